"""8-bit products and distillation on the GPU, at the edges of what their documentation settles: sums that cancel, values at
the ends of the range, rows without a finite logit, masses other than 1, operands inside wider buffers."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip('torch')

from oracle import lowbit  # noqa: E402
from test_gpu_lowbit import U, check_distill, logits, sum_error, teacher_of  # noqa: E402


@pytest.fixture(scope='module')
def ctx():
    from ocr_amd.engine import HipContext
    c = HipContext(0)
    yield c
    c.close()


# --------------------------------------------------------------------------------------- product
# few rows; tiles of 128; k in pieces; tiles of 256 (510 of them on 256 compute units, three blocks of k)
@pytest.mark.parametrize('out_dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('block_rows', [1, 128])
@pytest.mark.parametrize('mnk', [(1, 97, 16), (40, 70, 384), (64, 33, 1024), (200, 130, 384), (300, 97, 1280), (4100, 7600, 384)])
def test_products_that_cancel_leave_the_small_ones(ctx, mnk, block_rows, out_dtype):
    """Every group of 16 neighbours in k holds 448 * 448, its negative and one product i j, |i| <= 7, |j| <= 2, at places of
    their own.  All products are integers and every partial sum, in any order, is below K / 16 (448^2 + 14) < 2^24 for K up to
    1280: a float32 holds it, so the sums are exact and the result is the exact integer, rounded once."""
    m, n, k = mnk
    g = torch.Generator().manual_seed(m + n + k)
    groups = k // 16
    at = torch.stack([torch.randperm(16, generator=g)[:3] for _ in range(groups)]) + 16 * torch.arange(groups)[:, None]
    a, b = torch.zeros(m, k), torch.zeros(n, k)
    a[:, at[:, 0]], a[:, at[:, 1]], b[:, at[:, 0]], b[:, at[:, 1]] = 448.0, 448.0, 448.0, -448.0
    small_a = torch.randint(-7, 8, (m, groups), generator=g).float()
    small_b = torch.randint(-2, 3, (n, groups), generator=g).float()
    a[:, at[:, 2]], b[:, at[:, 2]] = small_a, small_b
    want = (small_a.cuda() @ small_b.cuda().t().contiguous()).to(out_dtype)      # integers: exact
    aq, bq = ctx.quantize_fp8(a.cuda()), ctx.quantize_fp8(b.cuda(), block_rows=block_rows)
    assert torch.equal(aq.q[:, :k].float().cpu(), a) and torch.equal(bq.q[:, :k].float().cpu(), b)
    assert torch.equal(ctx.gemm_fp8(aq, bq, out_dtype=out_dtype), want)
    if m <= 300:
        assert torch.equal(ctx.linear_fp8(a.cuda(), bq, out_dtype=out_dtype), want)
        assert torch.equal(ctx.linear_fp8(a.bfloat16().cuda(), bq, out_dtype=out_dtype), want)


def values_64(m):
    """Fp8Matrix -> its values in float64, on the GPU."""
    e = m.scale[:, :-(-m.rows // m.block_rows)].double().t() - 127
    row, col = torch.arange(m.rows, device='cuda') // m.block_rows, torch.arange(m.cols, device='cuda') // 128
    return m.q[:, :m.cols].double() * torch.exp2(e[row][:, col])


# Several blocks of k in workgroups that walk several tiles, the next tile's first block on its way while this one's last is
# multiplied and its results leave: 510 tiles of 256 on 256 compute units (bfloat16), 600 and 1256 tiles of 128 on 512 workgroups.
# Two blocks, three, five with a ragged last one; ragged last tiles in both directions.
@pytest.mark.parametrize('out_dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('block_rows', [1, 128])
@pytest.mark.parametrize('bias', [False, True])
@pytest.mark.parametrize('mnk', [(4100, 7600, 256), (4100, 7600, 384), (4100, 7600, 600), (3000, 3100, 256), (3000, 3100, 600), (20001, 999, 384)])
def test_products_of_many_tiles_and_blocks(ctx, mnk, bias, block_rows, out_dtype):
    """Every element against float64 on the GPU: float32 sums of K terms in any order, (K + 2) 2u sum |a b|, and for a bfloat16
    result half a step of that."""
    m, n, k = mnk
    g = torch.Generator().manual_seed(m + k)
    x = torch.randn(m, k, generator=g) * torch.exp2(torch.randint(-4, 5, (m, 1), generator=g).float())
    w = torch.randn(n, k, generator=g) * torch.exp2(torch.randint(-4, 5, (1, k), generator=g).float())
    a, b = ctx.quantize_fp8(x.cuda()), ctx.quantize_fp8(w.cuda(), block_rows=block_rows)
    v = torch.randn(n, generator=g).cuda() if bias else None
    got = ctx.gemm_fp8(a, b, bias=v, out_dtype=out_dtype)
    a64, b64 = values_64(a), values_64(b).t().contiguous()
    want, mass = a64 @ b64, a64.abs() @ b64.abs()
    if bias:
        want, mass = want + v.double(), mass + v.double().abs()
    tol = (k + 2) * 2 * U * mass
    if out_dtype == torch.bfloat16:
        tol = tol * 1.01 + 2.0 ** -8 * want.abs()
    assert bool(((got.double() - want).abs() <= tol).all())
    for _ in range(3):
        assert torch.equal(ctx.gemm_fp8(a, b, bias=v, out_dtype=out_dtype), got)


@pytest.mark.parametrize('out_dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('m', [5, 200])
def test_operand_values_at_the_ends_of_the_range(ctx, m, out_dtype):
    """Bytes times scale count as the bfloat16 number nearest to them, on either side: multiples of 2^-133 below 2^-126, infinite
    from 2^128 on, and exact between.  One value per row, the other operand a power of two."""
    from ocr_amd.engine import Fp8Matrix
    # byte and exponent of the scale: around 2^-126 and 2^-133 (ties, and bits that are lost), 2^-127 as a scale, around 2^128
    cases = [(0x08, -120), (0x04, -120), (0x0F, -120), (0x01, -117), (0x01, -124), (0x01, -125), (0x03, -125), (0x09, -127), (0x07, -127), (0x05, -126), (0x38, -126),
             (0x37, -126), (0x40, -127), (0x3D, -127), (0x7E, -127), (0x38, 127), (0x3F, 127), (0x40, 127), (0x7E, 119), (0x7E, 120), (0x78, 120), (0xB8, -126),
             (0x8F, -126), (0xC0, 127)]
    table = lowbit.e4m3_table()
    q = torch.zeros((m, 128), dtype=torch.uint8)
    scale = torch.full((1, -(-m // 16) * 16), 127, dtype=torch.uint8)
    for r in range(m):
        byte, e = cases[r % len(cases)]
        q[r, r % 128], scale[0, r] = byte, e + 127
    one = torch.zeros((3, 128), dtype=torch.uint8)
    one[:] = 0x38                                                     # 1
    # powers of two that bring every value to the middle of the range: 2^120 for the small ones, 2^-120 for the large
    other = Fp8Matrix(one.cuda().view(torch.float8_e4m3fn), torch.tensor([[247, 7, 127] + [127] * 13], dtype=torch.uint8).cuda(), 3, 128, 1)
    small = Fp8Matrix(q.cuda().view(torch.float8_e4m3fn), scale.cuda(), m, 128, 1)
    got = ctx.gemm_fp8(small, other, out_dtype=out_dtype).double().cpu()
    flipped = ctx.gemm_fp8(other, small, out_dtype=out_dtype).double().cpu()
    for r in range(m):
        byte, e = cases[r % len(cases)]
        n = 0 if e < 0 else 1
        value = torch.tensor(table[byte] * 2.0 ** e, dtype=torch.float64).float().bfloat16()           # (exact in float32)
        want = float(value) * 2.0 ** (120 if n == 0 else -120)
        assert got[r, n] == want and flipped[n, r] == want, (r, got[r, n], want)


@pytest.mark.parametrize('out_dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('block_rows', [1, 128])
@pytest.mark.parametrize('mnk', [(5, 40, 300), (65, 129, 300), (130, 67, 1000), (300, 97, 2048)])
def test_operands_are_the_last_columns_of_wider_buffers(ctx, mnk, block_rows, out_dtype):
    """Bytes and scales of both operands end where their buffers end; what lies in front are other columns (NaN)."""
    m, n, k = mnk
    g = torch.Generator().manual_seed(k)
    a = ctx.quantize_fp8(torch.randn(m, k, generator=g).cuda())
    w = ctx.quantize_fp8(torch.randn(n, k, generator=g).cuda(), block_rows=block_rows)

    def last_columns(t, wider):
        big = torch.full((t.shape[0], t.shape[1] + wider), 255, dtype=torch.uint8, device='cuda')
        big[:, wider:] = t.view(torch.uint8)
        return big[:, wider:]
    wide = [x._replace(q=last_columns(x.q, 256), scale=last_columns(x.scale, 944)) for x in (a, w)]
    assert torch.equal(ctx.gemm_fp8(*wide, out_dtype=out_dtype), ctx.gemm_fp8(a, w, out_dtype=out_dtype))


@pytest.mark.parametrize('out_dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('m', [5, 200])
def test_a_scale_of_255_makes_its_block_nan(ctx, m, out_dtype):
    """In the scales of either operand: that row or column of the product and nothing else, zeros in the block included."""
    a, b = ctx.quantize_fp8(torch.randn(m, 300).cuda()), ctx.quantize_fp8(torch.zeros(40, 300).cuda())
    a.scale[1, m // 2], b.scale[2, 7] = 255, 255
    bad = torch.isnan(ctx.gemm_fp8(a, b, out_dtype=out_dtype))
    assert bad[m // 2].all() and bad[:, 7].all() and int(bad.sum()) == 40 + m - 1


@pytest.mark.parametrize('block_rows', [1, 128])
@pytest.mark.parametrize('transpose', [False, True])
def test_quantise_beyond_32_bits(ctx, transpose, block_rows):
    """More than 2^31 elements in and bytes out: the first and last rows equal those of a matrix of their own."""
    rows, cols = 65536 + 256, 33000
    part = torch.randn(256, cols, generator=torch.Generator().manual_seed(1)).bfloat16().cuda()
    want = ctx.quantize_fp8(part, block_rows=block_rows, transpose=transpose)
    x = part.repeat(rows // 256, 1)
    assert x.numel() > 2 ** 31
    got = ctx.quantize_fp8(x, block_rows=block_rows, transpose=transpose)
    del x
    for first in (0, 256 * (rows // 512), rows - 256):
        if transpose:
            assert torch.equal(got.q.view(torch.uint8)[:, first:first + 256], want.q.view(torch.uint8))
            assert torch.equal(got.scale[first // 128:first // 128 + 2, :-(-cols // block_rows)], want.scale[:, :-(-cols // block_rows)])
        else:
            blocks = 256 // block_rows
            assert torch.equal(got.q.view(torch.uint8)[first:first + 256], want.q.view(torch.uint8))
            assert torch.equal(got.scale[:, first // block_rows:first // block_rows + blocks], want.scale[:, :blocks])


# ---------------------------------------------------------------------------------- distillation
# one row length for each form: 16, 32 and 64 lanes a row, a row in LDS on one wave and on four, a row read twice
FORMS = [(97, 6), (97, 30), (97, 50), (3, 3), (3, 20), (1000, 6), (6719, 6), (40000, 6)]


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('v,k', FORMS)
@pytest.mark.filterwarnings('ignore:invalid value encountered in subtract')      # the tolerance's own p_rest of those rows
def test_a_teacher_row_without_a_finite_logit(ctx, v, k, dtype):
    """What ocrhip_top_logits returns for it (entries and log normaliser -infinity): entries without probability, so with the
    normaliser everything lies outside them, and without it the row counts nothing."""
    t = 2.0
    x = logits(4, v, v, dtype).cuda()
    teacher = logits(4, v, v + 1).cuda()
    teacher[1:3] = -float('inf')
    n = min(k, v)
    z, i, lse = ctx.top_logits(teacher, n, temperature=t)
    assert (z[1:3] == -float('inf')).all() and (lse[1:3] == -float('inf')).all()
    if n < k:
        z = torch.cat([z, torch.zeros(4, k - n, device='cuda')], 1)
        i = torch.cat([i, torch.full((4, k - n), -1, dtype=torch.int32, device='cuda')], 1)
    for l in (lse, None):
        out = check_distill(ctx, x, z, i, l, t, None)
        assert torch.isfinite(out['loss']).all() and torch.isfinite(out['grad'].float()).all()
        assert l is not None or not (out['loss'][1:3].any() or out['grad'][1:3].any())


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('v,k', [f for f in FORMS if f[1] < f[0]])
def test_a_nan_next_to_a_rest_without_mass(ctx, v, k, dtype):
    """Nothing finite outside the entries and p_rest > 0: an infinite loss, but NaN with a NaN or +infinity among the student's
    logits or the teacher's entries."""
    x = torch.full((6, v), -float('inf'))
    z, i = torch.zeros(6, k), torch.arange(k, dtype=torch.int32).repeat(6, 1)
    x[:, :k] = torch.randn(6, k, generator=torch.Generator().manual_seed(v + k))
    lse = torch.full((6,), float(torch.log(torch.tensor(float(k)))) + 1.0)
    x[1, k - 1], z[2, 0], x[3, 0], z[4, k // 2] = float('nan'), float('nan'), float('inf'), float('inf')
    x[5, v - 1] = float('nan')
    out = ctx.distill_loss(x.to(dtype).cuda(), z.cuda(), i.cuda(), top_lse=lse.cuda(), want_grad=True)
    assert out['loss'][0] == float('inf') and torch.isnan(out['loss'][1:]).all()
    assert not torch.isnan(out['grad'][0]).any() and torch.isnan(out['grad'][1:]).all()


@pytest.mark.parametrize('v,k', FORMS)
def test_extreme_temperatures(ctx, v, k):
    """At 4.3e-39 only the largest logit is left, at 3e38 all are alike: log sum exp(x / t) = max / t and log V, to half a step; the
    gradient t (q - p) has no NaN."""
    k = min(k, v)
    x = torch.zeros(2, v)
    x[0, v // 2], x[1, v - 1] = 1.0, 0.5
    for t in (4.3e-39, 3e38):
        for dtype in (torch.float32, torch.bfloat16):
            val, idx, lse = ctx.top_logits(x.to(dtype).cuda(), k, temperature=t)
            assert idx[:, 0].tolist() == [v // 2, v - 1] and val[:, 0].tolist() == [1.0, 0.5]
            want = torch.tensor([1.0, 0.5]).double() / torch.tensor(t).double() if t < 1 else torch.full((2,), v).double().log()
            assert ((lse.cpu().double() - want).abs() <= 2.0 ** -22 * want).all()       # exp and sum 2^-23 of 1 + log V each, the store
            out = ctx.distill_loss(x.to(dtype).cuda(), val, idx, top_lse=lse, temperature=t, want_grad=True)
            assert not torch.isnan(out['loss']).any() and not torch.isnan(out['grad'].float()).any()


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('v,k', FORMS + [(33, 33), (64, 64)])
def test_gradient_where_the_mass_is_not_1(ctx, v, k, dtype):
    """A log normaliser too large and too small (p of more than 1 in all, no rest), and every class named: the gradient is the
    derivative of the loss, against the formula and against differences.

    Against the formula: q is off by q (eps + eps_v) relative to itself, times the mass P, as in check_distill.  Against
    differences along d of 0 and +-1, h = 2^-6 (s + h d exact): h^2 / 6 times a third derivative of at most 2 P, the two losses off
    by 2u of theirs and P times the error of the logarithm each, the gradient's own error along d."""
    t, h = 1.0, 2.0 ** -6
    n = min(k, v)
    x = (logits(6, v, v).cuda() * 8).round().div(8).to(dtype)          # few bits: s + h d is exact in float32
    z, i, lse = teacher_of(ctx, x, n, t, 7)
    lse = lse + torch.tensor([0.0, 0.5, -0.5, -1.5, -3.0, 2.0], device='cuda')
    if n < k:
        z = torch.cat([z, torch.zeros(6, k - n, device='cuda')], 1)
        i = torch.cat([i, torch.full((6, k - n), -1, dtype=torch.int32, device='cuda')], 1)
    out = ctx.distill_loss(x, z, i, top_lse=lse, temperature=t, want_grad=True)
    s64, z64, i64, l64 = x.double().cpu().numpy(), z.double().cpu().numpy(), i.cpu().numpy(), lse.cpu().numpy()
    loss, grad = lowbit.distill(s64, z64, i64, l64, t, None)
    mass = np.where(i64 >= 0, np.exp(z64 - l64[:, None].astype(np.float64)), 0.0).sum(1)
    full = np.maximum(mass, 1.0) if n < v else mass
    rest = np.maximum(0.0, 1.0 - mass) if n < v else 0.0 * mass
    e = np.exp(s64 - s64.max(1, keepdims=True))
    q = e / e.sum(1, keepdims=True)
    inside = np.zeros((6, v + 1), dtype=bool)
    np.put_along_axis(inside, np.where(i64 >= 0, i64, v).astype(np.int64), True, 1)
    q_rest = np.where(inside[:, :v], 0.0, q).sum(1)
    ratio = rest / np.where(q_rest > 0, q_rest, 1.0)
    eps = sum_error(v)
    assert (np.abs(out['loss'].double().cpu().numpy() - loss) <= full * eps * 2 + 2 * U * np.abs(loss)).all()
    own = 4 * U * (s64.max(1, keepdims=True) - s64) + 2.0 ** -22
    half = 2.0 ** -8 * 1.01 if dtype == torch.bfloat16 else 0.0
    tol = q * (full + ratio)[:, None] * (2 * eps + own + 4 * U) + (half + 2 * U) * np.abs(grad) + 1e-37
    assert (np.abs(out['grad'].double().cpu().numpy() - grad) <= tol).all()
    if dtype == torch.float32:
        d = (torch.randint(0, 3, x.shape, generator=torch.Generator().manual_seed(9)) - 1).float().cuda()
        up = ctx.distill_loss(x + h * d, z, i, top_lse=lse, temperature=t)['loss'].double().cpu().numpy()
        down = ctx.distill_loss(x - h * d, z, i, top_lse=lse, temperature=t)['loss'].double().cpu().numpy()
        slope = (out['grad'].double() * d).sum(1).cpu().numpy()
        tol = h * h / 6 * 2 * full + (2 * U * (np.abs(up) + np.abs(down)) + 4 * full * eps) / (2 * h) + 4 * full * eps
        assert (np.abs((up - down) / (2 * h) - slope) <= tol).all()


@pytest.mark.parametrize('rest', [False, True])
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('v,k', [f for f in FORMS if f[1] > 3])
def test_entries_of_one_class_add_up(ctx, v, k, dtype, rest):
    """Classes named several times - next to each other, far apart, by entries without probability, by every entry - count with
    their whole probability; a student that agrees with the teacher's classes has the loss of its rest alone."""
    x = logits(6, v, v, dtype).cuda()
    z, i, lse = teacher_of(ctx, x, min(k, v), 1.0, 3)
    if v < k:
        z = torch.cat([z, z[:, :1].expand(6, k - v)], 1).contiguous()
        i = torch.cat([i, i[:, :1].expand(6, k - v)], 1).contiguous()
    i[1, 1] = i[1, 0]
    i[2, k - 1] = i[2, 0]
    i[3] = i[3, 0].item()
    i[4, 1], z[4, 0] = i[4, 0], -float('inf')
    i[5, 1], i[5, 3] = i[5, 0], i[5, 2]
    top = x.float().gather(1, i[:, :1].long())[5, 0]
    x[5] = -30.0
    z[5] = -40.0                                               # row 5: all mass on one class, half of it in each of two entries
    z[5, :2], x[5, i[5, 0].long()] = top - 0.6931472, top.to(dtype)
    lse = torch.logsumexp(z, 1) + 0.1                          # p of less than 1 whatever the entries name
    out = check_distill(ctx, x, z, i, lse if rest else None, 1.0, None)
    if not rest:
        # p = q = 1 but for what 29 times exp(-70) and log 2's rounding leave; each of the two alone would give -log 2
        assert abs(float(out['loss'][5])) < 1e-6


@pytest.mark.parametrize('v', [4000, 8000, 20001, 262144])
def test_small_probabilities_beside_a_large_one_are_not_lost(ctx, v):
    """One class at 0 and all others at -16.75, 2^-24.2 of it each: added to 1 one by one in float32 they are all lost.  The
    largest class's gradient is 1 / S, S = 1 + (V - 1) e^-16.75: S may lose the up to 31 that share a float32 sum with the 1
    (2^-24.1 each), its other terms are off by 2^-22 and 4u * 16.75 of themselves, and the gradient by 4u for its roundings."""
    x = torch.full((3, v), -16.75)
    i = torch.tensor([[v - 1], [1], [v // 2]], dtype=torch.int32)
    for r, at in enumerate((0, v - 1, v // 3)):
        x[r, at] = 0.0
    out = ctx.distill_loss(x.cuda(), torch.zeros(3, 1).cuda(), i.cuda(), want_grad=True)
    small = np.exp(-16.75)
    s = 1.0 + (v - 1) * small
    tol = 31 * small + (s - 1) * (2.0 ** -22 + 4 * U * 16.75) + 4 * U
    tol = tol if v > 8192 else tol - 24 * small                  # rows in LDS: 4 classes share one
    for r, at in enumerate((0, v - 1, v // 3)):
        assert abs(float(out['grad'][r, at]) - 1.0 / s) <= tol, (r, float(out['grad'][r, at]) - 1.0 / s, tol)


@pytest.mark.parametrize('v,k', [(4000, 8), (8000, 8), (500, 64), (20001, 8), (262144, 64)])
def test_log_normaliser_of_small_probabilities_beside_a_large_one(ctx, v, k):
    """The same rows: log S, S = 1 + (V - 1) e^-16.75, off by what S is off by relative to itself and half a step of the store."""
    x = torch.full((3, v), -16.75)
    for r, at in enumerate((0, v - 1, v // 3)):
        x[r, at] = 0.0
    small = np.exp(-16.75)
    s = 1.0 + (v - 1) * small
    tol = (31 if v > 8192 else 7) * small + (s - 1) * (2.0 ** -22 + 4 * U * 16.75) + U * np.log(s)
    for dtype in (torch.float32, torch.bfloat16):                 # -16.75 has six bits
        lse = ctx.top_logits(x.to(dtype).cuda(), k)[2].double().cpu().numpy()
        assert (np.abs(lse - np.log(s)) <= tol).all(), (lse - np.log(s), tol)
