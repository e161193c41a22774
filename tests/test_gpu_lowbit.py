"""8-bit products and distillation on the GPU against the plain float64 forms (oracle/lowbit.py).

Tolerances (u = 2^-24, half a float32 step relative to the value):
  * quantised bytes and exponents are determined: equal.
  * products: every product of two e4m3 values is exact in float32; a float32 sum of K terms in any order is off by at most
    (K - 1) * 2u * sum |a b| (2u: an adder that truncates), the bias addition and the store by u each, a bfloat16 store by
    2^-8 relative to the value.  For a bfloat16 result the matrix instruction drops from every product what lies 2^-13 below
    the largest of its group of at most 16 neighbours in k (documented at ocrhip_gemm_fp8): 16 * 2^-13 * max |a| * max |b|
    per group.
  * sums of exponentials: the argument (a difference, times 1 / temperature and log2 e: four roundings) is off by 4u |arg|,
    exp by 2^-22, a chain of n float32 additions by n u; relative to the sum that is
    eps = u (4 (ln V + 1) + n) + 2^-22, the mean of |arg| under the distribution being at most ln V + 1.
    n = V / 16 up to 2048 classes and V / 64 + 64 beyond: the fewest lanes that share a row.
  * loss: an error of that sum enters with the factor q_rest - p_rest; what enters to first order is float64; u for the store.
  * gradient: q_v is off by q_v (eps + eps_v), eps_v the error of its own exponential, p_rest / q_rest of q_v likewise.
"""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip('torch')

from oracle import lowbit  # noqa: E402

U = 2.0 ** -24


@pytest.fixture(scope='module')
def ctx():
    from ocr_amd.engine import HipContext
    c = HipContext(0)
    yield c
    c.close()


def values(rows, cols, seed, dtype=torch.float32):
    """Columns of different scale, rows of zeros, large and tiny values."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, cols, generator=g) * torch.exp2(torch.randint(-6, 7, (cols,), generator=g).float())
    x[torch.rand(rows, generator=g) < 0.1] = 0.0
    x[torch.rand(rows, cols, generator=g) < 0.01] *= 1000.0
    return x.to(dtype)


def parts(m):
    """Fp8Matrix -> (values (rows, padded cols), exponents (row blocks, column blocks))."""
    rb = -(-m.rows // m.block_rows)
    return (lowbit.e4m3_table()[m.q.view(torch.uint8).cpu().numpy()], m.scale[:, :rb].cpu().numpy().astype(np.int64).T - 127)


# -------------------------------------------------------------------------------------- quantise
@pytest.mark.parametrize('transpose', [False, True])
@pytest.mark.parametrize('block_rows', [1, 128])
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('shape', [(1, 1), (1, 128), (3, 97), (17, 256), (130, 300), (257, 129), (64, 1030), (300, 64), (5, 2500)])
def test_quantise_is_the_definition(ctx, shape, dtype, block_rows, transpose):
    x = values(*shape, seed=shape[0] * 1000 + shape[1], dtype=dtype)
    m = ctx.quantize_fp8(x.cuda(), block_rows=block_rows, transpose=transpose)
    ref = (x.t() if transpose else x).double().numpy()
    q, e = lowbit.quantize(ref, block_rows)
    got_q, got_e = parts(m)
    assert (m.rows, m.cols) == ref.shape and got_q.shape[1] % 128 == 0
    np.testing.assert_array_equal(got_e, e)
    np.testing.assert_array_equal(got_q[:, :m.cols], q)
    assert not m.q.view(torch.uint8)[:, m.cols:].any()          # zero behind the last column


@pytest.mark.parametrize('transpose', [False, True])
@pytest.mark.parametrize('block_rows', [1, 128])
def test_quantise_special_values(ctx, block_rows, transpose):
    x = values(140, 260, 5)
    x[3, 5], x[3, 200], x[60, 7], x[61, :128] = float('nan'), float('inf'), -float('inf'), float('nan')
    x[70, :128] = 2.0 ** -140                                    # subnormal block (scale clamped at 2^-127)
    x[71, :128] = 3.4028234e38
    x[72, 128:256] = torch.linspace(-1, 1, 128) * 2.0 ** -126
    x[73, 128:256] = -0.0
    x[74, :128] = torch.tensor([448.0, -448.0, 17.0, 19.0, 2.0 ** -9, 2.0 ** -10, 3 * 2.0 ** -10, 432.0] * 16)       # ties
    x[75, :128] = torch.tensor([1.75, 1.7500001] * 64)
    m = ctx.quantize_fp8(x.cuda(), block_rows=block_rows, transpose=transpose)
    q, e = lowbit.quantize((x.t() if transpose else x).double().numpy(), block_rows)
    got_q, got_e = parts(m)
    np.testing.assert_array_equal(got_e, e)
    np.testing.assert_array_equal(got_q[:, :m.cols], q)


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('transpose', [False, True])
def test_quantise_strides_and_offsets(ctx, dtype, transpose):
    """Row strides beyond the columns, bases off every alignment, permuted and expanded views."""
    big = values(50, 700, 6, dtype).cuda()
    for view in (big[:, 3:300], big[5:, 1:130], big[::3, 7:500], big[7:8, 11:400], big.t(), big[0].expand(20, 700), big.view(10, 5, 700)[:, 2],
                 big.view(10, 5, 700), big[2, 5:300], big[:, ::2]):
        m = ctx.quantize_fp8(view, transpose=transpose)
        ref = view.reshape(-1, view.shape[-1])
        q, e = lowbit.quantize((ref.t() if transpose else ref).double().cpu().numpy(), 1)
        got_q, got_e = parts(m)
        np.testing.assert_array_equal(got_e, e)
        np.testing.assert_array_equal(got_q[:, :m.cols], q)


def test_quantise_leaves_what_is_not_its_own(ctx):
    """Rows behind the last, bytes between the rounded columns and the row stride, scales behind the last block."""
    import ctypes
    x = values(5, 200, 7).cuda()
    q = torch.full((7, 512), 0xAB, dtype=torch.uint8, device='cuda')
    sc = torch.full((3, 32), 0xCD, dtype=torch.uint8, device='cuda')
    from ocr_amd._lib import check
    p = lambda t: ctypes.c_void_p(t.data_ptr())
    check(ctx.lib.ocrhip_quantize_fp8(ctx._h, p(x), 0, 5, 200, 200, 1, 0, p(q), 512, p(sc), 32, ctx._on()))
    q, sc = q.cpu().numpy(), sc.cpu().numpy()
    assert (q[5:] == 0xAB).all() and (q[:, 256:] == 0xAB).all() and (q[:5, 200:256] == 0).all()
    assert (sc[2:] == 0xCD).all() and (sc[:, 5:] == 0xCD).all() and (sc[:2, :5] != 0xCD).all()


def test_empty_inputs(ctx):
    m = ctx.quantize_fp8(torch.empty(0, 200, device='cuda'))
    assert m.q.shape == (0, 256) and m.rows == 0
    w = ctx.quantize_fp8(values(7, 200, 8).cuda(), block_rows=128)
    assert ctx.gemm_fp8(m, w).shape == (0, 7)
    assert ctx.gemm_fp8(ctx.quantize_fp8(values(3, 200, 8).cuda()), ctx.quantize_fp8(torch.empty(0, 200, device='cuda'))).shape == (3, 0)
    assert ctx.linear_fp8(torch.empty(2, 0, 200, device='cuda'), w).shape == (2, 0, 7)
    v, i, l = ctx.top_logits(torch.empty(0, 97, device='cuda'), 5)
    assert v.shape == (0, 5) and i.shape == (0, 5) and l.shape == (0,)
    out = ctx.distill_loss(torch.empty(0, 97, device='cuda'), v, i, want_grad=True)
    assert out['loss'].shape == (0,) and out['grad'].shape == (0, 97)


# --------------------------------------------------------------------------------------- product
def check_product(got, a, w, bias, out_dtype):
    av = lowbit.dequantize(parts(a)[0][:, :a.cols], parts(a)[1], a.block_rows)
    wv = lowbit.dequantize(parts(w)[0][:, :w.cols], parts(w)[1], w.block_rows)
    ref, mass = av @ wv.T, np.abs(av) @ np.abs(wv).T
    if bias is not None:
        b = bias.double().cpu().numpy()
        ref, mass = ref + b, mass + np.abs(b)
    tol = (a.cols + 2) * 2 * U * mass
    if out_dtype == torch.bfloat16:
        group = lambda v: np.abs(np.pad(v, ((0, 0), (0, -v.shape[1] % 16)))).reshape(v.shape[0], -1, 16).max(2)   # noqa: E731
        tol = tol * 1.01 + 2.0 ** -8 * np.abs(ref) * 1.01 + 16 * 2.0 ** -13 * (group(av) @ group(wv).T)
    err = np.abs(got.double().cpu().numpy() - ref)
    assert got.dtype == out_dtype and got.shape == ref.shape
    worst = float((err / (tol + 1e-37)).max())
    assert worst <= 1, 'worst error %g of the tolerance' % worst


SIZES = [(1, 1, 1), (1, 97, 256), (2, 6719, 256), (16, 16, 128), (17, 33, 129), (63, 97, 256), (5, 300, 1000), (64, 64, 64), (65, 129, 640),
         (128, 256, 512), (200, 97, 97), (257, 255, 130), (300, 520, 384), (1000, 40, 256), (33, 1024, 2048), (130, 260, 4100), (515, 513, 127)]


@pytest.mark.parametrize('out_dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('block_rows', [1, 128])
@pytest.mark.parametrize('mnk', SIZES)
def test_product(ctx, mnk, block_rows, out_dtype):
    m, n, k = mnk
    a = ctx.quantize_fp8(values(m, k, m + n).cuda())
    w = ctx.quantize_fp8(values(n, k, m + k).cuda() * 0.05, block_rows=block_rows)
    bias = torch.randn(n, generator=torch.Generator().manual_seed(n)).cuda() if (m + n) % 2 else None
    got = ctx.gemm_fp8(a, w, bias=bias, out_dtype=out_dtype)
    check_product(got, a, w, bias, out_dtype)
    assert torch.equal(got, ctx.gemm_fp8(a, w, bias=bias, out_dtype=out_dtype))          # one order of the sums


@pytest.mark.parametrize('out_dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('mnk', [(65, 64, 66000), (130, 40, 20000), (300, 97, 2048), (100, 97, 512), (65, 1, 300000)])
def test_product_of_few_tiles_and_many_blocks(ctx, mnk, out_dtype):
    """k in pieces: a few, and more than the 16 of one batch of the join; a last piece that is shorter."""
    m, n, k = mnk
    a = ctx.quantize_fp8(values(m, k, k).cuda())
    w = ctx.quantize_fp8(values(n, k, n).cuda() * 0.05, block_rows=128)
    bias = torch.randn(n, generator=torch.Generator().manual_seed(n)).cuda()
    got = ctx.gemm_fp8(a, w, bias=bias, out_dtype=out_dtype)
    check_product(got, a, w, bias, out_dtype)
    assert torch.equal(got, ctx.gemm_fp8(a, w, bias=bias, out_dtype=out_dtype))


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('mnk', [(1, 6719, 256), (1, 1, 1), (3, 97, 256), (16, 300, 200), (17, 129, 97), (40, 4096, 1000), (64, 256, 512), (8, 64, 8192),
                                 (300, 97, 512), (2, 40, 20000), (32, 97, 512), (32, 97, 513), (17, 40, 1000)])
def test_linear_equals_quantise_and_product(ctx, mnk, dtype):
    m, n, k = mnk
    x = values(m, k, k + 1, dtype).cuda()
    w = ctx.quantize_fp8(values(n, k, 3).cuda() * 0.05, block_rows=128)
    bias = torch.randn(n, generator=torch.Generator().manual_seed(n)).cuda()
    got = ctx.linear_fp8(x, w, bias=bias)
    a = ctx.quantize_fp8(x)
    check_product(got, a, w, bias, torch.float32)
    for by in (1, 128):
        w2 = ctx.quantize_fp8(values(n, k, 3).cuda() * 0.05, block_rows=by)
        check_product(ctx.linear_fp8(x, w2, out_dtype=torch.bfloat16), a, w2, None, torch.bfloat16)


def test_linear_takes_batches_and_strided_rows(ctx):
    w = ctx.quantize_fp8(values(97, 256, 4).cuda(), block_rows=128)
    x = values(60, 700, 9).cuda()
    for view in (x[:, 3:259], x.view(4, 15, 700)[:, :, 100:356], x[5, 1:257], x[:1, 2:258], x[::7, :256]):
        got = ctx.linear_fp8(view, w)
        assert got.shape == view.shape[:-1] + (97,)
        assert torch.equal(got.view(-1, 97), ctx.linear_fp8(view.reshape(-1, 256).contiguous(), w))


@pytest.mark.parametrize('m', [1, 20, 300])
def test_product_scales_over_the_whole_range(ctx, m):
    """Exponents far apart between rows, blocks and operands, from 2^-127 on; sums that leave float32 are infinite."""
    g = torch.Generator().manual_seed(m)
    x = torch.randn(m, 512, generator=g) * torch.exp2(torch.randint(-60, 61, (m, 4), generator=g).float()).repeat_interleave(128, 1)
    w = torch.randn(70, 512, generator=g) * torch.exp2(torch.randint(-40, 41, (70, 4), generator=g).float()).repeat_interleave(128, 1)
    a, b = ctx.quantize_fp8(x.cuda()), ctx.quantize_fp8(w.cuda())
    check_product(ctx.gemm_fp8(a, b), a, b, None, torch.float32)
    a = ctx.quantize_fp8((torch.ones(m, 128) * 2.0 ** 100).cuda())
    b = ctx.quantize_fp8((torch.ones(3, 128) * torch.tensor([[2.0 ** 100], [2.0 ** -100], [-2.0 ** 100]])).cuda())
    got = ctx.gemm_fp8(a, b).cpu()
    assert (got[:, 0] == float('inf')).all() and (got[:, 1] == 128.0).all() and (got[:, 2] == -float('inf')).all()


@pytest.mark.parametrize('m', [1, 40, 300])
def test_nan_stays_in_its_row_and_column(ctx, m):
    x, w = values(m, 300, 1).cuda(), values(70, 300, 2).cuda()
    x[m // 2, 299], w[69, 1] = float('nan'), float('inf')
    got = ctx.gemm_fp8(ctx.quantize_fp8(x), ctx.quantize_fp8(w))
    bad = torch.isnan(got)
    assert bad[m // 2].all() and bad[:, 69].all() and int(bad.sum()) == 70 + m - 1
    assert torch.equal(torch.isnan(ctx.linear_fp8(x, ctx.quantize_fp8(w))), bad)


def test_product_leaves_what_is_not_its_own(ctx):
    """Rows behind the last and columns between N and the row stride of the output; operands with a longer row stride;
    bytes of an operand's last rows that another matrix shares."""
    import ctypes
    from ocr_amd._lib import check
    p = lambda t: ctypes.c_void_p(t.data_ptr())
    for m, n, k in ((3, 33, 200), (70, 97, 256), (300, 130, 130)):
        a, w = ctx.quantize_fp8(values(m, k, 1).cuda()), ctx.quantize_fp8(values(n, k, 2).cuda(), block_rows=128)
        for out_dtype, code in ((torch.float32, 0), (torch.bfloat16, 1)):
            aq = torch.full((m + 2, 512), 0x7F, dtype=torch.uint8, device='cuda')
            aq[:m, :a.q.shape[1]] = a.q.view(torch.uint8)
            asc = torch.full((a.scale.shape[0], a.scale.shape[1] + 16), 255, dtype=torch.uint8, device='cuda')
            asc[:, :m] = a.scale[:, :m]
            out = torch.full((m + 2, n + 5), -7.0, dtype=out_dtype, device='cuda')
            ws_bytes = ctx.lib.ocrhip_gemm_fp8_workspace(m, n, k)
            ws = torch.empty(max(1, ws_bytes), dtype=torch.uint8, device='cuda')
            check(ctx.lib.ocrhip_gemm_fp8(ctx._h, p(aq), 512, p(asc), asc.shape[1], p(w.q), w.q.shape[1], p(w.scale), w.scale.shape[1], 128, m, n, k, None,
                                          p(out), code, n + 5, p(ws), ws_bytes, ctx._on()))
            assert torch.equal(out[:m, :n], ctx.gemm_fp8(a, w, out_dtype=out_dtype))
            assert (out[m:] == -7).all() and (out[:, n:] == -7).all()


# rows that start anywhere in a line, results that start anywhere, several tiles of a row per workgroup (2 and 14 for the last
# two), few rows and columns, and whole lines: the same sums wherever they are put, and nothing beside them
@pytest.mark.parametrize('out_dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('block_rows', [1, 128])
@pytest.mark.parametrize('mnk', [(65, 129, 128), (100, 160, 300), (129, 300, 128), (300, 520, 256), (200, 1000, 256), (130, 6719, 128),
                                 (2000, 6719, 128), (17000, 6719, 64)])
def test_product_lands_in_any_rows(ctx, mnk, block_rows, out_dtype):
    import ctypes
    from ocr_amd._lib import check
    m, n, k = mnk
    code, e = (0, 4) if out_dtype == torch.float32 else (1, 2)
    a = ctx.quantize_fp8(torch.randn(m, k, generator=torch.Generator().manual_seed(m)).cuda())
    w = ctx.quantize_fp8(torch.randn(n, k, generator=torch.Generator().manual_seed(n)).cuda(), block_rows=block_rows)
    bias = torch.randn(n, generator=torch.Generator().manual_seed(k)).cuda()
    ws_bytes = ctx.lib.ocrhip_gemm_fp8_workspace(m, n, k)
    ws = torch.empty(max(1, ws_bytes), dtype=torch.uint8, device='cuda')

    def run(ld, first):
        buf = torch.full((first + (m + 1) * ld,), -7.0, dtype=out_dtype, device='cuda')
        p = lambda t: ctypes.c_void_p(t.data_ptr())          # noqa: E731
        check(ctx.lib.ocrhip_gemm_fp8(ctx._h, p(a.q), a.q.shape[1], p(a.scale), a.scale.shape[1], p(w.q), w.q.shape[1], p(w.scale), w.scale.shape[1],
                                      block_rows, m, n, k, p(bias), ctypes.c_void_p(buf.data_ptr() + first * e), code, ld, p(ws), ws_bytes, ctx._on()))
        rows = buf[first:].view(m + 1, ld)
        assert (buf[:first] == -7).all() and (rows[m] == -7).all() and (rows[:, n:] == -7).all()
        return rows[:m, :n]
    whole = run(-(-n // 64) * 64, 0)
    if m <= 300:
        check_product(whole, a, w, bias, out_dtype)
    for ld, first in ((n, 0), (n, 1), (n, 31), (n + 1, 0), (n + 3, 5), (-(-n // 64) * 64, 3)):
        assert torch.equal(run(ld, first), whole), (ld, first)


def test_product_beyond_32_bits(ctx):
    """A's bytes and C's elements lie beyond 2^31: the last rows equal those of a product of their own."""
    m, n, k = (1 << 24) + 300, 136, 128                       # A 2.1 GB, C 2.3 G elements (bfloat16)
    x = values(4096, k, 1).cuda()
    small = ctx.quantize_fp8(x)
    from ocr_amd.engine import Fp8Matrix
    reps = -(-m // 4096)
    q = small.q.view(torch.uint8).repeat(reps, 1)[:m].contiguous().view(torch.float8_e4m3fn)
    lds = (m + 15) // 16 * 16
    scale = torch.full((1, lds), 127, dtype=torch.uint8, device='cuda')
    scale[0, :m] = small.scale[0, :4096].repeat(reps)[:m]
    w = ctx.quantize_fp8(values(n, k, 2).cuda(), block_rows=128)
    got = ctx.gemm_fp8(Fp8Matrix(q, scale, m, k, 1), w, out_dtype=torch.bfloat16)
    want = ctx.gemm_fp8(small, w, out_dtype=torch.bfloat16)
    for first in (0, 4096 * 2048, 4096 * (m // 4096)):
        count = min(4096, m - first)
        assert torch.equal(got[first:first + count], want[:count])


# ------------------------------------------------------------------------------------ top logits
def logits(rows, v, seed, dtype=torch.float32, spread=2.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, v, generator=g) * spread
    x[torch.arange(rows), torch.randint(0, v, (rows,), generator=g)] += 10.0
    return x.to(dtype)


def sum_error(v):
    n = v / 16 if v <= 2048 else v / 64 + 64
    return U * (4 * (np.log(v) + 1) + n) + 2.0 ** -22


def check_top(ctx, x, k, t):
    got_v, got_i, got_l = ctx.top_logits(x, k, temperature=t)
    x64 = x.reshape(-1, x.shape[-1]).double().cpu().numpy()
    t = float(np.float32(t))
    val, idx, lse = lowbit.top_logits(x64, k, t)
    np.testing.assert_array_equal(got_i.cpu().numpy().reshape(-1, k), idx)
    np.testing.assert_array_equal(got_v.cpu().numpy().reshape(-1, k).astype(np.float64), val)
    # the result is a float32: what lies half a step beyond its largest, 2^128 (1 - 2^-25), rounds to infinity (a masked row
    # of the type's lowest value at a temperature below 1: -3.4e38 / 0.25 = -1.36e39)
    lse = np.where(np.abs(lse) >= 2.0 ** 128 * (1 - 2.0 ** -25), np.copysign(np.inf, lse), lse)
    got_l, fin = got_l.cpu().numpy().reshape(-1).astype(np.float64), np.isfinite(lse)
    np.testing.assert_array_equal(np.isnan(got_l), np.isnan(lse))
    np.testing.assert_array_equal(got_l[~fin & ~np.isnan(lse)], lse[~fin & ~np.isnan(lse)])
    high = np.abs(val[fin, 0]) / t
    assert (np.abs(got_l[fin] - lse[fin]) <= sum_error(x.shape[-1]) + 4 * U * high + 2 * U * np.abs(lse[fin])).all()


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('v,k', [(1, 1), (2, 2), (5, 5), (64, 64), (65, 10), (97, 10), (97, 64), (300, 1), (513, 16), (1000, 64), (2047, 33),
                                 (6719, 32), (20001, 64), (70000, 8), (262144, 64)])
def test_top_logits(ctx, v, k, dtype):
    check_top(ctx, logits(5 if v > 3000 else 37, v, v + k, dtype).cuda(), k, 1.0 if v % 2 else 2.5)


@pytest.mark.parametrize('v', [40, 97, 1000, 6719, 40000])
def test_top_logits_ties_masks_and_special_rows(ctx, v):
    """Constant rows, two values only, masked classes, rows without a finite logit, ascending and descending rows."""
    k = min(v, 37)
    x = torch.zeros(13, v)
    x[1] = -3.0
    x[2, ::3] = 1.0
    x[3] = -float('inf')
    x[4] = -float('inf')
    x[4, v // 2] = 2.0
    x[5] = torch.finfo(torch.float32).min
    x[5, 1::2] = -1.0
    x[6] = torch.arange(v) * 0.01
    x[7] = -torch.arange(v) * 0.01
    x[8, ::2] = -0.0
    x[9, v - 1], x[9, 0] = 5.0, 5.0
    x[10, v // 3:] = -float('inf')
    x[11] = torch.linspace(-1, 1, v).roll(v // 2)
    x[12, -k:] = 7.0
    check_top(ctx, x.cuda(), k, 1.0)
    check_top(ctx, x.bfloat16().cuda(), k, 1.0)


@pytest.mark.parametrize('v', [97, 6719, 40000])
def test_top_logits_with_nan_and_infinity(ctx, v):
    x = logits(4, v, 3)
    x[0, 5], x[0, v - 1] = float('nan'), -float('nan')
    x[1, 7] = float('inf')
    x[2] = float('nan')
    x[3, 9], x[3, 10] = float('inf'), float('nan')
    got_v, got_i, got_l = ctx.top_logits(x.cuda(), 8)
    val, idx, _ = lowbit.top_logits(x.double().numpy(), 8, 1.0)
    np.testing.assert_array_equal(got_i.cpu().numpy(), idx)
    np.testing.assert_array_equal(got_v.cpu().numpy().astype(np.float64), val)
    l = got_l.cpu()
    assert torch.isnan(l[0]) and l[1] == float('inf') and torch.isnan(l[2]) and torch.isnan(l[3])


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('v,k', [(1, 1), (3, 3), (4, 1), (7, 7), (8, 8), (9, 5), (16, 16), (17, 16), (40, 16), (97, 1), (97, 16), (127, 10), (128, 16),
                                 (17, 17), (40, 33), (65, 64), (97, 17), (97, 64), (128, 64), (129, 64), (129, 10)])
def test_top_logits_of_short_rows(ctx, v, k, dtype):
    """Up to 128 classes, and one more: one class far above the rest, equal values within a lane's classes and across lanes,
    masked classes, rows without a finite logit, infinities, zeros of both signs, NaN; and more rows than one pass of the
    grid holds."""
    g = torch.Generator().manual_seed(v * 100 + k)
    x = torch.randn(24, v, generator=g)
    x[0] = 0.0
    x[1] = torch.randint(0, 2, (v,), generator=g).float()
    x[2] = torch.arange(v).float()
    x[3] = -torch.arange(v).float()
    x[4] = -float('inf')
    x[5] = -float('inf')
    x[5, v // 2] = 1.0
    x[6, v - 1] = float('inf')
    x[7] = torch.finfo(dtype).min
    x[8, ::2] = torch.finfo(dtype).min
    x[9] = torch.where(torch.arange(v) % 2 == 0, 0.0, -0.0)
    x[10] = 3e38
    x[11] = torch.randint(-2, 3, (v,), generator=g).float() * 1e-40
    x[12, : v // 2 + 1] = 5.0
    x[13, v // 2:] = 5.0
    x[14, v // 3] = float('nan')
    x[15] = float('nan')
    x = x.to(dtype)
    for t in (1.0, 0.25):
        check_top(ctx, x.cuda(), k, t)
    many = x.cuda().repeat(1500, 1)[:35001]
    val, idx, lse = ctx.top_logits(many, k)
    want = ctx.top_logits(x.cuda(), k)
    for got, w in zip((val, idx, lse), want):
        w = w.repeat(1500, 1)[:35001] if w.dim() == 2 else w.repeat(1500)[:35001]
        assert torch.equal(got.nan_to_num(1e9) if got.is_floating_point() else got, w.nan_to_num(1e9) if w.is_floating_point() else w)


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('v,k', [(130, 20), (150, 32), (260, 64), (300, 20), (500, 64), (520, 64), (700, 64), (769, 64), (1500, 32), (3000, 64), (6719, 32), (9000, 64), (20000, 64)])
def test_top_logits_of_masked_rows(ctx, v, k, dtype):
    """Many classes at one low value, in rows of every length: fewer classes left than asked for, none, about as many, in one
    place and spread; two levels of equal values; equal values above and below the K-th; NaN among them."""
    g = torch.Generator().manual_seed(v + k)
    low = torch.finfo(dtype).min
    rows = []
    for left in (0, 1, k - 1, k, k + 1, 3 * k, v // 2, v - 1):
        for fill in (-float('inf'), low, 0.0):
            for spread in (False, True):
                r = torch.full((v,), fill)
                at = torch.randperm(v, generator=g)[:left] if spread else torch.arange(v - left, v)
                r[at] = torch.randn(len(at), generator=g)
                rows.append(r)
    levels = torch.zeros(6, v)
    levels[0, ::2] = 1.0
    levels[1, 3::7] = 1.0
    levels[2, :k // 2] = 2.0
    levels[2, v // 2:v // 2 + k] = 1.0
    levels[3] = torch.randint(0, 3, (v,), generator=g).float()
    levels[4, v // 2], levels[4, 1] = float('nan'), float('inf')
    levels[5] = -float('inf')
    levels[5, v - 1] = float('nan')
    x = torch.cat([torch.stack(rows), levels]).to(dtype)
    check_top(ctx, x.cuda(), k, 1.0)


def test_top_logits_strides_and_offsets(ctx):
    big = logits(60, 300, 4).cuda()
    for dt in (torch.float32, torch.bfloat16):
        b = big.to(dt)
        for view in (b[:, 3:100], b[1:, 1:298], b[::4, 5:], b.view(4, 15, 300)[:, :, :97], b[3, 7:], b.t(), b.view(4, 15, 300)):
            check_top(ctx, view, 9, 1.0)


# ---------------------------------------------------------------------------------- distillation
def teacher_of(ctx, x, k, t, seed):
    """Entries of a teacher near the student x (float64 math on the CPU), shuffled, with a few that are none."""
    g = torch.Generator().manual_seed(seed)
    tl = x.float().cpu() + 0.7 * torch.randn(x.shape, generator=g)
    z, i = torch.topk(tl, k)
    perm = torch.randperm(k, generator=g)
    lse = torch.logsumexp(tl.double() / t, -1).float()
    return z[:, perm].contiguous().cuda(), i[:, perm].to(torch.int32).contiguous().cuda(), lse.cuda()


def check_distill(ctx, x, z, i, lse, t, w, loose=1.0):
    out = ctx.distill_loss(x, z, i, top_lse=lse, temperature=t, row_weight=w, want_grad=True)
    V, K = x.shape[-1], z.shape[-1]
    s = x.reshape(-1, V).double().cpu().numpy()
    zz, ii = z.reshape(-1, K).double().cpu().numpy(), i.reshape(-1, K).cpu().numpy()
    ll = None if lse is None else lse.reshape(-1).cpu().numpy()
    ww = None if w is None else w.reshape(-1).cpu().numpy()
    t = float(np.float32(t))
    loss, grad = lowbit.distill(s, zz, ii, ll, t, ww)
    got_l = out['loss'].reshape(-1).double().cpu().numpy()
    got_g = out['grad'].reshape(-1, V).double().cpu().numpy()
    assert out['loss'].shape == x.shape[:-1] and out['grad'].shape == x.shape and out['grad'].dtype == x.dtype
    eps = sum_error(V)
    half = 2.0 ** -8 * 1.01 if x.dtype == torch.bfloat16 else 0.0
    for r in range(s.shape[0]):
        wr = 1.0 if ww is None else float(ww[r])
        if not np.isfinite(loss[r]) or not np.isfinite(grad[r]).all():
            assert np.array_equal(np.isnan(got_l[r]), np.isnan(loss[r])) and (np.isnan(loss[r]) or got_l[r] == loss[r])
            if np.isnan(loss[r]):
                assert np.isnan(grad[r]).all() and np.isnan(got_g[r]).all()
                continue
        if wr == 0:
            assert got_l[r] == 0 and not got_g[r].any()
            continue
        m = s[r].max()
        e = np.exp((s[r] - m) / t)
        q = e / e.sum()
        valid = ii[r][(ii[r] >= 0) & (ii[r] < V)]
        inside = np.zeros(V, dtype=bool)
        inside[valid] = True
        q_rest = q[~inside].sum()
        p_rest = 0.0
        if ll is not None and not inside.all():
            p_rest = max(0.0, 1.0 - np.exp(zz[r][(ii[r] >= 0) & (ii[r] < V)] / t - ll[r]).sum())
        if np.isfinite(loss[r]):
            tol = abs(wr) * t * t * (abs(q_rest - p_rest) * eps + eps * eps + 1e-13) + 2 * U * abs(loss[r])
            beyond = abs(loss[r]) > 3.4028235e38               # float32 (a mask of the type's lowest value)
            assert got_l[r] == np.inf if beyond else abs(got_l[r] - loss[r]) <= tol, (r, got_l[r], loss[r], tol)
        ratio = p_rest / q_rest if q_rest > 0 else 0.0
        own = 4 * U * np.abs(np.where(np.isfinite(s[r]), s[r] - m, 0.0)) / t + 2.0 ** -22
        tol = abs(wr) * t * q * (1 + ratio) * (2 * eps + own + 4 * U) + (half + 2 * U) * np.abs(grad[r]) + 1e-37 * max(1.0, abs(wr) * t)
        err = np.abs(got_g[r] - grad[r])
        assert (err <= tol).all(), (r, int((err - tol).argmax()), float((err / tol).max()))
    return out


@pytest.mark.parametrize('rest', [False, True])
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('v,k', [(1, 1), (2, 1), (5, 5), (65, 64), (97, 10), (97, 1), (130, 7), (97, 17), (97, 32), (128, 32), (97, 33), (128, 64), (20, 20), (33, 33), (513, 16), (1000, 64), (2047, 33), (2500, 4), (6719, 32),
                                 (20001, 64), (70000, 8), (262144, 64)])
def test_distillation(ctx, v, k, dtype, rest):
    rows = 3 if v > 3000 else 21
    t = 1.0 if v % 2 else 3.0
    x = logits(rows, v, v, dtype).cuda()
    z, i, lse = teacher_of(ctx, x, k, t, k)
    w = torch.rand(rows, generator=torch.Generator().manual_seed(1)).cuda()
    check_distill(ctx, x, z, i, lse if rest else None, t, w)


@pytest.mark.parametrize('rest', [False, True])
@pytest.mark.parametrize('v,k', [(97, 6), (97, 30), (97, 50), (128, 32), (1000, 6), (6719, 6), (40000, 6)])
def test_distillation_of_odd_rows(ctx, v, k, rest):
    """Entries that are none, classes named twice, entries without probability, rows without any, masked classes, a student
    without mass where the teacher has some, weights of 0 over NaN, rows on which both agree."""
    t = 2.0
    x = logits(16, v, v + 1).cuda()
    z, i, lse = teacher_of(ctx, x, k, t, 5)
    i[0, 2], i[0, 4] = -1, v                                   # none
    i[1, 1], z[1, 1] = i[1, 0].item(), z[1, 0].item()          # a class twice
    lse[1] = float(np.log(np.exp(z[1].cpu().double().numpy() / t).sum())) + 0.3
    i[2] = -1                                                  # a row without entries
    z[3] = -float('inf')                                       # entries without probability
    z[4, 0] = -float('inf')
    x[5, v // 2:] = -float('inf')                              # masked classes, some of them entries perhaps
    i[5] = torch.arange(k, dtype=torch.int32)
    x[6] = -float('inf')
    x[6, :k] = 1.0                                             # nothing finite outside the entries
    i[6] = torch.arange(k, dtype=torch.int32)
    lse[6] = float(np.log(np.exp(z[6].cpu().double().numpy() / t).sum()))
    x[7, i[7, 0].long()] = -float('inf')                       # q = 0 where p > 0
    x[8] = torch.finfo(torch.float32).min                      # the lowest value as a mask
    x[8, i[8].long()] = torch.randn(k, device='cuda')
    x[9, 3], x[10, i[10, 1].long()], x[11, 4] = float('nan'), float('nan'), float('inf')
    w = torch.ones(16, device='cuda')
    w[11], w[12] = 0.5, 0.0
    x[12] = float('nan')
    w[13] = -1.5
    z[14] = x[14, i[14].long()]
    lse[14] = torch.logsumexp(x[14].double() / t, 0).float()
    z[15] = z[15] + 100.0                                      # far beyond lse: p > 1, no rest
    lse[15] += 50.0
    if v > 97:
        x[9, 3], x[9, v - 1] = 0.0, float('nan')
    check_distill(ctx, x, z, i, lse if rest else None, t, w)
    y = x.bfloat16()
    y[8][y[8] == -float('inf')] = torch.finfo(torch.bfloat16).min
    check_distill(ctx, y, z, i, lse if rest else None, t, w)


def test_distillation_of_a_nan_entry_is_nan(ctx):
    x = logits(3, 97, 1).cuda()
    z, i, lse = teacher_of(ctx, x, 5, 1.0, 2)
    z[1, 3] = float('nan')
    for l in (None, lse):
        out = ctx.distill_loss(x, z, i, top_lse=l, want_grad=True)
        assert torch.isnan(out['loss']).tolist() == [False, True, False]
        assert torch.isnan(out['grad'][1]).all() and not torch.isnan(out['grad'][[0, 2]]).any()


@pytest.mark.parametrize('v', [97, 1000, 6719, 40000])
def test_distillation_without_a_teacher_is_zero_whatever_the_logits_are(ctx, v):
    x = logits(4, v, 1).cuda()
    x[0, 1], x[1, v - 1], x[2] = float('nan'), float('inf'), float('nan')
    z, i = torch.zeros(4, 3, device='cuda'), torch.full((4, 3), -1, dtype=torch.int32, device='cuda')
    i[3] = torch.arange(3, dtype=torch.int32)
    z[3] = -float('inf')
    out = ctx.distill_loss(x, z, i, want_grad=True)
    assert not out['loss'].any() and not out['grad'].any()


@pytest.mark.parametrize('rest', [False, True])
def test_distillation_where_teacher_and_student_nearly_agree(ctx, rest):
    """Losses of 1e-9 next to terms of order 1."""
    x = logits(8, 6719, 2).cuda()
    tl = x.double() + 3e-4 * torch.randn(x.shape, generator=torch.Generator().manual_seed(3)).cuda()
    z, i = torch.topk(tl, 40)
    lse = torch.logsumexp(tl, -1).float()
    check_distill(ctx, x, z.float(), i.to(torch.int32), lse if rest else None, 1.0, None)


def test_distillation_gradient_against_differences(ctx):
    """Directional derivatives: loss(s + h d) - loss(s - h d) over 2 h against grad . d.  h = 2^-6: the truncation is h^2 / 6
    times a third derivative of at most 2 |d|^3 per row (a softmax cumulant), the two losses are off by 2^-24 of theirs each
    plus the documented error, and s + h d is exact (d of 0 and +-1, s with few bits)."""
    for v, k, rest in ((97, 10, False), (97, 10, True), (6719, 32, True)):
        x = (logits(6, v, v).cuda() * 256).round() / 256
        z, i, lse = teacher_of(ctx, x, k, 1.0, 7)
        g = torch.Generator().manual_seed(9)
        d = (torch.randint(0, 3, x.shape, generator=g) - 1).float().cuda()
        h = 2.0 ** -6
        l = lse if rest else None
        up = ctx.distill_loss(x + h * d, z, i, top_lse=l)['loss'].double()
        down = ctx.distill_loss(x - h * d, z, i, top_lse=l)['loss'].double()
        out = ctx.distill_loss(x, z, i, top_lse=l, want_grad=True)
        slope = (out['grad'].double() * d).sum(1)
        tol = h * h / 6 * 2 + (2 * U * (up + down) + 2 * sum_error(v)) / (2 * h) + sum_error(v) * 4
        assert ((up - down) / (2 * h) - slope).abs().le(tol).all()


def test_distillation_parts_and_repeats(ctx):
    x = logits(50, 1000, 3).cuda()
    z, i, lse = teacher_of(ctx, x, 20, 1.0, 4)
    both = ctx.distill_loss(x, z, i, top_lse=lse, want_grad=True)
    only_loss = ctx.distill_loss(x, z, i, top_lse=lse)
    only_grad = ctx.distill_loss(x, z, i, top_lse=lse, want_loss=False, want_grad=True)
    again = ctx.distill_loss(x, z, i, top_lse=lse, want_grad=True)
    assert only_loss['grad'] is None and only_grad['loss'] is None
    assert torch.equal(both['loss'], only_loss['loss']) and torch.equal(both['grad'], only_grad['grad'])
    assert torch.equal(both['loss'], again['loss']) and torch.equal(both['grad'], again['grad'])


def test_distillation_strides_offsets_and_batches(ctx):
    big = logits(60, 300, 4).cuda()
    for dt in (torch.float32, torch.bfloat16):
        b = big.to(dt)
        for view in (b[:, 3:100], b[1:, 1:298], b[::4, 5:], b.view(4, 15, 300)[:, :, :97], b.view(4, 15, 300), b[3, 7:]):
            flat = view.reshape(-1, view.shape[-1])
            z, i, lse = teacher_of(ctx, flat, 6, 1.0, 8)
            z, i, lse = z.view(view.shape[:-1] + (6,)), i.view(view.shape[:-1] + (6,)), lse.view(view.shape[:-1])
            check_distill(ctx, view, z, i, lse, 1.0, None)


def test_distillation_leaves_what_is_not_its_own(ctx):
    import ctypes
    from ocr_amd._lib import check
    p = lambda t: ctypes.c_void_p(t.data_ptr())
    for v in (97, 1000, 6719, 40001):
        for dt, code in ((torch.float32, 0), (torch.bfloat16, 1)):
            for lead in (0, 1, 3, 5):                          # bases and strides off every alignment
                x = logits(5, v, 1, dt).cuda()
                z, i, lse = teacher_of(ctx, x, 4, 1.0, 2)
                want = ctx.distill_loss(x, z, i, want_grad=True)
                buf = torch.full((7 * (v + 3) + lead,), -7.0, dtype=dt, device='cuda')
                grad = buf[lead:].view(7, v + 3)
                loss = torch.full((7,), -7.0, device='cuda')
                check(ctx.lib.ocrhip_distill_loss(ctx._h, p(x), code, 5, v, v, p(z), p(i), 4, None, 1.0, None, p(loss), p(grad), v + 3, ctx._on()))
                assert torch.equal(grad[:5, :v], want['grad']) and torch.equal(loss[:5], want['loss'])
                assert (grad[5:] == -7).all() and (grad[:, v:] == -7).all() and (loss[5:] == -7).all() and (buf[:lead] == -7).all()


def test_logits_beyond_32_bits(ctx):
    """(rows, V) of more than 2^32 elements: the last rows equal those of calls of their own."""
    rows, v = 33000, 131073
    part = logits(64, v, 1, torch.bfloat16).cuda()
    x = torch.empty((rows, v), dtype=torch.bfloat16, device='cuda')
    for r in range(0, rows, 64):
        x[r:r + 64] = part[:min(64, rows - r)]
    z, i, lse = teacher_of(ctx, part, 8, 1.0, 2)
    reps = -(-rows // 64)
    tz, ti, tl = z.repeat(reps, 1)[:rows], i.repeat(reps, 1)[:rows], lse.repeat(reps)[:rows]
    out = ctx.distill_loss(x, tz, ti, top_lse=tl, want_grad=True)
    want = ctx.distill_loss(part, z, i, top_lse=lse, want_grad=True)
    assert torch.equal(out['loss'], want['loss'].repeat(reps)[:rows])
    for first in (0, 64 * 257, 64 * (rows // 64)):
        n = min(64, rows - first)
        assert torch.equal(out['grad'][first:first + n], want['grad'][:n])
    del out
    val, idx, l = ctx.top_logits(x, 5)
    wv, wi, wl = ctx.top_logits(part, 5)
    assert torch.equal(val, wv.repeat(reps, 1)[:rows]) and torch.equal(idx, wi.repeat(reps, 1)[:rows]) and torch.equal(l, wl.repeat(reps)[:rows])


def test_many_short_rows(ctx):
    """More rows than a launch has workgroups in one dimension of 65535."""
    x = logits(1000, 33, 6).cuda()
    z, i, lse = teacher_of(ctx, x, 3, 1.0, 2)
    want = ctx.distill_loss(x, z, i, want_grad=True)
    wv, wi, _ = ctx.top_logits(x, 4)
    wm = ctx.quantize_fp8(x)
    reps = 300
    out = ctx.distill_loss(x.repeat(reps, 1), z.repeat(reps, 1), i.repeat(reps, 1), want_grad=True)
    assert torch.equal(out['loss'], want['loss'].repeat(reps)) and torch.equal(out['grad'], want['grad'].repeat(reps, 1))
    val, idx, _ = ctx.top_logits(x.repeat(reps, 1), 4)
    assert torch.equal(val, wv.repeat(reps, 1)) and torch.equal(idx, wi.repeat(reps, 1))
    m = ctx.quantize_fp8(x.repeat(reps, 1))
    assert torch.equal(m.q.view(torch.uint8), wm.q.view(torch.uint8).repeat(reps, 1)) and torch.equal(m.scale[:, :1000 * reps], wm.scale[:, :1000].repeat(1, reps))


# ------------------------------------------------------------------------ together, streams, graphs
def step(ctx, x, w8, wt8, bias, z, i, lse, weight):
    """One training step of a class layer in 8 bits: logits, loss, gradients of the input and of the weight."""
    y = ctx.linear_fp8(x, w8, bias=bias)
    out = ctx.distill_loss(y, z, i, top_lse=lse, row_weight=weight, want_grad=True)
    g = out['grad']
    dx = ctx.gemm_fp8(ctx.quantize_fp8(g), wt8)
    dw = ctx.gemm_fp8(ctx.quantize_fp8(g, transpose=True), ctx.quantize_fp8(x, transpose=True))
    return y, out['loss'], g, dx, dw


def step_inputs(ctx, rows=300, v=97, k=256, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, k, generator=g).cuda()
    w = (torch.randn(v, k, generator=g) * k ** -0.5).cuda()
    bias = (torch.randn(v, generator=g) * 0.1).cuda()
    z, i, lse = ctx.top_logits(x @ w.t() + bias, 10)
    weight = torch.full((rows,), 1.0 / rows).cuda()
    return x, ctx.quantize_fp8(w, block_rows=128), ctx.quantize_fp8(w, block_rows=128, transpose=True), bias, z, i, lse, weight


@pytest.mark.parametrize('v', [97, 1000])
def test_a_training_step_of_the_class_layer(ctx, v):
    """Teacher: float32 class layer; student: the same in 8 bits.  Every stage against float64 on what the stage before gave."""
    x, w8, wt8, bias, z, i, lse, weight = step_inputs(ctx, v=v)
    y, loss, g, dx, dw = step(ctx, x, w8, wt8, bias, z, i, lse, weight)
    a = ctx.quantize_fp8(x)
    check_product(y, a, w8, bias, torch.float32)
    check_distill(ctx, y, z, i, lse, 1.0, weight)
    check_product(dx, ctx.quantize_fp8(g), wt8, None, torch.float32)
    check_product(dw, ctx.quantize_fp8(g, transpose=True), ctx.quantize_fp8(x, transpose=True), None, torch.float32)
    # the transposed weight holds the same numbers
    np.testing.assert_array_equal(lowbit.dequantize(parts(w8)[0][:, :w8.cols], parts(w8)[1], 128).T,
                                  lowbit.dequantize(parts(wt8)[0][:, :wt8.cols], parts(wt8)[1], 128))
    assert float(loss.sum()) >= 0.0


def test_graph_capture_and_replays(ctx):
    static = step_inputs(ctx, seed=0)
    sets = [step_inputs(ctx, seed=s) for s in (1, 2, 3)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(ctx, *static)
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):                                         # two graphs of the same work on the same handle
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = step(ctx, *static)
            top = ctx.top_logits(outs[0], 7)
        graphs.append((graph, outs, top))
    flat = lambda s: [t for m in s for t in (m[:2] if isinstance(m, tuple) else (m,))]
    for s in sets:
        for dst, src in zip(flat(static), flat(s)):
            dst.view(torch.uint8).copy_(src.view(torch.uint8))
        want = step(ctx, *s)
        want_top = ctx.top_logits(want[0], 7)
        for graph, outs, top in graphs:
            graph.replay()
            torch.cuda.synchronize()
            for a, b in zip(outs + tuple(top), want + tuple(want_top)):
                assert torch.equal(a, b)


def test_two_streams_at_once(ctx):
    a, b = step_inputs(ctx, rows=3000, seed=4), step_inputs(ctx, rows=2000, v=1000, seed=5)
    want = step(ctx, *a), step(ctx, *b)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(3):
        with torch.cuda.stream(s1):
            ga = step(ctx, *a)
        with torch.cuda.stream(s2):
            gb = step(ctx, *b)
        torch.cuda.synchronize()
        for x, y in zip(ga + gb, want[0] + want[1]):
            assert torch.equal(x, y)


def test_stage_timers_name_the_operators(ctx):
    ctx.profile_enable(True)
    try:
        step(ctx, *step_inputs(ctx))
        ctx.top_logits(torch.randn(4, 97).cuda(), 3)
        names = ' '.join(r['name'] for r in ctx.profile_collect())
    finally:
        ctx.profile_enable(False)
    for part in ('quantize_fp8', 'gemm_fp8', 'distill_loss', 'top_logits'):
        assert part in names
