"""8-bit products and distillation, CPU side: the plain float64 forms (oracle/lowbit.py) against independent definitions,
and every refusal of the C entry points and of their Python callers.  The argument checks run before the handle is looked
at, so a null handle reaches all of them without a GPU; nothing is launched."""
import ctypes

import numpy as np
import pytest

torch = pytest.importorskip('torch')

from oracle import lowbit  # noqa: E402


# ------------------------------------------------------------------------------------ plain forms
def test_e4m3_values_and_rounding_are_those_of_the_format():
    table = lowbit.e4m3_table()
    by_torch = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()
    np.testing.assert_array_equal(table, by_torch)
    x = np.concatenate([np.linspace(-448, 448, 40001), np.random.default_rng(0).normal(0, 0.02, 20000)]).astype(np.float32)
    np.testing.assert_array_equal(lowbit.round_e4m3(x), torch.from_numpy(x).to(torch.float8_e4m3fn).double().numpy())


def test_scale_exponent_is_the_least_that_fits():
    rng = np.random.default_rng(1)
    for a in np.concatenate([np.exp2(rng.uniform(-126, 127, 300)), [448.0, 449.0, 224.0, 1.75, 1.7500001, 3.5, 2.0 ** -140]]):
        a = float(np.float32(a))
        e = lowbit.scale_exponent(a)
        assert a <= 448 * 2.0 ** e and (e == -127 or a > 448 * 2.0 ** (e - 1))
    assert lowbit.scale_exponent(0.0) == 0


@pytest.mark.parametrize('with_lse', [False, True])
def test_plain_gradient_is_the_derivative_of_the_plain_loss(with_lse):
    rng = np.random.default_rng(2)
    V, K, t, w = 23, 5, 1.7, 0.6
    s, teacher = rng.normal(0, 2, V), rng.normal(0, 2, V)
    idx = np.array([3, 7, 7, -1, 22])                   # a class twice, an entry that is none
    z = teacher[idx]
    lse = float(np.log(np.exp(teacher / t).sum())) + 0.7 if with_lse else None      # + 0.7: 7 twice must not exceed 1
    _, grad = lowbit.distill_row(s, z, idx, lse, t, w)
    h = 1e-5
    for v in range(V):
        up, down = s.copy(), s.copy()
        up[v] += h
        down[v] -= h
        d = (lowbit.distill_row(up, z, idx, lse, t, w)[0] - lowbit.distill_row(down, z, idx, lse, t, w)[0]) / (2 * h)
        assert abs(d - grad[v]) < 1e-8                   # truncation h^2 * f''' ~ 1e-10, cancellation eps / h ~ 1e-11


def test_plain_loss_over_all_classes_is_the_divergence():
    rng = np.random.default_rng(3)
    s, z = rng.normal(0, 1, 11), rng.normal(0, 1, 11)
    p, q = np.exp(z) / np.exp(z).sum(), np.exp(s) / np.exp(s).sum()
    loss, grad = lowbit.distill_row(s, z, np.arange(11), None, 1.0, 1.0)
    assert abs(loss - (p * np.log(p / q)).sum()) < 1e-14
    np.testing.assert_allclose(grad, q - p, atol=1e-15)


# --------------------------------------------------------------------------------------- refusals
P = 1 << 20          # a pointer that is never followed; the buffers below lie megabytes apart


def _call(name, **over):
    from ocr_amd import _lib
    lib = _lib.load()
    order = {
        'quantize_fp8': dict(h=None, x=P, x_dtype=0, rows=10, cols=200, ld_x=200, block_rows=1, transpose=0, q=64 * P, ld_q=256, scale=128 * P,
                             ld_scale=16, stream=None),
        'gemm_fp8': dict(h=None, a=P, ld_a=256, a_scale=8 * P, ld_as=16, b=16 * P, ld_b=256, b_scale=24 * P, ld_bs=16, b_rows=1, M=10, N=7, K=200,
                         bias=32 * P, c=40 * P, c_dtype=0, ld_c=7, ws=48 * P, ws_bytes=1 << 20, stream=None),
        'linear_fp8': dict(h=None, x=P, x_dtype=0, ld_x=200, b=16 * P, ld_b=256, b_scale=24 * P, ld_bs=16, b_rows=1, M=10, N=7, K=200, bias=32 * P,
                           c=40 * P, c_dtype=0, ld_c=7, ws=48 * P, ws_bytes=1 << 20, stream=None),
        'top_logits': dict(h=None, x=P, dtype=0, rows=4, V=97, ld=97, K=10, t=1.0, values=8 * P, index=16 * P, lse=24 * P, stream=None),
        'distill_loss': dict(h=None, x=P, dtype=0, rows=4, V=97, ld=97, values=8 * P, index=16 * P, K=10, lse=None, t=1.0, weight=None, loss=24 * P,
                             grad=32 * P, ld_grad=97, stream=None),
    }[name]
    assert not set(over) - set(order)
    order.update(over)
    rc = getattr(lib, 'ocrhip_' + name)(*order.values())
    return rc, lib.ocrhip_last_error().decode()


@pytest.mark.parametrize('name', ['quantize_fp8', 'gemm_fp8', 'linear_fp8', 'top_logits', 'distill_loss'])
def test_good_arguments_reach_the_handle(name):
    rc, msg = _call(name)
    assert rc == -1 and msg == 'null handle'


@pytest.mark.parametrize('name,over,part', [
    ('quantize_fp8', dict(x_dtype=2), 'F32 or BF16'),
    ('quantize_fp8', dict(x=None), 'x is null'),
    ('quantize_fp8', dict(x=P + 2), 'aligned'),
    ('quantize_fp8', dict(rows=-1), 'rows'),
    ('quantize_fp8', dict(cols=1 << 31, ld_x=1 << 31), 'columns'),
    ('quantize_fp8', dict(ld_x=199), 'elements apart'),
    ('quantize_fp8', dict(rows=1 << 20, ld_x=1 << 39), 'elements apart'),
    ('quantize_fp8', dict(block_rows=64), 'scale per 64'),
    ('quantize_fp8', dict(transpose=2), 'transpose'),
    ('quantize_fp8', dict(ld_q=200), 'multiple of 128'),
    ('quantize_fp8', dict(ld_q=128), 'multiple of 128'),
    ('quantize_fp8', dict(ld_scale=10), 'multiple of 16'),
    ('quantize_fp8', dict(rows=17), 'multiple of 16'),
    ('quantize_fp8', dict(transpose=1), 'multiple of 16'),
    ('quantize_fp8', dict(q=None), 'output is null'),
    ('quantize_fp8', dict(q=64 * P + 8), '16-byte'),
    ('quantize_fp8', dict(q=P + 64), 'overlap'),
    ('quantize_fp8', dict(scale=64 * P + 128), 'overlap'),
    ('gemm_fp8', dict(K=0), 'K must be'),
    ('gemm_fp8', dict(K=(1 << 22) + 1, ld_a=(1 << 22) + 128, ld_b=(1 << 22) + 128), 'K must be'),
    ('gemm_fp8', dict(ld_b=1 << 23), 'exceeds'),
    ('gemm_fp8', dict(M=-1), 'rows'),
    ('gemm_fp8', dict(c_dtype=2), 'F32 or BF16'),
    ('gemm_fp8', dict(c=None), 'output is null'),
    ('gemm_fp8', dict(ld_c=6), 'elements apart'),
    ('gemm_fp8', dict(bias=32 * P + 1), 'bias'),
    ('gemm_fp8', dict(a=None), 'a is null'),
    ('gemm_fp8', dict(a_scale=None), 'a is null'),
    ('gemm_fp8', dict(ld_a=128), 'multiple of 128'),
    ('gemm_fp8', dict(ld_b=200), 'multiple of 128'),
    ('gemm_fp8', dict(b_rows=2), 'scale per 2'),
    ('gemm_fp8', dict(N=17, ld_c=17), 'multiple of 16'),
    ('gemm_fp8', dict(a=P + 1), '16-byte'),
    ('gemm_fp8', dict(c=P + 128), 'overlaps'),
    ('gemm_fp8', dict(c=16 * P), 'overlaps'),
    ('gemm_fp8', dict(c=8 * P + 16), 'overlaps'),
    ('gemm_fp8', dict(c=24 * P), 'overlaps'),
    ('gemm_fp8', dict(c=32 * P), 'overlaps'),
    ('linear_fp8', dict(x_dtype=1, x=P + 1), 'aligned'),
    ('linear_fp8', dict(ld_x=100), 'elements apart'),
    ('linear_fp8', dict(M=500, ws=None), 'workspace'),
    ('linear_fp8', dict(M=500, ws=48 * P + 4), 'workspace'),
    ('linear_fp8', dict(c=P), 'overlaps'),
    ('linear_fp8', dict(ws=P), 'overlaps'),
    ('linear_fp8', dict(ws=40 * P), 'overlaps'),
    ('top_logits', dict(V=0, K=1, ld=1), 'classes'),
    ('top_logits', dict(V=262145, ld=262145), 'classes'),
    ('top_logits', dict(K=0), 'entries'),
    ('top_logits', dict(K=65), 'entries'),
    ('top_logits', dict(V=9, ld=9), '10 of 9'),
    ('top_logits', dict(t=0.0), 'temperature'),
    ('top_logits', dict(t=float('nan')), 'temperature'),
    ('top_logits', dict(t=float('inf')), 'temperature'),
    ('top_logits', dict(t=1e-39), 'temperature'),
    ('top_logits', dict(ld=96), 'elements apart'),
    ('top_logits', dict(x=None), 'null'),
    ('top_logits', dict(values=None), 'null output'),
    ('top_logits', dict(index=16 * P + 2), 'aligned'),
    ('distill_loss', dict(loss=None, grad=None), 'ask for'),
    ('distill_loss', dict(values=None), 'entries are null'),
    ('distill_loss', dict(index=None), 'entries are null'),
    ('distill_loss', dict(dtype=2), 'F32 or BF16'),
    ('distill_loss', dict(K=100), 'entries'),
    ('distill_loss', dict(ld_grad=90), 'elements apart'),
    ('distill_loss', dict(grad=P), 'overlaps'),
    ('distill_loss', dict(grad=P + 97 * 4 * 3), 'overlaps'),
    ('distill_loss', dict(weight=3), 'aligned'),
    ('distill_loss', dict(t=-1.0), 'temperature'),
])
def test_refusals_of_the_c_entries(name, over, part):
    rc, msg = _call(name, **over)
    assert rc == -1 and part in msg and msg.startswith(name), msg


@pytest.mark.parametrize('name,over', [
    ('gemm_fp8', dict(c=P + 9 * 256 + 200)),                   # the zeros behind the last row's columns
    ('gemm_fp8', dict(M=500, ld_as=512, ws=P, c=60 * P)), ('gemm_fp8', dict(ws=16 * P + 64)), ('gemm_fp8', dict(ws=8 * P)), ('gemm_fp8', dict(ws=24 * P)),
    ('gemm_fp8', dict(ws=32 * P)), ('linear_fp8', dict(ws=16 * P)), ('linear_fp8', dict(ws=32 * P)),
    ('top_logits', dict(values=P + 64)), ('top_logits', dict(index=P + 64)), ('top_logits', dict(lse=P + 4 * 97 * 4 - 4)),
    ('top_logits', dict(index=8 * P)), ('top_logits', dict(index=8 * P + 156)), ('top_logits', dict(lse=8 * P)), ('top_logits', dict(lse=16 * P + 8)),
    ('distill_loss', dict(grad=8 * P)), ('distill_loss', dict(grad=16 * P + 40)), ('distill_loss', dict(grad=24 * P)), ('distill_loss', dict(lse=32 * P)),
    ('distill_loss', dict(weight=32 * P)), ('distill_loss', dict(loss=P)), ('distill_loss', dict(loss=8 * P)), ('distill_loss', dict(loss=16 * P + 156)),
    ('distill_loss', dict(weight=24 * P)), ('distill_loss', dict(lse=24 * P + 12)),
    ('distill_loss', dict(ld=200, ld_grad=200, grad=P + 96 * 4)),
])
def test_outputs_that_share_memory_are_refused(name, over):
    rc, msg = _call(name, **over)
    assert rc == -1 and 'overlap' in msg and msg.startswith(name), msg


@pytest.mark.parametrize('name,over', [
    ('distill_loss', dict(ld=200, ld_grad=200, grad=P + 97 * 4)),            # logits and gradient side by side
    ('distill_loss', dict(x=P + 103 * 4, ld=200, ld_grad=200, grad=P)),
    ('linear_fp8', dict(ld_x=256, ld_c=256, c=P + 200 * 4)),
    ('linear_fp8', dict(ld_x=256, ld_c=256, c=P - 7 * 4)),
    ('top_logits', dict(lse=16 * P + 160)), ('top_logits', dict(index=8 * P + 160)),
    ('gemm_fp8', dict(ld_a=384, ld_c=96, c=P + 256)),
])
def test_neighbours_in_one_buffer_are_no_overlap(name, over):
    rc, msg = _call(name, **over)
    assert rc == -1 and msg == 'null handle', msg


def test_a_workspace_that_is_too_small_is_a_capacity_error():
    from ocr_amd import _lib
    need = _lib.load().ocrhip_linear_fp8_workspace(500, 7, 200)
    assert need >= 500 * 256 + 2 * 512
    rc, msg = _call('linear_fp8', M=500, ws_bytes=need - 1)
    assert rc == -2 and str(need) in msg


def test_workspaces_of_empty_and_negative_sizes_are_nothing():
    from ocr_amd import _lib
    lib = _lib.load()
    for m, n, k in ((0, 5, 5), (5, 0, 5), (5, 5, 0), (-1, 5, 5), (1 << 62, 5, 5), (70, 1 << 62, 5), (70, 5, 1 << 62), (1 << 31, 5, 5)):
        assert lib.ocrhip_gemm_fp8_workspace(m, n, k) == 0 and lib.ocrhip_linear_fp8_workspace(m, n, k) == 0


@pytest.fixture()
def ctx():
    """A context without a handle on the CPU: everything that raises before the library is called."""
    from ocr_amd import _lib
    from ocr_amd.engine import HipContext
    c = object.__new__(HipContext)
    c.lib, c.device, c._h, c.options = _lib.load(), torch.device('cpu'), None, {}
    c._on = lambda: ctypes.c_void_p(0)
    return c


def _matrix(rows, cols, by=1, **over):
    from ocr_amd.engine import Fp8Matrix
    kb, rb = -(-cols // 128), -(-rows // by)
    m = dict(q=torch.zeros((rows, kb * 128), dtype=torch.uint8).view(torch.float8_e4m3fn), scale=torch.full((kb, -(-rb // 16) * 16), 127, dtype=torch.uint8),
             rows=rows, cols=cols, block_rows=by)
    m.update(over)
    return Fp8Matrix(**m)


def test_refusals_of_the_python_callers(ctx):
    x = torch.zeros(4, 200)
    v, i = torch.zeros(4, 3), torch.zeros(4, 3, dtype=torch.int32)
    cases = [
        (lambda: ctx.quantize_fp8(x.half()), 'float32 or bfloat16'),
        (lambda: ctx.quantize_fp8(x.to('meta')), 'is on meta'),
        (lambda: ctx.quantize_fp8(torch.tensor(1.0)), 'no dimensions'),
        (lambda: ctx.quantize_fp8(x, block_rows=32), 'block_rows'),
        (lambda: ctx.gemm_fp8(_matrix(4, 200, by=128), _matrix(7, 200)), 'scale per row'),
        (lambda: ctx.gemm_fp8(_matrix(4, 200), _matrix(7, 100)), 'columns'),
        (lambda: ctx.gemm_fp8(_matrix(4, 200)._replace(rows=5), _matrix(7, 200)), 'of 5 x 200'),
        (lambda: ctx.gemm_fp8(_matrix(4, 200), _matrix(7, 200, by=128, block_rows=16)), 'scale per 16'),
        (lambda: ctx.gemm_fp8(_matrix(4, 200), _matrix(7, 200, q=torch.zeros(7, 256))), 'float8_e4m3fn'),
        (lambda: ctx.gemm_fp8(_matrix(4, 200), _matrix(7, 200, q=torch.zeros(7, 256, dtype=torch.int8))), 'float8_e4m3fn'),
        (lambda: ctx.gemm_fp8(_matrix(4, 200), _matrix(7, 200, scale=torch.zeros(2, 16))), 'uint8'),
        (lambda: ctx.gemm_fp8(_matrix(4, 200), _matrix(7, 200, scale=torch.zeros(1, 16, dtype=torch.uint8))), 'scales (1, 16)'),
        (lambda: ctx.gemm_fp8(_matrix(4, 200), _matrix(7, 200), bias=torch.zeros(4)), 'shape (7,)'),
        (lambda: ctx.gemm_fp8(_matrix(4, 200), _matrix(7, 200), bias=torch.zeros(7, dtype=torch.float64)), 'bias must be'),
        (lambda: ctx.gemm_fp8(_matrix(4, 200), _matrix(7, 200), out_dtype=torch.float16), 'out_dtype'),
        (lambda: ctx.linear_fp8(torch.zeros(3, 100), _matrix(7, 200)), '100 columns'),
        (lambda: ctx.top_logits(x, 0), '1 .. 64'),
        (lambda: ctx.top_logits(x, 65), '1 .. 64'),
        (lambda: ctx.top_logits(x[:, :5], 6), '6 of 5'),
        (lambda: ctx.top_logits(x, 3, temperature=0.0), 'temperature'),
        (lambda: ctx.distill_loss(x, v[:2], i[:2]), 'shape (4, 3)'),
        (lambda: ctx.distill_loss(x, v, i.long()), 'top_index must be'),
        (lambda: ctx.distill_loss(x, v, i, top_lse=torch.zeros(3)), 'shape (4,)'),
        (lambda: ctx.distill_loss(x, v, i, row_weight=torch.zeros(4, 1)), 'shape (4,)'),
        (lambda: ctx.distill_loss(x, v, i, want_loss=False), 'ask for'),
        (lambda: ctx.distill_loss(x, torch.zeros(4, 0), torch.zeros(4, 0, dtype=torch.int32)), 'entries'),
    ]
    for k, (call, part) in enumerate(cases):
        with pytest.raises(ValueError) as e:
            call()
        assert part in str(e.value), (k, str(e.value))
