"""The recogniser's dense layers as 8-bit block-scaled products (option fp8_dense = 1, `compute_dtype = BF16`).

The class layer is checked exactly: its input rows are the tap 'seq1' (bfloat16 values), so its quantised operands are
determined and the logits are their float64 product but for float32 sums: (K - 1) 2u sum |a b|, u = 2^-24, and u each for
bias and store.  The whole is checked against the bfloat16 recogniser: a value is off by at most 2^-4 of itself after
rounding to e4m3 (no value of these inputs lies below the normal numbers of its block in a way that matters to a norm), a
product of two such by sqrt(2) 2^-4 of its norm when the errors are independent; five such layers follow one another (input
projection, linear, twice, and the classes), the recurrence is taken as not amplifying: sqrt(5) sqrt(2) 2^-4 = 0.198.
"""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip('torch')

from oracle import ctc as octc, lowbit, nets  # noqa: E402

U = 2.0 ** -24
BAR = 5 ** 0.5 * 2 ** 0.5 / 16


@pytest.fixture(scope='module')
def ctx():
    from ocr_amd.engine import HipContext
    c = HipContext(0)
    yield c
    c.close()


def rel(a, b):
    return float(np.linalg.norm((np.asarray(a, np.float64) - b).ravel()) / max(1e-30, np.linalg.norm(np.asarray(b, np.float64).ravel())))


def check_class_layer(params, seq, logits):
    w, b = (np.asarray(params['Prediction.' + k], np.float64) for k in ('weight', 'bias'))
    a = lowbit.dequantize(*lowbit.quantize(seq, 1), 1)
    q = lowbit.dequantize(*lowbit.quantize(w, 128), 128)
    want = a @ q.T + b
    tol = (a.shape[1] - 1) * 2 * U * (np.abs(a) @ np.abs(q).T) + 2 * U * (np.abs(want) + np.abs(b))
    assert (np.abs(logits - want) <= tol).all(), float((np.abs(logits - want) - tol).max())


# one row and one time step; up to 64 rows and beyond (two forms of the product), the Chinese and the English alphabet
@pytest.mark.parametrize('n,wpad,vocab', [(1, 8, 97), (3, 64, 97), (4, 72, 97), (33, 192, 97), (2, 64, 6719), (9, 128, 6719)])
def test_recogniser_with_8_bit_dense_layers(ctx, n, wpad, vocab):
    from ocr_amd._lib import BF16
    params = nets.init_crnn_params(vocab_size=vocab, seed=2)
    ctx.crnn_load_weights(params)
    x = torch.from_numpy(np.random.default_rng(n * 7 + wpad).uniform(-1, 1, (n, 64, wpad, 1)).astype(np.float32)).cuda()

    def run(dtype):
        out = ctx.crnn_forward(x, want_logits=True, want_tokens=True, compute_dtype=dtype)
        torch.cuda.synchronize()
        ctx.check_errors()
        seq = [np.asarray(ctx.crnn_activation(k), np.float64).reshape(-1, 256) for k in ('seq0', 'seq1')] if dtype == BF16 else None
        return out['logits'].cpu().numpy(), out['tokens'].cpu().numpy(), out['scores'].cpu().numpy(), seq
    plain, f32 = run(BF16), run(0)
    ctx.set_option('fp8_dense', 1)
    try:
        logits, tokens, scores, seq = run(BF16)
        again = run(BF16)
        f32_on = run(0)
    finally:
        ctx.set_option('fp8_dense', 0)
    check_class_layer(params, seq[1], logits.reshape(-1, vocab))
    assert 0 < rel(logits, plain[0]) <= BAR and 0 < rel(seq[0], plain[3][0]) <= BAR and rel(seq[1], plain[3][1]) <= BAR
    rt, rs = octc.ctc_greedy(logits, None, 0)
    np.testing.assert_array_equal(tokens, rt)
    np.testing.assert_array_equal(scores, rs)
    np.testing.assert_array_equal(again[0], logits)
    # the float32 recogniser does not know the option, and off is off
    np.testing.assert_array_equal(f32_on[0], f32[0])
    np.testing.assert_array_equal(run(BF16)[0], plain[0])


# blocks of k that the columns do not fill (64, 192), per-step recurrence
@pytest.mark.parametrize('hidden', [64, 128, 192, 512])
def test_other_lstm_widths(ctx, hidden):
    from ocr_amd._lib import BF16
    params = nets.init_crnn_params(vocab_size=211, hidden=hidden, seed=3)
    ctx.crnn_load_weights(params)
    x = torch.from_numpy(np.random.default_rng(hidden).uniform(-1, 1, (6, 64, 100, 1)).astype(np.float32)).cuda()
    plain = ctx.crnn_forward(x, compute_dtype=BF16)['logits'].cpu().numpy()
    ctx.set_option('fp8_dense', 1)
    try:
        logits = ctx.crnn_forward(x, compute_dtype=BF16)['logits'].cpu().numpy()
        ctx.check_errors()
    finally:
        ctx.set_option('fp8_dense', 0)
    check_class_layer(params, np.asarray(ctx.crnn_activation('seq1'), np.float64).reshape(-1, hidden), logits.reshape(-1, 211))
    assert 0 < rel(logits, plain) <= BAR


def test_resnet_recogniser_does_not_know_the_option(ctx):
    from ocr_amd._lib import BF16
    ctx.crnn_load_weights(nets.init_crnn_params(vocab_size=97, hidden=256, seed=3, backbone='resnet'))
    x = torch.from_numpy(np.random.default_rng(1).uniform(-1, 1, (2, 64, 64, 1)).astype(np.float32)).cuda()
    plain = ctx.crnn_forward(x, compute_dtype=BF16)['logits']
    ctx.set_option('fp8_dense', 1)
    try:
        got = ctx.crnn_forward(x, compute_dtype=BF16)['logits']
    finally:
        ctx.set_option('fp8_dense', 0)
    assert torch.equal(got, plain)


def test_packed_batch_with_8_bit_dense_layers(ctx):
    """Several widths in one call; then a smaller one: the buffers of the larger one hold other values behind its rows."""
    from ocr_amd._lib import BF16
    params = nets.init_crnn_params(vocab_size=97, seed=2)
    ctx.crnn_load_weights(params)
    rng = np.random.default_rng(5)
    widths = np.array([64] * 3 + [128] * 35 + [192] * 2 + [320], dtype=np.int32)
    packed = torch.from_numpy(rng.uniform(-1, 1, int(64 * widths.sum())).astype(np.float32)).cuda()
    plain = ctx.crnn_forward_packed(packed, widths, want_logits=True, compute_dtype=BF16)['logits'].cpu().numpy()
    ctx.set_option('fp8_dense', 1)
    try:
        for k in (len(widths), 2, 1):
            out = ctx.crnn_forward_packed(packed[:64 * int(widths[:k].sum())], widths[:k], want_logits=True, compute_dtype=BF16)
            ctx.check_errors()
            lg = out['logits'].cpu().numpy()
            check_class_layer(params, np.asarray(ctx.crnn_activation('seq1'), np.float64).reshape(-1, 256), lg)
            assert 0 < rel(lg, plain[:lg.shape[0]]) <= BAR
    finally:
        ctx.set_option('fp8_dense', 0)


def test_student_of_the_float32_recogniser(ctx):
    """The float32 recogniser's top logits against the 8-bit recogniser's logits, as a user would measure or train it: the
    loss and its gradient are what the definition gives for the two sets of logits."""
    from ocr_amd._lib import BF16
    ctx.crnn_load_weights(nets.init_crnn_params(vocab_size=97, seed=2))
    x = torch.from_numpy(np.random.default_rng(3).uniform(-1, 1, (5, 64, 96, 1)).astype(np.float32)).cuda()
    teacher = ctx.crnn_forward(x, want_logits=True)['logits'].reshape(-1, 97)
    values, index, lse = ctx.top_logits(teacher, 8, temperature=2.0)
    ctx.set_option('fp8_dense', 1)
    try:
        student = ctx.crnn_forward(x, want_logits=True, compute_dtype=BF16)['logits'].reshape(-1, 97)
        ctx.check_errors()
    finally:
        ctx.set_option('fp8_dense', 0)
    got = ctx.distill_loss(student, values, index, lse, temperature=2.0, want_grad=True)
    loss, grad = lowbit.distill(student.cpu().numpy(), values.cpu().numpy(), index.cpu().numpy(), lse.cpu().numpy(), 2.0, None)
    # 97 classes: a float32 sum of exponentials off by eps (four roundings of an argument of mean magnitude ln V + 1 at most,
    # six additions, the exponential's own 2^-22), the loss by eps times the factor |q_rest - p_rest| <= 1, a gradient entry
    # by twice that, its own exponential's argument of magnitude `far` and the store
    eps = U * (4 * (np.log(97) + 1) + 7) + 2.0 ** -22
    far = float((student.max(dim=1, keepdim=True).values - student).max()) / 2.0
    loss_tol, grad_tol = 4.0 * eps + 2 * U * np.abs(loss).max(), 2.0 * 2 * (2 * eps + U * (4 * far + 8))
    assert np.abs(got['loss'].cpu().numpy() - loss).max() <= loss_tol
    assert np.abs(got['grad'].cpu().numpy() - grad).max() <= grad_tol
    # a divergence, of distributions that the float32 lse lets sum to 1 within 2u |lse|
    assert (loss >= -4.0 * 2 * U * (1 + float(lse.abs().max()))).all()


def test_option_values(ctx):
    for v in (-1, 2):
        with pytest.raises(Exception, match='fp8_dense is 0 or 1'):
            ctx.set_option('fp8_dense', v)
