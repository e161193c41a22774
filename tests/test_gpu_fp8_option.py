"""When the recogniser's dense layers get their 8-bit weights: with the option fp8_dense and not without."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip('torch')

from oracle import nets  # noqa: E402


def context():
    from ocr_amd.engine import HipContext
    return HipContext(0)


def launches(ctx, call):
    ctx.profile_enable(True)
    try:
        call()
        return [r['name'] for r in ctx.profile_collect()]
    finally:
        ctx.profile_enable(False)


@pytest.mark.parametrize('backbone', ['vgg', 'resnet'])
def test_loading_weights_quantises_only_with_the_option(backbone):
    params = nets.init_crnn_params(vocab_size=97, seed=2, backbone=backbone)
    ctx = context()
    try:
        assert 'quantize_fp8' not in launches(ctx, lambda: ctx.crnn_load_weights(params))
        assert ('quantize_fp8' in launches(ctx, lambda: ctx.set_option('fp8_dense', 1))) == (backbone == 'vgg')
        assert 'quantize_fp8' not in launches(ctx, lambda: (ctx.set_option('fp8_dense', 0), ctx.set_option('fp8_dense', 1)))
        assert ('quantize_fp8' in launches(ctx, lambda: ctx.crnn_load_weights(params))) == (backbone == 'vgg')
    finally:
        ctx.close()


@pytest.mark.parametrize('vocab,hidden', [(97, 256), (211, 64), (6719, 256)])
def test_the_order_of_option_and_weights_does_not_matter(vocab, hidden):
    """The option before the weights, behind them, switched off and on again, and over other weights."""
    from ocr_amd._lib import BF16
    first, second = (nets.init_crnn_params(vocab_size=vocab, hidden=hidden, seed=s) for s in (2, 3))
    x = torch.from_numpy(np.random.default_rng(1).uniform(-1, 1, (5, 64, 96, 1)).astype(np.float32)).cuda()

    def run(*steps):
        ctx = context()
        try:
            for s in steps:
                ctx.set_option('fp8_dense', s) if isinstance(s, int) else ctx.crnn_load_weights(s)
            out = ctx.crnn_forward(x, want_logits=True, compute_dtype=BF16)['logits'].cpu()
            ctx.check_errors()
            return out
        finally:
            ctx.close()
    want = run(first, 1)
    assert torch.equal(run(1, first), want) and torch.equal(run(second, 1, first), want) and torch.equal(run(1, second, 0, first, 1), want)
    assert torch.equal(run(first, 1, 0, 1), want) and not torch.equal(run(first), want) and torch.equal(run(first, 1, 0), run(first))
