"""8-bit products and distillation, CPU side, at the edges of what their documentation settles: what the C entries accept and
refuse there, and the plain float64 forms (oracle/lowbit.py)."""
import numpy as np
import pytest

from oracle import lowbit
from test_lowbit_cpu import P, _call


@pytest.mark.parametrize('name', ['top_logits', 'distill_loss'])
@pytest.mark.parametrize('t,good', [(2.0 ** -149, False), (2.9e-39, False), (3.5e-39, False), (4.2e-39, False), (4.3e-39, True), (2.0 ** -127, True),
                                    (1e-38, True), (3.4e38, True)])
def test_temperatures(name, t, good):
    """log2(e) / temperature is a float32 number from 4.3e-39 on; below it 0 times infinity would be NaN."""
    rc, msg = _call(name, t=t)
    assert rc == -1 and (msg == 'null handle' if good else 'temperature' in msg and msg.startswith(name)), msg


@pytest.mark.parametrize('shift', [0.7, 0.0, -0.9, -3.0])
@pytest.mark.parametrize('every', [False, True])
def test_plain_gradient_is_the_derivative_whatever_the_mass(shift, every):
    """The entries' probabilities sum to less than 1, to 1 or to more (a log normaliser of another temperature), and with every
    class named there is no rest whatever they sum to."""
    rng = np.random.default_rng(5)
    V, t, w = 13, 1.7, 0.6
    s, teacher = rng.normal(0, 2, V), rng.normal(0, 2, V)
    idx = rng.permutation(V) if every else np.array([3, 7, 1, -1, 12])
    z = teacher[idx]
    lse = float(np.log(np.exp(teacher / t).sum())) + shift
    _, grad = lowbit.distill_row(s, z, idx, lse, t, w)
    h = 1e-5
    for v in range(V):
        up, down = s.copy(), s.copy()
        up[v] += h
        down[v] -= h
        d = (lowbit.distill_row(up, z, idx, lse, t, w)[0] - lowbit.distill_row(down, z, idx, lse, t, w)[0]) / (2 * h)
        # truncation h^2 times a third derivative ~ 1e-10, cancellation eps / h ~ 1e-11, times the mass
        assert abs(d - grad[v]) < 1e-8 * max(1.0, np.exp(-shift))


@pytest.mark.parametrize('with_lse', [False, True])
def test_plain_loss_of_a_class_named_twice_is_that_of_its_whole_probability(with_lse):
    """A class's probability split over several entries (z - log 2 twice, z - log 3 three times) is the class named once; a
    student that agrees entirely has no loss."""
    rng = np.random.default_rng(6)
    teacher = rng.normal(0, 2, 9)
    lse = float(np.log(np.exp(teacher).sum())) if with_lse else None
    once = np.arange(9)
    split = np.concatenate([[4, 2, 4, 2, 2], [0, 1, 3, 5, 6, 7, 8]])
    z = teacher[split] - np.array([np.log(2), np.log(3), np.log(2), np.log(3), np.log(3)] + [0.0] * 7)
    for s in (rng.normal(0, 2, 9), teacher):
        a, b = lowbit.distill_row(s, teacher, once, lse, 1.0, 1.0), lowbit.distill_row(s, z, split, lse, 1.0, 1.0)
        assert abs(a[0] - b[0]) < 1e-14 * 16 and np.abs(a[1] - b[1]).max() < 1e-15 * 16
    assert abs(b[0]) < 1e-14


@pytest.mark.parametrize('over,good', [
    (dict(cols=32, ld_x=128, q=P + 128, ld_q=512), True),                     # x and the bytes in columns of one buffer of 512-byte rows
    (dict(cols=32, ld_x=128, q=P + 112, ld_q=512), False),
    (dict(cols=32, ld_x=128, q=P + 384, ld_q=512), True),
    (dict(cols=32, ld_x=128, q=P + 400, ld_q=512), False),
    (dict(cols=130, ld_x=132, q=64 * P, ld_q=512, x=64 * P + 9 * 512 + 256), True),      # x right behind the last row's bytes
    (dict(cols=130, ld_x=132, q=64 * P, ld_q=512, x=64 * P + 9 * 512 + 252), False),
    (dict(q=64 * P, ld_q=512, scale=64 * P + 256, ld_scale=512), True),       # bytes and scales in columns of one buffer
    (dict(q=64 * P, ld_q=512, scale=64 * P + 240, ld_scale=512), False),
    (dict(q=64 * P, ld_q=512, scale=64 * P + 496, ld_scale=512), True),
    (dict(x=128 * P + 1024 + 12, scale=128 * P, ld_scale=1024), True),        # x right behind the last scale (10 of a row of 1024)
    (dict(x=128 * P + 1024 + 8, scale=128 * P, ld_scale=1024), False),
])
def test_quantised_columns_of_a_wider_buffer_are_no_overlap(over, good):
    """Only the columns rounded up to 128 and the scales of existing blocks are written."""
    rc, msg = _call('quantize_fp8', **over)
    assert rc == -1 and (msg == 'null handle' if good else 'overlap' in msg), msg
