"""8-bit products and distillation, CPU side, at the edges of what their documentation settles: what the C entries accept and
refuse there, and the plain float64 forms (oracle/lowbit.py)."""
import pytest

from test_lowbit_cpu import _call


@pytest.mark.parametrize('name', ['top_logits', 'distill_loss'])
@pytest.mark.parametrize('t,good', [(2.0 ** -149, False), (2.9e-39, False), (3.5e-39, False), (4.2e-39, False), (4.3e-39, True), (2.0 ** -127, True),
                                    (1e-38, True), (3.4e38, True)])
def test_temperatures(name, t, good):
    """log2(e) / temperature is a float32 number from 4.3e-39 on; below it 0 times infinity would be NaN."""
    rc, msg = _call(name, t=t)
    assert rc == -1 and (msg == 'null handle' if good else 'temperature' in msg and msg.startswith(name)), msg
