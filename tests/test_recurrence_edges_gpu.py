"""DeviceLinearRecurrence on the GPU where there is little or nothing to do."""
import pytest

from tests.test_recurrence_gpu import MODES, Case, host

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows", [1, 130, 700])
def test_no_sequences_among_the_rows(cuda, mode, dtype, rows):
    # one offset and no sequence: every row is padding, whatever it holds
    c = Case([], 72, dtype, mode, packed=True, tail=rows)
    for m in (c.gate, c.x, c.grad_out):
        m[::2] = float("nan")
    out, last = c.forward()
    gg, gi, g0 = c.backward()
    assert (host(out) == 0).all() and (host(gg) == 0).all() and (host(gi) == 0).all()
    assert last.shape == (0, 72) and g0.shape == (0, 72)
