"""The delta rule with buffers for more rows and sequences than a call has."""
import pytest

from tests.test_delta_gpu import Case

pytestmark = pytest.mark.gpu


class Larger(Case):
    """With the buffers of another case."""

    larger = None

    def sizes(self):
        return self.larger or super().sizes()


# One sequence of 4608 rows takes 9 parts; a row of chunks more 5, and with them less memory.
@pytest.mark.parametrize("dtype,heads,key_heads,dk,dv,more", [
    ("bf16", 16, 8, 128, 128, (4672, 1)), ("bf16", 16, 8, 128, 128, (5120, 3)), ("bf16", 8, 4, 128, 64, (4672, 1)),
    ("f32", 8, 4, 128, 64, (4672, 1))])
def test_buffers_for_more(cuda, dtype, heads, key_heads, dk, dv, more):
    c = Larger([4608], heads, key_heads, dk, dv, dtype, seed=51)
    c.larger = (*more, heads, key_heads, dk, dv)
    c.check()
