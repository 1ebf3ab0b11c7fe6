"""The delta rule at the ends of the precision and range that its header states for float32 values."""
import numpy as np
import pytest

from tests import delta_reference as R
from tests.test_delta_gpu import Case, host

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("size,q,k", [(2.0 ** -78, 1.0, 1.0), (1.0, 2.0 ** -38, 1.0), (1.0, 1.0, 2.0 ** -30), (2.0 ** 50, 2.0 ** 20, 1.0)])
def test_sizes_that_keep_all_bits(cuda, size, q, k):
    c = Case([130, 70], 2, 1, 64, 48, "f32", seed=71, size=size)
    c.q.mul_(q)
    c.k.mul_(k)
    c.check(backward=k == 1.0)  # the bounds of the gradients suppose unit keys


@pytest.mark.parametrize("ratio", [2.0 ** -8, 2.0 ** -20, 2.0 ** -30])
def test_value_dimensions_beside_larger_ones(cuda, ratio):
    """A value counts to 2^-32 of the largest of its 16 value dimensions: where the roundings of tests.delta_reference are
    2^-21 of a term of size M, 2^-32 of the others' M come on top, 2^-11 of theirs in the same count."""
    import torch

    c = Case([130, 70], 2, 1, 64, 48, "f32", seed=72)
    by = torch.tensor(np.where(np.arange(48) % 3 == 0, 1.0, ratio), device="cuda")
    for m in (c.v, c.grad_out):
        m.copy_((m.double() * by).float())
    for m in (c.init, c.grad_last):
        m.copy_((m.double() * by[:, None]).float())
    f = c.reference()
    out, last = c.run()
    got, want = c.back(), R.backward(f, host(c.grad_out), host(c.grad_last))
    for r in (f, want):
        r.most = r.most + 2.0 ** -11 * np.repeat(r.most.reshape(2, 2, 3, 16).max(3), 16, axis=2)
    b = R.bounds(f, want)
    R.assert_within(host(out), f.out, b.out, "f32", "out")
    R.assert_within(host(last), f.last, b.last, "f32", "last")
    for n in ("q", "k", "v", "beta", "decay", "init"):
        R.assert_within(host(getattr(got, n)), getattr(want, n), getattr(b, n), "f32", "grad " + n)


def test_states_that_start_anew(cuda):
    """What the tokens of a chunk bring counts to 2^-62 of the state before it: behind a decay of -inf nothing of a state 2^36
    times as large is left, and the outputs keep their bits."""
    c = Case([130, 70], 2, 1, 64, 48, "f32", seed=73)
    c.init.mul_(2.0 ** 36)
    c.decay[0], c.decay[130] = -float("inf"), -float("inf")
    out, last = c.run()
    c.init.zero_()
    f = c.reference()
    b = R.bounds(f)
    R.assert_within(host(out), f.out, b.out, "f32", "out")
    R.assert_within(host(last), f.last, b.last, "f32", "last")
