"""Gradients of the delta rule where the groups of 16 value dimensions that one warp has differ in size, or hold nothing."""
import numpy as np
import pytest

from tests import delta_reference as R
from tests.test_delta_gpu import Case, host

pytestmark = pytest.mark.gpu

# (heads, key heads, key_dim, value_dim): 3 groups, 8 groups, an odd last one
HEADS = [(2, 2, 64, 48), (2, 1, 128, 128), (1, 1, 40, 67)]


def grouped(c, name, factors):
    """Scales the tensor's groups of 16 value dimensions."""
    import torch

    t = getattr(c, name)
    by = torch.tensor(np.repeat(factors, 16)[:c.dv], device="cuda")
    dim = 2  # (sequences, heads, value_dim, key_dim) as well as (rows, heads, value_dim)
    by = by.view((1,) * dim + (-1,) + (1,) * (t.dim() - dim - 1))
    t.copy_((t.double() * by).to(t.dtype))


@pytest.mark.parametrize("heads,key_heads,dk,dv", HEADS)
@pytest.mark.parametrize("dtype,size", [("f32", 1e-6), ("f32", 1e-12), ("f32", 1.0), ("bf16", 1e-6), ("bf16", 1e-12), ("f16", 1e-3)])
@pytest.mark.parametrize("name", ["grad_out", "v", "grad_last", "init"])
def test_a_group_of_zeros(cuda, dtype, size, name, heads, key_heads, dk, dv):
    """The others are as good as without it: the bounds scale with what is there."""
    c = Case([130, 70], heads, key_heads, dk, dv, dtype, seed=31)
    groups = -(-dv // 16)
    if name == "v":
        c.init = None
    for at in (0, groups - 1):
        f = np.full(groups, size)
        f[at] = 0.0
        d = Case([130, 70], heads, key_heads, dk, dv, dtype, seed=31)
        if name == "v":
            d.init = None
        grouped(d, name, f)
        if name == "grad_out":  # nothing else brings a gradient
            d.check(use_last=False)
        elif name == "grad_last":
            d.check(use_out=False)
        else:
            d.check()


@pytest.mark.parametrize("heads,key_heads,dk,dv", HEADS)
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("step", [4, 8, 16])
@pytest.mark.parametrize("names", [("grad_out",), ("v", "init"), ("grad_last",), ("grad_out", "v", "init")])
def test_groups_of_different_sizes(cuda, dtype, step, names, heads, key_heads, dk, dv):
    """Group after group 2^step smaller or larger, down to 2^-(3 step)."""
    if dtype == "f16" and step == 16:
        step = 3  # its values end at 2^-24
    groups = -(-dv // 16)
    for turn in (1, -1):
        c = Case([130, 70], heads, key_heads, dk, dv, dtype, seed=32)
        f = 2.0 ** (-step * (np.arange(groups)[::turn] % 4))
        for n in names:
            grouped(c, n, f)
        c.check(use_last="grad_last" in names, use_out="grad_out" in names or "v" in names)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("size", [1e-10, 1e-18, 1e-24])
def test_small_gradients_of_outputs_beside_large_ones_of_states(cuda, dtype, size):
    """grad_q is made of grad_out alone: its bound is that of tests.delta_reference.bounds without the states' gradient, of
    scale |grad_out| M, with the largest gradient of the sequence for each value dimension."""
    c = Case([130, 70], 2, 1, 64, 48, dtype, seed=33)
    c.grad_out.mul_(size)
    f = c.reference()
    c.run()
    got, want = c.back(), R.backward(f, host(c.grad_out), host(c.grad_last))
    bound = np.zeros((c.rows, c.heads, 1))
    go = np.abs(host(c.grad_out))
    for s in range(2):
        a, b = c.offsets[s], c.offsets[s + 1]
        unit = R.UNIT * np.sqrt(-(-(b - a) // 64))
        bound[a:b] = 2 * unit * f.scale * np.sqrt(((go[a:b].max(0) * f.most[s]) ** 2).sum(1))[:, None]
    bound = bound.reshape(c.rows, 1, 2, 1).sum(2)
    R.assert_within(host(got.q), want.q, bound, dtype, "grad q")
