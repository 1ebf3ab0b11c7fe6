"""The float64 form of the delta rule's gradients against differences (no GPU)."""
import numpy as np
import pytest

from tests import delta_reference as R


@pytest.mark.parametrize("seed", range(2))
def test_gradients_are_differences(seed):
    r = np.random.RandomState(seed)
    rows, heads, key_heads, dk, dv, offsets, scale = 9, 4, 2, 5, 3, [1, 4, 4, 8], 0.7
    x = dict(q=r.randn(rows, key_heads, dk), k=r.randn(rows, key_heads, dk), v=r.randn(rows, heads, dv),
             decay=-np.abs(r.randn(rows, heads)), beta=r.rand(rows, heads), init=r.randn(3, heads, dv, dk))
    x["k"] /= np.linalg.norm(x["k"], axis=2, keepdims=True)
    go, gl = r.randn(rows, heads, dv), r.randn(3, heads, dv, dk)

    def value():
        f = R.forward(x["q"], x["k"], x["v"], x["decay"], x["beta"], offsets, x["init"], scale)
        return (f.out * go).sum() + (f.last * gl).sum(), f

    g = R.backward(value()[1], go, gl)
    for name in ("q", "k", "v", "decay", "beta", "init"):
        flat = x[name].reshape(-1)
        got = np.broadcast_to(getattr(g, name), x[name].shape).reshape(-1)
        for i in r.choice(flat.size, min(flat.size, 6), replace=False):
            h, old = 1e-6, flat[i]
            flat[i] = old + h
            up = value()[0]
            flat[i] = old - h
            down = value()[0]
            flat[i] = old
            assert abs((up - down) / (2 * h) - got[i]) <= 1e-7 * (1 + abs(got[i])) * 50, (name, i)
