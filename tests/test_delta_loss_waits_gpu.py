"""Waits that are cut short: a status, and the context goes on."""
import numpy as np
import pytest

from lc_parallel_primitive_b200 import _lib as L
from tests.test_delta_gpu import Case, host

pytestmark = pytest.mark.gpu


@pytest.fixture
def one_poll(cuda):
    import torch

    lib = L.lib()
    torch.cuda.synchronize()
    L.check(lib.lcpp_set_spin_limit(1))
    yield
    torch.cuda.synchronize()
    L.check(lib.lcpp_set_spin_limit(0))


@pytest.mark.parametrize("dtype,lengths,heads,dk,dv", [("bf16", [500, 300], 4, 128, 128), ("f32", [700], 2, 128, 96), ("f16", [4200], 1, 64, 40)])
def test_delta_rule(one_poll, dtype, lengths, heads, dk, dv):
    """A poll may last until what it waits for is there: the call then is as ever, and else its status says that it is not."""
    import torch
    from lc_parallel_primitive_b200 import last_device_error

    c = Case(lengths, heads, heads, dk, dv, dtype, seed=61)
    L.check(L.lib().lcpp_set_spin_limit(0))
    want = [t.clone() for t in c.run()]
    g = c.back()
    want += [g.q, g.k, g.v, g.decay, g.beta, g.init]
    L.check(L.lib().lcpp_set_spin_limit(1))
    for _ in range(5):
        got = [t.clone() for t in c.run(check=False)]
        g = c.back(check=False)
        got += [g.q, g.k, g.v, g.decay, g.beta, g.init]
        torch.cuda.synchronize()
        status = last_device_error()
        assert status in (0, L.ERR_LOOKBACK_TIMEOUT)
        if status == 0:
            assert all(torch.equal(a, b) for a, b in zip(got, want))
    L.check(L.lib().lcpp_set_spin_limit(0))
    got = [t.clone() for t in c.run()]
    g = c.back()
    got += [g.q, g.k, g.v, g.decay, g.beta, g.init]
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert all(np.isfinite(host(t)).all() for t in got)


def test_cross_entropy(one_poll):
    """The products of a tile of 4096 channels take longer than a poll of a microsecond."""
    import torch
    from lc_parallel_primitive_b200 import last_device_error
    from tests.test_cross_entropy_gpu import Case as Loss

    lib = L.lib()
    L.check(lib.lcpp_set_spin_limit(0))
    c = Loss(600, 4096, 2000, "bf16", seed=62)
    want = [t.clone() for t in c.run()]
    L.check(lib.lcpp_set_spin_limit(1))
    for _ in range(3):
        c.run(check=False)
        torch.cuda.synchronize()
        assert last_device_error() == L.ERR_LOOKBACK_TIMEOUT
    L.check(lib.lcpp_set_spin_limit(0))
    assert all(torch.equal(a, b) for a, b in zip(c.run(), want))
