"""Sizes of the cross entropy's temp buffer: what serves so many rows serves fewer."""
import time

import pytest

from lc_parallel_primitive_b200 import _lib as L


def size(dtype, rows, channels, vocab, backward, aligned=1):
    return L.lib().lcpp_cross_entropy_temp_bytes(dtype, rows, channels, vocab, backward, aligned)


@pytest.mark.parametrize("dtype", [L.F32, L.F16, L.BF16])
@pytest.mark.parametrize("channels,vocab", [(4096, 128000), (1000, 100003), (64, 300), (40, 33000)])
@pytest.mark.parametrize("backward", [0, 1])
def test_a_buffer_for_more_rows_serves_fewer(dtype, channels, vocab, backward):
    sizes = [size(dtype, r, channels, vocab, backward) for r in range(128, 20000, 128)]
    assert all(a <= b for a, b in zip(sizes, sizes[1:]))


def test_large_batches_are_sized_at_once():
    start = time.perf_counter()
    assert size(L.BF16, 1 << 24, 1024, 32000, 1) > 1 << 35
    assert time.perf_counter() - start < 1.0
