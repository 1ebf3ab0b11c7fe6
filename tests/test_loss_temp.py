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


@pytest.mark.parametrize("rows,vocab", [(16, 300000), (256, 262145), (1, 1000000)])
def test_float32_sums_of_the_hidden_gradient_are_of_4096_terms(rows, vocab):
    """64 splits at most, so a piece of G (three planes of 2 bytes, 256 rows) has 64 x 4096 tokens at most.  Beside it there
    are five planes of the weight and 64 sums of 256 rows."""
    g = size(L.F32, rows, 64, vocab, 1) - 10 * vocab * 64
    assert g <= 3 * 256 * 2 * 64 * 4096 + 64 * 256 * 64 * 4 + 4 * vocab + (1 << 20)
