"""What the sequence operators refuse about the memory that they are given: addresses and overlaps.

At the C ABI with made-up addresses; every call here is refused on the host, so nothing is launched.
"""
import ctypes

import pytest

from lc_parallel_primitive_b200 import _lib as L

BIG = 1 << 40


def place(i, shift=0):
    """Addresses that are far apart and aligned."""
    return (i << 44) + shift


def forward(gate=L.GATE_SIGMOID, dtype=L.F32, g=place(1), gs=64, x=place(2), xs=64, out=place(3), os=64, rows=300, d=64,
            seqs=3, length=100, offsets=None, init=place(4), ins=64, last=place(5), saved=place(6), temp=place(7),
            nbytes=BIG):
    return L.lib().lcpp_linear_recurrence_forward(gate, dtype, g, gs, x, xs, out, os, rows, d, seqs, length, offsets,
                                                  init, ins, last, saved, temp, nbytes, None)


def backward(gate=L.GATE_SIGMOID, dtype=L.F32, g=place(1), gs=64, x=place(2), xs=64, saved=place(6), init=place(4), ins=64,
             go=place(3), gos=64, gl=place(5), gg=place(8), ggs=64, gi=place(9), gis=64, g0=place(10), rows=300, d=64,
             seqs=3, length=100, offsets=None, temp=place(7), nbytes=BIG):
    return L.lib().lcpp_linear_recurrence_backward(gate, dtype, g, gs, x, xs, saved, init, ins, go, gos, gl, gg, ggs, gi,
                                                   gis, g0, rows, d, seqs, length, offsets, temp, nbytes, None)


def select(dtype=L.F32, z=place(1), stride=100, scores=place(2), finished=place(3), so=place(4), to=place(5), po=place(6),
           fo=place(7), batches=2, beams=4, vocab=100, eos=-1, temp=place(8), nbytes=BIG):
    return L.lib().lcpp_beam_select(dtype, z, stride, scores, finished, so, to, po, fo, batches, beams, vocab, eos, temp,
                                    nbytes, None)


@pytest.mark.parametrize("shift", [1, 4, 8])
@pytest.mark.parametrize("call", [forward, backward])
def test_recurrence_temp_holds_vectors(call, shift):
    # the look-back's records are read 16 bytes at a time
    assert call(temp=place(7, shift)) == L.ERR_INVALID_ARG


@pytest.mark.parametrize("shift", [1, 4])
def test_selection_temp_holds_keys(shift):
    # keys are 8 bytes
    assert select(temp=place(8, shift)) == L.ERR_INVALID_ARG


@pytest.mark.parametrize("call", [forward, backward])
def test_offsets_are_whole_words(call):
    assert call(offsets=place(11, 2)) == L.ERR_INVALID_ARG


@pytest.mark.parametrize("view", ["strided", "expanded"])
def test_python_temp_is_one_piece(view):
    # its size is the number of bytes from its address on, which a view with gaps or repeats does not have
    import torch
    from lc_parallel_primitive_b200 import CommandList, DeviceBeamSearch, DeviceLinearRecurrence

    temp = {"strided": torch.zeros(1 << 16, dtype=torch.int32)[::2],
            "expanded": torch.zeros(1, dtype=torch.int32).expand(1 << 16)}[view]
    x, c = torch.zeros((4, 8)), CommandList()
    s, i = torch.zeros((1, 4)), torch.zeros((1, 4), dtype=torch.int32)
    m = DeviceLinearRecurrence()
    with pytest.raises(ValueError, match="temp_storage must be contiguous"):
        m.Forward(c, temp, x, x, x, 4)
    with pytest.raises(ValueError, match="temp_storage must be contiguous"):
        m.Backward(c, temp, x, x, x, x, x, x, 4)
    with pytest.raises(ValueError, match="temp_storage must be contiguous"):
        DeviceBeamSearch().Select(c, temp, x, s, None, s, i, i, None)
    assert len(c) == 0
