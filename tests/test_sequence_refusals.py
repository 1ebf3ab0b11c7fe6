"""What the sequence operators refuse, at the C ABI (no GPU needed) and in Python."""
import ctypes

import pytest

from lc_parallel_primitive_b200 import _lib as L

BAD = ctypes.c_void_p(256)
BIG = 1 << 40


def forward(gate=L.GATE_SIGMOID, dtype=L.BF16, g=BAD, gs=64, x=BAD, xs=64, out=BAD, os=64, rows=10, d=64, seqs=1,
            length=10, offsets=None, temp=BAD, nbytes=BIG):
    return L.lib().lcpp_linear_recurrence_forward(gate, dtype, g, gs, x, xs, out, os, rows, d, seqs, length, offsets,
                                                  None, 0, None, None, temp, nbytes, None)


def backward(gate=L.GATE_SIGMOID, dtype=L.BF16, saved=BAD, gg=BAD, ggs=64, gi=BAD, rows=10, seqs=1, nbytes=BIG, go=BAD,
             gos=64):
    return L.lib().lcpp_linear_recurrence_backward(gate, dtype, BAD, 64, BAD, 64, saved, None, 0, go, gos, None, gg, ggs,
                                                   gi, 64, None, rows, 64, seqs, 10, None, BAD, nbytes, None)


def step(gate=L.GATE_SIGMOID, dtype=L.BF16, g=BAD, gs=64, states=BAD, rows_in=10, parents=None,
         states_out=ctypes.c_void_p(1 << 20), out=BAD, rows=10):
    return L.lib().lcpp_linear_recurrence_step(gate, dtype, g, gs, BAD, 64, states, rows_in, parents, states_out, out, 64,
                                               rows, 64, None)


def select(dtype=L.BF16, z=BAD, stride=100, scores=BAD, out=BAD, batches=2, beams=4, vocab=100, eos=-1, nbytes=BIG):
    return L.lib().lcpp_beam_select(dtype, z, stride, scores, None, out, BAD, BAD, None, batches, beams, vocab, eos, BAD,
                                    nbytes, None)


def reorder(x=BAD, row_in=64, out=ctypes.c_void_p(1 << 30), row_out=64, parents=BAD, layers=2, rows_in=4, rows=4,
            width=64):
    return L.lib().lcpp_beam_reorder(x, 4 * 64, row_in, out, 4 * 64, row_out, parents, layers, rows_in, rows, width, None)


@pytest.mark.parametrize("kw", [dict(gate=2), dict(gate=-1), dict(dtype=L.I32), dict(dtype=L.F64), dict(dtype=L.NONE),
                                dict(g=None), dict(x=None), dict(out=None), dict(gs=63), dict(xs=10), dict(os=0),
                                dict(gs=1 << 31), dict(rows=9), dict(seqs=2), dict(seqs=0), dict(rows=1 << 33),
                                dict(d=1 << 21, gs=1 << 21, xs=1 << 21, os=1 << 21)])
def test_forward_refuses(kw):
    assert forward(**kw) == L.ERR_INVALID_ARG


def test_temp_too_small():
    assert forward(nbytes=8) == L.ERR_TEMP_TOO_SMALL and forward(temp=None) == L.ERR_TEMP_TOO_SMALL
    assert backward(nbytes=8) == L.ERR_TEMP_TOO_SMALL
    assert select(nbytes=8) == L.ERR_TEMP_TOO_SMALL


def test_nothing_to_do():
    assert forward(d=0) == L.OK and forward(rows=0, seqs=0) == L.OK
    assert step(rows=0) == L.OK and select(batches=0) == L.OK
    assert reorder(rows=0) == L.OK and reorder(layers=0) == L.OK and reorder(width=0) == L.OK


@pytest.mark.parametrize("kw", [dict(gate=5), dict(dtype=L.I64), dict(saved=None), dict(gg=None), dict(gi=None),
                                dict(ggs=63), dict(gos=63), dict(rows=11), dict(seqs=0)])
def test_backward_refuses(kw):
    assert backward(**kw) == L.ERR_INVALID_ARG


@pytest.mark.parametrize("kw", [dict(gate=5), dict(dtype=L.U32), dict(g=None), dict(gs=63), dict(states_out=None),
                                dict(rows_in=9), dict(rows=1 << 31),
                                dict(parents=BAD, states_out=BAD),  # in place, but rows move
                                dict(parents=BAD, states_out=ctypes.c_void_p(256 + 9 * 64 * 4))])
def test_step_refuses(kw):
    assert step(**kw) == L.ERR_INVALID_ARG


@pytest.mark.parametrize("kw", [dict(dtype=L.I32), dict(beams=0), dict(beams=33), dict(vocab=0), dict(vocab=1 << 31),
                                dict(stride=99), dict(z=None), dict(scores=None), dict(out=None), dict(eos=100),
                                dict(batches=1 << 30)])
def test_select_refuses(kw):
    assert select(**kw) == L.ERR_INVALID_ARG


@pytest.mark.parametrize("kw", [dict(x=None), dict(out=None), dict(parents=None), dict(row_in=63), dict(row_out=63),
                                dict(out=BAD), dict(out=ctypes.c_void_p(256 + 7 * 64)), dict(rows=1 << 31)])
def test_reorder_refuses(kw):
    assert reorder(**kw) == L.ERR_INVALID_ARG


ODD = ctypes.c_void_p(257)


@pytest.mark.parametrize("call", [
    lambda: forward(g=ODD), lambda: forward(out=ODD), lambda: forward(dtype=L.F32, x=ctypes.c_void_p(258)),
    lambda: backward(gg=ODD), lambda: backward(saved=ctypes.c_void_p(258)), lambda: backward(go=ODD),
    lambda: step(g=ODD), lambda: step(states=ctypes.c_void_p(258)), lambda: step(out=ODD),
    lambda: select(z=ODD), lambda: select(scores=ctypes.c_void_p(258)), lambda: reorder(parents=ODD)])
def test_a_part_of_an_element_is_no_address(call):
    assert call() == L.ERR_INVALID_ARG


@pytest.mark.parametrize("place", ["scores", "tokens", "parents", "finished"])
@pytest.mark.parametrize("onto", ["scores", "finished"])
def test_select_refuses_outputs_over_inputs(place, onto):
    at = {n: ctypes.c_void_p((i + 2) << 16) for i, n in enumerate(["scores", "tokens", "parents", "finished"])}
    inputs = dict(scores=ctypes.c_void_p(1 << 12), finished=ctypes.c_void_p(1 << 13))
    at[place] = ctypes.c_void_p(inputs[onto].value + 4)
    assert L.lib().lcpp_beam_select(L.BF16, ctypes.c_void_p(1 << 30), 100, inputs["scores"], inputs["finished"], at["scores"],
                                    at["tokens"], at["parents"], at["finished"], 2, 4, 100, -1, BAD, BIG,
                                    None) == L.ERR_INVALID_ARG


def test_reorder_refuses_layers_over_each_other():
    out = ctypes.c_void_p(1 << 30)
    assert L.lib().lcpp_beam_reorder(BAD, 256, 64, out, 63, 64, BAD, 2, 4, 4, 64, None) == L.ERR_INVALID_ARG


def test_sizes():
    lib = L.lib()
    assert lib.lcpp_linear_recurrence_saved_bytes(129, 64) >= 2 * 64 * 4
    assert lib.lcpp_linear_recurrence_temp_bytes(1 << 20, 4096) > 0
    assert lib.lcpp_beam_select_temp_bytes(4, 4, 32000) > 0 and lib.lcpp_beam_select_temp_bytes(4, 33, 32000) == 0
    # the other primitives keep their types
    assert lib.lcpp_dtype_size(L.BF16) == 0 and lib.lcpp_reduce_temp_bytes(L.BF16, 10) == 0
    assert lib.lcpp_segment_reduce_fixed(0, L.F16, BAD, BAD, 4, 4, None) == L.ERR_INVALID_ARG


def test_python_refuses_host_tensors():
    import torch
    from lc_parallel_primitive_b200 import CommandList, DeviceBeamSearch, DeviceLinearRecurrence

    x = torch.zeros((4, 8))
    c = CommandList()
    with pytest.raises(ValueError, match="CUDA"):
        DeviceLinearRecurrence().Forward(c, x, x, x, x, 4)
    with pytest.raises(ValueError, match="CUDA"):
        DeviceBeamSearch().Reorder(c, x, x, torch.zeros(4, dtype=torch.int32))
    with pytest.raises(TypeError, match="element type"):
        DeviceLinearRecurrence().Forward(c, x, x.int(), x, x, 4)
    with pytest.raises(ValueError, match="mode"):
        DeviceLinearRecurrence().Forward(c, x, x, x, x, 4, mode="tanh")
    assert len(c) == 0


@pytest.mark.gpu
def test_python_refuses_wrong_buffers(cuda):
    import torch
    from lc_parallel_primitive_b200 import CommandList, DeviceBeamSearch, DeviceLinearRecurrence, temp_buffer

    m, bs, c = DeviceLinearRecurrence(), DeviceBeamSearch(), CommandList()
    x = torch.zeros((6, 8), device="cuda")
    temp = temp_buffer(m.GetTempStorageBytes(6, 8))

    def refused(error, match, fn, *a, **kw):
        with pytest.raises(error, match=match):
            fn(c, *a, **kw)

    refused(TypeError, "same element type", m.Forward, temp, x, x.half(), x, 6)
    refused(ValueError, "same shape", m.Forward, temp, x, x[:5], x, 6)
    refused(ValueError, "adjacent", m.Forward, temp, x, torch.zeros((8, 6), device="cuda").t(), x, 6)
    refused(ValueError, "overlap", m.Forward, temp, x, x[:1].expand(6, 8), x, 6)
    refused(ValueError, "whole number", m.Forward, temp, x, x, x, 4)
    refused(TypeError, "32-bit", m.Forward, temp, x, x, x, torch.tensor([0, 6], device="cuda"))
    refused(ValueError, "d_init must have the shape", m.Forward, temp, x, x, x, 6, d_init=x)
    refused(ValueError, "d_last must have the shape", m.Forward, temp, x, x, x, 6, d_last=x)
    refused(ValueError, "batch stride", m.Forward, temp, torch.zeros((2, 4, 8), device="cuda")[:, :3], x, x, 3)
    refused(ValueError, "d_saved", m.Backward, temp, x, x, None, x, x, x, 6)
    refused(ValueError, "GetSavedStateBytes", m.Backward, temp, x, x, temp[:1], x, x, x, 6)
    refused(ValueError, "one device", m.Forward, temp.cpu(), x, x, x, 6)
    refused(ValueError, "shape", m.Step, x, x, x, torch.zeros((5, 8), device="cuda"))
    refused(TypeError, "element type", m.Step, x, x, x, x.clone(), None, d_parents=torch.zeros(6, device="cuda"))
    s = torch.zeros((2, 3), device="cuda")
    i = torch.zeros((2, 3), dtype=torch.int32, device="cuda")
    refused(ValueError, "row for each score", bs.Select, temp, x[:5], s, None, s.clone(), i, i.clone(), None)
    refused(TypeError, "d_tokens_out", bs.Select, temp, x, s, None, s.clone(), i.long(), i.clone(), None)
    refused(ValueError, "same layers", bs.Reorder, x, torch.zeros((6, 9), device="cuda"), i.reshape(-1))
    assert len(c) == 0


@pytest.mark.gpu
def test_status_is_raised_at_commit(cuda):
    import torch
    from lc_parallel_primitive_b200 import CommandList, DeviceLinearRecurrence, LcppError, Stream, temp_buffer

    m, c = DeviceLinearRecurrence(), CommandList()
    x = torch.zeros((600, 80), device="cuda")
    m.Forward(c, torch.zeros(1, dtype=torch.uint8, device="cuda"), x, x, torch.empty_like(x), 600)
    with pytest.raises(LcppError) as e:
        Stream() << c.commit()
    assert e.value.status == L.ERR_TEMP_TOO_SMALL
    m.Step(c, x, x, x, x, None, d_parents=torch.zeros(600, dtype=torch.int32, device="cuda"))
    with pytest.raises(LcppError) as e:
        Stream() << c.commit()
    assert e.value.status == L.ERR_INVALID_ARG
    assert temp_buffer(m.GetTempStorageBytes(600, 80)).is_cuda
