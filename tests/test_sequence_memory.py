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


# Matrices of 300 rows x 64 float32 elements, 76800 bytes; a row is 256 bytes.
ROW, MATRIX, STATES = 256, 300 * 256, 3 * 256


@pytest.mark.parametrize("kw", [
    dict(out=place(1, ROW)), dict(out=place(2, 4)), dict(out=place(1, MATRIX - 4)),  # shifted against an input
    dict(out=place(1), os=128), dict(out=place(2), gs=128, xs=128),                  # another stride
    dict(out=place(1, 128), os=128, gs=128),                                         # half a row aside, strided
    dict(last=place(4), ins=0), dict(last=place(4), ins=128), dict(last=place(4, ROW)),
    dict(last=place(1)), dict(last=place(3, MATRIX - 4)), dict(out=place(4)),
    dict(saved=place(1)), dict(saved=place(3)), dict(saved=place(4)), dict(saved=place(5, STATES - 4)),
    dict(temp=place(3)), dict(temp=place(6)), dict(temp=place(1, MATRIX - 16)),
    dict(offsets=place(3), out=place(3)), dict(offsets=place(5, 4)), dict(offsets=place(7, 4)),
    dict(dtype=L.BF16, out=place(1, 2))])
def test_forward_refuses_overlaps(kw):
    assert forward(**kw) == L.ERR_INVALID_ARG


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_forward_within_one_buffer(cuda, dtype):
    # gate, input and output as columns of one buffer do not overlap
    import torch
    from tests import sequence_reference as R
    from tests.test_recurrence_gpu import Case, host

    c = Case([150, 150], 64, dtype, "sigmoid", seed=40)
    f = c.reference()
    buf = torch.full((300, 192), 77.0, dtype=c.gate.dtype, device="cuda")
    buf[:, :64], buf[:, 128:] = c.gate, c.x
    c.gate, c.x = buf[:, :64], buf[:, 128:]
    out, last = c.forward(out=buf[:, 64:128])
    R.assert_within(host(out), f["out"], f["out_err"], dtype, "out")
    R.assert_within(host(last), f["last"], f["last_err"], "f32", "last")


@pytest.mark.parametrize("kw", [
    dict(gg=place(1, ROW)), dict(gi=place(2, 4)), dict(gg=place(3, MATRIX - 4)),  # shifted against an input
    dict(gg=place(1), ggs=128), dict(gi=place(3), gs=128, xs=128, gos=128),       # another stride
    dict(gg=place(9)), dict(gi=place(8, ROW)),                                    # one gradient over the other
    dict(g0=place(5)), dict(g0=place(5, ROW)), dict(g0=place(4), ins=0), dict(g0=place(4, 4)),
    dict(g0=place(8)), dict(g0=place(1)), dict(g0=place(6)),
    dict(gg=place(6)), dict(gi=place(4)), dict(gg=place(5)),
    dict(temp=place(3)), dict(temp=place(6)), dict(temp=place(10)), dict(temp=place(4)),
    dict(offsets=place(8)), dict(offsets=place(10, 4)), dict(offsets=place(7, 4)),
    dict(dtype=L.BF16, gg=place(1, 2))])
def test_backward_refuses_overlaps(kw):
    assert backward(**kw) == L.ERR_INVALID_ARG


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_backward_within_one_buffer(cuda, dtype):
    # operands and gradients as columns of one buffer
    import torch
    from tests import sequence_reference as R
    from tests.test_recurrence_gpu import Case, host

    c = Case([150, 150], 64, dtype, "sigmoid", seed=41)
    f = c.reference()
    want = R.backward(f, host(c.grad_out), host(c.grad_last))
    buf = torch.full((300, 320), 77.0, dtype=c.gate.dtype, device="cuda")
    for name, at in (("gate", 0), ("x", 128), ("grad_out", 256)):
        buf[:, at:at + 64] = getattr(c, name)
        setattr(c, name, buf[:, at:at + 64])
    c.forward()
    gg, gi, g0 = c.backward(grad_gate=buf[:, 64:128], grad_in=buf[:, 192:256])
    R.assert_within(host(gg), want["grad_gate"], want["grad_gate_err"], dtype, "grad_gate")
    R.assert_within(host(gi), want["grad_in"], want["grad_in_err"], dtype, "grad_in")
    R.assert_within(host(g0), want["grad_init"], want["grad_init_err"], "f32", "grad_init")


@pytest.mark.gpu
def test_grad_init_in_the_place_of_init(cuda):
    # a state is read by the lanes that write its gradient later, and by no others
    import torch
    from lc_parallel_primitive_b200 import CommandList, DeviceLinearRecurrence, Stream
    from tests import sequence_reference as R
    from tests.test_recurrence_gpu import Case, host

    c = Case([3, 0, 300, 1, 1, 150], 72, "f32", "sigmoid", seed=42, packed=True)
    f = c.reference()
    want = R.backward(f, host(c.grad_out), host(c.grad_last))
    c.forward()
    m, cl = DeviceLinearRecurrence(), CommandList()
    m.create()
    gg, gi = c.matrix(), c.matrix()
    m.Backward(cl, c.temp, c.gate, c.x, c.saved, c.grad_out, gg, gi, c.sequences, d_init=c.init,
               d_grad_last=c.grad_last, d_grad_init=c.init)
    Stream() << cl.commit()
    torch.cuda.synchronize()
    R.assert_within(host(gg), want["grad_gate"], want["grad_gate_err"], "f32", "grad_gate")
    R.assert_within(host(gi), want["grad_in"], want["grad_in_err"], "f32", "grad_in")
    R.assert_within(host(c.init), want["grad_init"], want["grad_init_err"], "f32", "grad_init")


def step(gate=L.GATE_SIGMOID, dtype=L.F32, g=place(1), gs=64, x=place(2), xs=64, states=place(3), rows_in=300, parents=None,
         new=place(4), out=place(5), os=64, rows=300, d=64):
    return L.lib().lcpp_linear_recurrence_step(gate, dtype, g, gs, x, xs, states, rows_in, parents, new, out, os, rows, d,
                                               None)


@pytest.mark.parametrize("kw", [
    dict(new=place(3, ROW)), dict(new=place(3, 4)), dict(states=place(4, MATRIX - 4)),  # shifted states
    dict(out=place(3, ROW)), dict(out=place(3), os=128), dict(out=place(4, 4)),
    dict(dtype=L.BF16, out=place(3)), dict(dtype=L.BF16, out=place(4)),
    dict(out=place(1, ROW)), dict(out=place(2), os=128), dict(new=place(1, 4)),
    dict(parents=place(6), new=place(3)), dict(parents=place(6), out=place(3)),
    dict(parents=place(5, 4)), dict(parents=place(4, 4)),
    dict(parents=place(6), rows_in=400, out=place(3, MATRIX))])
def test_step_refuses_overlaps(kw):
    assert step(**kw) == L.ERR_INVALID_ARG


@pytest.mark.gpu
@pytest.mark.parametrize("out", ["gate", "in", "states", "new"])
def test_step_outputs_in_the_place_of_operands(cuda, out):
    # float32 without parents: every operand has the same layout, and each lane reads what it writes before
    import torch
    from lc_parallel_primitive_b200 import CommandList, DeviceLinearRecurrence, Stream
    from tests import sequence_reference as R
    from tests.test_recurrence_gpu import Case, host

    c = Case([1] * 33, 100, "f32", "sigmoid", seed=43)
    f = c.reference()
    new = torch.empty((33, 100), device="cuda")
    o = {"gate": c.gate, "in": c.x, "states": c.init, "new": new}[out]
    m, cl = DeviceLinearRecurrence(), CommandList()
    m.create()
    m.Step(cl, c.gate, c.x, c.init, new, o)
    Stream() << cl.commit()
    torch.cuda.synchronize()
    R.assert_within(host(new), f["out"], f["out_err"], "f32", "states")
    R.assert_within(host(o), f["out"], f["out_err"], "f32", "out")


@pytest.mark.gpu
def test_step_within_one_buffer(cuda):
    # old and new states as the halves of one buffer, gate, input and output as columns of another
    import torch
    from lc_parallel_primitive_b200 import CommandList, DeviceLinearRecurrence, Stream
    from tests import sequence_reference as R
    from tests.test_recurrence_gpu import Case, host

    c = Case([1] * 9, 72, "bf16", "sigmoid", seed=44)
    f = c.reference()
    states = torch.cat([c.init, torch.zeros_like(c.init)])
    buf = torch.cat([c.gate, c.x, torch.zeros_like(c.x)], dim=1)
    m, cl = DeviceLinearRecurrence(), CommandList()
    m.create()
    m.Step(cl, buf[:, :72], buf[:, 72:144], states[:9], states[9:], buf[:, 144:],
           d_parents=torch.arange(9, dtype=torch.int32, device="cuda"))
    Stream() << cl.commit()
    torch.cuda.synchronize()
    R.assert_within(host(states[9:]), f["out"], f["out_err"], "f32", "states")
    R.assert_within(host(buf[:, 144:]), f["out"], f["out_err"], "bf16", "out")


@pytest.mark.parametrize("kw", [
    dict(so=place(5)), dict(so=place(6, 28)), dict(to=place(6, 4)), dict(fo=place(4, 31)), dict(fo=place(5, 4)),
    dict(so=place(1)), dict(to=place(1, 3196)), dict(po=place(1, 1600)), dict(fo=place(1, 3199)),
    dict(temp=place(4)), dict(temp=place(1)), dict(temp=place(2)), dict(temp=place(3)), dict(fo=place(8)),
    dict(stride=200, to=place(1, 800 + 396))])
def test_select_refuses_overlaps(kw):
    # 8 rows of 100 float32 logits, 3200 bytes; outputs of 32 bytes (8 of finished)
    assert select(**kw) == L.ERR_INVALID_ARG


@pytest.mark.gpu
def test_select_within_one_buffer(cuda):
    # scores and choices as rows of one buffer, logits as columns of another
    import numpy as np
    import torch
    from lc_parallel_primitive_b200 import CommandList, DeviceBeamSearch, Stream, temp_buffer
    from tests import sequence_reference as R

    wide = torch.randn((8, 500), generator=torch.Generator().manual_seed(45)).cuda()
    logits = wide[:, 100:400]
    scores = torch.zeros((2, 4), device="cuda")
    scores[:] = torch.tensor([0.0, -0.5, -1.0, -1.5])
    words = torch.zeros((2, 2, 4), dtype=torch.int32, device="cuda")
    both = torch.stack([scores, torch.zeros_like(scores)])
    m, c = DeviceBeamSearch(), CommandList()
    m.create()
    m.Select(c, temp_buffer(m.GetTempStorageBytes(2, 4, 300)), logits, both[0], None, both[1], words[0], words[1], None)
    Stream() << c.commit()
    torch.cuda.synchronize()
    s, t, p, _, gap = R.beam_select(logits.cpu().numpy(), scores.cpu().numpy(), None, -1)
    assert (gap > 1e-4).all()  # no two choices of this seed that rounding could swap
    assert np.allclose(both[1].cpu().numpy(), s, rtol=0, atol=1e-5)
    assert np.array_equal(words[0].cpu().numpy(), t) and np.array_equal(words[1].cpu().numpy(), p)


def reorder(x=place(1), lin=256, rin=64, out=place(2), lout=256, rout=64, parents=place(3), layers=2, rows_in=4, rows=4,
            width=64):
    return L.lib().lcpp_beam_reorder(x, lin, rin, out, lout, rout, parents, layers, rows_in, rows, width, None)


@pytest.mark.parametrize("kw", [
    dict(out=place(1)), dict(out=place(1, 448)), dict(x=place(2, 255)), dict(out=place(1, 64), lin=512, lout=512),
    dict(out=place(1, 200), lin=512, lout=512), dict(out=place(1, 300), lin=512, lout=512),  # into the next layer
    dict(out=place(1, 63), lin=512, lout=512, rin=128, rout=128), dict(out=place(1, 65), lin=512, lout=512, rin=128, rout=128),
    dict(out=place(1, 256), lin=512, lout=256), dict(out=place(1, 64), lin=0)])
def test_reorder_refuses_overlaps(kw):
    assert reorder(**kw) == L.ERR_INVALID_ARG


@pytest.mark.gpu
@pytest.mark.parametrize("split", [1, 2])
@pytest.mark.parametrize("width", [16, 33])
def test_reorder_between_halves_of_one_buffer(cuda, split, width):
    # (layers, 2, rows, width) and (layers, rows, 2, width): old and new states alternate, and do not overlap
    import torch
    from lc_parallel_primitive_b200 import CommandList, DeviceBeamSearch, Stream

    shape = (3, 2, 5, width) if split == 1 else (3, 5, 2, width)
    buf = torch.randn(shape, device="cuda")
    old, new = buf.unbind(split)
    parents = torch.tensor([4, 0, 0, -1, 2], dtype=torch.int32, device="cuda")
    want = torch.where(parents[:, None] >= 0, old[:, parents.clamp(min=0).long()], torch.zeros((), device="cuda"))
    before = old.clone()
    m, c = DeviceBeamSearch(), CommandList()
    m.create()
    m.Reorder(c, old, new, parents)
    Stream() << c.commit()
    torch.cuda.synchronize()
    assert torch.equal(new, want) and torch.equal(old, before)


@pytest.mark.parametrize("kw", [
    dict(lout=64), dict(lout=128), dict(lout=192), dict(lout=191, rout=128), dict(lout=100, rout=70, layers=3),
    dict(lout=130, rout=64, layers=3, rows=3)])
def test_reorder_refuses_rows_of_layers_over_each_other(kw):
    # two layers' rows in one place would be written in any order
    assert reorder(**kw) == L.ERR_INVALID_ARG


@pytest.mark.gpu
@pytest.mark.parametrize("layers,rows,layer,row", [(3, 4, 64, 192), (3, 4, 64, 200), (3, 4, 320, 64), (2, 2, 96, 224),
                                                   (3, 4, 160, 64), (2, 4, 192, 128)])
def test_reorder_to_interleaved_layers(cuda, layers, rows, layer, row):
    # rows of 32 bytes whose places are apart, though not all one behind the other
    import torch
    from lc_parallel_primitive_b200 import CommandList, DeviceBeamSearch, Stream

    places = sorted(l * layer + i * row for l in range(layers) for i in range(rows))
    assert all(b - a >= 32 for a, b in zip(places, places[1:]))
    x = torch.randint(0, 255, (layers, rows, 32), device="cuda", dtype=torch.uint8)
    buf = torch.full((2 * layer + 3 * row + 32,), 7, dtype=torch.uint8, device="cuda")
    out = buf.as_strided((layers, rows, 32), (layer, row, 1))
    m, c = DeviceBeamSearch(), CommandList()
    m.create()
    m.Reorder(c, x, out, torch.arange(rows - 1, -1, -1, dtype=torch.int32, device="cuda"))
    Stream() << c.commit()
    torch.cuda.synchronize()
    assert torch.equal(out, x.flip(1))


@pytest.mark.gpu
@pytest.mark.parametrize("eos", [1 << 32, (1 << 32) + 2, 1 << 31, -(1 << 40)])
def test_select_refuses_an_end_token_that_is_none(cuda, eos):
    # not the token that its lowest 32 bits are
    import torch
    from lc_parallel_primitive_b200 import CommandList, DeviceBeamSearch, temp_buffer

    z, s = torch.zeros((4, 10), device="cuda"), torch.zeros((1, 4), device="cuda")
    i, m, c = torch.zeros((1, 4), dtype=torch.int32, device="cuda"), DeviceBeamSearch(), CommandList()
    with pytest.raises(ValueError, match="eos_token"):
        m.Select(c, temp_buffer(m.GetTempStorageBytes(1, 4, 10)), z, s, None, s.clone(), i, i.clone(), None, eos_token=eos)
    assert len(c) == 0


@pytest.mark.parametrize("kw", [dict(parents=place(2)), dict(parents=place(2, 500)), dict(out=place(3, 8))])
def test_reorder_refuses_outputs_over_parents(kw):
    assert reorder(**kw) == L.ERR_INVALID_ARG


@pytest.mark.gpu
def test_reorder_from_no_rows(cuda):
    # an empty pool has no memory; its negative parents give zeros, as everywhere
    import torch
    from lc_parallel_primitive_b200 import CommandList, DeviceBeamSearch, Stream, last_device_error

    out = torch.full((2, 3, 40), 7.0, device="cuda")
    m, c = DeviceBeamSearch(), CommandList()
    m.create()
    m.Reorder(c, torch.empty((2, 0, 40), device="cuda"), out, torch.full((3,), -1, dtype=torch.int32, device="cuda"))
    Stream() << c.commit()
    torch.cuda.synchronize()
    assert (out == 0).all() and last_device_error() == L.OK


@pytest.mark.gpu
def test_empty_tensors_have_no_strides(cuda):
    # as they come from numpy, where an empty array's strides say nothing
    import numpy as np
    import torch
    from lc_parallel_primitive_b200 import CommandList, DeviceLinearRecurrence, Stream, temp_buffer

    def empty():
        return torch.from_numpy(np.empty((0, 8), np.float32)).as_strided((0, 8), (1, 0)).cuda().as_strided((0, 8), (1, 0))

    m, c = DeviceLinearRecurrence(), CommandList()
    m.create()
    m.Forward(c, temp_buffer(m.GetTempStorageBytes(0, 8)), empty(), empty(), empty(), 4, d_init=empty())
    Stream() << c.commit()
    torch.cuda.synchronize()
