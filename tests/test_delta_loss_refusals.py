"""What the delta rule and the cross entropy refuse, at the C ABI with made-up addresses (nothing is launched) and in
Python."""
import ctypes

import pytest

from lc_parallel_primitive_b200 import _lib as L

BIG = 1 << 42
ROWS, HEADS, KEYS, DK, DV = 300, 4, 2, 64, 32


def place(i, shift=0):
    return (i << 44) + shift


def shape(rows=ROWS, seqs=3, length=100, offsets=None, heads=HEADS, key_heads=KEYS, dk=DK, dv=DV, scale=0.125):
    return L.DeltaShape(rows, seqs, length, offsets, heads, key_heads, dk, dv, scale)


def inputs(q=place(1), k=place(2), v=place(3), qs=KEYS * DK, ks=KEYS * DK, vs=HEADS * DV, decay=place(4), beta=place(5), ds=HEADS,
           bs=HEADS, init=place(6)):
    return L.DeltaInputs(q, k, v, qs, ks, vs, decay, beta, ds, bs, init)


def split(kw, names):
    return {k: kw[k] for k in kw if k in names}, {k: kw[k] for k in kw if k not in names}


SHAPE = ("rows", "seqs", "length", "offsets", "heads", "key_heads", "dk", "dv", "scale")
INPUTS = ("q", "k", "v", "qs", "ks", "vs", "decay", "beta", "ds", "bs", "init")


def forward(dtype=L.F32, out=place(7), os=HEADS * DV, last=place(8), saved=place(9), temp=place(10), nbytes=BIG, **kw):
    s, rest = split(kw, SHAPE)
    return L.lib().lcpp_delta_rule_forward(dtype, shape(**s), inputs(**rest), out, os, last, saved, temp, nbytes, None)


def backward(dtype=L.F32, saved=place(9), go=place(7), gos=HEADS * DV, gl=place(8), gq=place(11), gk=place(12), gv=place(13),
             gd=place(14), gb=place(15), g0=place(16), temp=place(10), nbytes=BIG, **kw):
    s, rest = split(kw, SHAPE)
    return L.lib().lcpp_delta_rule_backward(dtype, shape(**s), inputs(**rest), saved,
                                            L.DeltaGrads(go, gos, gl, gq, gk, gv, gd, gb, g0), temp, nbytes, None)


def step(dtype=L.F32, rows_in=ROWS, parents=None, new=place(8), out=place(7), os=HEADS * DV, **kw):
    s, rest = split(kw, SHAPE)
    return L.lib().lcpp_delta_rule_step(dtype, shape(**s), inputs(**rest), rows_in, parents, new, out, os, None)


def loss(dtype=L.F32, h=place(1), hs=64, w=place(2), ws=64, t=place(3), out=place(4), logsum=place(5), rows=300, d=64, v=1000,
         temp=place(6), nbytes=BIG):
    return L.lib().lcpp_cross_entropy_forward(dtype, h, hs, w, ws, t, out, logsum, rows, d, v, temp, nbytes, None)


def loss_back(dtype=L.F32, h=place(1), hs=64, w=place(2), ws=64, t=place(3), logsum=place(5), g=place(4), gs=1, gh=place(7),
              ghs=64, gw=place(8), gws=64, rows=300, d=64, v=1000, temp=place(6), nbytes=BIG):
    return L.lib().lcpp_cross_entropy_backward(dtype, h, hs, w, ws, t, logsum, g, gs, gh, ghs, gw, gws, rows, d, v, temp, nbytes, None)


SHAPES = [dict(heads=0), dict(key_heads=0), dict(key_heads=3), dict(heads=1 << 17, key_heads=1), dict(dk=0), dict(dv=0), dict(dk=129),
          dict(dv=129)]
SEQUENCES = [dict(length=99), dict(seqs=4), dict(seqs=0), dict(rows=1 << 33), dict(seqs=1 << 29), dict(offsets=place(20, 2))]
STRIDES = [dict(qs=KEYS * DK - 1), dict(ks=0), dict(vs=HEADS * DV - 1), dict(ds=3), dict(bs=3), dict(qs=1 << 31)]
MISSING = [dict(q=None), dict(k=None), dict(v=None), dict(beta=None)]
ODD = [dict(q=place(1, 2)), dict(k=place(2, 1)), dict(v=place(3, 2)), dict(decay=place(4, 2)), dict(beta=place(5, 1)),
       dict(init=place(6, 2)), dict(dtype=L.BF16, q=place(1, 1))]
TYPES = [dict(dtype=L.I32), dict(dtype=L.F64), dict(dtype=L.NONE), dict(dtype=-1)]


@pytest.mark.parametrize("kw", SHAPES + SEQUENCES + STRIDES + MISSING + ODD + TYPES + [
    dict(out=None), dict(os=HEADS * DV - 1), dict(out=place(7, 2)), dict(last=place(8, 1)), dict(saved=place(9, 8)), dict(temp=place(10, 8))])
def test_forward_refuses(kw):
    assert forward(**kw) == L.ERR_INVALID_ARG


@pytest.mark.parametrize("kw", SHAPES + SEQUENCES + STRIDES + MISSING + ODD + TYPES + [
    dict(saved=None), dict(gq=None), dict(gk=None), dict(gv=None), dict(gb=None), dict(gos=5), dict(go=place(7, 1)), dict(gd=place(14, 2)),
    dict(saved=place(9, 8)), dict(temp=place(10, 4))])
def test_backward_refuses(kw):
    assert backward(**kw) == L.ERR_INVALID_ARG


@pytest.mark.parametrize("kw", SHAPES + STRIDES + MISSING + ODD + TYPES + [
    dict(new=None), dict(out=None), dict(rows_in=ROWS - 1), dict(rows=1 << 31), dict(parents=place(21, 2)),
    dict(parents=place(21), new=place(6)), dict(new=place(6, 4)), dict(new=place(6, ROWS * HEADS * DV * DK * 4 - 4))])
def test_step_refuses(kw):
    assert step(**kw) == L.ERR_INVALID_ARG


# sizes in bytes, float32
QK, V, GATES, STATE = ROWS * KEYS * DK * 4, ROWS * HEADS * DV * 4, ROWS * HEADS * 4, 3 * HEADS * DV * DK * 4


@pytest.mark.parametrize("kw", [dict(out=place(1)), dict(out=place(2, QK - 4)), dict(out=place(3)), dict(out=place(4)), dict(out=place(5)),
                                dict(out=place(6)), dict(last=place(1)), dict(last=place(6, 4)), dict(last=place(7)), dict(temp=place(1)),
                                dict(temp=place(7)), dict(temp=place(8)), dict(temp=place(9)), dict(saved=place(3)), dict(saved=place(8)),
                                dict(offsets=place(7, 16)), dict(offsets=place(10, 16))])
def test_forward_refuses_overlaps(kw):
    assert forward(**kw) == L.ERR_INVALID_ARG


@pytest.mark.parametrize("name", ["gq", "gk", "gv", "gd", "gb", "g0", "temp"])
@pytest.mark.parametrize("at", [1, 2, 3, 4, 5, 6, 7, 8, 9, 11, 13, 14, 16])
def test_backward_refuses_overlaps(name, at):
    own = dict(gq=11, gk=12, gv=13, gd=14, gb=15, g0=16, temp=10)[name]
    if at != own:
        assert backward(**{name: place(at, 16)}) == L.ERR_INVALID_ARG


@pytest.mark.parametrize("kw", [dict(out=place(1)), dict(out=place(3)), dict(out=place(4)), dict(out=place(6)), dict(out=place(8)),
                                dict(new=place(2)), dict(new=place(5)), dict(parents=place(7, 4)), dict(parents=place(8, 4))])
def test_step_refuses_overlaps(kw):
    assert step(**kw) == L.ERR_INVALID_ARG


@pytest.mark.parametrize("kw", TYPES + [
    dict(h=None), dict(w=None), dict(t=None), dict(hs=63), dict(ws=63), dict(hs=1 << 31), dict(d=0), dict(v=0), dict(rows=1 << 25),
    dict(v=1 << 31), dict(d=1 << 21, hs=1 << 21, ws=1 << 21), dict(h=place(1, 2)), dict(w=place(2, 1)), dict(t=place(3, 2)),
    dict(temp=place(6, 16)), dict(dtype=L.BF16, h=place(1, 1))])
@pytest.mark.parametrize("call", [loss, loss_back])
def test_loss_refuses(call, kw):
    assert call(**kw) == L.ERR_INVALID_ARG


@pytest.mark.parametrize("kw", [dict(out=None, logsum=None), dict(out=place(4, 2)), dict(logsum=place(5, 1)), dict(out=place(1)),
                                dict(out=place(2, 4)), dict(out=place(3)), dict(logsum=place(4, 4)), dict(temp=place(4)), dict(temp=place(1, 32))])
def test_loss_forward_refuses(kw):
    assert loss(**kw) == L.ERR_INVALID_ARG


@pytest.mark.parametrize("kw", [dict(logsum=None), dict(g=None), dict(gh=None, gw=None), dict(ghs=63), dict(gws=63), dict(gh=place(7, 2)),
                                dict(g=place(4, 2)), dict(gs=1 << 31), dict(gh=place(1)), dict(gh=place(2, 256)), dict(gw=place(2)),
                                dict(gw=place(7, 64)), dict(gh=place(3)), dict(gw=place(4)), dict(gw=place(5)), dict(temp=place(7)),
                                dict(temp=place(8, 64)), dict(temp=place(4))])
def test_loss_backward_refuses(kw):
    assert loss_back(**kw) == L.ERR_INVALID_ARG


def test_temp_too_small():
    for call in (forward, backward, loss, loss_back):
        assert call(nbytes=8) == L.ERR_TEMP_TOO_SMALL and call(temp=None) == L.ERR_TEMP_TOO_SMALL


def test_nothing_to_do():
    assert forward(rows=0, seqs=0, length=0) == L.OK and backward(rows=0, seqs=0, length=0) == L.OK
    assert step(rows=0) == L.OK and loss(rows=0) == L.OK and loss_back(rows=0, gw=None) == L.OK


def test_sizes():
    lib = L.lib()
    small, large = (lib.lcpp_delta_rule_temp_bytes(L.BF16, shape(), b) for b in (0, 1))
    assert 0 < small < large and lib.lcpp_delta_rule_temp_bytes(L.I32, shape(), 0) == 0
    assert lib.lcpp_delta_rule_saved_bytes(shape()) > 0 and lib.lcpp_delta_rule_saved_bytes(shape(dk=200)) == 0
    small, large = (lib.lcpp_cross_entropy_temp_bytes(L.BF16, 300, 64, 1000, b, 1) for b in (0, 1))
    assert 0 < small <= large < lib.lcpp_cross_entropy_temp_bytes(L.BF16, 300, 64, 1000, 1, 0)
    assert lib.lcpp_cross_entropy_temp_bytes(L.I64, 300, 64, 1000, 1, 1) == 0
    assert lib.lcpp_delta_rule_temp_bytes(L.F32, None, 0) == 0
    assert lib.lcpp_delta_rule_forward(L.F32, None, None, None, 0, None, None, None, 0, None) == L.ERR_INVALID_ARG


def test_python_refuses_host_tensors():
    import torch
    from lc_parallel_primitive_b200 import CommandList, DeviceCrossEntropy, DeviceDeltaRule

    c = CommandList()
    q, g = torch.zeros(4, 2, 8), torch.zeros(4, 2)
    with pytest.raises(ValueError, match="CUDA"):
        DeviceDeltaRule().Forward(c, q, q, q, q, g, g, q, 4)
    with pytest.raises(ValueError, match="CUDA"):
        DeviceDeltaRule().Step(c, q, q, q, g, g, None, torch.zeros(4, 2, 8, 8), q)
    with pytest.raises(ValueError, match="d_saved"):
        DeviceDeltaRule().Backward(c, q, q, q, q, g, g, None, q, q, q, q, g, g, 4)
    with pytest.raises(TypeError, match="element type"):
        DeviceDeltaRule().Forward(c, q, q, q.half(), q, g, g, q, 4)
    x = torch.zeros(4, 8)
    with pytest.raises(ValueError, match="CUDA"):
        DeviceCrossEntropy().Forward(c, x, x, x, torch.zeros(4, dtype=torch.int32), x[:, 0])
    with pytest.raises(TypeError, match="unsupported"):
        DeviceCrossEntropy.GetTempStorageBytes(4, 8, 4, torch.int32)
    with pytest.raises(ValueError, match="temp_storage must be contiguous"):
        DeviceCrossEntropy().Forward(c, torch.zeros(1 << 16, dtype=torch.int32)[::2], x, x, torch.zeros(4, dtype=torch.int32), x[:, 0])
    assert len(c) == 0


@pytest.mark.gpu
def test_python_refuses_wrong_buffers(cuda):
    import torch
    from lc_parallel_primitive_b200 import CommandList, DeviceCrossEntropy, DeviceDeltaRule, LcppError, Stream, temp_buffer

    m, c = DeviceDeltaRule(), CommandList()
    new = lambda *s, t=torch.float32: torch.zeros(s, dtype=t, device="cuda")  # noqa: E731
    q, v, g, s = new(6, 2, 8), new(6, 4, 8), new(6, 4), new(1, 4, 8, 8)
    temp = temp_buffer(m.GetTempStorageBytes(6, 1, 4, 2, 8, 8, torch.float32))
    saved = temp_buffer(m.GetSavedStateBytes(6, 1, 4, 2, 8, 8))

    def refused(error, match, fn, *a, **kw):
        with pytest.raises(error, match=match):
            fn(c, *a, **kw)

    refused(ValueError, "same shape", m.Forward, temp, q, new(6, 1, 8), v, g, g, v, 6)
    refused(ValueError, "rows of d_q", m.Forward, temp, q, q, v[:5], g, g, v, 6)
    refused(ValueError, "whole number for each", m.Forward, temp, q, q, new(6, 3, 8), g, g, v, 6)
    refused(ValueError, "from 1 to 128", m.Forward, temp, new(6, 2, 129), new(6, 2, 129), v, g, g, v, 6)
    refused(ValueError, "heads of a row", m.Forward, temp, new(6, 8, 2).transpose(1, 2), q, v, g, g, v, 6)
    refused(ValueError, "overlap", m.Forward, temp, q[:1].expand(6, 2, 8), q, v, g, g, v, 6)
    refused(ValueError, "shape", m.Forward, temp, new(6, 16), q, v, g, g, v, 6)
    refused(TypeError, "element type", m.Forward, temp, q, q, v, g.half(), g, v, 6)
    refused(ValueError, "d_decay and d_beta", m.Forward, temp, q, q, v, g, new(6, 2), v, 6)
    refused(ValueError, "d_out", m.Forward, temp, q, q, v, g, g, q, 6)
    refused(ValueError, "d_init must have the shape", m.Forward, temp, q, q, v, g, g, v, 6, d_init=new(2, 4, 8, 8))
    refused(ValueError, "d_last must be contiguous", m.Forward, temp, q, q, v, g, g, v, 6, d_last=new(1, 4, 8, 16)[..., ::2])
    refused(ValueError, "whole number of sequences", m.Forward, temp, q, q, v, g, g, v, 4)
    refused(ValueError, "GetSavedStateBytes", m.Forward, temp, q, q, v, g, g, v, 6, d_saved=saved[:2])
    refused(ValueError, "d_grad_q must have the shape", m.Backward, temp, q, q, v, g, g, saved, v, v, q, v, g, g, 6)
    refused(ValueError, "d_grad_k must be contiguous", m.Backward, temp, q, q, v, g, g, saved, v, q, new(6, 2, 16)[..., ::2], v, g, g, 6)
    refused(ValueError, "d_states_out", m.Step, q, q, v, g, g, s, s, v)
    refused(ValueError, "one device", m.Forward, temp.cpu(), q, q, v, g, g, v, 6)
    e, x, w = DeviceCrossEntropy(), new(6, 8), new(9, 8)
    t, o = new(6, t=torch.int32), new(6)
    refused(ValueError, "d_weight must have the shape", e.Forward, temp, x, new(9, 7), t, o)
    refused(TypeError, "d_targets", e.Forward, temp, x, w, t.long(), o)
    refused(ValueError, "one for each row", e.Forward, temp, x, w, t[:5], o)
    refused(TypeError, "d_loss", e.Forward, temp, x, w, t, o.double())
    refused(ValueError, "d_logsum", e.Forward, temp, x, w, t, o, o[:5])
    refused(ValueError, "d_grad_loss", e.Backward, temp, x, w, t, o, new(12)[::2], x.clone(), w.clone())
    refused(ValueError, "d_grad_loss", e.Backward, temp, x, w, t, o, o[:5], x.clone(), w.clone())
    refused(ValueError, "same shape", e.Backward, temp, x, w, t, o, o, w, w.clone())
    assert len(c) == 0
    e.Forward(c, new(1, t=torch.uint8), x, w, t, o)
    with pytest.raises(LcppError) as err:
        Stream() << c.commit()
    assert err.value.status == L.ERR_TEMP_TOO_SMALL
    m.Step(c, q, q, v, g, g, new(6, 4, 8, 8), new(6, 4, 8, 8), v.clone(), d_parents=new(6, t=torch.int32))
    Stream() << c.commit()
    m.Step(c, q, q, v, g, g, None, new(6, 4, 8, 8), v)  # over its input
    with pytest.raises(LcppError) as err:
        Stream() << c.commit()
    assert err.value.status == L.ERR_INVALID_ARG
