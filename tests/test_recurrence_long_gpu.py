"""DeviceLinearRecurrence on the GPU with ten or more tiles for every CTA, where stages, slots and barriers of a CTA are
used again and again, against the float64 form on some of the channels."""
import numpy as np
import pytest

from lc_parallel_primitive_b200 import _lib as L
from tests import sequence_reference as R
from tests.test_recurrence_gpu import Case, host

pytestmark = pytest.mark.gpu

TILE_ROWS, TILE_BYTES = 128, 128  # of a tile: rows, and bytes of a row


def lengths(rows, seed):
    """Random lengths, short ones and empty ones among them, that fill the rows."""
    r = np.random.RandomState(seed)
    out = []
    while sum(out) < rows:
        out.append(min(int(r.choice([0, 1, r.randint(2, 40), r.randint(100, 900)])), rows - sum(out)))
    return out


def channels(d, dtype, seed):
    """The channels at the edges of the first and last tiles, and some others."""
    width = TILE_BYTES // (4 if dtype == "f32" else 2)
    edge = [0, 1, width - 1, width, 2 * width - 1, (d - 1) // width * width - 1, (d - 1) // width * width, d - 2, d - 1]
    more = np.random.RandomState(seed).randint(0, d, 24)
    return np.unique(np.clip(np.concatenate([edge, more]), 0, d - 1))


def check(c, seed):
    import torch

    width = TILE_BYTES // (4 if c.dtype == "f32" else 2)
    tiles = -(-c.rows // TILE_ROWS) * -(-c.d // width)
    assert tiles >= 10 * torch.cuda.get_device_properties(0).multi_processor_count
    out, last = c.forward()
    gg, gi, g0 = c.backward()
    cols = channels(c.d, c.dtype, seed)
    at = torch.from_numpy(cols).cuda()

    def some(t):
        return host(t[:, at])

    f = R.recurrence(some(c.gate), some(c.x), c.offsets, some(c.init), c.mode)
    want = R.backward(f, some(c.grad_out), some(c.grad_last))
    R.assert_within(some(out), f["out"], f["out_err"], c.dtype, "out")
    R.assert_within(some(last), f["last"], f["last_err"], "f32", "last")
    R.assert_within(some(gg), want["grad_gate"], want["grad_gate_err"], c.dtype, "grad_gate")
    R.assert_within(some(gi), want["grad_in"], want["grad_in_err"], c.dtype, "grad_in")
    R.assert_within(some(g0), want["grad_init"], want["grad_init_err"], "f32", "grad_init")


# (rows, channels): the look-back's window is the short one with more than 24 column tiles, the long one with fewer
@pytest.mark.parametrize("dtype,rows,d,mode,pad,shift,packed", [
    ("f32", 3000, 2048, "sigmoid", 0, 0, False),    # 64 column tiles, 16-byte copies
    ("bf16", 3100, 4096, "sigmoid", 0, 0, False),
    ("f16", 3100, 4096, "linear", 0, 0, True),
    ("f32", 6300, 1001, "linear", 0, 0, True),      # 32 column tiles, 4-byte copies
    ("bf16", 6300, 2047, "sigmoid", 0, 1, False),   # odd addresses and strides
    ("f16", 6300, 2047, "sigmoid", 2, 0, True),
    ("bf16", 65536, 136, "sigmoid", 0, 0, False),   # 3 column tiles, 512 row tiles
    ("f32", 50000, 97, "linear", 3, 1, True)])
def test_many_tiles_a_cta(cuda, dtype, rows, d, mode, pad, shift, packed):
    seed = rows + d
    check(Case(lengths(rows, seed) if packed else [rows // 2, rows // 2], d, dtype, mode, seed=seed, packed=packed, pad=pad,
               shift=shift), seed)


def test_two_streams_at_once(cuda):
    # two chains of tiles under way together, each with its temp buffer: the bits of either alone
    import torch
    from lc_parallel_primitive_b200 import CommandList, DeviceLinearRecurrence, Stream, last_device_error

    cases = [Case([2000], 64, "f32", "sigmoid", seed=50), Case([700, 0, 1500], 72, "bf16", "linear", seed=51, packed=True)]
    want = [[host(t).copy() for t in c.forward() + c.backward()] for c in cases]
    got, streams = [], [torch.cuda.Stream(), torch.cuda.Stream()]
    m = DeviceLinearRecurrence()
    m.create()
    for c in cases:
        S = len(c.lengths)
        got.append([c.matrix(), torch.zeros((S, c.d), device="cuda"), c.matrix(), c.matrix(), torch.zeros((S, c.d), device="cuda")])
    torch.cuda.synchronize()
    for _ in range(20):
        for c, (out, last, gg, gi, g0), s in zip(cases, got, streams):
            cl = CommandList()
            m.Forward(cl, c.temp, c.gate, c.x, out, c.sequences, d_init=c.init, d_last=last, d_saved=c.saved, mode=c.mode)
            m.Backward(cl, c.temp, c.gate, c.x, c.saved, c.grad_out, gg, gi, c.sequences, d_init=c.init,
                       d_grad_last=c.grad_last, d_grad_init=g0, mode=c.mode)
            Stream(s) << cl.commit()
    torch.cuda.synchronize()
    L.check(last_device_error())
    for w, g in zip(want, got):
        for p, q in zip(w, g):
            assert np.array_equal(p, host(q))
