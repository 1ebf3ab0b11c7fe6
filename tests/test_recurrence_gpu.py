"""DeviceLinearRecurrence on the GPU against the float64 row-by-row form."""
import numpy as np
import pytest

from lc_parallel_primitive_b200 import _lib as L
from tests import sequence_reference as R

pytestmark = pytest.mark.gpu

MODES = ["linear", "sigmoid"]
DTYPES = ["f32", "f16", "bf16"]


def torch_dtype(name):
    import torch

    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[name]


def host(t):
    return t.detach().float().cpu().numpy()


class Case:
    """Inputs on the device, in buffers whose rows may be wider than the channels or start off alignment."""

    def __init__(self, lengths, d, dtype, mode, seed=0, packed=False, pad=0, shift=0, init="random", tail=0, lead=0):
        import torch

        r = np.random.RandomState(seed)
        self.lengths, self.d, self.dtype, self.mode = list(lengths), d, dtype, mode
        self.offsets = np.concatenate([[0], np.cumsum(self.lengths)]).astype(np.int64) + lead
        self.rows = int(self.offsets[-1]) + tail
        self.pad, self.shift = pad, shift
        gate = r.randn(self.rows, d) + np.linspace(-1, 6, d)
        if mode == "linear":
            gate = np.where(r.rand(self.rows, d) < 0.5, 1, -1) * R.sigmoid(gate)
        self.gate, self.x = self.matrix(gate), self.matrix(r.randn(self.rows, d))
        self.init = None
        S = len(self.lengths)
        if init == "random":
            self.init = torch.from_numpy(r.randn(S, d).astype(np.float32)).cuda()
        elif init == "shared":
            self.init = torch.from_numpy(r.randn(1, d).astype(np.float32)).cuda().expand(S, d)
        self.grad_out = self.matrix(r.randn(self.rows, d))
        self.grad_last = torch.from_numpy(r.randn(S, d).astype(np.float32)).cuda()
        uniform = len(set(self.lengths)) == 1 and not lead and not tail
        self.sequences = (self.lengths[0] if uniform and not packed
                          else torch.from_numpy(self.offsets.astype(np.int32)).cuda())

    def matrix(self, a=None):
        import torch

        width = self.d + self.pad
        buf = torch.full((self.rows * width + self.shift,), 77.0, dtype=torch_dtype(self.dtype), device="cuda")
        m = buf[self.shift:].view(self.rows, width)[:, :self.d] if self.rows else buf[:0].view(0, self.d)
        if a is not None:
            m.copy_(torch.from_numpy(np.asarray(a)))
        return m

    def forward(self, out=None, last=None, saved=True):
        import torch
        from lc_parallel_primitive_b200 import CommandList, DeviceLinearRecurrence, Stream, last_device_error, temp_buffer

        m = DeviceLinearRecurrence()
        m.create()
        c, s = CommandList(), Stream()
        self.temp = temp_buffer(m.GetTempStorageBytes(self.rows, self.d))
        self.temp.fill_(0x5A5A5A5A)
        self.saved = temp_buffer(m.GetSavedStateBytes(self.rows, self.d)) if saved else None
        if saved:
            self.saved.fill_(-1)
        self.out = self.matrix() if out is None else out
        self.last = torch.full((len(self.lengths), self.d), 55.0, device="cuda") if last is None else last
        m.Forward(c, self.temp, self.gate, self.x, self.out, self.sequences, d_init=self.init, d_last=self.last,
                  d_saved=self.saved, mode=self.mode)
        s << c.commit()
        torch.cuda.synchronize()
        L.check(last_device_error())
        return self.out, self.last

    def backward(self, grad_gate=None, grad_in=None, use_out=True, use_last=True):
        import torch
        from lc_parallel_primitive_b200 import CommandList, DeviceLinearRecurrence, Stream, last_device_error

        m = DeviceLinearRecurrence()
        m.create()
        c, s = CommandList(), Stream()
        gg = self.matrix() if grad_gate is None else grad_gate
        gi = self.matrix() if grad_in is None else grad_in
        g0 = torch.full((len(self.lengths), self.d), 55.0, device="cuda")
        self.temp.fill_(0x5A5A5A5A)
        m.Backward(c, self.temp, self.gate, self.x, self.saved, self.grad_out if use_out else None, gg, gi,
                   self.sequences, d_init=self.init, d_grad_last=self.grad_last if use_last else None,
                   d_grad_init=g0, mode=self.mode)
        s << c.commit()
        torch.cuda.synchronize()
        L.check(last_device_error())
        return gg, gi, g0

    def reference(self):
        init = None if self.init is None else host(self.init)
        return R.recurrence(host(self.gate), host(self.x), self.offsets, init, self.mode)

    def check(self, backward=True, **kw):
        f = self.reference()
        out, last = self.forward()
        R.assert_within(host(out), f["out"], f["out_err"], self.dtype, "out")
        R.assert_within(host(last), f["last"], f["last_err"], "f32", "last")
        if backward:
            want = R.backward(f, host(self.grad_out) if kw.get("use_out", True) else None,
                              host(self.grad_last) if kw.get("use_last", True) else None)
            gg, gi, g0 = self.backward(**kw)
            R.assert_within(host(gg), want["grad_gate"], want["grad_gate_err"], self.dtype, "grad_gate")
            R.assert_within(host(gi), want["grad_in"], want["grad_in_err"], self.dtype, "grad_in")
            R.assert_within(host(g0), want["grad_init"], want["grad_init_err"], "f32", "grad_init")


@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("length", [1, 2, 7, 127, 128, 129, 1000])
def test_one_sequence(cuda, mode, dtype, length):
    Case([length], 70, dtype, mode, seed=length).check()


@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [1, 2, 3, 8, 31, 64, 65, 128, 136, 257, 1000])
def test_channels(cuda, mode, dtype, d):
    Case([150, 150], d, dtype, mode, seed=d).check()


@pytest.mark.parametrize("dtype", DTYPES)
def test_long_sequences(cuda, dtype):
    # many tiles in a chain, in both directions
    Case([9001, 9001], 40, dtype, "sigmoid", seed=3).check()


def test_many_tiles_across_channels(cuda):
    Case([4100], 520, "bf16", "sigmoid", seed=4).check()


RAGGED = {
    "mixed": [3, 0, 1, 127, 128, 129, 0, 0, 300, 1, 1, 64],
    "ones": [1] * 400,
    "empties": [0] * 70 + [5] + [0] * 100 + [200] + [0] * 40,
    "all empty": [0, 0, 0],
    "tile edges": [128, 128, 256, 1, 127],
    "one long": [0, 2000, 0],
}


@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("name", sorted(RAGGED))
def test_packed(cuda, mode, dtype, name):
    Case(RAGGED[name], 72, dtype, mode, seed=7, packed=True).check()


@pytest.mark.parametrize("lead,tail", [(0, 5), (3, 0), (130, 300), (1, 1)])
def test_padding_rows_come_out_zero(cuda, lead, tail):
    c = Case([100, 0, 77], 72, "f32", "sigmoid", seed=8, packed=True, lead=lead, tail=tail)
    for m in (c.gate, c.x, c.grad_out):  # whatever the padding holds
        m[:lead] = float("nan")
        m[c.rows - tail:] = float("inf")
    f = R.recurrence(np.nan_to_num(host(c.gate)), np.nan_to_num(host(c.x)), c.offsets, host(c.init), c.mode)
    out, last = c.forward()
    R.assert_within(host(out), f["out"], f["out_err"], "f32", "out")
    R.assert_within(host(last), f["last"], f["last_err"], "f32", "last")
    want = R.backward(f, np.nan_to_num(host(c.grad_out)), host(c.grad_last))
    gg, gi, g0 = c.backward()
    R.assert_within(host(gg), want["grad_gate"], want["grad_gate_err"], "f32", "grad_gate")
    R.assert_within(host(gi), want["grad_in"], want["grad_in_err"], "f32", "grad_in")
    R.assert_within(host(g0), want["grad_init"], want["grad_init_err"], "f32", "grad_init")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("pad,shift", [(1, 0), (8, 0), (0, 1), (8, 3), (5, 2), (24, 8)])
def test_strides_and_alignment(cuda, dtype, pad, shift):
    c = Case([200, 200], 64, dtype, "sigmoid", seed=9, pad=pad, shift=shift)
    c.check()
    if pad:  # nothing is written between the rows
        width = c.d + pad
        gaps = c.out.as_strided((c.rows - 1, pad), (width, 1), c.out.storage_offset() + c.d)
        assert (gaps == 77.0).all()


def test_mixed_alignment(cuda):
    c = Case([150], 64, "bf16", "sigmoid", seed=10)
    odd = Case([150], 64, "bf16", "sigmoid", seed=11, pad=1, shift=1)
    c.x = odd.x  # one unaligned operand among aligned ones
    c.check()


@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("init", ["none", "shared"])
def test_initial_states(cuda, mode, init):
    Case([129, 0, 40], 66, "f32", mode, seed=12, init=init).check()


@pytest.mark.parametrize("use_out,use_last", [(True, False), (False, True), (False, False)])
def test_missing_gradients_are_zero(cuda, use_out, use_last):
    Case([300, 20], 66, "f32", "sigmoid", seed=13).check(use_out=use_out, use_last=use_last)


def test_batched_view(cuda):
    # (batch, time, channels) halves of one projection
    import torch

    c = Case([70, 70, 70], 64, "bf16", "sigmoid", seed=14)
    both = torch.cat([c.gate, c.x], dim=1).view(3, 70, 128)
    c.gate, c.x = both[:, :, :64], both[:, :, 64:]
    out, last = c.forward(out=torch.empty((3, 70, 64), dtype=torch.bfloat16, device="cuda"))
    c.gate, c.x = c.gate.reshape(210, 64), c.x.reshape(210, 64)
    f = c.reference()
    R.assert_within(host(out).reshape(210, 64), f["out"], f["out_err"], "bf16", "out")
    R.assert_within(host(last), f["last"], f["last_err"], "f32", "last")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_in_place(cuda, dtype):
    c = Case([500, 300], 130, dtype, "sigmoid", seed=15)
    f = c.reference()
    want = R.backward(f, host(c.grad_out), host(c.grad_last))
    c.forward()
    gg, gi, _ = c.backward(grad_gate=c.gate, grad_in=c.grad_out)
    R.assert_within(host(gg), want["grad_gate"], want["grad_gate_err"], dtype, "grad_gate")
    R.assert_within(host(gi), want["grad_in"], want["grad_in_err"], dtype, "grad_in")
    c = Case([500, 300], 130, dtype, "sigmoid", seed=15)
    out, last = c.forward(out=c.x, last=c.init, saved=False)
    R.assert_within(host(out), f["out"], f["out_err"], dtype, "out")
    R.assert_within(host(last), f["last"], f["last_err"], "f32", "last")


def test_sequences_do_not_leak_into_each_other(cuda):
    # infinities and NaN of one sequence stay in it, forward and backward, also within a tile
    c = Case([50, 60, 200, 40], 66, "f32", "linear", seed=16, packed=True)
    lo, hi = int(c.offsets[1]), int(c.offsets[2])
    c.gate[lo:hi], c.x[lo:hi] = float("inf"), float("nan")
    c.grad_out[lo:hi] = float("nan")
    out, last = c.forward()
    gg, gi, g0 = c.backward()
    clean = Case([50, 60, 200, 40], 66, "f32", "linear", seed=16, packed=True)
    want_out, want_last = clean.forward()
    want_gg, want_gi, want_g0 = clean.backward()
    keep = np.r_[0:lo, hi:c.rows]
    for got, want in ((out, want_out), (gg, want_gg), (gi, want_gi)):
        assert np.array_equal(host(got)[keep], host(want)[keep])
        assert np.isnan(host(got)[lo:hi]).all()
    seqs = [0, 2, 3]
    assert np.array_equal(host(last)[seqs], host(want_last)[seqs])
    assert np.array_equal(host(g0)[seqs], host(want_g0)[seqs])


def test_gate_extremes(cuda):
    # a gate of -inf forgets exactly, one of +inf keeps exactly, and a NaN stays one
    c = Case([300], 64, "f32", "sigmoid", seed=17)
    c.gate[10, :16], c.gate[20:40, 16:32], c.gate[5, 32] = float("-inf"), float("inf"), float("nan")
    c.gate[50, 33], c.gate[60, 34] = -200.0, 200.0
    out = host(c.forward()[0])
    assert np.array_equal(out[10, :16], host(c.x)[10, :16])
    assert (out[20:40, 16:32] == out[19, 16:32]).all()
    assert np.isnan(out[5:, 32]).all() and np.isfinite(out[:5, 32]).all()
    assert out[50, 33] == host(c.x)[50, 33] and out[60, 34] == out[59, 34]
    gg, gi, g0 = (host(t) for t in c.backward())
    fine = [i for i in range(64) if i != 32]
    assert np.isfinite(gg[:, fine]).all() and np.isfinite(gi[:, fine]).all() and np.isfinite(g0[:, fine]).all()
    assert (gg[10, :16] == 0).all() and (gi[20:40, 16:32] == 0).all()


@pytest.mark.parametrize("mode", MODES)
def test_gradients_against_differences(cuda, mode):
    # d loss / d input of loss = sum(w out) + sum(w' last), by central differences of the float64 form
    c = Case([9, 0, 6], 3, "f32", mode, seed=18, packed=True)
    c.forward()
    got = [host(t).astype(np.float64) for t in c.backward()]
    gate, x, init = (host(t).astype(np.float64) for t in (c.gate, c.x, c.init))
    w, wl = host(c.grad_out).astype(np.float64), host(c.grad_last).astype(np.float64)

    def loss(gate, x, init):
        f = R.recurrence(gate, x, c.offsets, init, mode)
        return (f["out"] * w).sum() + (f["last"] * wl).sum()

    # step 1e-4: the third-derivative term is below 1e-7 for these O(1) values, rounding 1e-16 / 1e-4 below 1e-10;
    # 1e-5 also covers the float32 gradients' own bound at this length
    for k, base in enumerate((gate, x, init)):
        for at in np.ndindex(base.shape):
            args = [gate.copy(), x.copy(), init.copy()]
            args[k][at] += 1e-4
            up = loss(*args)
            args[k][at] -= 2e-4
            assert abs((up - loss(*args)) / 2e-4 - got[k][at]) < 1e-5, (k, at)


def test_temp_is_scratch_only(cuda):
    # two calls in a row through one temp buffer, and the same bits each time
    a, b = Case([3000], 130, "bf16", "sigmoid", seed=19), Case([700, 700], 130, "bf16", "sigmoid", seed=20)
    first = [host(t).copy() for t in a.forward() + a.backward()]
    b.forward()
    again = [host(t) for t in a.forward() + a.backward()]
    for p, q in zip(first, again):
        assert np.array_equal(p, q)


def test_other_stream(cuda):
    import torch
    from lc_parallel_primitive_b200 import CommandList, DeviceLinearRecurrence, Stream, temp_buffer

    c = Case([2000], 64, "f32", "sigmoid", seed=21)
    want = host(c.forward()[0])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    m, cl = DeviceLinearRecurrence(), CommandList()
    m.create()
    out = torch.empty_like(c.gate)
    m.Forward(cl, temp_buffer(m.GetTempStorageBytes(c.rows, c.d)), c.gate, c.x, out, 2000, d_init=c.init)
    Stream(side) << cl.commit()
    side.synchronize()
    assert np.array_equal(host(out), want)


def test_graph_capture(cuda):
    import torch
    from lc_parallel_primitive_b200 import CommandList, DeviceLinearRecurrence, Stream

    c = Case([2000], 64, "f32", "sigmoid", seed=22)
    want = host(c.forward()[0])
    m = DeviceLinearRecurrence()
    m.create()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        cl = CommandList()
        m.Forward(cl, c.temp, c.gate, c.x, c.out, 2000, d_init=c.init, d_last=c.last)
        Stream() << cl.commit()
    for _ in range(3):
        c.out.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert np.array_equal(host(c.out), want)


def test_look_back_gives_up(cuda):
    # waits cut to two polls run out somewhere in a long chain: a status, and the context goes on
    import torch

    c = Case([20000], 64, "f32", "sigmoid", seed=24)
    want = host(c.forward()[0])
    lib = L.lib()
    L.check(lib.lcpp_set_spin_limit(1))
    try:
        with pytest.raises(L.LcppError) as e:
            for _ in range(20):
                c.forward()
        assert e.value.status == L.ERR_LOOKBACK_TIMEOUT
    finally:
        torch.cuda.synchronize()
        L.check(lib.lcpp_set_spin_limit(0))
    assert np.array_equal(host(c.forward()[0]), want)


def test_long_cache_offsets_pass_32_bits(cuda):
    # element offsets beyond 2^32: rows of a wide buffer
    import torch

    stride, rows, d = (1 << 24) + 16, 300, 64  # the last rows start past 2^32 elements
    buf = torch.zeros(rows * stride, dtype=torch.bfloat16, device="cuda")
    c = Case([rows], d, "bf16", "sigmoid", seed=23)
    wide = buf.view(rows, stride)[:, :d]
    wide.copy_(c.gate)
    c.gate = wide
    c.check()


# ---- one token -----------------------------------------------------------------------------------
def step(c, states, states_out, parents=None, out=True):
    import torch
    from lc_parallel_primitive_b200 import CommandList, DeviceLinearRecurrence, Stream

    m, cl = DeviceLinearRecurrence(), CommandList()
    m.create()
    o = c.matrix() if out else None
    m.Step(cl, c.gate, c.x, states, states_out, o, d_parents=parents, mode=c.mode)
    Stream() << cl.commit()
    torch.cuda.synchronize()
    return o


@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,d,pad,shift", [(1, 1, 0, 0), (4, 64, 0, 0), (5, 67, 0, 0), (33, 128, 8, 0),
                                              (7, 130, 1, 1), (64, 1000, 0, 0), (3, 4099, 0, 2)])
def test_step(cuda, mode, dtype, rows, d, pad, shift):
    import torch

    c = Case([1] * rows, d, dtype, mode, seed=rows, pad=pad, shift=shift)
    f = c.reference()
    new = torch.empty_like(c.init)
    out = step(c, c.init, new)
    R.assert_within(host(new), f["out"], f["out_err"], "f32", "states")
    R.assert_within(host(out), f["out"], f["out_err"], dtype, "out")
    old = c.init.clone()
    step(c, old, old, out=False)  # in place, output not wanted
    assert torch.equal(old, new)


def test_step_follows_parents(cuda):
    import torch
    from lc_parallel_primitive_b200 import last_device_error

    c = Case([1] * 6, 100, "bf16", "sigmoid", seed=30)
    pool = torch.randn((9, 100), device="cuda")
    parents = torch.tensor([8, 0, 0, -1, 3, 3], dtype=torch.int32, device="cuda")
    c.init = torch.where(parents[:, None] >= 0, pool[parents.clamp(min=0).long()], torch.zeros((), device="cuda"))
    f = c.reference()
    new = torch.empty((6, 100), device="cuda")
    out = step(c, pool, new, parents)
    R.assert_within(host(new), f["out"], f["out_err"], "f32", "states")
    R.assert_within(host(out), f["out"], f["out_err"], "bf16", "out")
    # a parent that does not exist is reported and reads nothing
    parents[1] = 9
    c.init[1] = 0
    f = c.reference()
    step(c, pool, new, parents)
    R.assert_within(host(new), f["out"], f["out_err"], "f32", "states")
    assert last_device_error() == L.ERR_INVALID_ARG and last_device_error() == L.OK


def test_step_continues_forward(cuda):
    # a prompt through Forward, then tokens through Step: the states of one long Forward
    import torch

    c = Case([40], 96, "f32", "sigmoid", seed=31)
    f = c.reference()
    gate, x = c.gate, c.x
    c.gate, c.x, c.rows, c.lengths, c.sequences = gate[:30], x[:30], 30, [30], 30
    _, state = c.forward(saved=False)
    c.rows = 1
    for t in range(30, 40):
        c.gate, c.x = gate[t:t + 1], x[t:t + 1]
        step(c, state, state)
    R.assert_within(host(state), f["last"], f["last_err"], "f32", "state")
    assert torch.isfinite(state).all()
