"""DeviceDeltaRule on the GPU against the float64 token-by-token form."""
import numpy as np
import pytest

from lc_parallel_primitive_b200 import _lib as L
from tests import delta_reference as R

pytestmark = pytest.mark.gpu
DTYPES = ["f32", "f16", "bf16"]


def torch_dtype(name):
    import torch

    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[name]


def host(t):
    return t.detach().double().cpu().numpy()


class Case:
    """Inputs on the device, in buffers whose rows may be wider or start off alignment."""

    def __init__(self, lengths, heads, key_heads, dk, dv, dtype, seed=0, packed=False, pad=0, shift=0, lead=0, tail=0,
                 init=True, decay="mixed", beta=None, scale=None, size=1.0, fill=77.0):
        import torch

        r = np.random.RandomState(seed)
        self.lengths, self.heads, self.key_heads, self.dk, self.dv = list(lengths), heads, key_heads, dk, dv
        self.dtype, self.pad, self.shift, self.fill = dtype, pad, shift, fill
        self.offsets = np.concatenate([[0], np.cumsum(self.lengths)]).astype(np.int64) + lead
        rows = self.rows = int(self.offsets[-1]) + tail
        S = len(self.lengths)
        k = r.randn(rows, key_heads, dk)
        q = r.randn(rows, key_heads, dk)
        k /= np.linalg.norm(k, axis=2, keepdims=True) * 1.01  # unit keys, also when rounded
        q /= np.linalg.norm(q, axis=2, keepdims=True)
        self.q, self.k = self.matrix(key_heads, dk, q), self.matrix(key_heads, dk, k)
        self.v = self.matrix(heads, dv, size * r.randn(rows, heads, dv))
        d = -np.log1p(np.exp(-(r.randn(rows, heads) + np.linspace(1, 6, heads))))
        if decay == "resets":
            d[r.rand(rows, heads) < 0.05] = -np.inf
            d[r.rand(rows, heads) < 0.05] = -120.0
        self.decay = None if decay is None else self.gates(d)
        self.beta = self.gates(r.rand(rows, heads) if beta is None else np.full((rows, heads), float(beta)))
        self.init = torch.from_numpy((size * r.randn(S, heads, dv, dk) * 0.3).astype(np.float32)).cuda() if init else None
        self.scale = scale
        self.grad_out = self.matrix(heads, dv, r.randn(rows, heads, dv) * size)
        self.grad_last = torch.from_numpy((r.randn(S, heads, dv, dk) * size / np.sqrt(dk)).astype(np.float32)).cuda()
        uniform = len(set(self.lengths)) == 1 and self.lengths[0] > 0 and not lead and not tail
        self.sequences = (self.lengths[0] if uniform and not packed
                          else torch.from_numpy(self.offsets.astype(np.int32)).cuda())

    def matrix(self, heads, dim, a=None):
        import torch

        width = heads * dim + self.pad
        buf = torch.full((self.rows * width + self.shift,), self.fill, dtype=torch_dtype(self.dtype), device="cuda")
        m = buf[self.shift:].view(self.rows, width)[:, :heads * dim].unflatten(1, (heads, dim))
        if a is not None:
            m.copy_(torch.from_numpy(np.asarray(a)))
        return m

    def gates(self, a):
        import torch

        width = self.heads + self.pad
        m = torch.full((self.rows, width), self.fill, device="cuda")[:, :self.heads]
        m.copy_(torch.from_numpy(a))
        return m

    def sizes(self):
        return self.rows, len(self.lengths), self.heads, self.key_heads, self.dk, self.dv

    def run(self, saved=True, last=None, stream=None, check=True):
        import torch
        from lc_parallel_primitive_b200 import CommandList, DeviceDeltaRule, Stream, last_device_error, temp_buffer

        self.module = m = DeviceDeltaRule()
        m.create()
        c, s = CommandList(), stream or Stream()
        self.temp = temp_buffer(m.GetTempStorageBytes(*self.sizes(), torch_dtype(self.dtype)))
        self.temp.fill_(-1)  # NaN in every type
        self.saved = temp_buffer(m.GetSavedStateBytes(*self.sizes())) if saved else None
        if saved:
            self.saved.fill_(-1)
        self.out = self.matrix(self.heads, self.dv)
        self.last = torch.full((len(self.lengths), self.heads, self.dv, self.dk), 55.0, device="cuda") if last is None else last
        m.Forward(c, self.temp, self.q, self.k, self.v, self.decay, self.beta, self.out, self.sequences, d_init=self.init,
                  d_last=self.last, d_saved=self.saved, scale=self.scale)
        s << c.commit()
        if check:
            torch.cuda.synchronize()
            L.check(last_device_error())
        return self.out, self.last

    def back(self, use_out=True, use_last=True, stream=None, check=True):
        import torch
        from lc_parallel_primitive_b200 import CommandList, Stream, last_device_error

        c, s = CommandList(), stream or Stream()
        self.temp.fill_(-1)
        dt = torch_dtype(self.dtype)
        new = lambda shape, t=torch.float32: torch.full(shape, 55.0, dtype=t, device="cuda")  # noqa: E731
        g = R.Result()
        g.q, g.k, g.v = new(self.q.shape, dt), new(self.k.shape, dt), new(self.v.shape, dt)
        g.beta, g.init = new(self.beta.shape), new(self.last.shape)
        g.decay = None if self.decay is None else new(self.beta.shape)
        self.module.Backward(c, self.temp, self.q, self.k, self.v, self.decay, self.beta, self.saved,
                             self.grad_out if use_out else None, g.q, g.k, g.v, g.decay, g.beta, self.sequences,
                             d_init=self.init, d_grad_last=self.grad_last if use_last else None, d_grad_init=g.init,
                             scale=self.scale)
        s << c.commit()
        if check:
            torch.cuda.synchronize()
            L.check(last_device_error())
        return g

    def inside(self, a):
        """Rows of sequences; the others as zeros."""
        keep = np.zeros(self.rows, bool)
        keep[self.offsets[0]:self.offsets[-1]] = True
        return np.where(keep.reshape((-1,) + (1,) * (a.ndim - 1)), a, 0.0)

    def reference(self):
        scale = self.dk ** -0.5 if self.scale is None else self.scale
        f = lambda t: None if t is None else self.inside(host(t))  # noqa: E731
        return R.forward(f(self.q), f(self.k), f(self.v), f(self.decay), f(self.beta), self.offsets,
                         None if self.init is None else host(self.init), scale)

    def check(self, backward=True, **kw):
        f = self.reference()
        out, last = self.run(saved=backward)
        b = R.bounds(f, dtype=self.dtype)
        R.assert_within(host(out), f.out, b.out, self.dtype, "out")
        R.assert_within(host(last), f.last, b.last, "f32", "last")
        if backward:
            self.check_back(f, **kw)

    def check_back(self, f, use_out=True, use_last=True):
        got = self.back(use_out, use_last)
        want = R.backward(f, self.inside(host(self.grad_out)) if use_out else None, host(self.grad_last) if use_last else None)
        b = R.bounds(f, want)
        for n in ("q", "k", "v", "beta", "decay", "init"):
            if getattr(got, n) is not None:
                R.assert_within(host(getattr(got, n)), getattr(want, n), getattr(b, n), self.dtype if n in "qkv" else "f32",
                                "grad " + n)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lengths", [[1], [2, 2], [63], [64], [65, 65], [128], [130, 1, 0, 64, 63, 0], [0, 0], [200]])
def test_lengths(cuda, dtype, lengths):
    Case(lengths, 2, 1, 64, 64, dtype, seed=1).check()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads,key_heads,dk,dv", [(1, 1, 128, 128), (3, 3, 1, 1), (4, 2, 16, 128), (6, 2, 100, 36), (2, 2, 65, 127),
                                                   (3, 1, 128, 17), (1, 1, 60, 72), (5, 5, 8, 33), (2, 1, 127, 64)])
def test_shapes(cuda, dtype, heads, key_heads, dk, dv):
    Case([70, 131], heads, key_heads, dk, dv, dtype, seed=2).check()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kw", [dict(pad=8), dict(pad=3), dict(shift=1), dict(shift=1, pad=5), dict(lead=5, tail=70), dict(packed=True),
                                dict(init=False), dict(decay=None), dict(decay="resets"), dict(beta=0), dict(beta=1),
                                dict(beta=1.9), dict(scale=0.3), dict(scale=0.0), dict(scale=-2.0)])
def test_variants(cuda, dtype, kw):
    Case([90, 90], 4, 2, 72, 40, dtype, seed=3, **kw).check()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("size", [1e-20, 1e-8, 1e8])
def test_magnitudes(cuda, dtype, size):
    # values, states and gradients of any size: the products' scales follow them
    Case([130], 2, 2, 64, 48, dtype, seed=4, size=size).check()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("use_out,use_last", [(False, True), (True, False), (False, False)])
def test_missing_gradients(cuda, dtype, use_out, use_last):
    Case([70, 70], 2, 1, 64, 32, dtype, seed=5).check(use_out=use_out, use_last=use_last)


@pytest.mark.parametrize("dtype", DTYPES)
def test_equal_keys(cuda, dtype):
    # the triangular matrices are as far from the identity as they get
    c = Case([128], 2, 2, 64, 32, dtype, seed=6, decay=None, beta=1)
    c.k.copy_(c.k[:1].expand_as(c.k))
    c.check()


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_outside_hold_anything(cuda, dtype):
    c = Case([70, 65], 2, 1, 64, 40, dtype, seed=7, lead=3, tail=130)
    f = c.reference()
    for t in (c.q, c.k, c.v, c.decay, c.beta, c.grad_out):
        t[:3], t[138:] = float("nan"), float("inf")
    out, last = c.run()
    b = R.bounds(f, dtype=dtype)
    R.assert_within(host(out), f.out, b.out, dtype, "out")
    R.assert_within(host(last), f.last, b.last, "f32", "last")
    assert (host(out)[:3] == 0).all() and (host(out)[138:] == 0).all()
    c.check_back(f)


@pytest.mark.parametrize("dtype", DTYPES)
def test_what_is_not_finite_stays_in_its_sequence_and_head(cuda, dtype):
    c = Case([100, 100, 100], 4, 4, 64, 32, dtype, seed=8)
    f = c.reference()
    c.v[150, 1, 3], c.k[120, 2, 5], c.init[1, 3, 0, 0] = float("inf"), float("nan"), float("inf")
    out, last = c.run()
    b, o, la = R.bounds(f, dtype=dtype), host(out), host(last)
    for s in (0, 2):
        R.assert_within(o[100 * s:100 * s + 100], f.out[100 * s:100 * s + 100], b.out[100 * s:100 * s + 100], dtype, "out")
        R.assert_within(la[s], f.last[s], b.last[s], "f32", "last")
    R.assert_within(o[:, 0], f.out[:, 0], b.out[:, 0], dtype, "out of another head")
    assert not np.isfinite(o[150:200, 1, 3]).any() and not np.isfinite(la[1, 2]).any()
    # nothing that is finite is wrong
    ok = np.isfinite(o)
    R.assert_within(np.where(ok, o, f.out), f.out, b.out, dtype, "finite outputs")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lengths,heads,key_heads,dk,dv", [([4200], 2, 1, 64, 40), ([2100, 2100], 1, 1, 128, 128), ([3000, 1, 0, 700], 1, 1, 40, 72)])
def test_sequences_in_parts(cuda, dtype, lengths, heads, key_heads, dk, dv):
    # few chains: cut into parts, and states joined through the parts' maps
    Case(lengths, heads, key_heads, dk, dv, dtype, seed=9).check()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_many_sequences_of_different_lengths(cuda, dtype):
    # more chains than SMs: long ones first
    r = np.random.RandomState(10)
    lengths = np.minimum(r.lognormal(3, 1.3, 120).astype(int), 300)
    Case(lengths, 2, 2, 32, 24, dtype, seed=10).check()


@pytest.mark.parametrize("seqs,heads,dv", [(8, 16, 128), (8, 16, 100), (40, 4, 64)])
def test_full_ctas(cuda, seqs, heads, dv):
    # 8 warps a CTA, several chunks each
    Case([140] * seqs, heads, heads // 2, 128, dv, "bf16", seed=11).check()


def test_last_may_be_init(cuda):
    c = Case([70, 70], 2, 1, 64, 40, "f32", seed=12)
    f = c.reference()
    out, last = c.run(last=c.init)
    b = R.bounds(f)
    R.assert_within(host(out), f.out, b.out, "f32", "out")
    R.assert_within(host(last), f.last, b.last, "f32", "last")


def test_batches_of_four_dimensions(cuda):
    import torch

    c = Case([70, 70], 4, 2, 64, 40, "bf16", seed=13)
    out, last = c.run()
    want, states = out.clone(), last.clone()
    c.q, c.k, c.v = (t.unflatten(0, (2, 70)) for t in (c.q, c.k, c.v))
    matrix = c.matrix
    c.matrix = lambda *a: matrix(*a).unflatten(0, (2, 70))
    out, last = c.run()
    assert torch.equal(out.flatten(0, 1), want) and torch.equal(last, states)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_runs_give_the_same_bits(cuda, dtype):
    import torch

    r = np.random.RandomState(14)
    c = Case(r.randint(1, 400, 100), 4, 2, 64, 64, dtype, seed=14)
    out, last = c.run()
    g = c.back()
    for _ in range(3):
        o2, l2 = c.run()
        g2 = c.back()
        assert torch.equal(o2, out) and torch.equal(l2, last)
        assert all(torch.equal(getattr(g, n), getattr(g2, n)) for n in ("q", "k", "v", "decay", "beta", "init"))


def test_two_streams_at_once(cuda):
    import torch
    from lc_parallel_primitive_b200 import Stream

    cases = [Case([1000, 900], 8, 4, 128, 128, "bf16", seed=15), Case([70] * 40, 8, 8, 64, 64, "f32", seed=16)]
    want = [tuple(t.clone() for t in c.run()) + (c.back(),) for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    for _ in range(3):
        got = []
        for c, s in zip(cases, streams):
            with torch.cuda.stream(s):
                o = c.run(stream=Stream(s), check=False)
                got.append(o + (c.back(stream=Stream(s), check=False),))
        torch.cuda.synchronize()
        for (o, la, g), (wo, wl, wg) in zip(got, want):
            assert torch.equal(o, wo) and torch.equal(la, wl) and torch.equal(g.k, wg.k) and torch.equal(g.decay, wg.decay)


@pytest.mark.parametrize("lengths", [[200, 100], [4200]])
def test_captured_and_replayed(cuda, lengths):
    import torch
    from lc_parallel_primitive_b200 import CommandList, DeviceDeltaRule, Stream, temp_buffer

    c = Case(lengths, 2, 1, 64, 40, "bf16", seed=17)
    m, cl = DeviceDeltaRule(), CommandList()
    m.create()
    temp, saved = temp_buffer(m.GetTempStorageBytes(*c.sizes())), temp_buffer(m.GetSavedStateBytes(*c.sizes()))
    out, last = c.matrix(2, 40), torch.empty_like(c.grad_last)
    gq, gk, gv = (torch.empty(t.shape, dtype=t.dtype, device="cuda") for t in (c.q, c.k, c.v))
    gd, gb = torch.empty(c.rows, 2, device="cuda"), torch.empty(c.rows, 2, device="cuda")

    def go():
        m.Forward(cl, temp, c.q, c.k, c.v, c.decay, c.beta, out, c.sequences, d_init=c.init, d_last=last, d_saved=saved)
        m.Backward(cl, temp, c.q, c.k, c.v, c.decay, c.beta, saved, c.grad_out, gq, gk, gv, gd, gb, c.sequences, d_init=c.init,
                   d_grad_last=c.grad_last)
        Stream() << cl.commit()

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        go()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        go()
    c.v.mul_(0.5)  # other inputs
    c.init.mul_(-1)
    graph.replay()
    graph.replay()
    torch.cuda.synchronize()
    f = c.reference()
    g = R.backward(f, host(c.grad_out), host(c.grad_last))
    b = R.bounds(f, g, "bf16")
    R.assert_within(host(out), f.out, b.out, "bf16", "out")
    R.assert_within(host(last), f.last, b.last, "f32", "last")
    R.assert_within(host(gk), g.k, b.k, "bf16", "grad k")
    R.assert_within(host(gd), g.decay, b.decay, "f32", "grad decay")


def step(c, states_in, parents=None, states_out=None, rows=None):
    import torch
    from lc_parallel_primitive_b200 import CommandList, DeviceDeltaRule, Stream, last_device_error

    m, cl = DeviceDeltaRule(), CommandList()
    m.create()
    new = torch.full((c.rows, c.heads, c.dv, c.dk), 55.0, device="cuda") if states_out is None else states_out
    out = c.matrix(c.heads, c.dv)
    m.Step(cl, c.q, c.k, c.v, c.decay, c.beta, states_in, new, out, d_parents=parents, scale=c.scale)
    Stream() << cl.commit()
    torch.cuda.synchronize()
    return new, out, last_device_error()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,heads,key_heads,dk,dv,kw", [
    (1, 1, 1, 128, 128, {}), (5, 4, 2, 64, 40, {}), (7, 3, 3, 33, 7, {}), (3, 6, 2, 60, 72, dict(pad=3)),
    (4, 2, 1, 128, 9, dict(shift=1)), (9, 2, 2, 1, 1, dict(decay=None)), (6, 2, 1, 64, 64, dict(decay="resets")),
    (2, 2, 2, 128, 128, dict(scale=2.0))])
def test_step(cuda, dtype, rows, heads, key_heads, dk, dv, kw):
    import torch

    c = Case([1] * rows, heads, key_heads, dk, dv, dtype, seed=20, **kw)
    f = c.reference()
    b = R.bounds(f)
    new, out, status = step(c, c.init)
    L.check(status)
    R.assert_within(host(new), f.last, b.last, "f32", "states")
    R.assert_within(host(out), f.out, b.out, dtype, "out")
    # in place
    states = c.init.clone()
    step(c, states, states_out=states)
    assert torch.equal(states, new)
    # from zeros, and from parents: repeated, none, and beyond the end
    zeros, out0, _ = step(c, None)
    c.init, init = None, c.init
    f0 = c.reference()
    R.assert_within(host(zeros), f0.last, b.last, "f32", "states from zeros")
    if rows >= 4:
        parents = torch.tensor([2, 2, -1] + [0] * (rows - 3), dtype=torch.int32, device="cuda")
        c.init = torch.cat([init[parents[:2].long()], torch.zeros_like(init[:1]), init[:1].expand(rows - 3, -1, -1, -1)])
        fp = c.reference()
        new, out, status = step(c, init, parents)
        L.check(status)
        R.assert_within(host(new), fp.last, b.last + R.bounds(fp).last, "f32", "states of parents")
        parents[0] = rows
        new, out, status = step(c, init, parents)
        assert status == L.ERR_INVALID_ARG
        assert torch.equal(new[0], zeros[0])


@pytest.mark.parametrize("dtype", DTYPES)
def test_tokens_one_by_one_are_the_sequence(cuda, dtype):
    import torch

    c = Case([75, 75], 2, 1, 64, 40, dtype, seed=21)
    f = c.reference()
    b = R.bounds(f)
    states, outs = c.init.clone(), []
    rows = torch.tensor([0, 75], device="cuda")
    for t in range(75):
        one = Case([1, 1], 2, 1, 64, 40, dtype, seed=21)
        for n in ("q", "k", "v", "decay", "beta"):
            getattr(one, n).copy_(getattr(c, n)[rows + t])
        states, out, status = step(one, states)
        outs.append(out)
    got = host(torch.stack(outs, 1).flatten(0, 1))
    R.assert_within(got, f.out, b.out, dtype, "out")
    R.assert_within(host(states), f.last, b.last, "f32", "last")
