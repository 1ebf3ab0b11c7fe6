"""DeviceCrossEntropy on the GPU against float64, with element-wise bounds.

u = 2^-24.  A logit is a sum of products that are exact (16-bit operands) in float32, cut off at every step of 16 products: off
by z_err = (channels / 16 * pairs + 4) 2u sum_d |h_d w_d| with pairs 1, or 6 for float32: its operands in two float16 parts
take 3 products, leave 2^-23 of each factor and leave out the lower parts' product, 2^-22, together 8u.  logsum is off by the largest z_err and the sum's roundings (exp2 2 ulp of the term, its
argument |z| u, log2 and the last product 4 u |logsum|), the loss by that and one z_err more.
G = g (p - [target]), p = exp(z - logsum): off by g p times the errors of z and of logsum (which is the row's, of its
largest logits) and (|z| + |logsum|) 2u + 8u of the argument's and exp2's roundings, and, rounded between the products, by r |G| with r half an ulp of
the type (float32 in three parts: 2^-24; shares of the largest gradient add 2u).  Its products with weight and hidden add
the errors' absolute values, and cut off (terms / 16 * pairs + 4) 2u of their absolute terms.  float16 shares that are
below its smallest normal number times 2^14 are off by 2^-25 / 2^14 of the largest gradient instead, and what of a share
(or of its bf16 parts) is below float32's smallest normal number, 2^-126, may be lost: two parts' 2^-126 of the largest.
"""
import numpy as np
import pytest

from lc_parallel_primitive_b200 import _lib as L

pytestmark = pytest.mark.gpu
DTYPES = ["f32", "f16", "bf16"]
U = 2.0 ** -24
HALF_ULP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
SMALLEST = {"f32": 1e-37, "f16": 2.0 ** -24, "bf16": 1e-37}


def torch_dtype(name):
    import torch

    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[name]


class Case:
    def __init__(self, rows, channels, vocab, dtype, seed=0, pad=0, shift=0, ignored=0.1, gain="random", sharp=1.5, size=1.0):
        import torch

        g = torch.Generator(device="cuda").manual_seed(seed)
        normal = lambda *s: torch.randn(s, generator=g, device="cuda", dtype=torch.float64)  # noqa: E731
        self.rows, self.channels, self.vocab, self.dtype, self.pad, self.shift = rows, channels, vocab, dtype, pad, shift
        w = normal(vocab, channels) * (2 / np.sqrt(channels))
        t = torch.randint(0, vocab, (rows,), generator=g, device="cuda")
        self.hidden = self.matrix(rows, size * (normal(rows, channels) + sharp * w[t]))
        self.weight = self.matrix(vocab, w)
        out = torch.rand(rows, generator=g, device="cuda") < ignored
        self.targets = torch.where(out, -1 - torch.randint(0, 100, (rows,), generator=g, device="cuda"), t).int()
        if gain == "random":
            self.gain = normal(rows).float()
        elif gain == "zeros":
            self.gain = torch.zeros(rows, device="cuda")
        else:
            self.gain = torch.full((1,), float(gain), device="cuda").expand(rows)

    def matrix(self, rows, a=None):
        import torch

        width = self.channels + self.pad
        m = torch.full((rows * width + self.shift,), 77.0, dtype=torch_dtype(self.dtype), device="cuda")[self.shift:].view(
            rows, width)[:, :self.channels]
        return m if a is None else m.copy_(a)

    def temp(self):
        from lc_parallel_primitive_b200 import DeviceCrossEntropy, temp_buffer

        t = temp_buffer(DeviceCrossEntropy.GetTempStorageBytes(self.rows, self.channels, self.vocab, torch_dtype(self.dtype),
                                                               aligned=not (self.shift or self.pad % 8)))
        return t.fill_(-1)

    def run(self, stream=None, temp=None, grads="both", check=True):
        import torch
        from lc_parallel_primitive_b200 import CommandList, DeviceCrossEntropy, Stream, last_device_error

        m, c, s = DeviceCrossEntropy(), CommandList(), stream or Stream()
        m.create()
        temp = self.temp() if temp is None else temp
        self.loss, self.logsum = (torch.full((self.rows,), 55.0, device="cuda") for _ in range(2))
        m.Forward(c, temp, self.hidden, self.weight, self.targets, self.loss, self.logsum)
        self.grad_hidden = self.matrix(self.rows) if grads != "weight" else None
        self.grad_weight = self.matrix(self.vocab) if grads != "hidden" else None
        s << c.commit()
        if grads:
            m.Backward(c, temp, self.hidden, self.weight, self.targets, self.logsum, self.gain, self.grad_hidden,
                       self.grad_weight)
            s << c.commit()
        if check:
            torch.cuda.synchronize()
            L.check(last_device_error())
        return self.loss, self.logsum, self.grad_hidden, self.grad_weight

    def check(self, grads="both"):
        import torch

        self.run(grads=grads)
        keep = self.targets >= 0
        h, w = self.hidden.double()[keep], self.weight.double()
        t, n = self.targets.long()[keep], int(keep.sum())
        pairs = 6 if self.dtype == "f32" else 1
        z = h @ w.t()
        z_err = (self.channels / 16 * pairs + 4) * 2 * U * (h.abs() @ w.abs().t())
        logsum = torch.logsumexp(z, 1)
        top = z_err.amax(1) if n else logsum
        err = top + (z.abs().amax(1) + 16) * 2 * U + 4 * U * logsum.abs() if n else logsum
        right = z.gather(1, t[:, None]).squeeze(1)

        def rows(got, want, err, what):
            full, bound = torch.zeros(self.rows, dtype=torch.float64, device="cuda"), torch.zeros(
                self.rows, dtype=torch.float64, device="cuda")
            full[keep], bound[keep] = want, err
            self.within(got, full, bound, "f32", what)

        rows(self.logsum, logsum, err, "logsum")
        rows(self.loss, logsum - right, err + top + 2 * U * (logsum.abs() + right.abs()), "loss")
        if not grads:
            return
        g = self.gain.double()[keep][:, None]
        p = torch.exp(z - logsum[:, None])
        G = p.scatter_add(1, t[:, None], torch.full((n, 1), -1.0, dtype=torch.float64, device="cuda"))
        top_gain = float(g.abs().max()) if n else 0.0
        r = U if self.dtype == "f32" else HALF_ULP[self.dtype]
        G_err = g.abs() * (p * (z_err + err[:, None] + 2 * U * (z.abs() + logsum[:, None].abs()) + 8 * U) + (r + 4 * U) * G.abs())
        G_err = G_err + (2.0 ** -39 if self.dtype == "f16" else 2 * 2.0 ** -126) * top_gain
        G = g * G
        cut = lambda terms: (terms / 16 * pairs + 4) * 2 * U  # noqa: E731
        if self.grad_hidden is not None:
            want, bound = (torch.zeros(self.rows, self.channels, dtype=torch.float64, device="cuda") for _ in range(2))
            want[keep] = G @ w
            bound[keep] = G_err @ w.abs() + cut(self.vocab) * (G.abs() @ w.abs())
            self.within(self.grad_hidden, want, bound, self.dtype, "grad hidden")
        if self.grad_weight is not None:
            self.within(self.grad_weight, G.t() @ h, G_err.t() @ h.abs() + cut(n) * (G.abs().t() @ h.abs()), self.dtype, "grad weight")

    def within(self, got, want, err, dtype, what):
        tol = err + HALF_ULP[dtype] * (want.abs() + err) + SMALLEST[dtype]
        off = (got.double() - want).abs()
        bad = ~(off <= tol)
        assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()} out of bounds, worst "
                               f"{float((off / tol).nan_to_num(1e9).max())} times its bound")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,channels,vocab", [(1, 1, 1), (1, 8, 9), (3, 5, 2), (2, 64, 256), (255, 64, 257), (256, 128, 512),
                                                 (257, 63, 255), (700, 65, 1000), (1000, 200, 5003), (129, 1000, 130), (40, 33, 20011),
                                                 (2000, 16, 31)])
def test_sizes(cuda, dtype, rows, channels, vocab):
    Case(rows, channels, vocab, dtype, seed=1).check()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kw", [dict(pad=8), dict(pad=3), dict(shift=1), dict(shift=3, pad=5), dict(gain=0.25), dict(gain="zeros"),
                                dict(ignored=0.0), dict(ignored=0.95), dict(ignored=1.1), dict(sharp=8.0), dict(size=30.0),
                                dict(size=0.0)])
def test_variants(cuda, dtype, kw):
    Case(300, 72, 700, dtype, seed=2, **kw).check()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("grads", ["hidden", "weight", ""])
def test_what_is_wanted(cuda, dtype, grads):
    Case(300, 72, 700, dtype, seed=3).check(grads=grads)


@pytest.mark.parametrize("dtype,rows,vocab", [("bf16", 9000, 33000), ("f32", 2900, 33000)])
def test_pieces_of_the_vocabulary(cuda, dtype, rows, vocab):
    # the logits' gradient takes more than one piece: sums of the hidden gradient go on from piece to piece
    Case(rows, 40, vocab, dtype, seed=4).check()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_rows_and_tokens_of_any_size(cuda, dtype):
    import torch

    c = Case(300, 72, 700, dtype, seed=18)
    c.hidden *= (10.0 ** -torch.linspace(0, 18, 300, device="cuda"))[:, None].to(c.hidden.dtype)
    c.weight *= (10.0 ** -torch.linspace(0, 15, 700, device="cuda"))[torch.randperm(700, device="cuda")][:, None].to(c.weight.dtype)
    c.hidden[40], c.weight[50] = 0, 0
    c.check()


def test_an_infinity_of_float32_stays_in_its_row(cuda):
    import torch

    rows, row = 300, 7
    c = Case(rows, 72, 700, "f32", seed=17, ignored=0.0)
    want = [t.clone() for t in c.run()]
    c.hidden[row, 3] = float("inf")
    loss, logsum, gh, gw = c.run()
    rest = torch.arange(rows, device="cuda") != row
    assert not loss[row].isfinite() and not gh[row].isfinite().any()
    assert torch.equal(loss[rest], want[0][rest]) and torch.equal(logsum[rest], want[1][rest]) and torch.equal(gh[rest], want[2][rest])


@pytest.mark.parametrize("pad,shift", [(0, 0), (3, 1)])
def test_weight_gradient_of_many_rows(cuda, pad, shift):
    """Sums over up to 4096 rows are cut off at each of 256 steps, by up to 2u of what they have come to, half of the whole on
    average: 256 u; the roundings of G, of the parts' sums and the smaller products' cuts add less than 16 u."""
    c = Case(40000, 64, 300, "f32", seed=19, ignored=0.0, gain=1 / 40000, pad=pad, shift=shift)
    c.run()
    h, w = c.hidden.double(), c.weight.double()
    p = (h @ w.t()).softmax(1)
    p[range(40000), c.targets.long()] -= 1
    want = p.t() @ h / 40000
    assert float((c.grad_weight.double() - want).norm() / want.norm()) <= (256 + 16) * U


@pytest.mark.parametrize("dtype", DTYPES)
def test_sum_over_the_vocabulary_in_parts(cuda, dtype):
    # few tiles of the hidden gradient: several parts of the sum, each with its own
    Case(60, 100, 40003, dtype, seed=5).check()


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_that_take_no_part_hold_anything(cuda, dtype):
    import torch

    c = Case(300, 72, 700, dtype, seed=6, ignored=0.3)
    want = [t.clone() for t in c.run()]
    out = c.targets < 0
    c.hidden[out] = float("nan")
    c.hidden[out.nonzero()[0]] = float("inf")
    c.gain = torch.where(out, float("nan"), c.gain)
    got = c.run()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert (got[0][out] == 0).all() and (got[1][out] == 0).all() and (got[2][out] == 0).all()


def test_targets_beyond_the_vocabulary(cuda):
    import torch
    from lc_parallel_primitive_b200 import last_device_error

    c = Case(300, 72, 700, "bf16", seed=7, ignored=0.0)
    c.targets[5] = -1
    want = [t.clone() for t in c.run()]
    c.targets[5] = 700
    got = c.run(check=False)
    torch.cuda.synchronize()
    assert last_device_error() == L.ERR_INVALID_ARG
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_what_is_not_finite_stays_in_its_row(cuda):
    import torch

    c = Case(300, 72, 700, "f32", seed=8, ignored=0.0)
    want = [t.clone() for t in c.run()]
    c.hidden[7, 3] = float("nan")
    loss, logsum, gh, gw = c.run()
    rest = torch.arange(300, device="cuda") != 7
    assert loss[7].isnan() and gh[7].isnan().all()
    assert torch.equal(loss[rest], want[0][rest]) and torch.equal(gh[rest], want[2][rest])
    c.hidden[7, 3] = 1.0
    c.gain[9] = float("inf")
    loss, logsum, gh, gw = c.run()
    rest = torch.arange(300, device="cuda") != 9
    assert gh[rest].isfinite().all() and not gh[9].isfinite().any()


@pytest.mark.parametrize("dtype", DTYPES)
def test_large_logits(cuda, dtype):
    # exp of them would overflow: the largest is taken out first
    import torch

    c = Case(64, 64, 300, dtype, seed=9, ignored=0.0)
    c.hidden[:32] *= 400
    c.hidden[32:] = 0
    c.run()
    z = c.hidden.double() @ c.weight.double().t()
    want = torch.logsumexp(z, 1)
    assert ((c.logsum.double() - want).abs() <= 1e-5 * (1 + z.abs().amax(1))).all()
    assert ((c.logsum[32:].double() - np.log(300)).abs() <= 1e-6 * np.log(300)).all()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_runs_give_the_same_bits(cuda, dtype):
    import torch

    c = Case(700, 264, 9001, dtype, seed=10)
    want = [t.clone() for t in c.run()]
    for _ in range(4):
        assert all(torch.equal(a, b) for a, b in zip(c.run(), want))


def test_two_streams_at_once(cuda):
    import torch
    from lc_parallel_primitive_b200 import Stream

    cases = [Case(900, 512, 20000, "bf16", seed=11), Case(300, 100, 5000, "f16", seed=12)]
    want = [[t.clone() for t in c.run()] for c in cases]
    streams, temps = [torch.cuda.Stream() for _ in cases], [c.temp() for c in cases]
    torch.cuda.synchronize()
    for _ in range(4):
        got = []
        for c, s, t in zip(cases, streams, temps):
            with torch.cuda.stream(s):
                got.append(c.run(stream=Stream(s), temp=t, check=False))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_captured_and_replayed(cuda):
    import torch

    c = Case(300, 72, 700, "bf16", seed=13)
    temp = c.temp()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        c.run(temp=temp, check=False)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = c.run(temp=temp, check=False)
    c.hidden.mul_(0.5)
    c.targets[::3] = -1
    graph.replay()
    graph.replay()
    torch.cuda.synchronize()
    held = [t.clone() for t in got]
    assert all(torch.equal(a, b) for a, b in zip(c.run(temp=temp), held))
    c.check()


def test_gradient_is_a_difference(cuda):
    import torch

    c = Case(40, 32, 100, "f32", seed=14, gain=1.0)
    _, _, gh, gw = [t.clone() for t in c.run()]
    r = torch.Generator(device="cuda").manual_seed(0)
    for t, g in ((c.hidden, gh), (c.weight, gw)):
        d = torch.randn(t.shape, generator=r, device="cuda")
        h, old = 2.0 ** -6, t.clone()
        t.copy_(old + h * d)
        up = c.run(grads="")[0].double().sum()
        t.copy_(old - h * d)
        down = c.run(grads="")[0].double().sum()
        t.copy_(old)
        want, got = float(up - down) / (2 * h), float((g.double() * d).sum())
        # the losses' sums are off by 40 * 16 * 2^-24 / h at most; the third derivative's part is h^2 of the gradients' size
        size = float(d.norm())
        assert abs(want - got) <= 40 * 16 * U / h * 8 + h * h * size * 2, (want, got)


def test_no_rows(cuda):
    import torch
    from lc_parallel_primitive_b200 import CommandList, DeviceCrossEntropy, Stream, temp_buffer

    m, c = DeviceCrossEntropy(), CommandList()
    m.create()
    x, w, t = torch.zeros(0, 8, device="cuda"), torch.ones(5, 8, device="cuda"), torch.zeros(0, dtype=torch.int32, device="cuda")
    v = torch.zeros(0, device="cuda")
    g = torch.full((5, 8), 55.0, device="cuda")
    temp = temp_buffer(m.GetTempStorageBytes(0, 8, 5, torch.float32))
    m.Forward(c, temp, x, w, t, v, v)
    m.Backward(c, temp, x, w, t, v, v, x.clone(), g)
    Stream() << c.commit()
    torch.cuda.synchronize()
    assert (g == 0).all()
