"""DeviceBeamSearch on the GPU against the float64 form."""
import numpy as np
import pytest

from lc_parallel_primitive_b200 import _lib as L
from tests import sequence_reference as R

pytestmark = pytest.mark.gpu

DTYPES = ["f32", "f16", "bf16"]


def torch_dtype(name):
    import torch

    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[name]


def select(logits, scores, finished, eos):
    """(scores, tokens, parents, finished) as numpy arrays; logits a device tensor."""
    import torch
    from lc_parallel_primitive_b200 import CommandList, DeviceBeamSearch, Stream, last_device_error, temp_buffer

    b, k = scores.shape
    m, c = DeviceBeamSearch(), CommandList()
    m.create()
    temp = temp_buffer(m.GetTempStorageBytes(b, k, logits.shape[-1]))
    temp.fill_(0x5A5A5A5A)
    s = torch.from_numpy(scores).cuda()
    f = None if finished is None else torch.from_numpy(finished).cuda()
    out = [torch.full((b, k), 99, dtype=t, device="cuda")
           for t in (torch.float32, torch.int32, torch.int32, torch.uint8)]
    m.Select(c, temp, logits, s, f, *out, eos_token=eos)
    Stream() << c.commit()
    torch.cuda.synchronize()
    L.check(last_device_error())
    return [t.cpu().numpy() for t in out]


def inputs(b, k, v, dtype, seed, banned=0.0):
    import torch

    r = np.random.RandomState(seed)
    z = r.randn(b * k, v) * 3
    z[r.rand(b * k, v) < banned] = -np.inf
    logits = torch.from_numpy(z).to(torch_dtype(dtype)).cuda()
    scores = np.sort(-r.rand(b, k) * 4 - 5, axis=1)[:, ::-1].astype(np.float32).copy()
    return logits, scores


def bound(want, vocab):
    # score + ((z - m) - log s): each of the three float32 operations rounds a value of at most |score| + |logp|
    # (3u), the inputs are exact, and s, a sum of vocab positive terms each with a 2-ulp exponential and an argument
    # rounded by u |z - m|, is off by at most (4 + 40 + log2(vocab) + 8) u relative (pairwise over threads, a few
    # terms in a row), which log turns into an absolute error; log itself 1 ulp of at most 16.
    u = 2.0 ** -24
    return 3 * u * (np.abs(want) + 40) + (52 + np.log2(vocab + 1) + vocab / 256) * u + 16 * u


def check(logits, scores, finished, eos):
    z = logits.float().cpu().numpy().reshape(-1, logits.shape[-1])
    ws, wt, wp, wf, gap = R.beam_select(z, scores, finished, eos)
    s, t, p, f = select(logits, scores, finished, eos)
    fine = np.isfinite(ws)
    assert np.array_equal(np.isneginf(s), ~fine)
    tol = bound(ws[fine], z.shape[1])
    assert (np.abs(s[fine] - ws[fine]) <= tol).all()
    # where two scores of different beams are nearer than both their bounds, either order is right
    sure = gap > 2 * (tol.max() if tol.size else 0)
    assert sure.mean() > 0.9 or len(sure) < 4, gap
    assert np.array_equal(t[sure], wt[sure]) and np.array_equal(p[sure], wp[sure])
    assert np.array_equal(f[sure], wf[sure])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("b,k,v", [(1, 1, 1), (1, 1, 1000), (1, 4, 32000), (3, 4, 1001), (2, 8, 5000), (5, 3, 257),
                                   (2, 16, 4099), (1, 32, 3000), (7, 5, 40), (2, 2, 70001), (40, 2, 777)])
def test_select(cuda, dtype, b, k, v):
    logits, scores = inputs(b, k, v, dtype, seed=b * 100 + k)
    check(logits, scores, None, -1)


@pytest.mark.parametrize("dtype", DTYPES)
def test_large_vocabulary(cuda, dtype):
    logits, scores = inputs(2, 4, 300001, dtype, seed=1)
    check(logits, scores, None, 7)


@pytest.mark.parametrize("k,v", [(4, 3), (8, 1), (32, 5), (2, 2)])
def test_fewer_tokens_than_beams(cuda, k, v):
    logits, scores = inputs(3, k, v, "f32", seed=2)
    check(logits, scores, None, -1)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("banned", [0.3, 0.99])
def test_banned_tokens(cuda, dtype, banned):
    logits, scores = inputs(4, 4, 900, dtype, seed=3, banned=banned)
    check(logits, scores, None, 5)


def test_finished_beams_stay(cuda):
    logits, scores = inputs(6, 4, 800, "f32", seed=4)
    r = np.random.RandomState(4)
    finished = (r.rand(6, 4) < 0.5).astype(np.uint8)
    finished[0], finished[1] = 1, 0
    logits[:, 2] += 9.0  # the eos token comes up often
    check(logits, scores, finished, 2)
    s, t, p, f = select(logits, scores, finished, 2)
    assert np.array_equal(s[0], scores[0]) and (t[0] == 2).all() and np.array_equal(p[0], np.arange(4)) and f[0].all()


def test_first_step_has_one_live_beam(cuda):
    # all beams but the first at -inf: the four best tokens of beam 0
    logits, scores = inputs(3, 4, 5000, "bf16", seed=5)
    scores[:, 1:], scores[:, 0] = -np.inf, 0
    check(logits, scores, None, -1)
    _, _, p, _ = select(logits, scores, None, -1)
    assert (p == np.arange(3)[:, None] * 4).all()


def test_rows_with_nothing(cuda):
    # rows all -inf or NaN, an entry whose beams all are, scores of NaN
    logits, scores = inputs(4, 3, 500, "f32", seed=6)
    logits[0] = float("-inf")
    logits[4] = float("nan")
    logits[6:9] = float("-inf")
    logits[9, ::2] = float("nan")
    scores[3, 1] = np.nan
    check(logits, scores, None, 3)
    s, t, p, f = select(logits, scores, None, 3)
    assert np.isneginf(s[2]).all() and (t[2] == 3).all() and f[2].all() and np.array_equal(p[2], [6, 7, 8])


def test_lowest_value_as_a_mask(cuda):
    # masks of the type's lowest finite value: no NaN, and never preferred
    import torch

    for dtype in DTYPES:
        logits, scores = inputs(2, 4, 600, dtype, seed=7)
        low = torch.finfo(logits.dtype).min
        logits[:, 3:590] = low
        z = logits.float().cpu().numpy()
        s, t, p, f = select(logits, scores, None, -1)
        ws, wt, wp, wf, gap = R.beam_select(z, scores, None, -1)
        assert np.allclose(s, ws, rtol=1e-5) and np.array_equal(t, wt) and np.array_equal(p, wp)


def test_infinite_logits_share_the_probability(cuda):
    logits, scores = inputs(1, 2, 400, "f32", seed=8)
    logits[0, [5, 300]] = float("inf")
    check(logits, scores, None, -1)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("v", [5, 300, 5000, 40000])
def test_equal_logits_go_by_token(cuda, dtype, v):
    import torch

    logits = torch.zeros((8, v), dtype=torch_dtype(dtype), device="cuda")
    logits[1::2] = -0.0
    scores = np.tile(np.array([0, -1000, -2000, -3000], np.float32), (2, 1))
    s, t, p, f = select(logits, scores, None, -1)
    k = min(4, v)
    assert (t[:, :k] == np.arange(k)).all() and (p[:, :k] == [[0], [4]]).all()
    # a few levels, so that ties straddle every boundary
    r = np.random.RandomState(9)
    logits = torch.from_numpy(r.randint(0, 3, (8, v)).astype(np.float32)).to(torch_dtype(dtype)).cuda()
    s, t, p, f = select(logits, scores, None, -1)
    z = logits.float().cpu().numpy()
    ws, wt, wp, wf, gap = R.beam_select(z, scores, None, -1)
    assert np.array_equal(t, wt) and np.array_equal(p, wp)


def test_equal_scores_go_by_beam(cuda):
    import torch

    z = torch.randn((1, 900), device="cuda").repeat(4, 1)
    s, t, p, f = select(z, np.zeros((1, 4), np.float32), None, -1)
    best = int(z[0].argmax())
    assert (t == best).all() and np.array_equal(p, [[0, 1, 2, 3]]) and (s == s[0, 0]).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("pad,shift", [(1, 0), (8, 0), (0, 1), (5, 3)])
def test_strides_and_alignment(cuda, dtype, pad, shift):
    import torch

    logits, scores = inputs(2, 4, 9003, dtype, seed=10)
    buf = torch.full((8 * (9003 + pad) + shift,), 60000.0, dtype=logits.dtype, device="cuda")  # best, if read
    view = buf[shift:].view(8, 9003 + pad)[:, :9003]
    view.copy_(logits)
    check(view, scores, None, -1)
    want, got = select(logits, scores, None, -1), select(view, scores, None, -1)
    assert all(np.array_equal(p, q) for p, q in zip(want[1:], got[1:]))


def test_repeats_bit_for_bit(cuda):
    logits, scores = inputs(3, 8, 50000, "f32", seed=11)
    first = select(logits, scores, None, -1)
    for _ in range(3):
        assert all(np.array_equal(p, q) for p, q in zip(first, select(logits, scores, None, -1)))


def test_logits_past_32_bits(cuda):
    # the last rows start beyond 2^32 elements
    import torch

    stride = (1 << 30) + 8
    buf = torch.zeros(5 * stride, dtype=torch.bfloat16, device="cuda")
    logits, scores = inputs(1, 5, 2000, "bf16", seed=12)
    view = buf.view(5, stride)[:, :2000]
    view.copy_(logits)
    check(view, scores, None, -1)


# ---- reordering ----------------------------------------------------------------------------------
def reorder(x, out, parents):
    import torch
    from lc_parallel_primitive_b200 import CommandList, DeviceBeamSearch, Stream

    m, c = DeviceBeamSearch(), CommandList()
    m.create()
    m.Reorder(c, x, out, parents)
    Stream() << c.commit()
    torch.cuda.synchronize()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "uint8", "int64"])
@pytest.mark.parametrize("layers,rows,width", [(1, 1, 1), (3, 4, 64), (2, 5, 33), (1, 7, 1000), (4, 3, 4099), (70, 2, 16),
                                               (1, 300, 7)])
def test_reorder(cuda, dtype, layers, rows, width):
    import torch

    x = torch.randint(0, 100, (layers, rows, width), device="cuda").to(getattr(torch, dtype))
    r = np.random.RandomState(rows)
    parents = torch.from_numpy(r.randint(0, rows, rows).astype(np.int32)).cuda()
    out = torch.full_like(x, 101)
    reorder(x, out, parents)
    assert torch.equal(out, x[:, parents.long()])
    if layers == 1:
        out = torch.full_like(x[0], 101)
        reorder(x[0], out, parents)
        assert torch.equal(out, x[0, parents.long()])


@pytest.mark.parametrize("off,pad", [(1, 0), (0, 3), (3, 5), (4, 4), (0, 16)])
def test_reorder_strides(cuda, off, pad):
    import torch

    big = torch.randint(0, 100, (3, 6, 40 + pad + off), device="cuda", dtype=torch.uint8)
    x = big[:, :, off:off + 40]
    parents = torch.tensor([5, 5, 0, 2], dtype=torch.int32, device="cuda")
    dst = torch.full((3, 4, 50), 101, dtype=torch.uint8, device="cuda")
    reorder(x, dst[:, :, 7:47], parents)
    assert torch.equal(dst[:, :, 7:47], x[:, parents.long()])
    assert (dst[:, :, :7] == 101).all() and (dst[:, :, 47:] == 101).all()


def test_reorder_missing_parents(cuda):
    import torch
    from lc_parallel_primitive_b200 import last_device_error

    x = torch.randn((2, 4, 100), device="cuda")
    out = torch.empty_like(x)
    parents = torch.tensor([0, -1, 3, -5], dtype=torch.int32, device="cuda")
    reorder(x, out, parents)
    assert torch.equal(out[:, [0, 2]], x[:, [0, 3]]) and (out[:, [1, 3]] == 0).all()
    assert last_device_error() == L.OK
    parents[1] = 4  # no such row: reported, nothing read
    reorder(x, out, parents)
    assert (out[:, 1] == 0).all() and torch.equal(out[:, 2], x[:, 3])
    assert last_device_error() == L.ERR_INVALID_ARG and last_device_error() == L.OK
