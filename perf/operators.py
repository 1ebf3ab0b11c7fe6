"""Measured cases of the sequence operators: the gated linear recurrence (forward, forward with
backward, one token) and beam search (selection, reordering of states).

`run` computes a case in plain torch (`own` false: float32, rounded once at the end) or through
DeviceLinearRecurrence / DeviceBeamSearch (`own` true); `exact` computes it in float64.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
BYTES = {"bf16": 2, "f16": 2, "f32": 4}
EOS = 2  # end-of-sequence token of the selection cases


def listed():
    return [
        # Prefill of one short prompt: a few microseconds of work, launch latency counts.
        dict(name="forward_prompt", op="forward", seqs=1, rows=128, packed=False, channels=1024, dtype="bf16", mode="sigmoid"),
        # Prefill of one long document: the time axis is the only source of parallel work beside the channels.
        dict(name="forward_long", op="forward", seqs=1, rows=65536, packed=False, channels=2048, dtype="bf16", mode="sigmoid"),
        # Packed prompts of lognormal lengths (some empty), coefficients computed by the caller, odd channel count.
        dict(name="forward_packed", op="forward", seqs=512, rows=65536, packed=True, channels=1001, dtype="f32", mode="linear"),
        # Training step of one layer: a batch of equal sequences.
        dict(name="train_batch", op="train", seqs=8, rows=16384, packed=False, channels=2048, dtype="bf16", mode="sigmoid"),
        # The same in float32 with odd sizes: ragged tiles in time and channels.
        dict(name="train_odd", op="train", seqs=3, rows=3063, packed=False, channels=509, dtype="f32", mode="linear"),
        # Training on packed documents of lognormal lengths.
        dict(name="train_packed", op="train", seqs=300, rows=32768, packed=True, channels=1536, dtype="f16", mode="sigmoid"),
        # One token for four beams of one request.
        dict(name="step_one", op="step", rows=4, beams=4, channels=1024, dtype="bf16", mode="sigmoid"),
        # One token for a full serving batch, four beams each.
        dict(name="step_many", op="step", rows=2048, beams=4, channels=4096, dtype="bf16", mode="sigmoid"),
        # Selection for one request.
        dict(name="select_one", op="select", batches=1, beams=4, vocab=32000, dtype="bf16"),
        # Selection for a full batch over a large odd vocabulary in float32.
        dict(name="select_many", op="select", batches=64, beams=8, vocab=100003, dtype="f32"),
        # States of a small model follow the four beams of one request.
        dict(name="reorder_one", op="reorder", layers=8, rows=4, beams=4, channels=1024, dtype="f32"),
        # States of all layers of a large model follow the beams of a full batch.
        dict(name="reorder_many", op="reorder", layers=32, rows=512, beams=8, channels=4096, dtype="f32"),
    ]


def _spread(rng, low, high):
    """A whole number from low to high, even over its logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


MOST_BYTES = 800e6  # the largest listed case's


def draw(rng):
    while True:
        op = rng.choice(["forward", "train", "step", "select", "reorder"])
        dtype = rng.choice(["bf16", "f16", "f32"])
        if op in ("forward", "train"):
            packed = rng.random() < 0.4
            channels = _spread(rng, 128, 4096)
            if rng.random() < 0.6:
                channels = max(8, channels // 8 * 8)
            if packed:
                rows = _spread(rng, 512, 65536)
                seqs = max(1, rows // rng.randint(80, 160))
            else:
                seqs = _spread(rng, 1, 32)
                rows = seqs * _spread(rng, 64, 65536)
            case = dict(op=op, seqs=seqs, rows=rows, packed=packed, channels=channels, dtype=dtype,
                        mode=rng.choice(["sigmoid", "sigmoid", "linear"]))
        elif op == "step":
            beams = rng.choice([1, 2, 4, 8])
            channels = _spread(rng, 512, 4096)
            if rng.random() < 0.6:
                channels = channels // 8 * 8
            case = dict(op=op, rows=beams * _spread(rng, 1, 512), beams=beams, channels=channels, dtype=dtype,
                        mode=rng.choice(["sigmoid", "linear"]))
        elif op == "select":
            case = dict(op=op, batches=_spread(rng, 1, 96), beams=rng.choice([1, 2, 3, 4, 5, 8, 12, 16]),
                        vocab=_spread(rng, 8000, 131072), dtype=dtype)
        else:
            beams = rng.choice([2, 4, 5, 8])
            case = dict(op=op, layers=_spread(rng, 4, 48), rows=beams * _spread(rng, 1, 96), beams=beams,
                        channels=_spread(rng, 512, 4096), dtype=dtype)
        if work(case)["bytes"] <= MOST_BYTES and 3072 not in case.values():
            return case


def work(case):
    e = BYTES[case["dtype"]]
    if case["op"] in ("forward", "train"):
        n = case["rows"] * case["channels"]
        states = 4 * case["seqs"] * case["channels"]
        if case["op"] == "forward":  # gate, in, initial states -> out, last states
            return {"bytes": 3 * e * n + 2 * states, "flops": 10 * n}
        # forward as above; backward: gate, in, grad_out, grad_last, initial states -> grad_gate, grad_in, grad_init
        return {"bytes": 8 * e * n + 5 * states, "flops": 30 * n}
    if case["op"] == "step":  # gate, in, old state, parent -> out, new state
        n = case["rows"] * case["channels"]
        return {"bytes": (3 * e + 8) * n + 4 * case["rows"], "flops": 10 * n}
    if case["op"] == "select":
        rows = case["batches"] * case["beams"]
        return {"bytes": e * rows * case["vocab"] + 5 * rows + 13 * rows, "flops": 4 * rows * case["vocab"]}
    n = case["layers"] * case["rows"] * case["channels"]
    return {"bytes": 2 * e * n + 4 * case["rows"], "flops": 0}


# ---- inputs ------------------------------------------------------------------------------------
def _lengths(case, seed):
    """Sequence lengths: lognormal (mu 4, sigma 1.5) with some empty, scaled to fill the rows exactly."""
    r = np.random.RandomState(seed % (1 << 31))
    n = r.lognormal(4.0, 1.5, case["seqs"])
    n[r.rand(case["seqs"]) < 0.02] = 0
    if n.sum() == 0:
        n[0] = 1
    edge = np.floor(np.cumsum(n) * (case["rows"] / n.sum()) + 0.5).astype(np.int64)
    edge[-1] = case["rows"]
    return np.diff(np.concatenate([[0], np.minimum(edge, case["rows"])]))


def _recurrence_inputs(case, shape, normal):
    """(gate, in): gate logits with memories from a few tokens to some hundreds across the channels, or decays and
    inputs scaled as a normalised recurrence has them."""
    dt = DTYPES[case["dtype"]]
    bias = torch.linspace(-1.0, 5.0, shape[-1], device="cuda")
    gate = normal(shape) + bias
    x = normal(shape)
    if case["mode"] == "linear":
        gate = torch.sigmoid(gate)
        x = x * torch.sqrt(1 - gate * gate)
    return gate.to(dt), x.to(dt)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def normal(shape):
        return torch.randn(shape, generator=g, device="cuda")

    op, dt = case["op"], DTYPES[case["dtype"]]
    s = {"case": case, "op": op}
    if op in ("forward", "train"):
        rows, d, seqs = case["rows"], case["channels"], case["seqs"]
        s["gate"], s["in"] = _recurrence_inputs(case, (rows, d), normal)
        s["init"] = normal((seqs, d))
        if case["packed"]:
            lengths = _lengths(case, seed)
            offsets = np.concatenate([[0], np.cumsum(lengths)])
            s["offsets"] = torch.from_numpy(offsets.astype(np.int32)).cuda()
        else:
            lengths = np.full(seqs, rows // seqs)
        # the sequences that are not empty, their first and last rows and the longest length, for the plain form
        start, full = np.cumsum(lengths) - lengths, np.flatnonzero(lengths)
        s["full"], s["first"], s["end"] = (torch.from_numpy(v).cuda() for v in (full, start[full], (start + lengths)[full] - 1))
        s["start"], s["lengths"], s["longest"] = start, lengths, int(lengths.max())
        if op == "train":
            s["grad_out"] = (normal((rows, d)) / math.sqrt(d)).to(dt)
            s["grad_last"] = normal((seqs, d)) / math.sqrt(d)
    elif op == "step":
        rows, d = case["rows"], case["channels"]
        s["gate"], s["in"] = _recurrence_inputs(case, (rows, d), normal)
        s["states"] = normal((rows, d))
        s["parents"] = _parents(case, g)
    elif op == "select":
        b, k, v = case["batches"], case["beams"], case["vocab"]
        z = normal((b * k, v)) * 2.5
        z[:, :8] += 4.0
        z.masked_fill_(torch.rand((b * k, v), generator=g, device="cuda") < 0.02, float("-inf"))  # banned tokens
        s["logits"] = z.to(dt)
        s["scores"] = torch.sort(-20 - 3 * torch.rand((b, k), generator=g, device="cuda"), dim=1, descending=True)[0]
        finished = torch.rand((b, k), generator=g, device="cuda") < 0.1
        finished[:, 0] = False
        s["finished"] = finished.to(torch.uint8)
    else:
        s["states"] = normal((case["layers"], case["rows"], case["channels"])).to(dt)
        s["parents"] = _parents(case, g)
    if own:
        _prepare_own(s)
    return s


def _parents(case, g):
    rows, k = case["rows"], case["beams"]
    first = torch.arange(rows, device="cuda") // k * k
    return (first + torch.randint(0, k, (rows,), generator=g, device="cuda")).to(torch.int32)


# ---- plain forms -------------------------------------------------------------------------------
def _coefficients(gate, x, mode):
    """(a, b) of h = a h' + b, in the type of `gate`."""
    if mode == "linear":
        return gate, x
    a = 1 / (1 + torch.exp(-gate))
    return a, (1 - a) * x


def _affine_scan(a, b, longest):
    """All h_t = a_t h_{t-1} + b_t along dim 0, by doubling; `longest`: no chain is longer."""
    step = 1
    while step < longest:
        b = torch.cat([b[:step], b[step:] + a[step:] * b[:-step]])
        a = torch.cat([a[:step], a[step:] * a[:-step]])
        step *= 2
    return b


def _plain_forward(s):
    """(out, last, a, previous state of each row), float32."""
    a, b = _coefficients(s["gate"].float(), s["in"].float(), s["case"]["mode"])
    full, first, end = s["full"], s["first"], s["end"]
    cut, head = a.clone(), b.clone()
    head[first] = b[first] + a[first] * s["init"][full]
    cut[first] = 0  # no chain passes a sequence's first row
    h = _affine_scan(cut, head, s["longest"])
    last = s["init"].clone()
    last[full] = h[end]
    before = torch.cat([h[:1], h[:-1]])
    before[first] = s["init"][full]
    return h, last, a, before


def _plain_train(s):
    h, last, a, before = _plain_forward(s)
    full, first, end = s["full"], s["first"], s["end"]
    grad = s["grad_out"].to(torch.float32, copy=True)
    grad[end] += s["grad_last"][full]
    follow = torch.cat([a[1:], a[:1]])
    follow[end] = 0
    lam = _affine_scan(follow.flip(0), grad.flip(0), s["longest"]).flip(0)
    grad_init = s["grad_last"].clone()
    grad_init[full] = (a * lam)[first]
    if s["case"]["mode"] == "linear":
        grad_gate, grad_in = lam * before, lam
    else:
        grad_gate, grad_in = lam * (before - s["in"].float()) * a * (1 - a), (1 - a) * lam
    dt = s["gate"].dtype
    return {"out": h.to(dt), "last": last, "grad_gate": grad_gate.to(dt), "grad_in": grad_in.to(dt), "grad_init": grad_init}


def _ordered(v):
    """int64 with the order of float32 values (NaN as -inf, the two zeros alike)."""
    v = torch.where(torch.isnan(v), torch.full_like(v, float("-inf")), v) + 0.0
    i = v.view(torch.int32)
    return (i ^ ((i >> 31) & 0x7FFFFFFF)).long()


def _plain_select(s):
    b, k, v = s["case"]["batches"], s["case"]["beams"], s["case"]["vocab"]
    low = float("-inf")
    z = s["logits"].float()
    top = z.amax(1, keepdim=True)
    logsum = torch.log(torch.exp(z - top).sum(1, keepdim=True))
    # a beam's k best tokens, equal logits by token
    key = (_ordered(z) << 32) + (v - 1 - torch.arange(v, device=z.device))
    token = v - 1 - (torch.topk(key, k, dim=1)[0] & 0xFFFFFFFF)
    best = torch.gather(z, 1, token)
    score = s["scores"].reshape(-1, 1) + ((best - top) - logsum)
    # a finished beam has one candidate: it stays as it is
    done = s["finished"].reshape(-1, 1) != 0
    stay = torch.where(torch.arange(k, device=z.device) == 0, s["scores"].reshape(-1, 1), torch.full_like(score, low))
    score = torch.where(done, stay, score).reshape(b, k * k)
    token = torch.where(done, torch.full_like(token, EOS), token).reshape(b, k * k)
    # the k best of all, equal scores by beam and place in its list
    key = (_ordered(score) << 32) + (k * k - 1 - torch.arange(k * k, device=z.device))
    place = k * k - 1 - (torch.topk(key, k, dim=1)[0] & 0xFFFFFFFF)
    token = torch.gather(token, 1, place).to(torch.int32)
    parent = torch.arange(b, device=z.device)[:, None] * k + place // k
    finished = (s["finished"].reshape(-1)[parent] != 0) | (token == EOS)
    return {"scores": torch.gather(score, 1, place), "tokens": token, "parents": parent.to(torch.int32),
            "finished": finished.to(torch.uint8)}


def _plain(s):
    op = s["op"]
    if op == "forward":
        h, last, _, _ = _plain_forward(s)
        return {"out": h.to(s["gate"].dtype), "last": last}
    if op == "train":
        return _plain_train(s)
    if op == "step":
        a, b = _coefficients(s["gate"].float(), s["in"].float(), s["case"]["mode"])
        h = a * s["states"][s["parents"].long()] + b
        return {"states": h, "out": h.to(s["gate"].dtype)}
    if op == "select":
        return _plain_select(s)
    return {"states": s["states"][:, s["parents"].long()]}


# ---- through the framework ---------------------------------------------------------------------
def _prepare_own(s):
    """The buffers, temp storage and modules that a program keeps from call to call."""
    import lc_parallel_primitive_b200 as P

    case, op = s["case"], s["op"]
    s["stream"], s["cmdlist"] = P.Stream(), P.CommandList()
    if op in ("forward", "train", "step"):
        s["module"] = P.DeviceLinearRecurrence()
    else:
        s["module"] = P.DeviceBeamSearch()
    s["module"].create()
    if op in ("forward", "train"):
        rows, d = s["gate"].shape
        s["sequences"] = s["offsets"] if case["packed"] else rows // case["seqs"]
        s["temp"] = P.temp_buffer(s["module"].GetTempStorageBytes(rows, d))
        s["out"], s["last"] = torch.empty_like(s["gate"]), torch.empty_like(s["init"])
        if op == "train":
            s["saved"] = P.temp_buffer(s["module"].GetSavedStateBytes(rows, d))
            s["grad_gate"], s["grad_in"] = torch.empty_like(s["gate"]), torch.empty_like(s["gate"])
            s["grad_init"] = torch.empty_like(s["init"])
    elif op == "step":
        s["new"], s["out"] = torch.empty_like(s["states"]), torch.empty_like(s["gate"])
    elif op == "select":
        b, k, v = case["batches"], case["beams"], case["vocab"]
        s["temp"] = P.temp_buffer(s["module"].GetTempStorageBytes(b, k, v))
        s["scores_out"] = torch.empty_like(s["scores"])
        s["tokens"] = torch.empty((b, k), dtype=torch.int32, device="cuda")
        s["parents"] = torch.empty_like(s["tokens"])
        s["finished_out"] = torch.empty_like(s["finished"])
    else:
        s["new"] = torch.empty_like(s["states"])


def _own(s):
    op, m, c = s["op"], s["module"], s["cmdlist"]
    if op == "forward":
        m.Forward(c, s["temp"], s["gate"], s["in"], s["out"], s["sequences"], d_init=s["init"], d_last=s["last"],
                  mode=s["case"]["mode"])
        s["stream"] << c.commit()
        return {"out": s["out"], "last": s["last"]}
    if op == "train":
        mode = s["case"]["mode"]
        m.Forward(c, s["temp"], s["gate"], s["in"], s["out"], s["sequences"], d_init=s["init"], d_last=s["last"],
                  d_saved=s["saved"], mode=mode)
        m.Backward(c, s["temp"], s["gate"], s["in"], s["saved"], s["grad_out"], s["grad_gate"], s["grad_in"],
                   s["sequences"], d_init=s["init"], d_grad_last=s["grad_last"], d_grad_init=s["grad_init"], mode=mode)
        s["stream"] << c.commit()
        return {"out": s["out"], "last": s["last"], "grad_gate": s["grad_gate"], "grad_in": s["grad_in"],
                "grad_init": s["grad_init"]}
    if op == "step":
        m.Step(c, s["gate"], s["in"], s["states"], s["new"], s["out"], d_parents=s["parents"], mode=s["case"]["mode"])
        s["stream"] << c.commit()
        return {"states": s["new"], "out": s["out"]}
    if op == "select":
        m.Select(c, s["temp"], s["logits"], s["scores"], s["finished"], s["scores_out"], s["tokens"], s["parents"],
                 s["finished_out"], eos_token=EOS)
        s["stream"] << c.commit()
        return {"scores": s["scores_out"], "tokens": s["tokens"], "parents": s["parents"], "finished": s["finished_out"]}
    m.Reorder(c, s["states"], s["new"], s["parents"])
    s["stream"] << c.commit()
    return {"states": s["new"]}


def run(state):
    return _own(state) if own else _plain(state)


# ---- from the definition, in 64 bits -----------------------------------------------------------
def exact(case, seed):
    if case["op"] in ("forward", "train") and case["rows"] * case["channels"] > 3 * 10**8:
        return None
    s = prepare(case, seed)
    with torch.no_grad():
        if case["op"] in ("forward", "train"):
            return _exact_recurrence(s)
        if case["op"] == "step":
            g, x = s["gate"].double(), s["in"].double()
            old = s["states"].double().index_select(0, s["parents"].long())
            if case["mode"] == "linear":
                h = torch.addcmul(x, g, old)
            else:
                h = torch.lerp(x, old, torch.sigmoid(g))
            return {"states": h, "out": h}
        if case["op"] == "select":
            return _exact_select(s)
        return {"states": s["states"].double().index_select(1, s["parents"].long())}


def _exact_recurrence(s):
    """One token after the other, all sequences that are long enough at once."""
    mode, train = s["case"]["mode"], s["op"] == "train"
    g, x = s["gate"].double(), s["in"].double()
    order = np.argsort(-s["lengths"], kind="stable")
    counts, start = s["lengths"][order], torch.from_numpy(s["start"][order]).cuda()
    order = torch.from_numpy(order).cuda()
    live = [int(np.searchsorted(-counts, -t, side="left")) for t in range(int(counts[0]))]  # sequences with count > t
    a_of = (lambda r: g[r]) if mode == "linear" else (lambda r: torch.sigmoid(g[r]))
    state = s["init"].double()[order]
    out = torch.empty_like(g)
    for t, n in enumerate(live):
        r = start[:n] + t
        a = a_of(r)
        state[:n] = torch.addcmul(x[r], a, state[:n]) if mode == "linear" else torch.lerp(x[r], state[:n], a)
        out[r] = state[:n]
    back = torch.argsort(order)
    got = {"out": out, "last": state[back]}
    if not train:
        return got
    grad = s["grad_out"].double()
    init = s["init"].double()[order]
    mu = s["grad_last"].double()[order]
    dg, dx = torch.empty_like(g), torch.empty_like(g)
    for t in range(len(live) - 1, -1, -1):
        n = live[t]
        r = start[:n] + t
        a = a_of(r)
        lam = grad[r] + mu[:n]
        h = out[r - 1] if t else init[:n]
        if mode == "linear":
            dg[r], dx[r] = lam * h, lam
        else:
            dg[r], dx[r] = lam * (h - x[r]) * a * (1 - a), lam * (1 - a)
        mu[:n] = a * lam
    got.update(grad_gate=dg, grad_in=dx, grad_init=mu[back])
    return got


def _exact_select(s):
    k = s["case"]["beams"]
    logp = torch.log_softmax(s["logits"].double(), dim=1)
    best = torch.sort(logp, dim=1, descending=True)[0][:, :k]
    score = s["scores"].double().reshape(-1, 1) + best
    done = s["finished"].reshape(-1) != 0
    score[done] = float("-inf")
    score[done, 0] = s["scores"].double().reshape(-1)[done]
    score = torch.sort(score.reshape(s["case"]["batches"], k * k), dim=1, descending=True)[0][:, :k]
    return {"scores": score, "tokens": None, "parents": None, "finished": None}
