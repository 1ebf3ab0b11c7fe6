"""Measured cases of the gated delta rule (forward, forward with backward, one token) and of the softmax cross
entropy over a vocabulary from hidden states (loss, loss with gradients).

`run` computes a case in plain torch (`own` false: float32, rounded once at the end) or through DeviceDeltaRule /
DeviceCrossEntropy (`own` true); `exact` computes it in float64, the delta rule token by token.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
BYTES = {"bf16": 2, "f16": 2, "f32": 4}
CHUNK = 64  # rows that the plain form of the delta rule takes at once


def _delta(name, op, seqs, rows, heads, key_heads, key_dim, value_dim, dtype, packed=False):
    return dict(name=name, op=op, seqs=seqs, rows=rows, packed=packed, heads=heads, key_heads=key_heads, key_dim=key_dim,
                value_dim=value_dim, dtype=dtype)


def _step(name, rows, beams, heads, key_heads, key_dim, value_dim, dtype):
    return dict(name=name, op="step", rows=rows, beams=beams, heads=heads, key_heads=key_heads, key_dim=key_dim,
                value_dim=value_dim, dtype=dtype)


def _loss(name, op, rows, channels, vocab, dtype):
    return dict(name=name, op=op, rows=rows, channels=channels, vocab=vocab, dtype=dtype)


def listed():
    return [
        # Prefill of one short prompt of a small model: two chunks, launch latency counts.
        _delta("delta_prompt", "forward", 1, 128, 8, 8, 128, 128, "bf16"),
        # Prefill of one long document: few heads and one sequence, so the chain over its chunks decides.
        _delta("delta_long", "forward", 1, 65536, 16, 8, 128, 128, "bf16"),
        # Packed prompts of lognormal lengths (some empty) in float32, small heads of an odd size.
        _delta("delta_packed", "forward", 256, 32768, 6, 6, 60, 72, "f32", packed=True),
        # Training step of one layer: a batch of equal sequences.
        _delta("delta_train", "train", 8, 16384, 16, 16, 128, 128, "bf16"),
        # Training on packed documents of lognormal lengths, two value heads a key head.
        _delta("delta_train_packed", "train", 100, 12288, 8, 4, 64, 128, "f16", packed=True),
        # One token for four beams of one request.
        _step("delta_step_one", 4, 4, 16, 8, 128, 128, "bf16"),
        # One token for a full serving batch, four beams each.
        _step("delta_step_many", 256, 4, 32, 16, 128, 128, "bf16"),
        # Log-likelihood of one short prompt.
        _loss("loss_prompt", "loss", 48, 1024, 32000, "bf16"),
        # Evaluation over a text: odd rows, channels and vocabulary.
        _loss("loss_text", "loss", 4093, 1001, 50021, "f16"),
        # Training step of a small model in float32.
        _loss("loss_train_small", "loss_train", 2048, 512, 32000, "f32"),
        # Training step over a short batch with a large odd vocabulary.
        _loss("loss_train_odd", "loss_train", 1777, 1000, 100003, "f16"),
        # Training step of a large model.
        _loss("loss_train_large", "loss_train", 8192, 4096, 128000, "bf16"),
    ]


def _spread(rng, low, high):
    """A whole number from low to high, even over its logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


# the largest listed case's of its kind
MOST = {"forward": 8.2e8, "train": 5.7e8, "step": 1e9, "loss": 8.6e12, "loss_train": 2.5e13}


def draw(rng):
    while True:
        op = rng.choice(["forward", "forward", "train", "train", "step", "loss", "loss_train", "loss_train"])
        dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
        if op in ("loss", "loss_train"):
            channels = _spread(rng, 256, 4096)
            if rng.random() < 0.6:
                channels = channels // 8 * 8
            case = _loss(None, op, _spread(rng, 16, 16384), channels, _spread(rng, 4000, 131072), dtype)
        else:
            key_heads = rng.choice([1, 2, 4, 6, 8, 16])
            heads = key_heads * rng.choice([1, 1, 2, 3])
            if rng.random() < 0.6:
                key_dim, value_dim = rng.choice([(64, 64), (64, 128), (128, 64), (128, 128), (128, 128)])
            else:
                key_dim, value_dim = _spread(rng, 16, 128), _spread(rng, 16, 128)
            if op == "step":
                beams = rng.choice([1, 2, 4, 8])
                case = _step(None, beams * _spread(rng, 1, 128), beams, heads, key_heads, key_dim, value_dim, dtype)
            elif rng.random() < 0.4:
                rows = _spread(rng, 256, 32768)
                case = _delta(None, op, max(1, rows // rng.randint(80, 160)), rows, heads, key_heads, key_dim, value_dim,
                              dtype, packed=True)
            else:
                seqs = _spread(rng, 1, 32)
                rows = seqs * _spread(rng, 32, 65536 if op == "forward" else 16384)
                case = _delta(None, op, seqs, rows, heads, key_heads, key_dim, value_dim, dtype)
        del case["name"]
        size = work(case)["flops" if op in ("loss", "loss_train") else "bytes"]
        if size <= MOST[op]:
            return case


def work(case):
    e = BYTES[case["dtype"]]
    if case["op"] in ("loss", "loss_train"):
        n, d, v = case["rows"], case["channels"], case["vocab"]
        if case["op"] == "loss":  # hidden, weight, targets -> loss, log of the sum
            return {"bytes": e * d * (n + v) + 12 * n, "flops": 2 * n * d * v}
        # ... and gradient of the loss -> gradients of hidden and weight
        return {"bytes": 2 * e * d * (n + v) + 16 * n, "flops": 6 * n * d * v}
    qk, val = case["rows"] * case["key_heads"] * case["key_dim"], case["rows"] * case["heads"] * case["value_dim"]
    gates = 4 * case["rows"] * case["heads"]  # bytes of the decays, or of the strengths
    state = case["heads"] * case["key_dim"] * case["value_dim"]
    # a token decays the state, reads it by the key, adds the product of key and value, and reads it by the query
    flops = 7 * case["rows"] * state
    if case["op"] == "step":  # q, k, v, decay, beta, old state, parent -> out, new state
        return {"bytes": e * (2 * qk + 2 * val) + 2 * gates + 8 * case["rows"] * state + 4 * case["rows"], "flops": flops}
    states = 4 * case["seqs"] * state
    if case["op"] == "forward":  # q, k, v, decay, beta, first states -> out, last states
        return {"bytes": e * (2 * qk + 2 * val) + 2 * gates + 2 * states, "flops": flops}
    # ... gradients of out and of the last states -> gradients of all inputs
    return {"bytes": e * (4 * qk + 4 * val) + 4 * gates + 4 * states, "flops": 3 * flops}


# ---- inputs ------------------------------------------------------------------------------------
def _lengths(case, seed):
    """Sequence lengths: lognormal (mu 4, sigma 1.5) with some empty, scaled to fill the rows exactly."""
    if not case["packed"]:
        return np.full(case["seqs"], case["rows"] // case["seqs"])
    r = np.random.RandomState(seed % (1 << 31))
    n = r.lognormal(4.0, 1.5, case["seqs"])
    n[r.rand(case["seqs"]) < 0.02] = 0
    if n.sum() == 0:
        n[0] = 1
    edge = np.floor(np.cumsum(n) * (case["rows"] / n.sum()) + 0.5).astype(np.int64)
    edge[-1] = case["rows"]
    return np.diff(np.concatenate([[0], np.minimum(edge, case["rows"])]))


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    op, dt = case["op"], DTYPES[case["dtype"]]
    s = {"case": case, "op": op}
    if op in ("loss", "loss_train"):
        n, d, v = case["rows"], case["channels"], case["vocab"]
        weight = normal(v, d) * (2 / math.sqrt(d))  # logits of a deviation of two, the right token's six higher
        targets = torch.randint(0, v, (n,), generator=g, device="cuda")
        hidden = normal(n, d) + 1.5 * weight[targets]
        ignored = torch.rand(n, generator=g, device="cuda") < 0.1  # prompt tokens, which are not trained on
        ignored[0] = False
        s["weight"], s["hidden"] = weight.to(dt), hidden.to(dt)
        s["targets"] = torch.where(ignored, -1, targets).to(torch.int32)
        s["grad_loss"] = (1 / (~ignored).sum()).float().expand(n).contiguous()  # of the mean
    else:
        rows, h, hk, dk, dv = (case[n] for n in ("rows", "heads", "key_heads", "key_dim", "value_dim"))
        q, k = normal(rows, hk, dk), normal(rows, hk, dk)
        s["q"], s["k"] = ((t / t.norm(dim=2, keepdim=True)).to(dt) for t in (q, k))
        s["v"] = normal(rows, h, dv).to(dt)
        # memories from a few tokens to some hundreds across the heads
        s["decay"] = torch.nn.functional.logsigmoid(normal(rows, h) + torch.linspace(1.0, 6.0, h, device="cuda"))
        s["beta"] = torch.sigmoid(normal(rows, h))
        if op == "step":
            s["states"] = normal(rows, h, dv, dk) * 0.3
            first = torch.arange(rows, device="cuda") // case["beams"] * case["beams"]
            s["parents"] = (first + torch.randint(0, case["beams"], (rows,), generator=g, device="cuda")).to(torch.int32)
        else:
            seqs = case["seqs"]
            s["init"] = normal(seqs, h, dv, dk) * 0.3
            s["lengths"] = _lengths(case, seed)
            s["start"] = np.cumsum(s["lengths"]) - s["lengths"]
            if case["packed"]:
                s["offsets"] = torch.from_numpy(np.append(s["start"], rows).astype(np.int32)).cuda()
            if op == "train":
                s["grad_out"] = (normal(rows, h, dv) / math.sqrt(dv)).to(dt)
                s["grad_last"] = normal(seqs, h, dv, dk) / math.sqrt(dv * dk)
            _plan_chunks(s)
    if own:
        _prepare_own(s)
    return s


def _plan_chunks(s):
    """For the plain form: the rows of each chunk (the row after the last is zeros), chunks of a sequence in a row,
    longest sequences first; and the chunks that are done together."""
    rows, lengths, start = s["case"]["rows"], s["lengths"], s["start"]
    order = np.argsort(-lengths, kind="stable")
    counts = -(-lengths[order] // CHUNK)
    first = np.cumsum(counts) - counts
    seq = np.repeat(order, counts)
    at = start[seq] + (np.arange(counts.sum()) - np.repeat(first, counts)) * CHUNK
    index = at[:, None] + np.arange(CHUNK)
    index = np.where(index < (start + lengths)[seq][:, None], index, rows)
    s["index"], s["order"] = torch.from_numpy(index).cuda(), torch.from_numpy(order.copy()).cuda()
    live = [int((counts > c).sum()) for c in range(int(counts[0]))]
    s["first"], s["live"] = torch.from_numpy(first).cuda(), live


# ---- plain forms -------------------------------------------------------------------------------
def _chunked(t, s):
    """(chunks, heads, CHUNK, ...) of a tensor (rows, heads, ...), float32, zeros past a sequence's end."""
    t = torch.cat([t.float(), torch.zeros_like(t[:1], dtype=torch.float32)])
    return t[s["index"]].transpose(1, 2).contiguous()


def _rows(t, s):
    """The inverse of _chunked."""
    t = t.transpose(1, 2)
    out = torch.zeros((s["case"]["rows"] + 1, *t.shape[2:]), device="cuda")
    out[s["index"].reshape(-1)] = t.reshape(-1, *t.shape[2:])
    return out[:-1]


def _unit_lower_inverse(m):
    """(I + m)^-1 of strictly lower triangular matrices, row after row."""
    inv = torch.eye(CHUNK, device="cuda").expand_as(m).contiguous()
    for i in range(1, CHUNK):
        inv[..., i, :i] = -(m[..., i:i + 1, :i] @ inv[..., :i, :i]).squeeze(-2)
    return inv


def _plain_delta(s):
    """The delta rule by chunks: within one, tokens act on one another through the inverse of a triangular matrix."""
    case = s["case"]
    group, scale, dt = case["heads"] // case["key_heads"], case["key_dim"] ** -0.5, s["v"].dtype
    q, k, v = (_chunked(s[n], s) for n in ("q", "k", "v"))
    q, k = (t.repeat_interleave(group, 1) for t in (q * scale, k))
    beta = _chunked(s["beta"], s).unsqueeze(-1)
    total = torch.cumsum(_chunked(s["decay"], s).double(), 2)  # 64 bits: differences of long sums
    lower = torch.ones(CHUNK, CHUNK, dtype=torch.bool, device="cuda").tril()
    gap = (total.unsqueeze(-1) - total.unsqueeze(-2)).float()
    decay = torch.where(lower, torch.exp(gap), torch.zeros_like(gap))
    near = decay * (k @ k.transpose(-1, -2))
    near = near.tril(-1)
    read = decay * (q @ k.transpose(-1, -2))
    since = torch.exp(total.float()).unsqueeze(-1)  # from the chunk's start
    until = torch.exp((total[..., -1:] - total).float()).unsqueeze(-1)  # to its end
    whole = since[..., -1:, :]
    inverse = _unit_lower_inverse(near * beta.transpose(-1, -2))
    out, w, before = torch.empty_like(v), torch.empty_like(v), []
    state = s["init"].transpose(-1, -2)[s["order"]].contiguous()  # (sequences, heads, key_dim, value_dim)
    for c, n in enumerate(s["live"]):
        i = s["first"][:n] + c
        kc, old = k[i], state[:n].clone()
        w[i] = inverse[i] @ (v[i] - since[i] * (kc @ old))
        u = beta[i] * w[i]
        out[i] = since[i] * (q[i] @ old) + read[i] @ u
        state[:n] = whole[i] * old + (until[i] * kc).transpose(-1, -2) @ u
        before.append(old)
    last = torch.empty_like(state)
    last[s["order"]] = state
    got = {"out": _rows(out, s).to(dt), "last": last.transpose(-1, -2).contiguous()}
    if s["op"] == "forward":
        return got
    # backward: `tail` is the gradient of the state after the chunk, z that of the values before their strength
    grad_out = _chunked(s["grad_out"], s)
    inverse = _unit_lower_inverse(near * beta)
    dq, dwrite, derase, z = torch.empty_like(q), torch.empty_like(k), torch.empty_like(k), torch.empty_like(v)
    dtotal = torch.empty_like(total, dtype=torch.float32)
    tail = s["grad_last"].transpose(-1, -2)[s["order"]].contiguous()
    for c in range(len(s["live"]) - 1, -1, -1):
        n = s["live"][c]
        i = s["first"][:n] + c
        x, old, kc, qc, go = tail[:n].clone(), before[c], k[i], q[i], grad_out[i]
        du = read[i].transpose(-1, -2) @ go + until[i] * (kc @ x)
        z[i] = inverse[i].transpose(-1, -2) @ du
        y, u = beta[i] * z[i], beta[i] * w[i]
        dread = decay[i] * (go @ u.transpose(-1, -2))
        dnear = -(decay[i] * (y @ u.transpose(-1, -2))).tril(-1)
        oldt = old.transpose(-1, -2)
        dq[i] = since[i] * (go @ oldt) + dread @ kc
        derase[i] = dnear @ kc - since[i] * (y @ oldt)
        carry = until[i] * (u @ x.transpose(-1, -2))
        dwrite[i] = carry + dread.transpose(-1, -2) @ qc + dnear.transpose(-1, -2) @ kc
        d = (qc * dq[i] + kc * (derase[i] - dwrite[i])).sum(-1)
        d[..., -1] += (kc * carry).sum((-1, -2)) + (whole[i] * old * x).sum((-1, -2))
        dtotal[i] = d
        tail[:n] = whole[i] * x + (since[i] * qc).transpose(-1, -2) @ go - (since[i] * kc).transpose(-1, -2) @ y
    ddecay = dtotal.flip(2).cumsum(2).flip(2)

    def shared(t):  # heads of one key head
        return _rows(t.reshape(t.shape[0], -1, group, *t.shape[2:]).sum(2), s).to(dt)

    dinit = torch.empty_like(tail)
    dinit[s["order"]] = tail
    got.update(grad_q=shared(dq * scale), grad_k=shared(derase + dwrite), grad_v=_rows(beta * z, s).to(dt),
               grad_decay=_rows(ddecay, s), grad_beta=_rows((w * z).sum(-1), s),
               grad_init=dinit.transpose(-1, -2).contiguous())
    return got


def _plain_step(s):
    group = s["case"]["heads"] // s["case"]["key_heads"]
    q, k = (s[n].float().repeat_interleave(group, 1).unsqueeze(-1) for n in ("q", "k"))
    old = torch.exp(s["decay"])[..., None, None] * s["states"][s["parents"].long()]
    u = s["beta"][..., None, None] * (s["v"].float().unsqueeze(-1) - old @ k)
    new = old + u @ k.transpose(-1, -2)
    return {"states": new, "out": ((new @ q).squeeze(-1) * s["case"]["key_dim"] ** -0.5).to(s["v"].dtype)}


def _plain_loss(s):
    """Pieces of the rows, each with all its logits."""
    n, v = s["case"]["rows"], s["case"]["vocab"]
    hidden, weight, dt = s["hidden"].float(), s["weight"].float(), s["weight"].dtype
    valid = s["targets"] >= 0
    target = s["targets"].long().clamp(min=0)
    loss, logsum = torch.empty(n, device="cuda"), torch.empty(n, device="cuda")
    train = s["op"] == "loss_train"
    if train:
        grad_hidden, grad_weight = torch.empty_like(hidden), torch.zeros_like(weight)
    piece = max(1, (1 << 29) // v)
    for i in range(0, n, piece):
        r = slice(i, i + piece)
        z = hidden[r] @ weight.t()
        top = z.amax(1, keepdim=True)
        total = (top + torch.log(torch.exp(z - top).sum(1, keepdim=True)))
        right = z.gather(1, target[r, None])
        loss[r] = torch.where(valid[r], (total - right).squeeze(1), torch.zeros_like(loss[r]))
        logsum[r] = torch.where(valid[r], total.squeeze(1), torch.zeros_like(loss[r]))
        if train:
            p = torch.exp(z - total)
            p.scatter_add_(1, target[r, None], torch.full_like(right, -1.0))
            p *= torch.where(valid[r], s["grad_loss"][r], torch.zeros_like(loss[r]))[:, None]
            grad_hidden[r] = p @ weight
            grad_weight += p.t() @ hidden[r]
    got = {"loss": loss, "logsum": logsum}
    if train:
        got.update(grad_hidden=grad_hidden.to(dt), grad_weight=grad_weight.to(dt))
    return got


def _plain(s):
    if s["op"] in ("forward", "train"):
        return _plain_delta(s)
    return _plain_step(s) if s["op"] == "step" else _plain_loss(s)


# ---- through the framework ---------------------------------------------------------------------
def _prepare_own(s):
    """The buffers, temp storage and modules that a program keeps from call to call."""
    import lc_parallel_primitive_b200 as P

    case, op = s["case"], s["op"]
    s["stream"], s["cmdlist"] = P.Stream(), P.CommandList()
    if op in ("loss", "loss_train"):
        s["module"] = P.DeviceCrossEntropy()
        s["module"].create()
        s["temp"] = P.temp_buffer(s["module"].GetTempStorageBytes(
            case["rows"], case["channels"], case["vocab"], s["weight"].dtype, backward=op == "loss_train"))
        s["loss"], s["logsum"] = (torch.empty(case["rows"], device="cuda") for _ in range(2))
        if op == "loss_train":
            s["grad_hidden"], s["grad_weight"] = torch.empty_like(s["hidden"]), torch.empty_like(s["weight"])
        return
    s["module"] = P.DeviceDeltaRule()
    s["module"].create()
    s["out"] = torch.empty_like(s["v"])
    if op == "step":
        s["new"] = torch.empty_like(s["states"])
        return
    s["sequences"] = s["offsets"] if case["packed"] else case["rows"] // case["seqs"]
    sizes = (case["rows"], case["seqs"], case["heads"], case["key_heads"], case["key_dim"], case["value_dim"])
    s["temp"] = P.temp_buffer(s["module"].GetTempStorageBytes(*sizes, s["v"].dtype, backward=op == "train"))
    s["last"] = torch.empty_like(s["init"])
    if op == "train":
        s["saved"] = P.temp_buffer(s["module"].GetSavedStateBytes(*sizes))
        for n in ("q", "k", "v", "decay", "beta", "init"):
            s["grad_" + n] = torch.empty_like(s[n])


def _own(s):
    op, m, c = s["op"], s["module"], s["cmdlist"]
    if op in ("loss", "loss_train"):
        m.Forward(c, s["temp"], s["hidden"], s["weight"], s["targets"], s["loss"], d_logsum=s["logsum"])
        got = {"loss": s["loss"], "logsum": s["logsum"]}
        if op == "loss_train":
            m.Backward(c, s["temp"], s["hidden"], s["weight"], s["targets"], s["logsum"], s["grad_loss"],
                       s["grad_hidden"], s["grad_weight"])
            got.update(grad_hidden=s["grad_hidden"], grad_weight=s["grad_weight"])
    elif op == "step":
        m.Step(c, s["q"], s["k"], s["v"], s["decay"], s["beta"], s["states"], s["new"], s["out"], d_parents=s["parents"])
        got = {"states": s["new"], "out": s["out"]}
    else:
        m.Forward(c, s["temp"], s["q"], s["k"], s["v"], s["decay"], s["beta"], s["out"], s["sequences"],
                  d_init=s["init"], d_last=s["last"], d_saved=s.get("saved"))
        got = {"out": s["out"], "last": s["last"]}
        if op == "train":
            m.Backward(c, s["temp"], s["q"], s["k"], s["v"], s["decay"], s["beta"], s["saved"], s["grad_out"],
                       s["grad_q"], s["grad_k"], s["grad_v"], s["grad_decay"], s["grad_beta"], s["sequences"],
                       d_init=s["init"], d_grad_last=s["grad_last"], d_grad_init=s["grad_init"])
            got.update({n: s[n] for n in ("grad_q", "grad_k", "grad_v", "grad_decay", "grad_beta", "grad_init")})
    s["stream"] << c.commit()
    return got


def run(state):
    return _own(state) if own else _plain(state)


# ---- from the definition, in 64 bits -----------------------------------------------------------
def exact(case, seed):
    if case["op"] in ("forward", "train"):
        # a few launches a token: forward some 60 us, with backward some 300; and its arithmetic
        tokens = case["rows"] if case["seqs"] == 1 else case["rows"] // case["seqs"] * (8 if case["packed"] else 1)
        state = case["heads"] * case["key_dim"] * case["value_dim"]
        seconds = tokens * (6e-5 if case["op"] == "forward" else 3e-4)
        if seconds + case["rows"] * state * (1.2e-11 if case["op"] == "forward" else 8e-11) > 15:
            return None
    s = prepare(case, seed)
    with torch.no_grad():
        if case["op"] in ("forward", "train"):
            return _exact_delta(s)
        if case["op"] == "step":
            got, out = _exact_token(s, torch.arange(case["rows"], device="cuda"), s["states"].double()[s["parents"].long()])
            return {"states": got, "out": out}
        return _exact_loss(s)


def _exact_inputs(s, r):
    """q, k, v, decay factor, beta of the rows r, a key head's for each of its value heads."""
    group = s["case"]["heads"] // s["case"]["key_heads"]
    q, k = (s[n][r].double().unsqueeze(2).expand(-1, -1, group, -1).flatten(1, 2) for n in ("q", "k"))
    return q / math.sqrt(s["case"]["key_dim"]), k, s["v"][r].double(), s["decay"][r].double().exp(), s["beta"][r].double()


def _exact_token(s, r, state):
    """(new state, output) of one token for each row of r; state (rows, heads, value_dim, key_dim)."""
    q, k, v, a, b = _exact_inputs(s, r)
    state = state * a[:, :, None, None]
    u = b[:, :, None] * (v - torch.einsum("nhvk,nhk->nhv", state, k))
    state = state + torch.einsum("nhv,nhk->nhvk", u, k)
    return state, torch.einsum("nhvk,nhk->nhv", state, q)


def _exact_delta(s):
    """One token after the other, all sequences that are long enough at once."""
    train, case = s["op"] == "train", s["case"]
    order = np.argsort(-s["lengths"], kind="stable")
    counts, start = s["lengths"][order], torch.from_numpy(s["start"][order].copy()).cuda()
    order = torch.from_numpy(order.copy()).cuda()
    back = torch.argsort(order)
    live = [int(np.searchsorted(-counts, -t, side="left")) for t in range(int(counts[0]))]  # sequences with count > t
    state = s["init"].double()[order]
    out = torch.zeros(s["v"].shape, dtype=torch.float64, device="cuda")
    span = max(1, min(128, int(4e9 / (8 * max(1, state.numel())))))  # tokens between two kept states
    kept = []
    for t, n in enumerate(live):
        if train and t % span == 0:
            kept.append(state.clone())
        new, out[start[:n] + t] = _exact_token(s, start[:n] + t, state[:n])
        state[:n] = new
    got = {"out": out, "last": state[back]}
    if not train:
        return got
    grad = {n: torch.zeros(s[n].shape, dtype=torch.float64, device="cuda") for n in ("q", "k", "v", "decay", "beta")}
    go, scale = s["grad_out"].double(), 1 / math.sqrt(case["key_dim"])
    d = s["grad_last"].double()[order]  # of the state
    for block in range(len(kept) - 1, -1, -1):
        t0, t1 = block * span, min(len(live), (block + 1) * span)
        states = [kept[block][:live[t0]]]  # before token t0, t0 + 1, ...
        for t in range(t0, t1 - 1):
            n = live[t]
            states.append(_exact_token(s, start[:n] + t, states[-1][:n])[0])
        for t in range(t1 - 1, t0 - 1, -1):
            n = live[t]
            r = start[:n] + t
            q, k, v, a, b = _exact_inputs(s, r)
            before = states.pop()[:n]
            faded = before * a[:, :, None, None]
            miss = v - torch.einsum("nhvk,nhk->nhv", faded, k)
            u = b[:, :, None] * miss
            new = faded + torch.einsum("nhv,nhk->nhvk", u, k)
            dout = go[r]
            dq = torch.einsum("nhvk,nhv->nhk", new, dout)
            dnew = d[:n] + torch.einsum("nhv,nhk->nhvk", dout, q)
            du = torch.einsum("nhvk,nhk->nhv", dnew, k)
            dmiss = b[:, :, None] * du
            dk = torch.einsum("nhvk,nhv->nhk", dnew, u) - torch.einsum("nhvk,nhv->nhk", faded, dmiss)
            dfaded = dnew - torch.einsum("nhv,nhk->nhvk", dmiss, k)
            shape = (n, case["key_heads"], -1, case["key_dim"])
            grad["q"][r], grad["k"][r] = scale * dq.reshape(shape).sum(2), dk.reshape(shape).sum(2)
            grad["v"][r], grad["beta"][r] = dmiss, (du * miss).sum(2)
            grad["decay"][r] = (dfaded * faded).sum((2, 3))
            d[:n] = dfaded * a[:, :, None, None]
    got.update({"grad_" + n: v for n, v in grad.items()})
    got["grad_init"] = d[back]
    return got


def _exact_loss(s):
    """Pieces of the vocabulary, each with all rows: first the sums, then the gradients."""
    n, v = s["case"]["rows"], s["case"]["vocab"]
    keep = (s["targets"] >= 0).nonzero().squeeze(1)
    hidden, target = s["hidden"].double()[keep], s["targets"][keep].long()
    step = max(1, (1 << 28) // n)
    logsum = torch.full((len(keep),), -math.inf, dtype=torch.float64, device="cuda")
    for i in range(0, v, step):
        z = hidden @ s["weight"][i:i + step].double().t()
        logsum = torch.logaddexp(logsum, torch.logsumexp(z, 1))
    right = torch.einsum("nd,nd->n", hidden, s["weight"][target].double())

    def spread(t):
        full = torch.zeros((n, *t.shape[1:]), dtype=torch.float64, device="cuda")
        full[keep] = t
        return full

    got = {"loss": spread(logsum - right), "logsum": spread(logsum)}
    if s["op"] == "loss":
        return got
    gain = s["grad_loss"].double()[keep, None]
    dh = -gain * s["weight"][target].double()
    dw = torch.zeros(s["weight"].shape, dtype=torch.float64, device="cuda").index_add_(0, target, -gain * hidden)
    for i in range(0, v, step):
        w = s["weight"][i:i + step].double()
        p = gain * torch.exp(hidden @ w.t() - logsum[:, None])
        dh += p @ w
        dw[i:i + step] += p.t() @ hidden
    got.update(grad_hidden=spread(dh), grad_weight=dw)
    return got
