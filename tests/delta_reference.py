"""The gated delta rule token by token in float64 (numpy), its gradients, and error bounds for a chunked float32
implementation.

Per sequence, head and value dimension the state is a vector s with s_t = a (s - b k (k.s)) + b v k (s of the token before).
For |k|^2 b <= 2 and a <= 1 that map is a contraction, so an error made at a token does not grow.  Let X be the largest
|s| of a sequence, V the largest |v|; then every quantity of a chunk that belongs to the value dimension (k.s, v - k.s, w,
u, and the products of rows of the triangular inverse, whose entries are at most 1 for unit keys) is at most V + X =: M.

One chunk makes: r from a product over 128 key columns, w from one over 64 tokens with entries of the inverse, which is
itself two products over 64 entries, s from one over 64 tokens; every term is off by at most 2^-21 of itself (2^-22 left
out of a product of float16 pairs, the parts' roundings 2^-23 each, a float32 sum 2^-24 a step).  Taken as independent, the
roundings of a product of n terms add to sqrt(n): (sqrt(128) + sqrt(64) sqrt(64) + sqrt(64)) 2^-21 M < 84 * 2^-21 M = 4e-5 M
a chunk, sqrt(chunks) of that for a sequence.  out = scale q.s has it times scale |q|; the backward pass is the same
recurrence backwards over x = grad s with y = scale dO q: the largest |x| and |y| give its own M'.  Products of the two
sides over value dimensions or tokens add the squares: see bounds().

bf16 outputs (8 bits) are made from one float16 part (11 bits, off by 2^-12 of a value at most) of the state, of u and of
the scores A: the state's term is off by 2^-12 sum_d |q_d s_d| <= 2^-12 |q| M, and the chunk's sum over up to 64 tokens of
A_ij u_j, with |A_ij| <= |q| and |u_j| <= M (times scale all), by twice 2^-12 |q| M a term, sqrt(64) of that for
independent roundings: (1 + 2 sqrt(64)) 2^-12 = 17 * 2^-12 of scale |q| M together.
"""
import numpy as np

UNIT = 84 * 2.0 ** -21
HALF_ULP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
SMALLEST = {"f32": 1e-37, "f16": 2.0 ** -24, "bf16": 1e-37}


class Result:
    pass


def forward(q, k, v, decay, beta, offsets, init, scale):
    """q, k: (rows, key_heads, dk); v: (rows, heads, dv); decay (or None), beta: (rows, heads); init: (S, heads, dv, dk)
    or None; all float64."""
    rows, heads, dv = v.shape
    dk, group, S = q.shape[2], heads // q.shape[1], len(offsets) - 1
    r = Result()
    r.q, r.k = np.repeat(q, group, 1), np.repeat(k, group, 1)
    r.v, r.beta, r.scale, r.offsets, r.group = v, beta, scale, offsets, group
    r.a = np.ones((rows, heads)) if decay is None else np.exp(decay)
    r.out, r.last = np.zeros((rows, heads, dv)), np.zeros((S, heads, dv, dk))
    r.before = np.zeros((rows, heads, dv, dk))  # the state before each token
    r.most = np.zeros((S, heads, dv))           # M
    for s in range(S):
        state = np.zeros((heads, dv, dk)) if init is None else init[s].copy()
        top = np.linalg.norm(state, axis=2)
        for t in range(offsets[s], offsets[s + 1]):
            r.before[t] = state
            state = state * r.a[t][:, None, None]
            miss = v[t] - np.einsum("hvk,hk->hv", state, r.k[t])
            state = state + np.einsum("hv,hk->hvk", r.beta[t][:, None] * miss, r.k[t])
            r.out[t] = scale * np.einsum("hvk,hk->hv", state, r.q[t])
            top = np.maximum(top, np.linalg.norm(state, axis=2))
        r.last[s] = state
        part = v[offsets[s]:offsets[s + 1]]
        r.most[s] = top + (np.abs(part).max(0) if len(part) else 0)
    return r


def backward(r, grad_out, grad_last):
    rows, heads, dv = r.v.shape
    dk, S = r.q.shape[2], len(r.offsets) - 1
    g = Result()
    dq, dk_ = np.zeros((rows, heads, dk)), np.zeros((rows, heads, dk))
    g.v, g.beta, g.decay = np.zeros((rows, heads, dv)), np.zeros((rows, heads)), np.zeros((rows, heads))
    g.init, g.most = np.zeros((S, heads, dv, dk)), np.zeros((S, heads, dv))
    for s in range(S):
        x = np.zeros((heads, dv, dk)) if grad_last is None else grad_last[s].copy()
        top = np.linalg.norm(x, axis=2)
        for t in range(r.offsets[s + 1] - 1, r.offsets[s] - 1, -1):
            go = np.zeros((heads, dv)) if grad_out is None else grad_out[t]
            faded = r.before[t] * r.a[t][:, None, None]
            miss = r.v[t] - np.einsum("hvk,hk->hv", faded, r.k[t])
            u = r.beta[t][:, None] * miss
            state = faded + np.einsum("hv,hk->hvk", u, r.k[t])
            dq[t] = r.scale * np.einsum("hvk,hv->hk", state, go)
            x = x + r.scale * np.einsum("hv,hk->hvk", go, r.q[t])
            du = np.einsum("hvk,hk->hv", x, r.k[t])
            g.beta[t] = (du * miss).sum(1)
            y = r.beta[t][:, None] * du
            g.v[t] = y
            dk_[t] = np.einsum("hvk,hv->hk", x, u) - np.einsum("hvk,hv->hk", faded, y)
            x = x - np.einsum("hv,hk->hvk", y, r.k[t])
            g.decay[t] = (x * faded).sum((1, 2))
            x = x * r.a[t][:, None, None]
            top = np.maximum(top, np.linalg.norm(x, axis=2))
        g.init[s] = x
        part = np.zeros((1, heads, dv)) if grad_out is None else grad_out[r.offsets[s]:r.offsets[s + 1]]
        q = np.linalg.norm(r.q[r.offsets[s]:r.offsets[s + 1]], axis=2).max(initial=0)
        g.most[s] = top + abs(r.scale) * (np.abs(part).max(0) * q if len(part) else 0)
    shape = (rows, heads // r.group, r.group, dk)
    g.q, g.k = dq.reshape(shape).sum(2), dk_.reshape(shape).sum(2)
    return g


def bounds(r, g=None, dtype="f32"):
    """Absolute error bounds (before the output's rounding) of every output, by rows or sequences."""
    rows, heads, dv = r.v.shape
    S, out = len(r.offsets) - 1, Result()
    out.out, out.last = np.zeros(r.out.shape), np.zeros(r.last.shape)
    for n in ("q", "k", "v", "beta", "decay"):
        setattr(out, n, np.zeros((rows, heads, 1) if n in ("q", "k", "v") else (rows, heads)))
    out.init = np.zeros(r.last.shape)
    if g is not None:
        out.v = np.zeros((rows, heads, dv))
    for s in range(S):
        a, b = r.offsets[s], r.offsets[s + 1]
        unit = UNIT * np.sqrt(max(1, -(-(b - a) // 64)))
        out.last[s] = unit * r.most[s][:, :, None]
        if b > a:
            q = np.linalg.norm(r.q[a:b], axis=2).max()
            out.out[a:b] = (unit + (17 * 2.0 ** -12 if dtype == "bf16" else 0)) * abs(r.scale) * q * r.most[s]
        if g is None:
            continue
        out.init[s] = unit * g.most[s][:, :, None]
        if b == a:
            continue
        out.v[a:b] = unit * g.most[s]
        both = np.sqrt(((r.most[s] * g.most[s]) ** 2).sum(1))  # of w z, u x, y s, and scale dO s
        out.beta[a:b] = 2 * unit * both
        out.q[a:b], out.k[a:b] = 2 * unit * both[:, None], 4 * unit * both[:, None]
        # up to 64 rows' products of q, k with their gradients, and products with both states
        out.decay[a:b] = (np.sqrt(64) * 6 + 4) * unit * both
    if g is not None:
        shape = (rows, heads // r.group, r.group, 1)
        out.q, out.k = out.q.reshape(shape).sum(2), out.k.reshape(shape).sum(2)
    return out


def assert_within(got, want, err, dtype, what):
    tol = err + HALF_ULP[dtype] * (np.abs(want) + err) + SMALLEST[dtype]
    off = np.abs(got.astype(np.float64) - want)
    bad = ~(off <= tol)
    if bad.any():
        at = np.unravel_index(np.argmax(np.where(bad, off / tol, 0)), off.shape)
        raise AssertionError(f"{what}: {int(bad.sum())} of {off.size} values out of bounds; worst at {at}: got {got[at]!r} "
                             f"want {want[at]!r} bound {np.broadcast_to(tol, off.shape)[at]!r}")
