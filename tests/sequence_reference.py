"""Plain float64 forms of the sequence operators, row after row, with error
bounds for a float32 implementation of any summation order.

Bounds.  u = 2^-24.  With M_t = |a_t| M_{t-1} + |b_t| (all terms taken
positive) every product and sum of the recurrence, in whatever grouping, is at
most M_t, and an error made at one row reaches later rows through the same
products.  One row contributes the rounding of its product and sum, of the
grouping's product of gates and sum, and the gate's own error: 6u, and for the
sigmoid gate 4u (2-ulp exp2) + 2u (exponent's rounding per unit of |g|) |g| + 4u
(reciprocal, products).  So E_t = |a_t| E_{t-1} + k_t M_t with k_t that sum.
"""
import numpy as np

U = 2.0 ** -24
#: half an ulp, relative, of the element types (float32's own rounding is part of the bounds' terms)
HALF_ULP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
TINY = {"f32": 1e-37, "f16": 2.0 ** -24, "bf16": 1e-37}


def sigmoid(g):
    with np.errstate(over="ignore"):
        return 1.0 / (1.0 + np.exp(-g))


def _coefficients(gate, x, mode):
    if mode == "linear":
        return gate, x, np.ones_like(gate), np.full_like(gate, 6 * U)
    a, na = sigmoid(gate), sigmoid(-gate)
    return a, na * x, na, (14 + 2 * np.minimum(np.abs(gate), 100)) * U


def recurrence(gate, x, offsets, init, mode):
    """{"out", "last"} and their bounds {"out_err", "last_err"}; also what backward() needs."""
    gate, x = gate.astype(np.float64), x.astype(np.float64)
    rows, d = gate.shape
    S = len(offsets) - 1
    init = np.zeros((S, d)) if init is None else init.astype(np.float64)
    a, b, na, k = _coefficients(gate, x, mode)
    out, err, mag = np.zeros((rows, d)), np.zeros((rows, d)), np.zeros((rows, d))
    before, before_err = np.zeros((rows, d)), np.zeros((rows, d))
    last, last_err = init.copy(), np.zeros((S, d))
    for s in range(S):
        h, m, e = init[s], np.abs(init[s]), np.zeros(d)
        for r in range(offsets[s], offsets[s + 1]):
            before[r], before_err[r] = h, e
            h = a[r] * h + b[r]
            m = np.abs(a[r]) * m + np.abs(b[r])
            e = np.abs(a[r]) * e + k[r] * m
            out[r], err[r], mag[r] = h, e, m
        last[s], last_err[s] = h, e
    return {"out": out, "last": last, "out_err": err, "last_err": last_err, "a": a, "na": na, "k": k, "x": x,
            "before": before, "before_err": before_err, "offsets": offsets, "mode": mode}


def backward(f, grad_out, grad_last):
    """Gradients and bounds from recurrence()'s result."""
    rows, d = f["out"].shape
    S = len(f["offsets"]) - 1
    a, na, k, x, before = f["a"], f["na"], f["k"], f["x"], f["before"]
    go = np.zeros((rows, d)) if grad_out is None else grad_out.astype(np.float64)
    gl = np.zeros((S, d)) if grad_last is None else grad_last.astype(np.float64)
    out = {n: np.zeros((rows, d)) for n in ("grad_gate", "grad_in", "grad_gate_err", "grad_in_err")}
    out["grad_init"], out["grad_init_err"] = gl.copy(), np.zeros((S, d))
    for s in range(S):
        mu, m, e = gl[s], np.abs(gl[s]), np.zeros(d)
        for r in reversed(range(f["offsets"][s], f["offsets"][s + 1])):
            lam, lm = go[r] + mu, np.abs(go[r]) + m
            le = e + 2 * U * lm
            if f["mode"] == "linear":
                w, we, scale = before[r], f["before_err"][r], 1.0
                out["grad_in"][r], out["grad_in_err"][r] = lam, le
            else:
                scale = a[r] * na[r]
                w = before[r] - x[r]
                we = f["before_err"][r] + 2 * U * (np.abs(before[r]) + np.abs(x[r]))
                out["grad_in"][r] = na[r] * lam
                out["grad_in_err"][r] = na[r] * (le + 2 * k[r] * lm)
            out["grad_gate"][r] = lam * w * scale
            out["grad_gate_err"][r] = scale * (le * (np.abs(w) + we) + lm * we + 3 * k[r] * lm * np.abs(w))
            mu, m = a[r] * lam, np.abs(a[r]) * lm
            e = np.abs(a[r]) * le + k[r] * m
        out["grad_init"][s], out["grad_init_err"][s] = mu, e
    return out


def assert_within(got, want, err, dtype="f32", what=""):
    """|got - want| <= err + half an ulp of the element type."""
    got = got.astype(np.float64)
    tol = err + HALF_ULP[dtype] * (np.abs(want) + err) + TINY[dtype]
    off = np.abs(got - want)
    bad = ~(off <= tol)
    if bad.any():
        at = np.unravel_index(np.argmax(np.where(bad, off / tol, 0)), got.shape)
        raise AssertionError(f"{what}: {int(bad.sum())} of {got.size} values out of bounds; worst at {at}: "
                             f"got {got[at]!r} want {want[at]!r} bound {tol[at]!r}")


def beam_select(logits, scores, finished, eos):
    """(scores, tokens, parents, finished) of the selection, in float64, and for each entry the smallest gap
    between two scores that decided something (how near another order is)."""
    batches, beams = scores.shape
    z = logits.astype(np.float64).reshape(batches, beams, -1)
    V = z.shape[2]
    out_s, out_t = np.full((batches, beams), -np.inf), np.full((batches, beams), max(eos, 0), np.int32)
    out_p, out_f = np.zeros((batches, beams), np.int32), np.ones((batches, beams), np.uint8)
    gap = np.full(batches, np.inf)
    for b in range(batches):
        cand = []  # (-score, beam, place, token)
        for k in range(beams):
            sc = float(scores[b, k])
            if not sc > -np.inf:
                continue
            if finished is not None and finished[b, k]:
                cand.append((-sc, k, 0, max(eos, 0)))
                continue
            row = np.where(np.isnan(z[b, k]), -np.inf, z[b, k]) + 0.0
            m = row.max()
            if m == -np.inf:
                continue
            with np.errstate(invalid="ignore"):
                rel = np.where(row == m, 0.0, row - m)
                logp = rel - np.log(np.exp(rel).sum())
            order = np.lexsort((np.arange(V), -row))[:beams]
            cand += [(-(sc + logp[v]), k, j, int(v)) for j, v in enumerate(order) if sc + logp[v] > -np.inf]
        cand.sort()
        for j in range(beams):
            out_p[b, j] = b * beams + j
            if j < len(cand):
                s, k, _, v = cand[j]
                out_s[b, j], out_t[b, j], out_p[b, j] = -s, v, b * beams + k
                out_f[b, j] = (finished is not None and finished[b, k] != 0) or v == eos
        for p, q in zip(cand[:beams], cand[1:beams + 1]):
            if p[1] != q[1]:
                gap[b] = min(gap[b], q[0] - p[0])
    return out_s, out_t, out_p, out_f, gap
