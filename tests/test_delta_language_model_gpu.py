"""A small language model on the delta rule: its training step through DeviceDeltaRule and DeviceCrossEntropy against torch's
gradients in float64, and its decoding with beams (Step, Select, Reorder) against the whole sequence at once."""
import pytest

from lc_parallel_primitive_b200 import _lib as L

pytestmark = pytest.mark.gpu
VOCAB, WIDTH, HEADS, KEYS, DK, DV = 97, 48, 4, 2, 32, 24
LENGTHS = [70, 0, 3, 130, 64]


def parameters(dtype, seed=0):
    import torch

    g = torch.Generator(device="cuda").manual_seed(seed)
    new = lambda *s: (torch.randn(s, generator=g, device="cuda", dtype=torch.float64) / s[-1] ** 0.5).to(dtype)  # noqa: E731
    return {"embed": new(VOCAB, WIDTH) * 3, "q": new(KEYS * DK, WIDTH), "k": new(KEYS * DK, WIDTH), "v": new(HEADS * DV, WIDTH),
            "gates": new(2 * HEADS, WIDTH), "mix": new(WIDTH, HEADS * DV), "head": new(VOCAB, WIDTH) * 2}


def inputs(p, tokens):
    """(residual, q, k, v, decay, beta) of the layer."""
    import torch

    x = p["embed"][tokens]
    unit = lambda t: t / (t * t).sum(-1, keepdim=True).sqrt()  # noqa: E731
    q, k = (unit((x @ p[n].t()).unflatten(-1, (KEYS, DK))) for n in "qk")
    gates = x @ p["gates"].t()
    return (x, q, k, (x @ p["v"].t()).unflatten(-1, (HEADS, DV)), torch.nn.functional.logsigmoid(gates[..., :HEADS] + 3),
            torch.sigmoid(gates[..., HEADS:]))


def plain_layer(q, k, v, decay, beta, offsets):
    """Token by token, differentiable; (outputs, last states)."""
    import torch

    q, k = (t.repeat_interleave(HEADS // KEYS, 1) for t in (q, k))
    outs, last = [], []
    for a, b in zip(offsets, offsets[1:]):
        state = torch.zeros(HEADS, DV, DK, dtype=v.dtype, device="cuda")
        for t in range(a, b):
            state = state * decay[t].exp()[:, None, None]
            u = beta[t][:, None] * (v[t] - (state @ k[t][:, :, None]).squeeze(-1))
            state = state + u[:, :, None] * k[t][:, None, :]
            outs.append((state @ q[t][:, :, None]).squeeze(-1) * DK ** -0.5)
        last.append(state)
    return torch.stack(outs), torch.stack(last)


def layer(offsets):
    import torch
    import lc_parallel_primitive_b200 as P

    class Layer(torch.autograd.Function):
        @staticmethod
        def forward(ctx, q, k, v, decay, beta):
            m, c = P.DeviceDeltaRule(), P.CommandList()
            m.create()
            sizes = (len(q), offsets.numel() - 1, HEADS, KEYS, DK, DV)
            temp, saved = P.temp_buffer(m.GetTempStorageBytes(*sizes, v.dtype)), P.temp_buffer(m.GetSavedStateBytes(*sizes))
            out = torch.empty_like(v)
            m.Forward(c, temp, q, k, v, decay, beta, out, offsets, d_saved=saved)
            P.Stream() << c.commit()
            ctx.save_for_backward(q, k, v, decay, beta, saved)
            ctx.m, ctx.temp = m, temp
            return out

        @staticmethod
        def backward(ctx, grad):
            q, k, v, decay, beta, saved = ctx.saved_tensors
            c, got = P.CommandList(), [torch.empty_like(t) for t in (q, k, v, decay, beta)]
            ctx.m.Backward(c, ctx.temp, q, k, v, decay, beta, saved, grad.contiguous(), *got, offsets)
            P.Stream() << c.commit()
            return tuple(got)

    return Layer.apply


def loss_of(hidden, weight, targets):
    """Mean over the rows that take part."""
    import torch
    import lc_parallel_primitive_b200 as P

    class Loss(torch.autograd.Function):
        @staticmethod
        def forward(ctx, hidden, weight):
            m, c = P.DeviceCrossEntropy(), P.CommandList()
            m.create()
            temp = P.temp_buffer(m.GetTempStorageBytes(*hidden.shape, len(weight), weight.dtype))
            loss, logsum = (torch.empty(len(hidden), device="cuda") for _ in range(2))
            m.Forward(c, temp, hidden, weight, targets, loss, logsum)
            P.Stream() << c.commit()
            ctx.save_for_backward(hidden, weight, logsum)
            ctx.m, ctx.temp = m, temp
            return loss.sum() / (targets >= 0).sum()

        @staticmethod
        def backward(ctx, grad):
            hidden, weight, logsum = ctx.saved_tensors
            c, gh, gw = P.CommandList(), torch.empty_like(hidden), torch.empty_like(weight)
            one = (grad / (targets >= 0).sum()).float().reshape(1).expand(len(hidden))
            ctx.m.Backward(c, ctx.temp, hidden, weight, targets, logsum, one, gh, gw)
            P.Stream() << c.commit()
            return gh, gw

    return Loss.apply(hidden, weight)


@pytest.mark.parametrize("name,tolerance", [("f32", 2e-5), ("bf16", 0.05)])
def test_training_step(cuda, name, tolerance):
    # float32: 1e-6 an operator, some tens of additions of it; bf16: half an ulp (2^-8) at each of the about ten roundings of
    # the projections, activations and gradients on the way, the operators' among them
    import torch

    dtype = {"f32": torch.float32, "bf16": torch.bfloat16}[name]
    p = {n: t.requires_grad_() for n, t in parameters(dtype).items()}
    ref = {n: t.detach().double().requires_grad_() for n, t in p.items()}
    g = torch.Generator().manual_seed(1)
    rows = sum(LENGTHS)
    offsets = [0]
    for n in LENGTHS:
        offsets.append(offsets[-1] + n)
    tokens = torch.randint(0, VOCAB, (rows,), generator=g).cuda()
    targets = torch.randint(0, VOCAB, (rows,), generator=g).int().cuda()
    targets[::7] = -1
    device_offsets = torch.tensor(offsets, dtype=torch.int32, device="cuda")

    x, q, k, v, decay, beta = inputs(p, tokens)
    out = layer(device_offsets)(q, k, v, decay.float(), beta.float())
    loss = loss_of(x + out.flatten(1) @ p["mix"].t(), p["head"], targets)
    loss.backward()
    torch.cuda.synchronize()

    x, q, k, v, decay, beta = inputs(ref, tokens)
    out, _ = plain_layer(q, k, v, decay, beta, offsets)
    z = (x + out.flatten(1) @ ref["mix"].t()) @ ref["head"].t()
    want = torch.nn.functional.cross_entropy(z, targets.long(), ignore_index=-1)
    want.backward()
    assert abs(float(loss.detach()) - float(want.detach())) <= tolerance * float(want.detach())
    for n in p:
        a, b = p[n].grad.double(), ref[n].grad
        assert float((a - b).norm()) <= tolerance * float(b.norm()), (n, float((a - b).norm() / b.norm()))


def test_decoding_with_beams(cuda):
    import torch
    import lc_parallel_primitive_b200 as P

    p = parameters(torch.float32, seed=3)
    batches, beams, length, steps = 3, 4, 70, 6
    g = torch.Generator().manual_seed(4)
    prompts = torch.randint(0, VOCAB, (batches, length), generator=g).cuda()
    rows = batches * beams
    rule, search, c, s = P.DeviceDeltaRule(), P.DeviceBeamSearch(), P.CommandList(), P.Stream()
    rule.create()
    search.create()

    # the prompts at once
    x, *layer_in = inputs(p, prompts.reshape(-1))
    temp = P.temp_buffer(rule.GetTempStorageBytes(batches * length, batches, HEADS, KEYS, DK, DV, torch.float32, backward=False))
    out, last = torch.empty_like(layer_in[2]), torch.empty(batches, HEADS, DV, DK, device="cuda")
    rule.Forward(c, temp, *layer_in, out, length, d_last=last)
    s << c.commit()
    hidden = (x + out.flatten(1) @ p["mix"].t())[length - 1::length]
    logits = (hidden @ p["head"].t()).repeat_interleave(beams, 0)
    states, states_next = last.repeat_interleave(beams, 0).contiguous(), torch.empty(rows, HEADS, DV, DK, device="cuda")
    scores = torch.full((batches, beams), float("-inf"), device="cuda")
    scores[:, 0] = 0
    scores_next = torch.empty_like(scores)
    tokens, parents = (torch.empty((batches, beams), dtype=torch.int32, device="cuda") for _ in range(2))
    history, history_next = (torch.zeros((rows, steps), dtype=torch.int32, device="cuda") for _ in range(2))
    temp = P.temp_buffer(search.GetTempStorageBytes(batches, beams, VOCAB))
    for t in range(steps):
        search.Select(c, temp, logits, scores, None, scores_next, tokens, parents, None)
        search.Reorder(c, history, history_next, parents)
        s << c.commit()
        scores, scores_next, history, history_next = scores_next, scores, history_next, history
        history[:, t] = tokens.reshape(-1)
        x, *one = inputs(p, tokens.reshape(-1).long())
        out = torch.empty_like(one[2])
        rule.Step(c, *one, states, states_next, out, d_parents=parents.reshape(-1))
        s << c.commit()
        states, states_next = states_next, states
        logits = (x + out.flatten(1) @ p["mix"].t()) @ p["head"].t()
    torch.cuda.synchronize()
    P.check(P.last_device_error())

    # every beam's sequence token by token in float64: its score is the sum of its tokens' log probabilities
    ref = {n: t.double() for n, t in p.items()}
    for r in range(rows):
        line = torch.cat([prompts[r // beams], history[r].long()])
        x, *layer_in = inputs(ref, line)
        out, state = plain_layer(*layer_in, [0, len(line)])
        logp = torch.log_softmax((x + out.flatten(1) @ ref["mix"].t()) @ ref["head"].t(), 1)
        want = logp[length - 1:-1].gather(1, line[length:, None]).sum()
        # six log probabilities of logits that are off by some 1e-5 of their size
        assert abs(float(scores.reshape(-1)[r]) - float(want)) <= 6 * 1e-4, r
        assert float((states[r].double() - state[0]).norm()) <= 1e-5 * float(state.norm()) * 4, r
