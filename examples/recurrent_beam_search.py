"""A small gated recurrent language model on the package's sequence operators.

Trained with DeviceLinearRecurrence.Forward / Backward on packed sequences of
different lengths, then decoded with beam search: each token is one Step (whose
parents reorder the recurrent states on the way), one Select and one Reorder of
the beams' token histories.  The data is synthetic: digits that count up by a
step of their own, so that two tokens tell how a sequence goes on.

    python examples/recurrent_beam_search.py [--steps 200]
"""
from __future__ import annotations

import argparse
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))
import lc_parallel_primitive_b200 as lcpp  # noqa: E402

VOCAB, START, END = 12, 10, 11  # ten digits, start and end of a sequence


class Recurrence(torch.autograd.Function):
    """h_t = a_t h_{t-1} + (1 - a_t) x_t over packed rows, a = sigmoid(gate)."""

    @staticmethod
    def forward(ctx, gate, x, offsets):
        module, cmdlist = lcpp.DeviceLinearRecurrence(), lcpp.CommandList()
        module.create()
        rows, channels = gate.shape
        temp = lcpp.temp_buffer(module.GetTempStorageBytes(rows, channels))
        saved = lcpp.temp_buffer(module.GetSavedStateBytes(rows, channels))
        out = torch.empty_like(x)
        module.Forward(cmdlist, temp, gate, x, out, offsets, d_saved=saved)
        lcpp.Stream() << cmdlist.commit()
        ctx.save_for_backward(gate, x, offsets, saved)
        ctx.module, ctx.temp = module, temp
        return out

    @staticmethod
    def backward(ctx, grad_out):
        gate, x, offsets, saved = ctx.saved_tensors
        cmdlist = lcpp.CommandList()
        grad_gate, grad_x = torch.empty_like(gate), torch.empty_like(x)
        ctx.module.Backward(cmdlist, ctx.temp, gate, x, saved, grad_out.contiguous(), grad_gate, grad_x, offsets)
        lcpp.Stream() << cmdlist.commit()
        return grad_gate, grad_x, None


class Model(torch.nn.Module):
    def __init__(self, channels=128, layers=2):
        super().__init__()
        self.channels, self.layers = channels, layers
        self.embed = torch.nn.Embedding(VOCAB, channels)
        self.project = torch.nn.ModuleList(torch.nn.Linear(channels, 2 * channels) for _ in range(layers))
        self.mix = torch.nn.ModuleList(torch.nn.Linear(channels, channels) for _ in range(layers))
        self.head = torch.nn.Linear(channels, VOCAB)

    def run(self, tokens, recur):
        """Logits of the rows; recur(layer, gate, x) is the recurrence."""
        y = self.embed(tokens)
        for layer in range(self.layers):
            both = self.project[layer](y)  # gate and input are the halves of one projection, used in place
            h = recur(layer, both[:, :self.channels], both[:, self.channels:])
            y = y + torch.nn.functional.gelu(self.mix[layer](h))
        return self.head(y)

    def forward(self, tokens, offsets):
        return self.run(tokens, lambda layer, gate, x: Recurrence.apply(gate, x, offsets))


def batch(generator, sequences=64):
    """(tokens, targets, offsets) of packed sequences: start, digits, end."""
    rows, offsets = [], [0]
    for _ in range(sequences):
        length, first, step = (int(torch.randint(a, b, (1,), generator=generator)) for a, b in ((4, 20), (0, 10), (1, 10)))
        rows.append([START] + [(first + i * step) % 10 for i in range(length)] + [END])
        offsets.append(offsets[-1] + length + 1)
    tokens = torch.tensor([t for r in rows for t in r[:-1]], device="cuda")
    targets = torch.tensor([t for r in rows for t in r[1:]], device="cuda")
    return tokens, targets, torch.tensor(offsets, dtype=torch.int32, device="cuda")


def train(model, steps, seed=0):
    generator = torch.Generator().manual_seed(seed)
    optimizer = torch.optim.Adam(model.parameters(), lr=3e-3)
    losses = []
    for _ in range(steps):
        tokens, targets, offsets = batch(generator)
        loss = torch.nn.functional.cross_entropy(model(tokens, offsets), targets)
        optimizer.zero_grad()
        loss.backward()
        optimizer.step()
        losses.append(float(loss.detach()))
    return losses


@torch.no_grad()
def beam_search(model, prompts, beams=4, length=12):
    """(sequences, scores): the best continuations of equally long prompts (batch, time), (batch, beams, ...)."""
    recurrence, search = lcpp.DeviceLinearRecurrence(), lcpp.DeviceBeamSearch()
    recurrence.create()
    search.create()
    cmdlist, stream = lcpp.CommandList(), lcpp.Stream()
    batches, time = prompts.shape
    rows, channels, layers = batches * beams, model.channels, model.layers

    # the prompts in one pass, which leaves each layer's states
    prompt_states = torch.empty((layers, batches, channels), device="cuda")

    def prefill(layer, gate, x):
        out = torch.empty_like(x)
        temp = lcpp.temp_buffer(recurrence.GetTempStorageBytes(*gate.shape))
        recurrence.Forward(cmdlist, temp, gate, x, out, time, d_last=prompt_states[layer])
        stream << cmdlist.commit()
        return out

    logits = model.run(prompts.reshape(-1), prefill)[time - 1::time].repeat_interleave(beams, 0)
    states = prompt_states.repeat_interleave(beams, 1).contiguous()
    states_next = torch.empty_like(states)
    scores = torch.full((batches, beams), float("-inf"), device="cuda")
    scores[:, 0] = 0  # all beams are still alike: one of them goes on
    finished = torch.zeros((batches, beams), dtype=torch.uint8, device="cuda")
    history = torch.full((rows, length), END, dtype=torch.int32, device="cuda")
    history_next = torch.empty_like(history)
    scores_next, finished_next = torch.empty_like(scores), torch.empty_like(finished)
    tokens, parents = (torch.empty((batches, beams), dtype=torch.int32, device="cuda") for _ in range(2))
    temp = lcpp.temp_buffer(search.GetTempStorageBytes(batches, beams, VOCAB))
    for t in range(length):
        search.Select(cmdlist, temp, logits, scores, finished, scores_next, tokens, parents, finished_next, eos_token=END)
        search.Reorder(cmdlist, history, history_next, parents)
        stream << cmdlist.commit()
        scores, scores_next, finished, finished_next = scores_next, scores, finished_next, finished
        history, history_next = history_next, history
        history[:, t] = tokens.reshape(-1)

        def step(layer, gate, x):
            out = torch.empty_like(x)
            recurrence.Step(cmdlist, gate, x, states[layer], states_next[layer], out, d_parents=parents.reshape(-1))
            stream << cmdlist.commit()
            return out

        logits = model.run(tokens.reshape(-1).long(), step)
        states, states_next = states_next, states
    return history.reshape(batches, beams, length), scores


def main():
    parser = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    parser.add_argument("--steps", type=int, default=300)
    args = parser.parse_args()
    torch.manual_seed(0)
    model = Model().cuda()
    losses = train(model, args.steps)
    print(f"loss {losses[0]:.3f} -> {losses[-1]:.3f} in {args.steps} steps")
    prompts = torch.tensor([[START, 1, 3], [START, 9, 8], [START, 2, 7]], device="cuda")
    sequences, scores = beam_search(model, prompts)
    for prompt, beams, score in zip(prompts.tolist(), sequences.tolist(), scores.tolist()):
        print("prompt", prompt[1:])
        for tokens, s in zip(beams, score):
            print(f"  {s:8.3f}  {[t for t in tokens if t != END]}")


if __name__ == "__main__":
    main()
