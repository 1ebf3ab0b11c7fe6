"""The example's model: its gradients and its beam search against plain torch."""
import importlib.util
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu
PATH = Path(__file__).resolve().parent.parent / "examples" / "recurrent_beam_search.py"


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("recurrent_beam_search", PATH)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def plain_recurrence(offsets):
    import torch

    def recur(layer, gate, x):
        a = torch.sigmoid(gate)
        out = []
        for s in range(len(offsets) - 1):
            h = torch.zeros_like(x[0])
            for r in range(offsets[s], offsets[s + 1]):
                h = a[r] * h + (1 - a[r]) * x[r]
                out.append(h)
        return torch.stack(out)

    return recur


def test_gradients(cuda, example):
    import torch

    torch.manual_seed(1)
    model = example.Model(channels=24, layers=2).cuda()
    tokens, targets, offsets = example.batch(torch.Generator().manual_seed(2), sequences=5)
    loss = torch.nn.functional.cross_entropy(model(tokens, offsets), targets)
    loss.backward()
    got = [p.grad.double() for p in model.parameters()]
    wide = example.Model(channels=24, layers=2).cuda().double()
    wide.load_state_dict(model.state_dict())
    want = torch.nn.functional.cross_entropy(wide.run(tokens, plain_recurrence(offsets.tolist())), targets)
    want.backward()
    # float32 products over some hundred terms of a float64 computation of the same
    assert abs(float(loss.detach()) - float(want.detach())) < 1e-5
    for p, q in zip(got, wide.parameters()):
        assert float((p - q.grad).norm()) <= 1e-4 * float(q.grad.norm()) + 1e-7


def test_trains_and_decodes(cuda, example):
    import torch

    torch.manual_seed(3)
    model = example.Model(channels=64).cuda()
    losses = example.train(model, 60, seed=4)
    assert losses[-1] < 0.75 * losses[0]
    prompts = torch.tensor([[example.START, 1, 3], [example.START, 9, 8]], device="cuda")
    sequences, scores = example.beam_search(model, prompts, beams=3, length=5)
    # every hypothesis' score is the model's own log-probability of it
    assert (scores[:, :-1] >= scores[:, 1:]).all()
    for prompt, beams, score in zip(prompts.tolist(), sequences.tolist(), scores.tolist()):
        for tokens, s in zip(beams, score):
            total, at = 0.0, list(prompt)
            for t in tokens:
                with torch.no_grad():
                    logits = model.run(torch.tensor(at, device="cuda"), plain_recurrence([0, len(at)]))[-1].double()
                total += float(torch.log_softmax(logits, 0)[t])
                at.append(t)
                if t == example.END:
                    break
            assert abs(total - s) < 1e-3, (prompt, tokens)
