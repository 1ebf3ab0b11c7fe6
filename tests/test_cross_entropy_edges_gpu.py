"""DeviceCrossEntropy where a row is sure of its target, and at the ends of its sizes."""
import numpy as np
import pytest

from tests.test_cross_entropy_gpu import DTYPES, U, Case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_that_are_sure(cuda, dtype):
    """Logits of c for the target and 0 for the others (products of one factor, exact): the loss is log(1 + 299 exp(-c)), never
    below 0.  The sum's terms are off by exp2's 2^-22 and what its argument's roundings make of it, 2^-22 c; to the 1 in it
    fewer than 32 are added one after the other, by half an ulp of it (U) each; and its logarithm is off by 2^-22 of itself."""
    import torch

    c = Case(512, 300, 300, dtype, seed=41, ignored=0.0, gain=1.0)
    c.weight.copy_(torch.eye(300, device="cuda"))
    c.hidden.zero_()
    size = torch.linspace(15, 60, 512, device="cuda").to(c.hidden.dtype)
    c.hidden[torch.arange(512, device="cuda"), c.targets.long()] = size
    c.run()
    size = size.double()
    want = torch.log1p(299 * torch.exp(-size))
    assert float(c.loss.min()) >= 0.0
    assert ((c.loss.double() - want).abs() <= 32 * U + (3 + size) * 2.0 ** -22 * want).all()
    # logsum is c where the rest is less than half an ulp of c, and p = 1 then: the target's row of the gradient is 0
    sure = size > 30
    at = c.grad_hidden[torch.arange(512, device="cuda"), c.targets.long()]
    assert (at[sure] == 0).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_losses_are_not_negative(cuda, dtype):
    import torch

    c = Case(2000, 72, 700, dtype, seed=42, ignored=0.0, sharp=8.0, size=3.0)
    c.run(grads="")
    assert float(c.loss.min()) >= 0.0 and (c.loss <= 1e-3).sum() > 100
    assert not torch.isnan(c.loss).any() and np.isfinite(float(c.loss.max()))


@pytest.mark.parametrize("dtype,channels,vocab,rows,more", [("bf16", 256, 5000, 6144, 6400), ("f32", 40, 33000, 2560, 2816)])
def test_a_buffer_for_more_rows(cuda, dtype, channels, vocab, rows, more):
    # these fewer rows take more pieces or splits of their own
    import torch
    from lc_parallel_primitive_b200 import DeviceCrossEntropy, temp_buffer
    from tests.test_cross_entropy_gpu import torch_dtype

    c = Case(rows, channels, vocab, dtype, seed=43)
    want = [t.clone() for t in c.run()]
    got = c.run(temp=temp_buffer(DeviceCrossEntropy.GetTempStorageBytes(more, channels, vocab, torch_dtype(dtype))))
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_float32_sums_over_a_large_vocabulary(cuda):
    # two pieces of the vocabulary, the hidden gradient's sums in parts of 4096 tokens at most
    Case(16, 40, 300001, "f32", seed=44).check()
