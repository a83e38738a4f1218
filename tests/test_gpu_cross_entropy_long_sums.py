"""GPU: gradients whose sums run over a great many words or tokens and nearly cancel.

At most 1024 additions of 16 products follow one another in the tensor core, off by 2^-22 of the magnitudes each; the rest is FP32: 2^-14
covers it, the sums of the rounded probabilities and (for the weight) their correction, which is held in BF16."""

import pytest
import torch

pytestmark = pytest.mark.gpu

SUMS = 1024 * 2.0 ** -22 + 2.0 ** -14


@pytest.mark.parametrize("recompute", [False, True])
def test_two_million_words_that_are_all_alike(recompute):
    """All rows of the weight are one and the same: nothing is left of a row of the hidden states' gradient."""
    from hyper_multicore_b200 import mega_cross_entropy

    tokens, vocab = 130, 2_000_000
    g = torch.Generator().manual_seed(0)
    row = (torch.rand(1, 16, generator=g) + 0.5).bfloat16().cuda()
    weight = row.expand(vocab, 16).contiguous()
    x = (0.3 * torch.randn(tokens, 16, generator=g)).bfloat16().cuda().requires_grad_(True)
    targets = torch.randint(0, vocab, (tokens,), generator=g).cuda()
    (grad_x,) = torch.autograd.grad(mega_cross_entropy(x, weight, targets, reduction="sum", recompute=recompute), x)
    assert (grad_x.double().abs() <= SUMS * row.double()).all(), (grad_x.double().abs() / row.double()).max()


@pytest.mark.parametrize("tokens", [20_000, 140_000])
def test_tokens_that_are_all_alike(tokens):
    """Every token has the same hidden state, and words are targets about as often as it predicts."""
    from hyper_multicore_b200 import mega_cross_entropy

    g = torch.Generator().manual_seed(1)
    row = (torch.rand(1, 64, generator=g) + 0.5).bfloat16().cuda()
    weight = (0.1 * torch.randn(40, 64, generator=g)).bfloat16().cuda().requires_grad_(True)
    p = torch.softmax(row.double() @ weight.detach().double().t(), 1)[0]
    counts = (p * tokens).round().long()
    counts[0] += tokens - counts.sum()
    targets = torch.repeat_interleave(torch.arange(40, device="cuda"), counts)[torch.randperm(tokens, generator=g).cuda()]
    x = row.expand(tokens, 64).contiguous()
    (grad_w,) = torch.autograd.grad(mega_cross_entropy(x, weight, targets, reduction="sum", recompute=True), weight)
    exact = (p * tokens - counts).unsqueeze(1) * row.double()
    size = (p * tokens).unsqueeze(1) * row.double()
    # the logits' own errors, as in the cross entropy's other tests: the same for every token here
    error = 64 / 16 * 2.0 ** -22 * (row.double().abs() @ weight.detach().double().abs().t()).max()
    bound = (SUMS + 2 * error + 2.0 ** -19) * 2 * size + 2.0 ** -8 * exact.abs()
    assert ((grad_w.double() - exact).abs() <= bound).all(), ((grad_w.double() - exact).abs() / size).max()
