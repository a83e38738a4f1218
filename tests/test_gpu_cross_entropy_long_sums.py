"""GPU: gradients whose sums run over a great many words or tokens and nearly cancel.

At most 1024 additions of 16 products follow one another in the tensor core, off by 2^-22 of the magnitudes each; the rest is FP32: 2^-14
covers it and the sums of the rounded probabilities."""

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


@pytest.mark.parametrize("tokens", [20_000, 400_000])
def test_hidden_states_that_have_a_sign_in_common(tokens):
    """A head of zeros gives each of 64 words the same share, which BF16 holds, and words are targets as often as that: what the hidden
    states have in common nearly cancels between the product and the tokens of the word, whose sum is FP32."""
    from hyper_multicore_b200 import mega_cross_entropy

    g = torch.Generator().manual_seed(1)
    x = (torch.rand(tokens, 64, generator=g) + 0.5).bfloat16().cuda()
    weight = torch.zeros(64, 64).bfloat16().cuda().requires_grad_(True)
    targets = (torch.randperm(tokens, generator=g) % 64).cuda()
    (grad_w,) = torch.autograd.grad(mega_cross_entropy(x, weight, targets, reduction="sum", recompute=True), weight)
    total = x.double().sum(0)
    own = torch.zeros(64, 64, dtype=torch.float64, device="cuda").index_add_(0, targets, x.double())
    exact, size = total / 64 - own, total / 64 + own
    bound = SUMS * size + 2.0 ** -8 * exact.abs()
    assert ((grad_w.double() - exact).abs() <= bound).all(), ((grad_w.double() - exact).abs() / size).max()
