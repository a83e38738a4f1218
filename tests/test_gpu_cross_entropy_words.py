"""GPU: rows of the weight's gradient where one token holds almost all of a word, or where its terms nearly cancel.

A row is sum_{i: t_i != j} g_i p_ij x_i + sum_{i: t_i = j} g_i (p_ij - 1) x_i. The second sum is FP32; in the first a probability is off
by D = 2^-8 (BF16) + half a step of a kept logit + 2 E + 2^-19 (E as in the cross entropy's other tests), of which the BF16 part is scaled away as
a whole: the sum of |g_i| p_ij over the tokens is what it was before the rounding, up to R = 2^-14 (its correction, below 2^-8, is
held in BF16). As for a row of the hidden states' gradient, what is left is 2 D / (1 - D) sum_i |g_i| p_ij |s_i x_i - s_m x_m| for any
token m, s the gradient's signs: nothing where m holds all of the word or all x_i are alike, but for the errors that the scaling does not see,
kept + 2 E + 2^-19 + R of the sum. On top come the sums, T / 16 additions off by 2^-22 of the magnitudes and fewer than 256 in FP32 (2^-16),
and the row's own rounding."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

HALF = 2.0 ** -8
KEPT = math.log(2) * 2.0 ** -11


def check_words(grad_w, x, weight, targets, grad, words, kept):
    x64, w64 = x.double(), weight.double()
    logits = x64 @ w64.t()
    error = x.shape[1] / 16 * 2.0 ** -22 * (x64.abs() @ w64.abs().t()).max()
    p = torch.exp(logits - torch.logsumexp(logits, 1, keepdim=True))
    wrong = p.scatter(1, targets.unsqueeze(1), 0.0).sum(1)  # 1 - p of the target, also where that has no digits in 64 bits
    unseen = kept + 2 * error + 2.0 ** -19
    off = HALF + unseen
    for j in words:
        own = targets == j
        share = torch.where(own, 0.0, grad.double().abs() * p[:, j])
        signed = x64 * grad.double().sign().unsqueeze(1)
        target = torch.where(own, -grad.double() * wrong, 0.0)
        exact = share @ signed + target @ x64
        main = signed[share.argmax()]
        size = share @ x64.abs() + target.abs() @ x64.abs()
        bound = (2 * off / (1 - off) * (share @ (signed - main).abs()) + (unseen + 2.0 ** -14) * (share @ signed).abs()
                 + (len(x) / 16 * 2.0 ** -22 + 2.0 ** -16 + 2 * error + 2.0 ** -19) * size + HALF * exact.abs() + 1e-38)
        far = ((grad_w[j].double() - exact).abs() / bound).max().item()
        assert far <= 1, f"word {j}: {far:.2f} of its bound, {((grad_w[j].double() - exact).norm() / exact.norm()).item():.4f} of its norm"


def gradient(x, weight, targets, grad, recompute):
    from hyper_multicore_b200 import mega_cross_entropy

    weight = weight.detach().requires_grad_(True)
    loss = mega_cross_entropy(x, weight, targets, reduction="none", recompute=recompute)
    return torch.autograd.grad(loss, weight, grad)[0]


@pytest.mark.parametrize("recompute", [False, True])
@pytest.mark.parametrize("tokens,lead", [(100, 8.0), (300, 8.0), (300, 16.0), (700, 12.0)])
def test_words_that_one_token_takes_for_its_own(tokens, lead, recompute):
    """Every token favours a wrong word that no other token has to do with."""
    vocab, hidden = 2 * tokens, 256
    g = torch.Generator().manual_seed(tokens)
    own = torch.randn(vocab, hidden, generator=g) * hidden ** -0.5
    x = (lead * own[tokens:] + 0.3 * torch.randn(tokens, hidden, generator=g)).bfloat16().cuda()
    weight, targets = own.bfloat16().cuda(), torch.randint(0, tokens, (tokens,), generator=g).cuda()
    grad = (torch.rand(tokens, generator=g) + 0.5) * (torch.randint(0, 2, (tokens,), generator=g) * 2 - 1)
    grad = grad.cuda()
    got = gradient(x, weight, targets, grad, recompute)
    check_words(got, x, weight, targets, grad, range(0, vocab, 3), KEPT if tokens > 128 and not recompute else 0.0)


@pytest.mark.parametrize("recompute", [False, True])
@pytest.mark.parametrize("tokens,vocab", [(128, 40), (2000, 60), (3000, 300), (8000, 20000)])
def test_words_that_all_tokens_rate_alike(tokens, vocab, recompute):
    """A model that knows how frequent the words are and nothing else: what the tokens hold in common almost cancels."""
    g = torch.Generator().manual_seed(vocab)
    weight = torch.randn(vocab, 64, generator=g) * 0.2
    weight[:, 8:] = 0
    x = torch.randn(tokens, 64, generator=g)
    x[:, :8] = torch.randn(8, generator=g) * 2
    x, weight = x.bfloat16(), weight.bfloat16()
    p = torch.softmax(x[0].double() @ weight.double().t(), 0)
    targets = torch.multinomial(p, tokens, replacement=True, generator=g).cuda()
    x, weight, grad = x.cuda(), weight.cuda(), torch.ones(tokens).cuda()
    got = gradient(x, weight, targets, grad, recompute)
    check_words(got, x, weight, targets, grad, range(0, vocab, 1 + vocab // 300), KEPT if tokens > 128 and not recompute else 0.0)


@pytest.mark.parametrize("recompute", [False, True])
def test_tokens_left_out_and_gradients_of_zero(recompute):
    """Words that no token with a gradient rates, and a number of tokens that counts inside a block of 32."""
    g = torch.Generator().manual_seed(9)
    weight, x = torch.randn(500, 72, generator=g).mul_(0.1).bfloat16().cuda(), torch.randn(333, 72, generator=g).bfloat16().cuda()
    targets = torch.randint(0, 500, (333,), generator=g).cuda()
    grad = torch.rand(333, generator=g).cuda()
    grad[::3] = 0
    left_out = torch.arange(333, device="cuda") % 4 == 1
    got = gradient(x, weight, torch.where(left_out, -100, targets), grad, recompute)
    keep = ~left_out
    check_words(got, x[keep], weight, targets[keep], grad[keep], range(500), 0.0 if recompute else KEPT)
    nothing = gradient(x, weight, targets, torch.zeros_like(grad), recompute)
    assert torch.equal(nothing, torch.zeros_like(nothing))
