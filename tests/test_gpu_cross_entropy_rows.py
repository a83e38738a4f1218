"""GPU: rows of the hidden states' gradient where its terms nearly cancel or one of them holds almost everything.

A row is sum_{j != t} p_j (w_j - w_t). A probability reaches the product off by D = 2^-8 (BF16) + half a step of a kept logit +
2 E + 2^-19 (E and the last as in the cross entropy's other tests), but the row is scaled to the known sum 1 - p_t of what it was made of, and the
target's row enters with that sum: with q_j = p_j / (1 - p_t) and d_j the error of p_j, what is left is
(1 - p_t) sum_j q_j (d_j - d) (w_j - m) / (1 + d), d = sum_j q_j d_j, for any vector m, since the weights q_j (d_j - d) add up to nothing.
With m the row of the likeliest wrong word it is at most 2 D / (1 - D) sum_{j != t} p_j |w_j - m|: nothing where that word holds all, and
free of what the words' rows have in common. On top come the sums: of products, V / 16 additions off by 2^-22 of the magnitudes each;
of the rounded probabilities and in the epilogue, fewer than 128 FP32 additions (2^-17 of the magnitudes covers them); of 1 - p_t, the loss's
2 E + 2^-20 (1 + |lse|) times p_t; and the row's own rounding, 2^-8 of each value."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

HALF = 2.0 ** -8
KEPT = math.log(2) * 2.0 ** -11


def make(tokens, hidden, vocab, shared, lead, seed):
    """Rows of the weight with a component in common `shared` times their own size, tokens that favour a wrong word."""
    g = torch.Generator().manual_seed(seed)
    own = torch.randn(vocab, hidden, generator=g) * hidden ** -0.5
    weight = (own + shared * torch.randn(hidden, generator=g) * hidden ** -0.5).bfloat16()
    targets = torch.randint(0, vocab, (tokens,), generator=g)
    wrong = (targets + torch.randint(1, vocab, (tokens,), generator=g)) % vocab
    x = (lead * own[wrong] + 0.3 * torch.randn(tokens, hidden, generator=g)).bfloat16()
    return x.cuda(), weight.cuda(), targets.cuda()


def check_rows(grad_x, x, weight, targets, rows, kept):
    w = weight.double()
    for i in rows:
        t = targets[i].item()
        logits = w @ x[i].double()
        error = x.shape[1] / 16 * 2.0 ** -22 * (w.abs() @ x[i].double().abs()).max()
        lse = torch.logsumexp(logits, 0)
        p = torch.exp(logits - lse)
        p_target = p[t].item()
        p[t] = 0
        rest = p.sum()
        exact = p @ w - rest * w[t]
        main = w[p.argmax()]
        off = HALF + kept + 2 * error + 2.0 ** -19
        size = p @ w.abs() + rest * w[t].abs()
        bound = (2 * off / (1 - off) * (p @ (w - main).abs()) + (len(w) / 16 * 2.0 ** -22 + 2.0 ** -17) * size
                 + (2 * error + 2.0 ** -20 * (1 + lse.abs())) * p_target / rest * exact.abs() + HALF * exact.abs() + 1e-38)
        far = ((grad_x[i].double() - exact).abs() / bound).max().item()
        assert far <= 1, f"row {i}: {far:.2f} of its bound, {((grad_x[i].double() - exact).norm() / exact.norm()).item():.4f} of its norm"


@pytest.mark.parametrize("recompute", [False, True])
@pytest.mark.parametrize("tokens", [100, 300])
@pytest.mark.parametrize("shared", [0.0, 4.0, 10.0])
@pytest.mark.parametrize("lead", [8.0, 16.0])
def test_common_component_and_a_wrong_word_that_leads(lead, shared, tokens, recompute):
    from hyper_multicore_b200 import mega_cross_entropy

    x, weight, targets = make(tokens, 256, 1000, shared, lead, seed=int(lead + shared) + tokens)
    x.requires_grad_(True)
    grad = (torch.rand(tokens, device="cuda") + 0.5) * torch.randint(0, 2, (tokens,), device="cuda").mul(2).sub(1)
    kept = KEPT if tokens > 128 and not recompute else 0.0
    for reduction, dy in (("none", grad), ("sum", torch.ones((), device="cuda"))):
        loss = mega_cross_entropy(x, weight, targets, reduction=reduction, recompute=recompute)
        (grad_x,) = torch.autograd.grad(loss, x, dy)
        by = dy.double().view(-1, 1) if reduction == "none" else 1.0
        check_rows(grad_x.double() / by, x.detach(), weight, targets, range(tokens), kept)


@pytest.mark.parametrize("recompute", [False, True])
def test_sum_over_pieces_of_the_vocabulary(recompute):
    """4096 tokens of 70001 words: two pieces, whose sums add up."""
    from hyper_multicore_b200 import mega_cross_entropy

    x, weight, targets = make(4096, 64, 70001, 6.0, 10.0, seed=3)
    targets[::7] = -100
    x.requires_grad_(True)
    (grad_x,) = torch.autograd.grad(mega_cross_entropy(x, weight, targets, reduction="sum", recompute=recompute), x)
    rows = [i for i in range(0, 4096, 61) if i % 7]
    check_rows(grad_x, x.detach(), weight, targets, rows, 0.0 if recompute else KEPT)
    assert torch.equal(grad_x[::7], torch.zeros_like(grad_x[::7]))


@pytest.mark.parametrize("recompute", [False, True])
def test_words_that_are_all_alike(recompute):
    """A head of zeros: every p is 1 / V, which BF16 rounds the same way for all words."""
    from hyper_multicore_b200 import mega_cross_entropy

    vocab = 259  # 1 / 259 is 1.4 steps above a power of two: BF16 is off by 0.3 % of it
    g = torch.Generator().manual_seed(4)
    weight = torch.zeros(vocab, 64)
    weight[:, 8:] = torch.randn(vocab, 56, generator=g)
    x = torch.zeros(200, 64)
    x[:, :8] = torch.randn(200, 8, generator=g)
    weight, x = weight.bfloat16().cuda(), x.bfloat16().cuda().requires_grad_(True)
    targets = torch.randint(0, vocab, (200,), generator=g).cuda()
    (grad_x,) = torch.autograd.grad(mega_cross_entropy(x, weight, targets, reduction="sum", recompute=recompute), x)
    exact = weight.double().mean(0) - weight[targets].double()
    # all errors alike cancel: the sums' and the row's own rounding are left
    bound = HALF * exact.abs() + 2.0 ** -16 * (weight.double().abs().mean(0) + weight[targets].double().abs())
    assert ((grad_x.double() - exact).abs() <= bound).all()


def test_rows_without_a_wrong_word():
    """One word, a gradient of zero, and tokens so certain that no other word has a share: nothing divides by nothing."""
    from hyper_multicore_b200 import mega_cross_entropy

    x, weight, targets = make(200, 64, 300, 0.0, 0.0, seed=5)
    x.requires_grad_(True)
    for head, words, recompute in ((weight[:1], torch.zeros_like(targets), False), (weight, targets, True), (weight, targets, False)):
        for dy in (torch.zeros(200, device="cuda"), torch.ones(200, device="cuda")):
            (grad_x,) = torch.autograd.grad(mega_cross_entropy(x, head, words, reduction="none", recompute=recompute), x, dy)
            assert grad_x.isfinite().all()
            if head is not weight or not dy.any():
                assert torch.equal(grad_x, torch.zeros_like(grad_x))
    with torch.no_grad():
        certain = weight[targets].mul(4000).requires_grad_(True)  # other words are exp(-1000) and less
    for recompute in (False, True):
        (grad_x,) = torch.autograd.grad(mega_cross_entropy(certain, weight, targets, reduction="sum", recompute=recompute), certain)
        assert grad_x.isfinite().all()
