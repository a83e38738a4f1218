"""GPU: the cross entropy over a vocabulary and its gradients against the definition in 64 bits.

Tolerances. A logit is a sum of H exact products, added 16 at a time: H / 16 additions in FP32, each off by at most two
steps (2^-22) of the sum of magnitudes S_ij = sum_k |x_ik w_jk|, so E_i = H / 16 * 2^-22 max_j S_ij. A loss is the difference of
two such values and of FP32 logarithms: 2 E_i + 2^-20 (1 + |lse|). A probability carries exp's relative error, 2 E_i + 2^-20,
where its logit was kept half a step of 2^-10 of a power of two (log 2 * 2^-11; nothing is kept up to 128 tokens or with
recompute), and one rounding to BF16, 2^-8; the target's entry p - 1 stays in FP32. So grad_hidden is off by 2^-8 of itself (its own
rounding) and g (sum_j p_j |w_j| (2^-8 + kept + 2 E + 2^-19) + |w_target| (2 E + 2^-19)); grad_weight likewise over the tokens.
A kept logit more than 64 powers of two below the largest of its row's 128 columns counts as none: off by 2^-64 of that p."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

HALF = 2.0 ** -8  # half a step of BF16
KEPT = math.log(2) * 2.0 ** -11  # half a step of a kept logit
IGNORED = -100


def make(tokens, hidden, vocab, *, ignored=0.0, seed=0, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    weight = (torch.randn(vocab, hidden, generator=g) * scale * hidden ** -0.5).bfloat16()
    targets = torch.randint(0, vocab, (tokens,), generator=g)
    sure = torch.rand(tokens, 1, generator=g) * 12  # from lost to certain
    x = (torch.randn(tokens, hidden, generator=g) + sure * weight[targets].float()).bfloat16()
    targets[torch.rand(tokens, generator=g) < ignored] = IGNORED
    return x.cuda(), weight.cuda(), targets.cuda()


def run(x, weight, targets, reduction="mean", grad=None, ignore_index=IGNORED, **options):
    from hyper_multicore_b200 import mega_cross_entropy

    x, weight = x.detach().requires_grad_(True), weight.detach().requires_grad_(True)
    loss = mega_cross_entropy(x, weight, targets, ignore_index=ignore_index, reduction=reduction, **options)
    grad = torch.ones_like(loss) if grad is None else grad
    return (loss.detach(), *torch.autograd.grad(loss, (x, weight), grad))


def check(got, x, weight, targets, reduction="mean", grad=None, ignore_index=IGNORED, recompute=False):
    loss, grad_x, grad_w = got
    x64, w64 = x.double(), weight.double()
    counted = targets != ignore_index
    index = torch.where(counted, targets, 0).long().unsqueeze(1)
    logits = x64 @ w64.t()
    size = (x64.abs() @ w64.abs().t()).amax(1)
    error = x.shape[1] / 16 * 2.0 ** -22 * size
    lse = torch.logsumexp(logits, 1)
    losses = torch.where(counted, lse - logits.gather(1, index).squeeze(1), 0.0)
    loss_error = torch.where(counted, 2 * error + 2.0 ** -20 * (1 + lse.abs()), 0.0)
    n = counted.sum()
    want, bound, per_token = losses, loss_error, torch.ones_like(lse)
    if reduction != "none":
        by = n if reduction == "mean" else 1
        want, bound = losses.sum() / by, (loss_error.sum() + 2.0 ** -18 * losses.abs().sum()) / by
        per_token = per_token / by
    assert loss.dtype == torch.float32 and ((loss.double() - want).abs() <= bound).all(), (loss, want, bound)
    per_token = per_token * (1.0 if grad is None else grad.double()) * counted
    p = torch.exp(logits - lse.unsqueeze(1))
    rel = (2 * error + 2.0 ** -19).unsqueeze(1)
    kept = 0.0 if recompute or x.shape[0] <= 128 else KEPT
    onehot = torch.zeros_like(p).scatter_(1, index, 1.0)
    d = (p - onehot) * per_token.unsqueeze(1)
    slack = (p * (1 - onehot) * (HALF + kept + rel) + onehot * rel + 2.0 ** -64 * (kept > 0)) * per_token.abs().unsqueeze(1)
    for name, out, exact, off in (("grad_hidden", grad_x, d @ w64, slack @ w64.abs()),
                                  ("grad_weight", grad_w, d.t() @ x64, slack.t() @ x64.abs())):
        assert out.dtype == torch.bfloat16
        far = (out.double() - exact).abs() - HALF * exact.abs() - off - 1e-38
        assert far.max().item() <= 0, f"{name}: {far.max().item():.3e} beyond the bound"
        # on the whole a rounding is off by 2^-8 / sqrt(3) of the value or less, and twice that leaves room for p's
        assert (out.double() - exact).norm() <= HALF * exact.norm() + 1e-30, name


SIZES = [(1, 8, 1), (1, 64, 2), (2, 8, 255), (3, 1000, 256), (5, 72, 257), (33, 128, 1000), (64, 64, 64), (255, 64, 513),
         (257, 136, 511), (300, 256, 5003), (129, 1024, 4099), (513, 520, 1031)]


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("tokens,hidden,vocab", SIZES)
def test_loss_and_gradients_match_the_definition(tokens, hidden, vocab, reduction):
    x, weight, targets = make(tokens, hidden, vocab, ignored=0.2 if tokens > 4 else 0.0, seed=tokens + vocab)
    grad = torch.rand(tokens if reduction == "none" else (), device="cuda") + 0.5
    for recompute in (False, True):
        check(run(x, weight, targets, reduction, grad, recompute=recompute), x, weight, targets, reduction, grad, recompute=recompute)


@pytest.mark.parametrize("recompute", [False, True])
@pytest.mark.parametrize("tokens,hidden,vocab", [(4096, 64, 70001), (40, 4096, 20000), (2500, 256, 3000)])
def test_large_sizes_and_pieces_of_the_vocabulary(tokens, hidden, vocab, recompute):
    """The first one's probabilities take two pieces; its weight's gradient has words of both."""
    x, weight, targets = make(tokens, hidden, vocab, ignored=0.1, seed=vocab)
    got = run(x, weight, targets, recompute=recompute)
    check(got, x, weight, targets, recompute=recompute)
    again = run(x, weight, targets, recompute=recompute)
    assert all(torch.equal(a, b) for a, b in zip(got, again)), "the same call twice gives other bits"


def test_words_beyond_what_is_kept_are_computed_again():
    """20000 x 120001 words take more than 4 GiB: the loss is the same, a gradient differs by two roundings of p at most."""
    from hyper_multicore_b200 import kernels as K

    x, weight, targets = make(20_000, 64, 120_001, ignored=0.1, seed=23)
    held = K._size("hmc_vocab_loss_state_bytes", 20_000, 64, 120_001, True) - K._size("hmc_vocab_loss_state_bytes", 20_000, 64, 120_001, False)
    assert 0 < held < 2 * 20_000 * 120_001
    loss, grad_x, grad_w = run(x, weight, targets)
    other, want_x, want_w = run(x, weight, targets, recompute=True)
    assert torch.equal(loss, other)
    # one rounding of each result, and p's of both: at most 2 (2 * 2^-8 + KEPT) of sums of magnitudes, on the whole of their norms
    for got, want in ((grad_x, want_x), (grad_w, want_w)):
        assert not torch.equal(got, want)
        assert (got.double() - want.double()).norm() <= 2 * (2 * HALF + KEPT) * want.double().norm()
    check_rows = slice(19_900, 20_000)
    counted = targets[check_rows] != IGNORED
    p = torch.softmax(x[check_rows].double() @ weight.double().t(), 1)
    p.scatter_add_(1, torch.where(counted, targets[check_rows], 0).unsqueeze(1), torch.full((100, 1), -1.0, dtype=torch.float64, device="cuda"))
    exact = p * counted.unsqueeze(1) / (targets != IGNORED).sum() @ weight.double()
    assert (grad_x[check_rows].double() - exact).norm() <= HALF * exact.norm()


def test_kept_logits_far_below_the_largest():
    """Weights that put most words 100 powers of two below the rest of their 128, among them minus infinity."""
    x, weight, targets = make(300, 64, 1000, seed=24)
    x[:, 0] = 1.0
    weight[::3, 0] = -70.0
    weight[7] = 0.0
    weight[7, 0] = -float("inf")
    targets[targets % 3 == 0] += 1
    targets[targets == 7] = 8
    loss, grad_x, grad_w = run(x, weight, targets, "none")
    other, want_x, want_w = run(x, weight, targets, "none", recompute=True)
    assert torch.equal(loss, other) and loss.isfinite().all()
    assert torch.equal(grad_x.isnan(), want_x.isnan()) and torch.equal(grad_w.isnan(), want_w.isnan())
    kept = grad_w[1::3]
    assert (kept.double() - want_w[1::3].double()).norm() <= 2 * (2 * HALF + KEPT) * kept.double().norm()


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_no_token_counts(reduction):
    x, weight, targets = make(40, 64, 300, seed=1)
    targets.fill_(IGNORED)
    loss, grad_x, grad_w = run(x, weight, targets, reduction)
    assert loss.isnan().item() if reduction == "mean" else torch.equal(loss, torch.zeros_like(loss))
    assert torch.equal(grad_x, torch.zeros_like(grad_x)) and torch.equal(grad_w, torch.zeros_like(grad_w))


def test_only_one_token_counts():
    x, weight, targets = make(700, 64, 300, seed=2)
    targets[:] = IGNORED
    targets[650] = 299
    check(run(x, weight, targets), x, weight, targets)


def test_no_tokens():
    weight = torch.randn(30, 64, device="cuda").bfloat16()
    for reduction in ("mean", "sum", "none"):
        loss, grad_x, grad_w = run(torch.empty(0, 64, device="cuda").bfloat16(), weight, torch.empty(0, device="cuda").long(), reduction)
        assert loss.shape == ((0,) if reduction == "none" else ()) and grad_x.shape == (0, 64)
        assert torch.equal(grad_w, torch.zeros_like(grad_w))
        assert reduction == "none" or loss.isnan().item() == (reduction == "mean")


def test_ignored_tokens_are_not_read():
    """Padding may hold anything: neither the loss nor the weight's gradient sees it."""
    x, weight, targets = make(300, 128, 1000, ignored=0.4, seed=3)
    want = run(x, weight, targets)
    dirty = x.clone()
    dirty[targets == IGNORED] = float("nan")
    dirty[(targets == IGNORED).nonzero()[0]] = float("inf")
    got = run(dirty, weight, targets)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_ignore_index_may_be_a_word_and_targets_int32():
    x, weight, targets = make(200, 64, 50, seed=4)
    got = run(x, weight, targets.int(), ignore_index=7)
    check(got, x, weight, targets, ignore_index=7)
    assert (targets == 7).any()


def test_targets_outside_the_vocabulary_give_nan():
    x, weight, targets = make(20, 64, 50, seed=5)
    targets[3], targets[4] = 50, -1
    loss, grad_x, _ = run(x, weight, targets, "none")
    bad = torch.zeros(20, dtype=torch.bool, device="cuda")
    bad[3:5] = True
    assert torch.equal(loss.isnan(), bad) and torch.equal(grad_x.isnan().all(1), bad)
    assert run(x, weight, targets, "mean")[0].isnan()


def test_all_tokens_have_the_same_target():
    """One word's sum over every token: a chain of FP32 additions in the tokens' order."""
    x, weight, targets = make(1500, 1032, 400, seed=6)
    targets[:] = 123
    check(run(x, weight, targets), x, weight, targets)


def test_tokens_that_are_certain_keep_the_digits_of_their_gradient():
    """p rounds to 1 in BF16 here; p - 1 must not."""
    hidden, vocab = 256, 600
    g = torch.Generator().manual_seed(7)
    weight = torch.randn(vocab, hidden, generator=g).bfloat16() * 0.0625
    targets = torch.randint(0, vocab, (90,), generator=g)
    x = weight[targets] * 12 + (0.01 * torch.randn(90, hidden, generator=g)).bfloat16()
    x, weight, targets = x.cuda(), weight.cuda(), targets.cuda()
    p = torch.softmax(x.double() @ weight.double().t(), 1).gather(1, targets.unsqueeze(1))
    assert (1 - p).median() < 2.0 ** -4
    check(run(x, weight, targets, "none"), x, weight, targets, "none")


def test_large_logits():
    x, weight, targets = make(50, 64, 900, seed=8, scale=1.0)
    x = (x.float() * 40).bfloat16()
    check(run(x, weight, targets, "none"), x, weight, targets, "none")


def test_nan_and_infinite_hidden_states_stay_in_their_token():
    x, weight, targets = make(300, 64, 900, seed=9)
    want = run(x, weight, targets, "none")
    x[11, 3], x[270, 4] = float("nan"), float("inf")
    loss, grad_x, _ = run(x, weight, targets, "none")
    keep = torch.ones(300, dtype=torch.bool, device="cuda")
    keep[[11, 270]] = False
    assert torch.equal(loss[keep], want[0][keep]) and torch.equal(grad_x[keep], want[1][keep])
    assert loss[11].isnan() and loss[270].isnan()


def test_strides_alignment_and_batches():
    x, weight, targets = make(60, 128, 300, seed=10)
    wide = torch.randn(60, 200, device="cuda").bfloat16()
    big = torch.randn(300, 136, device="cuda").bfloat16()
    views = {
        "slice": wide[:, 8:136], "off the vector boundary": wide[:, 3:131], "transposed": x.t().contiguous().t(),
        "every other": wide[:, :128].repeat(2, 1)[::2], "broadcast": x[:1].expand(60, 128)}
    for name, rows in views.items():
        for head in (weight, big[:, :128], big[:, 3:131], weight.t().contiguous().t()):
            check(run(rows, head, targets), rows, head, targets)
    rows = wide[:, :128].reshape(3, 20, 128)
    loss, grad_x, grad_w = run(rows, weight, targets.view(3, 20), "none")
    assert loss.shape == (3, 20) and grad_x.shape == (3, 20, 128)
    check((loss.view(60), grad_x.view(60, 128), grad_w), rows.reshape(60, 128), weight, targets, "none")
    one = run(x[7], weight, targets[7], "none")  # a token without a batch
    assert one[0].shape == () and one[1].shape == (128,)
    check((one[0].view(1), one[1].view(1, 128), one[2]), x[7:8], weight, targets[7:8], "none")
    strided = torch.full((60, 2), IGNORED, device="cuda")
    strided[:, 0] = targets
    check(run(x, weight, strided[:, 0]), x, weight, targets)
    check(run(x, big[5:6, :128], torch.zeros_like(targets)), x, big[5:6, :128], torch.zeros_like(targets))


def test_one_gradient_alone_is_the_same():
    from hyper_multicore_b200 import mega_cross_entropy

    x, weight, targets = make(100, 64, 700, ignored=0.2, seed=11)
    loss, grad_x, grad_w = run(x, weight, targets)
    a = x.detach().requires_grad_(True)
    assert torch.equal(torch.autograd.grad(mega_cross_entropy(a, weight, targets), a)[0], grad_x)
    b = weight.detach().requires_grad_(True)
    assert torch.equal(torch.autograd.grad(mega_cross_entropy(x, b, targets), b)[0], grad_w)
    with torch.no_grad():
        assert torch.equal(mega_cross_entropy(a, b, targets), loss)


def test_gradient_agrees_with_differences_of_the_definition():
    x, weight, targets = make(30, 64, 200, seed=12)
    _, grad_x, grad_w = run(x, weight, targets, "sum")
    g = torch.Generator(device="cuda").manual_seed(3)
    step = 1e-5
    for i, (leaf, grad) in enumerate(((x, grad_x), (weight, grad_w))):
        direction = torch.randn(leaf.shape, generator=g, device="cuda", dtype=torch.float64)

        def value(sign):
            moved = [x.double(), weight.double()]
            moved[i] = moved[i] + sign * step * direction
            return torch.nn.functional.cross_entropy(moved[0] @ moved[1].t(), targets, reduction="sum").item()

        slope = (value(1) - value(-1)) / (2 * step)
        # every value of the gradient is off by 2^-8 of itself and of p's share: three times that over the whole sum
        assert abs((grad.double() * direction).sum().item() - slope) <= 3 * HALF * (grad.double() * direction).abs().sum().item()


def test_other_streams_and_captured_graphs():
    x, weight, targets = make(300, 128, 2000, ignored=0.3, seed=13)
    want = run(x, weight, targets)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = run(x, weight, targets)
    torch.cuda.current_stream().wait_stream(stream)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graphs, outputs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outputs.append(run(x, weight, targets))
        graphs.append(graph)
    other = make(300, 128, 2000, ignored=0.6, seed=14)  # another number of tokens counts, which only the device knows
    for mine, new in zip((x, weight, targets), other):
        mine.copy_(new)
    for graph in graphs:
        graph.replay()
    torch.cuda.synchronize()
    want = run(*other)
    for got in outputs:
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_rows_of_the_output_are_written_and_nothing_else():
    """Gradients that end inside a tile: guard rows behind them keep what they held."""
    from hyper_multicore_b200 import _lib, kernels as K

    x, weight, targets = make(70, 72, 300, ignored=0.2, seed=15)
    _, state = K.vocab_loss(x, weight, targets, ignore_index=IGNORED, reduction="mean")
    need = _lib.load().hmc_vocab_loss_grad_workspace_bytes(70, 72, 300)
    space = torch.full((need + 4096,), 0x5A, dtype=torch.uint8, device="cuda")
    gx, gw = (torch.full((n + 64, 72), 3.0, dtype=torch.bfloat16, device="cuda") for n in (70, 300))
    grad = torch.ones((), device="cuda")
    status = _lib.new_status(x.device)
    _lib.launch("hmc_vocab_loss_grad", x.device, state.data_ptr(), weight.data_ptr(), 72, 70, 72, 300, 1, 0, grad.data_ptr(),
                gx.data_ptr(), gw.data_ptr(), space.data_ptr(), need, status.data_ptr())
    _lib.raise_on_status(status, "gradient")
    _, want_x, want_w = run(x, weight, targets)
    assert torch.equal(gx[:70], want_x) and torch.equal(gw[:300], want_w)
    assert (gx[70:] == 3).all() and (gw[300:] == 3).all() and (space[need:] == 0x5A).all()


@pytest.mark.parametrize("tokens,hidden,vocab", [(70, 4096, 530_000), (530_000, 4096, 200)])
def test_offsets_beyond_31_bits(tokens, hidden, vocab):
    """A weight, and packed rows, of more than 2^31 values: the far end against the definition."""
    g = torch.Generator(device="cuda").manual_seed(1)
    weight = torch.randn(vocab, hidden, generator=g, device="cuda", dtype=torch.bfloat16).mul_(hidden ** -0.5)
    x = torch.randn(1000, hidden, generator=g, device="cuda", dtype=torch.bfloat16).repeat(tokens // 1000 + 1, 1)[:tokens]
    targets = torch.randint(0, vocab, (tokens,), generator=g, device="cuda")
    targets[-1] = vocab - 1
    loss, grad_x, grad_w = run(x, weight, targets, "none")
    rows = slice(max(0, tokens - 300), tokens)
    logits = x[rows].double() @ weight.double().t() if vocab < 1000 else torch.cat(
        [x[rows].double() @ w.double().t() for w in weight.split(65536)], 1)
    p = torch.softmax(logits, 1)
    want = torch.logsumexp(logits, 1) - logits.gather(1, targets[rows].unsqueeze(1)).squeeze(1)
    assert (loss[rows].double() - want).abs().max() <= 2.0 ** -14  # E = 256 * 2^-22 * 64 at the most, twice
    p.scatter_add_(1, targets[rows].unsqueeze(1), torch.full_like(want, -1).unsqueeze(1))
    far = sum(p[:, i:i + 65536] @ weight[i:i + 65536].double() for i in range(0, vocab, 65536))
    assert (grad_x[rows].double() - far).norm() <= HALF * far.norm()
    if tokens < 1000:  # a row of the weight's gradient needs every token
        tail = p[:, -500:].t() @ x.double()
        assert (grad_w[-500:].double() - tail).norm() <= HALF * tail.norm()
    else:
        whole = torch.zeros(vocab, hidden, dtype=torch.float64, device="cuda")
        for at in range(0, tokens, 50_000):
            part = slice(at, min(tokens, at + 50_000))
            q = torch.softmax(x[part].double() @ weight.double().t(), 1)
            q.scatter_add_(1, targets[part].unsqueeze(1), torch.full((q.shape[0], 1), -1.0, dtype=torch.float64, device="cuda"))
            whole += q.t() @ x[part].double()
        assert (grad_w.double() - whole).norm() <= HALF * whole.norm()


def test_calls_from_two_threads_on_two_streams():
    import threading

    cases = [make(300, 128, 2000, ignored=0.2, seed=s) for s in (21, 22)]
    want = [run(*c) for c in cases]
    torch.cuda.synchronize()
    got = [None, None]

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                got[i] = run(*cases[i])
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in (0, 1)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for mine, expected in zip(got, want):
        assert all(torch.equal(a, b) for a, b in zip(mine, expected))


def test_backward_twice_over_one_forward():
    from hyper_multicore_b200 import mega_cross_entropy

    x, weight, targets = make(100, 64, 700, ignored=0.2, seed=23)
    a, b = x.detach().requires_grad_(True), weight.detach().requires_grad_(True)
    loss = mega_cross_entropy(a, b, targets)
    first = torch.autograd.grad(loss, (a, b), retain_graph=True)
    second = torch.autograd.grad(loss, (a, b))
    assert all(torch.equal(p, q) for p, q in zip(first, second))
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss = mega_cross_entropy(a, b, targets)
        with torch.no_grad():
            b.mul_(2)
        torch.autograd.grad(loss, b)


def test_second_derivatives_and_batched_gradients_are_refused():
    from hyper_multicore_b200 import mega_cross_entropy

    x, weight, targets = make(10, 64, 50, seed=16)
    x.requires_grad_(True)
    (first,) = torch.autograd.grad(mega_cross_entropy(x, weight, targets), x, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable|does not require grad"):
        first.sum().backward()
    loss = mega_cross_entropy(x, weight, targets, reduction="none")
    with pytest.raises(RuntimeError, match="batched"):
        torch.autograd.grad(loss, x, torch.ones(3, 10, device="cuda"), is_grads_batched=True)


def test_end_of_a_training_step():
    """Experts, norm, head and loss in a row: the gradients that reach each are those of the pieces on their own."""
    from hyper_multicore_b200 import MegaCrossEntropy, MegaGate, MegaMoeExperts, MegaRmsNorm

    torch.manual_seed(0)
    tokens, hidden, vocab = 192, 256, 1000
    gate = MegaGate(hidden_size=hidden, num_experts=8, top_k=2, scoring_func="softmax", routed_scaling_factor=1.0).cuda()
    experts = MegaMoeExperts(hidden_size=hidden, intermediate_size=256, num_experts=8, top_k=2)
    norm = MegaRmsNorm(hidden, device="cuda")
    head = MegaCrossEntropy(hidden, vocab, device="cuda", initializer_range=0.1)
    w1 = (torch.randn(8, hidden, 512, device="cuda") * 0.05).bfloat16().requires_grad_(True)
    w2 = (torch.randn(8, 256, hidden, device="cuda") * 0.05).bfloat16().requires_grad_(True)
    x = torch.randn(1, tokens, hidden, device="cuda").bfloat16().requires_grad_(True)
    targets = torch.randint(0, vocab, (tokens,), device="cuda")
    targets[::5] = IGNORED
    _, probs, ids = gate(x)
    out = experts(x.view(tokens, hidden), ids, probs, expert_weights=(w1, w2))
    mixed = (x.view(tokens, hidden) + out)
    normed = norm(mixed)
    loss = head(normed, targets)
    loss.backward()
    experts.check_status()
    rows, unit = mixed.detach(), normed.detach()
    check((loss.detach(), run(unit, head.weight, targets)[1], head.weight.grad), unit, head.weight.detach(), targets)
    leaf = rows.clone().requires_grad_(True)
    again = norm(leaf)
    grad_leaf, grad_gain = torch.autograd.grad(again, (leaf, norm.weight), run(unit, head.weight, targets)[1])
    assert torch.equal(again, normed) and torch.equal(grad_gain, norm.weight.grad)
    for tensor in (x, w1, w2, gate.weight, head.weight, norm.weight):
        assert tensor.grad is not None and torch.isfinite(tensor.grad.float()).all() and tensor.grad.float().abs().max() > 0
    assert math.isfinite(loss.item()) and grad_leaf.abs().max() > 0


def test_module_computes_logits_again_where_asked_to():
    from hyper_multicore_b200 import MegaCrossEntropy

    x, weight, targets = make(300, 64, 500, seed=25)
    head = MegaCrossEntropy(64, 500, recompute=True, device="cuda")
    head.weight.data.copy_(weight)
    hidden = x.detach().requires_grad_(True)
    head(hidden, targets).backward()
    _, want_x, want_w = run(x, weight, targets, recompute=True)
    _, kept_x, _ = run(x, weight, targets)
    assert torch.equal(hidden.grad, want_x) and torch.equal(head.weight.grad, want_w) and not torch.equal(want_x, kept_x)


def test_module_shares_the_weight_of_an_existing_head():
    from hyper_multicore_b200 import MegaCrossEntropy

    linear = torch.nn.Linear(64, 300, bias=False, device="cuda", dtype=torch.bfloat16)
    head = MegaCrossEntropy.from_module(linear, reduction="sum")
    x, _, targets = make(20, 64, 300, seed=17)
    head(x, targets).backward()
    assert head.weight is linear.weight and torch.equal(linear.weight.grad, run(x, linear.weight, targets, "sum")[2])
