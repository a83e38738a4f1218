"""Performance cases of the end of a training step: row norms and the cross entropy over the vocabulary.

``mega_layer_norm`` and ``mega_rms_norm`` normalise rows of activations, ``mega_cross_entropy`` takes hidden states and the
head's weight to the loss without keeping the logits; each has its gradient. Sizes are those of the repository's
benchmark configurations (rows of 2560, 4096 and 7168 values; 1531, 4096, 8192 and 16384 tokens) and generic ones
around them. While ``own`` is false every case runs in elementary torch operations on FP32 copies of its inputs.
"""

import math

import torch

own = False

IGNORED = -100  # target of a token that has no loss
_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    return [
        # One decode step of one sequence: the norm before the head. Latency of a call.
        dict(name="layer_decode", kind="norm", center=True, tokens=1, hidden=4096, pad=0, dtype="bf16", affine="bf16",
             train=False),
        # A decode step of 16 sequences on the widest rows.
        dict(name="rms_decode", kind="norm", center=False, tokens=16, hidden=7168, pad=0, dtype="bf16", affine="bf16",
             train=False),
        # Prefill: rows that are read as a slice of a wider buffer (what a fused projection leaves).
        dict(name="rms_prefill_slice", kind="norm", center=False, tokens=8192, hidden=4096, pad=512, dtype="bf16",
             affine="fp32", train=False),
        # FP32 activations with an odd row length, whose rows start on no vector boundary.
        dict(name="layer_train_odd", kind="norm", center=True, tokens=2999, hidden=1001, pad=0, dtype="fp32", affine="fp32",
             train=True),
        # A short odd number of tokens (what sequence packing leaves over) with FP32 parameters.
        dict(name="layer_train_ragged", kind="norm", center=True, tokens=1531, hidden=2560, pad=0, dtype="bf16",
             affine="fp32", train=True),
        # FP16 training micro-batch of mid size.
        dict(name="rms_train_half", kind="norm", center=False, tokens=4096, hidden=4096, pad=0, dtype="fp16", affine="fp16",
             train=True),
        # A full training micro-batch.
        dict(name="layer_train", kind="norm", center=True, tokens=16384, hidden=7168, pad=0, dtype="bf16", affine="bf16",
             train=True),
        # Scoring of one decode step: log probabilities of the tokens that 16 sequences took.
        dict(name="loss_score", kind="loss", tokens=16, hidden=4096, vocab=131072, ignored=0.0, reduction="none",
             norm=False, train=False),
        # A small model's training step: launches and short tiles count.
        dict(name="loss_train_small", kind="loss", tokens=512, hidden=1024, vocab=32000, ignored=0.0, reduction="mean",
             norm=False, train=True),
        # Weighted losses of an odd number of tokens, three tenths of them prompt, over an odd vocabulary.
        dict(name="loss_train_ragged", kind="loss", tokens=3001, hidden=2048, vocab=50257, ignored=0.3, reduction="none",
             norm=False, train=True),
        # The end of a training step as it is used: RMSNorm, head, loss and the gradients of all three.
        dict(name="head_train", kind="loss", tokens=4096, hidden=4096, vocab=65536, ignored=0.1, reduction="mean",
             norm=True, train=True),
        # A full training micro-batch over a large vocabulary.
        dict(name="loss_train", kind="loss", tokens=8192, hidden=4096, vocab=131072, ignored=0.0, reduction="mean",
             norm=False, train=True),
    ]


def _log_int(rng, low, high):
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    """One more case: the same operators and options, sizes spread over the whole range."""
    if rng.random() < 0.5:
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        odd = rng.random() < 0.3
        hidden = _log_int(rng, 64, 7168) if odd else 64 * _log_int(rng, 1, 112)
        return dict(kind="norm", center=rng.random() < 0.5, tokens=_log_int(rng, 1, 16384), hidden=hidden,
                    pad=rng.choice([0, 0, 0, 64]), dtype=dtype, affine=rng.choice([dtype, "fp32"]), train=rng.random() < 0.6)
    train = rng.random() < 0.6
    hidden, vocab = 8 * _log_int(rng, 16, 512), _log_int(rng, 1000, 131072)
    return dict(kind="loss", tokens=_log_int(rng, 1, 8192), hidden=hidden, vocab=vocab, ignored=rng.choice([0.0, 0.0, 0.1, 0.5]),
                reduction=rng.choice(["mean", "sum", "none"]), norm=train and rng.random() < 0.3, train=train)


# ------------------------------------------------------------------------------------------------ inputs
def _normal(g, *shape, scale=1.0):
    return torch.randn(*shape, generator=g, device="cuda").mul_(scale)


def _prepare_norm(case, g):
    tokens, hidden, dtype = case["tokens"], case["hidden"], _DTYPES[case["dtype"]]
    # residual-stream activations: tokens of different size, a common offset, a few channels far larger than the others
    channel = 1 + 30 * (torch.rand(hidden, generator=g, device="cuda") < 0.002).float()
    x = torch.zeros(tokens, hidden + case["pad"], device="cuda")
    x[:, :hidden] = _normal(g, tokens, hidden) * channel * (0.5 + _normal(g, tokens, 1).abs()) + 0.3
    state = dict(case=case, x=x.to(dtype)[:, :hidden], weight=(1 + _normal(g, hidden, scale=0.1)).to(_DTYPES[case["affine"]]),
                 bias=_normal(g, hidden, scale=0.1).to(_DTYPES[case["affine"]]) if case["center"] else None, eps=1e-6)
    if case["train"]:
        state["grad"] = _normal(g, tokens, hidden).to(dtype)
    return state


def _prepare_loss(case, g):
    tokens, hidden, vocab = case["tokens"], case["hidden"], case["vocab"]
    weight = _normal(g, vocab, hidden, scale=hidden ** -0.5).bfloat16()
    # words are drawn by a power law; a model halfway through training gives most of them part of the mass
    place = torch.rand(tokens, generator=g, device="cuda")
    target = (torch.exp(place * math.log(vocab + 1)) - 1).long().clamp_(0, vocab - 1)
    learned = torch.rand(tokens, 1, generator=g, device="cuda") * 1.2 * math.log(vocab)
    x = _normal(g, tokens, hidden) + learned * weight[target].float()
    state = dict(case=case, x=x.bfloat16(), weight=weight, gain=None)
    if case["norm"]:
        state["gain"] = (1 + _normal(g, hidden, scale=0.1)).bfloat16()
    left_out = torch.randperm(tokens, generator=g, device="cuda")[: tokens - _counted(case)]
    target[left_out] = IGNORED
    state["target"] = target
    if case["train"]:
        shape = (tokens,) if case["reduction"] == "none" else ()
        state["grad"] = torch.rand(shape, generator=g, device="cuda") + 0.5
        if case["reduction"] != "mean":
            state["grad"] /= tokens
    return state


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    state = _prepare_norm(case, g) if case["kind"] == "norm" else _prepare_loss(case, g)
    if case["train"]:
        for name in ("x", "weight", "bias", "gain"):
            if state.get(name) is not None:
                state[name] = state[name].detach().requires_grad_(True)
    return state


# ------------------------------------------------------------------------------------------------ plain forms
def _plain_norm(x, weight, bias, eps):
    """Rows of x normalised in FP32; also the normalised rows and their scale, for the gradient."""
    x = x.float()
    if bias is not None:
        x = x - x.mean(-1, keepdim=True)
    rstd = torch.rsqrt((x * x).mean(-1, keepdim=True) + eps)
    unit = x * rstd
    y = unit * weight.float()
    return y if bias is None else y + bias.float(), unit, rstd


def _plain_norm_grad(grad, unit, rstd, weight, center):
    grad = grad.float()
    inner = grad * weight.float()
    grad_x = inner - unit * (inner * unit).mean(-1, keepdim=True)
    if center:
        grad_x = grad_x - inner.mean(-1, keepdim=True)
    return grad_x * rstd, (grad * unit).sum(0), grad.sum(0)


def _plain_loss(x, weight, target, reduction):
    """Loss of FP32 logits; also the softmax, for the gradient."""
    logits = x.float() @ weight.float().t()
    top = logits.amax(-1, keepdim=True)
    counted = target != IGNORED
    index = torch.where(counted, target, 0).unsqueeze(1)
    own_logit = logits.gather(1, index)
    p = logits.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    loss = torch.where(counted, (total.log() + (top - own_logit)).squeeze(1), 0.0)
    if reduction != "none":
        loss = loss.sum()
    if reduction == "mean":
        loss = loss / counted.sum()
    return loss, p.div_(total), index, counted


def _plain_loss_grad(grad, p, index, counted, x, weight, reduction):
    if reduction == "mean":
        grad = grad / counted.sum()
    grad = (grad * counted).unsqueeze(1)
    p = p.scatter_add_(1, index, torch.full_like(index, -1, dtype=p.dtype)).mul_(grad)
    return p @ weight.float(), p.t() @ x.float()


@torch.no_grad()
def _run_plain_norm(s):
    case, x, weight, bias = s["case"], s["x"], s["weight"], s["bias"]
    y, unit, rstd = _plain_norm(x, weight, bias, s["eps"])
    if not case["train"]:
        return y.to(x.dtype)
    grad_x, grad_weight, grad_bias = _plain_norm_grad(s["grad"], unit, rstd, weight, case["center"])
    grads = (grad_x.to(x.dtype), grad_weight.to(weight.dtype))
    return (y.to(x.dtype), *grads, grad_bias.to(bias.dtype)) if case["center"] else (y.to(x.dtype), *grads)


@torch.no_grad()
def _run_plain_loss(s):
    case, x, weight, gain = s["case"], s["x"], s["weight"], s["gain"]
    h = x
    if gain is not None:
        y, unit, rstd = _plain_norm(x, gain, None, 1e-6)
        h = y.to(x.dtype)  # the head reads BF16 rows
    loss, p, index, counted = _plain_loss(h, weight, s["target"], case["reduction"])
    if not case["train"]:
        return loss
    grad_h, grad_weight = _plain_loss_grad(s["grad"], p, index, counted, h, weight, case["reduction"])
    grad_h, grad_weight = grad_h.to(h.dtype), grad_weight.to(weight.dtype)
    if gain is None:
        return loss, grad_h, grad_weight
    grad_x, grad_gain, _ = _plain_norm_grad(grad_h, unit, rstd, gain, False)
    return loss, grad_x.to(x.dtype), grad_weight, grad_gain.to(gain.dtype)


# ------------------------------------------------------------------------------------------------ the framework's calls
def _run_own_norm(s):
    from hyper_multicore_b200 import mega_layer_norm, mega_rms_norm

    case, x, weight, bias = s["case"], s["x"], s["weight"], s["bias"]
    if not case["train"]:
        with torch.no_grad():
            return (mega_layer_norm(x, weight, bias, eps=s["eps"]) if case["center"]
                    else mega_rms_norm(x, weight, eps=s["eps"]))
    if case["center"]:
        y = mega_layer_norm(x, weight, bias, eps=s["eps"])
        return (y.detach(), *torch.autograd.grad(y, (x, weight, bias), s["grad"]))
    y = mega_rms_norm(x, weight, eps=s["eps"])
    return (y.detach(), *torch.autograd.grad(y, (x, weight), s["grad"]))


def _run_own_loss(s):
    from hyper_multicore_b200 import mega_cross_entropy, mega_rms_norm

    case, x, weight, gain, target = s["case"], s["x"], s["weight"], s["gain"], s["target"]
    if not case["train"]:
        with torch.no_grad():
            return mega_cross_entropy(x, weight, target, ignore_index=IGNORED, reduction=case["reduction"])
    h = x if gain is None else mega_rms_norm(x, gain, eps=1e-6)
    loss = mega_cross_entropy(h, weight, target, ignore_index=IGNORED, reduction=case["reduction"])
    leaves = (x, weight) if gain is None else (x, weight, gain)
    return (loss.detach(), *torch.autograd.grad(loss, leaves, s["grad"]))


def run(state):
    if own:
        return _run_own_norm(state) if state["case"]["kind"] == "norm" else _run_own_loss(state)
    return _run_plain_norm(state) if state["case"]["kind"] == "norm" else _run_plain_loss(state)


# ------------------------------------------------------------------------------------------------ work and exact values
def _counted(case):
    """Tokens of a case that have a loss: one at least."""
    return max(1, case["tokens"] - int(case["ignored"] * case["tokens"]))


def work(case):
    tokens, hidden = case["tokens"], case["hidden"]
    if case["kind"] == "norm":
        size, affine = _DTYPES[case["dtype"]].itemsize, _DTYPES[case["affine"]].itemsize
        rows, vectors = tokens * hidden * size, hidden * affine * (2 if case["center"] else 1)
        # forward: x, parameters -> y; with the gradient also grad -> grad_x, grad_parameters
        return {"bytes": (4 if case["train"] else 2) * rows + (2 if case["train"] else 1) * vectors,
                "flops": (18 if case["train"] else 7) * tokens * hidden}
    # tokens without a loss need no logits; the two gradients are a product of the same size each
    product = 2 * _counted(case) * case["vocab"] * hidden
    rows, weight = 2 * tokens * hidden, 2 * case["vocab"] * hidden
    losses = 4 * tokens if case["reduction"] == "none" else 4
    return {"bytes": (2 if case["train"] else 1) * (rows + weight) + 8 * tokens + (2 if case["train"] else 1) * losses,
            "flops": (3 if case["train"] else 1) * product}


def _exact_norm(x, weight, bias, eps):
    if bias is None:
        return x / torch.sqrt(x.pow(2).mean(-1, keepdim=True) + eps) * weight
    var, mean = torch.var_mean(x, -1, correction=0, keepdim=True)
    return (x - mean) / torch.sqrt(var + eps) * weight + bias


def exact(case, seed):
    """The definitions in FP64, differentiated by autograd; the loss over a few thousand tokens at a time."""
    s = prepare(case, seed)
    leaves = [n for n in ("x", "weight", "bias", "gain") if s.get(n) is not None]
    v = {n: s[n].detach().double().requires_grad_(case["train"]) for n in leaves}
    if case["kind"] == "norm":
        y = _exact_norm(v["x"], v["weight"], v.get("bias"), s["eps"])
        if not case["train"]:
            return y
        return (y.detach(), *torch.autograd.grad(y, [v[n] for n in leaves], s["grad"].double()))
    h = v["x"]
    if case["norm"]:
        h = _exact_norm(v["x"], v["gain"], None, 1e-6)
    h_in = h.detach().requires_grad_(case["train"])
    weights = torch.ones(case["tokens"], dtype=torch.float64, device="cuda")
    if case["train"]:
        weights = weights * s["grad"].double()
    if case["reduction"] == "mean":
        weights = weights / _counted(case)
    losses, grad_h, grad_weight = [], [], 0.0
    for at in range(0, case["tokens"], 2048):
        rows, target = h_in[at:at + 2048], s["target"][at:at + 2048]
        logits = rows @ v["weight"].t()
        counted = target != IGNORED
        loss = torch.logsumexp(logits, 1) - logits.gather(1, target.clamp(min=0).unsqueeze(1)).squeeze(1)
        loss = loss * counted
        losses.append(loss.detach())
        if case["train"]:
            part, more = torch.autograd.grad(loss, (h_in, v["weight"]), weights[at:at + 2048])
            grad_h.append(part[at:at + 2048])
            grad_weight = grad_weight + more
        del logits, loss
    total = torch.cat(losses)
    if case["reduction"] != "none":
        total = total.sum() / (_counted(case) if case["reduction"] == "mean" else 1)
    if not case["train"]:
        return total
    grad_h = torch.cat(grad_h)
    if not case["norm"]:
        return total, grad_h, grad_weight
    grad_x, grad_gain = torch.autograd.grad(h, (v["x"], v["gain"]), grad_h)
    return total, grad_x, grad_weight, grad_gain
