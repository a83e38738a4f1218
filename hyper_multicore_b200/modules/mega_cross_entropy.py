"""MegaCrossEntropy: the head of a model and its loss over the vocabulary in one; logits are held in 16 bits, or not at all.

The reference ends before the head; this is the operator that follows the last norm in training and in scoring.
"""

from __future__ import annotations

import math
from typing import Any

import torch

from .. import _lib, kernels
from ._rows import as_rows, first_order, plain_grad, refuse_tangents


def _fits(hidden, weight, targets, ignore_index, reduction) -> bool:
    """All of ``_validate`` in one expression, which builds no message; that one then says what is wrong."""
    return (type(hidden) is torch.Tensor and hidden.is_cuda and hidden.ndim > 0 and hidden.dtype == torch.bfloat16
            and isinstance(weight, torch.Tensor) and weight.ndim == 2 and weight.dtype == torch.bfloat16
            and hidden.shape[-1] == weight.shape[1] and weight.shape[1] % 8 == 0 and 0 < weight.shape[1] < 1 << 30
            and 0 < weight.shape[0] < (1 << 31) - 256 and weight.device == hidden.device
            and isinstance(targets, torch.Tensor) and targets.dtype in (torch.int64, torch.int32)
            and targets.shape == hidden.shape[:-1] and targets.device == hidden.device and targets.numel() < (1 << 31) - 256
            and type(ignore_index) is int and -(1 << 63) <= ignore_index < 1 << 63 and reduction in _lib.HMC_REDUCE)


def _validate(hidden, weight, targets, ignore_index, reduction) -> None:
    if _fits(hidden, weight, targets, ignore_index, reduction):
        return
    for name, tensor in (("hidden", hidden), ("weight", weight), ("targets", targets)):
        if not isinstance(tensor, torch.Tensor):
            raise TypeError(f"{name} must be a Tensor.")
    if reduction not in _lib.HMC_REDUCE:
        raise ValueError(f"reduction must be one of {tuple(_lib.HMC_REDUCE)}, got {reduction!r}.")
    if not isinstance(ignore_index, int) or isinstance(ignore_index, bool) or not -(1 << 63) <= ignore_index < 1 << 63:
        raise ValueError(f"ignore_index must be an integer of 64 bits, got {ignore_index!r}.")
    if weight.ndim != 2 or weight.shape[0] == 0 or weight.shape[1] == 0 or weight.shape[1] % 8:
        raise ValueError(f"weight must be [vocab, hidden] with hidden a multiple of 8, got {tuple(weight.shape)}.")
    if hidden.ndim < 1 or hidden.shape[-1] != weight.shape[1]:
        raise ValueError(f"hidden must end in [{weight.shape[1]}], got {tuple(hidden.shape)}.")
    if targets.shape != hidden.shape[:-1]:
        raise ValueError(f"targets must have shape {tuple(hidden.shape[:-1])}, got {tuple(targets.shape)}.")
    if targets.numel() >= (1 << 31) - 256 or weight.shape[0] >= (1 << 31) - 256 or weight.shape[1] >= 1 << 30:
        raise ValueError("tokens and vocab must be below 2^31 - 256, hidden below 2^30.")
    if hidden.dtype != torch.bfloat16 or weight.dtype != torch.bfloat16:
        raise TypeError(f"hidden and weight must be BF16, got {hidden.dtype} and {weight.dtype}.")
    if targets.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"targets must be INT32 or INT64, got {targets.dtype}.")
    if not hidden.is_cuda:
        raise TypeError(f"MegaCrossEntropy requires CUDA tensors (there is no CPU path), got {hidden.device}.")
    for name, tensor in (("weight", weight), ("targets", targets)):
        if tensor.device != hidden.device:
            raise ValueError(f"{name} must be on {hidden.device}, got {tensor.device}.")


def _weight_rows(weight: torch.Tensor) -> torch.Tensor:
    """The weight in place where its rows are adjacent values that start on 16-byte boundaries, a copy otherwise."""
    if weight.is_neg():
        weight = weight.resolve_neg()
    one_row = weight.shape[0] == 1
    if (weight.stride(1) == 1 and (one_row or (weight.stride(0) % 8 == 0 and weight.stride(0) >= weight.shape[1]))
            and weight.data_ptr() % 16 == 0):
        return weight if not one_row or weight.stride(0) == weight.shape[1] else weight.view(-1).view(1, -1)
    return weight.clone(memory_format=torch.contiguous_format)


def _forward(rows, weight, targets, ignore_index, reduction, keep=False):
    """(loss, state); without a token the empty tensor, sum or mean."""
    if targets.numel() == 0:
        f32 = dict(dtype=torch.float32, device=rows.device)
        loss = torch.empty(0, **f32) if reduction == "none" else torch.full((), math.nan if reduction == "mean" else 0.0, **f32)
        return loss, None
    return kernels.vocab_loss(rows, weight, targets, ignore_index=ignore_index, reduction=reduction, keep=keep)


class _CrossEntropyFunction(torch.autograd.Function):
    """Loss of packed rows with its matching backward; first order."""

    @staticmethod
    def forward(ctx, hidden, weight, targets, ignore_index, reduction, keep):  # pylint: disable=arguments-differ
        rows_of_weight = _weight_rows(weight)
        loss, state = _forward(hidden, rows_of_weight, targets, ignore_index, reduction, keep)
        ctx.save_for_backward(state, rows_of_weight)
        ctx.tokens, ctx.reduction, ctx.keep = hidden.shape[0], reduction, keep
        return loss

    @staticmethod
    @first_order
    def backward(ctx, grad_loss):  # pylint: disable=arguments-differ
        state, weight = ctx.saved_tensors
        if ctx.tokens == 0:
            return (torch.empty((0, weight.shape[1]), dtype=torch.bfloat16, device=weight.device),
                    torch.zeros(weight.shape, dtype=torch.bfloat16, device=weight.device), None, None, None, None)
        grad = plain_grad(grad_loss, "MegaCrossEntropy's backward").resolve_neg().contiguous()
        grad_hidden, grad_weight = kernels.vocab_loss_grad(grad, state, weight, ctx.tokens, reduction=ctx.reduction, keep=ctx.keep,
                                                           need_hidden=ctx.needs_input_grad[0], need_weight=ctx.needs_input_grad[1])
        return grad_hidden, grad_weight, None, None, None, None


def mega_cross_entropy(hidden: torch.Tensor, weight: torch.Tensor, targets: torch.Tensor, *, ignore_index: int = -100,
                       reduction: str = "mean", recompute: bool = False) -> torch.Tensor:
    """Cross entropy of ``hidden @ weight.T`` against ``targets``, FP32. Where a gradient follows, the call holds its logits in 16 bits
    until then, up to 4 GiB of them: as much as BF16 logits would take. With ``recompute=True`` it holds none.

    ``hidden`` BF16 [..., H] with any strides, ``weight`` BF16 [V, H] with H a multiple of 8, ``targets`` INT32 or INT64 [...].
    ``reduction`` "none" gives a loss per token (0 where the target is ``ignore_index``), "sum" and "mean" run over the other
    tokens; the mean over none of them is NaN, as in torch. Ignored tokens are not read: whatever their hidden states hold,
    their gradient is zero and they add nothing to the weight's. A target outside [0, V) that is not ``ignore_index`` is not
    noticed on the host: its loss is NaN, and so are the gradients it enters. Differentiable once, in reverse, in ``hidden`` and ``weight``;
    the gradients are BF16, and so are the probabilities that enter them; a token's keep their sum. What is held are the logits'
    distances from the largest of 128, of as many words as fit 4 GiB (none up to 128 tokens); the others are computed again, with
    ``recompute`` all of them, which takes a quarter longer. Every call whose graph lives holds its own. The backward pass takes
    scratch of up to 512 MiB for probabilities (4096 words of them where that is more) and a 64th of that for their sums, 8 bytes per
    element of ``hidden`` and per word, and 40 MiB. A wait inside a kernel that gives up makes the loss, or the gradients, NaN.
    """
    if recompute is not False and recompute is not True:
        raise ValueError(f"recompute must be a bool, got {recompute!r}.")
    refuse_tangents("MegaCrossEntropy", hidden, weight)
    _validate(hidden, weight, targets, ignore_index, reduction)
    rows = as_rows(hidden, weight.shape[1])
    flat = targets if targets.ndim == 1 and targets.is_contiguous() else targets.reshape(-1).contiguous()
    if torch.is_grad_enabled() and (hidden.requires_grad or weight.requires_grad):
        loss = _CrossEntropyFunction.apply(rows, weight, flat, ignore_index, reduction, not recompute)
    else:
        loss = _forward(rows, _weight_rows(weight), flat, ignore_index, reduction)[0]
    return loss.view(targets.shape) if reduction == "none" and targets.ndim != 1 else loss


class MegaCrossEntropy(torch.nn.Module):
    """Own the head's weight [vocab, hidden] and give the loss of hidden states against targets."""

    def __init__(self, hidden_size: int, vocab_size: int, *, ignore_index: int = -100, reduction: str = "mean",
                 recompute: bool = False, initializer_range: float = 0.02, device: Any | None = None) -> None:
        super().__init__()
        for name, value in (("hidden_size", hidden_size), ("vocab_size", vocab_size)):
            if not isinstance(value, int) or isinstance(value, bool) or value <= 0:
                raise ValueError(f"{name} must be a positive integer, got {value!r}.")
        if hidden_size % 8:
            raise ValueError(f"hidden_size must be a multiple of 8, got {hidden_size}.")
        if reduction not in _lib.HMC_REDUCE:
            raise ValueError(f"reduction must be one of {tuple(_lib.HMC_REDUCE)}, got {reduction!r}.")
        if not isinstance(recompute, bool):
            raise ValueError(f"recompute must be a bool, got {recompute!r}.")
        if not math.isfinite(initializer_range) or initializer_range < 0.0:
            raise ValueError("initializer_range must be finite and nonnegative")
        self.hidden_size, self.vocab_size = hidden_size, vocab_size
        self.ignore_index, self.reduction, self.recompute = ignore_index, reduction, recompute
        self.weight = torch.nn.Parameter(torch.empty(vocab_size, hidden_size, device=device, dtype=torch.bfloat16))
        torch.nn.init.normal_(self.weight, mean=0.0, std=initializer_range)

    @classmethod
    def from_module(cls, module: torch.nn.Module, **configuration: Any) -> "MegaCrossEntropy":
        """Share the weight of an existing bias-free head (``weight`` BF16 [vocab, hidden]) without copying it."""
        weight = getattr(module, "weight", None)
        if not isinstance(weight, torch.nn.Parameter) or weight.ndim != 2 or weight.dtype != torch.bfloat16:
            raise ValueError("source head requires a BF16 weight Parameter shaped [vocab, hidden]")
        if getattr(module, "bias", None) is not None:
            raise ValueError("source head must not have a bias")
        result = cls(weight.shape[1], weight.shape[0], device="meta", **configuration)
        result.weight = weight
        return result

    def forward(self, hidden: torch.Tensor, targets: torch.Tensor) -> torch.Tensor:
        return mega_cross_entropy(hidden, self.weight, targets, ignore_index=self.ignore_index, reduction=self.reduction,
                                  recompute=self.recompute)
