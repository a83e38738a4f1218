"""Views of activations as rows, and gradients that are simply their memory."""

from __future__ import annotations

from collections.abc import Callable

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

_functorch = torch._C._functorch  # pylint: disable=protected-access


def as_rows(tensor: torch.Tensor, width: int) -> torch.Tensor:
    """``tensor`` [..., width] as [rows, width] with adjacent values; rows may lie any distance apart, so that a slice of a
    wider buffer and a broadcast row are read in place."""
    if tensor.is_neg():
        tensor = tensor.resolve_neg()
    rows = tensor if tensor.ndim == 2 else tensor.reshape(-1, width)
    return rows if width == 1 or rows.stride(1) == 1 else rows.contiguous()


def as_vector(tensor: torch.Tensor) -> torch.Tensor:
    """``tensor`` [width] as adjacent values; a lazily negated view is one of other values, contiguous or not."""
    if tensor.is_neg():
        tensor = tensor.resolve_neg()
    return tensor if tensor.is_contiguous() else tensor.contiguous()


def plain_grad(grad: torch.Tensor, what: str) -> torch.Tensor:
    """``grad``; one that is batched by vmap (``is_grads_batched``) and so no memory of its own is refused."""
    if _functorch.is_legacy_batchedtensor(grad) or _functorch.is_functorch_wrapped_tensor(grad):
        raise RuntimeError(f"{what} does not take gradients batched by vmap (is_grads_batched); call its backward once each")
    return grad


def refuse_tangents(what: str, *tensors: torch.Tensor | None) -> None:
    """An error where forward mode would differentiate ``what``: a dual tensor requires no gradient, so nothing else stops it from
    being read as its value alone, a derivative of zero."""
    if forward_ad._current_level < 0:  # pylint: disable=protected-access
        return
    if any(isinstance(t, torch.Tensor) and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise RuntimeError(f"{what} has no forward-mode derivative; differentiate it in reverse")


def first_order(backward: Callable) -> Callable:
    """``once_differentiable`` that costs nothing where no graph of the gradient is recorded."""
    guarded = once_differentiable(backward)

    def run(ctx, *grads):
        return guarded(ctx, *grads) if torch.is_grad_enabled() else backward(ctx, *grads)

    return run
