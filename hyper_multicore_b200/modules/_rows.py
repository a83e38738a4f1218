"""Views of activations as rows, and gradients that are simply their memory."""

from __future__ import annotations

import torch


def as_rows(tensor: torch.Tensor, width: int) -> torch.Tensor:
    """``tensor`` [..., width] as [rows, width] with adjacent values; rows may lie any distance apart, so that a slice of a
    wider buffer and a broadcast row are read in place."""
    rows = tensor.resolve_neg().reshape(-1, width)
    return rows if width == 1 or rows.stride(1) == 1 else rows.contiguous()


def plain_grad(grad: torch.Tensor, what: str) -> torch.Tensor:
    """``grad`` as memory a kernel can read; a gradient batched by vmap (``is_grads_batched``) is refused."""
    functorch = torch._C._functorch  # pylint: disable=protected-access
    if functorch.is_legacy_batchedtensor(grad) or functorch.is_functorch_wrapped_tensor(grad):
        raise RuntimeError(f"{what} does not take gradients batched by vmap (is_grads_batched); call its backward once each")
    return grad.resolve_neg()
