"""MegaLayerNorm and MegaRmsNorm: norms of rows with their gradients.

The reference's only norm is the RMSNorm inside its mHC boundary (hyper_multicore/modules/mega_mhc/module.py:44-185); these
are the norms around it: the one before the head of a model, and those of blocks without residual streams.
"""

from __future__ import annotations

import math
from typing import Any

import torch
from torch.autograd.function import once_differentiable

from .. import _lib, kernels
from ._rows import as_rows, plain_grad


def _validate(x, weight, bias, eps) -> None:
    if not isinstance(x, torch.Tensor):
        raise TypeError("x must be a Tensor.")
    if x.dtype not in _lib.HMC_DTYPE:
        raise TypeError(f"x must be BF16, FP16 or FP32, got {x.dtype}.")
    if x.ndim < 1 or not 1 <= x.shape[-1] <= _lib.HMC_NORM_MAX_HIDDEN:
        raise ValueError(f"x must end in [hidden] with 1 <= hidden <= {_lib.HMC_NORM_MAX_HIDDEN}, got {tuple(x.shape)}.")
    if x.numel() // x.shape[-1] >= 1 << 31:
        raise ValueError("x must have fewer than 2^31 rows.")
    first = None
    for name, parameter in (("weight", weight), ("bias", bias)):
        if parameter is None:
            continue
        if not isinstance(parameter, torch.Tensor):
            raise TypeError(f"{name} must be a Tensor or None.")
        if tuple(parameter.shape) != (x.shape[-1],):
            raise ValueError(f"{name} must have shape {(x.shape[-1],)}, got {tuple(parameter.shape)}.")
        if parameter.dtype not in (x.dtype, torch.float32):
            raise TypeError(f"{name} must have dtype {x.dtype} or FP32, got {parameter.dtype}.")
        if first is not None and parameter.dtype != first:
            raise TypeError(f"weight and bias must have one dtype, got {first} and {parameter.dtype}.")
        first = parameter.dtype
        if parameter.device != x.device:
            raise ValueError(f"{name} must be on {x.device}, got {parameter.device}.")
    if not (isinstance(eps, (int, float)) and math.isfinite(eps) and eps >= 0):
        raise ValueError(f"eps must be finite and not negative, got {eps!r}.")
    if not x.is_cuda:
        raise TypeError(f"row norms on the sm_100a backend require CUDA tensors (there is no CPU path), got {x.device}.")


class _RowNormFunction(torch.autograd.Function):
    """Norm of [T, H] rows with its matching backward; first order."""

    @staticmethod
    def forward(ctx, x, weight, bias, center, eps):  # pylint: disable=arguments-differ
        rows = as_rows(x, x.shape[-1])
        w, b = (None if p is None else p.contiguous() for p in (weight, bias))
        y, mean, rstd = kernels.row_norm(rows, w, b, center=center, eps=eps, keep=True)
        ctx.save_for_backward(rows, w, mean, rstd)
        ctx.shape = x.shape
        ctx.affine_dtype = next((p.dtype for p in (weight, bias) if p is not None), x.dtype)
        return y.view(x.shape)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):  # pylint: disable=arguments-differ
        rows, weight, mean, rstd = ctx.saved_tensors
        grad_rows = as_rows(plain_grad(grad, "a row norm's backward"), rows.shape[1])
        need_x, need_weight, need_bias = ctx.needs_input_grad[:3]
        grad_x, grad_weight, grad_bias = kernels.row_norm_grad(
            grad_rows, rows, weight, mean, rstd, affine_dtype=ctx.affine_dtype, need_x=need_x, need_weight=need_weight,
            need_bias=need_bias)
        return grad_x.view(ctx.shape) if need_x else None, grad_weight, grad_bias, None, None


def _norm(x, weight, bias, center, eps):
    _validate(x, weight, bias, eps)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, bias)):
        return _RowNormFunction.apply(x, weight, bias, center, float(eps))
    w, b = (None if p is None else p.contiguous() for p in (weight, bias))
    return kernels.row_norm(as_rows(x, x.shape[-1]), w, b, center=center, eps=float(eps), keep=False)[0].view(x.shape)


def mega_layer_norm(x: torch.Tensor, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None, *,
                    eps: float = 1e-5) -> torch.Tensor:
    """(x - mean) / sqrt(var + eps) * weight + bias over the last dimension of ``x`` [..., H].

    ``x`` BF16, FP16 or FP32 with any strides; ``weight`` and ``bias`` [H] of that dtype or FP32, both the same, or None. The
    result has the dtype of ``x`` and no gaps; statistics and sums are FP32. Differentiable once in all three.
    """
    return _norm(x, weight, bias, True, eps)


def mega_rms_norm(x: torch.Tensor, weight: torch.Tensor | None = None, *, eps: float = 1e-6) -> torch.Tensor:
    """x / sqrt(mean(x^2) + eps) * weight over the last dimension of ``x`` [..., H]; types as ``mega_layer_norm``."""
    return _norm(x, weight, None, False, eps)


def _check_module(hidden_size, eps) -> None:
    if not isinstance(hidden_size, int) or isinstance(hidden_size, bool) or not 1 <= hidden_size <= _lib.HMC_NORM_MAX_HIDDEN:
        raise ValueError(f"hidden_size must be an integer in [1, {_lib.HMC_NORM_MAX_HIDDEN}], got {hidden_size!r}.")
    if not (isinstance(eps, (int, float)) and math.isfinite(eps) and eps >= 0):
        raise ValueError(f"eps must be finite and not negative, got {eps!r}.")


class MegaLayerNorm(torch.nn.Module):
    """Layer norm over the last dimension with weight and (by default) bias."""

    def __init__(self, hidden_size: int, *, eps: float = 1e-5, bias: bool = True, device: Any | None = None,
                 dtype: torch.dtype = torch.bfloat16) -> None:
        super().__init__()
        _check_module(hidden_size, eps)
        self.hidden_size, self.eps = hidden_size, float(eps)
        self.weight = torch.nn.Parameter(torch.ones(hidden_size, device=device, dtype=dtype))
        if bias:
            self.bias = torch.nn.Parameter(torch.zeros(hidden_size, device=device, dtype=dtype))
        else:
            self.register_parameter("bias", None)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return mega_layer_norm(x, self.weight, self.bias, eps=self.eps)


class MegaRmsNorm(torch.nn.Module):
    """RMSNorm over the last dimension with weight."""

    def __init__(self, hidden_size: int, *, eps: float = 1e-6, device: Any | None = None,
                 dtype: torch.dtype = torch.bfloat16) -> None:
        super().__init__()
        _check_module(hidden_size, eps)
        self.hidden_size, self.eps = hidden_size, float(eps)
        self.weight = torch.nn.Parameter(torch.ones(hidden_size, device=device, dtype=dtype))

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return mega_rms_norm(x, self.weight, eps=self.eps)
