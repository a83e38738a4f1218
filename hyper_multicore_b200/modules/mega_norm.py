"""MegaLayerNorm and MegaRmsNorm: norms of rows with their gradients.

The reference's only norm is the RMSNorm inside its mHC boundary (hyper_multicore/modules/mega_mhc/module.py:44-185); these
are the norms around it: the one before the head of a model, and those of blocks without residual streams.
"""

from __future__ import annotations

import math
from typing import Any

import torch

from .. import _lib, kernels
from ._rows import as_rows, as_vector, first_order, plain_grad, refuse_tangents


def _fits(x, weight, bias, eps) -> bool:
    """All of ``_validate`` in one expression, which builds no message; that one then says what is wrong."""
    if type(x) is not torch.Tensor or not x.is_cuda or x.ndim == 0 or type(eps) is not float or not 0.0 <= eps < math.inf:
        return False
    dtype, index = x.dtype, x.get_device()
    shape = x.shape[-1:]
    if not (1 <= shape[0] <= _lib.HMC_NORM_MAX_HIDDEN and x.numel() <= shape[0] * _lib.HMC_NORM_MAX_ROWS and dtype in _lib.HMC_DTYPE):
        return False
    affine = (dtype, torch.float32)
    if weight is not None:
        if not (isinstance(weight, torch.Tensor) and weight.shape == shape and weight.is_cuda and weight.get_device() == index
                and weight.dtype in affine):
            return False
        affine = (weight.dtype,)
    return bias is None or (isinstance(bias, torch.Tensor) and bias.shape == shape and bias.is_cuda and bias.get_device() == index
                            and bias.dtype in affine)


def _validate(x, weight, bias, eps) -> None:
    if not isinstance(x, torch.Tensor):
        raise TypeError("x must be a Tensor.")
    if x.dtype not in _lib.HMC_DTYPE:
        raise TypeError(f"x must be BF16, FP16 or FP32, got {x.dtype}.")
    if x.ndim < 1 or not 1 <= x.shape[-1] <= _lib.HMC_NORM_MAX_HIDDEN:
        raise ValueError(f"x must end in [hidden] with 1 <= hidden <= {_lib.HMC_NORM_MAX_HIDDEN}, got {tuple(x.shape)}.")
    if x.numel() // x.shape[-1] > _lib.HMC_NORM_MAX_ROWS:
        raise ValueError(f"x must have at most {_lib.HMC_NORM_MAX_ROWS} rows.")
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
    """Norm of rows with its matching backward; first order."""

    @staticmethod
    def forward(ctx, x, weight, bias, center, eps):  # pylint: disable=arguments-differ
        y, rows, weight, bias, stats = _forward(x, weight, bias, center, eps, True)
        ctx.save_for_backward(rows, weight, stats)
        ctx.of = center, x.shape, None if weight is not None else x.dtype if bias is None else bias.dtype
        return y

    @staticmethod
    @first_order
    def backward(ctx, grad):  # pylint: disable=arguments-differ
        rows, weight, stats = ctx.saved_tensors
        center, shape, affine_dtype = ctx.of
        need_x, need_weight, need_bias, _, _ = ctx.needs_input_grad
        grad = as_rows(plain_grad(grad, "a row norm's backward"), shape[-1])
        grad_x, grad_weight, grad_bias = kernels.row_norm_grad(grad, rows, weight, stats, center, affine_dtype, need_x, need_weight,
                                                               need_bias, rows.device)
        if need_x and len(shape) != 2:
            grad_x = grad_x.view(shape)
        return grad_x, grad_weight, grad_bias, None, None


def _forward(x, weight, bias, center, eps, keep):
    """(y, x as rows, parameters as the kernel reads them, statistics)"""
    rows = as_rows(x, x.shape[-1])
    if weight is not None:
        weight = as_vector(weight)
    if bias is not None:
        bias = as_vector(bias)
    y, stats = kernels.row_norm(rows, weight, bias, center, eps, keep, x.device)
    return y if x.ndim == 2 else y.view(x.shape), rows, weight, bias, stats


def _norm(x, weight, bias, center, eps):
    refuse_tangents("a row norm", x, weight, bias)
    if not _fits(x, weight, bias, eps):
        _validate(x, weight, bias, eps)
    if torch.is_grad_enabled() and (x.requires_grad or (weight is not None and weight.requires_grad)
                                    or (bias is not None and bias.requires_grad)):
        return _RowNormFunction.apply(x, weight, bias, center, float(eps))
    return _forward(x, weight, bias, center, float(eps), False)[0]


def mega_layer_norm(x: torch.Tensor, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None, *,
                    eps: float = 1e-5) -> torch.Tensor:
    """(x - mean) / sqrt(var + eps) * weight + bias over the last dimension of ``x`` [..., H].

    ``x`` BF16, FP16 or FP32 with any strides; ``weight`` and ``bias`` [H] of that dtype or FP32, both the same, or None. The
    result has the dtype of ``x`` and no gaps; statistics and sums are FP32. Differentiable once, in reverse, in all three. Few rows with
    their gradient are bound by the host: 110 to 130 us a call and its backward pass, where torch's own layer norm takes 70.
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
