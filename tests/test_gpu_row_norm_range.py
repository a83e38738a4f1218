"""GPU: row norms at the ends of their range, with the tolerances of the row norms' other tests."""

import pytest
import torch

from tests.test_gpu_row_norm import check, make, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("center", [True, False])
@pytest.mark.parametrize("hidden,dtype", [(64, torch.bfloat16), (1024, torch.bfloat16), (1024, torch.float32), (4096, torch.bfloat16),
                                          (7168, torch.float32), (9216, torch.bfloat16), (1002, torch.float32), (33000, torch.float32)])
@pytest.mark.parametrize("exponent", [-62, -66, -70])
def test_tiny_rows_without_eps(center, hidden, dtype, exponent):
    """Values of +-2^-70 and eps = 0: their squares are whole multiples of 2^-140, which FP32 still holds and adds without a
    rounding, and 1 / rstd is 2^-70 however it is taken; only rstd^2 = 2^140 is out of range."""
    x, weight, bias, grad = make(5, hidden, dtype, torch.float32, center, seed=hidden)
    sign = torch.ones(hidden, device="cuda")
    sign[::2] = -1
    sign = sign[torch.randperm(hidden, generator=torch.Generator().manual_seed(1)).cuda()]
    x = (sign * 2.0 ** exponent).expand(5, hidden).to(dtype).contiguous()
    y, grads = run(x, weight, bias, grad, center, eps=0.0)
    assert all(t.isfinite().all() for t in (y, *(g for g in grads if g is not None)))
    check(y, grads, x, weight, bias, grad, center, 0.0)


@pytest.mark.parametrize("hidden", [1, 64, 1000])
def test_lazily_negated_tensors(hidden):
    """A conjugate's imaginary part is a view that is negated when it is read."""
    x, weight, bias, grad = make(6, hidden, torch.float32, torch.float32, True, seed=2)
    negated = [torch._neg_view(-t) for t in (x, weight, bias, grad)]
    assert all(n.is_neg() and torch.equal(n, t) for n, t in zip(negated, (x, weight, bias, grad)))
    want, want_grads = run(x, weight, bias, grad, True)
    y, grads = run(*negated, True)
    assert torch.equal(y, want) and all(torch.equal(a, b) for a, b in zip(grads, want_grads))
