"""CPU: the modules refuse forward-mode derivatives instead of dropping them."""

import pytest
import torch
from torch.autograd import forward_ad

from hyper_multicore_b200 import (MegaCrossEntropy, MegaGate, MegaRmsNorm, hyper_mega_mhc, mega_cross_entropy, mega_layer_norm,
                                  mega_rms_norm)

CALLS = {
    "layer norm": (lambda x, w, b: mega_layer_norm(x, w, b), [(3, 8), (8,), (8,)]),
    "RMSNorm": (lambda x, w: mega_rms_norm(x, w), [(3, 8), (8,)]),
    "RMSNorm module": (lambda x: MegaRmsNorm(8)(x), [(3, 8)]),
    "cross entropy": (lambda x, w: mega_cross_entropy(x, w, torch.zeros(3, dtype=torch.int64)), [(3, 8), (10, 8)]),
    "cross entropy module": (lambda x: MegaCrossEntropy(8, 10, recompute=True)(x, torch.zeros(3, dtype=torch.int64)), [(3, 8)]),
}


@pytest.mark.parametrize("name,which", [(name, i) for name, (_, shapes) in CALLS.items() for i in range(len(shapes))])
@pytest.mark.parametrize("requires_grad", [False, True])
def test_tangents_are_refused(name, which, requires_grad):
    call, shapes = CALLS[name]
    tensors = [torch.randn(s).bfloat16().requires_grad_(requires_grad) for s in shapes]
    with forward_ad.dual_level():
        tensors[which] = forward_ad.make_dual(tensors[which], torch.ones(shapes[which]).bfloat16())
        with pytest.raises(RuntimeError, match="no forward-mode derivative"):
            call(*tensors)
        with torch.no_grad(), pytest.raises(RuntimeError, match="no forward-mode derivative"):
            call(*tensors)
        with pytest.raises(TypeError, match="CUDA"):  # the others have no tangent: the next refusal
            call(*(forward_ad.unpack_dual(t).primal for t in tensors))


@pytest.mark.parametrize("which", range(2))
def test_tangents_of_the_gate_are_refused(which):
    gate = MegaGate(hidden_size=64, num_experts=8, top_k=2, scoring_func="softmax", routed_scaling_factor=1.0)
    hidden = torch.randn(1, 4, 64).bfloat16()
    with forward_ad.dual_level():
        if which == 0:
            hidden = forward_ad.make_dual(hidden, torch.ones_like(hidden))
        else:
            weight = gate.weight.detach()
            del gate.weight
            gate.weight = forward_ad.make_dual(weight, torch.ones_like(weight))
        with pytest.raises(RuntimeError, match="no forward-mode derivative"):
            gate(hidden)


@pytest.mark.parametrize("which", range(9))
def test_tangents_of_the_mhc_boundary_are_refused(which):
    tensors = [torch.randn(4, 8) for _ in range(9)]
    with forward_ad.dual_level():
        tensors[which] = forward_ad.make_dual(tensors[which], torch.ones(4, 8))
        with pytest.raises(RuntimeError, match="no forward-mode derivative"):
            hyper_mega_mhc(*tensors)
