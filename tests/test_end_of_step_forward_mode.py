"""CPU: the row norms and the cross entropy refuse forward-mode derivatives instead of dropping them."""

import pytest
import torch
from torch.autograd import forward_ad

from hyper_multicore_b200 import MegaCrossEntropy, MegaRmsNorm, mega_cross_entropy, mega_layer_norm, mega_rms_norm

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
