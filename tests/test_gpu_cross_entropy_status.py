"""GPU: a chain whose status says that a wait gave up answers with NaN, never with numbers that look like any others.

No wait is made to run out: the words are set beforehand, as such a wait would leave them."""

import pytest
import torch

from tests.test_gpu_cross_entropy import IGNORED, make, run

pytestmark = pytest.mark.gpu


def words(first):
    from hyper_multicore_b200 import _lib

    status = torch.zeros(_lib.HMC_STATUS_WORDS, dtype=torch.int32, device="cuda")
    status[0] = first
    return status


@pytest.mark.parametrize("tokens,keep", [(20, False), (100, True), (300, False), (300, True)])
def test_a_forward_that_gave_up_has_no_loss_and_no_gradient(tokens, keep):
    from hyper_multicore_b200 import kernels as K

    x, weight, targets = make(tokens, 64, 700, ignored=0.2, seed=tokens)
    counted = targets != IGNORED
    for reduction in ("none", "mean", "sum"):
        options = dict(ignore_index=IGNORED, reduction=reduction, keep=keep)
        loss, state = K.vocab_loss(x, weight, targets, status=words(1), **options)
        assert loss.isnan().all() if reduction != "none" else torch.equal(loss.isnan(), counted)
        # the state remembers it
        grad_x, grad_w = K.vocab_loss_grad(torch.ones_like(loss), state, weight, tokens, reduction=reduction, need_hidden=True,
                                           need_weight=True, keep=keep)
        assert torch.equal(grad_x.isnan().all(1), counted) and not grad_x[~counted].any() and grad_w.isnan().all()
        # the next call in the same memory does not
        good, state = K.vocab_loss(x, weight, targets, status=words(0), **options)
        assert torch.equal(good, run(x, weight, targets, reduction)[0])


@pytest.mark.parametrize("tokens,keep,vocab", [(100, False, 700), (300, True, 700), (300, False, 700), (4096, True, 70001)])
def test_a_gradient_that_gave_up_is_nan(tokens, keep, vocab):
    from hyper_multicore_b200 import kernels as K

    x, weight, targets = make(tokens, 64, vocab, ignored=0.2, seed=tokens)
    counted = targets != IGNORED
    loss, state = K.vocab_loss(x, weight, targets, ignore_index=IGNORED, reduction="mean", keep=keep)
    options = dict(reduction="mean", need_hidden=True, need_weight=True, keep=keep)
    grad_x, grad_w = K.vocab_loss_grad(torch.ones_like(loss), state, weight, tokens, status=words(1), **options)
    assert torch.equal(grad_x.isnan().all(1), counted) and not grad_x[~counted].any() and grad_w.isnan().all()
    again = K.vocab_loss_grad(torch.ones_like(loss), state, weight, tokens, status=words(0), **options)
    want = run(x, weight, targets, recompute=not keep)
    assert torch.equal(again[0], want[1]) and torch.equal(again[1], want[2])
