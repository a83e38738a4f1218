"""GPU: what a call of the cross entropy holds until its gradient is taken, as its documentation says."""

import pytest
import torch

pytestmark = pytest.mark.gpu

TOKENS, HIDDEN, VOCAB = 2048, 256, 65536


def held(grads=True, **options):
    """(bytes that live as long as the loss, most bytes during the call)"""
    from hyper_multicore_b200 import mega_cross_entropy

    x = torch.randn(TOKENS, HIDDEN, device="cuda").bfloat16().requires_grad_(grads)
    weight = torch.randn(VOCAB, HIDDEN, device="cuda").bfloat16().requires_grad_(grads)
    targets = torch.randint(0, VOCAB, (TOKENS,), device="cuda")
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    loss = mega_cross_entropy(x, weight, targets, **options)
    torch.cuda.synchronize()
    return torch.cuda.memory_allocated() - before, torch.cuda.max_memory_allocated() - before, loss


SLACK = 4 << 20  # the allocator's blocks
ROWS = 2 * TOKENS * HIDDEN + 5 * 4 * TOKENS  # the rows that count, and five words of each
SCRATCH = TOKENS * VOCAB // 16 + 4 * TOKENS


def test_by_default_logits_are_held_in_16_bits():
    live, most, _ = held()
    logits = 2 * TOKENS * VOCAB
    assert logits < live <= ROWS + logits + logits // 64 + SLACK
    assert most <= live + SCRATCH + SLACK


@pytest.mark.parametrize("options", [dict(recompute=True), dict(grads=False)])
def test_nothing_of_tokens_times_vocabulary_is_held_otherwise(options):
    live, most, loss = held(**options)
    assert live <= ROWS + SLACK and most <= ROWS + SCRATCH + SLACK
    assert loss.requires_grad == ("grads" not in options)


def test_scratch_of_the_gradient():
    """512 MiB of probabilities and a 64th of that for their sums, 8 bytes per element of the hidden states and per word, and 40 MiB."""
    from hyper_multicore_b200 import _lib

    size = _lib.load().hmc_vocab_loss_grad_workspace_bytes
    for tokens, hidden, vocab in ((1, 8, 530_000), (129, 4096, 131072), (2048, 4096, 131072), (8192, 4096, 131072), (65536, 1024, 131072)):
        probs = min(512 << 20, 2 * tokens * (vocab + 255))
        assert size(tokens, hidden, vocab) <= probs * 65 // 64 + 8 * tokens * hidden + 8 * vocab + (40 << 20)
