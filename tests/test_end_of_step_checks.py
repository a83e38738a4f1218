"""CPU: what the row norms and the cross entropy refuse, from Python and at the C boundary, without a device."""

import ctypes
import math

import pytest
import torch

from hyper_multicore_b200 import (MegaCrossEntropy, MegaLayerNorm, MegaRmsNorm, _lib, mega_cross_entropy, mega_layer_norm,
                                  mega_rms_norm)

BF16 = torch.bfloat16


@pytest.mark.parametrize("error,match,call", [
    (TypeError, "must be a Tensor", lambda: mega_layer_norm([1.0])),
    (TypeError, "BF16, FP16 or FP32", lambda: mega_rms_norm(torch.zeros(2, 8, dtype=torch.float64))),
    (ValueError, "must end in", lambda: mega_rms_norm(torch.zeros((), dtype=BF16))),
    (ValueError, "must end in", lambda: mega_rms_norm(torch.zeros(4, 0, dtype=BF16))),
    (ValueError, "rows", lambda: mega_rms_norm(torch.zeros(1, 1).expand((1 << 31) - 1, 1))),
    (ValueError, "weight must have shape", lambda: mega_rms_norm(torch.zeros(2, 8), torch.ones(7))),
    (TypeError, "weight must have dtype", lambda: mega_rms_norm(torch.zeros(2, 8), torch.ones(8, dtype=BF16))),
    (TypeError, "one dtype", lambda: mega_layer_norm(torch.zeros(2, 8, dtype=BF16), torch.ones(8), torch.ones(8, dtype=BF16))),
    (ValueError, "eps must be", lambda: mega_layer_norm(torch.zeros(2, 8), eps=-1.0)),
    (ValueError, "eps must be", lambda: mega_layer_norm(torch.zeros(2, 8), eps=math.nan)),
    (TypeError, "require CUDA", lambda: mega_layer_norm(torch.zeros(2, 8))),
    (ValueError, "hidden_size", lambda: MegaLayerNorm(0)),
    (ValueError, "eps", lambda: MegaRmsNorm(8, eps=math.inf)),
])
def test_norm_refusals(error, match, call):
    with pytest.raises(error, match=match):
        call()


def _loss(x=(4, 16), w=(10, 16), t=(4,), x_dtype=BF16, w_dtype=BF16, t_dtype=torch.int64, **options):
    return mega_cross_entropy(torch.zeros(x, dtype=x_dtype), torch.zeros(w, dtype=w_dtype), torch.zeros(t, dtype=t_dtype), **options)


@pytest.mark.parametrize("error,match,call", [
    (TypeError, "targets must be a Tensor", lambda: mega_cross_entropy(torch.zeros(1, 8), torch.zeros(2, 8), 1)),
    (ValueError, "reduction", lambda: _loss(reduction="average")),
    (ValueError, "recompute", lambda: _loss(recompute=1)),
    (ValueError, "recompute", lambda: MegaCrossEntropy(16, 10, recompute=None)),
    (ValueError, "ignore_index", lambda: _loss(ignore_index=1.5)),
    (ValueError, "ignore_index", lambda: _loss(ignore_index=1 << 63)),
    (ValueError, "multiple of 8", lambda: _loss(x=(4, 12), w=(10, 12))),
    (ValueError, "weight must be", lambda: _loss(w=(10, 2, 16))),
    (ValueError, "weight must be", lambda: _loss(w=(0, 16))),
    (ValueError, "hidden must end", lambda: _loss(x=(4, 24))),
    (ValueError, "targets must have shape", lambda: _loss(t=(5,))),
    (ValueError, "targets must have shape", lambda: _loss(x=(2, 2, 16))),
    (TypeError, "must be BF16", lambda: _loss(x_dtype=torch.float32)),
    (TypeError, "must be BF16", lambda: _loss(w_dtype=torch.float16)),
    (TypeError, "INT32 or INT64", lambda: _loss(t_dtype=torch.int16)),
    (TypeError, "requires CUDA", _loss),
    (ValueError, "multiple of 8", lambda: MegaCrossEntropy(12, 10)),
    (ValueError, "vocab_size", lambda: MegaCrossEntropy(16, 0)),
    (ValueError, "reduction", lambda: MegaCrossEntropy(16, 10, reduction="")),
    (ValueError, "bias", lambda: MegaCrossEntropy.from_module(torch.nn.Linear(16, 10, dtype=BF16))),
    (ValueError, "BF16 weight", lambda: MegaCrossEntropy.from_module(torch.nn.Linear(16, 10, bias=False))),
])
def test_loss_refusals(error, match, call):
    with pytest.raises(error, match=match):
        call()


def test_c_entries_refuse_without_touching_a_device():
    lib = _lib.load()
    buffer = (ctypes.c_char * 4096)()
    at = (ctypes.addressof(buffer) + 255) // 256 * 256

    def refused(code, text):
        assert code == -1 and text in lib.hmc_last_error(), lib.hmc_last_error()

    norm = lambda **c: lib.hmc_row_norm(*{**dict(  # noqa: E731
        x=at, xs=8, rows=2, hidden=8, dtype=0, w=None, b=None, adt=0, center=1, eps=1e-6, y=at, mean=None, rstd=None,
        stream=None), **c}.values())
    refused(norm(rows=-1), b"rows")
    refused(norm(rows=(1 << 31) - 1), b"rows")
    refused(norm(hidden=0), b"hidden")
    refused(norm(hidden=(1 << 20) + 1), b"hidden")
    refused(norm(dtype=3), b"dtype")
    refused(norm(adt=1), b"parameters")
    refused(norm(x=None), b"null")
    refused(norm(eps=-1.0), b"eps")
    refused(norm(xs=-8), b"strides")
    refused(norm(center=0, b=at), b"neither bias")
    refused(norm(rstd=at), b"together")
    grad = lambda **c: lib.hmc_row_norm_grad(*{**dict(  # noqa: E731
        x=at, xs=8, g=at, gs=8, rows=2, hidden=8, dtype=0, w=None, adt=0, center=1, mean=at, rstd=at, gx=at, gw=at, gb=None,
        ws=at, wb=1 << 40, stream=None), **c}.values())
    refused(grad(wb=0), b"workspace")
    refused(grad(ws=at + 4), b"workspace")
    refused(grad(mean=None), b"null")
    refused(grad(center=0, gb=at), b"no bias")
    loss = lambda **c: lib.hmc_vocab_loss(*{**dict(  # noqa: E731
        x=at, xs=16, w=at, ws=16, t=at, wide=1, tokens=4, hidden=16, vocab=10, ignored=-100, red=1, keep=1, state=at, loss=at, space=at,
        sb=1 << 40, status=None, stream=None), **c}.values())
    refused(loss(tokens=0), b"tokens")
    refused(loss(vocab=0), b"vocab")
    refused(loss(hidden=12, ws=16), b"multiple of 8")
    refused(loss(ws=12), b"weight rows")
    refused(loss(ws=8), b"weight rows")
    refused(loss(w=at + 2), b"weight rows")
    refused(loss(red=3), b"reduction")
    refused(loss(t=None), b"null")
    refused(loss(sb=8), b"workspace")
    refused(loss(state=at + 8), b"boundaries")
    back = lambda **c: lib.hmc_vocab_loss_grad(*{**dict(  # noqa: E731
        state=at, w=at, ws=16, tokens=4, hidden=16, vocab=10, red=1, keep=1, g=at, gh=at, gw=at, space=at, sb=1 << 40, status=None,
        stream=None), **c}.values())
    refused(back(g=None), b"null")
    refused(back(gh=at + 2), b"aligned")
    refused(back(sb=8), b"workspace")
    assert back(gh=None, gw=None) == 0  # nothing asked for


def test_workspaces_hold_every_smaller_call():
    lib = _lib.load()
    for hidden in (1, 64, 4096):
        sizes = [lib.hmc_row_norm_grad_workspace_bytes(rows, hidden) for rows in [*range(1, 700), 4096, 16384]]
        assert sizes == sorted(sizes)
    for vocab in (1, 50257, 131072):
        for size in (lambda t, v=vocab: lib.hmc_vocab_loss_workspace_bytes(t, v), lambda t, v=vocab: lib.hmc_vocab_loss_state_bytes(t, 64, v, 0)):
            sizes = [size(t) for t in (1, 2, 255, 256, 257, 4096, 8192, 65536)]
            assert sizes == sorted(sizes)
        # kept logits: none up to 128 tokens, 4 GiB and a 64th of it at the most
        for tokens in (1, 128, 129, 4096, 20_000, 65536, 1 << 20):
            held = lib.hmc_vocab_loss_state_bytes(tokens, 64, vocab, 1) - lib.hmc_vocab_loss_state_bytes(tokens, 64, vocab, 0)
            assert (held == 0) if tokens <= 128 else (0 <= held <= (4 << 30) * 65 // 64 + 256)
            assert tokens > 4096 or tokens <= 128 or held > 2 * tokens * vocab
    # probabilities of a piece: half a GiB, and no fewer than 4096 words
    assert lib.hmc_vocab_loss_grad_workspace_bytes(8192, 8, 1 << 20) < 600 << 20


def test_modules_move_between_types_and_devices():
    norm = MegaLayerNorm(16, device="meta").to_empty(device="cpu")
    assert norm.weight.dtype == BF16 and norm.bias.shape == (16,) and MegaLayerNorm(16, bias=False).bias is None
    head = MegaCrossEntropy(16, 10)
    assert head.weight.shape == (10, 16) and head.weight.dtype == BF16 and list(head.state_dict()) == ["weight"]
