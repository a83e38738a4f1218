"""GPU: layer norm and RMSNorm of rows and their gradients against the definition in 64 bits.

Tolerances. `half` is half a step of the output's type. The FP32 sums of a row are chains of at most 32 values per
thread, 5 shuffles and 32 warps (long rows: a thread's share, 64 at the sizes used here), a column's of the rows of a
block, 8 slices and 37 partial sums: fewer than 128 additions each, every one off by at most 2^-24 of the sum of
magnitudes. A unit value u = (x - mean) rstd inherits the mean's error times rstd, so it is off by 128 * 2^-24 of
`spread` (1 + |u|) with spread = 1 + rstd mean|x|; 256 covers the few operations after it."""

import pytest
import torch

pytestmark = pytest.mark.gpu

STEP = 2.0 ** -24
CHAIN = 256 * STEP


def make(tokens, hidden, dtype, affine, center, seed=0, offset=0.3):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(tokens, hidden, generator=g) * (0.5 + torch.rand(tokens, 1, generator=g) * 3) + offset).to(dtype)
    weight = (1 + 0.2 * torch.randn(hidden, generator=g)).to(affine)
    bias = (0.2 * torch.randn(hidden, generator=g)).to(affine) if center else None
    grad = torch.randn(tokens, hidden, generator=g).to(dtype)
    return [t.cuda() if t is not None else None for t in (x, weight, bias, grad)]


def call(x, weight, bias, center, eps):
    from hyper_multicore_b200 import mega_layer_norm, mega_rms_norm

    return mega_layer_norm(x, weight, bias, eps=eps) if center else mega_rms_norm(x, weight, eps=eps)


def definition(x, weight, bias, center, eps):
    x = x.double()
    mean = x.mean(-1, keepdim=True) if center else torch.zeros_like(x[..., :1])
    rstd = 1 / torch.sqrt(((x - mean) ** 2).mean(-1, keepdim=True) + eps)
    u = (x - mean) * rstd
    y = u if weight is None else u * weight.double()
    return (y if bias is None else y + bias.double()), u, rstd


def check(y, grads, x, weight, bias, grad, center, eps):
    """Every value of the output and of the three gradients within its bound."""
    def inside(name, got, want, bound):
        half = torch.finfo(got.dtype).eps / 2
        tiny = torch.finfo(got.dtype).smallest_normal
        off = (got.double() - want).abs() - half * want.abs() - bound - tiny
        assert off.max().item() <= 0, f"{name}: {off.max().item():.3e} beyond the bound at {off.argmax().item()}"

    want, u, rstd = definition(x, weight, bias, center, eps)
    w = torch.ones(x.shape[-1], dtype=torch.float64, device=x.device) if weight is None else weight.double()
    spread = 1 + (rstd * x.double().abs().mean(-1, keepdim=True) if center else 0)
    size = (1 + u.abs()) * spread
    inside("y", y, want, CHAIN * (size * w.abs() + (0 if bias is None else bias.double().abs())))
    if grads is None:
        return
    g, d = grad.double() * w, grad.double()
    along = (g * u).mean(-1, keepdim=True)
    grad_x = g - u * along - (g.mean(-1, keepdim=True) if center else 0)
    inside("grad_x", grads[0], rstd * grad_x, CHAIN * rstd * (g.abs() * spread + size * (g.abs() * size).mean(-1, keepdim=True)))
    if weight is not None:
        inside("grad_weight", grads[1], (d * u).sum(0), CHAIN * (d.abs() * size).sum(0))
    if bias is not None:
        inside("grad_bias", grads[2], d.sum(0), CHAIN * d.abs().sum(0))


def run(x, weight, bias, grad, center, eps=1e-6):
    leaves = [t.detach().requires_grad_(True) for t in (x, weight, bias) if t is not None]
    it = iter(leaves)
    args = [next(it) if t is not None else None for t in (x, weight, bias)]
    y = call(*args, center, eps)
    found = dict(zip((i for i, t in enumerate(args) if t is not None), torch.autograd.grad(y, leaves, grad)))
    return y.detach(), [found.get(i) for i in range(3)]


TYPES = [(torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32), (torch.float16, torch.float16),
         (torch.float16, torch.float32), (torch.float32, torch.float32)]
SIZES = [(1, 1), (3, 7), (5, 8), (700, 40), (2, 64), (33, 1000), (17, 1001), (1, 1024), (6, 1032), (300, 2560), (3, 4096),
         (5, 4097), (9, 7168), (2, 8192), (3, 9000),
         (2, 16384), (2, 33000)]


@pytest.mark.parametrize("center", [True, False])
@pytest.mark.parametrize("dtype,affine", TYPES)
@pytest.mark.parametrize("tokens,hidden", SIZES)
def test_norm_and_gradients_match_the_definition(tokens, hidden, dtype, affine, center):
    x, weight, bias, grad = make(tokens, hidden, dtype, affine, center, seed=tokens * 31 + hidden)
    y, grads = run(x, weight, bias, grad, center)
    assert y.dtype == dtype and grads[0].dtype == dtype and grads[1].dtype == affine
    check(y, grads, x, weight, bias, grad, center, 1e-6)
    assert torch.equal(call(x, weight, bias, center, 1e-6), y), "the forward that keeps nothing gives other bits"


@pytest.mark.parametrize("center", [True, False])
@pytest.mark.parametrize("tokens,hidden,dtype", [
    (5000, 768, torch.bfloat16), (3000, 300, torch.bfloat16), (1501, 1001, torch.bfloat16), (1501, 1002, torch.float16),
    (777, 3001, torch.float32), (900, 1536, torch.float16), (700, 3584, torch.bfloat16), (600, 5120, torch.float32),
    (601, 8192, torch.bfloat16), (320, 12288, torch.bfloat16), (320, 9216, torch.float32), (500, 6145, torch.bfloat16)])
def test_many_rows_and_their_parameter_gradients(center, tokens, hidden, dtype):
    x, weight, bias, grad = make(tokens, hidden, dtype, torch.float32, center, seed=3)
    y, grads = run(x, weight, bias, grad, center)
    check(y, grads, x, weight, bias, grad, center, 1e-6)
    again = run(x, weight, bias, grad, center)
    assert torch.equal(again[0], y) and all(torch.equal(a, b) for a, b in zip(again[1], grads) if a is not None)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_offset_far_from_zero_costs_no_digits(dtype):
    """Rows around 1000 with a spread of one: the variance of the differences, not a difference of large squares."""
    x, weight, bias, grad = make(37, 2048, dtype, torch.float32, True, seed=5, offset=1000.0)
    y, grads = run(x, weight, bias, grad, True)
    check(y, grads, x, weight, bias, grad, True, 1e-6)


@pytest.mark.parametrize("center", [True, False])
def test_parameters_may_be_absent(center):
    x, weight, bias, grad = make(11, 520, torch.bfloat16, torch.bfloat16, center, seed=7)
    y, grads = run(x, None, None, grad, center)
    check(y, grads, x, None, None, grad, center, 1e-6)
    if center:
        for w, b in ((weight, None), (None, bias)):
            y, grads = run(x, w, b, grad, True)
            check(y, grads, x, w, b, grad, True, 1e-6)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_strides_alignment_and_batches(dtype):
    base, weight, bias, grad = make(60, 264, dtype, dtype, True, seed=9)
    views = {
        "slice": base[:, 8:256], "slice off the vector boundary": base[:, 3:251], "every other row": base[::2, :248],
        "broadcast row": base[:1, :248].expand(60, 248), "transposed": base[:, :60].t().contiguous().t(),
        "batched": base[:, :248].reshape(3, 4, 5, 248), "permuted batch": base[:, :248].reshape(6, 10, 248).transpose(0, 1),
        "one vector": base[5, :248],
    }
    for name, x in views.items():
        hidden = x.shape[-1]
        for dy in (torch.randn(x.shape, device="cuda").to(dtype), torch.ones((), device="cuda", dtype=dtype).expand(x.shape)):
            y, grads = run(x, weight[:hidden], bias[:hidden], dy, True)
            assert y.shape == x.shape and grads[0].shape == x.shape, name
            rows = x.reshape(-1, hidden)
            check(y.reshape(rows.shape), [grads[0].reshape(rows.shape), *grads[1:]], rows, weight[:hidden], bias[:hidden],
                  dy.reshape(rows.shape), True, 1e-6)
    odd = torch.empty(2 * 248 + 1, device="cuda", dtype=dtype)[1:]  # parameters off the vector boundary, one of them strided
    odd.copy_(weight.repeat(2)[:496])
    y, grads = run(base[:, :248], odd[::2], bias[1:249], grad[:, :248], True)
    check(y, grads, base[:, :248], odd[::2], bias[1:249], grad[:, :248], True, 1e-6)


def test_broadcast_input_gets_the_sum_of_its_rows_gradients():
    from hyper_multicore_b200 import mega_rms_norm

    x = torch.randn(1, 512, device="cuda").requires_grad_(True)
    grad = torch.randn(40, 512, device="cuda")
    (got,) = torch.autograd.grad(mega_rms_norm(x.expand(40, 512)), x, grad)
    x64 = x.detach().double().requires_grad_(True)
    (want,) = torch.autograd.grad(definition(x64.expand(40, 512), None, None, False, 1e-6)[0], x64, grad.double())
    assert (got.double() - want).abs().max() <= CHAIN * 40 * grad.abs().max().item() * 8


def test_gradient_agrees_with_differences_of_the_definition():
    for center in (True, False):
        x, weight, bias, grad = make(7, 333, torch.float32, torch.float32, center, seed=13)
        _, grads = run(x, weight, bias, grad, center)
        g = torch.Generator(device="cuda").manual_seed(1)
        for i, leaf in enumerate((x, weight, bias)):
            if leaf is None:
                continue
            direction = torch.randn(leaf.shape, generator=g, device="cuda", dtype=torch.float64)
            step = 1e-5

            def value(sign):
                moved = [t.double() if t is not None else None for t in (x, weight, bias)]
                moved[i] = moved[i] + sign * step * direction
                return (definition(*moved, center, 1e-6)[0] * grad.double()).sum().item()

            slope = (value(1) - value(-1)) / (2 * step)
            got = (grads[i].double() * direction).sum().item()
            # central differences: step^2 and 2^-53 / step, both below 1e-7 of the magnitudes; the FP32 sums decide
            assert abs(got - slope) <= CHAIN * (grads[i].double() * direction).abs().sum().item() * 8 + 1e-6


def test_rows_of_zeros_infinities_and_nan_stay_among_themselves():
    from hyper_multicore_b200 import mega_layer_norm, mega_rms_norm

    x = torch.randn(8, 1024, device="cuda").bfloat16()
    clean = x.clone()
    x[1], x[3, 5], x[4, 7] = 0, float("inf"), float("nan")
    for norm in (mega_layer_norm, mega_rms_norm):
        y, want = norm(x), norm(clean)
        for row in (0, 2, 5, 6, 7):
            assert torch.equal(y[row], want[row])
        assert torch.equal(y[1], torch.zeros_like(y[1])), "a row of zeros is divided by sqrt(eps)"
        assert y[4].isnan().all() and y[3].isnan().any()


def test_no_rows():
    x = torch.empty(0, 64, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    weight = torch.ones(64, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    y = call(x, weight, None, True, 1e-6)
    grad_x, grad_weight = torch.autograd.grad(y, (x, weight), torch.empty_like(y))
    assert y.shape == (0, 64) and grad_x.shape == (0, 64) and torch.equal(grad_weight, torch.zeros_like(grad_weight))


def test_rows_beyond_31_bits_of_elements():
    hidden, tokens = 4096, (1 << 31) // 4096 + 5
    x = torch.randn(64, hidden, device="cuda").bfloat16().repeat(tokens // 64 + 1, 1)[:tokens]
    y, grads = run(x, torch.ones(hidden, device="cuda", dtype=torch.bfloat16), None, x, False)
    for rows in (slice(0, 64), slice(tokens - 64, tokens)):
        check(y[rows], [grads[0][rows], None, None], x[rows], None, None, x[rows], False, 1e-6)


def test_early_started_launches_wait_for_what_they_read():
    """Launches may be placed while the one before them runs: behind a slow copy in their own stream, and behind another stream's."""
    from hyper_multicore_b200 import mega_cross_entropy

    new, weight, bias, grad = make(600, 1024, torch.bfloat16, torch.bfloat16, True, seed=41)
    head = (0.05 * torch.randn(3000, 1024, device="cuda")).bfloat16()
    targets = torch.randint(0, 3000, (600,), device="cuda")
    want = run(new, weight, bias, grad, True)
    want_loss = mega_cross_entropy(new[:64], head, targets[:64], reduction="none")
    x, w = torch.zeros_like(new), torch.zeros_like(head)
    torch.cuda.synchronize()
    torch.cuda._sleep(20_000_000)
    x.copy_(new)
    w.copy_(head)
    loss = mega_cross_entropy(x[:64], w, targets[:64], reduction="none")
    got = run(x, weight, bias, grad, True)
    torch.cuda.synchronize()
    assert torch.equal(loss, want_loss)
    assert torch.equal(got[0], want[0]) and all(torch.equal(a, b) for a, b in zip(got[1], want[1]))
    x.zero_()
    w.zero_()
    torch.cuda.synchronize()
    maker, user = torch.cuda.Stream(), torch.cuda.Stream()
    with torch.cuda.stream(user):
        call(new, weight, bias, True, 1e-6)  # a launch of ours is the last one in the stream
    with torch.cuda.stream(maker):
        torch.cuda._sleep(20_000_000)
        x.copy_(new)
        w.copy_(head)
    user.wait_stream(maker)
    with torch.cuda.stream(user):
        y = call(x, weight, bias, True, 1e-6)
        loss = mega_cross_entropy(x[:64], w, targets[:64], reduction="none")
    torch.cuda.synchronize()
    assert torch.equal(y, want[0]) and torch.equal(loss, want_loss)


@pytest.mark.parametrize("dtype,hidden", [(torch.bfloat16, 2560), (torch.bfloat16, 1001), (torch.bfloat16, 300), (torch.float32, 520)])
def test_nothing_is_written_behind_the_rows(dtype, hidden):
    from hyper_multicore_b200 import _lib

    rows, code = 700, _lib.HMC_DTYPE[dtype]
    x, weight, bias, grad = make(rows, hidden, dtype, dtype, True, seed=hidden)
    want = run(x, weight, bias, grad, True)
    y, dx = (torch.full((rows + 3, hidden), 7.0, device="cuda", dtype=dtype) for _ in range(2))
    mean, rstd = (torch.full((rows + 8,), 7.0, device="cuda") for _ in range(2))
    dw, db = (torch.full((hidden + 8,), 7.0, device="cuda", dtype=dtype) for _ in range(2))
    need = _lib.load().hmc_row_norm_grad_workspace_bytes(rows, hidden)
    space = torch.full((need + 256,), 0x5A, dtype=torch.uint8, device="cuda")
    _lib.launch("hmc_row_norm", x.device, x.data_ptr(), hidden, rows, hidden, code, weight.data_ptr(), bias.data_ptr(), code, 1,
                1e-6, y.data_ptr(), mean.data_ptr(), rstd.data_ptr())
    _lib.launch("hmc_row_norm_grad", x.device, x.data_ptr(), hidden, grad.data_ptr(), hidden, rows, hidden, code, weight.data_ptr(),
                code, 1, mean.data_ptr(), rstd.data_ptr(), dx.data_ptr(), dw.data_ptr(), db.data_ptr(), space.data_ptr(), need)
    assert torch.equal(y[:rows], want[0]) and torch.equal(dx[:rows], want[1][0])
    assert torch.equal(dw[:hidden], want[1][1]) and torch.equal(db[:hidden], want[1][2])
    for guard in (y[rows:], dx[rows:], mean[rows:], rstd[rows:], dw[hidden:], db[hidden:]):
        assert (guard == 7).all()
    assert (space[need:] == 0x5A).all()


def test_first_call_of_a_process_may_be_captured():
    """Shared memory limits and residency are asked for at the first launch of a kernel: that may happen under capture."""
    import subprocess
    import sys
    from pathlib import Path

    code = """
import torch
from hyper_multicore_b200 import mega_cross_entropy, mega_layer_norm
x = torch.randn(700, 2048, device="cuda").bfloat16().requires_grad_(True)
w = torch.randn(1000, 2048, device="cuda").bfloat16().mul_(0.02).requires_grad_(True)
t = torch.randint(0, 1000, (700,), device="cuda")
def step():
    loss = mega_cross_entropy(mega_layer_norm(x), w, t)
    return (loss.detach(), *torch.autograd.grad(loss, (x, w)))
torch.autograd.grad((x * 2).sum(), x)
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    got = step()
graph.replay()
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(got, step()))
"""
    root = Path(__file__).resolve().parent.parent
    subprocess.run([sys.executable, "-c", code], check=True, cwd=root, timeout=300)


def test_order_of_sums_does_not_depend_on_earlier_calls():
    """Two row lengths that share a block size: the second one's bits are those it has in a process of its own."""
    import subprocess
    import sys
    from pathlib import Path

    code = """
import sys, hashlib
import torch
from hyper_multicore_b200 import mega_layer_norm
for hidden in map(int, sys.argv[1:]):
    g = torch.Generator().manual_seed(hidden)
    x, dy = (torch.randn(2000, hidden, generator=g).cuda() for _ in range(2))
    weight, bias = (torch.randn(hidden, generator=g).cuda().requires_grad_(True) for _ in range(2))
    grads = torch.autograd.grad(mega_layer_norm(x, weight, bias), (weight, bias), dy)
print(hashlib.sha256(b"".join(q.cpu().numpy().tobytes() for q in grads)).hexdigest())
"""
    root = Path(__file__).resolve().parents[1]

    def digest(*sizes):
        return subprocess.run([sys.executable, "-c", code, *map(str, sizes)], check=True, cwd=root, timeout=300,
                              capture_output=True, text=True).stdout

    assert digest(1537, 1791) == digest(1791)


def test_the_most_rows_there_may_be():
    """Blocks step through rows in 32 bits: the last step must not run over."""
    from hyper_multicore_b200 import _lib, mega_rms_norm

    rows = _lib.HMC_NORM_MAX_ROWS
    x = torch.ones(1, 8, device="cuda", dtype=torch.bfloat16).expand(rows, 8)
    y = mega_rms_norm(x)
    assert torch.equal(y[-5:], torch.ones(5, 8, device="cuda", dtype=torch.bfloat16)) and y.shape[0] == rows


def test_other_streams_and_captured_graphs():
    x, weight, bias, grad = make(130, 1024, torch.bfloat16, torch.bfloat16, True, seed=17)
    want = run(x, weight, bias, grad, True)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = run(x, weight, bias, grad, True)
    torch.cuda.current_stream().wait_stream(stream)
    assert torch.equal(got[0], want[0]) and all(torch.equal(a, b) for a, b in zip(got[1], want[1]))
    graphs, outputs = [], []
    for _ in range(2):  # two graphs over the same inputs, each with workspaces of its own
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outputs.append(run(x, weight, bias, grad, True))
        graphs.append(graph)
    other, _, _, other_grad = make(130, 1024, torch.bfloat16, torch.bfloat16, True, seed=18)
    x.copy_(other)
    grad.copy_(other_grad)
    for graph in graphs:
        graph.replay()
    torch.cuda.synchronize()
    want = run(other, weight, bias, other_grad, True)
    for got in outputs:
        assert torch.equal(got[0], want[0]) and all(torch.equal(a, b) for a, b in zip(got[1], want[1]))


def test_second_derivatives_and_batched_gradients_are_refused():
    x = torch.randn(4, 64, device="cuda", requires_grad=True)
    y = call(x, None, None, True, 1e-6)
    (first,) = torch.autograd.grad(y.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable|does not require grad"):
        first.sum().backward()
    y = call(x, None, None, True, 1e-6)
    with pytest.raises(RuntimeError, match="batched"):
        torch.autograd.grad(y, x, torch.ones(3, 4, 64, device="cuda"), is_grads_batched=True)


def test_modules_hold_their_parameters():
    from hyper_multicore_b200 import MegaLayerNorm, MegaRmsNorm

    x = torch.randn(3, 5, 256, device="cuda").bfloat16()
    layer, rms = MegaLayerNorm(256, device="cuda"), MegaRmsNorm(256, device="cuda", dtype=torch.float32)
    assert {n for n, _ in layer.named_parameters()} == {"weight", "bias"} and {n for n, _ in rms.named_parameters()} == {"weight"}
    for module, center in ((layer, True), (rms, False)):
        y = module(x)
        y.backward(torch.ones_like(y))
        check(y.detach().reshape(15, 256), None, x.reshape(15, 256), module.weight, getattr(module, "bias", None), None, center,
              module.eps)
        assert all(p.grad is not None for p in module.parameters())
