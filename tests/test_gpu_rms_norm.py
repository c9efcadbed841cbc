"""The root-mean-square norm with the residual's addition, forward, backward and microscaled, against the oracle in 64 bits."""

import pytest
import torch

from fast_llm_amd.functional.microscaling import mx_quantize
from fast_llm_amd.functional.normalization import rms_norm, rms_norm_quantize
from fast_llm_amd.layers.normalization import RMSNorm
from oracle import mx_oracle

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
# A wavefront per row, 4 and 16 of them, with one, two and four vectors per lane, at the ends of each; odd lengths and one past the
# longest that registers hold (a value per load); rows alone, and more than the workgroups of a backward take at once.
SHAPES = [(1, 8), (3, 512), (5, 520), (9, 1032), (2, 2048), (1, 2056), (3, 4096), (2, 8192), (2, 8200), (1, 32768), (2, 1), (7, 33), (3, 1001),
          (1, 32776), (2100, 64), (600, 2064)]  # fmt: skip


def _inputs(rows, columns, dtype, weight_dtype, device, seed=0):
    generator = torch.Generator().manual_seed(seed + rows + columns)
    sizes = torch.exp(torch.randn(columns, generator=generator))
    x, residual = ((torch.randn(rows, columns, generator=generator) * sizes).to(dtype) for _ in range(2))
    weight = (1 + 0.2 * torch.randn(columns, generator=generator)).to(weight_dtype)
    grads = [torch.randn(rows, columns, generator=generator).to(dtype) for _ in range(2)]
    return x, residual, weight, grads


def _steps(columns: int) -> float:
    """Relative error of an fp32 sum over a row's columns as it is added up, in half steps of fp32: up to 32 or columns / 256 values one after the
    other in a lane, 6 levels of lanes, up to 16 wavefronts."""
    return max(32, columns / 256) + 6 + 16


@pytest.mark.parametrize(("rows", "columns"), SHAPES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("weight_f32", [False, True])
@pytest.mark.parametrize("with_residual", [False, True])
def test_forward_and_microscaled(rows, columns, dtype, weight_f32, with_residual, device):
    x, residual, weight, _ = _inputs(rows, columns, dtype, torch.float32 if weight_f32 else dtype, device)
    residual = residual if with_residual else None
    expected, stream = mx_oracle.rms_norm(x, weight, residual, 1e-5)
    on_gpu = (x.to(device), weight.to(device), None if residual is None else residual.to(device))
    result = rms_norm(*on_gpu)
    normalized = result[0] if with_residual else result
    if with_residual:
        assert torch.equal(result[1].cpu(), stream)
    # Half the sum's error in the root, four more roundings to fp32 on the way, the result's own.
    tolerance = ((_steps(columns) / 2 + 4) * 2.0**-24 + torch.finfo(dtype).eps / 2) * expected.abs() + torch.finfo(dtype).smallest_normal
    assert ((normalized.cpu().double() - expected).abs() <= tolerance).all()
    for format in ("e4m3", "e2m1"):
        again, stream_again, quantized = rms_norm_quantize(*on_gpu, format=format)
        assert torch.equal(again, normalized)
        assert torch.equal(stream_again.cpu(), stream)
        plain = mx_quantize(normalized, format)
        assert torch.equal(quantized.values, plain.values) and torch.equal(quantized.scales, plain.scales)


@pytest.mark.parametrize(("rows", "columns"), SHAPES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("weight_f32", [False, True])
@pytest.mark.parametrize("with_residual", [False, True])
def test_gradients(rows, columns, dtype, weight_f32, with_residual, device):
    x, residual, weight, grads = _inputs(rows, columns, dtype, torch.float32 if weight_f32 else dtype, device)
    leaves = [t.to(device).requires_grad_(True) for t in ((x, weight, residual) if with_residual else (x, weight))]
    result = rms_norm(*leaves)
    outputs = result if with_residual else (result,)
    ours = torch.autograd.grad(outputs, leaves, [g.to(device) for g in grads[: len(outputs)]])
    stream = x if not with_residual else (x.double() + residual.double()).to(dtype)
    grad_stream = grads[1] if with_residual else None
    grad_input, grad_weight = mx_oracle.rms_norm_backward(grads[0], grad_stream, stream, weight, 1e-5)
    wide, g, w = stream.double(), grads[0].double(), weight.double()
    inverse = 1 / torch.sqrt(wide.square().mean(-1, keepdim=True) + 1e-5)
    # Every term's size, with the errors of both sums (three times half of one in the powers of the root) and eight roundings to fp32.
    size = inverse * ((g * w).abs() + wide.abs() * inverse**2 * (g * w * wide).abs().mean(-1, keepdim=True))
    size = size + (grad_stream.double().abs() if with_residual else 0)
    tolerance = (2.5 * _steps(columns) + 8) * 2.0**-24 * size + torch.finfo(dtype).eps / 2 * grad_input.abs() + torch.finfo(dtype).smallest_normal
    assert ((ours[0].cpu().double() - grad_input).abs() <= tolerance).all()
    if with_residual:
        assert torch.equal(ours[2], ours[0])
    # The rows of a workgroup one after the other, then up to 512 parts.
    size = (g * wide * inverse).abs().sum(0)
    steps = rows / 512 + 1 + 4 + 512 / 64 + 6 + _steps(columns) / 2 + 4
    tolerance = steps * 2.0**-24 * size + torch.finfo(weight.dtype).eps / 2 * grad_weight.abs() + torch.finfo(dtype).smallest_normal
    assert ours[1].dtype == weight.dtype
    assert ((ours[1].cpu().double() - grad_weight).abs() <= tolerance).all()


def test_gradients_are_those_of_differences(device):
    x, residual, weight, grads = (t for t in _inputs(4, 200, torch.float32, torch.float32, device))
    leaves = [t.to(device).requires_grad_(True) for t in (x, weight, residual)]
    ours = torch.autograd.grad(rms_norm(*leaves, eps=1e-3), leaves, [g.to(device) for g in grads])

    def loss(x, weight, residual):
        wide = x.double() + residual.double()
        normalized = wide / torch.sqrt(wide.square().mean(-1, keepdim=True) + 1e-3) * weight.double()
        return (normalized * grads[0].double()).sum() + (wide * grads[1].double()).sum()

    originals = [x.double(), weight.double(), residual.double()]
    for which, at in ((0, (0, 3)), (0, (3, 199)), (2, (1, 100)), (1, (7,)), (1, (199,))):
        ends = []
        for sign in (1, -1):
            moved = [t.clone() for t in originals]
            moved[which][at] += sign * 1e-5
            ends.append(loss(*moved))
        # fp32 against differences in 64 bits: 1e-16 * 1e3 / 1e-5 from the subtraction, 2^-24 * 100 of values of order ten.
        assert abs((ends[0] - ends[1]) / 2e-5 - ours[which][at].item()) < 1e-4 * max(1, abs(ours[which][at].item()))


def test_gradients_that_are_not_asked_for_or_do_not_come(device):
    x, residual, weight, grads = _inputs(5, 264, torch.bfloat16, torch.bfloat16, device)
    x, residual, weight = (t.to(device) for t in (x, residual, weight))
    grads = [g.to(device) for g in grads]
    both = [t.detach().requires_grad_(True) for t in (x, weight, residual)]
    full = torch.autograd.grad(rms_norm(*both), both, grads)
    # Only the weight, only the residual.
    only = weight.detach().requires_grad_(True)
    normalized, stream = rms_norm(x, only, residual)
    assert torch.equal(torch.autograd.grad((normalized, stream), only, grads)[0], full[1])
    only = residual.detach().requires_grad_(True)
    assert torch.equal(torch.autograd.grad(rms_norm(x, weight, only), only, grads)[0], full[2])
    # Nothing behind the norm, nothing behind the stream.
    both = [t.detach().requires_grad_(True) for t in (x, weight, residual)]
    _, stream = rms_norm(*both)
    got = torch.autograd.grad(stream, both, grads[1])
    assert torch.equal(got[0], grads[1]) and not got[1].any() and torch.equal(got[2], grads[1])
    normalized, _ = rms_norm(*both)
    got = torch.autograd.grad(normalized, both, grads[0])
    zero = torch.autograd.grad(rms_norm(*both), both, [grads[0], torch.zeros_like(grads[0])])
    assert all(torch.equal(a, b) for a, b in zip(got, zero))
    # The same tensor twice: both gradients.
    leaf = x.detach().requires_grad_(True)
    twice = torch.autograd.grad(rms_norm(leaf, weight, leaf), leaf, grads)[0]
    once = [x.detach().requires_grad_(True), x.detach().requires_grad_(True)]
    parts = torch.autograd.grad(rms_norm(once[0], weight, once[1]), once, grads)
    assert torch.equal(twice, parts[0] + parts[1])
    with pytest.raises(RuntimeError, match="once_differentiable"):
        leaf, grad = x.detach().requires_grad_(True), grads[0].detach().requires_grad_(True)
        torch.autograd.grad(rms_norm(leaf, weight), leaf, grad, create_graph=True)[0].sum().backward()


def test_shapes_strides_and_rows_that_are_special(device):
    weight = torch.randn(96, device=device).bfloat16()
    x = torch.randn(4, 5, 96, device=device).bfloat16()
    flat = rms_norm(x.flatten(0, 1), weight)
    assert torch.equal(rms_norm(x, weight), flat.view_as(x))
    assert torch.equal(rms_norm(x.transpose(0, 1), weight), flat.view_as(x).transpose(0, 1))
    wide = torch.randn(6, 200, device=device).bfloat16()
    view = wide[:, 3:99]  # neither contiguous nor aligned
    assert torch.equal(rms_norm(view, weight), rms_norm(view.contiguous(), weight))
    # Aligned to 2 bytes only: a value per load, the same result up to the order of the sum.
    storage = torch.zeros(5 * 96 + 1, dtype=torch.bfloat16, device=device)
    storage[1:] = x[0].flatten()
    odd = rms_norm(storage[1:].view(5, 96), weight)
    assert ((odd.float() - rms_norm(x[0], weight).float()).abs() <= 2.0**-8 * odd.float().abs()).all()
    assert rms_norm(x[:0], weight).shape == (0, 5, 96)
    empty = rms_norm(x[:0].detach().requires_grad_(True), leaf := weight.detach().requires_grad_(True))
    empty.sum().backward()
    assert not leaf.grad.any()
    special = torch.zeros(4, 96, device=device)
    special[1, 5], special[2, 7], special[3] = float("inf"), float("nan"), 1e30
    got = rms_norm(special, torch.ones(96, device=device), eps=1e-6)
    assert not got[0].any() and got[1, 0] == 0 and torch.isnan(got[1, 5]) and torch.isnan(got[2]).all() and not got[3].any()
    _, _, quantized = rms_norm_quantize(special, torch.ones(96, device=device), eps=1e-6)
    assert quantized.scales[0].tolist() == [0, 0, 0, 0] and quantized.scales[1].tolist() == [255, 0, 0, 0]
    assert quantized.scales[2].tolist() == [255, 255, 255, 0]


def test_quantized_has_no_backward(device):
    x, weight = torch.randn(4, 64, device=device, requires_grad=True), torch.ones(64, device=device)
    normalized, _, _ = rms_norm_quantize(x, weight)
    with pytest.raises(RuntimeError, match="backward"):
        normalized.sum().backward()
    with torch.no_grad():
        assert torch.equal(rms_norm_quantize(x, weight)[0], normalized)


def test_module_and_graph(device):
    norm = RMSNorm(512, eps=1e-4, device=device)
    x, residual = (torch.randn(70, 512, device=device).bfloat16() for _ in range(2))
    assert torch.equal(norm(x), rms_norm(x, norm.weight, eps=1e-4))
    assert all(torch.equal(a, b) for a, b in zip(norm(x, residual), rms_norm(x, norm.weight, residual, 1e-4)))
    static, grads = [x.clone().requires_grad_(True), residual.clone().requires_grad_(True)], [torch.randn_like(x) for _ in range(2)]
    weight = norm.weight.detach().clone().requires_grad_(True)

    def step(x, residual):
        outputs = rms_norm(x, weight, residual)
        return (*(o.detach() for o in outputs), *torch.autograd.grad(outputs, (x, weight, residual), grads))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*static)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step(*static)
    for _ in range(3):
        new = [torch.randn_like(x) for _ in range(2)]
        with torch.no_grad():
            for target, source in zip(static, new):
                target.copy_(source)
        graph.replay()
        eager = step(*(t.clone().requires_grad_(True) for t in new))
        assert all(torch.equal(a, b) for a, b in zip(captured, eager))
        torch.cuda.synchronize()


@pytest.mark.parametrize(("rows", "columns"), [((1 << 26) + 5, 8), ((1 << 24) + 3, 3)])
def test_more_rows_than_a_launch_counts_threads(rows, columns, device):
    x = torch.randn(1 << 16, columns, device=device, dtype=torch.float16).repeat(rows // (1 << 16) + 1, 1)[:rows]
    weight = torch.randn(columns, device=device, dtype=torch.float16)
    first, _, quantized = rms_norm_quantize(x[: 1 << 16], weight)
    normalized, _, values = rms_norm_quantize(x, weight)
    for start in range(0, rows, 1 << 22):
        end = min(start + (1 << 22), rows)
        assert torch.equal(normalized[start:end], first.repeat(64, 1)[: end - start])
        assert torch.equal(values.values[start:end], quantized.values.repeat(64, 1)[: end - start])
        assert torch.equal(values.scales[start:end], quantized.scales.repeat(64, 1)[: end - start])


@pytest.mark.parametrize("columns", [9, 100, 513, 1027, 2044, 2049, 4091, 8190, 8194, 32763])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("offset", [0, 1])
def test_rows_of_any_length_and_alignment(columns, dtype, offset, device):
    """What a row's last lane shares with the lane before it counts once, and is written once or with the same value; nothing else is written."""
    rows = 7
    x, residual, weight, grads = _inputs(rows, columns, dtype, dtype, device)

    def placed(values):
        storage = torch.full((values.numel() + 16,), 3.0, dtype=dtype, device=device)
        view = storage[offset : offset + values.numel()].view(values.shape)
        view.copy_(values)
        return view

    leaves = [placed(t).requires_grad_(True) for t in (x, residual, weight)]
    normalized, stream = rms_norm(leaves[0], leaves[2], leaves[1])
    expected, expected_stream = mx_oracle.rms_norm(x, weight, residual, 1e-5)
    assert torch.equal(stream.cpu(), expected_stream)
    tolerance = ((_steps(columns) / 2 + 4) * 2.0**-24 + torch.finfo(dtype).eps / 2) * expected.abs() + torch.finfo(dtype).smallest_normal
    assert ((normalized.cpu().double() - expected).abs() <= tolerance).all()
    # Placed or not: the same kernel's bits, or those of the one for whole vectors up to the order of a sum.
    grad_input, grad_residual, grad_weight = torch.autograd.grad((normalized, stream), leaves, [placed(g) for g in grads])
    assert torch.equal(grad_input, grad_residual)
    plain = [t.to(device).requires_grad_(True) for t in (x, residual, weight)]
    results = torch.autograd.grad(rms_norm(plain[0], plain[2], plain[1]), plain, [g.to(device) for g in grads])
    wide_grad, wide_weight = mx_oracle.rms_norm_backward(grads[0], grads[1], expected_stream, weight, 1e-5)
    for ours, theirs, wide in ((grad_input, results[0], wide_grad), (grad_weight, results[2], wide_weight)):
        # Sums of either order are off by a few steps of fp32 of the largest of their terms, results by half a step each.
        slack = 2.0**-12 * wide.abs().max() if dtype == torch.float32 else 2 * torch.finfo(dtype).eps * wide.abs().max()
        assert (ours.double().cpu() - wide).abs().max() <= slack and (ours - theirs).double().abs().max().cpu() <= slack
    _, _, quantized = rms_norm_quantize(leaves[0].detach(), leaves[2].detach(), leaves[1].detach())
    reference = mx_quantize(normalized)
    assert torch.equal(quantized.values, reference.values) and torch.equal(quantized.scales, reference.scales)
