"""The layer on microscaled expert weights: the operators as they are used, one after the other."""

import pytest
import torch

from fast_llm_amd.functional.microscaling import mx_mlp, mx_quantize_expert_weights
from fast_llm_amd.functional.normalization import rms_norm_quantize
from fast_llm_amd.layers.moe import DroplessMoEMLP, MicroscaledMoEMLP
from fast_llm_amd.layers.normalization import RMSNorm

pytestmark = pytest.mark.gpu


def _layer(device, **options):
    torch.manual_seed(0)
    return DroplessMoEMLP(512, 640, 8, 2, device=device, **options).eval()


@pytest.mark.parametrize("format", ["e4m3", "e2m1"])
@pytest.mark.parametrize("tokens", [1, 40, 2000])
@pytest.mark.parametrize("options", [{}, {"shared_experts": 1, "gated": False}, {"router_input_scale": 0.5, "router_per_expert_scale": True}], ids=str)
def test_layer_is_its_operators_one_after_the_other(format, tokens, options, device):
    layer, norm = _layer(device, **options), RMSNorm(512, device=device)
    with torch.no_grad():
        norm.weight.normal_(1, 0.1)
    quantized = MicroscaledMoEMLP(layer, norm, format=format)
    x, residual = (torch.randn(tokens, 512, device=device).bfloat16() for _ in range(2))
    output, stream = quantized(x, residual)
    with torch.no_grad():
        normalized, expected_stream, rows = rms_norm_quantize(x, norm.weight, residual, norm.eps, format)
        scores, top_experts = layer.route(normalized)
        weights = mx_quantize_expert_weights(layer.layer_1, layer.layer_2, layer.experts)
        expected = mx_mlp(rows, scores, top_experts, *weights, layer.experts, gated=layer.gated, activation_type=layer.activation, dtype=x.dtype)
    assert torch.equal(stream, expected_stream) and torch.equal(output, expected)
    assert torch.equal(stream, x + residual)
    # Against the layer in 16 bits: weights with a relative step of up to a half and saturation up to a quarter; both formats are far under the norm
    # of the output itself, and uncorrelated results would be sqrt(2) of it apart.
    with torch.no_grad():
        full = layer(normalized)
    assert (output.double() - full.double()).norm() < 0.5 * full.double().norm()


def test_layer_without_a_norm_and_with_a_routing_of_the_callers_own(device):
    layer = _layer(device)
    quantized = MicroscaledMoEMLP(layer)
    x = torch.randn(3, 7, 512, device=device).bfloat16()
    output = quantized(x)
    assert output.shape == x.shape and not output.requires_grad
    with torch.no_grad():
        scores, top_experts = layer.route(x.flatten(0, 1))
    assert torch.equal(quantized(x, scores=scores, top_experts=top_experts), output)
    with pytest.raises(ValueError, match="residual"):
        quantized(x, x)
    with pytest.raises(RuntimeError, match="inference"):
        quantized.train()
    with pytest.raises(ValueError, match="no tokens"):  # as the layer itself
        quantized(x[:0])


def test_layer_keeps_no_16_bit_expert_weights_and_leaves_its_source_alone(device):
    layer = _layer(device, router_normalization=torch.nn.LayerNorm(512, device=device, dtype=torch.bfloat16)).train()
    quantized = MicroscaledMoEMLP(layer, RMSNorm(512, device=device))
    assert layer.training and layer.router_normalization.training and layer.layer_1.shape == (8 * 2 * 640, 512)
    state = quantized.state_dict()
    largest = 8 * 2 * 640 * 512 // 2
    assert max(t.numel() * t.element_size() for t in state.values()) == largest
    x = torch.randn(5, 512, device=device).bfloat16()
    output = quantized(x)
    with torch.no_grad():
        layer.router.zero_()
    assert all(torch.equal(a, b) for a, b in zip(quantized(x), output))  # a snapshot
    other = MicroscaledMoEMLP(_layer(device, router_normalization=torch.nn.LayerNorm(512, device=device, dtype=torch.bfloat16)), RMSNorm(512, device=device))
    for buffer in other.buffers():
        buffer.zero_()
    other.load_state_dict(state)
    assert all(torch.equal(a, b) for a, b in zip(other(x), output))


def test_router_normalization_by_the_module_trains(device):
    layer = _layer(device, router_normalization=RMSNorm(512, device=device)).train()
    x = torch.randn(40, 512, device=device).bfloat16().requires_grad_(True)
    layer(x, grad_scale=1.0).sum().backward()
    weight = layer.router_normalization.weight
    assert weight.grad is not None and weight.grad.any() and x.grad.any()


@pytest.mark.parametrize("tokens", [1, 700])
def test_layer_replays_from_a_graph(tokens, device):
    quantized = MicroscaledMoEMLP(_layer(device), RMSNorm(512, device=device))
    inputs = [[torch.randn(tokens, 512, device=device).bfloat16() for _ in range(2)] for _ in range(3)]
    eager = [quantized(*pair) for pair in inputs]
    static = [t.clone() for t in inputs[0]]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = quantized(*static)
    for _ in range(2):
        for pair, expected in zip(inputs, eager):
            for target, source in zip(static, pair):
                target.copy_(source)
            graph.replay()
            assert all(torch.equal(a, b) for a, b in zip(captured, expected))
            torch.cuda.synchronize()
