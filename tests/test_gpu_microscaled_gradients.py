"""The layer on microscaled expert weights has no backward: one that reaches it raises instead of losing its gradient."""

import pytest
import torch

from fast_llm_amd.layers.moe import DroplessMoEMLP, MicroscaledMoEMLP
from fast_llm_amd.layers.normalization import RMSNorm

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tokens", [3, 500])
@pytest.mark.parametrize("with_norm", [False, True])
def test_a_backward_that_reaches_the_layer_raises(tokens, with_norm, device):
    layer = MicroscaledMoEMLP(DroplessMoEMLP(128, 64, 4, 2, device=device), RMSNorm(128, device=device) if with_norm else None)
    x, residual = (torch.randn(tokens, 128, device=device).bfloat16() for _ in range(2))
    scores, top_experts = layer.router.route(x)
    scores, top_experts = scores.detach(), top_experts.detach()
    leaf = x.clone().requires_grad_(True)
    calls = [lambda: layer(leaf), lambda: layer(x, scores=scores.clone().requires_grad_(True), top_experts=top_experts)]
    if with_norm:
        calls += [lambda: layer(leaf, residual), lambda: layer(x, residual.clone().requires_grad_(True))]
    for call in calls:
        results = call()
        for result in results if with_norm else (results,):
            assert result.requires_grad
            with pytest.raises(RuntimeError, match="backward"):
                (leaf + result).sum().backward()  # the residual's way by itself would go through
        with torch.no_grad():
            again = call()
        for result, same in zip(results if with_norm else (results,), again if with_norm else (again,)):
            assert torch.equal(result, same)
        assert not (again[0] if with_norm else again).requires_grad
    results = layer(x, residual) if with_norm else (layer(x),)
    assert not any(result.requires_grad for result in results)
