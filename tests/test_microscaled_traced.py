"""What the operators on microscaled values compute is outside autograd and its tracers: they refuse what would lose a tangent or a result silently."""

import pytest
import torch
from torch.autograd import forward_ad

from fast_llm_amd.functional.microscaling import MicroscaledTensor, mx_mlp, mx_quantize
from fast_llm_amd.functional.normalization import rms_norm_quantize

X, WEIGHT = torch.randn(4, 64), torch.ones(64)
SCORES, TOP_EXPERTS = torch.ones(4, 1), torch.zeros(4, 1, dtype=torch.int64)


def _mlp(x, scores):
    weights = [MicroscaledTensor.empty(rows, 64, "e2m1", X.device) for rows in (128, 64)]
    return mx_mlp(x, scores, TOP_EXPERTS, *weights, 1, gated=True, activation_type="silu")


# The function and its arguments, of which any may carry a tangent.
CALLS = {
    "quantize": (lambda x: mx_quantize(x).values, (X,)),
    "norm": (lambda x, weight, residual: rms_norm_quantize(x, weight, residual)[0], (X, WEIGHT, X)),
    "norm_without_residual": (lambda x, weight: rms_norm_quantize(x, weight)[0], (X, WEIGHT)),
    "mlp": (_mlp, (X, SCORES)),
    "mlp_of_rows": (lambda scores: _mlp(MicroscaledTensor.empty(4, 64, "e4m3", X.device), scores), (SCORES,)),
}


@pytest.mark.parametrize("name", CALLS)
def test_tangents_are_refused(name):
    function, arguments = CALLS[name]
    with forward_ad.dual_level():
        for which in range(len(arguments)):
            dual = list(arguments)
            dual[which] = forward_ad.make_dual(dual[which], torch.ones_like(dual[which]))
            with pytest.raises(NotImplementedError, match="forward-mode"):
                function(*dual)
        with pytest.raises(RuntimeError, match="GPU only"):  # what carries none goes on
            function(*arguments)


@pytest.mark.parametrize("name", CALLS)
def test_the_tracer_is_refused(name):
    function, arguments = CALLS[name]
    with pytest.raises(NotImplementedError, match="tracer"):
        torch.jit.trace(function, arguments, check_trace=False)
