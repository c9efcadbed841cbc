"""
Root-mean-square norm with the residual's addition, on HIP kernels: in training with its backward, in serving with its result also
in microscaled values, which the products with quantised expert weights read. The reference has no counterpart on this path.
"""

import torch
from torch.autograd.function import once_differentiable

from fast_llm_amd import _lib
from fast_llm_amd.functional.microscaling import MicroscaledTensor, MicroscalingFormat, _tag
from fast_llm_amd.functional.utils import Assert, refuse_traced, without_backward


def _check(input_: torch.Tensor, weight: torch.Tensor, residual: torch.Tensor | None) -> None:
    assert weight.dim() == 1 and weight.size(0) == input_.size(-1) > 0, (weight.shape, input_.shape)
    if weight.dtype != input_.dtype and weight.dtype != torch.float32:
        raise ValueError(f"the weight has the input's type ({input_.dtype}) or float32, not {weight.dtype}")
    if residual is not None:
        Assert.eq(residual.shape, input_.shape)
        Assert.eq(residual.dtype, input_.dtype)


def _forward(
    input_: torch.Tensor, weight: torch.Tensor, residual: torch.Tensor | None, eps: float, quantized: MicroscaledTensor | None
) -> tuple[torch.Tensor, torch.Tensor]:
    """The normalised rows and the stream (the input itself without a residual)."""
    input_, weight = input_.contiguous(), weight.contiguous()
    normalized, stream = torch.empty_like(input_), None
    if residual is not None:
        residual, stream = residual.contiguous(), torch.empty_like(input_)
    device = _lib.require_device(input_, weight, residual)
    columns = input_.size(-1)
    _lib.call(
        "fm_rms_norm_forward", device, input_.data_ptr(), _lib.ptr(residual), weight.data_ptr(), _lib.ptr(stream),
        normalized.data_ptr(), None if quantized is None else quantized.values.data_ptr(),
        None if quantized is None else quantized.scales.data_ptr(), input_.numel() // columns, columns, eps,
        _lib.dtype_tag(input_.dtype), _lib.dtype_tag(weight.dtype), 0 if quantized is None else _tag(quantized.format),
    )  # fmt: skip
    return normalized, input_ if stream is None else stream


class _RMSNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, input_: torch.Tensor, weight: torch.Tensor, residual: torch.Tensor | None, eps: float):
        normalized, stream = _forward(input_, weight, residual, eps, None)
        ctx.save_for_backward(stream, weight)
        ctx.eps = eps
        ctx.set_materialize_grads(False)
        return normalized if residual is None else (normalized, stream)

    @staticmethod
    def backward(ctx, *grads: torch.Tensor | None):
        # Without the guard where no graph of the gradients is made: in small steps its host time counts.
        return (_backward_once if torch.is_grad_enabled() else _backward)(ctx, *grads)


def _backward(ctx, grad_normalized: torch.Tensor | None, grad_stream: torch.Tensor | None = None):
    stream, weight = ctx.saved_tensors
    _, needs_weight, needs_residual, _ = ctx.needs_input_grad
    if grad_normalized is None:
        # Nothing depends on the norm.
        return grad_stream, torch.zeros_like(weight) if needs_weight else None, grad_stream if needs_residual else None, None
    grad_normalized, weight = grad_normalized.contiguous(), weight.contiguous()
    if grad_stream is not None:
        grad_stream = grad_stream.contiguous()
    grad_input, grad_weight, workspace, size = torch.empty_like(stream), None, None, 0
    columns = weight.size(0)
    rows = stream.numel() // columns
    device = _lib.require_device(grad_normalized, grad_stream, stream, weight)
    if needs_weight:
        grad_weight = torch.empty_like(weight)
        size = _lib.lib().fm_rms_norm_backward_workspace_size(rows, columns)
        workspace = torch.empty(size, dtype=torch.uint8, device=device)
    _lib.call(
        "fm_rms_norm_backward", device, grad_normalized.data_ptr(), _lib.ptr(grad_stream), stream.data_ptr(),
        weight.data_ptr(), grad_input.data_ptr(), _lib.ptr(grad_weight), rows, columns, ctx.eps,
        _lib.dtype_tag(stream.dtype), _lib.dtype_tag(weight.dtype), _lib.ptr(workspace), size,
    )  # fmt: skip
    return grad_input, grad_weight, grad_input if needs_residual else None, None


_backward_once = once_differentiable(_backward)


def rms_norm(
    input_: torch.Tensor, weight: torch.Tensor, residual: torch.Tensor | None = None, eps: float = 1e-5
) -> torch.Tensor | tuple[torch.Tensor, torch.Tensor]:
    """
    stream = input_ + residual (rounded to their type; `input_` itself without one),
    normalized = stream / sqrt(mean(stream^2) + eps) * weight, over the last axis. Returns `normalized`, with a residual
    (`normalized`, `stream`). Differentiable (once) in `input_`, `weight` and `residual`; `weight` has the input's type or float32.
    Squares are summed in fp32: rows with values from 1.8e19 / sqrt(columns) on, whose sum overflows, become zeros.
    Rows of any length and alignment; can be captured into a graph, its backward while no eager graph of the same leaves is alive.
    """
    _check(input_, weight, residual)
    return _RMSNorm.apply(input_, weight, residual, eps)


def rms_norm_quantize(
    input_: torch.Tensor,
    weight: torch.Tensor,
    residual: torch.Tensor | None = None,
    eps: float = 1e-5,
    format: MicroscalingFormat | str = MicroscalingFormat.e4m3,
) -> tuple[torch.Tensor, torch.Tensor, MicroscaledTensor]:
    """
    `rms_norm` for inference: (`normalized`, `stream`, `mx_quantize(normalized, format)`) in one pass, bit for bit what the single
    calls give. Without a residual the stream is `input_`. No backward, no forward-mode derivative, not for `torch.jit`'s tracer.
    """
    refuse_traced(input_, weight, residual)
    _check(input_, weight, residual)
    columns = input_.size(-1)
    quantized = MicroscaledTensor.empty(input_.numel() // columns, columns, format, input_.device)
    normalized, stream = _forward(input_, weight, residual, eps, quantized)
    if torch.is_grad_enabled() and (input_.requires_grad or weight.requires_grad or (residual is not None and residual.requires_grad)):
        normalized, stream = without_backward(normalized), without_backward(stream)
    return normalized, stream, quantized
