"""
Values of 8 bits with a scale for each block of 128, and the dropless expert MLP on them, in training and in serving.

128 neighbours along a row share a power of two and are kept in e4m3, as include/fastmoe_hip.h states it. Every product sums along the rows of both
its operands, so that what is summed along another axis is quantised along that axis and kept transposed: the weights in two forms, gradients and
activations in one for the input gradient and one for the weights'. Between forward and backward the MLP keeps 8 bits per value: of its input's
rows, and of the first layer's output, from which the backward has the activation and its slope.

The reference has no counterpart. `block_mlp` has a backward. The operators by themselves have none (what is computed of values in 8 bits needs no
gradient), and refuse forward-mode derivatives and `torch.jit`'s tracer.
"""

import dataclasses
import typing

import torch
from torch.autograd.function import once_differentiable

from fast_llm_amd import _lib
from fast_llm_amd.functional.config import ActivationType
from fast_llm_amd.functional.mlp import _activation_tag
from fast_llm_amd.functional.sparse_copy import (
    SparseMap,
    copy_dense_to_sparse_backward,
    copy_sparse_to_dense,
    copy_sparse_to_dense_backward,
)
from fast_llm_amd.functional.utils import Assert, div, refuse_traced, without_backward
from fast_llm_amd.tensor import param_get_and_unset_is_zero

BLOCK = 128
# Scales of a block column are stored padded to a multiple of this many rows.
_SCALE_ROWS = 16


def _padded(size: int, multiple: int = BLOCK) -> int:
    return -(-size // multiple) * multiple


@dataclasses.dataclass()
class BlockScaledTensor:
    """[rows, columns] values that stand for element * 2^(scale - 127)."""

    # uint8 [rows, columns padded to a multiple of 128]
    values: torch.Tensor
    # uint8 [blocks of 128 columns, rows padded to a multiple of 16]: the scales of all rows' first blocks, then of their second ones ...
    scales: torch.Tensor
    columns: int

    def __post_init__(self):
        # One expression: it runs with every call that a tensor is made for.
        values, scales = self.values, self.scales
        assert (
            self.columns > 0
            and values.dtype == scales.dtype == torch.uint8
            and values.dim() == scales.dim() == 2
            and values.size(1) == _padded(self.columns)
            and scales.size(0) == values.size(1) // BLOCK
            and scales.size(1) == _padded(values.size(0), _SCALE_ROWS)
            and (values.stride(1) == 1 or values.size(0) == 0)
            and (scales.stride(1) == 1 or scales.size(1) == 0)
        ), (values.dtype, values.shape, scales.dtype, scales.shape, self.columns)

    @property
    def rows(self) -> int:
        return self.values.size(0)

    @property
    def shape(self) -> tuple[int, int]:
        return self.values.size(0), self.columns

    @property
    def elements(self) -> torch.Tensor:
        """The elements without their scales [rows, columns], a view."""
        return self.values.view(torch.float8_e4m3fn)[:, : self.columns]

    @property
    def block_scales(self) -> torch.Tensor:
        """The scales [rows, blocks], a view."""
        return self.scales.view(torch.float8_e8m0fnu)[:, : self.values.size(0)].t()

    @classmethod
    def empty(cls, rows: int, columns: int, device: torch.device) -> "BlockScaledTensor":
        assert columns > 0
        # Right by construction: the checks of `__post_init__` take as long as a small launch.
        out = cls.__new__(cls)
        padded = _padded(columns)
        out.columns = columns
        out.values = torch.empty((rows, padded), dtype=torch.uint8, device=device)
        out.scales = torch.empty((padded // BLOCK, _padded(rows, _SCALE_ROWS)), dtype=torch.uint8, device=device)
        return out


class BlockScaledWeights(typing.NamedTuple):
    """
    The expert weights of the sparse MLP in the forms that its products read (`block_quantize_expert_weights`); for inference without those of
    the backward.
    """

    layer_1: BlockScaledTensor  # [experts * ffn (* 2, gates then ups), hidden]: forward
    layer_1_transposed: BlockScaledTensor | None  # [experts * hidden, ffn (* 2)]: input gradient
    layer_2: BlockScaledTensor | None  # [experts * ffn, hidden]: input gradient
    layer_2_transposed: BlockScaledTensor  # [experts * hidden, ffn]: forward


def _pointers(tensor: BlockScaledTensor) -> tuple[int, int]:
    return tensor.values.data_ptr(), tensor.scales.data_ptr()


def _stride(tensor: torch.Tensor) -> int:
    """Bytes between rows; of one row alone, what the next would need."""
    return tensor.stride(0) if tensor.size(0) > 1 else tensor.size(1)


def _strides(tensor: BlockScaledTensor) -> tuple[int, int]:
    return _stride(tensor.values), _stride(tensor.scales)


def _map_pointers(sparse_map: SparseMap | None, rows: int, device: torch.device, aligned: bool = True) -> tuple:
    """(ends, pad begins), experts and the index type of a map of `rows` rows; `aligned`: its experts have to begin at multiples of 128."""
    if sparse_map is None:
        return (None, None), 1, 0
    experts, ends, pad_begins = sparse_map.num_experts, sparse_map.expert_ends, sparse_map.expert_pad_begins
    Assert.eq(rows, sparse_map.num_rows)
    Assert.eq(ends.numel(), pad_begins.numel(), experts)
    Assert.eq(ends.dtype, pad_begins.dtype)
    Assert.eq(ends.device, pad_begins.device, device)
    assert ends.is_contiguous() and pad_begins.is_contiguous()
    if aligned and (rows % BLOCK != 0 or sparse_map.pad_to_multiple % BLOCK != 0):
        raise ValueError(f"the experts' rows have to be padded to multiples of {BLOCK}, not {sparse_map.pad_to_multiple}")
    return (ends.data_ptr(), pad_begins.data_ptr()), experts, _lib.index_tag(ends.dtype)


def _rows_of(input_: torch.Tensor) -> torch.Tensor:
    """The rows of [..., columns], each contiguous."""
    columns = input_.size(-1)
    input_ = input_.detach().reshape(input_.numel() // max(columns, 1), columns)
    return input_ if input_.stride(1) == 1 or columns == 1 else input_.contiguous()


def _quantize(input_: torch.Tensor, groups: int, sparse_map: SparseMap | None, rows: bool, transposed: bool) -> tuple:
    refuse_traced(input_)
    input_ = _rows_of(input_)
    device = _lib.require_device(input_)
    all_rows, columns = input_.shape
    if groups < 1 or (sparse_map is not None and groups != 1):
        raise ValueError(f"{groups} groups" + (" of a sparse layout" if sparse_map is not None else ""))
    group_rows = div(all_rows, groups)
    pointers, experts, index_tag = _map_pointers(sparse_map, all_rows, device)
    along_rows = BlockScaledTensor.empty(all_rows, columns, device) if rows else None
    # (Without rows there is nothing to sum over, and a tensor has a column.)
    along_columns = BlockScaledTensor.empty(groups * columns, max(group_rows, 1), device) if transposed else None
    if transposed and group_rows == 0:
        along_columns.values.zero_(), along_columns.scales.zero_()
    _lib.call(
        "fm_block_quantize", device, input_.data_ptr(), *(_pointers(along_rows) if rows else (None, None)),
        *(_pointers(along_columns) if transposed else (None, None)), *pointers, groups, group_rows, columns, experts,
        input_.stride(0), _stride(along_rows.scales) if rows else 0, _stride(along_columns.scales) if transposed else 0,
        _lib.dtype_tag(input_.dtype), index_tag,
    )  # fmt: skip
    return along_rows, along_columns


def block_quantize(input_: torch.Tensor) -> BlockScaledTensor:
    """
    The rows of `input_` [..., columns] in blocks of 128 along the last axis: scale = the smallest power of two (from 2^-127 on) with
    (largest magnitude) <= 448 * scale, element = value / scale rounded to nearest even. A block with an infinity or NaN is NaN altogether.
    """
    return _quantize(input_, 1, None, True, False)[0]


def block_quantize_transposed(
    input_: torch.Tensor | BlockScaledTensor, *, groups: int = 1, sparse_map: SparseMap | None = None
) -> BlockScaledTensor:
    """
    `groups` matrices one after the other [groups * rows, columns], each transposed: [groups * columns, rows], in blocks of 128 along the former
    columns. With a map the rows that no token has count as zeros. What is of 8 bits already keeps its elements, but for those that become
    subnormal under their new block's scale.
    """
    if isinstance(input_, torch.Tensor):
        return _quantize(input_, groups, sparse_map, False, True)[1]
    refuse_traced()
    device = _lib.require_device(input_.values, input_.scales)
    if groups < 1 or (sparse_map is not None and groups != 1):
        raise ValueError(f"{groups} groups" + (" of a sparse layout" if sparse_map is not None else ""))
    rows = div(input_.rows, groups)
    pointers, experts, index_tag = _map_pointers(sparse_map, input_.rows, device)
    out = BlockScaledTensor.empty(groups * input_.columns, max(rows, 1), device)
    if rows == 0:
        out.values.zero_(), out.scales.zero_()
    _lib.call(
        "fm_block_transpose", device, *_pointers(input_), *_pointers(out), *pointers, groups, rows, input_.columns, experts,
        *_strides(input_), _stride(out.scales), index_tag,
    )  # fmt: skip
    return out


def block_quantize_both(
    input_: torch.Tensor, *, groups: int = 1, sparse_map: SparseMap | None = None
) -> tuple[BlockScaledTensor, BlockScaledTensor]:
    """`block_quantize` (with zeros for the rows that no token of `sparse_map` has) and `block_quantize_transposed` in one pass."""
    return _quantize(input_, groups, sparse_map, True, True)


def block_dequantize(input_: BlockScaledTensor, dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """The values that `input_` stands for, each rounded once to `dtype`."""
    refuse_traced()
    device = _lib.require_device(input_.values, input_.scales)
    out = torch.empty(input_.shape, dtype=dtype, device=device)
    _lib.call(
        "fm_block_dequantize", device, *_pointers(input_), out.data_ptr(), *input_.shape, *_strides(input_), _lib.dtype_tag(dtype)
    )
    return out


def block_quantize_expert_weights(
    weight_1: torch.Tensor, weight_2: torch.Tensor, num_experts: int, *, training: bool = True
) -> BlockScaledWeights:
    """The weights of the sparse MLP (layer 1 [experts * ffn (* 2), hidden], layer 2 [experts * ffn, hidden]) in both forms each, or without
    `training` in the one that its forward reads."""
    Assert.eq(weight_1.size(1), weight_2.size(1))
    if not training:
        return BlockScaledWeights(
            block_quantize(weight_1), None, None, block_quantize_transposed(weight_2, groups=num_experts)
        )
    return BlockScaledWeights(
        *block_quantize_both(weight_1, groups=num_experts), *block_quantize_both(weight_2, groups=num_experts)
    )


def block_copy_dense_to_sparse(input_: BlockScaledTensor, sparse_map: SparseMap) -> BlockScaledTensor:
    """`copy_dense_to_sparse` of rows of 8 bits. Padding rows of the result stay uninitialised."""
    refuse_traced()
    device = _lib.require_device(input_.values, input_.scales, sparse_map.sparse_rows)
    Assert.eq(input_.rows, sparse_map.num_rows_dense)
    Assert.eq(tuple(sparse_map.sparse_rows.shape), (sparse_map.num_rows_dense, sparse_map.num_experts_per_token))
    assert sparse_map.sparse_rows.is_contiguous()
    out = BlockScaledTensor.empty(sparse_map.num_rows, input_.columns, device)
    _lib.call(
        "fm_block_copy_dense_to_sparse", device, *_pointers(input_), sparse_map.sparse_rows.data_ptr(), *_pointers(out), *input_.shape,
        sparse_map.num_experts_per_token, sparse_map.num_rows, *_strides(input_), _stride(out.scales),
        _lib.index_tag(sparse_map.sparse_rows.dtype),
    )  # fmt: skip
    return out


def _has_worst_padding(sparse_map: SparseMap) -> bool:
    """
    Whether the layout has room for any routing of its tokens (or nothing says how many rows they have): a product's kernel is then chosen by its
    rows.
    """
    entries = sparse_map.num_rows_unpadded
    return entries is None or sparse_map.num_rows == (entries + sparse_map.num_experts * BLOCK) // BLOCK * BLOCK


def block_sparse_matmul(
    lhs: BlockScaledTensor,
    rhs: BlockScaledTensor,
    sparse_map: SparseMap | None = None,
    out: torch.Tensor | None = None,
    dtype: torch.dtype = torch.bfloat16,
    exact_sums: bool = False,
) -> torch.Tensor:
    """
    Rows of 8 bits times expert weights of 8 bits, both quantised along the axis that is summed over: both layers' products and their input gradients.
    Formula: out[i, j] = sum_k(lhs[i, k] * rhs[jd, k]), where jd = j + col_sparse_dim * sparse_index[i]
      sparse_index[i] = sum(expert_ends <= i)
    `out` (of any float type, rows contiguous) or `dtype` gives the result's type. Only the rows that tokens have are written: padding and
    the rows behind the last expert stay as they are in `out`, uninitialised without one. Experts may begin anywhere.
    Sums in fp32, rounded once. For results of 16 bits each product loses up to 2^-13 of the largest among the eight neighbours along k that it is
    one of: sums of normally distributed operands are 1.5e-5 of their root mean square off, and those whose large terms cancel may be off
    altogether. With `exact_sums` they are as exact as those for results in float32, at half the rate: for results that are quantised again, and for
    sums that cancel. (Operands then have the range of bfloat16: magnitudes from 3.3e38 on, quantised to 2^128, are infinities, and those below
    2^-126 are rounded to multiples of 2^-133.)
    """
    refuse_traced()
    Assert.eq(lhs.columns, rhs.columns)
    device = _lib.require_device(lhs.values, lhs.scales, rhs.values, rhs.scales, out)
    pointers, experts, index_tag = _map_pointers(sparse_map, lhs.rows, device, False)
    columns = div(rhs.rows, experts)
    if out is None:
        out = torch.empty((lhs.rows, columns), dtype=dtype, device=device)
    Assert.eq(tuple(out.shape), (lhs.rows, columns))
    assert out.stride(1) == 1 or columns == 1
    if columns == 0:
        return out
    name, entries = "fm_block_sparse_matmul", ()
    if sparse_map is not None and not _has_worst_padding(sparse_map):
        name, entries = "fm_block_sparse_matmul_counted", (sparse_map.num_rows_unpadded,)
    _lib.call(
        name, device, *_pointers(lhs), *_pointers(rhs), out.data_ptr(), *pointers, lhs.rows, columns,
        lhs.columns, experts, *entries, *_strides(lhs), *_strides(rhs), out.stride(0) if lhs.rows > 1 else columns, int(exact_sums),
        _lib.dtype_tag(out.dtype), index_tag,
    )  # fmt: skip
    return out


def block_input_row_sparse_matmul(
    lhs: BlockScaledTensor,
    rhs: BlockScaledTensor,
    sparse_map: SparseMap | None = None,
    out: torch.Tensor | None = None,
    accumulate: bool = False,
    dtype: torch.dtype = torch.bfloat16,
) -> torch.Tensor:
    """
    The weights' gradients from transposed forms lhs [rows, sparse rows] and rhs [columns, sparse rows] (`block_quantize_both`,
    `block_activation_backward`), which hold zeros where no token is.
    Formula: out[id, j] (+)= sum_ks(lhs[is, ks] * rhs[j, ks]), where ks are the rows of expert id // rows, is = id % rows
    `out` (of any float type, rows contiguous) or `dtype` gives the result's type. Sums are those of `block_sparse_matmul`: in fp32 and fp16 with
    `exact_sums`, in bf16 without; where large terms cancel in a gradient, its buffer is in fp32.
    """
    refuse_traced()
    Assert.eq(lhs.columns, rhs.columns)
    device = _lib.require_device(lhs.values, lhs.scales, rhs.values, rhs.scales, out)
    # (A tensor has a column: without rows that one counts for nothing.)
    empty = sparse_map is not None and sparse_map.num_rows == 0 and lhs.columns == 1
    pointers, experts, index_tag = _map_pointers(sparse_map, 0 if empty else lhs.columns, device)
    shape = (experts * lhs.rows, rhs.rows)
    if out is None:
        assert not accumulate
        out = torch.empty(shape, dtype=dtype, device=device)
    Assert.eq(tuple(out.shape), shape)
    assert out.stride(1) == 1 or shape[1] == 1
    if empty and not accumulate:
        out.zero_()
    if rhs.rows == 0 or empty:
        return out
    _lib.call(
        "fm_block_input_row_sparse_matmul", device, *_pointers(lhs), *_pointers(rhs), out.data_ptr(), *pointers, lhs.rows, rhs.rows,
        lhs.columns, experts, *_strides(lhs), *_strides(rhs), out.stride(0) if shape[0] > 1 else shape[1], int(accumulate),
        _lib.dtype_tag(out.dtype), index_tag,
    )  # fmt: skip
    return out


def block_activation_forward(
    input_: torch.Tensor, gated: bool, activation_type: ActivationType | str, sparse_map: SparseMap | None = None
) -> tuple[BlockScaledTensor, BlockScaledTensor]:
    """
    (`mlp_activation_forward` of `input_` [rows, columns] in 8 bits, of the fp32 result; `input_` itself in 8 bits, for the backward.) With a map
    the rows that no token has are zeros. Gated, gates and ups have whole blocks of 128 columns.
    """
    refuse_traced(input_)
    Assert.eq(input_.dim(), 2)
    input_ = _rows_of(input_)
    device = _lib.require_device(input_)
    rows, input_columns = input_.shape
    columns = div(input_columns, 2) if gated else input_columns
    pointers, experts, index_tag = _map_pointers(sparse_map, rows, device)
    output, checkpoint = BlockScaledTensor.empty(rows, columns, device), BlockScaledTensor.empty(rows, input_columns, device)
    _lib.call(
        "fm_block_activation_forward", device, input_.data_ptr(), *_pointers(output), *_pointers(checkpoint), *pointers, rows, columns,
        experts, input_.stride(0) if rows > 1 else input_columns, _stride(output.scales), _stride(checkpoint.scales), int(gated),
        _activation_tag(activation_type), _lib.dtype_tag(input_.dtype), index_tag,
    )  # fmt: skip
    return output, checkpoint


def block_activation_backward(
    grad_output: torch.Tensor,
    checkpoint: BlockScaledTensor,
    gated: bool,
    activation_type: ActivationType | str,
    sparse_map: SparseMap | None = None,
) -> tuple[BlockScaledTensor, BlockScaledTensor, BlockScaledTensor]:
    """
    The backward of `block_activation_forward` at what its checkpoint holds: the input's gradient along its rows (for the input gradient's product)
    and transposed (for the weights'), and the activation's result transposed, all in 8 bits of fp32 values. With a map the rows that no token has
    are zeros.
    """
    refuse_traced(grad_output)
    Assert.eq(grad_output.dim(), 2)
    grad_output = _rows_of(grad_output)
    device = _lib.require_device(grad_output, checkpoint.values, checkpoint.scales)
    rows, columns = grad_output.shape
    Assert.eq(checkpoint.shape, (rows, columns * (2 if gated else 1)))
    pointers, experts, index_tag = _map_pointers(sparse_map, rows, device)
    grad = BlockScaledTensor.empty(rows, checkpoint.columns, device)
    grad_transposed = BlockScaledTensor.empty(checkpoint.columns, max(rows, 1), device)
    output_transposed = BlockScaledTensor.empty(columns, max(rows, 1), device)
    if rows == 0:
        for tensor in (grad_transposed, output_transposed):
            tensor.values.zero_(), tensor.scales.zero_()
    _lib.call(
        "fm_block_activation_backward", device, grad_output.data_ptr(), *_pointers(checkpoint), *_pointers(grad), *_pointers(grad_transposed),
        *_pointers(output_transposed), *pointers, rows, columns, experts, grad_output.stride(0) if rows > 1 else columns,
        *_strides(checkpoint), _stride(grad.scales), _stride(grad_transposed.scales), _stride(output_transposed.scales), int(gated),
        _activation_tag(activation_type), _lib.dtype_tag(grad_output.dtype), index_tag,
    )  # fmt: skip
    return grad, grad_transposed, output_transposed


def _write_weight_gradient(weight: torch.Tensor, lhs: BlockScaledTensor, rhs: BlockScaledTensor, sparse_map: SparseMap) -> None:
    first_write = param_get_and_unset_is_zero(weight)
    block_input_row_sparse_matmul(lhs, rhs, sparse_map, out=weight.grad_buffer, accumulate=not first_write)


def _has_fine_results(tensor: torch.Tensor) -> bool:
    """
    Whether results of the tensor's type show the error of sums that are not exact: it is a sixteenth of half a step of fp16, which moves results
    that are rounded and added up by up to half again as much as the roundings do, and a 128th of half a step of bf16.
    """
    return tensor.dtype == torch.float16


class _BlockMLP(torch.autograd.Function):
    @staticmethod
    def forward(ctx, input_, scores, weight_1, weight_2, weights: BlockScaledWeights, gated, activation_type, sparse_map, training, _anchor):
        rows = block_copy_dense_to_sparse(block_quantize(input_), sparse_map)
        layer_1 = block_sparse_matmul(rows, weights.layer_1, sparse_map, dtype=input_.dtype, exact_sums=True)
        activation, checkpoint = block_activation_forward(layer_1, gated, activation_type, sparse_map)
        del layer_1
        layer_2 = block_sparse_matmul(
            activation, weights.layer_2_transposed, sparse_map, dtype=input_.dtype, exact_sums=_has_fine_results(input_)
        )
        del activation
        output = copy_sparse_to_dense(layer_2, scores, sparse_map)
        if training:
            # The backward's forms of the weights are the caller's, or are made of the weights when it comes to them: kept until then they would take
            # more than all else. (As these are saved, a weight that changes until then is noticed.)
            kept, saved = [rows, checkpoint], ()
            if weights.layer_1_transposed is None:
                saved = weight_1, weight_2
            else:
                kept += weights.layer_1_transposed, weights.layer_2
            ctx.save_for_backward(scores, layer_2, *(part for tensor in kept for part in (tensor.values, tensor.scales)), *saved)
            ctx.columns = [tensor.columns for tensor in kept]
            ctx.weights, ctx.options = (weight_1, weight_2), (gated, activation_type, sparse_map)
        return output

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_output: torch.Tensor):
        scores, layer_2, *saved = ctx.saved_tensors
        kept = [BlockScaledTensor(saved[2 * i], saved[2 * i + 1], columns) for i, columns in enumerate(ctx.columns)]
        del saved
        rows, checkpoint, layer_1_transposed, layer_2_weight = kept + [None] * (4 - len(kept))
        del kept
        (weight_1, weight_2), (gated, activation_type, sparse_map) = ctx.weights, ctx.options
        grad_layer_2, grad_scores = copy_sparse_to_dense_backward(grad_output, (sparse_map, layer_2, scores))
        grad_rows, grad_transposed = block_quantize_both(grad_layer_2, sparse_map=sparse_map)
        del grad_layer_2
        if layer_2_weight is None:
            layer_2_weight = block_quantize(weight_2)
        grad_activation = block_sparse_matmul(grad_rows, layer_2_weight, sparse_map, dtype=grad_output.dtype, exact_sums=True)
        del layer_2_weight
        grad, grad_1_transposed, activation_transposed = block_activation_backward(
            grad_activation, checkpoint, gated, activation_type, sparse_map
        )
        del grad_activation
        if weight_2.requires_grad:
            _write_weight_gradient(weight_2, activation_transposed, grad_transposed, sparse_map)
        del activation_transposed, grad_transposed
        grad_input = None
        if ctx.needs_input_grad[0]:
            if layer_1_transposed is None:
                layer_1_transposed = block_quantize_transposed(weight_1, groups=sparse_map.num_experts)
            grad_sparse = block_sparse_matmul(
                grad, layer_1_transposed, sparse_map, dtype=grad_output.dtype, exact_sums=_has_fine_results(grad_output)
            )
            del layer_1_transposed
            grad_input = copy_dense_to_sparse_backward(grad_sparse, (sparse_map, grad_output.shape))
        if weight_1.requires_grad:
            _write_weight_gradient(
                weight_1, grad_1_transposed, block_quantize_transposed(rows, sparse_map=sparse_map), sparse_map
            )
        return grad_input, grad_scores, *(None,) * 8


# An argument that makes autograd visit the node whatever else needs a gradient: the weights' gradients are side effects.
_ANCHOR = torch.empty(0, requires_grad=True)


def block_mlp(
    input_: torch.Tensor,
    scores: torch.Tensor,
    weight_1: torch.Tensor,
    weight_2: torch.Tensor,
    weights: BlockScaledWeights | None = None,
    *,
    gated: bool,
    activation_type: ActivationType | str,
    sparse_map: SparseMap,
    training: bool = True,
) -> torch.Tensor:
    """
    `mlp_autograd` of `input_` [tokens, hidden] with all products in 8 bits: dispatch, layer 1, activation, layer 2 and combine.
    `weight_1` [experts * ffn (* 2), hidden] and `weight_2` [experts * ffn, hidden] are what the gradients are of: they are written to their
    `grad_buffer`s (of any float type) as everywhere. `weights`: the same weights quantised (`block_quantize_expert_weights`), where there are
    several calls to one optimizer step; otherwise they are quantised here, for the backward in the backward, until when they have to stay as they
    are. Rows and gradients between the steps are of 8 bits; the results of both layers, of the activation's gradient and of the input's per slot
    are rounded to the input's type, sums are in fp32 (exact, as `block_sparse_matmul` says, where results are quantised again, in fp16, and for
    gradients in fp16 or fp32). Differentiable once.
    Gated, ffn is a multiple of 128.
    """
    refuse_traced(input_, scores, weight_1, weight_2)
    Assert.eq(input_.dim(), 2)
    hidden, experts = input_.size(1), sparse_map.num_experts
    ffn = div(weight_2.size(0), experts)
    Assert.eq(tuple(weight_1.shape), (experts * ffn * (2 if gated else 1), hidden))
    Assert.eq(weight_2.size(1), hidden)
    activation_type = ActivationType(activation_type)
    _activation_tag(activation_type)
    if gated and ffn % BLOCK != 0:
        raise NotImplementedError(f"a gated activation has whole blocks of {BLOCK} columns, not {ffn}")
    if weights is None:
        weights = block_quantize_expert_weights(weight_1, weight_2, experts, training=False)
    elif training and (weights.layer_1_transposed is None or weights.layer_2 is None):
        raise ValueError("the weights are quantised for inference: they have nothing for a backward")
    ffn_1 = ffn * (2 if gated else 1)
    Assert.eq(weights.layer_1.shape, (experts * ffn_1, hidden))
    Assert.eq(weights.layer_2_transposed.shape, (experts * hidden, ffn))
    for form, shape in ((weights.layer_1_transposed, (experts * hidden, ffn_1)), (weights.layer_2, (experts * ffn, hidden))):
        if form is not None:
            Assert.eq(form.shape, shape)
    input_, scores = input_.contiguous(), scores.contiguous()
    if sparse_map.num_rows == 0:
        # No token has an expert, in a layout for this routing alone: a block of rows that no expert has stands in for none at all.
        sparse_map = dataclasses.replace(sparse_map, num_rows=BLOCK)
    if not training:
        with torch.no_grad():
            output = _BlockMLP.apply(input_, scores, weight_1, weight_2, weights, gated, activation_type, sparse_map, False, None)
        return without_backward(output)
    return _BlockMLP.apply(
        input_, scores, weight_1, weight_2, weights, gated, activation_type, sparse_map, True, _ANCHOR
    )
