"""
Microscaled (MX) values and the dropless expert MLP on expert weights of 4 bits, for inference.

A block of 32 neighbours along a row shares a power of two; elements have 8 bits (e4m3) or 4 (e2m1). The formats, rounding and storage
are those of the OCP Microscaling Formats specification 1.0, as include/fastmoe_hip.h states them. Weights are quantised along
the axis that the product sums over: layer 1 as the layer stores it, [experts * ffn (* 2, gates then ups), hidden]; layer 2 transposed expert by
expert, [experts * hidden, ffn] (`mx_quantize_expert_weights`).

The reference has no counterpart. Nothing here has a backward or a forward-mode derivative, and `torch.jit`'s tracer is refused.
"""

import dataclasses
import enum

import torch

from fast_llm_amd import _lib
from fast_llm_amd.functional.config import ActivationType
from fast_llm_amd.functional.mlp import _activation_tag
from fast_llm_amd.functional.sparse_copy import SparseMap
from fast_llm_amd.functional.utils import Assert, div, refuse_traced, without_backward

MX_BLOCK = 32
# Rows are stored padded with zeros to a multiple of this many columns.
MX_COLUMN_MULTIPLE = 128


class MicroscalingFormat(str, enum.Enum):
    e4m3 = "e4m3"
    e2m1 = "e2m1"

    def __str__(self) -> str:
        return self.value


_BYTES = {MicroscalingFormat.e4m3: MX_COLUMN_MULTIPLE, MicroscalingFormat.e2m1: MX_COLUMN_MULTIPLE // 2}


def _padded(columns: int) -> int:
    return -(-columns // MX_COLUMN_MULTIPLE) * MX_COLUMN_MULTIPLE


@dataclasses.dataclass()
class MicroscaledTensor:
    """[rows, columns] values that stand for element * 2^(scale - 127)."""

    # uint8 [rows, padded columns (e4m3) or half of that (e2m1, the even column in the low half)]
    values: torch.Tensor
    # uint8 [rows, padded columns / 32]
    scales: torch.Tensor
    columns: int
    format: MicroscalingFormat

    def __post_init__(self):
        if type(self.format) is not MicroscalingFormat:
            self.format = MicroscalingFormat(self.format)
        # One expression: it runs with every call that a tensor is made for.
        groups, values, scales = _padded(self.columns) // MX_COLUMN_MULTIPLE, self.values, self.scales
        assert (
            self.columns > 0
            and values.dtype == scales.dtype == torch.uint8
            and values.dim() == scales.dim() == 2
            and values.size(0) == scales.size(0)
            and values.size(1) == groups * _BYTES[self.format]
            and scales.size(1) == groups * (MX_COLUMN_MULTIPLE // MX_BLOCK)
            and values.stride(1) == scales.stride(1) == 1
        ), (values.dtype, values.shape, scales.dtype, scales.shape, self.columns, self.format)

    @property
    def rows(self) -> int:
        return self.values.size(0)

    @property
    def shape(self) -> tuple[int, int]:
        return self.values.size(0), self.columns

    @property
    def elements(self) -> torch.Tensor:
        """The elements without their scales [rows, columns], a view (8-bit formats: torch has none for single 4-bit values)."""
        if self.format != MicroscalingFormat.e4m3:
            raise ValueError(f"elements of {self.format} are not a tensor of their own: use `mx_dequantize`")
        return self.values.view(torch.float8_e4m3fn)[:, : self.columns]

    @property
    def block_scales(self) -> torch.Tensor:
        """The scales of the blocks that have columns [rows, ceil(columns / 32)], a view."""
        return self.scales.view(torch.float8_e8m0fnu)[:, : -(-self.columns // MX_BLOCK)]

    def __getitem__(self, rows: slice) -> "MicroscaledTensor":
        """Some of the rows, a view."""
        return MicroscaledTensor(self.values[rows], self.scales[rows], self.columns, self.format)

    @classmethod
    def empty(cls, rows: int, columns: int, format: MicroscalingFormat | str, device: torch.device) -> "MicroscaledTensor":
        assert columns > 0
        # Right by construction: the checks of `__post_init__` take as long as a small launch.
        out = cls.__new__(cls)
        out.columns, out.format = columns, MicroscalingFormat(format)
        groups = _padded(columns) // MX_COLUMN_MULTIPLE
        out.values = torch.empty((rows, groups * _BYTES[out.format]), dtype=torch.uint8, device=device)
        out.scales = torch.empty((rows, groups * (MX_COLUMN_MULTIPLE // MX_BLOCK)), dtype=torch.uint8, device=device)
        return out


def _tag(format: MicroscalingFormat) -> int:
    return _lib.MX_FORMATS[format.value]


def _stride(tensor: torch.Tensor) -> int:
    """Bytes between rows; of one row alone, what the next would need."""
    return tensor.stride(0) if tensor.size(0) > 1 else tensor.size(1)


def _strides(tensor: MicroscaledTensor) -> tuple[int, int]:
    return _stride(tensor.values), _stride(tensor.scales)


def mx_quantize(input_: torch.Tensor, format: MicroscalingFormat | str = MicroscalingFormat.e4m3) -> MicroscaledTensor:
    """
    The rows of `input_` [..., columns] in blocks of 32 along the last axis:
    scale = 2^max(floor(log2(largest magnitude)) - emax, -127) with emax = 8 (e4m3) or 2 (e2m1), element = value / scale rounded to
    nearest even and saturated. A block with an infinity or NaN is NaN altogether.
    """
    refuse_traced(input_)
    format = MicroscalingFormat(format)
    columns = input_.size(-1)
    input_ = input_.detach().reshape(input_.numel() // max(columns, 1), columns)
    if input_.stride(1) != 1:
        input_ = input_.contiguous()
    device = _lib.require_device(input_)
    rows = input_.size(0)
    out = MicroscaledTensor.empty(rows, columns, format, device)
    _lib.call(
        "fm_mx_quantize", device, input_.data_ptr(), out.values.data_ptr(), out.scales.data_ptr(), rows, columns,
        input_.stride(0), _lib.dtype_tag(input_.dtype), _tag(format),
    )  # fmt: skip
    return out


def mx_dequantize(input_: MicroscaledTensor, dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """The values that `input_` stands for, each rounded once to `dtype`."""
    refuse_traced()
    device = _lib.require_device(input_.values, input_.scales)
    out = torch.empty(input_.shape, dtype=dtype, device=device)
    _lib.call(
        "fm_mx_dequantize", device, input_.values.data_ptr(), input_.scales.data_ptr(), out.data_ptr(), *input_.shape,
        *_strides(input_), _lib.dtype_tag(dtype), _tag(input_.format),
    )  # fmt: skip
    return out


def mx_quantize_expert_weights(
    weight_1: torch.Tensor, weight_2: torch.Tensor, num_experts: int
) -> tuple[MicroscaledTensor, MicroscaledTensor]:
    """
    The weights of the sparse MLP (layer 1 [experts * ffn (* 2), hidden], layer 2 [experts * ffn, hidden]) in e2m1, each in blocks
    along the axis that its product sums over: layer 2 becomes [experts * hidden, ffn].
    """
    hidden = weight_2.size(1)
    Assert.eq(weight_1.size(1), hidden)
    transposed = weight_2.detach().view(num_experts, div(weight_2.size(0), num_experts), hidden).transpose(1, 2).flatten(0, 1)
    return mx_quantize(weight_1, MicroscalingFormat.e2m1), mx_quantize(transposed, MicroscalingFormat.e2m1)


def mx_copy_dense_to_sparse(input_: MicroscaledTensor, sparse_map: SparseMap) -> MicroscaledTensor:
    """`copy_dense_to_sparse` of microscaled rows. Padding rows of the result stay uninitialised."""
    refuse_traced()
    device = _lib.require_device(input_.values, input_.scales, sparse_map.sparse_rows)
    Assert.eq(input_.rows, sparse_map.num_rows_dense)
    Assert.eq(tuple(sparse_map.sparse_rows.shape), (sparse_map.num_rows_dense, sparse_map.num_experts_per_token))
    assert sparse_map.sparse_rows.is_contiguous()
    out = MicroscaledTensor.empty(sparse_map.num_rows, input_.columns, input_.format, device)
    _lib.call(
        "fm_mx_copy_dense_to_sparse", device, input_.values.data_ptr(), input_.scales.data_ptr(),
        sparse_map.sparse_rows.data_ptr(), out.values.data_ptr(), out.scales.data_ptr(), input_.rows, input_.columns,
        sparse_map.num_experts_per_token, sparse_map.num_rows, *_strides(input_), _tag(input_.format),
        _lib.index_tag(sparse_map.sparse_rows.dtype),
    )  # fmt: skip
    return out


def _product_operands(lhs: MicroscaledTensor, rhs: MicroscaledTensor, sparse_map: SparseMap | None) -> tuple:
    """Experts, their ends and the ends of their rows, rows of `rhs` per expert."""
    refuse_traced()
    if rhs.format != MicroscalingFormat.e2m1:
        raise NotImplementedError(f"expert weights are in e2m1, not {rhs.format}")
    Assert.eq(lhs.columns, rhs.columns)
    if sparse_map is None:
        ends = torch.full((1,), lhs.rows, dtype=torch.int32, device=lhs.values.device)
        return 1, ends, ends, rhs.rows
    experts, ends, pad_begins = sparse_map.num_experts, sparse_map.expert_ends, sparse_map.expert_pad_begins
    Assert.eq(lhs.rows, sparse_map.num_rows)
    Assert.eq(ends.numel(), pad_begins.numel(), experts)
    Assert.eq(ends.dtype, pad_begins.dtype)
    assert ends.is_contiguous() and pad_begins.is_contiguous()
    return experts, ends, pad_begins, div(rhs.rows, experts)


def mx_sparse_matmul(
    lhs: MicroscaledTensor,
    rhs: MicroscaledTensor,
    sparse_map: SparseMap | None = None,
    out: torch.Tensor | None = None,
    dtype: torch.dtype = torch.bfloat16,
) -> torch.Tensor:
    """
    Both layers' product of microscaled rows with e2m1 expert weights (`output_sparse_matmul` with every expert's weight stored
    along the axis that is summed over).
    Formula: out[i, j] = sum_k(lhs[i, k] * rhs[jd, k]), where jd = j + col_sparse_dim * sparse_index[i]
      sparse_index[i] = sum(expert_ends <= i)
    `out` (of any float type, rows contiguous) or `dtype` gives the result's type. Only the rows that tokens have are written: padding and
    the rows behind the last expert stay as they are in `out`, uninitialised without one.
    """
    experts, ends, pad_begins, columns = _product_operands(lhs, rhs, sparse_map)
    if out is None:
        out = torch.empty((lhs.rows, columns), dtype=dtype, device=lhs.values.device)
    Assert.eq(tuple(out.shape), (lhs.rows, columns))
    assert out.stride(1) == 1 or columns == 1
    device = _lib.require_device(lhs.values, lhs.scales, rhs.values, rhs.scales, out, ends, pad_begins)
    _lib.call(
        "fm_mx_sparse_matmul", device, lhs.values.data_ptr(), lhs.scales.data_ptr(), rhs.values.data_ptr(),
        rhs.scales.data_ptr(), out.data_ptr(), ends.data_ptr(), pad_begins.data_ptr(), lhs.rows, columns, lhs.columns, experts,
        *_strides(lhs), *_strides(rhs), out.stride(0) if lhs.rows > 1 else columns, _tag(lhs.format),
        _lib.dtype_tag(out.dtype), _lib.index_tag(ends.dtype),
    )  # fmt: skip
    return out


def mx_sparse_matmul_activation(
    lhs: MicroscaledTensor,
    rhs: MicroscaledTensor,
    sparse_map: SparseMap | None,
    gated: bool,
    activation_type: ActivationType | str,
) -> MicroscaledTensor:
    """
    Layer 1 with its activation: `mx_sparse_matmul`, act(gate) * up (or act alone) of the fp32 sums, microscaled in `lhs`'s
    format: one rounding. Rows that no token has stay uninitialised.
    """
    experts, ends, pad_begins, columns = _product_operands(lhs, rhs, sparse_map)
    if gated:
        columns = div(columns, 2)
    device = _lib.require_device(lhs.values, lhs.scales, rhs.values, rhs.scales, ends, pad_begins)
    out = MicroscaledTensor.empty(lhs.rows, columns, lhs.format, device)
    _lib.call(
        "fm_mx_sparse_matmul_activation", device, lhs.values.data_ptr(), lhs.scales.data_ptr(), rhs.values.data_ptr(),
        rhs.scales.data_ptr(), out.values.data_ptr(), out.scales.data_ptr(), ends.data_ptr(), pad_begins.data_ptr(), lhs.rows,
        columns, lhs.columns, experts, *_strides(lhs), *_strides(rhs), int(gated),
        _activation_tag(ActivationType(activation_type)), _tag(lhs.format), _lib.index_tag(ends.dtype),
    )  # fmt: skip
    return out


# Up to this many rows per expert on average the MLP runs without a sparse map: up to 32 rows of an expert its weights are read once. (Measured in us, without | with a
# map and tiles: 8 experts, 4096 and 2 x 14336, 16 rows per expert 170 | 259, 32 rows 279 | 274; 64 experts, 2048 and 2 x 1408, 93 | 119 and 152 | 124.)
MX_FEW_TOKENS_ROWS = 24


def mx_mlp(
    input_: torch.Tensor | MicroscaledTensor,
    scores: torch.Tensor,
    top_experts: torch.Tensor,
    weight_1: MicroscaledTensor,
    weight_2: MicroscaledTensor,
    num_experts: int,
    *,
    gated: bool,
    activation_type: ActivationType | str,
    dtype: torch.dtype | None = None,
    router_counts=None,
) -> torch.Tensor:
    """
    The dropless expert MLP in inference on e2m1 weights (`mx_quantize_expert_weights`):
    output[t] = sum_j scores[t, j] * W2[e] act(W1[e] input[t]), e = top_experts[t, j], the activations microscaled between the
    layers in the input's format. Sums are in fp32, with one rounding of the output; with over `MX_FEW_TOKENS_ROWS` rows per expert layer 2's rows are
    also rounded to `dtype` (float32: not at all), as they are in `mlp_autograd`. Entries of `top_experts` outside [0, num_experts) add
    nothing. `input_` [tokens, hidden] may be a plain tensor: it is then quantised to e4m3. `dtype` of the output: the plain input's type,
    or bfloat16.
    `router_counts` as in `get_sparse_map`.
    """
    refuse_traced(scores)
    if isinstance(input_, torch.Tensor):
        requires_grad = input_.requires_grad or scores.requires_grad
        dtype = dtype or input_.dtype
        input_ = mx_quantize(input_)
    else:
        requires_grad = scores.requires_grad
    dtype = dtype or torch.bfloat16
    activation = _activation_tag(ActivationType(activation_type))
    (tokens, hidden), slots, ffn = input_.shape, top_experts.size(-1), weight_2.columns
    Assert.eq(tuple(top_experts.shape), tuple(scores.shape), (tokens, slots))
    Assert.eq(weight_1.columns, hidden)
    Assert.eq(weight_1.rows, num_experts * ffn * (2 if gated else 1))
    Assert.eq(weight_2.rows, num_experts * hidden)
    for weight in (weight_1, weight_2):
        if weight.format != MicroscalingFormat.e2m1:
            raise NotImplementedError(f"expert weights are in e2m1, not {weight.format}")
    device = _lib.require_device(
        input_.values, input_.scales, scores, top_experts, weight_1.values, weight_1.scales, weight_2.values, weight_2.scales
    )
    if tokens == 0 or slots == 0:
        return torch.zeros((tokens, hidden), dtype=dtype, device=device)
    assert not top_experts.is_floating_point()
    library, format_tag, dtype_tag, size = _lib.lib(), _tag(input_.format), _lib.dtype_tag(dtype), 0
    if tokens * slots <= MX_FEW_TOKENS_ROWS * num_experts:
        size = library.fm_mx_few_tokens_workspace_size(tokens, slots, hidden, ffn, num_experts, format_tag)
    name, counts = "fm_mx_few_tokens_forward", ()
    if not size:
        # With a sparse map, from the router's own counts where they are of these very experts.
        size = library.fm_mx_mlp_workspace_size(tokens, slots, hidden, ffn, num_experts, format_tag, dtype_tag)
        name, counts = "fm_mx_mlp_forward", (None, 0, 0)
        if router_counts is not None and router_counts.describes(top_experts):
            Assert.eq(router_counts.tokens, tokens)
            Assert.eq(router_counts.shared_experts + router_counts.experts_per_token, slots)
            Assert.eq(router_counts.shared_experts + router_counts.routed_experts, num_experts)
            _lib.require_device(top_experts, router_counts.workspace)
            counts = router_counts.workspace
            counts = counts.data_ptr(), counts.numel() * counts.element_size(), router_counts.shared_experts
    top_experts, scores = top_experts.to(torch.int64).contiguous(), scores.detach().float().contiguous()
    out = torch.empty((tokens, hidden), dtype=dtype, device=device)
    workspace = torch.empty(size, dtype=torch.uint8, device=device)
    _lib.call(
        name, device, input_.values.data_ptr(), input_.scales.data_ptr(), top_experts.data_ptr(), scores.data_ptr(),
        weight_1.values.data_ptr(), weight_1.scales.data_ptr(), weight_2.values.data_ptr(), weight_2.scales.data_ptr(),
        out.data_ptr(), tokens, slots, hidden, ffn, num_experts, *_strides(input_), *_strides(weight_1), *_strides(weight_2),
        int(gated), activation, format_tag, dtype_tag, *counts, workspace.data_ptr(), size,
    )  # fmt: skip
    return without_backward(out) if requires_grad else out
