"""The operators on microscaled values and the norm without a GPU: sizes, and what they refuse before any kernel is launched."""

import pytest
import torch

from fast_llm_amd import _lib
from fast_llm_amd.functional import microscaling, normalization
from fast_llm_amd.functional.microscaling import MicroscaledTensor
from fast_llm_amd.functional.sparse_copy import SparseMap

FAKE = 256  # a non-null, aligned "pointer" that validation must never dereference
INVALID, UNSUPPORTED = _lib.FM_ERR_INVALID_ARGUMENT, _lib.FM_ERR_UNSUPPORTED


def test_storage():
    tensor = MicroscaledTensor.empty(5, 130, "e2m1", torch.device("cpu"))
    assert tensor.values.shape == (5, 128) and tensor.scales.shape == (5, 8) and tensor.shape == (5, 130)
    tensor = MicroscaledTensor.empty(5, 130, "e4m3", torch.device("cpu"))
    assert tensor.values.shape == (5, 256) and tensor.elements.shape == (5, 130) and tensor.block_scales.shape == (5, 5)
    assert tensor[1:3].shape == (2, 130) and tensor[1:3].values.data_ptr() == tensor.values[1].data_ptr()
    with pytest.raises(ValueError, match="mx_dequantize"):
        MicroscaledTensor.empty(1, 32, "e2m1", torch.device("cpu")).elements
    with pytest.raises(ValueError):
        MicroscaledTensor.empty(1, 32, "e5m2", torch.device("cpu"))
    values, scales = torch.zeros(3, 128, dtype=torch.uint8), torch.zeros(3, 4, dtype=torch.uint8)
    MicroscaledTensor(values, scales, 97, "e4m3")
    for bad in ((values, scales, 129, "e4m3"), (values, scales, 97, "e2m1"), (values[:2], scales, 97, "e4m3"),
                (values.float(), scales, 97, "e4m3"), (values, scales[:, :3], 97, "e4m3"), (values, scales, 0, "e4m3")):  # fmt: skip
        with pytest.raises(AssertionError):
            MicroscaledTensor(*bad)


def test_there_is_no_cpu_path():
    x, weight = torch.zeros(4, 64), torch.ones(64)
    quantized = MicroscaledTensor.empty(4, 64, "e4m3", x.device)
    experts = MicroscaledTensor(torch.zeros(128, 64, dtype=torch.uint8), torch.zeros(128, 4, dtype=torch.uint8), 64, "e2m1")
    for call in (
        lambda: microscaling.mx_quantize(x),
        lambda: microscaling.mx_dequantize(quantized),
        lambda: microscaling.mx_sparse_matmul(quantized, experts),
        lambda: normalization.rms_norm(x, weight),
        lambda: normalization.rms_norm_quantize(x, weight, x),
        lambda: microscaling.mx_mlp(quantized, torch.ones(4, 1), torch.zeros(4, 1, dtype=torch.int64), experts, experts[:64], 1,
                                    gated=True, activation_type="silu"),
    ):  # fmt: skip
        with pytest.raises(RuntimeError, match="GPU only"):
            call()


def test_operands_that_do_not_fit():
    def tensor(rows, columns, format="e2m1"):
        return MicroscaledTensor.empty(rows, columns, format, torch.device("cpu"))

    ends = torch.tensor([128, 256], dtype=torch.int32)
    sparse_map = SparseMap(None, ends, ends, 100, 256, 200, 2, 2)
    with pytest.raises(NotImplementedError, match="e2m1"):
        microscaling.mx_sparse_matmul(tensor(256, 64, "e4m3"), tensor(64, 64, "e4m3"), sparse_map)
    for lhs, rhs in (((255, 64), (64, 64)), ((256, 64), (64, 96))):
        with pytest.raises(AssertionError):
            microscaling.mx_sparse_matmul(tensor(*lhs), tensor(*rhs), sparse_map)
    with pytest.raises(ValueError, match="%2"):  # rows of the weight that are no multiple of the experts
        microscaling.mx_sparse_matmul(tensor(256, 64), tensor(65, 64), sparse_map)
    with pytest.raises(ValueError, match="%2"):  # gates without their ups
        microscaling.mx_sparse_matmul_activation(tensor(256, 64), tensor(66, 64), sparse_map, True, "silu")
    scores, top_experts = torch.ones(4, 2), torch.zeros(4, 2, dtype=torch.int64)

    def mlp(weight_1=(128, 64), weight_2=(128, 32), scores=scores, activation="silu", gated=True):
        return microscaling.mx_mlp(tensor(4, 64, "e4m3"), scores, top_experts, tensor(*weight_1), tensor(*weight_2), 2,
                                   gated=gated, activation_type=activation)  # fmt: skip

    for bad in (dict(weight_1=(120, 64)), dict(weight_1=(128, 32)), dict(weight_2=(64, 32)), dict(weight_2=(128, 64)),
                dict(scores=scores[:3]), dict(gated=False)):  # fmt: skip
        with pytest.raises(AssertionError):
            mlp(**bad)
    with pytest.raises(NotImplementedError, match="sigmoid"):
        mlp(activation="sigmoid")
    with pytest.raises(NotImplementedError, match="e2m1"):
        mlp(weight_1=(128, 64, "e4m3"))
    x, weight = torch.zeros(4, 64, dtype=torch.bfloat16), torch.ones(64, dtype=torch.bfloat16)
    with pytest.raises(AssertionError):
        normalization.rms_norm(x, weight[:32])
    with pytest.raises(AssertionError):
        normalization.rms_norm(x, weight, x[:2])
    with pytest.raises(AssertionError):
        normalization.rms_norm(x, weight, x.float())
    with pytest.raises(ValueError, match="float32"):
        normalization.rms_norm(x, weight.half())


def test_quantisation_entry_points_validate_before_launching(library):
    def quantize(rows=4, columns=64, dtype=1, format=0, values=FAKE):
        return library.fm_mx_quantize(FAKE, values, FAKE, rows, columns, columns, dtype, format, None)

    assert quantize(rows=0) == 0
    for bad in (dict(rows=-1), dict(columns=0), dict(dtype=5), dict(format=2), dict(values=None), dict(values=FAKE + 8)):
        assert quantize(**bad) == INVALID, bad
    assert quantize(rows=1 << 41) == UNSUPPORTED

    def dequantize(rows=4, columns=64, value_stride=128, scale_stride=4, values=FAKE, output=FAKE, dtype=1):
        return library.fm_mx_dequantize(values, FAKE, output, rows, columns, value_stride, scale_stride, dtype, 0, None)

    assert dequantize(rows=0) == 0
    for bad in (dict(columns=0), dict(value_stride=64), dict(value_stride=136), dict(scale_stride=2), dict(values=None), dict(output=FAKE + 1), dict(dtype=3)):
        assert dequantize(**bad) == INVALID, bad

    def dispatch(tokens=4, columns=64, slots=2, rows=256, value_stride=128, scale_stride=4, index=1, out=FAKE):
        return library.fm_mx_copy_dense_to_sparse(FAKE, FAKE, FAKE, out, FAKE, tokens, columns, slots, rows, value_stride, scale_stride, 0, index, None)

    assert dispatch(tokens=0) == 0
    for bad in (dict(columns=0), dict(slots=0), dict(value_stride=120), dict(scale_stride=6), dict(index=3), dict(out=None), dict(out=FAKE + 4)):
        assert dispatch(**bad) == INVALID, bad


def test_products_validate_before_launching(library):
    def product(rows=256, columns=64, inner=64, experts=2, lhs=FAKE, rhs=FAKE, lhs_stride=128, rhs_stride=64, scale_stride=4, out=FAKE,
                out_stride=64, format=0, dtype=1, index=1):  # fmt: skip
        return library.fm_mx_sparse_matmul(lhs, FAKE, rhs, FAKE, out, FAKE, FAKE, rows, columns, inner, experts, lhs_stride, scale_stride,
                                           rhs_stride, scale_stride, out_stride, format, dtype, index, None)  # fmt: skip

    assert product(rows=0) == 0
    for bad in (dict(rows=-1), dict(columns=0), dict(inner=0), dict(experts=0), dict(experts=1025), dict(lhs=None), dict(rhs=FAKE + 8),
                dict(lhs_stride=64), dict(lhs_stride=136), dict(rhs_stride=32), dict(scale_stride=6), dict(out=None), dict(out=FAKE + 1),
                dict(out_stride=63), dict(format=2), dict(dtype=4), dict(index=9)):  # fmt: skip
        assert product(**bad) == INVALID, bad
    assert b"index" in library.fm_last_error()
    assert product(lhs_stride=1 << 30) == UNSUPPORTED

    def with_activation(activation=1, gated=1, out=FAKE):
        return library.fm_mx_sparse_matmul_activation(FAKE, FAKE, FAKE, FAKE, out, FAKE, FAKE, FAKE, 256, 64, 64, 2, 128, 4, 64, 4, gated, activation, 0, 1, None)

    assert with_activation(activation=5) == INVALID and with_activation(out=None) == INVALID and with_activation(out=FAKE + 4) == INVALID


def test_few_tokens_entry_point_validates_before_launching(library):
    size = library.fm_mx_few_tokens_workspace_size
    entries, ffn, hidden = 3 * 2, 128, 64  # ffn 100 is stored as 128
    assert size(3, 2, hidden, 100, 8, 0) == 768 + 256 + entries * hidden * 4 and entries * ffn == 768
    for bad in ((0, 2, 64, 64, 8, 0), (4097, 1, 64, 64, 8, 0), (2049, 2, 64, 64, 8, 0), (3, 2, 64, 64, 1025, 0), (3, 2, 64, 64, 8, 2)):
        assert size(*bad) == 0, bad

    def forward(tokens=3, experts=8, workspace=FAKE, workspace_size=1 << 20, activation=1, format=0, dtype=1, scores=FAKE, input_stride=128, weight_stride=64):
        return library.fm_mx_few_tokens_forward(FAKE, FAKE, FAKE, scores, FAKE, FAKE, FAKE, FAKE, FAKE, tokens, 2, 64, 100, experts, input_stride, 4,
                                                weight_stride, 4, 64, 4, 1, activation, format, dtype, workspace, workspace_size, None)  # fmt: skip

    for bad in (dict(workspace=None), dict(workspace=FAKE + 8), dict(workspace_size=2000), dict(activation=-1), dict(format=3), dict(dtype=3),
                dict(scores=None), dict(input_stride=120), dict(weight_stride=48)):  # fmt: skip
        assert forward(**bad) == INVALID, bad
    assert forward(tokens=4097) == UNSUPPORTED and forward(experts=1025) == UNSUPPORTED


def test_norm_validates_before_launching(library):
    def forward(rows=4, columns=64, eps=1e-5, dtype=1, weight_dtype=1, residual=FAKE, stream=FAKE, values=FAKE, scales=FAKE, format=0, input_=FAKE):
        return library.fm_rms_norm_forward(input_, residual, FAKE, stream, FAKE, values, scales, rows, columns, eps, dtype, weight_dtype, format, None)

    assert forward(rows=0) == 0
    for bad in (dict(rows=-1), dict(columns=0), dict(eps=-1.0), dict(eps=float("nan")), dict(dtype=7), dict(weight_dtype=2), dict(residual=None),
                dict(stream=None), dict(values=None), dict(values=FAKE + 8), dict(format=5), dict(input_=None)):  # fmt: skip
        assert forward(**bad) == INVALID, bad
    size = library.fm_rms_norm_backward_workspace_size
    assert size(0, 64) == 0 and size(4, 0) == 0 and size(1, 64) == 64 * 4 and size(1 << 20, 64) == size(1 << 21, 64) > 0

    def backward(grad=FAKE, grad_weight=FAKE, workspace=FAKE, workspace_size=1 << 20):
        return library.fm_rms_norm_backward(grad, None, FAKE, FAKE, FAKE, grad_weight, 4, 64, 1e-5, 1, 1, workspace, workspace_size, None)

    for bad in (dict(grad=None), dict(workspace=None), dict(workspace_size=255), dict(workspace=FAKE + 4)):
        assert backward(**bad) == INVALID, bad


def test_sizes_past_what_is_counted_in_32_bits_are_refused(library):
    assert library.fm_mx_quantize(FAKE, FAKE, FAKE, 1 << 31, 64, 64, 1, 0, None) == UNSUPPORTED
    assert library.fm_mx_quantize(FAKE, FAKE, FAKE, 1 << 30, 1 << 20, 1 << 20, 1, 0, None) == UNSUPPORTED
    assert library.fm_mx_dequantize(FAKE, FAKE, FAKE, 1 << 30, 1 << 20, 1 << 20, 1 << 15, 1, 0, None) == UNSUPPORTED
    assert library.fm_mx_copy_dense_to_sparse(FAKE, FAKE, FAKE, FAKE, FAKE, 1 << 24, 64, 2, 1 << 25, 128, 4, 0, 1, None) == UNSUPPORTED
    # 200 rows, or their scales, over more than 4 GiB
    few_tokens = library.fm_mx_few_tokens_forward
    for stride, scale_stride in ((1 << 25, 4), (128, 1 << 25)):
        status = few_tokens(FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, 200, 2, 64, 100, 8, stride, scale_stride, 64, 4, 64, 4, 1, 1, 0, 1, FAKE, 1 << 24, None)
        assert status == UNSUPPORTED, (stride, scale_stride)


def test_mlp_entry_point_validates_before_launching(library):
    size = library.fm_mx_mlp_workspace_size
    # 3 * 2 rows of 8 experts: 1024, int16; ffn 100 and hidden 64 are stored as 128
    fixed = 3 * 256 + -(-max(library.fm_sparse_map_workspace_size(3, 2, 8), library.fm_sparse_map_from_router_workspace_size(3, 8)) // 256) * 256
    assert size(3, 2, 64, 100, 8, 0, 1) == fixed + 1024 * 128 + 1024 * 4 + 1024 * 128 + 1024 * 4
    for bad in ((0, 2, 64, 64, 8, 0, 1), (3, 0, 64, 64, 8, 0, 1), (3, 2, 64, 64, 1025, 0, 1), (3, 2, 64, 64, 8, 2, 1), (3, 2, 64, 64, 8, 0, 3), (1 << 24, 2, 64, 64, 8, 0, 1)):
        assert size(*bad) == 0, bad

    def forward(tokens=3, workspace=FAKE, workspace_size=1 << 30, activation=1, format=0, dtype=1, scores=FAKE, input_stride=128, weight_stride=64, router=None, shared=0):
        return library.fm_mx_mlp_forward(FAKE, FAKE, FAKE, scores, FAKE, FAKE, FAKE, FAKE, FAKE, tokens, 2, 64, 100, 8, input_stride, 4, weight_stride, 4, 64, 4,
                                         1, activation, format, dtype, router, 0, shared, workspace, workspace_size, None)  # fmt: skip

    for bad in (dict(workspace=None), dict(workspace=FAKE + 16), dict(workspace_size=2000), dict(activation=-1), dict(format=3), dict(dtype=3),
                dict(scores=None), dict(input_stride=120), dict(weight_stride=48), dict(shared=-1), dict(router=FAKE, shared=2)):  # fmt: skip
        assert forward(**bad) == INVALID, bad
    assert forward(tokens=1 << 24) == UNSUPPORTED


def test_norm_is_not_computed_in_place(library):
    a, b, c, d = (FAKE * i for i in range(1, 5))
    for stream, normalized in ((a, c), (b, c), (c, a), (c, b), (c, c)):
        assert library.fm_rms_norm_forward(a, b, d, stream, normalized, None, None, 4, 64, 1e-5, 1, 1, 0, None) == INVALID, (stream, normalized)
        assert b"in place" in library.fm_last_error()
    for result in (a, b, c):
        assert library.fm_rms_norm_backward(a, b, c, d, result, None, 4, 64, 1e-5, 1, 1, None, 0, None) == INVALID, result
        assert b"in place" in library.fm_last_error()
