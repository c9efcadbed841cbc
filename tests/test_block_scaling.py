"""The operators on values of 8 bits with a scale per block of 128 without a GPU: sizes, rules, and what they refuse before any kernel is launched."""

import ctypes
import subprocess

import pytest
import torch
from torch.autograd import forward_ad

from fast_llm_amd import _lib
from fast_llm_amd.functional import block_scaling
from fast_llm_amd.functional.block_scaling import BlockScaledTensor, BlockScaledWeights
from fast_llm_amd.functional.sparse_copy import SparseMap
from fast_llm_amd.layers.moe import BlockScaledMoEMLP, DroplessMoEMLP
from oracle import block_oracle
from tests.dispatch import CSRC

FAKE = 256  # a non-null, aligned "pointer" that validation must never dereference
INVALID, UNSUPPORTED = _lib.FM_ERR_INVALID_ARGUMENT, _lib.FM_ERR_UNSUPPORTED
CPU = torch.device("cpu")


def _tensor(rows, columns):
    return BlockScaledTensor.empty(rows, columns, CPU)


def _weights(experts, hidden, ffn, gated=True):
    ffn_1 = ffn * (1 + gated)
    return BlockScaledWeights(_tensor(experts * ffn_1, hidden), _tensor(experts * hidden, ffn_1), _tensor(experts * ffn, hidden), _tensor(experts * hidden, ffn))


def _map(block=128, rows=256):
    ends = torch.tensor([rows // 2, rows], dtype=torch.int32)
    return SparseMap(torch.zeros(4, 2, dtype=torch.int32), ends, ends, 100, rows, 4, 2, 2, block)


def test_storage():
    tensor = _tensor(5, 130)
    assert tensor.values.shape == (5, 256) and tensor.scales.shape == (2, 16) and tensor.shape == (5, 130) and tensor.rows == 5
    assert tensor.elements.shape == (5, 130) and tensor.elements.dtype == torch.float8_e4m3fn
    assert tensor.block_scales.shape == (5, 2) and tensor.block_scales.dtype == torch.float8_e8m0fnu
    values, scales = torch.zeros(17, 128, dtype=torch.uint8), torch.zeros(1, 32, dtype=torch.uint8)
    BlockScaledTensor(values, scales, 97)
    for bad in ((values, scales, 129), (values, scales, 0), (values[:3], scales, 97), (values.float(), scales, 97), (values, scales[:, :17], 97),
                (values, scales.t(), 97), (values.t(), scales, 17)):  # fmt: skip
        with pytest.raises(AssertionError):
            BlockScaledTensor(*bad)


def test_the_oracle_quantises_as_torch_rounds():
    """Elements are what torch's e4m3 makes of the scaled values, and the scale is the smallest that needs no saturation."""
    generator = torch.Generator().manual_seed(0)
    values = torch.randn(40, 300, generator=generator, dtype=torch.float64) * torch.exp2(torch.randint(-30, 30, (40, 1), generator=generator))
    values[3] = 0
    elements, scales = block_oracle.quantize(values.float())
    exponents = (scales - 127).repeat_interleave(128, 1)[:, :300].double()
    assert torch.equal(elements, (values.float().double() * torch.exp2(-exponents)).float().to(torch.float8_e4m3fn).double())
    largest = torch.nn.functional.pad(values.float().double().abs(), (0, 84)).unflatten(1, (3, 128)).amax(-1)
    scale = torch.exp2(scales.double() - 127)
    assert (largest <= 448 * scale).all() and ((largest > 224 * scale) | (scales == 0)).all()
    assert (scales[3] == 0).all() and (elements[3] == 0).all()
    bad = torch.ones(2, 130)
    bad[0, 1], bad[1, 129] = float("inf"), float("nan")
    assert block_oracle.quantize(bad)[1].eq(255).tolist() == [[True, False], [False, True]]


def test_there_is_no_cpu_path():
    x, quantized, weight = torch.zeros(4, 256), _tensor(4, 128), torch.zeros(128, 256)
    for call in (
        lambda: block_scaling.block_quantize(x),
        lambda: block_scaling.block_quantize_transposed(x),
        lambda: block_scaling.block_quantize_transposed(quantized),
        lambda: block_scaling.block_quantize_both(x),
        lambda: block_scaling.block_dequantize(quantized),
        lambda: block_scaling.block_quantize_expert_weights(weight, weight, 1),
        lambda: block_scaling.block_copy_dense_to_sparse(quantized, _map()),
        lambda: block_scaling.block_sparse_matmul(quantized, quantized),
        lambda: block_scaling.block_input_row_sparse_matmul(quantized, quantized),
        lambda: block_scaling.block_activation_forward(x, True, "silu"),
        lambda: block_scaling.block_activation_backward(x, _tensor(4, 512), True, "silu"),
        lambda: block_scaling.block_mlp(x, torch.ones(4, 2), torch.zeros(512, 256), torch.zeros(256, 256), gated=True, activation_type="silu", sparse_map=_map()),
    ):  # fmt: skip
        with pytest.raises(RuntimeError, match="GPU only"):
            call()


@pytest.fixture
def on_device(monkeypatch):
    """The checks that follow those of the devices, with no call of the library."""
    monkeypatch.setattr(_lib, "require_device", lambda *tensors: CPU)
    calls = []
    monkeypatch.setattr(_lib, "call", lambda name, *args: calls.append(name))
    return calls


def test_operands_that_do_not_fit(on_device):
    x = torch.zeros(256, 256)
    for call in (
        lambda: block_scaling.block_quantize_both(x, groups=3),
        lambda: block_scaling.block_quantize_both(x, groups=0),
        lambda: block_scaling.block_quantize_both(x, groups=2, sparse_map=_map()),
        lambda: block_scaling.block_quantize_transposed(_tensor(256, 256), groups=2, sparse_map=_map()),
        lambda: block_scaling.block_sparse_matmul(_tensor(256, 64), _tensor(65, 64), _map()),
        lambda: block_scaling.block_activation_forward(torch.zeros(4, 3), True, "silu"),
        # Experts that begin where no block of 128 rows does.
        lambda: block_scaling.block_quantize_both(x, sparse_map=_map(64)),
        lambda: block_scaling.block_quantize_transposed(_tensor(256, 128), sparse_map=_map(1)),
        lambda: block_scaling.block_input_row_sparse_matmul(_tensor(64, 256), _tensor(64, 256), _map(64)),
        lambda: block_scaling.block_input_row_sparse_matmul(_tensor(64, 200), _tensor(64, 200), _map(rows=200)),
        lambda: block_scaling.block_activation_forward(x, True, "silu", _map(64)),
        lambda: block_scaling.block_activation_backward(x, _tensor(256, 512), True, "silu", _map(64)),
    ):
        with pytest.raises(ValueError):
            call()
    ends = _map().expert_ends
    for call in (
        lambda: block_scaling.block_quantize_both(x[:128], sparse_map=_map()),
        lambda: block_scaling.block_copy_dense_to_sparse(_tensor(5, 64), _map()),
        lambda: block_scaling.block_sparse_matmul(_tensor(256, 64), _tensor(64, 65), _map()),
        lambda: block_scaling.block_sparse_matmul(_tensor(255, 64), _tensor(64, 64), _map()),
        lambda: block_scaling.block_sparse_matmul(_tensor(256, 64), _tensor(64, 64), _map(), out=torch.zeros(256, 64)),
        lambda: block_scaling.block_sparse_matmul(_tensor(256, 64), _tensor(64, 64), _map(), out=torch.zeros(32, 256).t()),
        lambda: block_scaling.block_sparse_matmul(
            _tensor(256, 64), _tensor(64, 64), SparseMap(None, ends, ends.long(), 1, 256, 4, 2, 2)
        ),
        lambda: block_scaling.block_input_row_sparse_matmul(_tensor(64, 256), _tensor(64, 128), _map()),
        lambda: block_scaling.block_input_row_sparse_matmul(_tensor(64, 256), _tensor(32, 256), _map(), out=torch.zeros(64, 32)),
        lambda: block_scaling.block_input_row_sparse_matmul(_tensor(64, 256), _tensor(32, 256), _map(), accumulate=True),
        lambda: block_scaling.block_activation_backward(x, _tensor(256, 256), True, "silu"),
        lambda: block_scaling.block_quantize_expert_weights(torch.zeros(8, 64), torch.zeros(8, 32), 2),
    ):
        with pytest.raises(AssertionError):
            call()
    for call in (lambda: block_scaling.block_activation_forward(x, True, "sigmoid"), lambda: block_scaling.block_activation_backward(x, _tensor(256, 512), True, "sigmoid")):
        with pytest.raises((NotImplementedError, ValueError), match="sigmoid"):
            call()
    assert on_device == []
    block_scaling.block_sparse_matmul(_tensor(256, 64), _tensor(64, 64), _map(1))  # whose experts may begin anywhere
    assert on_device == ["fm_block_sparse_matmul"]


def test_mlps_that_do_not_fit(on_device):
    def mlp(weight_1=(512, 64), weight_2=(256, 64), weights=None, gated=True, activation="silu", columns=64):
        return block_scaling.block_mlp(torch.zeros(4, columns), torch.ones(4, 2), torch.zeros(weight_1), torch.zeros(weight_2), weights, gated=gated,
                                       activation_type=activation, sparse_map=_map())  # fmt: skip

    for bad in (dict(weight_1=(256, 64)), dict(weight_1=(512, 32)), dict(weight_2=(256, 32)), dict(gated=False), dict(columns=32),
                dict(weights=_weights(2, 64, 256)), dict(weights=_weights(2, 128, 128)), dict(weights=_weights(2, 64, 128, False)),
                dict(weights=BlockScaledWeights(*reversed(_weights(2, 64, 128))))):  # fmt: skip
        with pytest.raises(AssertionError):
            mlp(**bad)
    with pytest.raises(ValueError, match="%2"):
        mlp(weight_2=(255, 64))
    with pytest.raises(NotImplementedError, match="128"):
        mlp(weight_1=(400, 64), weight_2=(200, 64))
    with pytest.raises(NotImplementedError, match="sigmoid"):
        mlp(activation="sigmoid")
    assert on_device == []


def test_layers_that_are_refused():
    for bad in (dict(intermediate_size=192), dict(recompute_level="full")):
        arguments = dict(intermediate_size=128) | bad
        with pytest.raises(NotImplementedError):
            BlockScaledMoEMLP(64, experts=4, experts_per_token=2, device="cpu", **arguments)
    layer = BlockScaledMoEMLP(64, 100, 4, 2, gated=False, shared_experts=1, device="cpu")
    for half in (dict(scores=torch.ones(3, 2)), dict(top_experts=torch.zeros(3, 2, dtype=torch.int64))):
        with pytest.raises(ValueError, match="own"):
            layer(torch.zeros(3, 64, dtype=torch.bfloat16), **half)
    assert {n: p.shape for n, p in layer.named_parameters()} == {
        n: p.shape for n, p in DroplessMoEMLP(64, 100, 4, 2, gated=False, shared_experts=1, device="cpu").named_parameters()
    }


X, SCORES, WEIGHT_1, WEIGHT_2 = torch.randn(4, 128), torch.ones(4, 2), torch.randn(512, 128), torch.randn(256, 128)


def _mlp(*tensors):
    return block_scaling.block_mlp(*tensors, gated=True, activation_type="silu", sparse_map=_map())


# The function and its arguments, of which any may carry a tangent.
CALLS = {
    "quantize": (lambda x: block_scaling.block_quantize(x).values, (X,)),
    "quantize_transposed": (lambda x: block_scaling.block_quantize_transposed(x).values, (X,)),
    "quantize_both": (lambda x: block_scaling.block_quantize_both(x)[0].values, (X,)),
    "activation_forward": (lambda x: block_scaling.block_activation_forward(x, False, "silu")[0].values, (X,)),
    "activation_backward": (lambda x: block_scaling.block_activation_backward(x, _tensor(4, 128), False, "silu")[0].values, (X,)),
    "mlp": (_mlp, (X, SCORES, WEIGHT_1, WEIGHT_2)),
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


# ---- entry points ----------------------------------------------------------------------------------------
def test_quantisation_validates_before_launching(library):
    def quantize(input_=FAKE, values=FAKE, scales=FAKE, t_values=FAKE, t_scales=FAKE, ends=None, begins=None, groups=1, rows=256, columns=64,
                 experts=1, input_stride=64, scale_stride=256, t_scale_stride=64, dtype=1, index=1):  # fmt: skip
        return library.fm_block_quantize(input_, values, scales, t_values, t_scales, ends, begins, groups, rows, columns, experts, input_stride, scale_stride,
                                         t_scale_stride, dtype, index, None)  # fmt: skip

    assert quantize(rows=0) == 0
    for bad in (dict(rows=-1), dict(columns=0), dict(groups=-1), dict(dtype=5), dict(input_=None), dict(values=None), dict(t_scales=None),
                dict(values=None, scales=None, t_values=None, t_scales=None), dict(ends=FAKE), dict(ends=FAKE, begins=FAKE, index=4),
                dict(ends=FAKE, begins=FAKE, experts=0), dict(ends=FAKE, begins=FAKE, experts=1025), dict(ends=FAKE, begins=FAKE, groups=2),
                dict(ends=FAKE, begins=FAKE, t_values=None, t_scales=None), dict(input_stride=-1), dict(input_=FAKE + 1), dict(values=FAKE + 8), dict(scale_stride=255),
                dict(t_scale_stride=63)):  # fmt: skip
        assert quantize(**bad) == INVALID, bad

    def transpose(values=FAKE, out=FAKE, ends=None, groups=1, rows=256, columns=64, stride=128, scale_stride=256, out_scale_stride=64):
        return library.fm_block_transpose(values, FAKE, out, FAKE, ends, ends, groups, rows, columns, 2, stride, scale_stride, out_scale_stride, 1, None)

    assert transpose(rows=0) == 0
    for bad in (dict(rows=-1), dict(columns=0), dict(groups=-1), dict(values=None), dict(out=None), dict(out=FAKE + 4), dict(stride=64), dict(stride=136),
                dict(scale_stride=255), dict(out_scale_stride=60), dict(ends=FAKE, groups=2)):  # fmt: skip
        assert transpose(**bad) == INVALID, bad

    def dequantize(values=FAKE, out=FAKE, rows=20, columns=64, stride=128, scale_stride=32, dtype=1):
        return library.fm_block_dequantize(values, FAKE, out, rows, columns, stride, scale_stride, dtype, None)

    assert dequantize(rows=0) == 0
    for bad in (dict(columns=0), dict(stride=64), dict(stride=130), dict(scale_stride=16), dict(values=None), dict(out=None), dict(dtype=3), dict(out=FAKE + 1)):
        assert dequantize(**bad) == INVALID, bad

    def dispatch(values=FAKE, rows_of=FAKE, out=FAKE, tokens=4, columns=64, slots=2, rows=256, stride=128, scale_stride=16, out_scale_stride=256, index=1):
        return library.fm_block_copy_dense_to_sparse(values, FAKE, rows_of, out, FAKE, tokens, columns, slots, rows, stride, scale_stride, out_scale_stride, index,
                                                     None)  # fmt: skip

    assert dispatch(tokens=0) == 0
    for bad in (dict(columns=0), dict(slots=0), dict(stride=120), dict(scale_stride=3), dict(out_scale_stride=240), dict(index=3), dict(out=None),
                dict(out=FAKE + 4), dict(rows_of=None)):  # fmt: skip
        assert dispatch(**bad) == INVALID, bad


def test_products_validate_before_launching(library):
    def product(lhs=FAKE, rhs=FAKE, out=FAKE, ends=FAKE, begins=FAKE, rows=256, columns=64, inner=64, experts=2, lhs_stride=128, lhs_scale_stride=256,
                rhs_stride=128, rhs_scale_stride=128, out_stride=64, exact=0, dtype=1, index=1):  # fmt: skip
        return library.fm_block_sparse_matmul(lhs, FAKE, rhs, FAKE, out, ends, begins, rows, columns, inner, experts, lhs_stride, lhs_scale_stride, rhs_stride,
                                              rhs_scale_stride, out_stride, exact, dtype, index, None)  # fmt: skip

    assert product(rows=0) == 0
    for bad in (dict(rows=-1), dict(columns=0), dict(inner=0), dict(experts=0), dict(experts=1025), dict(dtype=3), dict(index=3), dict(lhs=None),
                dict(rhs=None), dict(out=None), dict(begins=None), dict(ends=None, begins=None), dict(lhs=FAKE + 8), dict(rhs=FAKE + 8), dict(out=FAKE + 1),
                dict(lhs_stride=64), dict(rhs_stride=136), dict(lhs_scale_stride=240), dict(rhs_scale_stride=100), dict(out_stride=63)):  # fmt: skip
        assert product(**bad) == INVALID, bad

    def gradient(lhs=FAKE, rhs=FAKE, out=FAKE, ends=FAKE, begins=FAKE, rows=64, columns=48, inner=256, experts=2, lhs_stride=256, lhs_scale_stride=64,
                 rhs_stride=256, rhs_scale_stride=48, out_stride=48, accumulate=0, dtype=1, index=1):  # fmt: skip
        return library.fm_block_input_row_sparse_matmul(lhs, FAKE, rhs, FAKE, out, ends, begins, rows, columns, inner, experts, lhs_stride, lhs_scale_stride,
                                                        rhs_stride, rhs_scale_stride, out_stride, accumulate, dtype, index, None)  # fmt: skip

    assert gradient(rows=0) == 0
    for bad in (dict(rows=-1), dict(columns=0), dict(inner=0), dict(experts=0), dict(experts=1025), dict(dtype=3), dict(index=3), dict(lhs=None),
                dict(rhs=None), dict(out=None), dict(begins=None), dict(ends=None, begins=None), dict(lhs=FAKE + 8), dict(out=FAKE + 1), dict(lhs_stride=128),
                dict(rhs_stride=264), dict(lhs_scale_stride=48), dict(rhs_scale_stride=40), dict(out_stride=47)):  # fmt: skip
        assert gradient(**bad) == INVALID, bad


def test_activations_validate_before_launching(library):
    def forward(input_=FAKE, output=FAKE, checkpoint=FAKE, ends=None, rows=256, columns=128, experts=1, input_stride=256, output_stride=256,
                checkpoint_stride=256, gated=1, activation=0, dtype=1):  # fmt: skip
        return library.fm_block_activation_forward(input_, output, FAKE, checkpoint, FAKE, ends, ends, rows, columns, experts, input_stride, output_stride,
                                                   checkpoint_stride, gated, activation, dtype, 1, None)  # fmt: skip

    assert forward(rows=0) == 0
    for bad in (dict(rows=-1), dict(columns=0), dict(input_=None), dict(output=None), dict(checkpoint=None), dict(input_stride=128), dict(output_stride=128),
                dict(checkpoint_stride=240), dict(activation=99), dict(dtype=3), dict(input_=FAKE + 1), dict(output=FAKE + 8),
                dict(ends=FAKE, experts=0)):  # fmt: skip
        assert forward(**bad) == INVALID, bad
    assert forward(columns=100) == UNSUPPORTED

    def backward(grad=FAKE, checkpoint=FAKE, outputs=(FAKE,) * 3, ends=None, rows=256, columns=128, experts=1, grad_stride=128, checkpoint_stride=256,
                 checkpoint_scale_stride=256, strides=(256, 256, 128), gated=1, activation=0, dtype=1):  # fmt: skip
        pointers = [p for output in outputs for p in (output, FAKE)]
        return library.fm_block_activation_backward(grad, checkpoint, FAKE, *pointers, ends, ends, rows, columns, experts, grad_stride, checkpoint_stride,
                                                    checkpoint_scale_stride, *strides, gated, activation, dtype, 1, None)  # fmt: skip

    assert backward(rows=0) == 0
    for bad in (dict(rows=-1), dict(columns=0), dict(grad=None), dict(checkpoint=None), dict(outputs=(None, FAKE, FAKE)), dict(outputs=(FAKE, None, FAKE)),
                dict(outputs=(FAKE, FAKE, FAKE + 8)), dict(grad_stride=127), dict(checkpoint_stride=128), dict(checkpoint_scale_stride=240),
                dict(strides=(240, 256, 128)), dict(strides=(256, 240, 128)), dict(strides=(256, 256, 112)), dict(activation=99), dict(dtype=3)):  # fmt: skip
        assert backward(**bad) == INVALID, bad
    assert backward(columns=100) == UNSUPPORTED


# ---- rules -----------------------------------------------------------------------------------------------
_PROGRAM = """
#include "fm_block_product.h"
using namespace fm::block;

extern "C" int takes(int64_t rows, int64_t columns, int64_t inner, int experts, int by_map) {
    static char ends[2];
    ProductArgs args{};
    args.rows = rows, args.columns = columns, args.inner = padded_columns(inner), args.experts = experts;
    args.x_stride = args.weight_stride = args.inner, args.x_scale_stride = (rows + 15) / 16 * 16, args.weight_scale_stride = (experts * columns + 15) / 16 * 16;
    args.out_stride = columns;
    if (by_map) args.expert_ends = ends, args.expert_pad_begins = ends + 1;
    return runs_on_tiles(args);
}
"""


@pytest.fixture(scope="module")
def rules(tmp_path_factory, library):
    from fast_llm_amd.build import _hipcc

    folder, library = tmp_path_factory.mktemp("block_dispatch"), _lib.LIBRARY_PATH
    (folder / "rules.hip").write_text(_PROGRAM)
    subprocess.run(
        [_hipcc(), "--offload-host-only", "-std=c++17", "-fPIC", "-shared", f"-I{CSRC}", str(folder / "rules.hip"), "-o", str(folder / "rules.so"),
         f"-L{library.parent}", f"-l:{library.name}", f"-Wl,-rpath,{library.parent}"],
        check=True, capture_output=True,
    )  # fmt: skip
    found = ctypes.CDLL(str(folder / "rules.so"))
    found.takes.argtypes = [ctypes.c_int64] * 3 + [ctypes.c_int] * 2
    return found.takes


def test_which_kernel_the_products_of_the_tests_run_on(rules):
    from tests import test_gpu_block_scaling as tested

    sizes = [(1, 1), (128, 64), (384, 100), (512, 256), (640, 130), (1416, 516)]
    ran = {rules(sum(-(-c // 128) * 128 for c in counts), columns, inner, len(counts), 1) for counts in tested.COUNTS + [[256, 700], [31, 0, 33, 2]] for inner, columns in sizes}
    assert ran == {0, 1}
    # Few rows per expert do not run on tiles, many do, whatever the length of the reduction.
    assert rules(8 * 128, 28672, 4096, 8, 1) == 0 and rules(8 * 1024, 28672, 4096, 8, 1) == 1
    assert rules(1, 28672, 4096, 1, 0) == 0 and rules(33, 28672, 4096, 1, 0) == 1
    assert rules(4096, 512, 1, 1, 0) == rules(4096, 512, 257, 1, 0) == 1
