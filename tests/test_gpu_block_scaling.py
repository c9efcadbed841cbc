"""Values of 8 bits with a scale per block of 128, the products on them and the expert MLP's step, against the oracle in 64 bits."""

import pytest
import torch

from fast_llm_amd.functional.block_scaling import (
    BlockScaledTensor, block_activation_backward, block_activation_forward, block_copy_dense_to_sparse, block_dequantize,
    block_input_row_sparse_matmul, block_mlp, block_quantize, block_quantize_both, block_quantize_expert_weights, block_quantize_transposed,
    block_sparse_matmul,
)  # fmt: skip
from fast_llm_amd.functional.sparse_copy import SparseMap, get_sparse_map
from fast_llm_amd.layers.moe import attach_grad_buffer
from oracle import block_oracle
from oracle.mx_oracle import activation as plain_activation

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
ACTIVATIONS = ["silu", "gelu", "relu", "squared_relu", "identity"]


def _values(tensor: BlockScaledTensor) -> torch.Tensor:
    return block_oracle.unpack(tensor.values.cpu(), tensor.scales.cpu(), tensor.columns)


def _assert_stored(ours: BlockScaledTensor, values: torch.Tensor) -> None:
    """`ours` holds `values` quantised, bit for bit, with zeros behind the rows' ends."""
    elements, scales = block_oracle.pack(*block_oracle.quantize(values))
    assert ours.shape == values.shape
    assert torch.equal(ours.values.cpu(), elements)
    assert torch.equal(ours.scales[:, : ours.rows].cpu(), scales)


def _map(counts: list[int], device, index_dtype=torch.int32, block: int = 128, phantom: int = 0) -> SparseMap:
    ends, pad_begins, begin = [], [], 0
    for count in counts:
        pad_begins.append(begin + count)
        begin += -(-count // block) * block
        ends.append(begin)
    to = dict(dtype=index_dtype, device=device)
    return SparseMap(
        None, torch.tensor(ends, **to), torch.tensor(pad_begins, **to), None, begin + phantom, sum(counts), len(counts), None, block
    )


def _experts(sparse_map: SparseMap) -> list[tuple[int, int, int]]:
    """(expert, first row, end of its tokens' rows)"""
    ends, pad_begins = sparse_map.expert_ends.tolist(), sparse_map.expert_pad_begins.tolist()
    return [(e, begin, end) for e, (begin, end) in enumerate(zip([0] + ends[:-1], pad_begins))]


def _real(sparse_map: SparseMap) -> torch.Tensor:
    real = torch.zeros(sparse_map.num_rows, dtype=torch.bool)
    for _, begin, end in _experts(sparse_map):
        real[begin:end] = True
    return real


def _unlike(generator, rows: int, columns: int, dtype) -> torch.Tensor:
    """Rows, and columns by blocks of 64, of unlike size."""
    sizes = torch.exp2(torch.randint(-8, 9, (rows, 1), generator=generator)) * torch.exp2(
        torch.randint(-3, 4, (-(-columns // 64),), generator=generator).repeat_interleave(64)[:columns]
    )
    return (torch.randn(rows, columns, generator=generator) * sizes).clamp(-6e4, 6e4).to(dtype)


# ---- quantisation ----------------------------------------------------------------------------------------
# One row, one column, parts of blocks on both axes, whole ones, odd lengths, more than a workgroup's share.
SHAPES = [(1, 1), (1, 4096), (3, 33), (128, 128), (127, 129), (130, 777), (9, 2050), (300, 260)]


@pytest.mark.parametrize(("rows", "columns"), SHAPES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_quantize_and_back(rows, columns, dtype, device):
    generator = torch.Generator().manual_seed(rows + columns)
    values = _unlike(generator, rows, columns, dtype)
    quantized = block_quantize(values.to(device))
    _assert_stored(quantized, values)
    elements, scales = block_oracle.quantize(values)
    assert torch.equal(quantized.elements.cpu().double(), elements)
    assert torch.equal(quantized.block_scales.view(torch.uint8).cpu().long(), scales)
    for back in DTYPES:
        assert torch.equal(block_dequantize(quantized, back).cpu(), block_oracle.values_of(elements, scales).to(back))


@pytest.mark.parametrize("groups", [1, 3])
@pytest.mark.parametrize(("rows", "columns"), SHAPES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_both_forms(rows, columns, groups, dtype, device):
    generator = torch.Generator().manual_seed(rows + columns + groups)
    values = _unlike(generator, groups * rows, columns, dtype)
    along_rows, transposed = block_quantize_both(values.to(device), groups=groups)
    _assert_stored(along_rows, values)
    expected = values.view(groups, rows, columns).transpose(1, 2).reshape(groups * columns, rows)
    _assert_stored(transposed, expected)
    _assert_stored(block_quantize_transposed(values.to(device), groups=groups), expected)
    # Of 8 bits already: what remains along the rows, quantised along the columns.
    remaining = block_oracle.kept(values).view(groups, rows, columns).transpose(1, 2).reshape(groups * columns, rows)
    _assert_stored(block_quantize_transposed(along_rows, groups=groups), remaining)


def test_quantize_at_the_edges(device):
    """Zeros of both signs, subnormal and smallest values, the largest ones, both sides of 448, ties, infinities and NaN, a block each."""
    values = torch.zeros(2, 1280)
    values[0, 1] = -0.0
    values[0, 128:132] = torch.tensor([2.0**-149, -(2.0**-140), 2.0**-126, 2.0**-130])
    values[0, 256:260] = torch.tensor([torch.finfo(torch.float32).max, -1e38, 1e-38, 1.0])
    values[0, 384:386] = torch.tensor([448.0, 2.0**-9])  # as it is, and the smallest element
    values[0, 512:514] = torch.tensor([torch.tensor(448.0).nextafter(torch.tensor(1e9)), 448.0])
    values[0, 640:649] = 256 + 8 * torch.arange(9)  # ties between 256 and 320
    values[0, 768:772] = torch.tensor([448.0, 1.5 * 2.0**-9, 2.5 * 2.0**-9, 2.0**-10])  # ties of subnormal elements
    values[0, 896], values[0, 1024], values[0, 1152] = float("inf"), float("nan"), -float("inf")
    values[0, 900] = 3.0
    values[1] = torch.randn(1280, generator=torch.Generator().manual_seed(1))
    for dtype in (torch.float32, torch.bfloat16):
        _assert_stored(block_quantize(values.to(device, dtype)), values.to(dtype))
        # (Transposed, the two rows are blocks of two.)
        along_rows, transposed = block_quantize_both(values.to(device, dtype))
        _assert_stored(along_rows, values.to(dtype))
        _assert_stored(transposed, values.to(dtype).t())
    lowest = torch.full((2, 200), torch.finfo(torch.bfloat16).min, dtype=torch.bfloat16)
    _assert_stored(block_quantize(lowest.to(device)), lowest)
    quantized = block_quantize(values.to(device))
    _assert_stored(block_quantize_transposed(quantized), _values(quantized).t())
    assert torch.equal(block_dequantize(quantized).cpu().double().isnan(), _values(quantized).isnan())


def test_strided_rows(device):
    generator = torch.Generator().manual_seed(3)
    for dtype in DTYPES:
        wide = _unlike(generator, 140, 700, dtype)
        for view in (wide[:, 3:600], wide[::2, 8:520], wide.t(), wide[:1], wide.view(2, 70, 700)[:, :, 1:]):
            rows = view.reshape(-1, view.size(-1))
            _assert_stored(block_quantize(view.to(device)), rows)
            on_device = wide.to(device)
            strided = on_device.as_strided(view.shape, view.stride(), view.storage_offset())
            for ours in block_quantize(strided), block_quantize_both(strided)[0]:
                _assert_stored(ours, rows)
            _assert_stored(block_quantize_transposed(strided), rows.t())


COUNTS = [[1], [0, 1, 0], [128, 0, 129, 2], [300, 0, 257, 1, 512], [0, 0], [3] * 70 + [0] * 60 + [140]]


@pytest.mark.parametrize("index_dtype", [torch.int16, torch.int32, torch.int64])
@pytest.mark.parametrize("counts", COUNTS, ids=str)
def test_rows_that_no_token_has_are_zeros(counts, index_dtype, device):
    generator = torch.Generator().manual_seed(len(counts))
    sparse_map = _map(counts, device, index_dtype, phantom=256)
    real = _real(sparse_map)[:, None]
    values = _unlike(generator, sparse_map.num_rows, 200, torch.bfloat16)
    expected = torch.where(real, values, 0)
    values = torch.where(real, values, float("nan")).to(device)
    along_rows, transposed = block_quantize_both(values, sparse_map=sparse_map)
    _assert_stored(along_rows, expected)
    _assert_stored(transposed, expected.t())
    _assert_stored(block_quantize_transposed(values, sparse_map=sparse_map), expected.t())
    _assert_stored(block_quantize_transposed(block_quantize(values), sparse_map=sparse_map), block_oracle.kept(expected).t())


@pytest.mark.parametrize(("tokens", "slots", "columns"), [(1, 1, 5), (37, 3, 200), (300, 2, 1408)])
def test_dispatch(tokens, slots, columns, device):
    generator = torch.Generator().manual_seed(tokens)
    top_experts = torch.randint(-1, 7, (tokens, slots), generator=generator)  # some select no expert
    rows = block_quantize(torch.randn(tokens, columns, generator=generator).to(device))
    sparse_map = get_sparse_map(top_experts.to(device), 6)
    sparse = block_copy_dense_to_sparse(rows, sparse_map)
    assert sparse.shape == (sparse_map.num_rows, columns)
    for token, targets in enumerate(sparse_map.sparse_rows.cpu().tolist()):
        for target in targets:
            if target >= 0:
                assert torch.equal(sparse.values[target], rows.values[token]) and torch.equal(sparse.scales[:, target], rows.scales[:, token])


# ---- products --------------------------------------------------------------------------------------------
def _whole(generator, shape, device) -> tuple[BlockScaledTensor, torch.Tensor]:
    """Whole numbers up to 2 times 1/2, 1 or 2, by block of 128: e4m3 holds every one, and scales differ from block to block and from row to row."""
    values = torch.tensor([0.0, 1, -1, 2, -2])[torch.randint(0, 5, shape, generator=generator)]
    sizes = torch.exp2(torch.randint(-1, 2, (shape[0], -(-shape[1] // 128)), generator=generator).float())
    values = values * sizes.repeat_interleave(128, dim=1)[:, : shape[1]]
    quantized = block_quantize(values.to(device))
    assert torch.equal(_values(quantized), values.double())
    return quantized, values


# The matrix instruction drops what lies under 2^-17 of the largest of its terms and the sum so far: nothing, where that is below 2^14 units of 1/4 (a
# quarter of the room is left for partial sums that are larger than the whole).
def _assert_exact(sums: torch.Tensor) -> None:
    assert sums.numel() == 0 or sums.abs().max() < 2**14 / 4


@pytest.mark.parametrize("counts", COUNTS + [[256, 700], [31, 0, 33, 2]], ids=str)
# Reductions of one slice and of parts of it, of an odd and an even number of slices; columns of parts of blocks of 16 and 32, and on both
# sides of the tiles.
@pytest.mark.parametrize(("inner", "columns"), [(1, 1), (128, 64), (384, 100), (512, 256), (640, 130), (1416, 516)])
def test_whole_numbers_are_multiplied_exactly(counts, inner, columns, device):
    if len(counts) > 100 and inner * columns > 100 * 400:
        pytest.skip("large on the CPU")
    generator = torch.Generator().manual_seed(inner + columns)
    sparse_map = _map(counts, device, phantom=128)
    lhs, wide = _whole(generator, (sparse_map.num_rows, inner), device)
    rhs, weight = _whole(generator, (len(counts) * columns, inner), device)
    # What padding rows hold is not looked at.
    real = _real(sparse_map).to(device)
    lhs.values[~real], lhs.scales[:, : lhs.rows][:, ~real] = 0x7F, 255
    out = torch.full((sparse_map.num_rows, columns), -7.0, device=device)
    assert block_sparse_matmul(lhs, rhs, sparse_map, out) is out
    expected = torch.full_like(out, -7.0).cpu()
    for expert, begin, end in _experts(sparse_map):
        expected[begin:end] = wide[begin:end] @ weight.view(len(counts), columns, inner)[expert].t()
        _assert_exact(expected[begin:end])
    assert torch.equal(out.cpu(), expected)  # what no token has is as it was
    for dtype in (torch.bfloat16, torch.float16):
        half = block_sparse_matmul(lhs, rhs, sparse_map, dtype=dtype)
        for _, begin, end in _experts(sparse_map):
            assert torch.equal(half[begin:end].cpu(), expected[begin:end].to(dtype))


@pytest.mark.parametrize("index_dtype", [torch.int16, torch.int32, torch.int64])
@pytest.mark.parametrize("counts", [[300, 259, 5], [9, 0, 30]], ids=str)
def test_strides_and_boundaries_of_any_kind(counts, index_dtype, device):
    generator = torch.Generator().manual_seed(5)
    inner, columns = 512, 132
    sparse_map = _map(counts, device, index_dtype, block=1, phantom=3)
    lhs, wide = _whole(generator, (sparse_map.num_rows, inner), device)
    rhs, weight = _whole(generator, (3 * columns, inner), device)

    def spread(tensor: BlockScaledTensor) -> BlockScaledTensor:
        values = torch.full((tensor.rows, 2 * tensor.values.size(1)), 0x7F, dtype=torch.uint8, device=device)
        scales = torch.full((tensor.scales.size(0), tensor.scales.size(1) + 48), 255, dtype=torch.uint8, device=device)
        values, scales = values[:, 16 : 16 + tensor.values.size(1)], scales[:, 32 : 32 + tensor.scales.size(1)]
        values.copy_(tensor.values), scales.copy_(tensor.scales)
        return BlockScaledTensor(values, scales, inner)

    for offset in (8, 9):  # columns in the middle of wider rows, aligned to vectors and not
        around = torch.full((sparse_map.num_rows, 2 * columns), -7.0, dtype=torch.float16, device=device)
        out = around[:, offset : offset + columns]
        block_sparse_matmul(spread(lhs), spread(rhs), sparse_map, out)
        for expert, begin, end in _experts(sparse_map):
            assert torch.equal(out[begin:end].cpu(), (wide[begin:end] @ weight[expert * columns : (expert + 1) * columns].t()).half())
        assert (around[:, :offset] == -7).all() and (around[:, offset + columns :] == -7).all() and (out[-3:] == -7).all()


def _tolerance(lhs: torch.Tensor, rhs: torch.Tensor, expected: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    """The matrix instruction aligns the 64 products that it adds, and the sum so far, to the largest of them and drops what lies
    under its last bit, at 2^-17 of it or below: per product of the reduction at most that; then the result's rounding, half a step. (Below the smallest
    normal value, in fp16 2^-14, steps get no smaller: there half of one is eps / 2 of that, in fp16 2^-25, whatever the value.)"""
    largest = lhs.abs().amax(-1, keepdim=True) * rhs.abs().amax(-1)[None]
    return 2.0**-17 * lhs.size(-1) * torch.maximum(largest, expected.abs()) + torch.finfo(dtype).eps / 2 * expected.abs().clamp_min(torch.finfo(dtype).smallest_normal)


@pytest.mark.parametrize("counts", [[40, 3], [300, 257]], ids=str)
@pytest.mark.parametrize(("inner", "columns"), [(200, 70), (1024, 300)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_products_of_values_of_all_sizes(counts, inner, columns, dtype, device):
    generator = torch.Generator().manual_seed(inner)
    sparse_map = _map(counts, device)
    lhs = block_quantize(_unlike(generator, sparse_map.num_rows, inner, torch.float32).to(device))
    rhs = block_quantize((_unlike(generator, len(counts) * columns, inner, torch.float32) * 2.0**-8).to(device))
    out = block_sparse_matmul(lhs, rhs, sparse_map, dtype=dtype)
    rows, weight = _values(lhs), _values(rhs).view(len(counts), columns, inner)
    for expert, begin, end in _experts(sparse_map):
        expected = rows[begin:end] @ weight[expert].t()
        finite = expected.abs() < torch.finfo(dtype).max / 2
        error = (out[begin:end].cpu().double() - expected).abs()
        assert (error[finite] <= _tolerance(rows[begin:end], weight[expert], expected, dtype)[finite]).all()


@pytest.mark.parametrize("counts", [[33], [290]], ids=str)
def test_blocks_of_nan_reach_their_rows_only(counts, device):
    generator = torch.Generator().manual_seed(9)
    sparse_map = _map(counts, device)
    values = torch.randn(sparse_map.num_rows, 512, generator=generator)
    values[5, 70], values[20, 511] = float("nan"), float("inf")
    weight = torch.randn(64, 512, generator=generator)
    weight[40, 0] = float("inf")
    out = block_sparse_matmul(block_quantize(values.to(device)), block_quantize(weight.to(device)), sparse_map)[: counts[0]].cpu()
    expected = torch.zeros(counts[0], 64, dtype=torch.bool)
    expected[5], expected[20], expected[:, 40] = True, True, True
    assert torch.equal(torch.isnan(out), expected)


@pytest.mark.parametrize("rows", [1, 40, 300])
def test_dense_products(rows, device):
    generator = torch.Generator().manual_seed(rows)
    (lhs, wide), (rhs, weight) = _whole(generator, (rows, 640), device), _whole(generator, (96, 640), device)
    assert torch.equal(block_sparse_matmul(lhs, rhs, dtype=torch.float32).cpu(), wide @ weight.t())
    assert torch.equal(block_input_row_sparse_matmul(lhs, rhs, dtype=torch.float32).cpu(), wide @ weight.t())


@pytest.mark.parametrize("accumulate", [False, True])
@pytest.mark.parametrize("counts", COUNTS + [[128], [1000, 0, 20]], ids=str)
@pytest.mark.parametrize(("rows", "columns"), [(1, 1), (100, 70), (256, 256), (300, 520)])
def test_weight_gradients_of_whole_numbers(counts, rows, columns, accumulate, device):
    if len(counts) > 100 and rows * columns > 100 * 400:
        pytest.skip("large on the CPU")
    generator = torch.Generator().manual_seed(rows + columns)
    sparse_map = _map(counts, device, phantom=128)
    real = _real(sparse_map)
    operands = []
    for size in (rows, columns):
        _, values = _whole(generator, (size, max(sparse_map.num_rows, 1)), device)
        values = values.t() * real[:, None]
        operands.append((block_quantize_transposed(values.contiguous().to(device), sparse_map=sparse_map), values))
    (lhs, a), (rhs, b) = operands
    # What lies behind the last expert is not looked at.
    end = int(sparse_map.expert_ends[-1])
    for tensor in (lhs, rhs):
        tensor.values[:, end:], tensor.scales[end // 128 :] = 0x7F, 255
    expected = torch.zeros(len(counts) * rows, columns)
    before = torch.randint(-8, 9, expected.shape, generator=generator).float()
    for expert, begin, past in _experts(sparse_map):
        expected[expert * rows : (expert + 1) * rows] = a[begin:past].t() @ b[begin:past]
    if accumulate:
        expected += before
    _assert_exact(expected)
    for dtype in DTYPES:
        for offset in (0, 8, 3):  # the whole, and columns in the middle of wider rows, aligned to vectors and not
            around = torch.full((len(counts) * rows, columns + 2 * offset), -7.0, dtype=dtype, device=device)
            out = around[:, offset : offset + columns]
            out.copy_(before if accumulate else torch.full_like(before, float("nan")))
            assert block_input_row_sparse_matmul(lhs, rhs, sparse_map, out=out, accumulate=accumulate) is out
            assert torch.equal(out.cpu(), expected.to(dtype))
            assert (around[:, :offset] == -7).all() and (around[:, offset + columns :] == -7).all()


# ---- the activation --------------------------------------------------------------------------------------
def _near(ours: BlockScaledTensor, expected: torch.Tensor, error: torch.Tensor) -> None:
    """`ours` holds `expected` quantised where that is known to within `error`: next to a border either side is right, at most a step apart. A
    block's scale is known but for a largest magnitude at the border of the next scale."""
    elements, scales = block_oracle.quantize(expected)
    blocks = torch.nn.functional.pad(expected.abs(), (0, -expected.size(1) % 128)).unflatten(1, (-1, 128)).amax(-1)
    slack = torch.nn.functional.pad(error, (0, -expected.size(1) % 128)).unflatten(1, (-1, 128)).amax(-1)
    lower, upper = (block_oracle.quantize((blocks + sign * slack).clamp_min(0).flatten()[:, None])[1].view(scales.shape) for sign in (-1, 1))
    bytes_ = ours.scales[:, : ours.rows].t().cpu().long()
    assert ((bytes_ >= lower) & (bytes_ <= upper)).all()
    step = torch.exp2(torch.maximum(torch.floor(torch.log2(expected.abs() + error + 1e-300)), (bytes_ - 127 - 6).repeat_interleave(128, 1)[:, : expected.size(1)]) - 3)
    assert ((_values(ours) - expected).abs() <= step / 2 + error + 1e-45).all()
    # Where the error is below 2^-12 of the value (it is not where the activation's tail is lost in its rounding, as gelu's is in 1 + tanh), it reaches over the one
    # border in a step, at least 2^-4 of the value wide, in 2 * 2^-12 / 2^-4 = 2^-7 of all cases: twice as many for chance.
    sure = error <= 2.0**-12 * expected.abs()
    assert ((_values(ours) != block_oracle.values_of(elements, scales)) & sure).sum() <= 2.0**-6 * sure.sum() + 1
    padding = ours.values.cpu()[:, expected.size(1) :]
    assert (padding == 0).all()


# Hardware exponentials and reciprocals are good to a few units in the last place of fp32, of values up to the size of the argument's: the error of act(x) and
# act'(x) is below 2^-19 (1 + |x|) (squares: |x|^2 2^-23), each product adds 2^-24 of itself.
def _activation_error(x: torch.Tensor) -> torch.Tensor:
    return 2.0**-19 * (1 + x.abs() + x * x / 16)


@pytest.mark.parametrize(("gated", "ffn"), [(True, 128), (True, 384), (False, 1), (False, 200), (False, 256)])
@pytest.mark.parametrize("activation", ACTIVATIONS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("counts", [None, [130, 0, 1]], ids=str)
def test_activation_there_and_back(counts, dtype, activation, gated, ffn, device):
    generator = torch.Generator().manual_seed(ffn)
    sparse_map = None if counts is None else _map(counts, device, phantom=128)
    rows = 70 if counts is None else sparse_map.num_rows
    real = torch.ones(rows, dtype=torch.bool) if counts is None else _real(sparse_map)
    input_ = (torch.randn(rows, ffn * (1 + gated), generator=generator) * torch.exp2(torch.randint(-2, 3, (rows, 1), generator=generator))).to(dtype)
    grad = torch.randn(rows, ffn, generator=generator).to(dtype)
    bad = torch.where(real[:, None], 0.0, float("nan"))
    output, checkpoint = block_activation_forward((input_ + bad).to(device, dtype), gated, activation, sparse_map)
    x, g = (torch.where(real[:, None], t.double(), 0.0) for t in (input_, grad))
    _assert_stored(checkpoint, x)
    up = x[:, ffn:].abs() if gated else torch.ones(())
    _near(output, plain_activation(x, gated, activation), _activation_error(x[:, :ffn]) * up * real[:, None])

    ours = block_activation_backward((grad + bad).to(device, dtype), checkpoint, gated, activation, sparse_map)
    kept = block_oracle.kept(x)
    up = kept[:, ffn:].abs() if gated else torch.ones(())
    error = _activation_error(kept[:, :ffn])
    expected = block_oracle.activation_gradient(g, kept, gated, activation)
    errors = error * up * g.abs()
    errors = torch.cat((errors, error * g.abs()), dim=1) if gated else errors
    result = plain_activation(kept, gated, activation)
    _near(ours[0], expected, errors)
    _near(ours[1], expected.t(), errors.t())
    _near(ours[2], result.t(), (error * up * real[:, None]).t())


def test_gradient_against_differences(device):
    """The gradient is that of the forward at what the checkpoint holds: central differences of the forward in 64 bits, within a step of e4m3."""
    generator = torch.Generator().manual_seed(2)
    input_ = torch.randn(40, 256, generator=generator)
    _, checkpoint = block_activation_forward(input_.to(device), True, "silu")
    grad, _, _ = block_activation_backward(torch.ones(40, 128, device=device), checkpoint, True, "silu")
    kept, step = _values(checkpoint), 1e-5
    differences = torch.empty_like(kept)
    for part in (slice(0, 128), slice(128, 256)):
        moved = torch.zeros_like(kept)
        moved[:, part] = step
        differences[:, part] = (plain_activation(kept + moved, True, "silu") - plain_activation(kept - moved, True, "silu")) / (2 * step)
    largest = differences.unflatten(1, (2, 128)).abs().amax(-1).repeat_interleave(128, 1)
    assert ((_values(grad) - differences).abs() <= 2.0**-4 * differences.abs() + 2.0**-17 * largest + 1e-6).all()


# ---- the MLP ---------------------------------------------------------------------------------------------
def _mlp_inputs(tokens, hidden, ffn, experts, slots, gated, dtype, device, seed=0):
    generator = torch.Generator().manual_seed(seed)
    input_ = torch.randn(tokens, hidden, generator=generator).to(dtype)
    logits = torch.randn(tokens, experts, generator=generator)
    logits[:, -1] = -10.0  # an expert without tokens
    top, top_experts = logits.topk(slots, dim=-1)
    weights = [(torch.randn(experts * rows, hidden, generator=generator) * 0.05).to(dtype) for rows in (ffn * (1 + gated), ffn)]
    grad = torch.randn(tokens, hidden, generator=generator).to(dtype)
    return input_, top.softmax(-1), top_experts, *weights, grad


def _difference(ours: torch.Tensor, theirs: torch.Tensor) -> float:
    return ((ours.detach().cpu().double() - theirs).norm() / theirs.norm()).item()


# Where an fp32 sum and the exact one lie on two sides of a border, a value of 8 bits differs by a step of 2^-3 of itself: with sums that differ by d of
# themselves that is d / 2^-3 of the values, and the rms of all their differences sqrt(d 2^-3). Sums are good to 2^-13, with the roundings to half precision
# that fall to the other side on the way (one in 2^4 or so, by 2^-9): sqrt(2^-13 2^-3) = 2^-8 per quantisation, of which three or four lie behind one
# another, and half a step of the result (bf16: 2^-9) on top.
MLP_TOLERANCE = 1e-2


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize(("gated", "activation"), [(True, "silu"), (False, "gelu"), (True, "squared_relu")])
@pytest.mark.parametrize(("tokens", "hidden", "ffn", "experts", "slots"), [(1, 128, 128, 4, 1), (70, 200, 256, 5, 2), (600, 264, 384, 4, 2)])
def test_mlp_step(tokens, hidden, ffn, experts, slots, gated, activation, dtype, device):
    inputs = _mlp_inputs(tokens, hidden, ffn, experts, slots, gated, dtype, device)
    input_, scores, top_experts, weight_1, weight_2, grad = inputs
    expected = block_oracle.mlp_step(input_, scores, top_experts, weight_1, weight_2, experts, gated, activation, grad, dtype)
    x, s = input_.to(device).requires_grad_(True), scores.to(device).requires_grad_(True)
    weights = [attach_grad_buffer(w.to(device).requires_grad_(True)) for w in (weight_1, weight_2)]
    sparse_map = get_sparse_map(top_experts.to(device), experts)
    for quantized in (None, block_quantize_expert_weights(*weights, experts)):
        for weight in weights:
            weight.grad_buffer.fill_(float("nan"))
            weight.param_grad_is_zero = True
        x.grad = s.grad = None
        output = block_mlp(x, s, *weights, quantized, gated=gated, activation_type=activation, sparse_map=sparse_map)
        output.backward(grad.to(device))
        ours = {"output": output, "grad_input": x.grad, "grad_scores": s.grad, "grad_weight_1": weights[0].grad_buffer, "grad_weight_2": weights[1].grad_buffer}
        for name, theirs in expected.items():
            assert _difference(ours[name], theirs) <= MLP_TOLERANCE, name
    # A second batch's gradients are added.
    first = [weight.grad_buffer.clone() for weight in weights]
    block_mlp(x, s, *weights, gated=gated, activation_type=activation, sparse_map=sparse_map).backward(grad.to(device))
    for weight, before in zip(weights, first):
        assert _difference(weight.grad_buffer, 2 * before.cpu().double()) <= torch.finfo(dtype).eps
    # Inference has the same result, to the bit, and no backward.
    inference = block_mlp(x, s, *weights, gated=gated, activation_type=activation, sparse_map=sparse_map, training=False)
    assert torch.equal(inference, output)
    with pytest.raises(RuntimeError, match="inference"):
        inference.sum().backward()
