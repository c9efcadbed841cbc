"""Microscaled values, the products with expert weights of 4 bits and the expert MLP on them, against the oracle in 64 bits."""

import pytest
import torch

from fast_llm_amd.functional import microscaling
from fast_llm_amd.functional.microscaling import (
    MicroscaledTensor, mx_copy_dense_to_sparse, mx_dequantize, mx_mlp, mx_quantize, mx_quantize_expert_weights, mx_sparse_matmul,
    mx_sparse_matmul_activation,
)  # fmt: skip
from fast_llm_amd.functional.routing import router
from fast_llm_amd.functional.sparse_copy import SparseMap, copy_sparse_to_dense, get_sparse_map
from oracle import mx_oracle

pytestmark = pytest.mark.gpu

FORMATS = ["e4m3", "e2m1"]
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def _stored(tensor: MicroscaledTensor) -> tuple[torch.Tensor, torch.Tensor]:
    return tensor.values.cpu(), tensor.scales.cpu()


def _values(tensor: MicroscaledTensor) -> torch.Tensor:
    return mx_oracle.unpack(*_stored(tensor), tensor.columns, tensor.format.value)


# ---- quantisation ----------------------------------------------------------------------------------------
@pytest.mark.parametrize("format", FORMATS)
@pytest.mark.parametrize("dtype", DTYPES)
# Whole and partial blocks and groups of 128, odd lengths (a value per load), a row alone, more than a workgroup's share.
@pytest.mark.parametrize(("rows", "columns"), [(1, 32), (1, 1), (3, 33), (5, 100), (2, 136), (33, 1416), (7, 4100), (130, 2048), (9, 257)])
def test_quantize_and_back(rows, columns, dtype, format, device):
    generator = torch.Generator().manual_seed(rows + columns)
    values = (torch.randn(rows, columns, generator=generator) * torch.exp2(torch.randint(-8, 9, (rows, 1), generator=generator))).to(dtype)
    quantized = mx_quantize(values.to(device), format)
    elements, scales = mx_oracle.quantize(values, format)
    for ours, theirs in zip(_stored(quantized), mx_oracle.pack(elements, scales, format)):
        assert torch.equal(ours, theirs)
    for back in DTYPES:
        assert torch.equal(mx_dequantize(quantized, back).cpu(), mx_oracle.values_of(elements, scales).to(back))
    if format == "e4m3":
        assert torch.equal(quantized.elements.double().cpu(), elements)
        assert torch.equal(quantized.block_scales.view(torch.uint8).cpu().long(), scales)


@pytest.mark.parametrize("format", FORMATS)
@pytest.mark.parametrize("columns", [256, 255])
def test_quantize_at_the_edges(columns, format, device):
    """Zeros of both signs, subnormal values, the largest ones, ties and borders of saturation, infinities and NaN, a block each."""
    values = torch.zeros(2, columns)
    values[0, 1] = -0.0
    values[0, 32:36] = torch.tensor([2.0**-149, -(2.0**-140), 2.0**-126, 2.0**-130])
    values[0, 64:68] = torch.tensor([torch.finfo(torch.float32).max, -1e38, 1e-38, 1.0])
    grid = torch.tensor(mx_oracle.E2M1)
    values[0, 96:103] = (grid[1:] + grid[:-1]) / 2
    values[0, 103] = 7.99
    values[0, 128:136] = 256 + 8 * torch.arange(8)  # ties of e4m3 between 256 and 320
    values[0, 136:140] = torch.tensor([448.0, 463.99, 464.0, 511.9])
    values[1, :3] = torch.tensor([1.0, float("inf"), 3.0])
    values[1, 40:42] = torch.tensor([float("nan"), float("-inf")])
    values[1, 64] = float("nan")
    quantized = mx_quantize(values.to(device), format)
    for ours, theirs in zip(_stored(quantized), mx_oracle.pack(*mx_oracle.quantize(values, format), format)):
        assert torch.equal(ours, theirs)
    back = mx_dequantize(quantized).cpu()
    assert torch.equal(torch.isnan(back), torch.isnan(mx_oracle.values_of(*mx_oracle.quantize(values, format))))


@pytest.mark.parametrize("format", FORMATS)
def test_quantize_strides_and_shapes(format, device):
    wide = torch.randn(40, 300, generator=torch.Generator().manual_seed(2)).to(device)
    for view in (wide[:, 8:200], wide[3:, 1:130], wide[::2], wide.t(), wide[:, ::3], wide[:0], wide.view(4, 10, 300)):
        plain = mx_quantize(view.contiguous(), format)
        ours = mx_quantize(view, format)
        assert ours.shape == (view.numel() // view.size(-1) if view.numel() else 0, view.size(-1))
        assert torch.equal(ours.values, plain.values) and torch.equal(ours.scales, plain.scales)
    rows = mx_quantize(wide, format)[5:9]
    assert torch.equal(mx_dequantize(rows), mx_dequantize(mx_quantize(wide, format))[5:9])
    assert mx_dequantize(rows[:0]).shape == (0, 300)


def test_quantize_more_than_a_gigabyte_of_values(device):
    """Byte offsets past 31 and 32 bits: rows at the end of 4.3 GB of input."""
    rows, columns = 1 << 20, 2056
    values = torch.zeros(rows, columns, dtype=torch.bfloat16, device=device)
    tail = torch.randn(300, columns, generator=torch.Generator().manual_seed(3)).bfloat16()
    values[-300:] = tail.to(device)
    quantized = mx_quantize(values, "e4m3")
    theirs = mx_oracle.pack(*mx_oracle.quantize(tail, "e4m3"), "e4m3")
    assert torch.equal(quantized.values[-300:].cpu(), theirs[0]) and torch.equal(quantized.scales[-300:].cpu(), theirs[1])
    assert not quantized.values[: rows - 300 : 1021].any()
    assert torch.equal(mx_dequantize(quantized, torch.bfloat16)[-300:].cpu(), mx_oracle.values_of(*mx_oracle.quantize(tail, "e4m3")).bfloat16())


@pytest.mark.parametrize("format", FORMATS)
@pytest.mark.parametrize(("tokens", "slots", "columns"), [(1, 1, 32), (70, 3, 200), (5, 8, 2048)])
def test_dispatch(tokens, slots, columns, format, device):
    generator = torch.Generator().manual_seed(tokens)
    experts = 6
    top_experts = torch.randint(-1, experts + 1, (tokens, slots), generator=generator)  # some select no expert
    rows = mx_quantize(torch.randn(tokens, columns, generator=generator).to(device), format)
    sparse_map = get_sparse_map(top_experts.to(device), experts)
    sparse = mx_copy_dense_to_sparse(rows, sparse_map)
    assert sparse.shape == (sparse_map.num_rows, columns) and sparse.format == rows.format
    for token, targets in enumerate(sparse_map.sparse_rows.cpu().tolist()):
        for target in targets:
            if target >= 0:
                assert torch.equal(sparse.values[target], rows.values[token]) and torch.equal(sparse.scales[target], rows.scales[token])


# ---- products --------------------------------------------------------------------------------------------
def _whole(generator, shape, device, format) -> MicroscaledTensor:
    """Small whole numbers, of which both formats hold every one whatever the block's scale."""
    table = torch.tensor([0.0, 1, -1, 2, -2, 3, -3, 4, -4, 6, -6])
    values = table[torch.randint(0, len(table), shape, generator=generator)]
    quantized = mx_quantize(values.to(device), format)
    assert torch.equal(_values(quantized), values.double())
    return quantized


def _map(counts: list[int], device, index_dtype=torch.int32, block: int = 128, phantom: int = 0) -> SparseMap:
    ends, pad_begins, begin = [], [], 0
    for count in counts:
        pad_begins.append(begin + count)
        begin += -(-count // block) * block
        ends.append(begin)
    to = dict(dtype=index_dtype, device=device)
    return SparseMap(None, torch.tensor(ends, **to), torch.tensor(pad_begins, **to), None, begin + phantom, sum(counts), len(counts), None)


def _real_rows(sparse_map: SparseMap) -> list[tuple[int, int, int]]:
    ends, pad_begins = sparse_map.expert_ends.tolist(), sparse_map.expert_pad_begins.tolist()
    return [(e, begin, end) for e, (begin, end) in enumerate(zip([0] + ends[:-1], pad_begins))]


# Experts without rows, with one, a part of a block of 32, and on both sides of the tiles of 256; many experts.
COUNTS = [[1], [0, 1, 0], [31, 0, 33, 2], [300, 0, 257, 1, 512], [256, 700], [0, 0], [3] * 70 + [0] * 60 + [40]]


@pytest.mark.parametrize("counts", COUNTS, ids=str)
# Reductions of one group of 128 and of parts of it, of less than, exactly and more than four slices, with a last chunk of 128; columns
# of parts of blocks of 4 and 32, and on both sides of the tiles.
@pytest.mark.parametrize(("inner", "columns"), [(1, 1), (96, 33), (128, 64), (384, 100), (512, 256), (640, 130), (1416, 516)])
@pytest.mark.parametrize("format", FORMATS)
def test_whole_numbers_are_multiplied_exactly(counts, inner, columns, format, device):
    if len(counts) > 100 and inner * columns > 100 * 400:
        pytest.skip("large on the CPU")
    generator = torch.Generator().manual_seed(inner + columns)
    sparse_map = _map(counts, device, phantom=128)
    lhs = _whole(generator, (sparse_map.num_rows, inner), device, format)
    rhs = _whole(generator, (len(counts) * columns, inner), device, "e2m1")
    out = torch.full((sparse_map.num_rows, columns), -7.0, device=device)
    assert mx_sparse_matmul(lhs, rhs, sparse_map, out) is out
    expected = torch.full_like(out, -7.0).cpu()
    wide, weight = _values(lhs).float(), _values(rhs).float().view(len(counts), columns, inner)
    for expert, begin, end in _real_rows(sparse_map):
        expected[begin:end] = wide[begin:end] @ weight[expert].t()  # below 2^24: exact
    assert torch.equal(out.cpu(), expected)  # what no token has is as it was
    half = mx_sparse_matmul(lhs, rhs, sparse_map, dtype=torch.bfloat16)
    for _, begin, end in _real_rows(sparse_map):
        assert torch.equal(half[begin:end].cpu(), expected[begin:end].bfloat16())


@pytest.mark.parametrize("many", [False, True])
@pytest.mark.parametrize("format", FORMATS)
@pytest.mark.parametrize("index_dtype", [torch.int16, torch.int32, torch.int64])
def test_strides_and_index_types(index_dtype, format, many, device):
    generator = torch.Generator().manual_seed(5)
    inner, columns = 512, 132
    # Boundaries of any kind.
    sparse_map = _map([300, 259, 5] if many else [9, 0, 30], device, index_dtype, block=1, phantom=3)
    experts = sparse_map.num_experts
    lhs = _whole(generator, (2 * sparse_map.num_rows, inner), device, format)
    rhs = _whole(generator, (2 * experts * columns, inner), device, "e2m1")
    plain = mx_sparse_matmul(*(MicroscaledTensor(t.values[::2].contiguous(), t.scales[::2].contiguous(), inner, t.format) for t in (lhs, rhs)),
                             sparse_map, dtype=torch.float16)  # fmt: skip
    for offset in (0, 1):  # columns in the middle of wider rows, aligned to groups of four and not
        wide = torch.full((sparse_map.num_rows, 2 * columns), -7.0, dtype=torch.float16, device=device)
        out = wide[:, 8 + offset : 8 + offset + columns]
        operands = [MicroscaledTensor(t.values[::2], t.scales[::2], inner, t.format) for t in (lhs, rhs)]
        mx_sparse_matmul(*operands, sparse_map, out)
        for _, begin, end in _real_rows(sparse_map):
            assert torch.equal(out[begin:end], plain[begin:end])
        assert (wide[:, : 8 + offset] == -7).all() and (wide[:, 8 + offset + columns :] == -7).all() and (out[-3:] == -7).all()


def _tolerance(lhs: torch.Tensor, weight: torch.Tensor, expected: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    """The matrix instruction aligns the 64 products that it adds, and the sum so far, to the largest of them and drops what lies
    under its last bit, at 2^-17 of it or below: per product of the reduction at most that; then the result's rounding, half a step."""
    largest = lhs.abs().amax(-1, keepdim=True) * weight.abs().amax(-1)[None]
    return 2.0**-17 * lhs.size(-1) * torch.maximum(largest, expected.abs()) + torch.finfo(dtype).eps / 2 * expected.abs() + 1e-30


@pytest.mark.parametrize("counts", [[40, 3], [300, 257]], ids=str)
@pytest.mark.parametrize(("inner", "columns"), [(200, 70), (1024, 300)])
@pytest.mark.parametrize("format", FORMATS)
@pytest.mark.parametrize("dtype", DTYPES)
def test_products_of_values_of_all_sizes(counts, inner, columns, format, dtype, device):
    generator = torch.Generator().manual_seed(inner)
    sparse_map = _map(counts, device)
    # Features and rows of unlike size, so that neighbouring blocks have different scales.
    sizes = torch.exp2(torch.randint(-3, 4, (1, inner), generator=generator))
    lhs = mx_quantize((torch.randn(sparse_map.num_rows, inner, generator=generator) * sizes).to(device), format)
    rhs = mx_quantize((torch.randn(len(counts) * columns, inner, generator=generator) * 0.02).to(device), "e2m1")
    # What padding rows hold is not looked at.
    for _, _, end in _real_rows(sparse_map):
        lhs.values[end : -(-end // 128) * 128] = 0x7F
        lhs.scales[end : -(-end // 128) * 128] = 255
    out = mx_sparse_matmul(lhs, rhs, sparse_map, dtype=dtype)
    rows, weight = _values(lhs), _values(rhs).view(len(counts), columns, inner)
    for expert, begin, end in _real_rows(sparse_map):
        expected = rows[begin:end] @ weight[expert].t()
        assert ((out[begin:end].cpu().double() - expected).abs() <= _tolerance(rows[begin:end], weight[expert], expected, dtype)).all()


@pytest.mark.parametrize("counts", [[40, 0, 3], [300, 257, 0]], ids=str)
@pytest.mark.parametrize(("inner", "columns"), [(96, 33), (512, 160), (640, 256)])
@pytest.mark.parametrize("format", FORMATS)
@pytest.mark.parametrize(("gated", "activation"), [(True, "identity"), (False, "relu"), (True, "relu"), (False, "squared_relu")])
def test_activation_is_microscaled_from_exact_sums(counts, inner, columns, format, gated, activation, device):
    """Whole numbers below 2^24 up to the activation's result: the bytes are known."""
    generator = torch.Generator().manual_seed(columns)
    sparse_map = _map(counts, device)
    lhs = _whole(generator, (sparse_map.num_rows, inner), device, format)
    rhs = _whole(generator, (len(counts) * columns * (1 + gated), inner), device, "e2m1")
    out = mx_sparse_matmul_activation(lhs, rhs, sparse_map, gated, activation)
    assert out.shape == (sparse_map.num_rows, columns) and out.format == lhs.format
    rows, weight = _values(lhs), _values(rhs).view(len(counts), -1, inner)
    for expert, begin, end in _real_rows(sparse_map):
        result = mx_oracle.activation(rows[begin:end] @ weight[expert].t(), gated, activation)
        assert result.abs().max() < 2**24 if len(result) else True
        theirs = mx_oracle.pack(*mx_oracle.quantize(result, format), format)
        assert torch.equal(out.values[begin:end].cpu(), theirs[0]) and torch.equal(out.scales[begin:end].cpu(), theirs[1])


@pytest.mark.parametrize("counts", [[33], [290]], ids=str)
@pytest.mark.parametrize("format", FORMATS)
def test_blocks_of_nan_reach_their_rows_only(counts, format, device):
    generator = torch.Generator().manual_seed(9)
    sparse_map = _map(counts, device)
    values = torch.randn(sparse_map.num_rows, 512, generator=generator)
    values[5, 70], values[20, 511] = float("nan"), float("inf")
    weight = torch.randn(64, 512, generator=generator)
    weight[40, 0] = float("inf")
    out = mx_sparse_matmul(mx_quantize(values.to(device), format), mx_quantize(weight.to(device), "e2m1"), sparse_map)[: counts[0]].cpu()
    expected = torch.zeros(counts[0], 64, dtype=torch.bool)
    expected[5], expected[20], expected[:, 40] = True, True, True
    assert torch.equal(torch.isnan(out), expected)
    activated = mx_sparse_matmul_activation(mx_quantize(values.to(device), format), mx_quantize(weight.to(device), "e2m1"), sparse_map, True, "silu")
    bad = (activated.scales[: counts[0], 0] == 255).cpu()  # up 8 (row 40) makes the one block of every row NaN
    assert bad.all()


def test_dense_product(device):
    generator = torch.Generator().manual_seed(1)
    for rows in (1, 300):
        lhs, rhs = _whole(generator, (rows, 640), device, "e4m3"), _whole(generator, (96, 640), device, "e2m1")
        assert torch.equal(mx_sparse_matmul(lhs, rhs, dtype=torch.float32).cpu().double(), _values(lhs) @ _values(rhs).t())


# ---- the expert MLP --------------------------------------------------------------------------------------
@pytest.mark.parametrize("few", [True, False])
# One workgroup row per entry or per expert; more rows of an expert than a wavefront's block.
@pytest.mark.parametrize(("tokens", "experts", "slots"), [(1, 8, 2), (3, 64, 6), (17, 4, 1), (40, 6, 3), (150, 5, 2)])
@pytest.mark.parametrize(("hidden", "ffn"), [(64, 40), (136, 128), (512, 520)])
@pytest.mark.parametrize(("format", "gated", "activation"), [("e4m3", True, "relu"), ("e2m1", False, "squared_relu"), ("e4m3", False, "identity")])
def test_mlp_with_exact_activations(few, tokens, experts, slots, hidden, ffn, format, gated, activation, device, monkeypatch):
    """Whole numbers up to the activations, which are rounded as the oracle rounds them; what follows is off by the tolerance of a
    product, a rounding per slot where the rows of layer 2 are stored, and that of the result."""
    monkeypatch.setattr(microscaling, "MX_FEW_TOKENS_ROWS", 10**6 if few else 0)
    generator = torch.Generator().manual_seed(tokens + hidden)
    rows = _whole(generator, (tokens, hidden), device, format)
    weight_1 = _whole(generator, (experts * ffn * (1 + gated), hidden), device, "e2m1")
    weight_2 = _whole(generator, (experts * hidden, ffn), device, "e2m1")
    logits = torch.randn(tokens, experts, generator=generator) + 2 * torch.randn(experts, generator=generator)
    top_logits, top_experts = torch.topk(logits, slots, dim=-1)
    scores = torch.softmax(top_logits, dim=-1)
    if tokens > 1:
        top_experts[1, 0] = -1  # an entry that selects no expert contributes nothing
        top_experts[tokens - 1, slots - 1] = experts
    arguments = (rows, scores.to(device), top_experts.to(device), weight_1, weight_2, experts)
    values = (_values(rows), scores, top_experts, _values(weight_1), _values(weight_2), experts, gated, activation, format)
    expected = mx_oracle.mlp(*values)
    # Of the slots' absolute contributions.
    weights = (values[0].abs(), scores, top_experts, values[3].abs(), values[4].abs(), experts, gated, activation if gated else "identity", format)
    for dtype in (torch.bfloat16, torch.float32):
        output = mx_mlp(*arguments, gated=gated, activation_type=activation, dtype=dtype)
        assert output.dtype == dtype and output.shape == (tokens, hidden)
        bound = mx_oracle.mlp(*weights)
        if activation == "squared_relu":
            weights_squared = (*weights[:7], "squared_relu", format)
            bound = mx_oracle.mlp(*weights_squared)
        tolerance = (2.0**-17 * ffn + torch.finfo(dtype).eps / 2 * 1.1) * bound + torch.finfo(dtype).eps / 2 * expected.abs() + 1e-6
        assert ((output.cpu().double() - expected).abs() <= tolerance).all()


@pytest.mark.parametrize("few", [True, False])
@pytest.mark.parametrize("format", FORMATS)
@pytest.mark.parametrize(("gated", "activation"), [(True, "silu"), (True, "gelu"), (False, "gelu")])
def test_mlp_of_a_layers_values(few, format, gated, activation, device, monkeypatch):
    """An activation next to a border may be rounded to either side: sums that are off by 2^-17 and a step of 2^-3 (e4m3) or 2^-1 (e2m1) make
    that one in 2^13 values, off by half a step at most, so under 2^-6 of the norm together with the roundings to bfloat16."""
    monkeypatch.setattr(microscaling, "MX_FEW_TOKENS_ROWS", 10**6 if few else 0)
    generator = torch.Generator().manual_seed(11)
    tokens, experts, slots, hidden, ffn = 90, 4, 2, 512, 704
    x = torch.randn(tokens, hidden, generator=generator).to(device)
    layer_1 = torch.randn(experts * ffn * (1 + gated), hidden, generator=generator).to(device) * 0.05
    layer_2 = torch.randn(experts * ffn, hidden, generator=generator).to(device) * 0.05
    weight_1, weight_2 = mx_quantize_expert_weights(layer_1, layer_2, experts)
    assert torch.equal(mx_dequantize(weight_2), mx_dequantize(mx_quantize(layer_2.view(experts, ffn, hidden).transpose(1, 2).reshape(-1, ffn), "e2m1")))
    scores, top_experts = torch.topk(torch.rand(tokens, experts, generator=generator), slots)
    rows = mx_quantize(x, format)
    output = mx_mlp(rows, scores.to(device), top_experts.to(device), weight_1, weight_2, experts, gated=gated, activation_type=activation)
    expected = mx_oracle.mlp(_values(rows), scores, top_experts, _values(weight_1), _values(weight_2), experts, gated, activation, format)
    assert output.dtype == torch.bfloat16
    assert (output.cpu().double() - expected).norm() <= 2.0**-6 * expected.norm()
    if format == "e4m3":  # a plain input is quantised first
        plain = mx_mlp(x.bfloat16(), scores.to(device), top_experts.to(device), weight_1, weight_2, experts, gated=gated, activation_type=activation)
        again = mx_mlp(mx_quantize(x.bfloat16()), scores.to(device), top_experts.to(device), weight_1, weight_2, experts, gated=gated, activation_type=activation)
        assert torch.equal(plain, again)


def test_mlp_without_tokens_and_without_a_backward(device):
    weight_1, weight_2 = mx_quantize_expert_weights(torch.randn(2 * 64, 32, device=device), torch.randn(2 * 32, 32, device=device), 2)

    def call(tokens, slots=1, **options):
        x = torch.randn(tokens, 32, device=device, dtype=torch.bfloat16)
        scores, top_experts = torch.ones(tokens, slots, device=device, **options), torch.zeros(tokens, slots, dtype=torch.int64, device=device)
        return mx_mlp(x, scores, top_experts, weight_1, weight_2, 2, gated=True, activation_type="silu")

    assert call(0).shape == (0, 32)
    assert torch.equal(call(3, 0), torch.zeros(3, 32, dtype=torch.bfloat16, device=device))
    assert not call(3).requires_grad
    with pytest.raises(RuntimeError, match="backward"):
        call(3, requires_grad=True).sum().backward()


@pytest.mark.parametrize("tokens", [2, 900])
def test_mlp_replays_from_a_graph_and_runs_on_any_stream(tokens, device):
    generator = torch.Generator().manual_seed(4)
    experts, slots, hidden, ffn = 4, 2, 512, 256
    weight_1, weight_2 = mx_quantize_expert_weights(
        torch.randn(experts * 2 * ffn, hidden, generator=generator).to(device), torch.randn(experts * ffn, hidden, generator=generator).to(device), experts
    )
    inputs = []
    for _ in range(3):
        scores, top_experts = torch.topk(torch.rand(tokens, experts, generator=generator), slots)
        inputs.append([t.to(device) for t in (torch.randn(tokens, hidden, generator=generator).bfloat16(), scores, top_experts)])

    def call(x, scores, top_experts):
        return mx_mlp(x, scores, top_experts, weight_1, weight_2, experts, gated=True, activation_type="silu")

    eager = [call(*arguments) for arguments in inputs]
    assert all(torch.equal(call(*arguments), result) for arguments, result in zip(inputs, eager))  # the same bits again
    other = torch.cuda.Stream()
    other.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(other):
        elsewhere = call(*inputs[0])
    torch.cuda.current_stream().wait_stream(other)
    assert torch.equal(elsewhere, eager[0])
    static = [t.clone() for t in inputs[0]]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        output = call(*static)
    for _ in range(2):
        for arguments, result in zip(inputs, eager):
            for target, source in zip(static, arguments):
                target.copy_(source)
            graph.replay()
            assert torch.equal(output, result)
            assert torch.equal(call(*arguments), result)
            torch.cuda.synchronize()


# ---- calls at the ends of what is allowed ----------------------------------------------------------------
@pytest.mark.parametrize("index_dtype", [torch.int16, torch.int32, torch.int64])
@pytest.mark.parametrize("format", FORMATS)
def test_tiles_take_strides_and_index_types(index_dtype, format, device):
    generator = torch.Generator().manual_seed(5)
    inner, columns = 640, 132
    sparse_map = _map([500, 259, 5], device, index_dtype, block=1, phantom=3)  # boundaries of any kind
    lhs = _whole(generator, (2 * sparse_map.num_rows, inner), device, format)
    rhs = _whole(generator, (2 * 3 * columns, inner), device, "e2m1")
    operands = [MicroscaledTensor(t.values[::2], t.scales[::2], inner, t.format) for t in (lhs, rhs)]
    rows, weight = (_values(t) for t in operands)
    for offset in (0, 1):  # aligned to groups of four and not
        wide = torch.full((sparse_map.num_rows, 2 * columns), -7.0, dtype=torch.bfloat16, device=device)
        mx_sparse_matmul(*operands, sparse_map, wide[:, 8 + offset : 8 + offset + columns])
        expected = torch.full(wide.shape, -7.0, dtype=torch.bfloat16)
        for expert, begin, end in _real_rows(sparse_map):
            product = rows[begin:end] @ weight[expert * columns : (expert + 1) * columns].t()
            expected[begin:end, 8 + offset : 8 + offset + columns] = product.bfloat16()
        assert torch.equal(wide.cpu(), expected)


@pytest.mark.parametrize("format", FORMATS)
# Of tiles of 256 x 256: 156, fewer than CUs; 453, over half a round after a whole one; 297 and 300, under half a round after a whole one, where the
# second halves of an expert's last tile have 40, 2, 0 and 0 rows.
@pytest.mark.parametrize("counts", [[9864, 3201], [30000, 8300], [25000, 130], [20096, 5128, 0]], ids=str)
def test_rounds_of_tiles(counts, format, device):
    generator = torch.Generator().manual_seed(sum(counts))
    inner, columns = 512, 516
    sparse_map = _map(counts, device)
    lhs = _whole(generator, (sparse_map.num_rows, inner), device, format)
    rhs = _whole(generator, (len(counts) * columns, inner), device, "e2m1")
    out = mx_sparse_matmul(lhs, rhs, sparse_map, dtype=torch.float32).cpu()
    rows, weight = _values(lhs).float(), _values(rhs).float().view(len(counts), columns, inner)
    for expert, begin, end in _real_rows(sparse_map):
        assert torch.equal(out[begin:end], rows[begin:end] @ weight[expert].t())


@pytest.mark.parametrize("format", FORMATS)
@pytest.mark.parametrize("of_rows", [True, False])
def test_scales_that_are_far_apart(of_rows, format, device):
    """The rows of scales of one tile lie over 2 GiB of memory, those of a block of 32 rows within 4 GiB."""
    generator = torch.Generator().manual_seed(3)
    lhs, rhs = _whole(generator, (200, 512), device, format), _whole(generator, (200, 512), device, "e2m1")
    plain = mx_sparse_matmul(lhs, rhs, dtype=torch.float32)
    tensor = lhs if of_rows else rhs
    apart = torch.empty(200, 1 << 24, dtype=torch.uint8, device=device)[:, :16]
    apart.copy_(tensor.scales)
    tensor.scales = apart
    assert torch.equal(mx_sparse_matmul(lhs, rhs, dtype=torch.float32), plain)


@pytest.mark.parametrize("rows", [8, 300])
@pytest.mark.parametrize("inner", [128, 640])
def test_scales_that_end_with_their_memory(rows, inner, device):
    generator = torch.Generator().manual_seed(rows + inner)
    lhs, rhs = _whole(generator, (rows, inner), device, "e4m3"), _whole(generator, (64, inner), device, "e2m1")
    expected = _values(lhs) @ _values(rhs).t()
    for tensor in (lhs, rhs):
        memory = torch.empty(tensor.rows, 1 << 16, dtype=torch.uint8, device=device)
        scales = memory[:, memory.size(1) - tensor.scales.size(1) :]
        scales.copy_(tensor.scales)
        tensor.scales = scales
    assert torch.equal(mx_sparse_matmul(lhs, rhs, dtype=torch.float32).cpu().double(), expected)


def test_a_row_by_itself_is_quantised(device):
    row = torch.randn(100, device=device)
    for ours, theirs in zip(_stored(mx_quantize(row)), _stored(mx_quantize(row[None]))):
        assert torch.equal(ours, theirs)
    assert mx_quantize(row.view(2, 1, 50).transpose(0, 2)).shape == (50, 2) and mx_quantize(row.view(2, 50)[:0]).shape == (0, 50)


@pytest.mark.parametrize("format", FORMATS)
@pytest.mark.parametrize("tokens", [3, 200])
def test_two_streams_at_once(tokens, format, device):
    """Calls on two streams share nothing but their inputs."""
    generator = torch.Generator().manual_seed(tokens)
    weight_1, weight_2 = mx_quantize_expert_weights(
        torch.randn(4 * 512, 256, generator=generator).to(device), torch.randn(4 * 256, 256, generator=generator).to(device), 4
    )
    inputs = [torch.randn(tokens, 256, generator=generator).to(device).bfloat16() for _ in range(2)]
    scores, top_experts = (t.to(device) for t in torch.topk(torch.rand(tokens, 4, generator=generator), 2))

    def call(x):
        rows = mx_quantize(x, format)
        return mx_mlp(rows, scores, top_experts, weight_1, weight_2, 4, gated=True, activation_type="silu")

    alone = [call(x) for x in inputs]
    streams = [torch.cuda.Stream(device) for _ in inputs]
    torch.cuda.synchronize()
    results = []
    for _ in range(8):
        for x, stream in zip(inputs, streams):
            with torch.cuda.stream(stream):
                results.append(call(x))
    torch.cuda.synchronize()
    for i, result in enumerate(results):
        assert torch.equal(result, alone[i % 2])


@pytest.mark.parametrize("format", FORMATS)
@pytest.mark.parametrize(("tokens", "experts", "slots"), [(300, 4, 2), (700, 60, 3), (33000, 2, 1)])
@pytest.mark.parametrize("counted", [False, True])
def test_mlp_is_its_operators_one_after_the_other(counted, tokens, experts, slots, format, device, monkeypatch):
    monkeypatch.setattr(microscaling, "MX_FEW_TOKENS_ROWS", 0)
    generator = torch.Generator().manual_seed(tokens)
    hidden, ffn = 264, 200
    weight_1, weight_2 = mx_quantize_expert_weights(
        torch.randn(experts * 2 * ffn, hidden, generator=generator).to(device), torch.randn(experts * ffn, hidden, generator=generator).to(device), experts
    )
    rows = mx_quantize(torch.randn(tokens, hidden, generator=generator).to(device), format)
    logits = torch.randn(tokens, experts, generator=generator).to(device)
    scores, top_experts, _, _, counts = router(logits, slots, return_counts=True)
    if not counted:
        counts, top_experts = None, top_experts.clone()
        top_experts[tokens // 2, 0] = -1
    sparse_map = get_sparse_map(top_experts, experts)
    between = mx_sparse_matmul_activation(mx_copy_dense_to_sparse(rows, sparse_map), weight_1, sparse_map, True, "silu")
    for dtype in DTYPES:
        expected = copy_sparse_to_dense(mx_sparse_matmul(between, weight_2, sparse_map, dtype=dtype), scores.float(), sparse_map)
        output = mx_mlp(
            rows, scores, top_experts, weight_1, weight_2, experts, gated=True, activation_type="silu", dtype=dtype, router_counts=counts
        )
        assert torch.equal(output, expected)


@pytest.mark.parametrize("format", FORMATS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("columns", [7, 8, 9, 31, 100, 129, 511, 515, 1029])
def test_quantize_rows_of_any_length_and_alignment(columns, dtype, format, device):
    generator = torch.Generator().manual_seed(columns)
    values = torch.randn(9, columns, generator=generator).to(dtype)
    elements, scales = mx_oracle.quantize(values, format)
    for stride, offset in ((columns, 1), (columns + 1, 0), (columns + 5, 3)):
        storage = torch.full((9 * stride + offset + 16,), 100.0, dtype=dtype, device=device)
        view = storage[offset : offset + 9 * stride].view(9, stride)[:, :columns]
        view.copy_(values)
        quantized = mx_quantize(view, format)
        for ours, theirs in zip(_stored(quantized), mx_oracle.pack(elements, scales, format)):
            assert torch.equal(ours, theirs)
        assert torch.equal(mx_dequantize(quantized, dtype).cpu(), mx_oracle.values_of(elements, scales).to(dtype))
