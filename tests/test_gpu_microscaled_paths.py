"""
The parts of the kernels for microscaled products that a rule on sizes chooses, each run by cases that are held to it without a GPU
(`test_mx_dispatch.py`): tiles for more than 128 experts, activations and both layers of the MLP on tiles; one, four and eight wavefronts that
share a reduction, by a map and by entries, with more chunks of it each than are fetched with one group of scales.
"""

import pytest
import torch

from fast_llm_amd.functional import microscaling
from fast_llm_amd.functional.microscaling import mx_copy_dense_to_sparse, mx_mlp, mx_sparse_matmul, mx_sparse_matmul_activation
from fast_llm_amd.functional.sparse_copy import copy_sparse_to_dense, get_sparse_map
from oracle import mx_oracle
from tests.mx_values import PRODUCT_UNIT, assert_exact, scaled
from tests.test_gpu_microscaling import _map, _real_rows

pytestmark = pytest.mark.gpu

FORMATS = ["e4m3", "e2m1"]

# ---- tiles -----------------------------------------------------------------------------------------------
# Rows of the experts, block of the map, reduction, columns: experts over and under half a tile, without rows and with one; more tiles than CUs.
MANY_EXPERTS = [
    ([300] * 60 + [100] * 35 + [0] * 20 + [1] * 15, 128, 512, 40),
    ([0] + [300] * 60 + [129] * 40 + [1] * 30, 128, 896, 300),
    ([256] * 150 + [100] * 150, 1, 640, 72),
]
ACTIVATIONS = [([300, 257, 1, 512], 512, 160), ([300, 257, 1, 512], 896, 130), ([500, 140], 768, 260)]
# Tokens, experts, slots, hidden, ffn. The last one's are all of one expert.
MLPS = [(900, 4, 2, 640, 896), (900, 4, 2, 768, 520), (1500, 3, 1, 512, 1100)]

# ---- few rows --------------------------------------------------------------------------------------------
# Rows of the experts, reduction, columns, wavefronts that share the reduction.
BY_MAP = [
    ([40, 3], 2304, 70, 8),  # 9 chunks: three wavefronts have none
    ([70, 0], 9000, 33, 8),  # 36: five each
    ([33, 5], 1416, 100, 4),
    ([34, 40], 4360, 12320, 4),  # 18: five each, the last three
    ([3, 33], 640, 200, 1),
    ([33, 1], 1416, 49160, 1),  # six
]
# Tokens, experts, slots, hidden, ffn, gated, wavefronts that share the reductions of the two layers.
BY_ENTRIES = [
    (1, 8, 2, 2304, 1100, True, 8, 4),  # a row of workgroups per entry
    (1, 64, 1, 1416, 9000, False, 4, 8),
    (40, 2, 2, 9000, 2100, False, 8, 8),  # per expert, with more than 32 rows
    (45, 2, 1, 2304, 2100, True, 8, 8),
    (40, 64, 2, 4360, 416, False, 4, 1),
    (40, 64, 2, 1416, 1536, True, 1, 4),
    (40, 64, 2, 1600, 1300, False, 4, 1),
]


def _check_products(counts, block, inner, columns, format, gates, device):
    """The product and, for every one of `gates`, the activation's result to the byte."""
    generator = torch.Generator(device).manual_seed(inner + columns)
    sparse_map, experts = _map(counts, device, block=block, phantom=5), len(counts)
    lhs, rows = scaled(generator, (sparse_map.num_rows, inner), format)
    rhs, weight = scaled(generator, (experts * columns, inner), "e2m1")
    out = torch.full((sparse_map.num_rows, columns), -7.0, device=device)
    mx_sparse_matmul(lhs, rhs, sparse_map, out)
    expected = torch.full_like(out, -7.0)
    for (_, begin, end), part in zip(_real_rows(sparse_map), weight.chunk(experts)):
        expected[begin:end] = sums = rows[begin:end] @ part.t()
        assert_exact(sums)
    assert torch.equal(out, expected)
    for gated, activation in gates:
        if gated:
            rhs, weight = scaled(generator, (2 * experts * columns, inner), "e2m1")
        result = mx_sparse_matmul_activation(lhs, rhs, sparse_map, gated, activation)
        for (_, begin, end), part in zip(_real_rows(sparse_map), weight.chunk(experts)):
            values = mx_oracle.activation((rows[begin:end] @ part.t()).cpu(), gated, activation)
            assert values.numel() == 0 or values.abs().max() < 2**24 * PRODUCT_UNIT**2
            stored, scales = mx_oracle.pack(*mx_oracle.quantize(values, format), format)
            assert torch.equal(result.values[begin:end].cpu(), stored) and torch.equal(result.scales[begin:end].cpu(), scales)


@pytest.mark.parametrize("format", FORMATS)
@pytest.mark.parametrize("case", MANY_EXPERTS, ids=["130", "131", "300"])
def test_tiles_of_more_than_128_experts(case, format, device):
    counts, block, inner, columns = case
    _check_products(counts, block, inner, columns, format, [(True, "relu"), (False, "identity")], device)


@pytest.mark.parametrize("format", FORMATS)
@pytest.mark.parametrize(("counts", "inner", "columns", "split"), BY_MAP)
def test_few_rows_by_a_map(counts, inner, columns, split, format, device):
    gates = [(False, "relu")]
    if inner < 9000:  # the product of a gate and an up is not exact there
        gates.append((True, "relu"))
    _check_products(counts, 128, inner, columns, format, gates, device)


@pytest.mark.parametrize("format", FORMATS)
@pytest.mark.parametrize(("gated", "activation"), [(True, "silu"), (False, "silu"), (True, "gelu"), (False, "gelu")])
@pytest.mark.parametrize(("counts", "inner", "columns"), ACTIVATIONS)
def test_smooth_activations_of_tiles(counts, inner, columns, gated, activation, format, device):
    """
    The sums, of about 1, are exact. v_exp_f32 and v_rcp_f32 are off by an ulp, so a sigmoid or tanh by 2^-20 at these arguments (up to 32: five bits
    of the exponential's), and gelu's 1 + tanh by that in absolute terms: results lie within 2^-19 of their argument's (times up's) size. What
    they are rounded to then lies between what both ends of that are rounded to (with the scales of the one or of the other).
    """
    generator = torch.Generator(device).manual_seed(inner + columns)
    sparse_map, experts = _map(counts, device), len(counts)
    lhs, rows = scaled(generator, (sparse_map.num_rows, inner), format)
    rhs, weight = scaled(generator, (experts * columns * (1 + gated), inner), "e2m1", 2.0**-6)
    out = mx_sparse_matmul_activation(lhs, rhs, sparse_map, gated, activation)
    for (_, begin, end), part in zip(_real_rows(sparse_map), weight.chunk(experts)):
        sums = (rows[begin:end] @ part.t()).cpu()
        assert_exact(sums, 2.0**-6)
        assert sums.abs().max() < 16 and sums.std() > 0.5
        result = mx_oracle.activation(sums, gated, activation)
        slack = 2.0**-19 * mx_oracle.activation(sums, gated, "identity").abs()
        ends = [mx_oracle.values_of(*mx_oracle.quantize(result + sign * slack, format)) for sign in (-1, 0, 1)]
        low, high = torch.stack(ends).amin(0), torch.stack(ends).amax(0)
        ours = mx_oracle.unpack(out.values[begin:end].cpu(), out.scales[begin:end].cpu(), columns, format)
        assert ((low <= ours) & (ours <= high)).all()
        # So nearly all are known exactly. Not where a result is next to nothing: sums have a deviation of at most 3.5 sqrt(896) / 2^6 = 1.6, one in 30
        # is below -3, where gelu is under 2^-8 and the slack may be half of the smallest step beside a block's largest value.
        assert (low == high).double().mean() > 0.95


def expected_mlp(x, first, second, scores, top_experts, experts, gated, activation, format):
    """
    In fp64: (the output, the slots' absolute contributions, what layer 2 may drop). Layer 1's sums and what the activation makes of them are exact, so its
    bytes are the oracle's. Layer 2 may drop, of each of its products, what lies under 2^-17 of the largest term or partial sum of its
    instruction (of a part of the reduction: twice the largest sum from its start on).
    """
    hidden, ffn = second.size(0) // experts, second.size(1)
    expected, absolute, room = (torch.zeros(len(x), hidden, dtype=torch.float64, device=x.device) for _ in range(3))
    for e, (gates_and_ups, part) in enumerate(zip(first.chunk(experts), second.chunk(experts))):
        token, slot = torch.where(top_experts == e)
        if not len(token):
            continue
        sums = x[token] @ gates_and_ups.t()
        assert_exact(sums)
        result = mx_oracle.activation(sums.cpu(), gated, activation)
        assert result.abs().max() < 2**24 * PRODUCT_UNIT**2
        act = mx_oracle.values_of(*mx_oracle.quantize(result, format)).to(x.device)
        largest = act.abs().amax(1, keepdim=True) * part.abs().amax(1)[None]
        sums, score, chunks = torch.zeros_like(largest), scores[token, slot, None].double(), []
        for start in range(0, ffn, 256):
            before = sums.clone()
            for step in range(start, min(start + 256, ffn), 64):
                sums += act[:, step : step + 64] @ part[:, step : step + 64].t()
                largest = torch.maximum(largest, 2 * sums.abs())
            if start + 256 <= ffn:
                chunks.append((sums - before).abs())
        # A chunk of 256 that is left out, or has twice its scale, shows in the expert's result.
        assert all((chunk > 2 * 2.0**-17 * ffn * largest).any() for chunk in chunks)
        expected.index_add_(0, token, sums * score)
        absolute.index_add_(0, token, sums.abs() * score)
        room.index_add_(0, token, 2.0**-17 * ffn * largest * score)
    return expected, absolute, room


def _check_mlp(tokens, experts, slots, hidden, ffn, gated, activation, top_experts, format, dtypes, device):
    generator = torch.Generator(device).manual_seed(tokens + hidden)
    rows, x = scaled(generator, (tokens, hidden), format)
    weight_1, first = scaled(generator, (experts * ffn * (1 + gated), hidden), "e2m1")
    weight_2, second = scaled(generator, (experts * hidden, ffn), "e2m1", 2.0**-12)  # results within fp16's range
    scores = torch.rand(tokens, slots, generator=generator, device=device)
    expected, absolute, room = expected_mlp(x, first, second, scores, top_experts, experts, gated, activation, format)
    for dtype in dtypes:
        output = mx_mlp(rows, scores, top_experts, weight_1, weight_2, experts, gated=gated, activation_type=activation, dtype=dtype)
        half_step = torch.finfo(dtype).eps / 2
        # A rounding per slot where rows are stored in the output's type, one of the result, and those of the sums in fp32.
        tolerance = room * 1.01 + (half_step + (slots + 1) * 2.0**-24) * absolute * 1.01 + half_step * expected.abs()
        tolerance += (slots + 1) * torch.finfo(dtype).smallest_normal
        assert ((output.double() - expected).abs() <= tolerance).all()


@pytest.mark.parametrize("format", FORMATS)
@pytest.mark.parametrize(("gated", "activation"), [(True, "relu"), (False, "squared_relu"), (False, "identity")])
@pytest.mark.parametrize("case", range(len(MLPS)))
def test_both_layers_on_tiles(case, gated, activation, format, device, monkeypatch):
    monkeypatch.setattr(microscaling, "MX_FEW_TOKENS_ROWS", 0)
    tokens, experts, slots, hidden, ffn = MLPS[case]
    top_experts = torch.rand(tokens, experts, generator=torch.Generator(device).manual_seed(case), device=device).topk(slots).indices
    top_experts[7, 0] = -1  # entries that select no expert contribute nothing
    top_experts[tokens - 1, slots - 1] = experts
    if case == len(MLPS) - 1:
        top_experts.fill_(1)
    _check_mlp(tokens, experts, slots, hidden, ffn, gated, activation, top_experts, format, (torch.bfloat16, torch.float16, torch.float32), device)


@pytest.mark.parametrize("format", FORMATS)
@pytest.mark.parametrize(("tokens", "experts", "slots", "hidden", "ffn", "gated", "first", "second"), BY_ENTRIES)
def test_few_tokens(tokens, experts, slots, hidden, ffn, gated, first, second, format, device, monkeypatch):
    monkeypatch.setattr(microscaling, "MX_FEW_TOKENS_ROWS", 10**6)
    top_experts = torch.rand(tokens, experts, generator=torch.Generator(device).manual_seed(hidden), device=device).topk(slots).indices
    if tokens > 1:
        top_experts[1, 0] = -1
    _check_mlp(tokens, experts, slots, hidden, ffn, gated, "relu", top_experts, format, (torch.float32, torch.bfloat16), device)


@pytest.mark.parametrize("format", FORMATS)
@pytest.mark.parametrize(("tokens", "experts", "slots", "hidden", "ffn"), MLPS)
def test_mlp_on_tiles_is_its_operators_one_after_the_other(tokens, experts, slots, hidden, ffn, format, device, monkeypatch):
    monkeypatch.setattr(microscaling, "MX_FEW_TOKENS_ROWS", 0)
    generator = torch.Generator(device).manual_seed(tokens)
    rows, _ = scaled(generator, (tokens, hidden), format, 2.0**-5)
    weight_1, _ = scaled(generator, (2 * experts * ffn, hidden), "e2m1")
    weight_2, _ = scaled(generator, (experts * hidden, ffn), "e2m1")
    scores, top_experts = torch.rand(tokens, experts, generator=generator, device=device).topk(slots)
    top_experts[tokens // 2, 0] = -1
    sparse_map = get_sparse_map(top_experts, experts)
    between = mx_sparse_matmul_activation(mx_copy_dense_to_sparse(rows, sparse_map), weight_1, sparse_map, True, "silu")
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        expected = copy_sparse_to_dense(mx_sparse_matmul(between, weight_2, sparse_map, dtype=dtype), scores, sparse_map)
        assert torch.equal(mx_mlp(rows, scores, top_experts, weight_1, weight_2, experts, gated=True, activation_type="silu", dtype=dtype), expected)
