"""Operators on values of 8 bits with a scale per block of 128 at their edges: what is no number, terms that cancel, weights that are quantised where they are needed."""

import pytest
import torch

from fast_llm_amd.functional.block_scaling import (
    block_activation_backward, block_activation_forward, block_copy_dense_to_sparse, block_input_row_sparse_matmul, block_mlp, block_quantize,
    block_quantize_both, block_quantize_transposed, block_sparse_matmul,
)  # fmt: skip
from fast_llm_amd.functional.sparse_copy import copy_dense_to_sparse_backward, copy_sparse_to_dense, copy_sparse_to_dense_backward, get_sparse_map
from fast_llm_amd.layers.moe import BlockScaledMoEMLP, attach_grad_buffer
from oracle import block_oracle
from tests.test_gpu_block_scaling import ACTIVATIONS, DTYPES, MLP_TOLERANCE, _difference, _map, _mlp_inputs, _values

pytestmark = pytest.mark.gpu


# ---- infinities and NaN in rows that count ---------------------------------------------------------------
NAN, INF = float("nan"), float("inf")


def _bad_blocks(bad: torch.Tensor) -> torch.Tensor:
    """[rows, blocks of 128 columns]: those with a bad value."""
    return torch.nn.functional.pad(bad, (0, -bad.size(1) % 128)).unflatten(1, (-1, 128)).any(-1)


def _assert_bad(tensor, bad: torch.Tensor, plain) -> None:
    """Blocks with a bad value are NaN, with zeros for elements; the others are those of `plain`, which has none."""
    blocks = _bad_blocks(bad)
    scales, expected = tensor.scales[:, : tensor.rows].t().cpu(), plain.scales[:, : tensor.rows].t().cpu()
    assert torch.equal(scales == 255, blocks)
    assert torch.equal(scales[~blocks], expected[~blocks])
    elements, expected = (t.values.cpu().unflatten(1, (-1, 128)) for t in (tensor, plain))
    assert not elements[blocks].any() and torch.equal(elements[~blocks], expected[~blocks])


@pytest.mark.parametrize("gated", [True, False])
@pytest.mark.parametrize("activation", ACTIVATIONS)
@pytest.mark.parametrize("dtype", DTYPES)
def test_infinities_and_nan_in_rows_that_count(dtype, activation, gated, device):
    generator = torch.Generator().manual_seed(1)
    rows, ffn = 130, 256
    x = torch.randn(rows, ffn * (1 + gated), generator=generator).to(dtype)
    grad = torch.randn(rows, ffn, generator=generator).to(dtype)
    plain_output, plain_checkpoint = block_activation_forward(x.to(device), gated, activation)
    plain_grads = block_activation_backward(grad.to(device), plain_checkpoint, gated, activation)

    # Into the gates, row by row; row 7 has one in each block, the last row is in the second block of rows.
    places = {(3, 5): NAN, (7, 0): NAN, (7, 255): INF, (20, 130): INF, (129, 1): -INF}
    bad_input, bad_output = torch.zeros(rows, x.size(1), dtype=torch.bool), torch.zeros(rows, ffn, dtype=torch.bool)
    y = x.clone()
    for (row, column), value in places.items():
        y[row, column] = value
        bad_input[row, column] = True
        # An infinity is one of the result's; x times a sigmoid has no limit at the lower end in which 0 times it were a number, and ReLUs are 0 there.
        bad_output[row, column] = not (value == -INF and activation in ("relu", "squared_relu"))
    if gated:
        y[40, ffn + 200] = NAN  # an up: its gate is what it was
        bad_input[40, ffn + 200] = bad_output[40, 200] = True
    output, checkpoint = block_activation_forward(y.to(device), gated, activation)
    _assert_bad(checkpoint, bad_input, plain_checkpoint)
    # (In its row's block -inf becomes 0, which is not what the plain block has: that block is compared by its scale alone.)
    special = activation in ("relu", "squared_relu")
    if special:
        assert output.scales[0, 129] != 255 and output.values[129, 1] & 0x7F == 0
        output.scales[0, 129], output.values[129, :128] = plain_output.scales[0, 129], plain_output.values[129, :128]
    _assert_bad(output, bad_output, plain_output)

    # Backward: whatever shares a block with a bad value is NaN.
    kept = _bad_blocks(bad_input).repeat_interleave(128, 1)
    gate, up = kept[:, :ffn], kept[:, ffn:] if gated else torch.zeros(rows, ffn, dtype=torch.bool)
    bad_gate = up if activation == "identity" else gate | up  # (whose slope is 1, whatever it is of)
    bad_grad = torch.cat((bad_gate, gate), dim=1) if gated else bad_gate
    grads = block_activation_backward(grad.to(device), checkpoint, gated, activation)
    _assert_bad(grads[0], bad_grad, plain_grads[0])
    _assert_bad(grads[1], bad_grad.t(), plain_grads[1])
    _assert_bad(grads[2], (gate | up).t(), plain_grads[2])

    # Into the gradient, which leaves the activation alone.
    g = grad.clone()
    g[9, 3], g[70, 140] = NAN, -INF
    bad = ~torch.isfinite(g)
    grads = block_activation_backward(g.to(device), plain_checkpoint, gated, activation)
    # Zero times an infinity is not a number either.
    bad = torch.cat((bad, bad), dim=1) if gated else bad
    _assert_bad(grads[0], bad, plain_grads[0])
    _assert_bad(grads[1], bad.t(), plain_grads[1])
    _assert_bad(grads[2], torch.zeros(rows, ffn, dtype=torch.bool).t(), plain_grads[2])


# ---- sums ------------------------------------------------------------------------------------------------
def _cancelling(generator, rows: int, columns: int, inner: int) -> tuple[torch.Tensor, torch.Tensor]:
    """Operands whose products have, in each eight neighbours along the reduction, two large ones that cancel, beside small ones."""
    lhs, rhs = torch.randn(rows, inner, generator=generator), torch.randn(columns, inner, generator=generator)
    lhs[:, ::8], lhs[:, 1::8], rhs[:, ::8], rhs[:, 1::8] = 400.0, 400.0, 4.0, -4.0
    return lhs, rhs


def _eights(lhs: torch.Tensor, rhs: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Of each eight neighbours along the reduction, [eights, rows, columns]: the sum and the largest magnitude of their products."""
    a, b = (torch.nn.functional.pad(t, (0, -t.size(1) % 8)).unflatten(1, (-1, 8)).transpose(0, 1) for t in (lhs, rhs))
    products = a[:, :, None] * b[:, None]
    return products.sum(-1), products.abs().amax(-1)


def _rounding(expected: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    """Half a step of the result (of its smallest normal value, below that)."""
    return torch.finfo(dtype).eps / 2 * expected.abs().clamp_min(torch.finfo(dtype).smallest_normal)


def _exact_tolerance(lhs: torch.Tensor, rhs: torch.Tensor) -> torch.Tensor:
    """
    Exact sums: each product is exact. An instruction adds 16 of them, two whole eights, to the sum so far: 16 additions, in any order, of at most (the sum so far and
    the magnitudes of the 16), each off by a step of fp32 at most. The sum so far is made of whole eights: it is no larger than the magnitudes of their sums.
    """
    sums, _ = _eights(lhs, rhs)
    instructions = -(-lhs.size(1) // 16)
    return 16 * 2.0**-23 * (lhs.abs() @ rhs.abs().t() + instructions * sums.abs().sum(0))


@pytest.mark.parametrize("accumulate", [False, True])
@pytest.mark.parametrize("counts", [[30], [300, 0, 257]], ids=str)
@pytest.mark.parametrize(("rows", "columns"), [(40, 70), (300, 264)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_weight_gradients_keep_small_terms_beside_large_ones(dtype, rows, columns, counts, accumulate, device):
    """In fp32, and in fp16, of which every bit is one that inexact sums would show."""
    generator = torch.Generator().manual_seed(rows + columns)
    sparse_map = _map(counts, device)
    lhs, rhs = _cancelling(generator, rows, columns, sparse_map.num_rows)
    before = (torch.randn(len(counts) * rows, columns, generator=generator) * 10).to(dtype)
    begin = 0
    for count in counts:  # zeros where no token is
        lhs[:, begin + count : begin + -(-count // 128) * 128] = 0
        begin += -(-count // 128) * 128
    a, b = block_quantize(lhs.to(device)), block_quantize(rhs.to(device))
    x, y = _values(a), _values(b)
    out = before.to(device)
    block_input_row_sparse_matmul(a, b, sparse_map, out=out, accumulate=accumulate)
    begin = 0
    for expert, count in enumerate(counts):
        part = slice(begin, begin + -(-count // 128) * 128)
        begin = part.stop
        expected, tolerance = x[:, part] @ y[:, part].t(), _exact_tolerance(x[:, part], y[:, part])
        if accumulate:
            earlier = before[expert * rows : (expert + 1) * rows].double()
            expected += earlier
            tolerance += 2.0**-24 * (expected.abs() + tolerance)  # one more addition in fp32
        error = (out[expert * rows : (expert + 1) * rows].cpu().double() - expected).abs()
        assert (error <= tolerance + _rounding(expected.abs() + tolerance, dtype)).all()


def _default_tolerance(lhs: torch.Tensor, rhs: torch.Tensor) -> torch.Tensor:
    """
    Sums without `exact_sums`: of every eight products the instruction keeps what lies above 2^-13 of the largest one's power of two, so that each of the other seven loses less than
    2^-13 of the largest (whose own 8 bits are all above that). An instruction adds eight such sums to the sum so far, each addition off by
    2^-21 of (the sum so far and the magnitudes of the 64 products) at most: they are aligned to the largest of them with 23 bits.
    """
    sums, largest = _eights(lhs, rhs)
    instructions = -(-lhs.size(1) // 64)
    return 7 * 2.0**-13 * largest.sum(0) + 8 * 2.0**-21 * (lhs.abs() @ rhs.abs().t() + instructions * (sums.abs().sum(0) + 7 * 2.0**-13 * largest.sum(0)))


@pytest.mark.parametrize("exact", [False, True])
@pytest.mark.parametrize("cancelling", [False, True])
@pytest.mark.parametrize("counts", [[40, 3], [300, 257]], ids=str)  # few rows, and tiles
@pytest.mark.parametrize(("inner", "columns"), [(200, 70), (1024, 264)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_products_are_as_exact_as_they_say(dtype, inner, columns, counts, cancelling, exact, device):
    generator = torch.Generator().manual_seed(inner + columns)
    sparse_map = _map(counts, device)
    lhs, rhs = _cancelling(generator, sparse_map.num_rows, len(counts) * columns, inner)
    if not cancelling:
        lhs, rhs = (torch.randn(t.shape, generator=generator) for t in (lhs, rhs))
    a, b = block_quantize(lhs.to(device)), block_quantize(rhs.to(device))
    x, w = _values(a), _values(b)
    out = block_sparse_matmul(a, b, sparse_map, dtype=dtype, exact_sums=exact).cpu().double()
    # fp32 results are exact sums in any case.
    tolerance_of = _exact_tolerance if exact or dtype == torch.float32 else _default_tolerance
    begin = 0
    for expert, count in enumerate(counts):
        weight = w[expert * columns : (expert + 1) * columns]
        # (All columns, and of the rows as many as the products of all eights fit the memory for.)
        rows = torch.arange(begin, begin + count)[:: max(count // 20, 1)]
        expected, tolerance = x[rows] @ weight.t(), tolerance_of(x[rows], weight)
        assert ((out[rows] - expected).abs() <= tolerance + _rounding(expected.abs() + tolerance, dtype)).all()
        begin += -(-count // 128) * 128


@pytest.mark.parametrize("accumulate", [False, True])
def test_weight_gradients_in_bf16_are_as_exact_as_they_say(accumulate, device):
    generator = torch.Generator().manual_seed(7)
    counts, rows, columns = [300, 0, 257], 40, 264
    sparse_map = _map(counts, device)
    lhs, rhs = (torch.randn(size, sparse_map.num_rows, generator=generator) for size in (rows, columns))
    before = (torch.randn(len(counts) * rows, columns, generator=generator) * 10).bfloat16()
    begin = 0
    for count in counts:
        lhs[:, begin + count : begin + -(-count // 128) * 128] = 0
        begin += -(-count // 128) * 128
    a, b = block_quantize(lhs.to(device)), block_quantize(rhs.to(device))
    x, y = _values(a), _values(b)
    out = block_input_row_sparse_matmul(a, b, sparse_map, out=before.to(device), accumulate=accumulate).cpu().double()
    begin = 0
    for expert, count in enumerate(counts):
        part, of_expert = slice(begin, begin + -(-count // 128) * 128), slice(expert * rows, (expert + 1) * rows)
        begin = part.stop
        expected, tolerance = x[:, part] @ y[:, part].t(), _default_tolerance(x[:, part], y[:, part])
        if accumulate:
            expected += before[of_expert].double()
            tolerance += 2.0**-24 * (expected.abs() + tolerance)
        assert ((out[of_expert] - expected).abs() <= tolerance + _rounding(expected.abs() + tolerance, torch.bfloat16)).all()


def test_a_layer_in_fp16_has_exact_sums_throughout(device):
    """It is its operators one after the other, all of them with `exact_sums`; without, the last ones have other bits."""
    torch.manual_seed(0)
    layer = BlockScaledMoEMLP(512, 640, 8, 2, device=device, dtype=torch.float16)
    x, grad = (torch.randn(1500, 512, device=device).half() for _ in range(2))
    with torch.no_grad():
        scores, top_experts = layer.route(x)
    y = x.clone().requires_grad_(True)
    output = layer(y, scores=scores, top_experts=top_experts)
    output.backward(grad)
    with torch.no_grad():
        sparse_map, weights = get_sparse_map(top_experts, 8), layer.quantize_weights()

        def product(rows, weight, exact=True):
            return block_sparse_matmul(rows, weight, sparse_map, dtype=torch.float16, exact_sums=exact)

        rows = block_copy_dense_to_sparse(block_quantize(x), sparse_map)
        hidden, checkpoint = block_activation_forward(product(rows, weights.layer_1), True, layer.activation, sparse_map)
        layer_2 = product(hidden, weights.layer_2_transposed)
        assert torch.equal(output, copy_sparse_to_dense(layer_2, scores, sparse_map))
        assert not torch.equal(output, copy_sparse_to_dense(product(hidden, weights.layer_2_transposed, False), scores, sparse_map))
        grad_2, _ = copy_sparse_to_dense_backward(grad, (sparse_map, layer_2, scores))
        grad_rows, grad_columns = block_quantize_both(grad_2, sparse_map=sparse_map)
        grad_1, grad_1_columns, hidden_columns = block_activation_backward(product(grad_rows, weights.layer_2), checkpoint, True, layer.activation, sparse_map)
        assert torch.equal(y.grad, copy_dense_to_sparse_backward(product(grad_1, weights.layer_1_transposed), (sparse_map, x.shape)))
        assert not torch.equal(y.grad, copy_dense_to_sparse_backward(product(grad_1, weights.layer_1_transposed, False), (sparse_map, x.shape)))
        # An exact sum in fp32, rounded once, is that in fp16.
        rows_columns = block_quantize_transposed(rows, sparse_map=sparse_map)
        for weight, lhs, rhs in ((layer.layer_2, hidden_columns, grad_columns), (layer.layer_1, grad_1_columns, rows_columns)):
            assert weight.grad_buffer.dtype == torch.float16
            assert torch.equal(weight.grad_buffer, block_input_row_sparse_matmul(lhs, rhs, sparse_map, dtype=torch.float32).half())


@pytest.mark.parametrize("rows", [1, 300])  # few rows, and tiles
def test_the_range_of_operands(rows, device):
    """Everything that 8 bits and a scale stand for; with exact sums what bf16 does: no 2^128, and multiples of 2^-133."""
    top, small = torch.finfo(torch.bfloat16).max, 2.0**-133

    def product(value: float, factor: float, exact: bool) -> float:
        lhs, rhs = (block_quantize(torch.full((n, 128), v, device=device)) for n, v in ((rows, value), (1, factor)))
        out = block_sparse_matmul(lhs, rhs, dtype=torch.bfloat16, exact_sums=exact)
        assert torch.equal(out.isnan(), out[:1].isnan().expand_as(out)) and torch.equal(out.nan_to_num(), out[:1].expand_as(out).nan_to_num())
        return out[0, 0].item()

    # (128 products of powers of two, or of numbers of four bits: exact in bf16.)
    for exact in (False, True):
        for value in (240 * 2.0**120, -(2.0**127), 2.0**-126, 2.0**-127, small, -3 * small):
            factor = 2.0**-40 if abs(value) > 1 else 2.0**120
            assert product(value, factor, exact) == 128 * value * factor
    assert product(top, 2.0**-40, False) == 128 * 2.0**88 and product(-top, 0.0, False) == 0
    assert product(top, 2.0**-40, True) == INF and torch.tensor(product(-top, 0.0, True)).isnan()
    assert product(small / 4, 2.0**120, False) == 128 * 2.0**-15 and product(small / 4, 2.0**120, True) == 0


@pytest.mark.parametrize("per_expert", [1, 20, 100, 300])
@pytest.mark.parametrize("exact", [False, True])
def test_the_padding_of_the_layout_changes_nothing(exact, per_expert, device):
    """Room for any routing, for this one alone, or no padding: the same products run on the same kernel, to the bit."""
    generator = torch.Generator().manual_seed(per_expert)
    experts, inner, columns = 8, 512, 1280
    top_experts = torch.rand(per_expert * experts // 2, experts, generator=generator).topk(2).indices.to(device)
    rows = block_quantize(torch.randn(top_experts.size(0), inner, generator=generator).to(device))
    weight = block_quantize(torch.randn(experts * columns, inner, generator=generator).to(device))
    results = []
    for options in ({}, {"dynamic_shape": True}, {"dynamic_shape": True, "pad_to_multiple": 1}):
        sparse_map = get_sparse_map(top_experts, experts, **options)
        out = block_sparse_matmul(block_copy_dense_to_sparse(rows, sparse_map), weight, sparse_map, exact_sums=exact)
        results.append(out[sparse_map.sparse_rows.long()])
    assert all(torch.equal(result, results[0]) for result in results)


# ---- weights that are quantised where they are needed ----------------------------------------------------
def _layer_step(layer, x, grad, **options):
    x = x.detach().requires_grad_(True)
    layer.zero_grad()
    layer.layer_1.param_grad_is_zero = layer.layer_2.param_grad_is_zero = True
    output = layer(x, **options)
    output.backward(grad)
    return [t.detach().clone() for t in (output, x.grad, layer.router.grad, layer.layer_1.grad_buffer, layer.layer_2.grad_buffer)]


@pytest.mark.parametrize("gated", [True, False])
def test_weights_quantised_in_the_step_are_those_quantised_before_it(gated, device):
    torch.manual_seed(0)
    layer = BlockScaledMoEMLP(512, 640, 8, 2, gated=gated, device=device)
    x, grad = (torch.randn(300, 512, device=device).bfloat16() for _ in range(2))
    expected = _layer_step(layer, x, grad, weights=layer.quantize_weights())
    assert all(torch.equal(a, b) for a, b in zip(_layer_step(layer, x, grad), expected))
    # Twice through the same graph.
    layer.layer_1.param_grad_is_zero = layer.layer_2.param_grad_is_zero = True
    y = x.clone().requires_grad_(True)
    output = layer(y)
    (first,) = torch.autograd.grad(output, y, grad, retain_graph=True)
    (second,) = torch.autograd.grad(output, y, grad)
    assert torch.equal(first, expected[1]) and torch.equal(second, first)
    # Inference needs half of the forms, and has the same result with either half or all of them.
    layer.eval()
    for weights in (None, layer.quantize_weights(), layer.quantize_weights(training=False)):
        assert torch.equal(layer(x, weights=weights), expected[0])
    inference = layer.quantize_weights(training=False)
    assert inference.layer_1_transposed is None and inference.layer_2 is None
    layer.train()
    with pytest.raises(ValueError, match="for inference"):
        layer(x, weights=inference)


def test_what_is_kept_between_forward_and_backward(device):
    """8 bits of each slot's input and of the first layer's output, each slot's output: no form of the weights, which would be the most of it."""
    torch.manual_seed(0)
    hidden, ffn, experts, tokens = 512, 640, 8, 64
    layer = BlockScaledMoEMLP(hidden, ffn, experts, 2, device=device)
    x = torch.randn(tokens, hidden, device=device).bfloat16().requires_grad_(True)
    rows = 2 * tokens + 128 * experts
    most = rows * ((hidden + 2 * ffn) * (1 + 1 / 128) + 2 * hidden) + (1 << 18)  # and what belongs to the routing
    forms = experts * hidden * 3 * ffn
    assert most < forms / 1.5
    layer(x).backward(torch.zeros_like(x))

    def held() -> int:
        """Bytes as they were asked for. (What is allocated may be up to 1 MiB more for each tensor, where the allocator has a larger block to hand.)"""
        return torch.cuda.memory_stats()["requested_bytes.all.current"]

    for weights in (None, layer.quantize_weights()):
        before = held()
        output = layer(x, weights=weights)
        assert held() - before <= most
        output.backward(torch.zeros_like(x))
        del output
    layer.eval()
    before = held()
    weights = layer.quantize_weights(training=False)
    assert held() - before <= forms * (1 + 1 / 64)


def test_weights_that_change_before_the_backward_are_noticed(device):
    torch.manual_seed(0)
    layer = BlockScaledMoEMLP(256, 256, 4, 2, device=device)
    x, grad = (torch.randn(50, 256, device=device).bfloat16() for _ in range(2))
    for name in ("layer_1", "layer_2"):
        output = layer(x)
        with torch.no_grad():
            getattr(layer, name).mul_(2)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            output.backward(grad)
    # Those that the caller has quantised are what the backward goes by.
    weights = layer.quantize_weights()
    expected = _layer_step(layer, x, grad, weights=weights)
    y = x.clone().requires_grad_(True)
    output = layer(y, weights=weights)
    with torch.no_grad():
        layer.layer_1.mul_(2)
    (ours,) = torch.autograd.grad(output, y, grad)
    assert torch.equal(ours, expected[1])


# ---- routings and sizes that the layer allows and seldom meets -------------------------------------------
@pytest.mark.parametrize("dynamic", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize(("hidden", "ffn", "gated"), [(129, 100, False), (8, 1, False), (320, 128, True)])
def test_mlp_step_of_tokens_without_experts_and_with_one_twice(hidden, ffn, gated, dtype, dynamic, device):
    tokens, experts, slots = 90, 5, 3
    input_, scores, top_experts, weight_1, weight_2, grad = _mlp_inputs(tokens, hidden, ffn, experts, slots, gated, dtype, device, seed=hidden)
    top_experts[::7] = -1  # the padding of a batch
    top_experts[1::7, 1] = -1
    top_experts[2::7] = top_experts[2::7, :1]  # the same expert in all slots
    expected = block_oracle.mlp_step(input_, scores, top_experts, weight_1, weight_2, experts, gated, "silu", grad, dtype)
    x, s = input_.to(device).requires_grad_(True), scores.to(device).requires_grad_(True)
    weights = [attach_grad_buffer(w.to(device).requires_grad_(True)) for w in (weight_1, weight_2)]
    sparse_map = get_sparse_map(top_experts.to(device), experts, dynamic_shape=dynamic)
    output = block_mlp(x, s, *weights, gated=gated, activation_type="silu", sparse_map=sparse_map)
    output.backward(grad.to(device))
    ours = {"output": output, "grad_input": x.grad, "grad_scores": s.grad, "grad_weight_1": weights[0].grad_buffer, "grad_weight_2": weights[1].grad_buffer}
    for name, theirs in expected.items():
        assert _difference(ours[name], theirs) <= MLP_TOLERANCE, name
    assert not output[::7].any() and not x.grad[::7].any() and not s.grad[::7].any()


@pytest.mark.parametrize("dynamic", [False, True])
@pytest.mark.parametrize("without", [slice(None), slice(None, None, 5)], ids=["all", "some"])
def test_tokens_without_experts_may_hold_anything(without, dynamic, device):
    input_, scores, top_experts, weight_1, weight_2, grad = (t.to(device) for t in _mlp_inputs(60, 256, 128, 4, 2, True, torch.bfloat16, device))
    top_experts[without] = -1
    weights = [attach_grad_buffer(w.requires_grad_(True)) for w in (weight_1, weight_2)]
    sparse_map = get_sparse_map(top_experts, 4, dynamic_shape=dynamic)
    results = []
    for value in (0.0, NAN):
        x, s, g = input_.clone(), scores.clone(), grad.clone()
        x[without], s[without], g[without] = value, value, value
        x.requires_grad_(True), s.requires_grad_(True)
        for weight in weights:
            weight.param_grad_is_zero = True
        output = block_mlp(x, s, *weights, gated=True, activation_type="silu", sparse_map=sparse_map)
        output.backward(g)
        results.append([t.detach().clone() for t in (output, x.grad, s.grad, *(w.grad_buffer for w in weights))])
    assert all(torch.equal(a, b) for a, b in zip(*results))
    assert not any(t[without].any() for t in results[1][:3])
    if without == slice(None):
        assert not any(t.any() for t in results[1])
