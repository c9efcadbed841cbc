"""
What is measured: serving the mixture-of-experts layer from microscaled (MX) expert weights, and the normalisation in front.

Four operators that a pass through a quantised layer calls one after the other: the root-mean-square norm with the residual's
addition (in serving with its result also in 8 bits, in training with its backward), the quantisation to blocks of 32 with a
shared power of two, the grouped product of 8- or 4-bit rows with 4-bit expert weights, and the whole expert MLP on them. Sizes
are the benchmark's (`fast_llm_amd.workloads.WORKLOADS`) and generic ones.

Definition of the MX formats used here (OCP Microscaling Formats 1.0): a block of 32 neighbours along a row shares the scale
2^e, e = floor(log2(largest magnitude)) - (8 for e4m3, 2 for e2m1), at least -127, stored as the byte e + 127; elements are
value / 2^e, rounded to nearest even and saturated at 448 or 6. Rows are stored padded with zeros to whole groups of 128 columns.
"""

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
# hidden, ffn, experts, experts per token
_MIXTRAL, _FINE_GRAINED, _WIDE, _RAGGED = (4096, 14336, 8, 2), (2048, 1408, 64, 6), (2048, 768, 128, 8), (1280, 3416, 16, 2)
_EPS = 1e-5
_PADDING = 128  # rows of a sparse map's blocks, and columns of the storage


# ---- the cases -------------------------------------------------------------------------------------------
def _norm(kind: str, tokens: int, hidden: int, dtype: str, residual: bool = True) -> dict:
    return {"kind": kind, "tokens": tokens, "hidden": hidden, "dtype": dtype, "residual": residual}


def _quantize(rows: int, columns: int, dtype: str, format: str) -> dict:
    return {"kind": "quantize", "rows": rows, "columns": columns, "dtype": dtype, "format": format}


def _product(tokens: int, inner: int, columns: int, experts: int, slots: int, dtype: str = "bf16", format: str = "e4m3", zipf: float = 0.0) -> dict:
    return {
        "kind": "product", "tokens": tokens, "inner": inner, "columns": columns, "experts": experts, "slots": slots,
        "dtype": dtype, "format": format, "zipf": zipf,
    }  # fmt: skip


def _mlp(tokens: int, shape: tuple, dtype: str = "bf16", format: str = "e4m3", gated: bool = True, activation: str = "silu", zipf: float = 0.0) -> dict:
    return {
        "kind": "mlp", "tokens": tokens, "hidden": shape[0], "ffn": shape[1], "experts": shape[2], "slots": shape[3],
        "dtype": dtype, "format": format, "gated": gated, "activation": activation, "zipf": zipf,
    }  # fmt: skip


def listed() -> list[dict]:
    cases = {
        # In front of the layer for one generated token: latency.
        "norm_token": _norm("norm_quantize", 1, 4096, "bf16"),
        # In front of the layer for several prompts at once.
        "norm_prompt": _norm("norm_quantize", 5001, 2048, "fp16"),
        # A training step's forward and backward in front of the wide and the fine-grained layer.
        "norm_step": _norm("norm_step", 16384, 2048, "bf16"),
        # The smallest benchmark configuration: tests and debugging runs in single precision, the first layer of a block.
        "norm_step_tiny": _norm("norm_step", 512, 256, "fp32", residual=False),
        # Activations of a feed-forward size of no whole block, in 8 bits.
        "quantize_rows": _quantize(12001, 3416, "bf16", "e4m3"),
        # The second layer of eight experts to 4 bits, and back as a check of a checkpoint's quality does it.
        "quantize_experts": _quantize(8 * 4096, 14336, "bf16", "e2m1"),
        # The first layer's product for one generated token: two experts' weights are read.
        "product_token": _product(1, 4096, 2 * 14336, 8, 2),
        # The first layer's product for several prompts, many small experts.
        "product_prompt": _product(5001, 2048, 2 * 1408, 64, 6, "fp16"),
        # The second layer's product of a long prompt, the rows in 4 bits as well.
        "product_four_bit": _product(8192, 14336, 4096, 8, 2, "bf16", "e2m1"),
        # Text generation for one user.
        "mlp_token": _mlp(1, _MIXTRAL),
        # Batched generation with many small experts.
        "mlp_batch": _mlp(96, _WIDE),
        # The benchmark's headline shape as a prompt.
        "mlp_prompt": _mlp(8192, _MIXTRAL),
    }
    return [{"name": name, **case} for name, case in cases.items()]


def _log_uniform(rng, low: int, high: int, multiple: int = 1) -> int:
    value = low * (high / low) ** rng.random()
    return max(low, min(high, round(value / multiple) * multiple))


# No case does more than the listed ones of its kind.
_MOST_NORM, _MOST_QUANTIZE, _MOST_FLOPS, _MOST_WEIGHTS = 16384 * 4096, 8 * 4096 * 14336, 6 * 8192 * 2 * 4096 * 14336, 8 * 3 * 4096 * 14336


def draw(rng) -> dict:
    while True:
        kind = rng.choice(("norm_quantize", "norm_step", "quantize", "product", "product", "mlp", "mlp", "mlp"))
        multiple = rng.choice((1, 8, 32, 128))
        if kind in ("norm_quantize", "norm_step"):
            # A prime number of columns is nobody's hidden size; multiples of 8 and of 2 are.
            hidden = _log_uniform(rng, 64, 8192, max(multiple, 2))
            tokens = _log_uniform(rng, 1, 16384)
            if tokens * hidden <= _MOST_NORM:
                return _norm(kind, tokens, hidden, rng.choice(("bf16", "bf16", "fp16", "fp32")), rng.random() < 0.8)
        elif kind == "quantize":
            rows, columns = _log_uniform(rng, 1, 32768), _log_uniform(rng, 32, 14336, multiple)
            if rows * columns <= _MOST_QUANTIZE:
                return _quantize(rows, columns, rng.choice(("bf16", "bf16", "fp16", "fp32")), rng.choice(("e4m3", "e2m1")))
        else:
            shape = rng.choice((_MIXTRAL, _FINE_GRAINED, _WIDE, _RAGGED, None, None))
            if shape is None:
                experts = rng.choice((8, 16, 32, 60, 64, 128))
                shape = (_log_uniform(rng, 512, 4096, max(multiple, 8)), _log_uniform(rng, 512, 8192, max(multiple, 8)), experts, rng.choice((1, 2, 4, 6, 8)))
            hidden, ffn, experts, slots = shape
            tokens = _log_uniform(rng, 1, 256) if rng.random() < 0.5 else _log_uniform(rng, 256, 16384)
            zipf = rng.choice((0.0, 0.6, 1.2)) if experts <= 16 else 0.0
            dtype, format = rng.choice(("bf16", "bf16", "fp16")), rng.choice(("e4m3", "e4m3", "e2m1"))
            if kind == "product":
                inner, columns = (hidden, 2 * ffn) if rng.random() < 0.5 else (ffn, hidden)
                case = _product(tokens, inner, columns, experts, slots, dtype, format, zipf)
                weights = experts * inner * columns
            else:
                activation = rng.choice(("silu", "silu", "gelu", "squared_relu"))
                case = _mlp(tokens, shape, dtype, format, rng.random() < 0.85, activation, zipf)
                weights = experts * hidden * ffn * (3 if case["gated"] else 2)
            # The plain form pads experts to the fullest one.
            fullest = tokens if zipf else min(tokens, 2 * tokens * slots // experts + 64)
            if work(case)["flops"] <= _MOST_FLOPS and weights <= _MOST_WEIGHTS and fullest * experts * max(hidden, 2 * ffn) <= 1 << 31:
                return case


# ---- inputs ----------------------------------------------------------------------------------------------
def _normal(generator: torch.Generator, shape: tuple, dtype: torch.dtype, std: float = 1.0) -> torch.Tensor:
    return (torch.randn(shape, generator=generator, device="cuda") * std).to(dtype)


def _hidden_states(generator: torch.Generator, rows: int, columns: int, dtype: torch.dtype) -> torch.Tensor:
    """Features of unlike size, as the residual stream has them."""
    sizes = torch.exp(0.5 * torch.randn(columns, generator=generator, device="cuda"))
    return (torch.randn(rows, columns, generator=generator, device="cuda") * sizes).to(dtype)


def _padded(columns: int) -> int:
    return -(-columns // _PADDING) * _PADDING


def _mx_weights(generator: torch.Generator, experts: int, rows: int, columns: int) -> dict:
    """Normal weights in e2m1, packed two to a byte, the even column in the low half."""
    values = torch.empty(experts * rows, _padded(columns) // 2, dtype=torch.uint8, device="cuda")
    scales = torch.empty(experts * rows, _padded(columns) // 32, dtype=torch.uint8, device="cuda")
    for expert in range(experts):
        part = slice(expert * rows, (expert + 1) * rows)
        weight = _normal(generator, (rows, columns), torch.float32, 0.02)
        values[part], scales[part] = _stored(*_mx_parts(weight, "e2m1"), "e2m1")
    return {"values": values, "scales": scales, "columns": columns, "format": "e2m1"}


def _stored(elements: torch.Tensor, exponents: torch.Tensor, format: str) -> tuple[torch.Tensor, torch.Tensor]:
    """Elements and exponents of `_mx_parts` as the bytes in which they are kept."""
    rows, blocks = exponents.shape
    scales = torch.zeros(rows, _padded(blocks * 32) // 32, dtype=torch.uint8, device="cuda")
    scales[:, :blocks] = (exponents + 127).to(torch.uint8)
    if format == "e4m3":
        values = torch.zeros(rows, _padded(blocks * 32), dtype=torch.uint8, device="cuda")
        values[:, : blocks * 32] = elements.flatten(1).to(torch.float8_e4m3fn).view(torch.uint8)
        return values, scales
    doubled = (elements.flatten(1).abs() * 2).to(torch.int32)  # 0, 1, 2, 3, 4, 6, 8, 12
    codes = torch.where(doubled <= 4, doubled, torch.where(doubled == 6, 5, torch.where(doubled == 8, 6, 7)))
    codes = (codes + 8 * torch.signbit(elements.flatten(1))).to(torch.uint8)
    values = torch.zeros(rows, _padded(blocks * 32) // 2, dtype=torch.uint8, device="cuda")
    values[:, : blocks * 16] = codes[:, ::2] | codes[:, 1::2] << 4
    return values, scales


def _routing(generator: torch.Generator, tokens: int, experts: int, slots: int, zipf: float) -> tuple[torch.Tensor, torch.Tensor]:
    logits = torch.randn(tokens, experts, generator=generator, device="cuda")
    if zipf:
        logits -= zipf * torch.arange(1, experts + 1, device="cuda").log()
    top_logits, top_experts = torch.topk(logits, slots, dim=-1)
    return torch.softmax(top_logits, dim=-1), top_experts


def prepare(case: dict, seed: int) -> dict:
    generator = torch.Generator("cuda").manual_seed(seed)
    dtype = _DTYPES[case["dtype"]]
    state = dict(case)
    if case["kind"] in ("norm_quantize", "norm_step"):
        rows, columns = case["tokens"], case["hidden"]
        state["input"] = _hidden_states(generator, rows, columns, dtype)
        state["stream"] = _hidden_states(generator, rows, columns, dtype) if case["residual"] else None
        state["weight"] = (1 + _normal(generator, (columns,), torch.float32, 0.1)).to(dtype)
        if case["kind"] == "norm_step":
            state["gradients"] = [_normal(generator, (rows, columns), dtype) for _ in range(1 + case["residual"])]
            for name in ("input", "weight", "stream"):
                if state[name] is not None:
                    state[name].requires_grad_(True)
    elif case["kind"] == "quantize":
        state["input"] = _hidden_states(generator, case["rows"], case["columns"], dtype)
    elif case["kind"] == "product":
        experts = case["experts"]
        state["weight"] = _mx_weights(generator, experts, case["columns"], case["inner"])
        _, top_experts = _routing(generator, case["tokens"], experts, case["slots"], case["zipf"])
        counts = torch.bincount(top_experts.flatten(), minlength=experts)
        entries = case["tokens"] * case["slots"]
        rows = (entries + experts * _PADDING) // _PADDING * _PADDING
        blocks = (counts + _PADDING - 1) // _PADDING * _PADDING
        index_dtype = torch.int16 if rows < 32768 else torch.int32
        ends = blocks.cumsum(0)
        state["expert_ends"], state["expert_pad_begins"] = ends.to(index_dtype), (ends - blocks + counts).to(index_dtype)
        state["sparse_rows"], state["fullest"] = rows, int(counts.max())
        sparse = _hidden_states(generator, rows, case["inner"], torch.float32)
        values, scales = _stored(*_mx_parts(sparse, case["format"]), case["format"])
        state["rows"] = {"values": values, "scales": scales, "columns": case["inner"], "format": case["format"]}
        # Padding rows are left as they are.
        state["out"] = torch.zeros(rows, case["columns"], dtype=dtype, device="cuda")
    else:
        hidden, ffn, experts = case["hidden"], case["ffn"], case["experts"]
        state["weight_1"] = _mx_weights(generator, experts, ffn * (2 if case["gated"] else 1), hidden)
        state["weight_2"] = _mx_weights(generator, experts, hidden, ffn)
        state["scores"], state["top_experts"] = _routing(generator, case["tokens"], experts, case["slots"], case["zipf"])
        state["fullest"] = int(torch.bincount(state["top_experts"].flatten(), minlength=experts).max())
        values, scales = _stored(*_mx_parts(_hidden_states(generator, case["tokens"], hidden, torch.float32), case["format"]), case["format"])
        state["rows"] = {"values": values, "scales": scales, "columns": hidden, "format": case["format"]}
    return state


# ---- plain forms -----------------------------------------------------------------------------------------
_MIDDLES = (0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0)
_E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _mx_parts(values: torch.Tensor, format: str) -> tuple[torch.Tensor, torch.Tensor]:
    """Elements [rows, blocks, 32] (as floats) and exponents [rows, blocks] of fp32 rows."""
    rows, columns = values.shape
    blocks = torch.nn.functional.pad(values, (0, -columns % 32)).view(rows, -1, 32)
    largest = blocks.abs().amax(-1)
    # frexp: largest = m 2^e with m in [1/2, 1)
    exponents = torch.where(largest > 0, torch.frexp(largest)[1] - 1 - (8 if format == "e4m3" else 2), -127).clamp_min(-127)
    scaled = torch.ldexp(blocks, -exponents[..., None])
    if format == "e4m3":
        return scaled.clamp(-448, 448).to(torch.float8_e4m3fn).float(), exponents
    size = scaled.abs()
    # The number of borders below; one met exactly goes to the even code.
    code = (size > _MIDDLES[0]).to(torch.uint8)
    code += size >= _MIDDLES[1]
    code += size > _MIDDLES[2]
    code += size >= _MIDDLES[3]
    code += size > _MIDDLES[4]
    code += size >= _MIDDLES[5]
    code += size > _MIDDLES[6]
    table = torch.tensor(_E2M1, device=values.device)
    return torch.copysign(table[code.int()], scaled), exponents


def _mx_values(stored: dict) -> torch.Tensor:
    """The fp32 values that stored rows stand for, padding included."""
    scales = torch.ldexp(torch.ones((), device="cuda"), stored["scales"].int() - 127)
    if stored["format"] == "e4m3":
        elements = stored["values"].view(torch.float8_e4m3fn).float()
    else:
        table = torch.tensor(_E2M1 + tuple(-value for value in _E2M1), device="cuda")
        elements = table[torch.stack((stored["values"] & 15, stored["values"] >> 4), dim=-1).flatten(1).int()]
    return elements * scales.repeat_interleave(32, dim=1)


def _activate(values: torch.Tensor, gated: bool, activation: str) -> torch.Tensor:
    gate, up = values.chunk(2, dim=-1) if gated else (values, None)
    if activation == "silu":
        gate = gate / (1 + torch.exp(-gate))
    elif activation == "gelu":
        gate = 0.5 * gate * (1 + torch.tanh(0.7978845608028654 * (gate + 0.044715 * gate * gate * gate)))
    else:
        gate = gate.clamp_min(0) * gate.clamp_min(0)
    return gate * up if gated else gate


def _plain_norm(state: dict):
    dtype, columns = state["input"].dtype, state["hidden"]
    input_, weight = state["input"].detach().float(), state["weight"].detach().float()
    # The stream that goes on is what is normalised: rounded to its type.
    stream = input_ if state["stream"] is None else (input_ + state["stream"].detach().float()).to(dtype).float()
    inverse = 1 / torch.sqrt((stream * stream).mean(-1, keepdim=True) + _EPS)
    normalized = (stream * inverse * weight).to(dtype)
    outputs = {"normalized": normalized}
    if state["stream"] is not None:
        outputs["stream"] = stream.to(dtype)
    if state["kind"] == "norm_quantize":
        elements, exponents = _mx_parts(normalized.float(), "e4m3")
        outputs["elements"] = elements.flatten(1)[:, :columns].to(torch.float8_e4m3fn)
        outputs["scales"] = (exponents + 127).to(torch.uint8).view(torch.float8_e8m0fnu)
        return outputs
    grad = state["gradients"][0].float()
    scaled = grad * weight
    grad_input = inverse * (scaled - stream * inverse * inverse * (scaled * stream).mean(-1, keepdim=True))
    if state["stream"] is not None:
        grad_input = grad_input + state["gradients"][1].float()
    outputs["grad_input"] = grad_input.to(dtype)
    outputs["grad_weight"] = (grad * stream * inverse).sum(0).to(dtype)
    return outputs


def _plain_quantize(state: dict):
    elements, exponents = _mx_parts(state["input"].float(), state["format"])
    if state["format"] == "e4m3":
        elements = elements.flatten(1)[:, : state["columns"]].to(torch.float8_e4m3fn)
        return {"elements": elements, "scales": (exponents + 127).to(torch.uint8).view(torch.float8_e8m0fnu)}
    return {"values": torch.ldexp(elements, exponents[..., None]).flatten(1)[:, : state["columns"]].to(state["input"].dtype)}


def _by_expert(rows: torch.Tensor, places: torch.Tensor, experts: int, fullest: int) -> torch.Tensor:
    padded = torch.zeros(experts * fullest, rows.size(1), device="cuda")
    padded[places] = rows
    return padded.view(experts, fullest, -1)


def _plain_product(state: dict):
    experts, fullest = state["experts"], state["fullest"]
    ends, pad_begins = state["expert_ends"].long(), state["expert_pad_begins"].long()
    row = torch.arange(state["sparse_rows"], device="cuda")
    expert = torch.searchsorted(ends, row, right=True).clamp_max(experts - 1)
    begins = torch.cat((ends.new_zeros(1), ends[:-1]))
    real = (row < pad_begins[expert]).nonzero()[:, 0]
    places = (expert * fullest + row - begins[expert])[real]
    weight = _mx_values(state["weight"]).view(experts, state["columns"], -1)
    sums = torch.bmm(_by_expert(_mx_values(state["rows"])[real], places, experts, fullest), weight.transpose(1, 2))
    out = torch.zeros_like(state["out"])
    out[real] = sums.view(experts * fullest, -1)[places].to(out.dtype)
    return out


def _plain_mlp(state: dict):
    experts, fullest, dtype = state["experts"], state["fullest"], _DTYPES[state["dtype"]]
    hidden, ffn, slots = state["hidden"], state["ffn"], state["slots"]
    flat = state["top_experts"].flatten()
    chosen = torch.nn.functional.one_hot(flat, experts)
    places = flat * fullest + (chosen.cumsum(0) - chosen).gather(1, flat[:, None])[:, 0]
    rows = _mx_values(state["rows"])[torch.arange(state["tokens"], device="cuda").repeat_interleave(slots)]
    weight_1 = _mx_values(state["weight_1"]).view(experts, -1, _padded(hidden))
    layer_1 = torch.bmm(_by_expert(rows, places, experts, fullest), weight_1.transpose(1, 2)).view(experts * fullest, -1)[places]
    del weight_1
    # Between the layers the rows are in the input's format.
    elements, exponents = _mx_parts(_activate(layer_1, state["gated"], state["activation"]), state["format"])
    activation = torch.ldexp(elements, exponents[..., None]).flatten(1)[:, :ffn]
    weight_2 = _mx_values(state["weight_2"]).view(experts, hidden, -1)[..., :ffn]
    layer_2 = torch.bmm(_by_expert(activation, places, experts, fullest), weight_2.transpose(1, 2)).view(experts * fullest, -1)[places]
    return (layer_2.view(-1, slots, hidden) * state["scores"][..., None]).sum(1).to(dtype)


# ---- one pass --------------------------------------------------------------------------------------------
def run(state: dict):
    if own:
        return _run_own(state)
    if state["kind"] in ("norm_quantize", "norm_step"):
        return _plain_norm(state)
    if state["kind"] == "quantize":
        return _plain_quantize(state)
    return _plain_product(state) if state["kind"] == "product" else _plain_mlp(state)


def _run_own(state: dict):
    if state["kind"] == "norm_quantize":
        from fast_llm_amd.functional.normalization import rms_norm_quantize

        normalized, stream, quantized = rms_norm_quantize(state["input"], state["weight"], state["stream"], eps=_EPS)
        outputs = {"normalized": normalized, "elements": quantized.elements, "scales": quantized.block_scales}
        if state["stream"] is not None:
            outputs["stream"] = stream
        return outputs
    if state["kind"] == "norm_step":
        from fast_llm_amd.functional.normalization import rms_norm

        leaves = [state[name] for name in ("input", "weight", "stream") if state[name] is not None]
        results = rms_norm(state["input"], state["weight"], state["stream"], eps=_EPS)
        results = results if state["stream"] is not None else (results,)
        grads = torch.autograd.grad(results, leaves, state["gradients"])
        outputs = {"normalized": results[0].detach(), "grad_input": grads[0], "grad_weight": grads[1]}
        if state["stream"] is not None:
            outputs["stream"] = results[1].detach()
        return outputs
    from fast_llm_amd.functional import microscaling

    if state["kind"] == "quantize":
        quantized = microscaling.mx_quantize(state["input"], state["format"])
        if state["format"] == "e4m3":
            return {"elements": quantized.elements, "scales": quantized.block_scales}
        return {"values": microscaling.mx_dequantize(quantized, state["input"].dtype)}
    if state["kind"] == "product":
        from fast_llm_amd.functional.sparse_copy import SparseMap

        sparse_map = SparseMap(
            None, state["expert_ends"], state["expert_pad_begins"], state["tokens"], state["sparse_rows"],
            state["tokens"] * state["slots"], state["experts"], state["slots"],
        )  # fmt: skip
        rows, weight = (microscaling.MicroscaledTensor(**state[name]) for name in ("rows", "weight"))
        return microscaling.mx_sparse_matmul(rows, weight, sparse_map, out=state["out"])
    rows, weight_1, weight_2 = (microscaling.MicroscaledTensor(**state[name]) for name in ("rows", "weight_1", "weight_2"))
    return microscaling.mx_mlp(
        rows, state["scores"], state["top_experts"], weight_1, weight_2, state["experts"],
        gated=state["gated"], activation_type=state["activation"], dtype=_DTYPES[state["dtype"]],
    )  # fmt: skip


# ---- the definitions in 64 bits --------------------------------------------------------------------------
def _exact_quantized(values: torch.Tensor, format: str) -> tuple[torch.Tensor, torch.Tensor]:
    """Elements and scales, [rows, columns] and [rows, blocks], by the definition: the grid's spacing at a value's size is
    2^(its exponent - mantissa bits), and no finer than at the smallest normal value."""
    mantissa, lowest, highest, top = (3, -6, 8, 448.0) if format == "e4m3" else (1, 0, 2, 6.0)
    values = values.double()
    rows, columns = values.shape
    largest = torch.nn.functional.pad(values.abs(), (0, -columns % 32)).unflatten(1, (-1, 32)).amax(-1)
    scales = torch.exp2((torch.floor(torch.log2(largest)) - highest).clamp(-127, 127))
    scaled = values / scales.repeat_interleave(32, dim=1)[:, :columns]
    spacing = torch.exp2(torch.floor(torch.log2(scaled.abs().clamp_min(2.0**-200))).clamp_min(lowest) - mantissa)
    return (torch.round(scaled / spacing) * spacing).clamp(-top, top), scales


def _exact_values(stored: dict, rows: slice | torch.Tensor) -> torch.Tensor:
    bytes_, scales = stored["values"][rows], stored["scales"][rows].double()
    if stored["format"] == "e2m1":
        bytes_ = torch.stack((bytes_ & 15, bytes_ >> 4), dim=-1).flatten(1)
        sign, exponent, fraction = bytes_ >> 3, (bytes_ >> 1 & 3).double(), (bytes_ & 1).double() / 2
        size = torch.where(exponent > 0, (1 + fraction) * torch.exp2(exponent - 1), fraction)
    else:
        sign, exponent, fraction = bytes_ >> 7, (bytes_ >> 3 & 15).double(), (bytes_ & 7).double() / 8
        size = torch.where(exponent > 0, (1 + fraction) * torch.exp2(exponent - 7), fraction * 2.0**-6)
    values = (1 - 2 * sign.double()) * size * torch.exp2(scales - 127).repeat_interleave(32, dim=1)
    return values[:, : stored["columns"]]


def _exact_norm(state: dict) -> dict:
    dtype = state["input"].dtype
    stream = state["input"].detach().double()
    if state["stream"] is not None:
        stream = (stream + state["stream"].detach().double()).to(dtype).double()
    weight = state["weight"].detach().double()
    if state["kind"] == "norm_step":
        stream, weight = stream.requires_grad_(True), weight.requires_grad_(True)
    normalized = stream / torch.sqrt(stream.pow(2).mean(dim=1, keepdim=True) + _EPS) * weight
    outputs = {"normalized": normalized.detach()}
    if state["stream"] is not None:
        outputs["stream"] = stream.detach()
    if state["kind"] == "norm_quantize":
        outputs["elements"], outputs["scales"] = _exact_quantized(normalized.to(dtype), "e4m3")
        return outputs
    grads = torch.autograd.grad(normalized, (stream, weight), state["gradients"][0].double())
    outputs["grad_input"] = grads[0] if state["stream"] is None else grads[0] + state["gradients"][1].double()
    outputs["grad_weight"] = grads[1]
    return outputs


def exact(case: dict, seed: int):
    state = prepare(case, seed)
    if case["kind"] in ("norm_quantize", "norm_step"):
        return _exact_norm(state)
    if case["kind"] == "quantize":
        elements, scales = _exact_quantized(state["input"], case["format"])
        if case["format"] == "e4m3":
            return {"elements": elements, "scales": scales}
        return {"values": elements * scales.repeat_interleave(32, dim=1)[:, : case["columns"]]}
    if case["kind"] == "product":
        out = torch.zeros(state["sparse_rows"], case["columns"], dtype=torch.float64, device="cuda")
        begin = 0
        for expert in range(case["experts"]):
            end = int(state["expert_pad_begins"][expert])
            weight = _exact_values(state["weight"], slice(expert * case["columns"], (expert + 1) * case["columns"]))
            out[begin:end] = _exact_values(state["rows"], slice(begin, end)) @ weight.t()
            begin = int(state["expert_ends"][expert])
        return out
    hidden, ffn = case["hidden"], case["ffn"]
    layer_1_rows = ffn * (2 if case["gated"] else 1)
    out = torch.zeros(case["tokens"], hidden, dtype=torch.float64, device="cuda")
    for expert in range(case["experts"]):
        token, slot = torch.where(state["top_experts"] == expert)
        if not token.numel():
            continue
        weight = _exact_values(state["weight_1"], slice(expert * layer_1_rows, (expert + 1) * layer_1_rows))
        layer_1 = _exact_values(state["rows"], token) @ weight.t()
        gate = layer_1[:, :ffn]
        if case["activation"] == "silu":
            activation = gate * torch.sigmoid(gate)
        elif case["activation"] == "gelu":
            activation = torch.nn.functional.gelu(gate, approximate="tanh")
        else:
            activation = torch.relu(gate) ** 2
        if case["gated"]:
            activation = activation * layer_1[:, ffn:]
        elements, scales = _exact_quantized(activation, case["format"])
        activation = elements * scales.repeat_interleave(32, dim=1)[:, :ffn]
        weight = _exact_values(state["weight_2"], slice(expert * hidden, (expert + 1) * hidden))
        out.index_add_(0, token, (activation @ weight.t()) * state["scores"][token, slot, None].double())
    return out


# ---- what a pass cannot do without -----------------------------------------------------------------------
def _mx_bytes(format: str) -> float:
    return (8 if format == "e4m3" else 4) / 8 + 1 / 32


def _selected(case: dict) -> float:
    """Experts that some token is expected to select."""
    return (1 - (1 - case["slots"] / case["experts"]) ** case["tokens"]) * case["experts"]


def work(case: dict) -> dict:
    size = 4 if case["dtype"] == "fp32" else 2
    if case["kind"] in ("norm_quantize", "norm_step"):
        values = case["tokens"] * case["hidden"]
        if case["kind"] == "norm_quantize":
            return {"bytes": values * (size * (4 if case["residual"] else 2) + _mx_bytes("e4m3")) + case["hidden"] * size, "flops": 8 * values}
        # Forward: input (and stream) in, result (and stream) out; backward: stream or input, gradients in, gradient out.
        return {"bytes": values * size * (8 if case["residual"] else 5) + 2 * case["hidden"] * size, "flops": 20 * values}
    if case["kind"] == "quantize":
        values = case["rows"] * case["columns"]
        there_and_back = 1 if case["format"] == "e4m3" else 2
        return {"bytes": there_and_back * values * (size + _mx_bytes(case["format"])), "flops": there_and_back * 4 * values}
    entries = case["tokens"] * case["slots"]
    if case["kind"] == "product":
        inner, columns = case["inner"], case["columns"]
        return {
            "bytes": _selected(case) * inner * columns * _mx_bytes("e2m1") + entries * (inner * _mx_bytes(case["format"]) + columns * size),
            "flops": 2 * entries * inner * columns,
        }
    products = case["hidden"] * case["ffn"] * (3 if case["gated"] else 2)
    return {
        "bytes": _selected(case) * products * _mx_bytes("e2m1") + case["tokens"] * case["hidden"] * (_mx_bytes(case["format"]) + size),
        "flops": 2 * entries * products,
    }
