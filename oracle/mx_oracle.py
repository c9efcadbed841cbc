"""CPU statement, in 64 bits, of the microscaled formats, the products on them and the root-mean-square norm."""

import torch

BLOCK, COLUMN_MULTIPLE = 32, 128
TOP = {"e4m3": 448.0, "e2m1": 6.0}
# Mantissa bits, exponent of the smallest normal value, exponent of the largest.
GRID = {"e4m3": (3, -6, 8), "e2m1": (1, 0, 2)}
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def quantize(values: torch.Tensor, format: str) -> tuple[torch.Tensor, torch.Tensor]:
    """(elements [rows, columns] float64, scale bytes [rows, ceil(columns / 32)] int64)."""
    mantissa, lowest, highest = GRID[format]
    values = values.double()
    rows, columns = values.shape
    blocks = torch.nn.functional.pad(values, (0, -columns % BLOCK)).unflatten(1, (-(-columns // BLOCK), BLOCK))
    largest = blocks.abs().amax(-1)
    bad = ~torch.isfinite(blocks).all(-1)
    exponent = torch.floor(torch.log2(largest.where(~bad, torch.ones(()).double()))) - highest
    bytes_ = exponent.clamp(-127, 127).nan_to_num(neginf=-127.0).long() + 127
    bytes_ = torch.where(largest == 0, 0, bytes_)
    scaled = blocks * torch.exp2(127.0 - bytes_.double())[..., None]
    spacing = torch.exp2(torch.floor(torch.log2(scaled.abs().clamp_min(2.0**-300))).clamp_min(lowest) - mantissa)
    elements = (torch.round(scaled / spacing) * spacing).clamp(-TOP[format], TOP[format])
    elements = torch.where(bad[..., None], torch.zeros(()).double(), elements)
    return elements.flatten(1)[:, :columns], torch.where(bad, 255, bytes_)


def values_of(elements: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """What elements and scale bytes stand for."""
    scale = torch.where(scales == 255, torch.nan, torch.exp2(scales.double() - 127))
    return elements * scale.repeat_interleave(BLOCK, dim=1)[:, : elements.size(1)]


def pack(elements: torch.Tensor, scales: torch.Tensor, format: str) -> tuple[torch.Tensor, torch.Tensor]:
    """The stored bytes: rows padded to whole groups of 128 columns with zeros."""
    rows, columns = elements.shape
    padded = -(-columns // COLUMN_MULTIPLE) * COLUMN_MULTIPLE
    elements = torch.nn.functional.pad(elements, (0, padded - columns))
    if format == "e4m3":
        values = elements.float().to(torch.float8_e4m3fn).view(torch.uint8)
    else:
        codes = torch.bucketize(elements.abs(), torch.tensor(E2M1, dtype=torch.float64)) + 8 * torch.signbit(elements).long()
        values = (codes[:, ::2] | codes[:, 1::2] << 4).to(torch.uint8)
    return values, torch.nn.functional.pad(scales, (0, padded // BLOCK - scales.size(1))).to(torch.uint8)


def unpack(values: torch.Tensor, scales: torch.Tensor, columns: int, format: str) -> torch.Tensor:
    """The values that stored bytes stand for, [rows, columns] float64."""
    if format == "e4m3":
        elements = values.view(torch.float8_e4m3fn).double()
    else:
        table = torch.tensor(E2M1 + tuple(-value for value in E2M1), dtype=torch.float64)
        elements = table[torch.stack((values & 15, values >> 4), dim=-1).flatten(1).long()]
    return values_of(elements[:, :columns], scales[:, : -(-columns // BLOCK)].long())


def activation(layer_1: torch.Tensor, gated: bool, name: str) -> torch.Tensor:
    gate, up = layer_1.chunk(2, dim=-1) if gated else (layer_1, None)
    gate = {
        "silu": lambda x: x * torch.sigmoid(x),
        "gelu": lambda x: torch.nn.functional.gelu(x, approximate="tanh"),
        "relu": torch.relu,
        "squared_relu": lambda x: torch.relu(x) ** 2,
        "identity": lambda x: x,
    }[name](gate)
    return gate * up if gated else gate


def mlp(
    rows: torch.Tensor, scores: torch.Tensor, top_experts: torch.Tensor, weight_1: torch.Tensor, weight_2: torch.Tensor,
    experts: int, gated: bool, name: str, format: str,
) -> torch.Tensor:  # fmt: skip
    """The expert MLP on the values of quantised operands: weight_1 [experts * ffn (* 2), hidden], weight_2 [experts * hidden, ffn]."""
    out = torch.zeros(rows.size(0), weight_2.size(0) // experts, dtype=torch.float64)
    for e, (w1, w2) in enumerate(zip(weight_1.chunk(experts), weight_2.chunk(experts))):
        token, slot = torch.where(top_experts == e)
        act = values_of(*quantize(activation(rows[token] @ w1.t(), gated, name), format))
        out.index_add_(0, token, (act @ w2.t()) * scores[token, slot, None].double())
    return out


def rms_norm(
    input_: torch.Tensor, weight: torch.Tensor, residual: torch.Tensor | None, eps: float
) -> tuple[torch.Tensor, torch.Tensor]:
    """(normalized in float64, stream): the stream is rounded to the input's type, and that is what is normalised."""
    stream = input_ if residual is None else (input_.double() + residual.double()).to(input_.dtype)
    wide = stream.double()
    return wide / torch.sqrt(wide.square().mean(-1, keepdim=True) + eps) * weight.double(), stream


def rms_norm_backward(
    grad: torch.Tensor, grad_stream: torch.Tensor | None, stream: torch.Tensor, weight: torch.Tensor, eps: float
) -> tuple[torch.Tensor, torch.Tensor]:
    """(gradient of the stream, of the weight), in float64."""
    grad, wide, weight = grad.double(), stream.double(), weight.double()
    inverse = 1 / torch.sqrt(wide.square().mean(-1, keepdim=True) + eps)
    grad_input = inverse * (grad * weight - wide * inverse**2 * (grad * weight * wide).mean(-1, keepdim=True))
    if grad_stream is not None:
        grad_input = grad_input + grad_stream.double()
    return grad_input, (grad * wide * inverse).flatten(0, -2).sum(0)
