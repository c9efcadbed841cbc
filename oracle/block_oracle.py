"""CPU statement, in 64 bits, of values of 8 bits with a scale for each block of 128, and of the expert MLP's step on them."""

import torch

from oracle.mx_oracle import activation

BLOCK, TOP = 128, 448.0


def quantize(values: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(elements [rows, columns] float64, scale bytes [rows, ceil(columns / 128)] int64): scale the smallest power of two that leaves the
    largest magnitude at 448 or below."""
    values = values.double()
    rows, columns = values.shape
    blocks = torch.nn.functional.pad(values, (0, -columns % BLOCK)).unflatten(1, (-(-columns // BLOCK), BLOCK))
    bad = ~torch.isfinite(blocks).all(-1)
    largest = blocks.abs().amax(-1).where(~bad, torch.zeros(()).double())
    mantissa, exponent = torch.frexp(largest)  # m 2^e, m in [1/2, 1), and 448 = 0.875 * 2^9
    exponent = torch.where(largest > 0, exponent - 9 + (mantissa > 0.875), -127).clamp_min(-127).double()
    scaled = blocks * torch.exp2(-exponent)[..., None]
    spacing = torch.exp2(torch.floor(torch.log2(scaled.abs().clamp_min(2.0**-300))).clamp_min(-6) - 3)
    elements = torch.where(bad[..., None], torch.zeros(()).double(), torch.round(scaled / spacing) * spacing)
    return elements.flatten(1)[:, :columns], torch.where(bad, 255, exponent.long() + 127)


def values_of(elements: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """What elements and scale bytes stand for."""
    scale = torch.where(scales == 255, torch.nan, torch.exp2(scales.double() - 127))
    return elements * scale.repeat_interleave(BLOCK, dim=1)[:, : elements.size(1)]


def kept(values: torch.Tensor) -> torch.Tensor:
    """What remains of values in 8 bits."""
    return values_of(*quantize(values))


def transposed_kept(values: torch.Tensor) -> torch.Tensor:
    """What remains in blocks along the columns, not transposed."""
    return kept(values.t().contiguous()).t()


def pack(elements: torch.Tensor, scales: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """The stored bytes: rows padded to whole blocks with zeros, and scales by block column (without what pads its rows)."""
    elements = torch.nn.functional.pad(elements, (0, -elements.size(1) % BLOCK))
    return elements.float().to(torch.float8_e4m3fn).view(torch.uint8), scales.to(torch.uint8).t()


def unpack(values: torch.Tensor, scales: torch.Tensor, columns: int) -> torch.Tensor:
    """The values that stored bytes stand for, [rows, columns] float64."""
    elements = values.view(torch.float8_e4m3fn).double()[:, :columns]
    return values_of(elements, scales[:, : values.size(0)].t().long())


def activation_gradient(grad: torch.Tensor, layer_1: torch.Tensor, gated: bool, name: str) -> torch.Tensor:
    layer_1 = layer_1.detach().requires_grad_(True)
    with torch.enable_grad():
        return torch.autograd.grad(activation(layer_1, gated, name), layer_1, grad)[0]


def mlp_step(input_, scores, top_experts, weight_1, weight_2, experts, gated, name, grad_output, dtype) -> dict:
    """Forward and backward of the MLP in 8 bits, weights unquantised as the layer has them; rounded to `dtype` where the layer does."""
    hidden, ffn = input_.size(1), weight_2.size(0) // experts
    ffn_1 = ffn * (2 if gated else 1)
    rows, scores, grad_output = kept(input_), scores.double(), grad_output.double()
    out = {
        "output": torch.zeros(input_.shape, dtype=torch.float64),
        "grad_input": torch.zeros(input_.shape, dtype=torch.float64),
        "grad_scores": torch.zeros(scores.shape, dtype=torch.float64),
        "grad_weight_1": torch.zeros(weight_1.shape, dtype=torch.float64),
        "grad_weight_2": torch.zeros(weight_2.shape, dtype=torch.float64),
    }
    for expert in range(experts):
        token, slot = torch.where(top_experts == expert)
        if not len(token):
            continue
        of_1, of_2 = slice(expert * ffn_1, (expert + 1) * ffn_1), slice(expert * ffn, (expert + 1) * ffn)
        w_1, w_2 = weight_1[of_1].double(), weight_2[of_2].double()
        x, score, grad = rows[token], scores[token, slot, None], grad_output[token]
        layer_1 = (x @ kept(w_1).t()).to(dtype).double()
        layer_2 = (kept(activation(layer_1, gated, name)) @ transposed_kept(w_2)).to(dtype).double()
        out["output"].index_add_(0, token, layer_2 * score)
        out["grad_scores"][token, slot] = (layer_2 * grad).sum(1)
        grad_2 = (grad * score).to(dtype).double()
        grad_activation = (kept(grad_2) @ kept(w_2).t()).to(dtype).double()
        saved = kept(layer_1)
        out["grad_weight_2"][of_2] = transposed_kept(activation(saved, gated, name)).t() @ transposed_kept(grad_2)
        grad_1 = activation_gradient(grad_activation, saved, gated, name)
        out["grad_input"].index_add_(0, token, (kept(grad_1) @ transposed_kept(w_1)).to(dtype).double())
        out["grad_weight_1"][of_1] = transposed_kept(grad_1).t() @ transposed_kept(x)
    return out
