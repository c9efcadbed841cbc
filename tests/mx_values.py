"""Microscaled operands whose products are known exactly and whose scales differ from block to block and from row to row."""

import torch

from fast_llm_amd.functional.microscaling import MicroscaledTensor, mx_dequantize, mx_quantize

# A block of 32 without a 2 is one in 10^7: its scale is what `scaled_values` gives it.
TABLE = (0.0, 1.0, -1.0, 2.0, -2.0)
# What all values are multiples of, and those of a product.
UNIT, PRODUCT_UNIT = 0.5, 0.25


def scaled_values(generator: torch.Generator, shape: tuple[int, int], factor: float = 1.0) -> torch.Tensor:
    """Whole numbers up to 2, every block of 32 along a row times 1/2, 1 or 2: fp32, on the generator's device."""
    rows, columns = shape
    options = dict(generator=generator, device=generator.device)
    values = torch.tensor(TABLE, device=generator.device)[torch.randint(0, len(TABLE), shape, **options)]
    scales = torch.exp2(torch.randint(-1, 2, (rows, -(-columns // 32)), **options).float())
    return values * scales.repeat_interleave(32, dim=1)[:, :columns] * factor


def scaled(generator: torch.Generator, shape: tuple[int, int], format: str, factor: float = 1.0) -> tuple[MicroscaledTensor, torch.Tensor]:
    """Such values as a microscaled tensor, which holds every one of them, and in fp64. `generator`: of the GPU."""
    values = scaled_values(generator, shape, factor)
    quantized = mx_quantize(values, format)
    assert torch.equal(mx_dequantize(quantized), values)
    if shape[1] >= 32 and shape[0] * shape[1] >= 32 * 32:
        assert quantized.scales[:, : shape[1] // 32].unique().numel() >= 3
    return quantized, values.double()


def assert_exact(sums: torch.Tensor, factor: float = 1.0) -> None:
    """The matrix instruction drops what lies under 2^-17 of the largest of its terms and the sum so far: nothing, where that is below 2^14 units (a quarter
    of the room is left for partial sums that are larger than the whole)."""
    assert sums.numel() == 0 or sums.abs().max() < 2**14 * PRODUCT_UNIT * factor
