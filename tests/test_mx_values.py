"""The operands of the tests of microscaled products tell a wrong scale from the right one: the mistakes are planted in the oracle."""

import pytest
import torch

from oracle import mx_oracle
from tests.mx_values import assert_exact, scaled_values


def _products(rows: tuple, weight: tuple, columns: int, format: str) -> torch.Tensor:
    return mx_oracle.values_of(*rows) @ mx_oracle.values_of(*weight).t()


@pytest.mark.parametrize("format", ["e4m3", "e2m1"])
@pytest.mark.parametrize("columns", [128, 640])
def test_scales_from_another_place_show(columns, format):
    generator = torch.Generator().manual_seed(columns)
    rows = mx_oracle.quantize(values := scaled_values(generator, (40, columns)), format)
    weight = mx_oracle.quantize(scaled_values(generator, (36, columns)), "e2m1")
    assert torch.equal(mx_oracle.values_of(*rows), values.double())
    right = _products(rows, weight, columns, format)
    assert_exact(right)
    assert torch.equal(right / 0.25, torch.round(right / 0.25))
    for shift, axis in ((1, 0), (8, 0), (1, 1), (2, 1)):  # of another row, of another block
        for which in (0, 1):
            operands = [rows, weight]
            operands[which] = operands[which][0], torch.roll(operands[which][1], shift, axis)
            wrong = _products(*operands, columns, format) != right
            assert wrong.double().mean() > 0.8, (shift, axis, which)
    # One block of one row: every product of that row but a few.
    scales = rows[1].clone()
    scales[7, columns // 32 - 1] += 1
    wrong = _products((rows[0], scales), weight, columns, format) != right
    assert wrong[7].double().mean() > 0.8 and wrong.any(1).sum() == 1
