"""The oracle of the microscaled formats and of the norm, against cases worked out by hand, torch's casts and differences."""

import pytest
import torch

from oracle import mx_oracle


def test_scales_and_elements_by_hand():
    row = torch.zeros(1, 96)
    row[0, :4] = torch.tensor([6.0, -0.75, 0.25, 1e-9])  # largest 6 = 1.5 * 2^2: scale 2^0 in e2m1, 2^-6 in e4m3
    row[0, 32:35] = torch.tensor([7.9, 5.0, -3.5])  # saturates; 5 and 3.5 are ties: to 4 (even) and 4 (even)
    elements, scales = mx_oracle.quantize(row, "e2m1")
    assert scales.tolist() == [[127, 127, 0]]
    assert elements[0, :4].tolist() == [6.0, -1.0, 0.0, 0.0]
    assert elements[0, 32:35].tolist() == [6.0, 4.0, -4.0]
    elements, scales = mx_oracle.quantize(row, "e4m3")
    assert scales.tolist() == [[127 - 6, 127 - 6, 0]]
    assert elements[0, :3].tolist() == [384.0, -48.0, 16.0]
    assert elements[0, 32:35].tolist() == [448.0, 320.0, -224.0]


def test_blocks_that_are_not_finite_and_the_lowest_scale():
    row = torch.zeros(1, 128)
    row[0, 0], row[0, 33], row[0, 64] = float("inf"), float("nan"), 2.0**-140
    elements, scales = mx_oracle.quantize(row, "e4m3")
    assert scales.tolist() == [[255, 255, 0, 0]]
    assert elements[0, 64] == 0.0 and elements[0, :64].eq(0).all()  # 2^-13 of the lowest scale: under half of e4m3's 2^-9
    assert torch.isnan(mx_oracle.values_of(elements, scales)[0, :64]).all()


@pytest.mark.parametrize("format", ["e4m3", "e2m1"])
def test_bytes_stand_for_the_values(format):
    values = torch.randn(7, 200, generator=torch.Generator().manual_seed(0)) * torch.logspace(-3, 3, 200)
    elements, scales = mx_oracle.quantize(values, format)
    stored = mx_oracle.pack(elements, scales, format)
    assert stored[0].shape == (7, 256 if format == "e4m3" else 128) and stored[1].shape == (7, 8)
    assert torch.equal(mx_oracle.unpack(*stored, 200, format), mx_oracle.values_of(elements, scales))
    if format == "e4m3":  # torch's cast rounds the same way
        scaled = values.double() * torch.exp2(127.0 - scales.double()).repeat_interleave(32, 1)[:, :200]
        assert torch.equal(scaled.clamp(-448, 448).float().to(torch.float8_e4m3fn).double(), elements)


def test_norm_gradients_are_those_of_differences():
    generator = torch.Generator().manual_seed(1)
    stream, weight, grad, grad_stream = (torch.randn(shape, generator=generator, dtype=torch.float64) for shape in ((3, 40), (40,), (3, 40), (3, 40)))
    grads = mx_oracle.rms_norm_backward(grad, grad_stream, stream, weight, 1e-3)

    def loss(stream, weight):
        normalized, _ = mx_oracle.rms_norm(stream, weight, None, 1e-3)
        return (normalized * grad).sum() + (stream * grad_stream).sum()

    step = 1e-6
    for tensor, gradient, at in ((stream, grads[0], (1, 7)), (stream, grads[0], (2, 39)), (weight, grads[1], (0,))):
        ends = []
        for sign in (1, -1):
            moved = tensor.clone()
            moved[at] += sign * step
            ends.append(loss(moved, weight) if tensor is stream else loss(stream, moved))
        # Second order in the step: (1e-6)^2 times third derivatives of order 1e2, and 1e-16 * 1e2 / 1e-6 from the subtraction.
        assert abs((ends[0] - ends[1]) / (2 * step) - gradient[at]) < 1e-7
