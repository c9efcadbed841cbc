"""Products of microscaled rows with scales that differ from block to block: a scale that is read from another place shows."""

import pytest
import torch

from fast_llm_amd.functional.microscaling import MicroscaledTensor, mx_sparse_matmul, mx_sparse_matmul_activation
from oracle import mx_oracle
from tests.mx_values import assert_exact, scaled
from tests.test_gpu_microscaling import _map, _real_rows

pytestmark = pytest.mark.gpu

FORMATS = ["e4m3", "e2m1"]
FEW, MANY = [40, 0, 3], [300, 0, 257, 1, 512]
# Of 128 columns: one and a part, then all remainders of four with one group of four slices and with more.
INNER = [96, 200, 512, 640, 768, 896, 1024, 1152, 1280, 1416, 1536, 1664]


def _expected(rows: torch.Tensor, weight: torch.Tensor, sparse_map) -> torch.Tensor:
    """NaN in the rows that no token has."""
    experts = sparse_map.num_experts
    out = torch.full((rows.size(0), weight.size(0) // experts), torch.nan, dtype=torch.float64, device=rows.device)
    for (_, begin, end), part in zip(_real_rows(sparse_map), weight.chunk(experts)):
        out[begin:end] = rows[begin:end] @ part.t()
        assert_exact(out[begin:end])
    return out


def _same(out: torch.Tensor, expected: torch.Tensor, fill: float) -> None:
    assert torch.equal(out, expected.nan_to_num(fill).to(out.dtype))


@pytest.mark.parametrize("counts", [FEW, MANY], ids=str)
@pytest.mark.parametrize("inner", INNER)
@pytest.mark.parametrize("columns", [33, 260])
@pytest.mark.parametrize("format", FORMATS)
def test_products(counts, inner, columns, format, device):
    generator = torch.Generator(device).manual_seed(inner + columns)
    sparse_map = _map(counts, device, phantom=128)
    (lhs, rows), (rhs, weight) = scaled(generator, (sparse_map.num_rows, inner), format), scaled(generator, (len(counts) * columns, inner), "e2m1")
    expected = _expected(rows, weight, sparse_map)
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        out = torch.full((sparse_map.num_rows, columns), -7.0, dtype=dtype, device=device)
        mx_sparse_matmul(lhs, rhs, sparse_map, out)
        _same(out, expected, -7.0)


@pytest.mark.parametrize("counts", [FEW, [500, 259, 5]], ids=str)
@pytest.mark.parametrize("inner", [512, 640, 896])
@pytest.mark.parametrize("index_dtype", [torch.int16, torch.int32, torch.int64])
@pytest.mark.parametrize("format", FORMATS)
def test_strides_and_index_types(counts, inner, index_dtype, format, device):
    generator, columns = torch.Generator(device).manual_seed(inner), 132
    sparse_map = _map(counts, device, index_dtype, block=1, phantom=3)  # boundaries of any kind
    (lhs, rows), (rhs, weight) = (
        scaled(generator, (2 * size, inner), kind) for size, kind in ((sparse_map.num_rows, format), (len(counts) * columns, "e2m1"))
    )
    expected = _expected(rows[::2], weight[::2], sparse_map)
    # Scales between others that are not theirs.
    operands = []
    for tensor in (lhs, rhs):
        wide = torch.randint(110, 140, (tensor.rows // 2, tensor.scales.size(1) + 12), dtype=torch.uint8, generator=generator, device=device)
        scales = wide[:, 8 : 8 + tensor.scales.size(1)]
        scales.copy_(tensor.scales[::2])
        operands.append(MicroscaledTensor(tensor.values[::2], scales, inner, tensor.format))
    for offset in (0, 1):  # aligned to groups of four and not
        wide = torch.full((sparse_map.num_rows, 2 * columns), -7.0, device=device)
        mx_sparse_matmul(*operands, sparse_map, wide[:, 8 + offset : 8 + offset + columns])
        _same(wide[:, 8 + offset : 8 + offset + columns], expected, -7.0)
        assert (wide[:, : 8 + offset] == -7).all() and (wide[:, 8 + offset + columns :] == -7).all()


@pytest.mark.parametrize("counts", [FEW, MANY], ids=str)
@pytest.mark.parametrize(("inner", "columns"), [(96, 33), (512, 160), (640, 256), (768, 70), (896, 130), (1152, 384)])
@pytest.mark.parametrize("format", FORMATS)
@pytest.mark.parametrize(("gated", "activation"), [(True, "relu"), (False, "squared_relu"), (True, "identity"), (False, "identity")])
def test_activations(counts, inner, columns, format, gated, activation, device):
    generator = torch.Generator(device).manual_seed(inner + columns)
    sparse_map = _map(counts, device)
    (lhs, rows) = scaled(generator, (sparse_map.num_rows, inner), format)
    rhs, weight = scaled(generator, (len(counts) * columns * (1 + gated), inner), "e2m1")
    out = mx_sparse_matmul_activation(lhs, rhs, sparse_map, gated, activation)
    sums = _expected(rows, weight, sparse_map)
    for _, begin, end in _real_rows(sparse_map):
        result = mx_oracle.activation(sums[begin:end].cpu(), gated, activation)
        assert result.numel() == 0 or result.abs().max() < 2**24 * 0.25**2  # multiples of that: exact in fp32
        values, scales = mx_oracle.pack(*mx_oracle.quantize(result, format), format)
        assert torch.equal(out.values[begin:end].cpu(), values) and torch.equal(out.scales[begin:end].cpu(), scales)


@pytest.mark.parametrize("format", FORMATS)
@pytest.mark.parametrize("inner", [640, 768, 896, 1152])
# More tiles of 256 x 256 than CUs: 453, and 297 and 300, where the last round's are in halves of 40, 2, 0 and 0 rows.
@pytest.mark.parametrize("counts", [[30000, 8300], [25000, 130], [20096, 5128, 0]], ids=str)
def test_rounds_of_tiles(counts, inner, format, device):
    generator, columns = torch.Generator(device).manual_seed(sum(counts)), 516
    sparse_map = _map(counts, device)
    (lhs, rows), (rhs, weight) = scaled(generator, (sparse_map.num_rows, inner), format), scaled(generator, (len(counts) * columns, inner), "e2m1")
    out = torch.full((sparse_map.num_rows, columns), -7.0, device=device)
    mx_sparse_matmul(lhs, rhs, sparse_map, out)
    _same(out, _expected(rows, weight, sparse_map), -7.0)


@pytest.mark.parametrize("format", FORMATS)
@pytest.mark.parametrize("of_rows", [True, False])
@pytest.mark.parametrize("rows", [30, 200])
def test_scales_that_are_far_apart(rows, of_rows, format, device):
    """The rows of scales of one tile lie over 2 GiB of memory, those of a block of 32 rows within 4 GiB."""
    generator = torch.Generator(device).manual_seed(3)
    (lhs, left), (rhs, right) = scaled(generator, (rows, 512), format), scaled(generator, (200, 512), "e2m1")
    tensor = lhs if of_rows else rhs
    apart = torch.empty(tensor.rows, 1 << 24, dtype=torch.uint8, device=device)[:, :16]
    apart.copy_(tensor.scales)
    tensor.scales = apart
    _same(mx_sparse_matmul(lhs, rhs, dtype=torch.float32), left @ right.t(), 0.0)


@pytest.mark.parametrize("rows", [8, 300])
@pytest.mark.parametrize("inner", [128, 640, 896])
def test_scales_that_end_with_their_memory(rows, inner, device):
    generator = torch.Generator(device).manual_seed(rows + inner)
    (lhs, left), (rhs, right) = scaled(generator, (rows, inner), "e4m3"), scaled(generator, (64, inner), "e2m1")
    for tensor in (lhs, rhs):
        memory = torch.empty(tensor.rows, 1 << 16, dtype=torch.uint8, device=device)
        scales = memory[:, memory.size(1) - tensor.scales.size(1) :]
        scales.copy_(tensor.scales)
        tensor.scales = scales
    _same(mx_sparse_matmul(lhs, rhs, dtype=torch.float32), left @ right.t(), 0.0)
