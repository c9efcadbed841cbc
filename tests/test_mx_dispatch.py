"""Which kernel the microscaled products of the tests run on, asked of the library's own rules without a GPU."""

import ctypes
import subprocess

import pytest

from tests import test_gpu_microscaled_paths as paths
from tests import test_gpu_microscaled_scales as scales
from tests.dispatch import CSRC

_PROGRAM = """
#include "fm_mx_product.h"
using namespace fm::mx;

static ProductArgs product(int64_t rows, int64_t columns, int64_t inner, int experts, int gated, int quantized, int format) {
    ProductArgs args{};
    args.format = format, args.gated = gated, args.rows = args.x_rows = rows, args.experts = experts;
    args.columns = columns, args.out_columns = quantized ? padded_columns(columns) : columns, args.inner = padded_columns(inner);
    args.x_stride = value_bytes(format, args.inner), args.weight_stride = value_bytes(FM_MX_E2M1, args.inner);
    args.x_scale_stride = args.weight_scale_stride = scale_bytes(args.inner);
    return args;
}
// By a map: 0 for tiles, or the wavefronts that share a reduction.
extern "C" int by_map(int64_t rows, int64_t columns, int64_t inner, int experts, int gated, int quantized, int format) {
    static char ends[2];
    ProductArgs args = product(rows, columns, inner, experts, gated, quantized, format);
    args.expert_ends = ends, args.expert_pad_begins = ends + 1;
    return runs_on_tiles(args) ? 0 : stream_split(args);
}
extern "C" int by_entries(int64_t entries, int64_t columns, int64_t inner, int experts, int gated, int quantized, int format) {
    static int64_t top_experts[1];
    ProductArgs args = product(entries, columns, inner, experts, gated, quantized, format);
    args.top_experts = top_experts, args.entries = static_cast<int>(entries), args.by_entry = entries < experts;
    return stream_split(args);
}
"""


@pytest.fixture(scope="module")
def rules(tmp_path_factory, library):
    from fast_llm_amd import _lib
    from fast_llm_amd.build import _hipcc

    folder, library = tmp_path_factory.mktemp("mx_dispatch"), _lib.LIBRARY_PATH
    (folder / "rules.hip").write_text(_PROGRAM)
    subprocess.run(
        [_hipcc(), "--offload-host-only", "-std=c++17", "-fPIC", "-shared", f"-I{CSRC}", str(folder / "rules.hip"), "-o", str(folder / "rules.so"),
         f"-L{library.parent}", f"-l:{library.name}", f"-Wl,-rpath,{library.parent}"],
        check=True, capture_output=True,
    )  # fmt: skip
    found = ctypes.CDLL(str(folder / "rules.so"))
    for function in (found.by_map, found.by_entries):
        function.argtypes = [ctypes.c_int64] * 3 + [ctypes.c_int] * 4
    return found


def _rows(counts, block=128, phantom=0):
    return sum(-(-count // block) * block for count in counts) + phantom


def _kinds(formats=(0, 1)):
    """(gated, quantised result, format)"""
    return [(gated, quantized, format) for format in formats for gated, quantized in ((0, 0), (0, 1), (1, 1))]


def test_scales_of_few_and_many_rows(rules):
    for inner in scales.INNER:
        for columns in (33, 260):
            for format in (0, 1):
                few = 1 if inner <= 768 else 4
                assert rules.by_map(_rows(scales.FEW, phantom=128), columns, inner, 3, 0, 0, format) == few
                assert rules.by_map(_rows(scales.MANY, phantom=128), columns, inner, 5, 0, 0, format) == (0 if inner >= 512 else 1), (inner, columns)
    for inner in (512, 640, 896):
        assert rules.by_map(_rows([500, 259, 5], 1, 3), 132, inner, 3, 0, 0, 0) == 0
    for inner, columns in ((512, 160), (640, 256), (768, 70), (896, 130), (1152, 384)):
        for kind in _kinds():
            assert rules.by_map(_rows(scales.MANY), columns, inner, 5, *kind) == 0, (inner, columns, kind)
    for counts in ([30000, 8300], [25000, 130], [20096, 5128, 0]):
        assert rules.by_map(_rows(counts), 516, 640, len(counts), 0, 0, 0) == 0


def test_tiles(rules):
    for counts, block, inner, columns in paths.MANY_EXPERTS:
        assert len(counts) > 128
        for kind in _kinds():
            assert rules.by_map(_rows(counts, block, 5), columns, inner, len(counts), *kind) == 0, (len(counts), kind)
    for counts, inner, columns in paths.ACTIVATIONS:
        for kind in _kinds():
            assert rules.by_map(_rows(counts), columns, inner, len(counts), *kind) == 0, (counts, kind)
    for tokens, experts, slots, hidden, ffn in paths.MLPS:
        rows = (tokens * slots + experts * 128) // 128 * 128
        for format in (0, 1):
            for gated in (0, 1):
                assert rules.by_map(rows, ffn, hidden, experts, gated, 1, format) == 0
            assert rules.by_map(rows, hidden, ffn, experts, 0, 0, format) == 0


def test_few_rows(rules):
    for counts, inner, columns, split in paths.BY_MAP:
        for gated, quantized, format in _kinds():
            assert rules.by_map(_rows(counts, phantom=5), columns, inner, len(counts), gated, quantized, format) == split, (inner, columns, gated)
    assert {case[-1] for case in paths.BY_MAP} == {1, 4, 8}
    for tokens, experts, slots, hidden, ffn, gated, first, second in paths.BY_ENTRIES:
        for format in (0, 1):
            assert rules.by_entries(tokens * slots, ffn, hidden, experts, gated, 1, format) == first, (hidden, ffn)
            assert rules.by_entries(tokens * slots, hidden, ffn, experts, 0, 0, format) == second, (hidden, ffn)
    assert {case[-2] for case in paths.BY_ENTRIES} == {case[-1] for case in paths.BY_ENTRIES} == {1, 4, 8}
    # More than one group of four chunks per wavefront, with every number of them.
    for split in (1, 4, 8):
        assert any(-(-(-(-inner // 256)) // split) > 4 for _, inner, _, s in paths.BY_MAP if s == split)
        assert any(-(-(-(-hidden // 256)) // first) > 4 for _, _, _, hidden, _, _, first, _ in paths.BY_ENTRIES if first == split)
