"""Which kernel the products of few and many rows run on (the tokens decide, not how the layout is padded), and what is quantised when."""

import ctypes
import subprocess

import pytest
import torch

from fast_llm_amd import _lib
from fast_llm_amd.functional import block_scaling
from fast_llm_amd.functional.block_scaling import BlockScaledTensor
from fast_llm_amd.functional.sparse_copy import SparseMap
from tests.dispatch import CSRC

CPU = torch.device("cpu")
_PROGRAM = """
#include "fm_block_product.h"
using namespace fm::block;

static ProductArgs arguments(int64_t rows, int64_t entries, int64_t columns, int64_t inner, int experts) {
    static char map[2];
    ProductArgs args{};
    args.rows = rows, args.entries = entries, args.columns = columns, args.inner = padded_columns(inner), args.experts = experts;
    args.x_stride = args.weight_stride = args.inner, args.x_scale_stride = (rows + 15) / 16 * 16, args.weight_scale_stride = (experts * columns + 15) / 16 * 16;
    args.out_stride = columns, args.expert_ends = map, args.expert_pad_begins = map + 1;
    return args;
}
extern "C" int tiles(int64_t rows, int64_t entries, int64_t columns, int64_t inner, int experts) { return runs_on_tiles(arguments(rows, entries, columns, inner, experts)); }
extern "C" int split(int64_t rows, int64_t entries, int64_t columns, int64_t inner, int experts) { return stream_split(arguments(rows, entries, columns, inner, experts)); }
"""


@pytest.fixture(scope="module")
def rules(tmp_path_factory, library):
    from fast_llm_amd.build import _hipcc

    folder, library = tmp_path_factory.mktemp("block_rules"), _lib.LIBRARY_PATH
    (folder / "rules.hip").write_text(_PROGRAM)
    subprocess.run(
        [_hipcc(), "--offload-host-only", "-std=c++17", "-fPIC", "-shared", f"-I{CSRC}", str(folder / "rules.hip"), "-o", str(folder / "rules.so"),
         f"-L{library.parent}", f"-l:{library.name}", f"-Wl,-rpath,{library.parent}"],
        check=True, capture_output=True,
    )  # fmt: skip
    found = ctypes.CDLL(str(folder / "rules.so"))
    for rule in (found.tiles, found.split):
        rule.argtypes = [ctypes.c_int64] * 4 + [ctypes.c_int]
    return found


def _worst(entries: int, experts: int) -> int:
    return (entries + experts * 128) // 128 * 128


@pytest.mark.parametrize(("experts", "inner", "columns"), [(8, 4096, 28672), (8, 14336, 4096), (64, 2048, 2816), (128, 768, 2048), (1, 512, 300)])
def test_the_tokens_decide_however_the_layout_is_padded(experts, inner, columns, rules):
    chosen = set()
    for per_expert in (1, 2, 4, 8, 16, 24, 32, 48, 64, 100, 128, 256, 1000):
        entries = per_expert * experts
        worst = _worst(entries, experts)
        padded = experts * -(-per_expert // 128) * 128  # as many for each expert, in a layout for them alone
        choices = {(rules.tiles(rows, entries, columns, inner, experts), rules.split(rows, entries, columns, inner, experts)) for rows in (entries, padded, worst)}
        # ... and as without the entries where the layout has room for any routing.
        choices.add((rules.tiles(worst, 0, columns, inner, experts), rules.split(worst, 0, columns, inner, experts)))
        assert len(choices) == 1, (per_expert, choices)
        chosen.add(choices.pop()[0])
    assert chosen == {0, 1}


@pytest.fixture
def calls(monkeypatch):
    """The calls of the library, none of which is made."""
    monkeypatch.setattr(_lib, "require_device", lambda *tensors: CPU)
    made = []
    monkeypatch.setattr(_lib, "call", lambda name, device, *args: made.append((name, args)))
    return made


def test_products_say_how_many_rows_tokens_have(calls):
    def product(num_rows, entries, experts=4):
        ends = torch.zeros(experts, dtype=torch.int32)
        sparse_map = SparseMap(None, ends, ends, None, num_rows, entries, experts, 2)
        block_scaling.block_sparse_matmul(BlockScaledTensor.empty(num_rows, 256, CPU), BlockScaledTensor.empty(experts * 64, 256, CPU), sparse_map)
        return calls.pop()

    for entries in (2, 130, 1000):
        name, args = product(_worst(entries, 4), entries)
        assert name == "fm_block_sparse_matmul" and len(args) == len(_lib.SIGNATURES[name][1]) - 1
        for rows in {entries, -(-entries // 128) * 128 + 128, 4 * 128 * -(-entries // 128)} - {_worst(entries, 4)}:
            name, args = product(rows, entries)
            assert name == "fm_block_sparse_matmul_counted" and len(args) == len(_lib.SIGNATURES[name][1]) - 1
            assert args[7:12] == (rows, 64, 256, 4, entries)
    assert product(640, None)[0] == "fm_block_sparse_matmul"  # nothing is known


def test_counted_products_validate_before_launching(library):
    def product(rows=256, columns=64, inner=64, experts=2, entries=100, out=256, lhs_stride=128, dtype=1):
        return library.fm_block_sparse_matmul_counted(256, 256, 256, 256, out, 256, 256, rows, columns, inner, experts, entries, lhs_stride, 256, 128, 128, 64, 0,
                                                      dtype, 1, None)  # fmt: skip

    assert product(rows=0) == 0 and product(rows=0, entries=0) == 0
    for bad in (dict(rows=-1), dict(entries=-1), dict(entries=2**31), dict(columns=0), dict(inner=0), dict(experts=0), dict(experts=1025), dict(out=None),
                dict(lhs_stride=64), dict(dtype=3)):  # fmt: skip
        assert product(**bad) == _lib.FM_ERR_INVALID_ARGUMENT, bad
        assert b"counted" in library.fm_last_error()


@pytest.mark.parametrize("weights", [False, True])
def test_inference_quantises_what_its_forward_reads(weights, calls):
    experts, hidden, ffn, tokens = 2, 128, 256, 3
    weight_1, weight_2 = torch.zeros(experts * 2 * ffn, hidden), torch.zeros(experts * ffn, hidden)
    quantized = block_scaling.block_quantize_expert_weights(weight_1, weight_2, experts, training=False) if weights else None
    calls.clear()
    ends = torch.zeros(experts, dtype=torch.int32)
    sparse_map = SparseMap(torch.zeros(tokens, 2, dtype=torch.int32), ends, ends, tokens, 256, 6, experts, 2)
    with torch.no_grad():
        block_scaling.block_mlp(torch.zeros(tokens, hidden), torch.ones(tokens, 2), weight_1, weight_2, quantized, gated=True, activation_type="silu",
                                sparse_map=sparse_map, training=False)  # fmt: skip
    # (rows' values, transposed values) of each quantisation: the input along its rows, and of the weights what the products sum along.
    made = [(args[1] is not None, args[3] is not None) for name, args in calls if name == "fm_block_quantize"]
    assert made == ([] if weights else [(True, False), (False, True)]) + [(True, False)]
    with pytest.raises(ValueError, match="for inference"):
        block_scaling.block_mlp(
            torch.zeros(tokens, hidden), torch.ones(tokens, 2), weight_1, weight_2,
            block_scaling.block_quantize_expert_weights(weight_1, weight_2, experts, training=False),
            gated=True, activation_type="silu", sparse_map=sparse_map,
        )  # fmt: skip
