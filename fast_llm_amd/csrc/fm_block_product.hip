// Entry points of the products of operands of 8 bits with a scale per block of 128: their checks, and which kernel they run on.
#include <algorithm>

#include "fm_block_product.h"

using namespace fm;

namespace {

int check_sizes(const char *name, int64_t rows, int64_t columns, int64_t inner, int64_t num_experts, int out_dtype) {
    FM_REQUIRE(valid_dtype(out_dtype), "%s: bad dtype %d", name, out_dtype);
    FM_REQUIRE(num_experts > 0 && num_experts <= 1024, "%s: num_experts = %lld is not in 1 .. 1024", name, static_cast<long long>(num_experts));
    FM_REQUIRE(rows >= 0 && rows < (int64_t(1) << 31) && columns > 0 && columns <= (int64_t(1) << 28) && inner > 0 && inner <= block::kMaxColumns &&
                   num_experts * std::max(rows, columns) < (int64_t(1) << 40), "%s: bad sizes", name);
    return FM_OK;
}

int check_result(const char *name, const void *out, int64_t columns, int64_t out_stride, int out_dtype) {
    FM_REQUIRE(out != nullptr, "%s: null tensor", name);
    FM_REQUIRE(out_stride >= columns, "%s: rows of the result overlap", name);
    FM_REQUIRE(reinterpret_cast<uintptr_t>(out) % dtype_size(out_dtype) == 0, "%s: misaligned result", name);
    return FM_OK;
}

}  // namespace

bool block::runs_on_tiles(const ProductArgs &args) {
    // The tiles read the weights once, at 4 TB/s where little is multiplied and there is a tile for every CU; with few rows the weights are read once
    // per 32 rows of an expert, at up to 6. So it depends on how many experts have over 32 rows, and on the tiles. Measured in us, few rows | tiles,
    // with tokens at random: 8 experts 4096 -> 2 x 14336, 1 token 42 | 60, 8 rows per expert 153 | 234, 24 rows 197 | 238; 14336 -> 4096 22 | 112, 80
    // | 164, 103 | 165; 64 experts 2048 -> 2 x 1408, 8 rows 65 | 83, 24 rows 84 | 87; 128 experts 2048 -> 2 x 768, 70 | 86 and 100 | 91. One expert,
    // 4096 -> 28672 (112 tiles): 32 rows 31 | 50, 48 rows 54 | 50; 14336 -> 4096 (16 tiles): 128 rows 98 | 155, 192 rows 145 | 150. Of a map the host
    // knows the rows with up to 128 of padding per expert (`rows_of_any_routing`); without one it knows them exactly.
    const int64_t tiles = (args.columns + 255) / 256 * args.experts, times = std::min(std::max(80 / tiles, int64_t(1)), int64_t(5));
    const bool many = args.expert_ends != nullptr ? rows_of_any_routing(args) > (128 + 24 * times) * args.experts : args.rows > 32 * times;
    return (many || !stream_product_takes(args)) && tile_product_takes(args);
}

namespace {

int sparse_matmul(const char *name, const void *lhs, const void *lhs_scales, const void *rhs, const void *rhs_scales, void *out, const void *expert_ends,
                  const void *expert_pad_begins, int64_t rows, int64_t columns, int64_t inner, int64_t num_experts, int64_t num_entries, int64_t lhs_stride,
                  int64_t lhs_scale_stride, int64_t rhs_stride, int64_t rhs_scale_stride, int64_t out_stride, int exact_sums, int out_dtype, int index_dtype,
                  void *stream) {
    if (int status = check_sizes(name, rows, columns, inner, num_experts, out_dtype)) return status;
    block::RowMap map;
    if (int status = block::check_map(name, map, expert_ends, expert_pad_begins, num_experts, index_dtype)) return status;
    FM_REQUIRE(expert_ends != nullptr || num_experts == 1, "%s: several experts and no map", name);
    if (rows == 0) return FM_OK;
    const int64_t padded = block::padded_columns(inner);
    if (int status = block::check_tensor(name, "lhs", lhs, lhs_scales, rows, padded, lhs_stride, lhs_scale_stride)) return status;
    if (int status = block::check_tensor(name, "rhs", rhs, rhs_scales, num_experts * columns, padded, rhs_stride, rhs_scale_stride)) return status;
    if (int status = check_result(name, out, columns, out_stride, out_dtype)) return status;
    block::ProductArgs args{};
    args.x = static_cast<const uint8_t *>(lhs), args.x_scales = static_cast<const uint8_t *>(lhs_scales);
    args.weight = static_cast<const uint8_t *>(rhs), args.weight_scales = static_cast<const uint8_t *>(rhs_scales), args.out = out;
    args.x_stride = lhs_stride, args.x_scale_stride = lhs_scale_stride, args.weight_stride = rhs_stride, args.weight_scale_stride = rhs_scale_stride;
    args.out_stride = out_stride, args.rows = rows, args.entries = num_entries, args.columns = columns, args.inner = padded, args.experts = num_experts, args.out_dtype = out_dtype;
    args.exact = exact_sums != 0;
    args.out_vectors = aligned16(out) && out_stride * dtype_size(out_dtype) % 16 == 0;
    args.expert_ends = expert_ends, args.expert_pad_begins = expert_pad_begins, args.index_dtype = index_dtype;
    const bool tiles = block::runs_on_tiles(args);
    if (!(tiles ? block::tile_product_takes(args) : block::stream_product_takes(args))) return fail(FM_ERR_UNSUPPORTED, "%s: too large", name);
    if (int status = tiles ? block::tile_product(args, static_cast<hipStream_t>(stream)) : block::stream_product(args, static_cast<hipStream_t>(stream))) return status;
    return check_launch(name);
}

}  // namespace

extern "C" int fm_block_sparse_matmul(const void *lhs, const void *lhs_scales, const void *rhs, const void *rhs_scales, void *out, const void *expert_ends,
                                      const void *expert_pad_begins, int64_t rows, int64_t columns, int64_t inner, int64_t num_experts, int64_t lhs_stride,
                                      int64_t lhs_scale_stride, int64_t rhs_stride, int64_t rhs_scale_stride, int64_t out_stride, int exact_sums, int out_dtype,
                                      int index_dtype, void *stream) {
    return sparse_matmul("fm_block_sparse_matmul", lhs, lhs_scales, rhs, rhs_scales, out, expert_ends, expert_pad_begins, rows, columns, inner, num_experts, 0, lhs_stride,
                         lhs_scale_stride, rhs_stride, rhs_scale_stride, out_stride, exact_sums, out_dtype, index_dtype, stream);
}

extern "C" int fm_block_sparse_matmul_counted(const void *lhs, const void *lhs_scales, const void *rhs, const void *rhs_scales, void *out, const void *expert_ends,
                                              const void *expert_pad_begins, int64_t rows, int64_t columns, int64_t inner, int64_t num_experts,
                                              int64_t num_entries, int64_t lhs_stride, int64_t lhs_scale_stride, int64_t rhs_stride, int64_t rhs_scale_stride,
                                              int64_t out_stride, int exact_sums, int out_dtype, int index_dtype, void *stream) {
    const char *name = "fm_block_sparse_matmul_counted";
    FM_REQUIRE(num_entries >= 0 && num_entries < (int64_t(1) << 31), "%s: num_entries = %lld", name, static_cast<long long>(num_entries));
    return sparse_matmul(name, lhs, lhs_scales, rhs, rhs_scales, out, expert_ends, expert_pad_begins, rows, columns, inner, num_experts, num_entries, lhs_stride,
                         lhs_scale_stride, rhs_stride, rhs_scale_stride, out_stride, exact_sums, out_dtype, index_dtype, stream);
}

extern "C" int fm_block_input_row_sparse_matmul(const void *lhs, const void *lhs_scales, const void *rhs, const void *rhs_scales, void *out,
                                                const void *expert_ends, const void *expert_pad_begins, int64_t rows, int64_t columns, int64_t inner,
                                                int64_t num_experts, int64_t lhs_stride, int64_t lhs_scale_stride, int64_t rhs_stride, int64_t rhs_scale_stride,
                                                int64_t out_stride, int accumulate, int out_dtype, int index_dtype, void *stream) {
    const char *name = "fm_block_input_row_sparse_matmul";
    if (int status = check_sizes(name, rows, columns, inner, num_experts, out_dtype)) return status;
    block::RowMap map;
    if (int status = block::check_map(name, map, expert_ends, expert_pad_begins, num_experts, index_dtype)) return status;
    FM_REQUIRE(expert_ends != nullptr || num_experts == 1, "%s: several experts and no map", name);
    if (rows == 0) return FM_OK;
    const int64_t padded = block::padded_columns(inner);
    if (int status = block::check_tensor(name, "lhs", lhs, lhs_scales, rows, padded, lhs_stride, lhs_scale_stride)) return status;
    if (int status = block::check_tensor(name, "rhs", rhs, rhs_scales, columns, padded, rhs_stride, rhs_scale_stride)) return status;
    if (int status = check_result(name, out, columns, out_stride, out_dtype)) return status;
    block::ProductArgs args{};
    args.x = static_cast<const uint8_t *>(lhs), args.x_scales = static_cast<const uint8_t *>(lhs_scales);
    args.weight = static_cast<const uint8_t *>(rhs), args.weight_scales = static_cast<const uint8_t *>(rhs_scales), args.out = out;
    args.x_stride = lhs_stride, args.x_scale_stride = lhs_scale_stride, args.weight_stride = rhs_stride, args.weight_scale_stride = rhs_scale_stride;
    args.out_stride = out_stride, args.rows = rows, args.columns = columns, args.inner = padded, args.experts = num_experts, args.out_dtype = out_dtype;
    args.by_inner = 1, args.accumulate = accumulate != 0;
    args.out_vectors = aligned16(out) && out_stride * dtype_size(out_dtype) % 16 == 0;
    args.expert_ends = expert_ends, args.expert_pad_begins = expert_pad_begins, args.index_dtype = index_dtype;
    if (!block::tile_product_takes(args)) return fail(FM_ERR_UNSUPPORTED, "%s: too large", name);
    if (int status = block::tile_product(args, static_cast<hipStream_t>(stream))) return status;
    return check_launch(name);
}
