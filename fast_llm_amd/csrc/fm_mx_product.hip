// Entry points of the products with e2m1 expert weights: their checks, and which kernel they run on.
#include "fm_mx_product.h"

using namespace fm;

namespace {

constexpr int64_t kMost32 = (int64_t(1) << 32) - 4096;

// What all of them ask of a microscaled tensor.
int check_tensor(const char *name, const char *what, const void *values, const void *scales, int64_t columns, int64_t value_stride, int64_t scale_stride,
                 int format) {
    FM_REQUIRE(values && scales, "%s: null %s", name, what);
    FM_REQUIRE(value_stride >= mx::value_bytes(format, columns) && scale_stride >= mx::scale_bytes(columns), "%s: rows of %s overlap", name, what);
    FM_REQUIRE(aligned16(values) && value_stride % 16 == 0, "%s: rows of %s are 16-byte aligned", name, what);
    FM_REQUIRE(reinterpret_cast<uintptr_t>(scales) % 4 == 0 && scale_stride % 4 == 0, "%s: rows of scales of %s are 4-byte aligned", name, what);
    // 32 rows are addressed in 32 bits from the first.
    if (value_stride > kMost32 / 64 || scale_stride > kMost32 / 64) return fail(FM_ERR_UNSUPPORTED, "%s: rows of %s are too long", name, what);
    return FM_OK;
}

int check_sizes(const char *name, int64_t rows, int64_t columns, int64_t inner, int64_t num_experts, int format) {
    FM_REQUIRE(mx::valid_format(format), "%s: bad format %d", name, format);
    FM_REQUIRE(rows >= 0 && rows < (int64_t(1) << 31) && columns > 0 && columns <= (int64_t(1) << 28) && inner > 0 && inner <= (int64_t(1) << 24), "%s: bad sizes", name);
    FM_REQUIRE(num_experts > 0 && num_experts <= 1024, "%s: num_experts = %lld is not in 1 .. 1024", name, static_cast<long long>(num_experts));
    return FM_OK;
}

int run(const mx::ProductArgs &args, void *stream) {
    return mx::runs_on_tiles(args) ? mx::tile_product(args, static_cast<hipStream_t>(stream)) : mx::stream_product(args, static_cast<hipStream_t>(stream));
}

}  // namespace

bool mx::runs_on_tiles(const ProductArgs &args) {
    // The tiles read the weights once, at 3.8 TB/s where little is multiplied and there is a tile for every CU; with few rows the weights are read once
    // per 32 rows of an expert, at 4.8 TB/s. So it depends on how many experts have over 32 rows, and on the tiles. Measured in us, few rows | tiles,
    // with both layers' weights of 8 experts (4096, 2 x 14336), 64 (2048, 2 x 1408) and 128 (2048, 2 x 768) and tokens at random: 16 rows per
    // expert 165 | 221, 75 | 82, 74 | 96; 32 rows 273 | 239, 135 | 89, 137 | 95. One expert, 4096 -> 28672 (112 tiles): 32 rows 28 | 34, 48 rows 45 | 36;
    // 14336 -> 4096 (16 tiles): 128 rows 83 | 102. Of a map the host knows the rows with up to 128 of padding per expert; without one (the
    // ends are those of the rows) it knows them exactly. (Rows per expert are an average: of 375 tokens with 8 slots over 128 experts, all in 8 experts, those are
    // read a dozen times each, 512 us in `mx_mlp` without a map and 376 with one, where they take 123 and 119 spread over all.)
    const int64_t tiles = (args.out_columns + 255) / 256 * (args.gated ? 2 : 1) * args.experts, times = min(max(80 / tiles, int64_t(1)), int64_t(4));
    const bool exact = args.expert_ends == args.expert_pad_begins;
    const bool many = args.rows > (exact ? 32 * times : 128 + 24 * times) * args.experts;
    return many && tile_product_takes(args);
}

extern "C" int fm_mx_sparse_matmul(const void *lhs, const void *lhs_scales, const void *rhs, const void *rhs_scales, void *out, const void *expert_ends,
                                   const void *expert_pad_begins, int64_t rows, int64_t columns, int64_t inner, int64_t num_experts,
                                   int64_t lhs_stride, int64_t lhs_scale_stride, int64_t rhs_stride, int64_t rhs_scale_stride, int64_t out_stride,
                                   int format, int out_dtype, int index_dtype, void *stream) {
    const char *name = "fm_mx_sparse_matmul";
    if (int status = check_sizes(name, rows, columns, inner, num_experts, format)) return status;
    FM_REQUIRE(valid_dtype(out_dtype), "%s: bad dtype %d", name, out_dtype);
    FM_REQUIRE(valid_index_dtype(index_dtype), "%s: bad index dtype %d", name, index_dtype);
    if (rows == 0) return FM_OK;
    const int64_t padded = mx::padded_columns(inner);
    if (int status = check_tensor(name, "lhs", lhs, lhs_scales, padded, lhs_stride, lhs_scale_stride, format)) return status;
    if (int status = check_tensor(name, "rhs", rhs, rhs_scales, padded, rhs_stride, rhs_scale_stride, FM_MX_E2M1)) return status;
    FM_REQUIRE(out && expert_ends && expert_pad_begins, "%s: null tensor", name);
    FM_REQUIRE(out_stride >= columns, "%s: rows of the result overlap", name);
    const int size = dtype_size(out_dtype);
    FM_REQUIRE(reinterpret_cast<uintptr_t>(out) % size == 0, "%s: misaligned result", name);
    mx::ProductArgs args{};
    args.x = static_cast<const uint8_t *>(lhs), args.x_scales = static_cast<const uint8_t *>(lhs_scales);
    args.weight = static_cast<const uint8_t *>(rhs), args.weight_scales = static_cast<const uint8_t *>(rhs_scales), args.out = out;
    args.x_rows = args.rows = rows, args.x_stride = lhs_stride, args.x_scale_stride = lhs_scale_stride;
    args.weight_stride = rhs_stride, args.weight_scale_stride = rhs_scale_stride, args.out_stride = out_stride;
    args.columns = args.out_columns = columns, args.inner = padded, args.experts = num_experts, args.format = format;
    args.out_dtype = out_dtype;
    args.out_vectors = aligned16(out) && out_stride * size % 16 == 0;
    args.expert_ends = expert_ends, args.expert_pad_begins = expert_pad_begins, args.index_dtype = index_dtype;
    if (int status = run(args, stream)) return status;
    return check_launch(name);
}

extern "C" int fm_mx_sparse_matmul_activation(const void *lhs, const void *lhs_scales, const void *rhs, const void *rhs_scales, void *out_values,
                                              void *out_scales, const void *expert_ends, const void *expert_pad_begins, int64_t rows, int64_t columns,
                                              int64_t inner, int64_t num_experts, int64_t lhs_stride, int64_t lhs_scale_stride, int64_t rhs_stride,
                                              int64_t rhs_scale_stride, int gated, int activation, int format, int index_dtype, void *stream) {
    const char *name = "fm_mx_sparse_matmul_activation";
    if (int status = check_sizes(name, rows, columns, inner, num_experts, format)) return status;
    FM_REQUIRE(activation >= FM_ACT_GELU && activation <= FM_ACT_IDENTITY, "%s: bad activation %d", name, activation);
    FM_REQUIRE(valid_index_dtype(index_dtype), "%s: bad index dtype %d", name, index_dtype);
    if (rows == 0) return FM_OK;
    const int64_t padded = mx::padded_columns(inner);
    if (int status = check_tensor(name, "lhs", lhs, lhs_scales, padded, lhs_stride, lhs_scale_stride, format)) return status;
    if (int status = check_tensor(name, "rhs", rhs, rhs_scales, padded, rhs_stride, rhs_scale_stride, FM_MX_E2M1)) return status;
    FM_REQUIRE(out_values && out_scales && expert_ends && expert_pad_begins, "%s: null tensor", name);
    FM_REQUIRE(aligned16(out_values) && aligned16(out_scales), "%s: results are 16-byte aligned", name);
    mx::ProductArgs args{};
    args.x = static_cast<const uint8_t *>(lhs), args.x_scales = static_cast<const uint8_t *>(lhs_scales);
    args.weight = static_cast<const uint8_t *>(rhs), args.weight_scales = static_cast<const uint8_t *>(rhs_scales);
    args.out = out_values, args.out_scales = static_cast<uint8_t *>(out_scales);
    args.x_rows = args.rows = rows, args.x_stride = lhs_stride, args.x_scale_stride = lhs_scale_stride;
    args.weight_stride = rhs_stride, args.weight_scale_stride = rhs_scale_stride;
    args.columns = columns, args.out_columns = mx::padded_columns(columns), args.inner = padded, args.experts = num_experts, args.format = format;
    args.out_stride = mx::value_bytes(format, args.out_columns), args.out_scale_stride = mx::scale_bytes(args.out_columns);
    args.gated = gated != 0, args.activation = activation;
    args.expert_ends = expert_ends, args.expert_pad_begins = expert_pad_begins, args.index_dtype = index_dtype;
    if (int status = run(args, stream)) return status;
    return check_launch(name);
}

namespace {

// Where the scratch of the few-token MLP lies: the activations' values and scales, then the second layer's fp32 sums.
struct FewTokensLayout {
    int64_t entries, ffn, hidden_stride;
    size_t scales_at, sums_at, size;
};

bool few_tokens_layout(FewTokensLayout &layout, int64_t tokens, int64_t slots, int64_t hidden, int64_t ffn, int64_t experts, int format) {
    if (tokens <= 0 || slots <= 0 || hidden <= 0 || ffn <= 0 || experts <= 0 || experts > 1024 || !mx::valid_format(format)) return false;
    if (tokens > mx::kMaxEntries || slots > mx::kMaxEntries || tokens * slots > mx::kMaxEntries) return false;
    if (hidden > (1 << 20) || ffn > (1 << 20) || tokens > 65535) return false;
    layout.entries = tokens * slots;
    layout.ffn = mx::padded_columns(ffn), layout.hidden_stride = (hidden + 3) / 4 * 4;
    // Rows are addressed in 32 bits.
    if (layout.entries * max(layout.ffn, mx::padded_columns(hidden)) >= kMost32) return false;
    const auto rounded = [](size_t bytes) { return (bytes + 255) / 256 * 256; };
    layout.scales_at = rounded(layout.entries * mx::value_bytes(format, layout.ffn));
    layout.sums_at = layout.scales_at + rounded(layout.entries * mx::scale_bytes(layout.ffn));
    layout.size = layout.sums_at + layout.entries * layout.hidden_stride * sizeof(float);
    return true;
}

}  // namespace

extern "C" size_t fm_mx_few_tokens_workspace_size(int64_t num_tokens, int64_t slots_per_token, int64_t hidden, int64_t ffn, int64_t num_experts, int format) {
    FewTokensLayout layout;
    return few_tokens_layout(layout, num_tokens, slots_per_token, hidden, ffn, num_experts, format) ? layout.size : 0;
}

extern "C" int fm_mx_few_tokens_forward(const void *input, const void *input_scales, const void *top_experts, const void *scores, const void *weight_1,
                                        const void *weight_1_scales, const void *weight_2, const void *weight_2_scales, void *output, int64_t num_tokens,
                                        int64_t slots_per_token, int64_t hidden, int64_t ffn, int64_t num_experts, int64_t input_stride,
                                        int64_t input_scale_stride, int64_t weight_1_stride, int64_t weight_1_scale_stride, int64_t weight_2_stride,
                                        int64_t weight_2_scale_stride, int gated, int activation, int format, int out_dtype, void *workspace,
                                        size_t workspace_size, void *stream) {
    const char *name = "fm_mx_few_tokens_forward";
    FM_REQUIRE(activation >= FM_ACT_GELU && activation <= FM_ACT_IDENTITY, "%s: bad activation %d", name, activation);
    FM_REQUIRE(mx::valid_format(format), "%s: bad format %d", name, format);
    FM_REQUIRE(valid_dtype(out_dtype), "%s: bad dtype %d", name, out_dtype);
    FewTokensLayout layout;
    if (!few_tokens_layout(layout, num_tokens, slots_per_token, hidden, ffn, num_experts, format))
        return fail(FM_ERR_UNSUPPORTED, "%s: at most %d (token, slot) pairs and 1024 experts", name, mx::kMaxEntries);
    FM_REQUIRE(top_experts && scores && output, "%s: null tensor", name);
    FM_REQUIRE(reinterpret_cast<uintptr_t>(output) % dtype_size(out_dtype) == 0, "%s: misaligned output", name);
    const int64_t padded = mx::padded_columns(hidden);
    if (int status = check_tensor(name, "the input", input, input_scales, padded, input_stride, input_scale_stride, format)) return status;
    if (int status = check_tensor(name, "layer 1", weight_1, weight_1_scales, padded, weight_1_stride, weight_1_scale_stride, FM_MX_E2M1)) return status;
    if (int status = check_tensor(name, "layer 2", weight_2, weight_2_scales, layout.ffn, weight_2_stride, weight_2_scale_stride, FM_MX_E2M1))
        return status;
    if (num_tokens * max(input_stride, input_scale_stride) >= kMost32) return fail(FM_ERR_UNSUPPORTED, "%s: rows of the input are too far apart", name);
    FM_REQUIRE(workspace && aligned16(workspace) && workspace_size >= layout.size, "%s: workspace of %zu bytes (16-byte aligned) needed, got %zu", name,
               layout.size, workspace_size);
    mx::ProductArgs layer_1{};
    layer_1.experts = num_experts, layer_1.format = format, layer_1.gated = gated != 0, layer_1.activation = activation;
    layer_1.top_experts = static_cast<const int64_t *>(top_experts);
    layer_1.entries = static_cast<int>(layout.entries), layer_1.by_entry = layout.entries < num_experts;
    mx::ProductArgs layer_2 = layer_1;
    uint8_t *scratch = static_cast<uint8_t *>(workspace);
    layer_1.entries_per_row = static_cast<int>(slots_per_token);
    layer_1.x = static_cast<const uint8_t *>(input), layer_1.x_scales = static_cast<const uint8_t *>(input_scales);
    layer_1.x_rows = num_tokens, layer_1.x_stride = input_stride, layer_1.x_scale_stride = input_scale_stride;
    layer_1.weight = static_cast<const uint8_t *>(weight_1), layer_1.weight_scales = static_cast<const uint8_t *>(weight_1_scales);
    layer_1.weight_stride = weight_1_stride, layer_1.weight_scale_stride = weight_1_scale_stride;
    layer_1.out = scratch, layer_1.out_scales = scratch + layout.scales_at;
    layer_1.out_stride = mx::value_bytes(format, layout.ffn), layer_1.out_scale_stride = mx::scale_bytes(layout.ffn);
    layer_1.columns = ffn, layer_1.out_columns = layout.ffn, layer_1.inner = padded;
    layer_2.gated = 0, layer_2.entries_per_row = 1;
    layer_2.x = scratch, layer_2.x_scales = layer_1.out_scales;
    layer_2.x_rows = layout.entries, layer_2.x_stride = layer_1.out_stride, layer_2.x_scale_stride = layer_1.out_scale_stride;
    layer_2.weight = static_cast<const uint8_t *>(weight_2), layer_2.weight_scales = static_cast<const uint8_t *>(weight_2_scales);
    layer_2.weight_stride = weight_2_stride, layer_2.weight_scale_stride = weight_2_scale_stride;
    layer_2.out = scratch + layout.sums_at, layer_2.out_stride = layout.hidden_stride, layer_2.out_vectors = 1, layer_2.out_dtype = FM_DTYPE_F32;
    layer_2.columns = layer_2.out_columns = hidden, layer_2.inner = layout.ffn;
    if (int status = mx::few_tokens(layer_1, layer_2, static_cast<const float *>(scores), output, out_dtype, static_cast<hipStream_t>(stream))) return status;
    return check_launch(name);
}

namespace {

// Where the scratch of the MLP with a sparse map lies: the map, the activations, and the rows in front of layer 1, which the rows behind layer 2 replace.
struct MlpLayout {
    int64_t rows;
    int index_dtype;
    size_t ends_at, pad_begins_at, map_at, map_size, rows_at, row_scales_at, activations_at, activation_scales_at, size;
};

bool mlp_layout(MlpLayout &layout, int64_t tokens, int64_t slots, int64_t hidden, int64_t ffn, int64_t experts, int format, int out_dtype) {
    if (tokens <= 0 || slots <= 0 || hidden <= 0 || ffn <= 0 || experts <= 0 || experts > 1024 || !mx::valid_format(format) || !valid_dtype(out_dtype)) return false;
    if (tokens >= (int64_t(1) << 24) || slots > 1024 || tokens * slots >= (int64_t(1) << 31) - 128 * 1024 || hidden > (1 << 24) || ffn > (1 << 24)) return false;
    constexpr int64_t kBlock = 128;
    layout.rows = (tokens * slots + experts * kBlock) / kBlock * kBlock;
    layout.index_dtype = layout.rows < 32768 ? FM_INDEX_I16 : FM_INDEX_I32;
    const size_t index_size = layout.rows < 32768 ? 2 : 4;
    size_t at = 0;
    const auto take = [&](size_t bytes) {
        const size_t start = at;
        at += (bytes + 255) / 256 * 256;
        return start;
    };
    const int64_t padded = mx::padded_columns(hidden), ffn_padded = mx::padded_columns(ffn);
    take(tokens * slots * index_size);  // sparse_rows
    layout.ends_at = take(experts * index_size), layout.pad_begins_at = take(experts * index_size);
    layout.map_size = max(fm_sparse_map_workspace_size(tokens, slots, experts), fm_sparse_map_from_router_workspace_size(tokens, experts));
    layout.map_at = take(layout.map_size);
    layout.activations_at = take(layout.rows * mx::value_bytes(format, ffn_padded)), layout.activation_scales_at = take(layout.rows * mx::scale_bytes(ffn_padded));
    layout.rows_at = at, layout.row_scales_at = at + (layout.rows * mx::value_bytes(format, padded) + 255) / 256 * 256;
    const size_t before = layout.row_scales_at - at + layout.rows * mx::scale_bytes(padded), after = layout.rows * hidden * dtype_size(out_dtype);
    take(max(before, after));
    layout.size = at;
    return true;
}

}  // namespace

extern "C" size_t fm_mx_mlp_workspace_size(int64_t num_tokens, int64_t slots_per_token, int64_t hidden, int64_t ffn, int64_t num_experts, int format,
                                           int out_dtype) {
    MlpLayout layout;
    return mlp_layout(layout, num_tokens, slots_per_token, hidden, ffn, num_experts, format, out_dtype) ? layout.size : 0;
}

extern "C" int fm_mx_mlp_forward(const void *input, const void *input_scales, const void *top_experts, const void *scores, const void *weight_1,
                                 const void *weight_1_scales, const void *weight_2, const void *weight_2_scales, void *output, int64_t num_tokens,
                                 int64_t slots_per_token, int64_t hidden, int64_t ffn, int64_t num_experts, int64_t input_stride,
                                 int64_t input_scale_stride, int64_t weight_1_stride, int64_t weight_1_scale_stride, int64_t weight_2_stride,
                                 int64_t weight_2_scale_stride, int gated, int activation, int format, int out_dtype, const void *router_workspace,
                                 size_t router_workspace_size, int64_t shared_experts, void *workspace, size_t workspace_size, void *stream) {
    const char *name = "fm_mx_mlp_forward";
    FM_REQUIRE(mx::valid_format(format), "%s: bad format %d", name, format);
    FM_REQUIRE(valid_dtype(out_dtype), "%s: bad dtype %d", name, out_dtype);
    FM_REQUIRE(activation >= FM_ACT_GELU && activation <= FM_ACT_IDENTITY, "%s: bad activation %d", name, activation);
    MlpLayout layout;
    if (!mlp_layout(layout, num_tokens, slots_per_token, hidden, ffn, num_experts, format, out_dtype)) return fail(FM_ERR_UNSUPPORTED, "%s: bad sizes", name);
    FM_REQUIRE(top_experts && scores && output, "%s: null tensor", name);
    FM_REQUIRE(shared_experts >= 0 && (router_workspace == nullptr || shared_experts < slots_per_token), "%s: bad shared_experts", name);
    // All that the launches below check, before the first of them.
    const int64_t padded = mx::padded_columns(hidden);
    if (int status = check_tensor(name, "the input", input, input_scales, padded, input_stride, input_scale_stride, format)) return status;
    if (int status = check_tensor(name, "layer 1", weight_1, weight_1_scales, padded, weight_1_stride, weight_1_scale_stride, FM_MX_E2M1)) return status;
    if (int status = check_tensor(name, "layer 2", weight_2, weight_2_scales, mx::padded_columns(ffn), weight_2_stride, weight_2_scale_stride, FM_MX_E2M1))
        return status;
    FM_REQUIRE(workspace && reinterpret_cast<uintptr_t>(workspace) % 256 == 0 && workspace_size >= layout.size,
               "%s: workspace of %zu bytes (256-byte aligned) needed, got %zu", name, layout.size, workspace_size);
    char *scratch = static_cast<char *>(workspace);
    void *ends = scratch + layout.ends_at, *pad_begins = scratch + layout.pad_begins_at, *map_scratch = scratch + layout.map_at;
    void *rows = scratch + layout.rows_at, *row_scales = scratch + layout.row_scales_at;
    void *activations = scratch + layout.activations_at, *activation_scales = scratch + layout.activation_scales_at;
    const int64_t *experts = static_cast<const int64_t *>(top_experts);
    const int index = layout.index_dtype;
    int status = router_workspace != nullptr
                     ? fm_sparse_map_from_router(experts, router_workspace, router_workspace_size, num_tokens, num_experts, slots_per_token - shared_experts,
                                                 shared_experts, 128, index, scratch, ends, pad_begins, map_scratch, layout.map_size, stream)
                     : fm_sparse_map(experts, num_tokens, slots_per_token, num_experts, 128, index, scratch, ends, pad_begins, map_scratch, layout.map_size, stream);
    if (status < 0) return status;
    status = fm_mx_copy_dense_to_sparse(input, input_scales, scratch, rows, row_scales, num_tokens, hidden, slots_per_token, layout.rows, input_stride,
                                        input_scale_stride, format, index, stream);
    if (status < 0) return status;
    status = fm_mx_sparse_matmul_activation(rows, row_scales, weight_1, weight_1_scales, activations, activation_scales, ends, pad_begins, layout.rows, ffn, hidden,
                                            num_experts, mx::value_bytes(format, padded), mx::scale_bytes(padded), weight_1_stride, weight_1_scale_stride, gated,
                                            activation, format, index, stream);
    if (status < 0) return status;
    const int64_t ffn_padded = mx::padded_columns(ffn);
    // Rows in the output's type, as the operators one by one hand them on and as the sparse MLP in 16 bits has them: a rounding per slot more than without a map
    // (bf16: 2.5e-3 from 64 bits against 1.7e-3). In fp32 layer 2 and the combine take 900 us for 814 (8192 tokens, 8 experts, 4096, 14336), 217 for 124
    // (5001, 64, 2048, 1408).
    status = fm_mx_sparse_matmul(activations, activation_scales, weight_2, weight_2_scales, rows, ends, pad_begins, layout.rows, hidden, ffn, num_experts,
                                 mx::value_bytes(format, ffn_padded), mx::scale_bytes(ffn_padded), weight_2_stride, weight_2_scale_stride, hidden, format,
                                 out_dtype, index, stream);
    if (status < 0) return status;
    return fm_copy_sparse_to_dense(rows, scores, scratch, output, num_tokens, hidden, slots_per_token, layout.rows, out_dtype, FM_DTYPE_F32, index, stream);
}
