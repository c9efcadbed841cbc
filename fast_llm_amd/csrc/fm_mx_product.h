// Arguments of the products of microscaled rows with e2m1 expert weights.
#pragma once

#include "fm_mx.h"

namespace fm {

namespace mx {

// Strides in bytes (those of `out` in elements where it is not microscaled).
struct ProductArgs {
    const uint8_t *x, *x_scales;            // [x_rows]
    const uint8_t *weight, *weight_scales;  // [experts * columns (* 2: gates and ups, expert by expert)]
    void *out;
    uint8_t *out_scales;  // null: `out` is not microscaled
    int64_t x_rows, x_stride, x_scale_stride, weight_stride, weight_scale_stride, out_stride, out_scale_stride;
    int64_t rows;         // of the sparse layout
    int64_t columns;      // of the result
    int64_t out_columns;  // that are written: with the padding where the result is microscaled
    int64_t inner;        // padded: a multiple of 128
    int64_t experts;
    int format;  // of x, and of a microscaled result
    int gated, activation;
    int out_dtype;    // where it is not microscaled
    int out_vectors;  // rows of `out` are aligned to 16 bytes
    // Rows by a sparse map ...
    const void *expert_ends, *expert_pad_begins;
    int index_dtype;
    // ... or by their entry: entry i is row i / entries_per_row of x and has row i of the result.
    const int64_t *top_experts;
    int entries, entries_per_row;
    int by_entry;  // a workgroup row per entry instead of one per expert
};

constexpr int kMaxEntries = 4096;  // the list in LDS, and the scan of every workgroup

// Which kernel a product by a map runs on (fm_mx_product.hip).
bool runs_on_tiles(const ProductArgs &args);
// How many wavefronts share a reduction in the kernel for few rows (fm_mx_stream.hip): 1, 4 or 8.
int stream_split(const ProductArgs &args);

// Many rows per expert (fm_mx_tiles.hip).
bool tile_product_takes(const ProductArgs &args);
int tile_product(const ProductArgs &args, hipStream_t stream);
// Few rows per expert (fm_mx_stream.hip).
int stream_product(const ProductArgs &args, hipStream_t stream);
// Both layers and the combine without a sparse map; layer_2.out is fp32 scratch.
int few_tokens(const ProductArgs &layer_1, const ProductArgs &layer_2, const float *scores, void *out, int out_dtype, hipStream_t stream);

}  // namespace mx

}  // namespace fm
