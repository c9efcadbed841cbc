// Arguments of the products of operands of 8 bits with a scale per block of 128.
#pragma once

#include "fm_block.h"

namespace fm {

namespace block {

// Strides in bytes, those of `out` in elements.
struct ProductArgs {
    const uint8_t *x, *x_scales;            // rows of the result
    const uint8_t *weight, *weight_scales;  // its columns (by rows: of each expert)
    void *out;
    int64_t x_stride, x_scale_stride, weight_stride, weight_scale_stride, out_stride;
    int64_t rows;     // of x (by rows: of the sparse layout)
    int64_t columns;  // of the result
    int64_t inner;    // padded: a multiple of 128
    int64_t experts;
    int out_dtype, accumulate;
    int out_vectors;  // rows of `out` are aligned to 16 bytes
    int by_inner;     // an expert has a range of the reduction and `rows` rows of the result; otherwise a range of rows
    const void *expert_ends, *expert_pad_begins;
    int index_dtype;
};

// Many rows per expert (fm_block_tiles.hip).
int tile_product(const ProductArgs &args, hipStream_t stream);
bool tile_product_takes(const ProductArgs &args);

}  // namespace block

}  // namespace fm
