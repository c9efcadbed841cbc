// Values of 8 bits with a scale for each block of 128: 128 neighbours along a row share a power of two, 2^(byte - 127), and are kept in e4m3. What
// the kernels that write, read and multiply them have in common.
//
// Rows are stored padded with zeros to whole blocks. The scales of all rows' first blocks come first, then those of their second blocks: a tile of
// the products then has its scales of a slice in one piece. The scale is the smallest power of two (from 2^-127 on) that leaves the block's largest
// magnitude at 448 or below, so nothing saturates; elements are value / scale rounded to nearest even. A power of two costs no accuracy next to a
// scale of 24 bits (but below 2^-14 of the largest value, where elements become subnormal), the matrix instructions apply it by themselves, and a
// block that is cut along the other axis keeps its elements: a change of scale is exact. A block with an infinity or NaN has scale byte 255, which
// makes all of it NaN, and zeros for elements.
#pragma once

#include "fm_mx.h"

namespace fm {

namespace block {

using mx::f32x16_t;
using mx::f32x4_t;
using mx::magnitude_bits;
using mx::u32x2_t;
using mx::u32x4_t;

constexpr int kBlock = 128, kScaleRows = 16;  // rows of scales are padded to a multiple of that many
constexpr int64_t padded_columns(int64_t columns) { return (columns + kBlock - 1) / kBlock * kBlock; }
constexpr int64_t padded_rows(int64_t rows) { return (rows + kScaleRows - 1) / kScaleRows * kScaleRows; }
// Values of a row are addressed in 32 bits, as bytes and as floats.
constexpr int64_t kMaxColumns = int64_t(1) << 28;

// The scale byte of a block, from the bits of its largest magnitude m 2^k, 1 <= m < 2: 448 = 1.75 * 2^8, so the exponent is k - 8 up to m = 1.75 and
// one more above, which the addition carries into. Subnormal magnitudes end at the lowest scale in any case.
__device__ __forceinline__ uint32_t scale_byte(uint32_t largest) {
    const int exponent = static_cast<int>((largest + 0x1fffffu) >> 23) - 8;
    return largest >= 0x7f800000u ? 255u : static_cast<uint32_t>(max(exponent, 0));
}
// What elements are multiplied by: 1 / scale, an exact product but for what vanishes next to the block's largest value.
__device__ __forceinline__ float inverse_scale(uint32_t byte) { return byte == 255u ? 0.f : __builtin_bit_cast(float, (254u - byte) << 23); }
__device__ __forceinline__ float scale_value(uint32_t byte) {
    // 2^-127 is a subnormal number; 255 stands for NaN.
    return byte == 255u ? __builtin_nanf("") : byte == 0u ? __builtin_bit_cast(float, 0x00400000u) : __builtin_bit_cast(float, byte << 23);
}

// Four elements of a block that is finite (nothing is over 448), or of any: of one that is not, `inverse` 0, zeros.
__device__ __forceinline__ uint32_t pack_finite(float a, float b, float c, float d, float inverse) {
    const int low = __builtin_amdgcn_cvt_pk_fp8_f32(a * inverse, b * inverse, 0, false);
    return static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(c * inverse, d * inverse, low, true));
}
__device__ __forceinline__ uint32_t pack_four(float a, float b, float c, float d, float inverse) { return pack_finite(a, b, c, d, inverse) & (inverse == 0.f ? 0u : ~0u); }
__device__ __forceinline__ void unpack_four(uint32_t word, float scale, float (&values)[4]) {
    values[0] = __builtin_amdgcn_cvt_f32_fp8(static_cast<int>(word), 0) * scale, values[1] = __builtin_amdgcn_cvt_f32_fp8(static_cast<int>(word), 1) * scale;
    values[2] = __builtin_amdgcn_cvt_f32_fp8(static_cast<int>(word), 2) * scale, values[3] = __builtin_amdgcn_cvt_f32_fp8(static_cast<int>(word), 3) * scale;
}

// The rows of a sparse layout that tokens have, by blocks of 128 rows: experts begin at multiples of 128.
struct RowMap {
    const void *expert_ends, *expert_pad_begins;  // null: all rows count
    int num_experts, index_dtype;
};

// What the entry points ask of a tensor in blocks (`columns` padded), and of a sparse map, which may be null.
int check_tensor(const char *name, const char *what, const void *values, const void *scales, int64_t rows, int64_t columns, int64_t value_stride,
                 int64_t scale_stride);
int check_map(const char *name, RowMap &map, const void *expert_ends, const void *expert_pad_begins, int64_t num_experts, int index_dtype);

// How many of the rows from `row0` (a multiple of 128) to row0 + 127 count, up to `rows` in all: they are the first ones. All lanes of the wavefront
// take part.
__device__ __forceinline__ int rows_in_block(const RowMap &map, int64_t row0, int64_t rows) {
    int64_t end = rows;
    if (map.expert_ends != nullptr) {
        const int lane = threadIdx.x & 63;
        int expert = 0;  // experts that end at or before the block: they come in order
        for (int base = 0; base < map.num_experts; base += 64) {
            const bool before = base + lane < map.num_experts && load_index(map.expert_ends, map.index_dtype, base + lane) <= row0;
            const int count = __popcll(__ballot(before));
            expert += count;
            if (count < 64) break;
        }
        end = expert < map.num_experts ? min(load_index(map.expert_pad_begins, map.index_dtype, expert), rows) : 0;
    }
    return __builtin_amdgcn_readfirstlane(static_cast<int>(max(min(end - row0, static_cast<int64_t>(kBlock)), static_cast<int64_t>(0))));
}

// kCount neighbours of a row as they lie in memory, at any alignment: the hardware takes vectors at any address.
template <typename T, int kCount>
struct __attribute__((packed, aligned(sizeof(T)))) Raw {
    T v[kCount];
};
// ... from `pointer` on, of which `left` exist; the others are zeros.
template <typename T, int kCount>
__device__ __forceinline__ Raw<T, kCount> load_part(const T *pointer, int left) {
    Raw<T, kCount> raw;
#pragma unroll
    for (int i = 0; i < kCount; ++i) raw.v[i] = i < left ? pointer[i] : from_float<T>(0.f);
    return raw;
}

// Rows `first_row` + kRowStep r, r < kRows, of a block of 128 x 128 that begins at `block`: kCount neighbours of each from `column` on. Those from
// `count` on are zeros, and so is what is behind the `columns` that there are. `exist`: rows that may be read. Where the columns are whole, no load
// is behind a branch, so that all are on their way at once.
template <int kRows, int kRowStep, typename T, int kCount>
__device__ __forceinline__ void load_block(const T *block, uint32_t stride, int first_row, int column, int exist, int count, int columns, Raw<T, kCount> (&raw)[kRows]) {
    if (columns == kBlock) {
#pragma unroll
        for (int r = 0; r < kRows; ++r)
            raw[r] = *reinterpret_cast<const Raw<T, kCount> *>(block + (static_cast<uint32_t>(min(first_row + r * kRowStep, exist - 1)) * stride + column));
        if (count < kBlock) {
#pragma unroll
            for (int r = 0; r < kRows; ++r)
#pragma unroll
                for (int i = 0; i < kCount; ++i) raw[r].v[i] = first_row + r * kRowStep < count ? raw[r].v[i] : from_float<T>(0.f);
        }
    } else {
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
            const int row = first_row + r * kRowStep;
            raw[r] = load_part<T, kCount>(block + (static_cast<uint32_t>(row) * stride + column), row < count ? columns - column : 0);
        }
    }
}

}  // namespace block

}  // namespace fm
