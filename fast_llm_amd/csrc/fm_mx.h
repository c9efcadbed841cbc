// Microscaled values: blocks of 32 neighbours along a row share a power of two, 2^(byte - 127), and are kept in e4m3 (8 bits) or
// e2m1 (4 bits, two to a byte, the even column in the low half). Rows are stored padded to whole groups of 128 columns: zeros, with
// scale byte 0. What the kernels that write, read and multiply them have in common.
//
// Of a block with the largest magnitude m the scale is 2^(floor(log2 m) - 8) for e4m3, whose largest value is 1.75 * 2^8, or
// 2^(floor(log2 m) - 2) for e2m1 (1.5 * 2^2), at least 2^-127; its elements are value / scale rounded to nearest even and saturated. A block
// with an infinity or NaN has scale byte 255, which makes all of it NaN, and zeros for elements.
#pragma once

#include "fm_gemm_common.h"

namespace fm {

namespace mx {

typedef __attribute__((__vector_size__(2 * sizeof(uint32_t)))) uint32_t u32x2_t;
typedef __attribute__((__vector_size__(4 * sizeof(uint32_t)))) uint32_t u32x4_t;
typedef __attribute__((__vector_size__(8 * sizeof(int)))) int i32x8_t;
typedef __attribute__((__vector_size__(4 * sizeof(float)))) float f32x4_t;
typedef __attribute__((__vector_size__(16 * sizeof(float)))) float f32x16_t;

constexpr int kBlock = 32, kPadding = 128;

inline bool valid_format(int format) { return format == FM_MX_E4M3 || format == FM_MX_E2M1; }
constexpr int64_t padded_columns(int64_t columns) { return (columns + kPadding - 1) / kPadding * kPadding; }
// Of a row's values and scales, for padded columns.
__host__ __device__ constexpr int64_t value_bytes(int format, int64_t columns) { return format == FM_MX_E4M3 ? columns : columns / 2; }
__host__ __device__ constexpr int64_t scale_bytes(int64_t columns) { return columns / kBlock; }

// ---- to microscaled values -------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t magnitude_bits(float value) { return __builtin_bit_cast(uint32_t, value) & 0x7fffffffu; }

// The maximum over the kLanes neighbouring lanes (4 or 8, aligned), in all of them. All lanes of the wavefront take part.
template <int kLanes>
__device__ __forceinline__ uint32_t max_of_neighbours(uint32_t value) {
    static_assert(kLanes == 4 || kLanes == 8, "lanes");
    const auto with = [&](auto control) {
        value = max(value, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(value), decltype(control)::value, 0xf, 0xf, true)));
    };
    with(std::integral_constant<int, 0xb1>{});  // lanes 1 0 3 2 of every four
    with(std::integral_constant<int, 0x4e>{});  // 2 3 0 1
    if constexpr (kLanes == 8) with(std::integral_constant<int, 0x141>{});  // the eight mirrored
    return value;
}

// The scale byte of a block, from the bits of its largest magnitude. floor(log2) of a normal value is its exponent field - 127; subnormal
// ones end at the lowest scale in any case; infinities and NaN have the largest bits of all.
__device__ __forceinline__ uint32_t scale_byte(int format, uint32_t largest) {
    const int exponent = static_cast<int>(largest >> 23), top = format == FM_MX_E4M3 ? 8 : 2;
    return exponent == 255 ? 255u : static_cast<uint32_t>(max(exponent - top, 0));
}
// What elements are multiplied by: 1 / scale, an exact product but for what vanishes next to the block's largest value.
__device__ __forceinline__ float inverse_scale(uint32_t byte) {
    return byte == 255u ? 0.f : __builtin_bit_cast(float, (254u - byte) << 23);
}

// Four scaled elements of a block, as they are kept: 32 bits of e4m3 or 16 of e2m1. (The conversions round to nearest even; the one to
// e4m3 makes a NaN of what is over 464, the one to e2m1 saturates.) Of a block that is not finite, `inverse` 0: zeros.
__device__ __forceinline__ uint32_t pack_four(int format, float a, float b, float c, float d, float inverse) {
    const uint32_t finite = inverse == 0.f ? 0u : ~0u;
    if (format == FM_MX_E4M3) {
        const auto saturated = [&](float value) { return __builtin_amdgcn_fmed3f(value * inverse, -448.f, 448.f); };
        const int low = __builtin_amdgcn_cvt_pk_fp8_f32(saturated(a), saturated(b), 0, false);
        return static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(saturated(c), saturated(d), low, true)) & finite;
    }
    const uint32_t low = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, a * inverse, b * inverse, 1.f, 0);
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(low, c * inverse, d * inverse, 1.f, 1) & 0xffffu & finite;
}

// Where eight columns from `column` on are read in a row of any length from 8: the row's last eight in place of what goes past its end.
__device__ __forceinline__ int window(int column, int columns) { return min(column, columns - 8); }
// Of such a window the values from `by` on (below 8) to the front, with zeros behind them.
__device__ __forceinline__ void shift_down(float (&values)[8], int by) {
#pragma unroll
    for (int step = 4; step > 0; step /= 2)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float next = i + step < 8 ? values[(i + step) % 8] : 0.f;
            values[i] = by & step ? next : values[i];
        }
}
constexpr int kNowhere = 0x7fffff00;  // past the end of any row

// Eight neighbours per lane, four neighbouring lanes a block: writes the elements (8 or 4 bytes) and, from the block's first lane, the scale.
// `column`: of the lane's first value, a multiple of 8. All lanes of the wavefront take part; `store`: whether this one's block exists.
__device__ __forceinline__ void store_eight(int format, const float (&values)[8], uint8_t *row_values, uint8_t *row_scales, int64_t column, bool store) {
    uint32_t largest = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) largest = max(largest, magnitude_bits(values[i]));
    const uint32_t byte = scale_byte(format, max_of_neighbours<4>(largest));
    const float inverse = inverse_scale(byte);
    if (!store) return;
    const uint32_t low = pack_four(format, values[0], values[1], values[2], values[3], inverse);
    const uint32_t high = pack_four(format, values[4], values[5], values[6], values[7], inverse);
    if (format == FM_MX_E4M3) *reinterpret_cast<u32x2_t *>(row_values + column) = u32x2_t{low, high};
    else *reinterpret_cast<uint32_t *>(row_values + column / 2) = low | high << 16;
    if (column % kBlock == 0) row_scales[column / kBlock] = static_cast<uint8_t>(byte);
}

// One value per lane, 32 neighbouring lanes a block: for rows of any length and alignment.
__device__ __forceinline__ void store_one(int format, float value, uint8_t *row_values, uint8_t *row_scales, int64_t column, bool store) {
    uint32_t largest = magnitude_bits(value);
#pragma unroll
    for (int offset = 16; offset > 0; offset >>= 1) largest = max(largest, static_cast<uint32_t>(__shfl_xor(static_cast<int>(largest), offset, 64)));
    const uint32_t byte = scale_byte(format, largest);
    const float inverse = inverse_scale(byte);
    const float neighbour = __shfl_xor(value, 1, 64);
    if (!store) return;
    if (format == FM_MX_E4M3) row_values[column] = static_cast<uint8_t>(pack_four(format, value, 0.f, 0.f, 0.f, inverse));
    else if (column % 2 == 0) row_values[column / 2] = static_cast<uint8_t>(pack_four(format, value, neighbour, 0.f, 0.f, inverse));
    if (column % kBlock == 0) row_scales[column / kBlock] = static_cast<uint8_t>(byte);
}

// ---- products --------------------------------------------------------------------------------------------
// D[m][n] += sum over 64 k of A[m][k] 2^sa B[n][k] 2^sb, A in e2m1, B in kFormat: lane l holds row l % 32 of both. Of A (and of B in e2m1) it
// holds the block l / 32: 16 bytes; of B in e4m3 the bytes 16 (l / 32) .. + 15 of the first block and then of the second. Its scales are those of its
// row's block l / 32, byte kStep of the two words. Of D it holds column n = l % 32, rows m = 8 (i / 4) + 4 (l / 32) + i % 4.
template <int kFormat, int kStepA, int kStepB>
__device__ __forceinline__ f32x16_t multiply(u32x4_t a, const u32x4_t (&b)[kFormat == FM_MX_E4M3 ? 2 : 1], uint32_t scales_a, uint32_t scales_b, f32x16_t c) {
    const i32x8_t wide_a = {static_cast<int>(a[0]), static_cast<int>(a[1]), static_cast<int>(a[2]), static_cast<int>(a[3])};
    i32x8_t wide_b;
    if constexpr (kFormat == FM_MX_E4M3)
        wide_b = i32x8_t{static_cast<int>(b[0][0]), static_cast<int>(b[0][1]), static_cast<int>(b[0][2]), static_cast<int>(b[0][3]),
                         static_cast<int>(b[1][0]), static_cast<int>(b[1][1]), static_cast<int>(b[1][2]), static_cast<int>(b[1][3])};
    else
        wide_b = i32x8_t{static_cast<int>(b[0][0]), static_cast<int>(b[0][1]), static_cast<int>(b[0][2]), static_cast<int>(b[0][3])};
    return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(wide_a, wide_b, c, 4, kFormat == FM_MX_E4M3 ? 0 : 4, kStepA, static_cast<int>(scales_a),
                                                           kStepB, static_cast<int>(scales_b));
}

}  // namespace mx

}  // namespace fm
