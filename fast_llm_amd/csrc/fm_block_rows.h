// Pieces of the kernels that quantise: values in registers -> elements and scales in memory, along the rows and along the columns.
#pragma once

#include "fm_block.h"

namespace fm {

namespace block {

// The maximum over 2, 4, 8 (DPP), 16 or 32 neighbouring lanes, in all of them. All lanes of the wavefront take part.
template <int kLanes>
__device__ __forceinline__ uint32_t max_of_lanes(uint32_t value) {
    static_assert(kLanes == 8 || kLanes == 32, "lanes");
    const auto with = [&](auto control) {
        value = max(value, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(value), decltype(control)::value, 0xf, 0xf, true)));
    };
    with(std::integral_constant<int, 0xb1>{});   // lanes 1 0 3 2 of every four
    with(std::integral_constant<int, 0x4e>{});   // 2 3 0 1
    with(std::integral_constant<int, 0x141>{});  // the eight mirrored
    if constexpr (kLanes == 32) {
        with(std::integral_constant<int, 0x140>{});  // the sixteen mirrored
        const auto swapped = __builtin_amdgcn_permlane16_swap(value, value, false, false);
        value = max(static_cast<uint32_t>(swapped[0]), static_cast<uint32_t>(swapped[1]));
    }
    return value;
}

// ---- rows alone: a wavefront has eight rows x 128 columns, a lane sixteen neighbours of one row ----------
constexpr int kRowThreads = 256, kRowsAtOnce = 8, kRowSteps = kBlock / (kRowThreads / 64) / kRowsAtOnce;

// Writes the elements and the scale of a row's block; `exists`: the row does. All lanes of the wavefront take part.
__device__ __forceinline__ void store_row(const float (&values)[16], uint8_t *elements, uint8_t *scale, bool exists) {
    uint32_t largest = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i) largest = max(largest, magnitude_bits(values[i]));
    const uint32_t byte = scale_byte(max_of_lanes<8>(largest));
    const float inverse = inverse_scale(byte);
    u32x4_t packed;
#pragma unroll
    for (int q = 0; q < 4; ++q) packed[q] = pack_four(values[4 * q], values[4 * q + 1], values[4 * q + 2], values[4 * q + 3], inverse);
    if (!exists) return;
    *reinterpret_cast<u32x4_t *>(elements) = packed;
    if (threadIdx.x % 8 == 0) *scale = static_cast<uint8_t>(byte);
}

// ---- rows and columns: a workgroup has 128 x 128, a lane eight neighbouring rows x four neighbouring columns ------
constexpr int kSquareThreads = 512, kLaneRows = 8, kLaneColumns = 4;

struct Square {
    uint32_t largest[kSquareThreads / 64][kBlock];  // of each wavefront's rows, by column
    uint32_t transposed[kBlock][kBlock / 4];        // the elements, column by column; see `transposed_at`
    uint8_t row_scales[kBlock], column_scales[kBlock];
};

// Where the eight rows of row group `group` of column 4 cg + c lie, in words: column by column in the order c, cg, units of 8 bytes swapped so that the writes
// of a wavefront (32 cg, two groups) meet every bank twice and the reads, whole columns, once.
__device__ __forceinline__ int transposed_at(int cg, int c, int group) { return (c * 32 + cg) * 32 + ((group ^ (cg >> 1 & 7) << 1) << 1); }

// The elements along the rows. `scales`: of this column of blocks, at the square's first row; `rows`: that exist.
__device__ __forceinline__ void store_rows(const float (&values)[kLaneRows][kLaneColumns], Square &shared, uint8_t *elements, int64_t stride, int rows) {
    const int cg = threadIdx.x & 31, group = threadIdx.x >> 5;
    uint32_t bytes[2] = {0, 0};
#pragma unroll
    for (int r = 0; r < kLaneRows; ++r) {
        uint32_t largest = 0;
#pragma unroll
        for (int c = 0; c < kLaneColumns; ++c) largest = max(largest, magnitude_bits(values[r][c]));
        const uint32_t byte = scale_byte(max_of_lanes<32>(largest));
        bytes[r / 4] |= byte << (r % 4 * 8);
        const uint32_t packed = pack_four(values[r][0], values[r][1], values[r][2], values[r][3], inverse_scale(byte));
        const int row = group * kLaneRows + r;
        if (row < rows) *reinterpret_cast<uint32_t *>(elements + row * stride + cg * kLaneColumns) = packed;
    }
    if (cg == 0) *reinterpret_cast<u32x2_t *>(shared.row_scales + group * kLaneRows) = u32x2_t{bytes[0], bytes[1]};
}

// The scales that `store_rows` found, after a barrier.
__device__ __forceinline__ void store_row_scales(const Square &shared, uint8_t *scales, int rows) {
    if (static_cast<int>(threadIdx.x) < rows) scales[threadIdx.x] = shared.row_scales[threadIdx.x];
}

// The elements along the columns, in two parts with a barrier before, between and after them: the maxima and then the elements to LDS, ...
__device__ __forceinline__ void column_maxima(const float (&values)[kLaneRows][kLaneColumns], Square &shared) {
    const int cg = threadIdx.x & 31, wave = threadIdx.x >> 6;
    u32x4_t largest = {};
#pragma unroll
    for (int c = 0; c < kLaneColumns; ++c) {
#pragma unroll
        for (int r = 0; r < kLaneRows; ++r) largest[c] = max(largest[c], magnitude_bits(values[r][c]));
        const auto swapped = __builtin_amdgcn_permlane32_swap(largest[c], largest[c], false, false);
        largest[c] = max(static_cast<uint32_t>(swapped[0]), static_cast<uint32_t>(swapped[1]));
    }
    if ((threadIdx.x & 32) == 0) *reinterpret_cast<u32x4_t *>(&shared.largest[wave][cg * kLaneColumns]) = largest;
}
__device__ __forceinline__ void stage_columns(const float (&values)[kLaneRows][kLaneColumns], Square &shared) {
    const int cg = threadIdx.x & 31, group = threadIdx.x >> 5;
    u32x4_t largest = {};
#pragma unroll
    for (int w = 0; w < kSquareThreads / 64; ++w) {
        const u32x4_t of_wave = *reinterpret_cast<const u32x4_t *>(&shared.largest[w][cg * kLaneColumns]);
#pragma unroll
        for (int c = 0; c < kLaneColumns; ++c) largest[c] = max(largest[c], of_wave[c]);
    }
    uint32_t bytes = 0;
    uint32_t *words = &shared.transposed[0][0];
#pragma unroll
    for (int c = 0; c < kLaneColumns; ++c) {
        const uint32_t byte = scale_byte(largest[c]);
        bytes |= byte << (c * 8);
        const float inverse = inverse_scale(byte);
        const uint32_t low = pack_four(values[0][c], values[1][c], values[2][c], values[3][c], inverse);
        const uint32_t high = pack_four(values[4][c], values[5][c], values[6][c], values[7][c], inverse);
        *reinterpret_cast<u32x2_t *>(words + transposed_at(cg, c, group)) = u32x2_t{low, high};
    }
    if (group == 0) *reinterpret_cast<uint32_t *>(shared.column_scales + cg * kLaneColumns) = bytes;
}
// ... and from there to memory: whole lines. `elements`: of the square's first column, from its first row on; `columns`: that exist.
__device__ __forceinline__ void store_columns(const Square &shared, uint8_t *elements, int64_t stride, uint8_t *scales, int columns) {
    const uint32_t *words = &shared.transposed[0][0];
#pragma unroll
    for (int pass = 0; pass < 2; ++pass) {
        const int at = pass * 64 + static_cast<int>(threadIdx.x) / 8, part = threadIdx.x % 8, cg = at % 32, column = cg * kLaneColumns + at / 32;
        const u32x4_t vector = *reinterpret_cast<const u32x4_t *>(words + transposed_at(cg, at / 32, 2 * part));
        if (column < columns) *reinterpret_cast<u32x4_t *>(elements + column * stride + part * 16) = vector;
    }
    if (static_cast<int>(threadIdx.x) < columns) scales[threadIdx.x] = shared.column_scales[threadIdx.x];
}

}  // namespace block

}  // namespace fm
