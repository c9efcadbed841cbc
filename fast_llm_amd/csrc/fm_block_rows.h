// Pieces of the kernels that quantise: values in registers -> elements and scales in memory, along the rows and along the columns.
#pragma once

#include "fm_block.h"

namespace fm {

namespace block {

constexpr int kSwapPairs = 0xb1, kSwapFours = 0x4e, kMirrorEight = 0x141, kRotateEight = 0x128;  // lanes 1 0 3 2, 2 3 0 1 of every four; 7 .. 0 of eight; 8 .. 15, 0 .. 7
template <int kControl>
__device__ __forceinline__ uint32_t from_lanes(uint32_t value) {
    return static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(value), kControl, 0xf, 0xf, true));
}

// The maximum over eight neighbouring lanes, in all of them. All lanes of the wavefront take part.
__device__ __forceinline__ uint32_t max_of_eight(uint32_t value) {
    value = max(value, from_lanes<kSwapPairs>(value));
    value = max(value, from_lanes<kSwapFours>(value));
    return max(value, from_lanes<kMirrorEight>(value));
}

// ---- rows alone: a wavefront has eight rows x 128 columns, a lane sixteen neighbours of one row ----------
constexpr int kRowThreads = 256, kRowsAtOnce = 8, kRowSteps = kBlock / (kRowThreads / 64) / kRowsAtOnce;

// Writes the elements and the scale of a row's block; `exists`: the row does. All lanes of the wavefront take part.
__device__ __forceinline__ void store_row(const float (&values)[16], uint8_t *elements, uint8_t *scale, bool exists) {
    uint32_t largest = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i) largest = max(largest, magnitude_bits(values[i]));
    const uint32_t byte = scale_byte(max_of_eight(largest));
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
// Bytes from a square's first row on are counted in 32 bits: rows of less than 2^24 elements of four bytes.
constexpr int64_t kMaxSquareStride = int64_t(1) << 24;

struct Square {
    uint32_t largest[kSquareThreads / 64][kBlock];  // of each wavefront's rows, by column
    uint32_t transposed[kBlock][kBlock / 4];        // the elements, column by column; see `transposed_at`
    float row_inverse[kBlock], column_inverse[kBlock];
    uint8_t row_scales[kBlock];
};

// Where the eight rows of row group `group` of column 4 cg + c lie, in words: column by column in the order c, cg, units of 8 bytes swapped so that
// the writes of a wavefront (32 cg, two groups) meet every bank twice and the reads, whole columns, once.
__device__ __forceinline__ int transposed_at(int cg, int c, int group) { return (c * 32 + cg) * 32 + ((group ^ (cg >> 1 & 7) << 1) << 1); }

// The largest magnitude over 32 lanes of each of eight values: of value 4 (l / 16 % 2) + 2 (l / 8 % 2) + l / 4 % 2 in lane l. Every step but the last
// two hands over half of what is left and keeps the other.
__device__ __forceinline__ uint32_t maxima_of_rows(const uint32_t (&rows)[kLaneRows], int lane) {
    uint32_t four[4], two[2];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const auto swapped = __builtin_amdgcn_permlane16_swap(rows[i], rows[i + 4], false, false);
        four[i] = max(static_cast<uint32_t>(swapped[0]), static_cast<uint32_t>(swapped[1]));
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) two[i] = max(lane & 8 ? four[i + 2] : four[i], from_lanes<kRotateEight>(lane & 8 ? four[i] : four[i + 2]));
    uint32_t one = max(lane & 4 ? two[1] : two[0], from_lanes<kMirrorEight>(lane & 4 ? two[0] : two[1]));
    one = max(one, from_lanes<kSwapPairs>(one));
    return max(one, from_lanes<kSwapFours>(one));
}

// The elements of a square's values, along the columns and (kRows) along the rows. `elements` and `scales`: of the square's first row and column in
// either form, `rows` and `columns` that exist. Ends with reads of LDS that its next call comes after. All threads take part.
template <bool kRows>
__device__ __forceinline__ void store_square(const float (&values)[kLaneRows][kLaneColumns], Square &shared, uint8_t *elements, uint32_t stride, uint8_t *scales, int rows,
                                             uint8_t *t_elements, int64_t t_stride, uint8_t *t_scales, int columns) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, cg = threadIdx.x & 31, group = threadIdx.x >> 5, thread = static_cast<int>(threadIdx.x);
    u32x4_t of_columns = {};
    uint32_t of_rows[kLaneRows];
#pragma unroll
    for (int r = 0; r < kLaneRows; ++r) {
        of_rows[r] = 0;
#pragma unroll
        for (int c = 0; c < kLaneColumns; ++c) {
            const uint32_t bits = magnitude_bits(values[r][c]);
            of_rows[r] = max(of_rows[r], bits), of_columns[c] = max(of_columns[c], bits);
        }
    }
#pragma unroll
    for (int c = 0; c < kLaneColumns; ++c) {
        const auto swapped = __builtin_amdgcn_permlane32_swap(of_columns[c], of_columns[c], false, false);
        of_columns[c] = max(static_cast<uint32_t>(swapped[0]), static_cast<uint32_t>(swapped[1]));
    }
    __builtin_amdgcn_sched_barrier(0);
    if (lane < 32) *reinterpret_cast<u32x4_t *>(&shared.largest[wave][cg * kLaneColumns]) = of_columns;
    if constexpr (kRows) {
        const uint32_t byte = scale_byte(maxima_of_rows(of_rows, lane));
        const int row = group * kLaneRows + (lane >> 4 & 1) * 4 + (lane >> 3 & 1) * 2 + (lane >> 2 & 1);
        if ((lane & 3) == 0) shared.row_inverse[row] = inverse_scale(byte), shared.row_scales[row] = static_cast<uint8_t>(byte);
        // The lanes read what others of the wavefront wrote: its LDS operations are carried out in order, and this keeps the compiler to it.
        asm volatile("" ::: "memory");
        float inverse[kLaneRows];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const f32x4_t four = *reinterpret_cast<const f32x4_t *>(&shared.row_inverse[group * kLaneRows + half * 4]);
#pragma unroll
            for (int i = 0; i < 4; ++i) inverse[half * 4 + i] = four[i];
        }
        const auto store = [&](auto pack) {
#pragma unroll
            for (int r = 0; r < kLaneRows; ++r) {
                const uint32_t in_square = group * kLaneRows + r, packed = pack(values[r][0], values[r][1], values[r][2], values[r][3], inverse[r]);
                if (static_cast<int>(in_square) < rows) *reinterpret_cast<uint32_t *>(elements + (in_square * stride + cg * kLaneColumns)) = packed;
            }
        };
        if (__any(byte == 255u)) store(pack_four);
        else store(pack_finite);
    }
    __syncthreads();
    if (thread < kBlock) {
        uint32_t largest = 0;
#pragma unroll
        for (int w = 0; w < kSquareThreads / 64; ++w) largest = max(largest, shared.largest[w][thread]);
        const uint32_t byte = scale_byte(largest);
        shared.column_inverse[thread] = inverse_scale(byte);
        if (thread < columns) t_scales[thread] = static_cast<uint8_t>(byte);
    } else if (kRows && thread < 2 * kBlock) {
        if (thread - kBlock < rows) scales[thread - kBlock] = shared.row_scales[thread - kBlock];
    }
    __syncthreads();
    const f32x4_t inverse = *reinterpret_cast<const f32x4_t *>(&shared.column_inverse[cg * kLaneColumns]);
    uint32_t *words = &shared.transposed[0][0];
    const auto stage = [&](auto pack) {
#pragma unroll
        for (int c = 0; c < kLaneColumns; ++c) {
            const uint32_t low = pack(values[0][c], values[1][c], values[2][c], values[3][c], inverse[c]);
            const uint32_t high = pack(values[4][c], values[5][c], values[6][c], values[7][c], inverse[c]);
            *reinterpret_cast<u32x2_t *>(words + transposed_at(cg, c, group)) = u32x2_t{low, high};
        }
    };
    if (__any(inverse[0] == 0.f || inverse[1] == 0.f || inverse[2] == 0.f || inverse[3] == 0.f)) stage(pack_four);
    else stage(pack_finite);
    __syncthreads();
    // Whole lines.
#pragma unroll
    for (int pass = 0; pass < 2; ++pass) {
        const int at = pass * 64 + thread / 8, part = thread % 8, column = at % 32 * kLaneColumns + at / 32;
        const u32x4_t vector = *reinterpret_cast<const u32x4_t *>(words + transposed_at(at % 32, at / 32, 2 * part));
        if (column < columns) *reinterpret_cast<u32x4_t *>(t_elements + column * t_stride + part * 16) = vector;
    }
}

}  // namespace block

}  // namespace fm
