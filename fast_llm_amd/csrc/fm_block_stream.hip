// Products of a few rows per expert with expert weights of 8 bits and a scale per block of 128: the weights come from memory once and that is the
// bound.
//
// A wavefront has 32 weight rows of one expert and up to 32 rows of the activations at a time. kSplit wavefronts share the reduction, a stretch of it
// each, and add up in LDS; kAcross of them sit side by side. The reduction is in chunks of 128, a block of the format and a line of memory of each
// weight row. A load instruction takes eight whole lines, and the fragments, 16 bytes of each of 32 rows, are read from the wavefront's own part of
// LDS (XOR-swizzled; a wavefront's LDS operations are carried out in order, so no barrier). kDepth chunks are on their way at a time. Activations,
// which all workgroups of an expert read, come from L2 as fragments, and the scales as bytes, those of 32 neighbouring rows side by side.
//
// One token and two of 8 experts, 4096 -> 2 x 14336: 40 us, 5.8 TB/s of weights; 96 tokens with 8 of 128, 2048 -> 2 x 768: 66 us, 6.1 TB/s. As
// fragments straight from memory, 16 bytes of each of 32 lines at a time, the first took 60 and 14336 -> 4096 112 for 22.
//
// Any number of rows per expert is right (they are walked and the weights read again); the caller decides up to where this is the faster way.
#include <algorithm>

#include "fm_block_product.h"

namespace fm {

namespace block {

namespace {

constexpr uint32_t kOutOfRange = 0x80000000u;
constexpr int kDepth = 2, kStreaming = 2;  // nt: weights are read once

__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer_of(const uint8_t *base, int64_t bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<char *>(uniform_pointer(reinterpret_cast<const char *>(base))), 0,
                                             __builtin_amdgcn_readfirstlane(static_cast<int>(max(bytes, static_cast<int64_t>(0)))), kBufferResourceFlags);
}

// Four neighbouring columns of a row, `left` of which exist.
template <typename Result>
__device__ __forceinline__ void store_four(Result *target, const f32x4_t &value, int vectors, int left) {
    if (vectors && left >= 4) {
        struct alignas(4 * sizeof(Result)) Four {
            Result v[4];
        } four;
#pragma unroll
        for (int c = 0; c < 4; ++c) four.v[c] = from_float<Result>(value[c]);
        *reinterpret_cast<Four *>(target) = four;
    } else {
#pragma unroll
        for (int c = 0; c < 4; ++c)
            if (c < left) target[c] = from_float<Result>(value[c]);
    }
}

template <bool kWide, int kSplit, int kAcross>
__global__ __launch_bounds__(kSplit * kAcross * 64) void stream_kernel(ProductArgs args) {
    constexpr int kWaves = kSplit * kAcross;
    __shared__ f32x4_t shared[kWaves * 4 * 64];  // the wavefronts' chunks of weights; then [wavefront][quad of a lane's sums][lane]
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), row_of_lane = lane & 31, half = lane >> 5;
    const int split = wave % kSplit, across = wave / kSplit, expert = blockIdx.y;
    int64_t first_row = 0, end = args.rows;
    if (args.expert_ends != nullptr) {
        first_row = expert > 0 ? max(load_index(args.expert_ends, args.index_dtype, expert - 1), static_cast<int64_t>(0)) : 0;
        end = min(load_index(args.expert_pad_begins, args.index_dtype, expert), args.rows);
    }
    if (end <= first_row) return;  // most experts of a map for a few tokens
    const int rows = static_cast<int>(end - first_row);

    const int columns = static_cast<int>(args.columns), chunks = static_cast<int>(args.inner / kBlock);
    const int own_chunks = (chunks + kSplit - 1) / kSplit, first_chunk = split * own_chunks, end_chunk = min(first_chunk + own_chunks, chunks);
    // Rows of an operand from `row` on, `valid` of which exist (maybe none, or less): what is behind them is zero.
    const auto values_of = [&](const uint8_t *values, int64_t row, int valid, int64_t stride) { return buffer_of(values + row * stride, valid > 0 ? (valid - 1) * stride + args.inner : 0); };
    const auto scales_of = [&](const uint8_t *scales, int64_t row, int valid, int64_t stride) { return buffer_of(scales + row, valid > 0 ? (chunks - 1) * stride + valid : 0); };
    const int first = (blockIdx.x * kAcross + across) * 32, weights_valid = min(columns - first, 32);
    const int64_t weight_row = static_cast<int64_t>(expert) * columns + first;
    const __amdgpu_buffer_rsrc_t weight = values_of(args.weight, weight_row, weights_valid, args.weight_stride);
    const __amdgpu_buffer_rsrc_t weight_scale_buffer = scales_of(args.weight_scales, weight_row, weights_valid, args.weight_scale_stride);
    // A load takes eight whole lines.
    const uint32_t weight_offset = (lane >> 3) * static_cast<uint32_t>(args.weight_stride) + (lane & 7) * 16, eight_rows = 8 * static_cast<uint32_t>(args.weight_stride);
    const uint32_t x_offset = row_of_lane * static_cast<uint32_t>(args.x_stride) + half * 16;
    const uint32_t weight_scale_stride = static_cast<uint32_t>(args.weight_scale_stride), x_scale_stride = static_cast<uint32_t>(args.x_scale_stride);

    u32x4_t weights[kDepth][4], x[kDepth][4];
    uint32_t weight_scales[kDepth], x_scales[kDepth];
    const auto fetch_weights = [&](int slot, int c) {
        const uint32_t at = c < end_chunk ? weight_offset + c * kBlock : kOutOfRange;
#pragma unroll
        for (int j = 0; j < 4; ++j) weights[slot][j] = __builtin_bit_cast(u32x4_t, __builtin_amdgcn_raw_buffer_load_b128(weight, static_cast<int>(at + j * eight_rows), 0, kStreaming));
        weight_scales[slot] = static_cast<uint8_t>(
            __builtin_amdgcn_raw_buffer_load_b8(weight_scale_buffer, static_cast<int>(c < end_chunk ? c * weight_scale_stride + row_of_lane : kOutOfRange), 0, 0));
    };
#pragma unroll
    for (int d = 0; d < kDepth; ++d) fetch_weights(d, first_chunk + d);
    FM_LDS(char) *const chunk_lds = (FM_LDS(char) *)shared + wave * (32 * kBlock);
    for (int base = 0; base < rows; base += 32) {
        const __amdgpu_buffer_rsrc_t x_buffer = values_of(args.x, first_row + base, min(rows - base, 32), args.x_stride);
        const __amdgpu_buffer_rsrc_t x_scale_buffer = scales_of(args.x_scales, first_row + base, min(rows - base, 32), args.x_scale_stride);
        const auto fetch_x = [&](int slot, int c) {
            const uint32_t at = c < end_chunk ? x_offset + c * kBlock : kOutOfRange;
#pragma unroll
            for (int j = 0; j < 4; ++j) x[slot][j] = __builtin_bit_cast(u32x4_t, __builtin_amdgcn_raw_buffer_load_b128(x_buffer, static_cast<int>(at + j * 32), 0, 0));
            x_scales[slot] = static_cast<uint8_t>(
                __builtin_amdgcn_raw_buffer_load_b8(x_scale_buffer, static_cast<int>(c < end_chunk ? c * x_scale_stride + row_of_lane : kOutOfRange), 0, 0));
        };
#pragma unroll
        for (int d = 0; d < kDepth; ++d) {
            if (base > 0) fetch_weights(d, first_chunk + d);
            fetch_x(d, first_chunk + d);
        }
        f32x16_t sums = {};
#pragma unroll 1
        for (int c = first_chunk; c < end_chunk; c += kDepth) {
#pragma unroll
            for (int d = 0; d < kDepth; ++d) {
                u32x4_t fragments[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int row = 8 * j + (lane >> 3);
                    *(FM_LDS(u32x4_t) *)(chunk_lds + row * kBlock + (((lane & 7) ^ ((row >> 1) & 7)) << 4)) = weights[d][j];
                }
                // The lanes read what others wrote: the hardware keeps a wavefront's LDS operations in order, and this the compiler.
                asm volatile("" ::: "memory");
#pragma unroll
                for (int j = 0; j < 4; ++j) fragments[j] = *(FM_LDS(u32x4_t) *)(chunk_lds + row_of_lane * kBlock + (((2 * j + half) ^ ((row_of_lane >> 1) & 7)) << 4));
                asm volatile("" ::: "memory");
                if constexpr (kWide) {
                    const uint32_t weight_scale = wide_scale(weight_scales[d]), x_scale = wide_scale(x_scales[d]);
#pragma unroll
                    for (int q = 0; q < 8; ++q) {
                        const auto wide = [&](const u32x4_t &part, uint32_t scale) {
                            const uint32_t low = part[q % 2 * 2], high = part[q % 2 * 2 + 1];
                            return u32x4_t{widened<0>(low, scale), widened<1>(low, scale), widened<0>(high, scale), widened<1>(high, scale)};
                        };
                        sums = multiply_wide(wide(fragments[q / 2], weight_scale), wide(x[d][q / 2], x_scale), sums);
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const u32x4_t a[2] = {fragments[2 * i], fragments[2 * i + 1]}, b[2] = {x[d][2 * i], x[d][2 * i + 1]};
                        sums = multiply(a, b, weight_scales[d], x_scales[d], sums);
                    }
                }
                fetch_weights(d, c + kDepth + d);
                fetch_x(d, c + kDepth + d);
            }
        }

        __syncthreads();
#pragma unroll
        for (int q = 0; q < 4; ++q) shared[(wave * 4 + q) * 64 + lane] = f32x4_t{sums[4 * q], sums[4 * q + 1], sums[4 * q + 2], sums[4 * q + 3]};
        __syncthreads();
        // A thread finishes the four columns 4 quad .. of a row.
        for (int item = threadIdx.x; item < kAcross * 256; item += kWaves * 64) {
            const int place = item / 256, in_chunk = item / 8 % 32, quad = item % 8, row = base + in_chunk, column = (blockIdx.x * kAcross + place) * 32 + quad * 4;
            const int at = (place * kSplit * 4 + quad / 2) * 64 + quad % 2 * 32 + in_chunk;
            f32x4_t sum = shared[at];
#pragma unroll
            for (int w = 1; w < kSplit; ++w) sum += shared[w * 256 + at];
            if (row >= rows) continue;
            FM_DISPATCH_DTYPE(args.out_dtype, Result, store_four(static_cast<Result *>(args.out) + (first_row + row) * args.out_stride + column, sum, args.out_vectors, columns - column));
        }
        __syncthreads();
    }
}

template <bool kWide>
int launch(const ProductArgs &args, hipStream_t stream) {
    const auto grid = [&](int across) { return dim3(static_cast<uint32_t>((args.columns + across * 32 - 1) / (across * 32)), static_cast<uint32_t>(args.experts)); };
    switch (stream_split(args)) {
        case 1: stream_kernel<kWide, 1, 4><<<grid(4), 256, 0, stream>>>(args); break;
        case 4: stream_kernel<kWide, 4, 1><<<grid(1), 256, 0, stream>>>(args); break;
        default: stream_kernel<kWide, 8, 1><<<grid(1), 512, 0, stream>>>(args); break;
    }
    return FM_OK;
}

}  // namespace

// As few wavefronts share a reduction as give the device twelve wavefronts per CU.
int stream_split(const ProductArgs &args) {
    // A map's rows have up to 128 of padding per expert; of its last ones it is not known whether there is anything in them.
    const int64_t busy = args.expert_ends == nullptr ? 1 : std::min(std::max(rows_of_any_routing(args) - 128 * args.experts, int64_t(2)), args.experts);
    const int64_t sets = (args.columns + 31) / 32 * busy, chunks = args.inner / kBlock;
    constexpr int kWanted = 12 * 256;
    if (sets >= kWanted || chunks < 4) return 1;
    return sets * 4 >= kWanted || chunks < 8 ? 4 : 8;
}

bool stream_product_takes(const ProductArgs &args) {
    // 32 rows, and the scales of all chunks, are addressed in 31 bits from the first. Workgroups in y: experts.
    constexpr int64_t kMost = (int64_t(1) << 31) - 4096;
    return std::max(args.x_stride, args.weight_stride) * 32 < kMost && std::max(args.x_scale_stride, args.weight_scale_stride) * (args.inner / kBlock + 1) < kMost &&
           (args.columns + 31) / 32 < (int64_t(1) << 22);
}

int stream_product(const ProductArgs &args, hipStream_t stream) { return args.out_dtype == FM_DTYPE_F32 || args.exact ? launch<true>(args, stream) : launch<false>(args, stream); }

}  // namespace block

}  // namespace fm
