// Products of a few microscaled rows per expert with e2m1 expert weights: the weights come from memory once and that is the bound.
//
// A workgroup has kSets x 32 weight rows of one expert (with the gated activation half of them gates and half the ups that go with them) and up
// to kGroups x 32 rows of the activations at a time; its wavefronts take every kWaves-th chunk of 256 along K and add up in LDS. A weight row is half a
// byte per element, so a chunk is one line of 128 bytes of each row: a load instruction takes eight whole lines, and the fragments, 16 bytes of
// each of 32 rows, are read from the wavefront's own part of LDS (XOR-swizzled; a wavefront's LDS operations are carried out in order, so
// no barrier). Activations, which all workgroups of an expert read, come from L2 as fragments; scales as 8 bytes per row and chunk.
//
// The rows are those of a sparse map, or are found without one: with few tokens a workgroup scans `top_experts` for its expert.
// Any number of rows per expert is right (they are walked and the weights read again); the caller decides up to where this is the faster way.
#include "fm_activation_math.h"
#include "fm_mx.h"
#include "fm_mx_product.h"

namespace fm {

namespace mx {

constexpr int kChunk = 256;
constexpr uint32_t kOutOfRange = 0xffffffffu;

enum Source { kByEntries, kByMap };

__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer_of(const uint8_t *pointer, int64_t bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<char *>(uniform_pointer(reinterpret_cast<const char *>(pointer))), 0,
                                             static_cast<int>(max(min(bytes, static_cast<int64_t>(0xfffffff0)), static_cast<int64_t>(0))), kBufferResourceFlags);
}
constexpr int kStreaming = 2;  // nt: weights are read once
template <int kCachePolicy = 0>
__device__ __forceinline__ u32x4_t load_16(__amdgpu_buffer_rsrc_t buffer, uint32_t offset) {
    return __builtin_bit_cast(u32x4_t, __builtin_amdgcn_raw_buffer_load_b128(buffer, static_cast<int>(offset), 0, kCachePolicy));
}
__device__ __forceinline__ u32x2_t load_8(__amdgpu_buffer_rsrc_t buffer, uint32_t offset) {
    return __builtin_bit_cast(u32x2_t, __builtin_amdgcn_raw_buffer_load_b64(buffer, static_cast<int>(offset), 0, 0));
}

// The scales of a lane's row in a chunk: word i / 2, byte 2 (i % 2), is that of its block 2 i + l / 32.
__device__ __forceinline__ void align_scales(u32x2_t &scales, bool second, int half) {
    scales[0] >>= 8 * half;
    scales[1] = second ? scales[1] >> (8 * half) : 0u;
}

template <int kFormat, bool kGated, int kSets, int kGroups, int kWaves, Source kSource, typename Result>
__global__ __launch_bounds__(kWaves * 64) void stream_kernel(ProductArgs args) {
    constexpr bool kQuantized = std::is_same<Result, uint8_t>::value;
    constexpr int kParts = kFormat == FM_MX_E4M3 ? 2 : 1;  // 16-byte parts of a lane's activations per MFMA
    constexpr int kOutputSets = kGated ? kSets / 2 : kSets, kSetBytes = 32 * 128;
    extern __shared__ __attribute__((aligned(16))) char shared[];  // the wavefronts' chunks and then sums; the list of entries
    int *list = reinterpret_cast<int *>(shared + kWaves * kSets * kSetBytes);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5;

    // The expert and its rows.
    int expert, rows;
    int64_t first_row = 0;
    if constexpr (kSource == kByEntries) {
        __shared__ int count;
        expert = args.by_entry ? static_cast<int>(args.top_experts[blockIdx.y]) : blockIdx.y;
        if (expert < 0 || expert >= args.experts) return;
        if (threadIdx.x == 0) count = 0;
        __syncthreads();
        bool seen = false;
        for (int i = threadIdx.x; i < args.entries; i += kWaves * 64) {
            if (args.top_experts[i] != expert) continue;
            // With a workgroup row per entry, the first entry of an expert does the work.
            if (args.by_entry && i < static_cast<int>(blockIdx.y)) seen = true;
            list[atomicAdd(&count, 1)] = i;  // in any order: every entry's sums are its own
        }
        if (__syncthreads_or(seen)) return;
        rows = __builtin_amdgcn_readfirstlane(count);
    } else {
        expert = blockIdx.y;
        first_row = expert > 0 ? load_index(args.expert_ends, args.index_dtype, expert - 1) : 0;
        const int64_t end = min(load_index(args.expert_pad_begins, args.index_dtype, expert), args.rows);
        rows = first_row >= 0 && end > first_row ? static_cast<int>(end - first_row) : 0;
    }
    if (rows == 0) return;

    const int first = blockIdx.x * kOutputSets * 32;  // of the result's columns
    const int columns = static_cast<int>(args.columns), inner = static_cast<int>(args.inner);
    const int64_t weight_stride = args.weight_stride, scale_stride = args.weight_scale_stride;
    __amdgpu_buffer_rsrc_t weight[kSets], weight_scales[kSets];
#pragma unroll
    for (int s = 0; s < kSets; ++s) {
        const int column = first + s % kOutputSets * 32, valid = min(columns - column, 32);
        const int64_t row = static_cast<int64_t>(expert) * columns * (kGated ? 2 : 1) + column + (kGated && s >= kOutputSets ? columns : 0);
        weight[s] = buffer_of(args.weight + row * weight_stride, valid * weight_stride);
        weight_scales[s] = buffer_of(args.weight_scales + row * scale_stride, valid * scale_stride);
    }
    uint32_t load_offset[4];  // of rows 8 i + l / 8; past the last row: out of the buffer
#pragma unroll
    for (int i = 0; i < 4; ++i) load_offset[i] = static_cast<uint32_t>((8 * i + (lane >> 3)) * weight_stride + (lane & 7) * 16);
    const uint32_t weight_scale_offset = static_cast<uint32_t>((lane & 31) * scale_stride);
    FM_LDS(char) *const chunk_lds = (FM_LDS(char) *)shared + wave * kSets * kSetBytes;
    const int chunks = (inner + kChunk - 1) / kChunk;
    const auto activate = [&](float value) {
        float result;
        FM_DISPATCH_ACTIVATION(args.activation, kActivation, result = activation_forward<kActivation>(value));
        return result;
    };

    for (int base = 0; base < rows; base += 32 * kGroups) {
        __amdgpu_buffer_rsrc_t x, x_scales;
        uint32_t x_offset[kGroups], x_scale_offset[kGroups];
        if constexpr (kSource == kByEntries) {
            x = buffer_of(args.x, args.x_rows * args.x_stride);
            x_scales = buffer_of(args.x_scales, args.x_rows * args.x_scale_stride);
        } else {
            x = buffer_of(args.x + (first_row + base) * args.x_stride, min(rows - base, 32 * kGroups) * args.x_stride);
            x_scales = buffer_of(args.x_scales + (first_row + base) * args.x_scale_stride, min(rows - base, 32 * kGroups) * args.x_scale_stride);
        }
#pragma unroll
        for (int g = 0; g < kGroups; ++g) {
            const int within = g * 32 + (lane & 31), row = base + within;
            int64_t at = within;
            if constexpr (kSource == kByEntries) at = row < rows ? list[row] / args.entries_per_row : 0;
            x_offset[g] = row < rows ? static_cast<uint32_t>(at * args.x_stride) : kOutOfRange;
            x_scale_offset[g] = row < rows ? static_cast<uint32_t>(at * args.x_scale_stride) : kOutOfRange;
        }
        f32x16_t sums[kSets][kGroups];
#pragma unroll
        for (int s = 0; s < kSets; ++s)
#pragma unroll
            for (int g = 0; g < kGroups; ++g) sums[s][g] = f32x16_t{};

        struct Chunk {
            u32x4_t weight[kSets][4];
            u32x2_t weight_scales[kSets], x_scales[kGroups];
            u32x4_t x[kGroups][4][kParts];
        };
        const auto fetch = [&](int c, Chunk &chunk) {
            const int k0 = c * kChunk;
            const bool exists = k0 + (lane & 7) * 32 < inner;  // inner is a multiple of 128
#pragma unroll
            for (int s = 0; s < kSets; ++s) {
#pragma unroll
                for (int i = 0; i < 4; ++i) chunk.weight[s][i] = load_16<kStreaming>(weight[s], exists ? load_offset[i] + k0 / 2 : kOutOfRange);
                chunk.weight_scales[s] = load_8(weight_scales[s], k0 < inner ? weight_scale_offset + k0 / 32 : kOutOfRange);
            }
#pragma unroll
            for (int g = 0; g < kGroups; ++g) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const bool there = k0 + i * 64 < inner && x_offset[g] != kOutOfRange;
#pragma unroll
                    for (int p = 0; p < kParts; ++p) {
                        // In e4m3 the halves of two blocks, in e2m1 one block.
                        const int at = kFormat == FM_MX_E4M3 ? k0 + i * 64 + p * 32 + half * 16 : (k0 + i * 64) / 2 + half * 16;
                        chunk.x[g][i][p] = load_16(x, there ? x_offset[g] + at : kOutOfRange);
                    }
                }
                chunk.x_scales[g] = load_8(x_scales, k0 < inner && x_scale_offset[g] != kOutOfRange ? x_scale_offset[g] + k0 / 32 : kOutOfRange);
            }
        };
        const auto multiply_chunk = [&](int c, Chunk &chunk) {
#pragma unroll
            for (int s = 0; s < kSets; ++s)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int row = 8 * i + (lane >> 3);
                    *(FM_LDS(u32x4_t) *)(chunk_lds + s * kSetBytes + row * 128 + (((lane & 7) ^ ((row >> 1) & 7)) << 4)) = chunk.weight[s][i];
                }
            const bool second = c * kChunk + 128 < inner;
#pragma unroll
            for (int s = 0; s < kSets; ++s) align_scales(chunk.weight_scales[s], second, half);
#pragma unroll
            for (int g = 0; g < kGroups; ++g) align_scales(chunk.x_scales[g], second, half);
            // The lanes read what others wrote: the hardware keeps a wavefront's LDS operations in order, and this the compiler.
            asm volatile("" ::: "memory");
            const auto step = [&](auto constant) {
                constexpr int i = decltype(constant)::value;
#pragma unroll
                for (int s = 0; s < kSets; ++s) {
                    const int row = lane & 31;
                    const u32x4_t fragment = *(FM_LDS(u32x4_t) *)(chunk_lds + s * kSetBytes + row * 128 + (((2 * i + half) ^ ((row >> 1) & 7)) << 4));
#pragma unroll
                    for (int g = 0; g < kGroups; ++g)
                        sums[s][g] = multiply<kFormat, i % 2 * 2, i % 2 * 2>(fragment, chunk.x[g][i], chunk.weight_scales[s][i / 2], chunk.x_scales[g][i / 2], sums[s][g]);
                }
            };
            step(std::integral_constant<int, 0>{});
            step(std::integral_constant<int, 1>{});
            step(std::integral_constant<int, 2>{});
            step(std::integral_constant<int, 3>{});
            asm volatile("" ::: "memory");  // and the next chunk's writes stay behind these reads
        };
        Chunk even, odd;
        fetch(wave, even);
        for (int c = wave; c < chunks; c += 2 * kWaves) {
            fetch(c + kWaves, odd);  // past the end: zeros, and no memory is touched
            multiply_chunk(c, even);
            if (c + kWaves >= chunks) break;
            fetch(c + 2 * kWaves, even);
            multiply_chunk(c + kWaves, odd);
        }
        __syncthreads();

        // Group by group, [wavefront][set][quad of a lane's sums][lane]. Thread t then finishes four columns 4 (t % 8) of row t / 8.
        f32x4_t *partial = reinterpret_cast<f32x4_t *>(shared);
#pragma unroll
        for (int g = 0; g < kGroups; ++g) {
#pragma unroll
            for (int s = 0; s < kSets; ++s)
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    partial[((wave * kSets + s) * 4 + q) * 64 + lane] = f32x4_t{sums[s][g][4 * q], sums[s][g][4 * q + 1], sums[s][g][4 * q + 2], sums[s][g][4 * q + 3]};
            __syncthreads();
            for (int item = threadIdx.x; item < kOutputSets * 256; item += kWaves * 64) {
                const int set = item / 256, token = item / 8 % 32, quad = item % 8, row = base + g * 32 + token;
                const auto total = [&](int s) {
                    const int at = (s * 4 + quad / 2) * 64 + quad % 2 * 32 + token;
                    f32x4_t sum = partial[at];
#pragma unroll
                    for (int w = 1; w < kWaves; ++w) sum += partial[w * kSets * 256 + at];
                    return sum;
                };
                f32x4_t value = total(set);
                const int column = first + set * 32 + quad * 4;
                const int64_t out_row = row >= rows ? 0 : kSource == kByEntries ? list[row] : first_row + row;
                if constexpr (kQuantized) {
                    // From the fp32 sums: one rounding, to the elements' type.
                    f32x4_t up = {1.f, 1.f, 1.f, 1.f};
                    if constexpr (kGated) up = total(set + kOutputSets);
                    uint32_t largest = 0;
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        value[c] = activate(value[c]);
                        if constexpr (kGated) value[c] *= up[c];
                        largest = max(largest, magnitude_bits(value[c]));
                    }
                    const uint32_t byte = scale_byte(kFormat, max_of_neighbours<8>(largest));
                    if (row >= rows || column >= args.out_columns) continue;
                    const uint32_t packed = pack_four(kFormat, value[0], value[1], value[2], value[3], inverse_scale(byte));
                    uint8_t *target = static_cast<uint8_t *>(args.out) + out_row * args.out_stride;
                    if (kFormat == FM_MX_E4M3) *reinterpret_cast<uint32_t *>(target + column) = packed;
                    else *reinterpret_cast<uint16_t *>(target + column / 2) = static_cast<uint16_t>(packed);
                    if (quad == 0) args.out_scales[out_row * args.out_scale_stride + column / 32] = static_cast<uint8_t>(byte);
                } else {
                    if (row >= rows) continue;
                    Result *target = static_cast<Result *>(args.out) + out_row * args.out_stride + column;
                    if (args.out_vectors && column + 3 < columns) {
                        struct alignas(4 * sizeof(Result)) Four {
                            Result v[4];
                        } four;
#pragma unroll
                        for (int c = 0; c < 4; ++c) four.v[c] = from_float<Result>(value[c]);
                        *reinterpret_cast<Four *>(target) = four;
                    } else {
#pragma unroll
                        for (int c = 0; c < 4; ++c)
                            if (column + c < columns) target[c] = from_float<Result>(value[c]);
                    }
                }
            }
            __syncthreads();
        }
    }
}

// out[t, :] = sum over the slots j of scores[t, j] * sums[t slots + j, :], in the order of the slots. Entries of no expert add nothing: of
// theirs nothing was written.
template <typename T>
__global__ __launch_bounds__(256) void combine_kernel(const float *sums, const int64_t *top_experts, const float *scores, T *out, int slots, int experts,
                                                      int hidden, int stride) {
    const int64_t token = blockIdx.y;
    const int column = (blockIdx.x * 256 + threadIdx.x) * 4;
    if (column >= hidden) return;
    f32x4_t total = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
    for (int j = 0; j < slots; ++j) {
        const int64_t expert = top_experts[token * slots + j];
        const f32x4_t value = *reinterpret_cast<const f32x4_t *>(sums + (token * slots + j) * stride + column);
        const float score = scores[token * slots + j];
        if (expert >= 0 && expert < experts) total += score * value;
    }
    T *target = out + token * hidden + column;
#pragma unroll
    for (int c = 0; c < 4; ++c)
        if (column + c < hidden) target[c] = from_float<T>(total[c]);
}

template <int kFormat, bool kGated, int kSets, int kGroups, int kWaves, Source kSource, typename Result>
static int launch_stream(const ProductArgs &args, int workgroup_rows, hipStream_t stream) {
    constexpr int kOutputs = (kGated ? kSets / 2 : kSets) * 32;
    const auto kernel = stream_kernel<kFormat, kGated, kSets, kGroups, kWaves, kSource, Result>;
    const int lds = kWaves * kSets * 4096 + (kSource == kByEntries ? (args.entries + 3) / 4 * 16 : 0);
    static std::atomic<uint64_t> configured{0};
    if (lds > 65536)
        if (int status = allow_lds(reinterpret_cast<const void *>(kernel), kWaves * kSets * 4096 + kMaxEntries * 4, configured)) return status;
    kernel<<<dim3(static_cast<uint32_t>((args.out_columns + kOutputs - 1) / kOutputs), workgroup_rows), kWaves * 64, lds, stream>>>(args);
    return FM_OK;
}

template <bool kGated, int kSets, Source kSource, typename Result>
static int launch_format(const ProductArgs &args, int workgroup_rows, hipStream_t stream) {
    return args.format == FM_MX_E4M3 ? launch_stream<FM_MX_E4M3, kGated, kSets, 1, 4, kSource, Result>(args, workgroup_rows, stream)
                                     : launch_stream<FM_MX_E2M1, kGated, kSets, 1, 4, kSource, Result>(args, workgroup_rows, stream);
}

int stream_product(const ProductArgs &args, int out_dtype, hipStream_t stream) {
    const int experts = static_cast<int>(args.experts);
    if (args.out_scales != nullptr)
        return args.gated ? launch_format<true, 2, kByMap, uint8_t>(args, experts, stream) : launch_format<false, 1, kByMap, uint8_t>(args, experts, stream);
    switch (out_dtype) {
        case FM_DTYPE_F32: return launch_format<false, 1, kByMap, float>(args, experts, stream);
        case FM_DTYPE_BF16: return launch_format<false, 1, kByMap, bf16_t>(args, experts, stream);
        default: return launch_format<false, 1, kByMap, f16_t>(args, experts, stream);
    }
}

int few_tokens(const ProductArgs &layer_1, const ProductArgs &layer_2, const float *scores, void *out, int out_dtype, hipStream_t stream) {
    const int workgroup_rows = layer_1.by_entry ? layer_1.entries : static_cast<int>(layer_1.experts);
    int status = layer_1.gated ? launch_format<true, 2, kByEntries, uint8_t>(layer_1, workgroup_rows, stream)
                               : launch_format<false, 1, kByEntries, uint8_t>(layer_1, workgroup_rows, stream);
    if (status == FM_OK) status = launch_format<false, 1, kByEntries, float>(layer_2, workgroup_rows, stream);
    if (status != FM_OK) return status;
    const int slots = layer_1.entries_per_row, tokens = layer_1.entries / slots, hidden = static_cast<int>(layer_2.columns);
    FM_DISPATCH_DTYPE(out_dtype, T, {
        combine_kernel<T><<<dim3((hidden + 1023) / 1024, tokens), 256, 0, stream>>>(
            static_cast<const float *>(layer_2.out), layer_1.top_experts, scores, static_cast<T *>(out), slots, static_cast<int>(layer_1.experts), hidden,
            static_cast<int>(layer_2.out_stride));
    });
    return FM_OK;
}

}  // namespace mx

}  // namespace fm
