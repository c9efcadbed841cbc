// Products of a few microscaled rows per expert with e2m1 expert weights: the weights come from memory once and that is the bound.
//
// A wavefront has 32 weight rows of one expert (with the gated activation 32 gates and the ups that go with them) and up to 32 rows of the activations at a
// time. kSplit wavefronts share the reduction, a stretch of it each, and add up in LDS; kAcross of them sit side by side. The reduction is in chunks
// of 256: half a byte per element, so a chunk is one line of 128 bytes of each weight row. A load instruction takes eight whole lines, and the
// fragments, 16 bytes of each of 32 rows, are read from the wavefront's own part of LDS (XOR-swizzled; a wavefront's LDS operations are carried
// out in order, so no barrier). Scales go the same way, those of four chunks at a time. A chunk of weights is on its way while the one before it is
// multiplied, the first one while the rows are being found: what is in flight and how soon it starts is the whole speed. Activations, which all
// workgroups of an expert read, come from L2 as fragments.
//
// Measured, the weights' bytes over the kernel's time: 4096 -> 2 x 14336, one row for each of 2 experts, 125 MB in 25.5 us (4.9 TB/s) as the gated
// layer 1 and in 26.9 us as a product by itself; 14336 -> 4096 62 MB in 15.6 us (4.0 TB/s); a probe that does nothing but read such rows takes
// 18 and 11.5 us (6.5, 5.4 TB/s).
//
// The rows are those of a sparse map, or are found without one: with few tokens a workgroup scans `top_experts` for its expert.
// Any number of rows per expert is right (they are walked and the weights read again); the caller decides up to where this is the faster way.
#include "fm_activation_math.h"
#include "fm_mx.h"
#include "fm_mx_product.h"

namespace fm {

namespace mx {

constexpr int kChunk = 256, kScaleChunks = 4;

template <int kFirst, int kLast, typename F>
__device__ __forceinline__ void for_each(const F &f) {
    if constexpr (kFirst < kLast) {
        f(std::integral_constant<int, kFirst>{});
        for_each<kFirst + 1, kLast>(f);
    }
}
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

// The scales of a row in a chunk, for the lanes of a group: byte 0 (and 2, where a row has two groups) of a word is that of the group's block.
__device__ __forceinline__ void align_scales(u32x2_t &scales, bool second, int group) {
    scales[0] >>= 8 * group;
    scales[1] = second ? scales[1] >> (8 * group) : 0u;
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

template <int kFormat, bool kGated, bool kQuantized, int kSplit, int kAcross, Source kSource>
__global__ __launch_bounds__(kSplit * kAcross * 64, kGated ? 3 : 4) void stream_kernel(ProductArgs args) {
    constexpr int kParts = kFormat == FM_MX_E4M3 ? 2 : 1;  // 16-byte parts of a lane's activations per MFMA
    constexpr int kSets = kGated ? 2 : 1, kSetBytes = 32 * 128, kWaves = kSplit * kAcross;
    constexpr int kScaleBytes = 32 * 8 * kScaleChunks;  // of 32 rows
    constexpr int kLds = kWaves * ((kSets + 1) * kScaleBytes + kSets * kSetBytes);
    extern __shared__ __attribute__((aligned(16))) char shared[];  // the wavefronts' chunks and then sums; the list of entries
    int *list = reinterpret_cast<int *>(shared + kLds);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), token_of_lane = lane & 31, group = lane >> 5;
    const int split = wave % kSplit, across = wave / kSplit;

    const int expert = kSource == kByEntries && args.by_entry ? static_cast<int>(args.top_experts[blockIdx.y]) : blockIdx.y;
    if (expert < 0 || expert >= args.experts) return;
    int rows;
    int64_t first_row = 0;
    if constexpr (kSource == kByMap) {
        first_row = expert > 0 ? load_index(args.expert_ends, args.index_dtype, expert - 1) : 0;
        const int64_t end = min(load_index(args.expert_pad_begins, args.index_dtype, expert), args.rows);
        rows = first_row >= 0 && end > first_row ? static_cast<int>(end - first_row) : 0;
        if (rows == 0) return;  // most experts of a map for a few tokens
    }

    // ---- weights -----------------------------------------------------------------------------------------------------
    const int first = (blockIdx.x * kAcross + across) * 32;  // of the result's columns
    const int columns = static_cast<int>(args.columns), inner = static_cast<int>(args.inner), chunks = (inner + kChunk - 1) / kChunk;
    const int64_t weight_stride = args.weight_stride, scale_stride = args.weight_scale_stride;
    // To the end of the last row and no further: loads of 16 bytes reach behind it.
    const auto scale_bytes_of = [&](int64_t count, int64_t stride) { return count > 0 ? (count - 1) * stride + inner / kBlock : 0; };
    __amdgpu_buffer_rsrc_t weight[kSets], weight_scale_buffers[kSets];
#pragma unroll
    for (int s = 0; s < kSets; ++s) {
        const int valid = min(columns - first, 32);  // may be negative: nothing is read
        const int64_t row = static_cast<int64_t>(expert) * columns * kSets + first + s * columns;
        weight[s] = buffer_of(args.weight + row * weight_stride, valid * weight_stride);
        weight_scale_buffers[s] = buffer_of(args.weight_scales + row * scale_stride, scale_bytes_of(valid, scale_stride));
    }
    const uint32_t weight_offset = static_cast<uint32_t>((lane >> 3) * weight_stride + (lane & 7) * 16);
    const uint32_t eight_rows = static_cast<uint32_t>(8 * weight_stride);
    // Past the end: zeros, and no memory is touched. (`inner` is a multiple of 128.)
    const int own_chunks = (chunks + kSplit - 1) / kSplit, first_chunk = split * own_chunks, end_chunk = min(first_chunk + own_chunks, chunks);
    u32x4_t raw[kSets][4], raw_scales[kSets];
    const auto fetch_weights = [&](int c) {
        const bool exists = c < end_chunk && c * kChunk + (lane & 7) * 32 < inner;
#pragma unroll
        for (int s = 0; s < kSets; ++s)
#pragma unroll
            for (int i = 0; i < 4; ++i) raw[s][i] = load_16<kStreaming>(weight[s], exists ? weight_offset + i * eight_rows + c * (kChunk / 2) : kOutOfRange);
    };
    // Scales of kScaleChunks chunks from `c` on: 16 bytes of row l / 2. (8 bytes a chunk come from as many lines of memory as the chunk itself.)
    const auto fetch_scales = [&](__amdgpu_buffer_rsrc_t buffer, uint32_t row_offset, int c) {
        const int byte = c * (kChunk / 32) + (lane & 1) * 16;
        return load_16(buffer, c < end_chunk && row_offset != kOutOfRange && byte < inner / 32 ? row_offset + byte : kOutOfRange);
    };
    const auto fetch_weight_scales = [&](int c) {
#pragma unroll
        for (int s = 0; s < kSets; ++s) raw_scales[s] = fetch_scales(weight_scale_buffers[s], static_cast<uint32_t>((lane >> 1) * scale_stride), c);
    };
    fetch_weight_scales(first_chunk);
    fetch_weights(first_chunk);

    // ---- rows, while the first weights are on their way ----------------------------------------------------------------
    if constexpr (kSource == kByEntries) {
        __shared__ int count;
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
        if (rows == 0) return;
    }

    FM_LDS(char) *const chunk_lds = (FM_LDS(char) *)shared + wave * kSets * kSetBytes;
    FM_LDS(char) *const scale_lds = (FM_LDS(char) *)shared + kWaves * kSets * kSetBytes + wave * (kSets + 1) * kScaleBytes;
    const auto activate = [&](float value) {
        float result;
        FM_DISPATCH_ACTIVATION(args.activation, kActivation, result = activation_forward<kActivation>(value));
        return result;
    };
    for (int base = 0; base < rows; base += 32) {
        if (base > 0) fetch_weight_scales(first_chunk), fetch_weights(first_chunk);
        __amdgpu_buffer_rsrc_t x, x_scale_buffer;
        if constexpr (kSource == kByEntries) {
            x = buffer_of(args.x, args.x_rows * args.x_stride);
            x_scale_buffer = buffer_of(args.x_scales, scale_bytes_of(args.x_rows, args.x_scale_stride));
        } else {
            x = buffer_of(args.x + (first_row + base) * args.x_stride, min(rows - base, 32) * args.x_stride);
            x_scale_buffer = buffer_of(args.x_scales + (first_row + base) * args.x_scale_stride, scale_bytes_of(min(rows - base, 32), args.x_scale_stride));
        }
        const auto row_of = [&](int token) {  // of x; -1: none
            if (base + token >= rows) return -1;
            return kSource == kByEntries ? list[base + token] / args.entries_per_row : token;
        };
        const int x_row = row_of(token_of_lane), scale_row = row_of(lane >> 1);
        const uint32_t x_offset = static_cast<uint32_t>(x_row * args.x_stride) + group * 16;
        const uint32_t x_scale_offset = scale_row >= 0 ? static_cast<uint32_t>(scale_row * args.x_scale_stride) : kOutOfRange;
        u32x4_t raw_x_scales = fetch_scales(x_scale_buffer, x_scale_offset, first_chunk);
        f32x16_t sums[kSets];
#pragma unroll
        for (int s = 0; s < kSets; ++s) sums[s] = f32x16_t{};
#pragma unroll 1
        for (int c = first_chunk; c < end_chunk; ++c) {
            const int k0 = c * kChunk, in_group = (c - first_chunk) % kScaleChunks;
            u32x4_t x_part[4][kParts];
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int p = 0; p < kParts; ++p) {
                    // In e4m3 the halves of two blocks, in e2m1 one block.
                    const int k = k0 + i * 64, byte = kFormat == FM_MX_E4M3 ? k + p * 32 : k / 2;
                    x_part[i][p] = load_16(x, x_row >= 0 && k < inner ? x_offset + byte : kOutOfRange);
                }
            if (in_group == 0) {
#pragma unroll
                for (int s = 0; s < kSets; ++s) *(FM_LDS(u32x4_t) *)(scale_lds + s * kScaleBytes + lane * 16) = raw_scales[s];
                *(FM_LDS(u32x4_t) *)(scale_lds + kSets * kScaleBytes + lane * 16) = raw_x_scales;
                fetch_weight_scales(c + kScaleChunks);
                raw_x_scales = fetch_scales(x_scale_buffer, x_scale_offset, c + kScaleChunks);
            }
#pragma unroll
            for (int s = 0; s < kSets; ++s)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int row = 8 * i + (lane >> 3);
                    *(FM_LDS(u32x4_t) *)(chunk_lds + s * kSetBytes + row * 128 + (((lane & 7) ^ ((row >> 1) & 7)) << 4)) = raw[s][i];
                }
            fetch_weights(c + 1);
            // The lanes read what others wrote: the hardware keeps a wavefront's LDS operations in order, and this the compiler.
            asm volatile("" ::: "memory");
            const bool second = k0 + 128 < inner;
            u32x2_t scales[kSets + 1];  // of the weights, and of x
#pragma unroll
            for (int s = 0; s <= kSets; ++s) {
                scales[s] = *(FM_LDS(u32x2_t) *)(scale_lds + s * kScaleBytes + token_of_lane * 32 + in_group * 8);
                align_scales(scales[s], second, group);
            }
            for_each<0, 4>([&](auto step) {
                constexpr int i = decltype(step)::value;
#pragma unroll
                for (int s = 0; s < kSets; ++s) {
                    const u32x4_t fragment =
                        *(FM_LDS(u32x4_t) *)(chunk_lds + s * kSetBytes + token_of_lane * 128 + (((2 * i + group) ^ ((token_of_lane >> 1) & 7)) << 4));
                    sums[s] = multiply<kFormat, i % 2 * 2, i % 2 * 2>(fragment, x_part[i], scales[s][i / 2], scales[kSets][i / 2], sums[s]);
                }
            });
            asm volatile("" ::: "memory");  // and the next chunk's writes stay behind these reads
        }
        __syncthreads();

        // [wavefront][set][quad of a lane's sums][lane]. A thread then finishes the four columns 4 quad .. of a row.
        f32x4_t *partial = reinterpret_cast<f32x4_t *>(shared);
#pragma unroll
        for (int s = 0; s < kSets; ++s)
#pragma unroll
            for (int q = 0; q < 4; ++q)
                partial[((wave * kSets + s) * 4 + q) * 64 + lane] = f32x4_t{sums[s][4 * q], sums[s][4 * q + 1], sums[s][4 * q + 2], sums[s][4 * q + 3]};
        __syncthreads();
        for (int item = threadIdx.x; item < kAcross * 256; item += kWaves * 64) {
            const int block = item / 256, token = item / 8 % 32, quad = item % 8, row = base + token;
            const auto total = [&](int s) {
                const int place = ((block * kSplit * kSets + s) * 4 + quad / 2) * 64 + quad % 2 * 32 + token;
                f32x4_t sum = partial[place];
#pragma unroll
                for (int w = 1; w < kSplit; ++w) sum += partial[w * kSets * 256 + place];
                return sum;
            };
            f32x4_t value = total(0);
            const int column = (blockIdx.x * kAcross + block) * 32 + quad * 4;
            const int64_t out_row = row >= rows ? 0 : kSource == kByEntries ? list[row] : first_row + row;
            if constexpr (kQuantized) {
                // From the fp32 sums: one rounding, to the elements' type.
                f32x4_t up = {1.f, 1.f, 1.f, 1.f};
                if constexpr (kGated) up = total(1);
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
                FM_DISPATCH_DTYPE(args.out_dtype, Result, store_four(static_cast<Result *>(args.out) + out_row * args.out_stride + column, value, args.out_vectors, columns - column));
            }
        }
        __syncthreads();
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

template <int kFormat, bool kGated, bool kQuantized, Source kSource, int kSplit, int kAcross>
static int launch_stream(const ProductArgs &args, int workgroup_rows, hipStream_t stream) {
    const auto kernel = stream_kernel<kFormat, kGated, kQuantized, kSplit, kAcross, kSource>;
    constexpr int kSums = kSplit * kAcross * ((kGated ? 2 : 1) * 4096 + (kGated ? 3 : 2) * 32 * 8 * kScaleChunks);
    const int lds = kSums + (kSource == kByEntries ? (args.entries + 3) / 4 * 16 : 0);
    static std::atomic<uint64_t> configured{0};
    if (lds > 65536)
        if (int status = allow_lds(reinterpret_cast<const void *>(kernel), kSums + kMaxEntries * 4, configured)) return status;
    kernel<<<dim3(static_cast<uint32_t>((args.out_columns + kAcross * 32 - 1) / (kAcross * 32)), workgroup_rows), kSplit * kAcross * 64, lds, stream>>>(args);
    return FM_OK;
}

// Rows of workgroups where the rows are found by their entries: one per entry where there are fewer of them than experts.
static int entry_workgroup_rows(const ProductArgs &args) { return args.by_entry ? args.entries : static_cast<int>(args.experts); }

// As few wavefronts share a reduction as give the device twelve wavefronts per CU.
int stream_split(const ProductArgs &args) {
    // A map's rows have 128 of padding per expert; of its last ones it is not known whether there is anything in them.
    const int64_t busy = args.top_experts == nullptr ? min(max(args.rows - 128 * args.experts, int64_t(2)), args.experts) : entry_workgroup_rows(args);
    const int64_t sets = (args.out_columns + 31) / 32 * busy, chunks = (args.inner + kChunk - 1) / kChunk;
    constexpr int kWanted = 12 * 256;
    if (sets >= kWanted || chunks < 4) return 1;
    return sets * 4 >= kWanted || chunks < 8 ? 4 : 8;
}

template <int kFormat, bool kGated, bool kQuantized, Source kSource>
static int launch_split(const ProductArgs &args, hipStream_t stream) {
    const int workgroup_rows = kSource == kByMap ? static_cast<int>(args.experts) : entry_workgroup_rows(args);
    switch (stream_split(args)) {
        case 1: return launch_stream<kFormat, kGated, kQuantized, kSource, 1, 4>(args, workgroup_rows, stream);
        case 4: return launch_stream<kFormat, kGated, kQuantized, kSource, 4, 1>(args, workgroup_rows, stream);
        default: return launch_stream<kFormat, kGated, kQuantized, kSource, 8, 1>(args, workgroup_rows, stream);
    }
}

template <bool kGated, bool kQuantized, Source kSource>
static int launch_format(const ProductArgs &args, hipStream_t stream) {
    return args.format == FM_MX_E4M3 ? launch_split<FM_MX_E4M3, kGated, kQuantized, kSource>(args, stream)
                                     : launch_split<FM_MX_E2M1, kGated, kQuantized, kSource>(args, stream);
}

int stream_product(const ProductArgs &args, hipStream_t stream) {
    if (args.out_scales == nullptr) return launch_format<false, false, kByMap>(args, stream);
    return args.gated ? launch_format<true, true, kByMap>(args, stream) : launch_format<false, true, kByMap>(args, stream);
}

int few_tokens(const ProductArgs &layer_1, const ProductArgs &layer_2, const float *scores, void *out, int out_dtype, hipStream_t stream) {
    int status = layer_1.gated ? launch_format<true, true, kByEntries>(layer_1, stream) : launch_format<false, true, kByEntries>(layer_1, stream);
    if (status == FM_OK) status = launch_format<false, false, kByEntries>(layer_2, stream);
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
