// Products of many microscaled rows per expert with e2m1 expert weights, on tiles of 256 rows x 256 weight rows.
//
// Eight wavefronts, two per SIMD, multiply 64 rows x 128 weight rows each (2 x 4 blocks of v_mfma_scale_f32_32x32x64_f8f6f4; D's rows are weight rows, so
// that a lane has four neighbouring columns of one row). K passes in slices of 128 through three LDS slots: a slice's bytes go straight
// from memory into LDS, two slices ahead of the multiplications; one barrier a slice. Scales, 16 bytes of a row at a time, take the
// same way every fourth slice.
//
// A row's slice is 128 bytes (e4m3) or 64 (e2m1), in LDS XOR-swizzled in units of 16 bytes so that eight lanes that read the same unit of
// neighbouring rows hit all banks.
#include "fm_activation_math.h"
#include "fm_mx_product.h"

namespace fm {

namespace mx {

namespace tiles {

constexpr int kTile = 256, kSlice = 128, kSlots = 3, kThreads = 512, kWaves = 8;
constexpr int kBlocksN = 4, kBlocksM = 2;
constexpr int kWeightBytes = kTile * kSlice / 2, kScaleBytes = 2 * kTile * 16;
template <int kFormat>
constexpr int kRowBytes = kFormat == FM_MX_E4M3 ? kSlice : kSlice / 2;
template <int kFormat>
constexpr int kSlotBytes = kTile * kRowBytes<kFormat> + kWeightBytes;
template <int kFormat>
constexpr int kLdsBytes = kSlots * kSlotBytes<kFormat> + 2 * kScaleBytes;
static_assert(kLdsBytes<FM_MX_E4M3> <= 160 * 1024, "LDS of a CU");

constexpr uint32_t kOutOfRange = 0x80000000u, kRange = 0x7fffffffu;
constexpr int kResident = 256;  // workgroups: one per CU

// 16 bytes of each lane -> LDS at `target` + 16 * lane; zeros for offsets out of range.
__device__ __forceinline__ void load_to_lds(const uint8_t *base, uint32_t offset, int target) {
    const __amdgpu_buffer_rsrc_t resource = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<char *>(uniform_pointer(reinterpret_cast<const char *>(base))), 0, static_cast<int>(kRange), kBufferResourceFlags);
    // M0 is not handed out by the register allocator and nothing else in this file uses it.
    asm volatile("s_mov_b32 m0, %0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
                 :
                 : "s"(__builtin_amdgcn_readfirstlane(target)), "v"(offset), "s"(resource)
                 : "memory");
}

// Returns once at most `kNewest` of the loads this wavefront has issued are on their way, and all that it has asked LDS for is there.
template <int kNewest>
__device__ __forceinline__ void wait_for_loads() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(kNewest) : "memory");
}

// Where unit `u` of 16 bytes of row `row` is in a slot's rows of kUnits units.
template <int kUnits>
__device__ __forceinline__ int unit_address(int row, int u) {
    return kUnits == 8 ? row * 128 + ((u ^ (row & 7)) << 4) : row * 64 + ((u ^ ((row >> 1) & 3)) << 4);
}

__device__ __forceinline__ u32x4_t read_lds(int address) { return *(FM_LDS(u32x4_t) *)static_cast<uintptr_t>(address); }

template <int kFormat, bool kGated, typename Result>
__global__ __launch_bounds__(kThreads, 1) void tile_kernel(ProductArgs args, GemmArgs placement) {
    constexpr bool kQuantized = std::is_same<Result, uint8_t>::value;
    constexpr int kUnits = kRowBytes<kFormat> / 16, kXBytes = kTile * kRowBytes<kFormat>;
    constexpr int kXLoads = kXBytes / 1024 / kWaves, kWeightLoads = kWeightBytes / 1024 / kWaves, kLoads = kXLoads + kWeightLoads;
    constexpr int kParts = kFormat == FM_MX_E4M3 ? 2 : 1;
    extern __shared__ __attribute__((aligned(1024))) char lds_generic[];
    const int lds = static_cast<int>(reinterpret_cast<uintptr_t>((FM_LDS(char) *)lds_generic));
    const int scales_at = lds + kSlots * kSlotBytes<kFormat>;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5;
    const int wave_n = wave & 1, wave_m = wave >> 1;
    const int slices = static_cast<int>(args.inner) / kSlice, columns = static_cast<int>(args.columns);
    constexpr int kColumns = kGated ? kTile / 2 : kTile;  // of the result

    // The 32 workgroups of an XCD take consecutive tiles.
    int logical = (blockIdx.x % 8) * (kResident / 8) + blockIdx.x / 8;
    RowTile tile;
    for (; locate_tile<kTile>(placement, logical, tile); logical += kResident) {
        const int expert = __builtin_amdgcn_readfirstlane(tile.expert), rows_valid = __builtin_amdgcn_readfirstlane(tile.rows_valid);
        const int col0 = __builtin_amdgcn_readfirstlane(tile.tile_n) * kColumns;
        const int64_t row0 = tile.row0;
        const uint8_t *x = args.x + row0 * args.x_stride;
        const int64_t weight_row = static_cast<int64_t>(expert) * columns * (kGated ? 2 : 1) + col0;
        const uint8_t *weight = args.weight + weight_row * args.weight_stride;

        uint32_t x_offset[kXLoads], weight_offset[kWeightLoads], scale_offset;
        // Row `t` of the tile's weight rows, from the tile's first; -1: there is none. (Gated: 64 gates and their ups by turns.)
        const auto weight_row_of = [&](int t) {
            const int column = kGated ? t / 128 * 64 + t % 64 : t;
            return col0 + column >= columns ? -1 : kGated && t % 128 >= 64 ? column + columns : column;
        };
#pragma unroll
        for (int j = 0; j < kXLoads; ++j) {
            const int slot = (wave * kXLoads + j) * 64 + lane, row = slot / kUnits, at = slot % kUnits;
            const int unit = kUnits == 8 ? at ^ (row & 7) : at ^ ((row >> 1) & 3);
            x_offset[j] = row < rows_valid ? static_cast<uint32_t>(row * args.x_stride + unit * 16) : kOutOfRange;
        }
#pragma unroll
        for (int j = 0; j < kWeightLoads; ++j) {
            const int slot = (wave * kWeightLoads + j) * 64 + lane, t = slot / 4, unit = slot % 4 ^ ((t >> 1) & 3), row = weight_row_of(t);
            weight_offset[j] = row >= 0 ? static_cast<uint32_t>(row * args.weight_stride + unit * 16) : kOutOfRange;
        }
        // The lower wavefronts load the scales of 64 rows each, the upper ones those of the weight rows.
        const uint8_t *scales = wave < 4 ? args.x_scales + row0 * args.x_scale_stride : args.weight_scales + weight_row * args.weight_scale_stride;
        if (wave < 4) {
            const int row = wave * 64 + lane;
            scale_offset = row < rows_valid ? static_cast<uint32_t>(row * args.x_scale_stride) : kOutOfRange;
        } else {
            const int row = weight_row_of((wave - 4) * 64 + lane);
            scale_offset = row >= 0 ? static_cast<uint32_t>(row * args.weight_scale_stride) : kOutOfRange;
        }
        // The first of the four slices whose scales are loaded together with those of slice 4 group: the row's last ones end with it.
        const auto first_of_group = [&](int group) { return min(group * 4, slices - 4); };
        const auto fetch_scales = [&](int group) {
            const bool exists = group * 4 < slices;
            load_to_lds(scales + first_of_group(group) * 4, exists ? scale_offset : kOutOfRange, scales_at + (group & 1) * kScaleBytes + wave * 1024);
        };
        const auto fetch = [&](int s, int slot) {
            const bool exists = s < slices;
            const int target = lds + slot * kSlotBytes<kFormat>;
#pragma unroll
            for (int j = 0; j < kXLoads; ++j)
                load_to_lds(x + static_cast<int64_t>(s) * kRowBytes<kFormat>, exists ? x_offset[j] : kOutOfRange, target + (wave * kXLoads + j) * 1024);
#pragma unroll
            for (int j = 0; j < kWeightLoads; ++j)
                load_to_lds(weight + static_cast<int64_t>(s) * (kSlice / 2), exists ? weight_offset[j] : kOutOfRange,
                            target + kXBytes + (wave * kWeightLoads + j) * 1024);
        };

        f32x16_t acc[kBlocksN][kBlocksM];
#pragma unroll
        for (int n = 0; n < kBlocksN; ++n)
#pragma unroll
            for (int m = 0; m < kBlocksM; ++m) acc[n][m] = f32x16_t{};
        fetch_scales(0);
        fetch(0, 0);
        fetch(1, 1);
        const bool multiplies = wave_m * 64 < rows_valid;
        int slot = 0;
#pragma unroll 1
        for (int s = 0; s < slices; ++s) {
            // Slice s is there, and slice s - 1 has been read: its slot takes slice s + 2.
            wait_for_loads<kLoads>();
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
            if (s % 4 == 0) fetch_scales(s / 4 + 1);
            fetch(s + 2, slot == 0 ? 2 : slot - 1);
            if (multiplies) {
                const int x_at = lds + slot * kSlotBytes<kFormat>, weight_at = x_at + kXBytes;
                const int scale_word = scales_at + (s / 4 & 1) * kScaleBytes + (s - first_of_group(s / 4)) * 4;
                uint32_t x_scales[kBlocksM], weight_scales[kBlocksN];
#pragma unroll
                for (int m = 0; m < kBlocksM; ++m)
                    x_scales[m] = *(FM_LDS(uint32_t) *)static_cast<uintptr_t>(scale_word + (wave_m * 64 + m * 32 + (lane & 31)) * 16) >> (8 * half);
#pragma unroll
                for (int n = 0; n < kBlocksN; ++n)
                    weight_scales[n] = *(FM_LDS(uint32_t) *)static_cast<uintptr_t>(scale_word + (kTile + wave_n * 128 + n * 32 + (lane & 31)) * 16) >> (8 * half);
                const auto step = [&](auto constant) {
                    constexpr int i = decltype(constant)::value;
                    u32x4_t a[kBlocksN], b[kBlocksM][kParts];
#pragma unroll
                    for (int m = 0; m < kBlocksM; ++m)
#pragma unroll
                        for (int p = 0; p < kParts; ++p)
                            b[m][p] = read_lds(x_at + unit_address<kUnits>(wave_m * 64 + m * 32 + (lane & 31), (kFormat == FM_MX_E4M3 ? 4 * i + 2 * p : 2 * i) + half));
#pragma unroll
                    for (int n = 0; n < kBlocksN; ++n) a[n] = read_lds(weight_at + unit_address<4>(wave_n * 128 + n * 32 + (lane & 31), 2 * i + half));
#pragma unroll
                    for (int n = 0; n < kBlocksN; ++n)
#pragma unroll
                        for (int m = 0; m < kBlocksM; ++m)
                            acc[n][m] = multiply<kFormat, 2 * i, 2 * i>(a[n], b[m], weight_scales[n], x_scales[m], acc[n][m]);
                };
                step(std::integral_constant<int, 0>{});
                step(std::integral_constant<int, 1>{});
            }
            slot = slot == 2 ? 0 : slot + 1;
        }
        wait_for_loads<0>();  // zeros of slices past the end
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");

        if constexpr (kQuantized) {
            const auto store = [&](auto activate) {
#pragma unroll
                for (int n = 0; n < (kGated ? 2 : 4); ++n)
#pragma unroll
                    for (int m = 0; m < kBlocksM; ++m) {
                        // The block of 32 columns of a row is in lanes l and l + 32: quad q of its lane's sums are columns 8 q + 4 half ..
                        float values[16];
                        uint32_t largest = 0;
#pragma unroll
                        for (int i = 0; i < 16; ++i) {
                            values[i] = activate(acc[n][m][i]);
                            if constexpr (kGated) values[i] *= acc[n + 2][m][i];
                            largest = max(largest, magnitude_bits(values[i]));
                        }
                        largest = max(largest, static_cast<uint32_t>(__shfl_xor(static_cast<int>(largest), 32, 64)));
                        const uint32_t byte = scale_byte(kFormat, largest);
                        const float inverse = inverse_scale(byte);
                        const int row = wave_m * 64 + m * 32 + (lane & 31), column = col0 + wave_n * (kGated ? 64 : 128) + n * 32;
                        if (row >= rows_valid || column >= args.out_columns) continue;
                        const int64_t out_row = row0 + row;
                        uint8_t *target = static_cast<uint8_t *>(args.out) + out_row * args.out_stride;
#pragma unroll
                        for (int q = 0; q < 4; ++q) {
                            const uint32_t packed = pack_four(kFormat, values[4 * q], values[4 * q + 1], values[4 * q + 2], values[4 * q + 3], inverse);
                            const int at = column + 8 * q + 4 * half;
                            if (kFormat == FM_MX_E4M3) *reinterpret_cast<uint32_t *>(target + at) = packed;
                            else *reinterpret_cast<uint16_t *>(target + at / 2) = static_cast<uint16_t>(packed);
                        }
                        if (half == 0) args.out_scales[out_row * args.out_scale_stride + column / 32] = static_cast<uint8_t>(byte);
                    }
            };
            FM_DISPATCH_ACTIVATION(args.activation, kActivation, store([](float value) { return activation_forward<kActivation>(value); }));
        } else {
#pragma unroll
            for (int n = 0; n < kBlocksN; ++n)
#pragma unroll
                for (int m = 0; m < kBlocksM; ++m) {
                    const int row = wave_m * 64 + m * 32 + (lane & 31);
                    if (row >= rows_valid) continue;
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        const int column = col0 + wave_n * 128 + n * 32 + 8 * q + 4 * half;
                        Result *target = static_cast<Result *>(args.out) + (row0 + row) * args.out_stride + column;
                        if (args.out_vectors && column + 3 < columns) {
                            struct alignas(4 * sizeof(Result)) Four {
                                Result v[4];
                            } four;
#pragma unroll
                            for (int c = 0; c < 4; ++c) four.v[c] = from_float<Result>(acc[n][m][4 * q + c]);
                            *reinterpret_cast<Four *>(target) = four;
                        } else {
#pragma unroll
                            for (int c = 0; c < 4; ++c)
                                if (column + c < columns) target[c] = from_float<Result>(acc[n][m][4 * q + c]);
                        }
                    }
                }
        }
    }
}

template <int kFormat, bool kGated, typename Result>
static int launch(const ProductArgs &args, hipStream_t stream) {
    const auto kernel = tile_kernel<kFormat, kGated, Result>;
    static std::atomic<uint64_t> configured{0};
    if (int status = allow_lds(reinterpret_cast<const void *>(kernel), kLdsBytes<kFormat>, configured)) return status;
    GemmArgs placement{};
    placement.expert_ends = args.expert_ends, placement.expert_pad_begins = args.expert_pad_begins, placement.index_dtype = args.index_dtype;
    placement.rows = args.rows, placement.num_experts = static_cast<int>(args.experts);
    constexpr int kColumns = kGated ? kTile / 2 : kTile;
    placement.tiles_n = static_cast<int>((args.out_columns + kColumns - 1) / kColumns);
    kernel<<<kResident, kThreads, kLdsBytes<kFormat>, stream>>>(args, placement);
    return FM_OK;
}

template <bool kGated, typename Result>
static int launch(const ProductArgs &args, hipStream_t stream) {
    return args.format == FM_MX_E4M3 ? launch<FM_MX_E4M3, kGated, Result>(args, stream) : launch<FM_MX_E2M1, kGated, Result>(args, stream);
}

}  // namespace tiles

bool tile_product_takes(const ProductArgs &args) {
    using namespace tiles;
    // Scales of four slices are loaded at once; offsets from a tile's first row are counted in 31 bits.
    const int64_t weight_rows = args.gated ? args.columns + kTile : kTile;
    return args.inner >= 4 * kSlice && args.x_stride * kTile < (int64_t(1) << 31) && args.weight_stride * weight_rows < (int64_t(1) << 31) &&
           (args.rows / kTile + args.experts + 1) * ((args.out_columns + 127) / 128) < (int64_t(1) << 30);
}

int tile_product(const ProductArgs &args, int out_dtype, hipStream_t stream) {
    using namespace tiles;
    if (args.out_scales != nullptr) return args.gated ? launch<true, uint8_t>(args, stream) : launch<false, uint8_t>(args, stream);
    switch (out_dtype) {
        case FM_DTYPE_F32: return launch<false, float>(args, stream);
        case FM_DTYPE_BF16: return launch<false, bf16_t>(args, stream);
        default: return launch<false, f16_t>(args, stream);
    }
}

}  // namespace mx

}  // namespace fm
