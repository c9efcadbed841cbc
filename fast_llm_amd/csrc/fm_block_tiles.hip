// Products of operands of 8 bits with a scale per block of 128, on tiles of 256 x 256: rows times expert weights, and weight gradients (the same
// product with an expert's part of the reduction in place of its part of the rows). Both operands lie along the reduction.
//
// One workgroup per CU walks over its tiles. Its four wavefronts, one per SIMD, multiply 128 rows x 128 weight rows each (4 x 4 blocks of
// v_mfma_scale_f32_32x32x64_f8f6f4, 256 accumulation registers; D's rows are weight rows, so that a lane has neighbouring columns of one row). The
// reduction passes in slices of 128, a block of the format, through two LDS slots of 64 KB, on into the next tile. A slice's bytes go straight from
// memory into LDS. A step multiplies half of a wavefront's rows over the whole slice, and what the next step needs is read beside it; what has been
// read makes room for the slice after the next one at once, two to three steps before that is read. Every product has one or two reads or loads in
// its shadow, and is kept in its place among them. The scales of a slice, a byte for each row, are next to each other: a wavefront brings those of
// its rows with one load, which pass LDS to the lanes that hold the rows. With exact sums (`kWide`) a step is 64 of the slice, and 256 conversions to
// bf16 go with 128 products of half the length.
//
// 16384 rows of 8 experts, 14336 -> 4096: 749 to 780 us by card, 2.47 to 2.57 PFLOP/s, matrix units busy 68 % at 1.6 to 1.7 GHz (bound by power, and
// by waits at the barriers of a step); with steps of half a slice, whose loads were asked for one to two steps ahead, and products that the compiler
// moved behind the loads, 830. With exact sums 1490 at 1.29 PFLOP/s, busy 66 % at 1.87 GHz: a conversion takes 12 cycles, two of them a product's
// whole shadow. Weight gradient 14336 x 4096 of as many rows: 900, as every 16 slices have an epilogue. Into fp32 that is added to (128 experts, 1536
// x 2048, 131072 rows) 1210, half of it memory at 4.9 TB/s.
//
// A row's slice is 128 bytes, in LDS XOR-swizzled in units of 16 bytes so that 16 lanes that read the same unit of neighbouring rows hit all 64
// banks. Of every 32 weight rows, LDS row 8 a + 4 h + b holds row 16 h + 4 a + b: a lane (h: its half of the wavefront) then has 16 neighbouring
// columns of its row, and results leave without a way through LDS, which is full of the next tile's slices.
#include <algorithm>
#include <atomic>
#include <type_traits>

#include "fm_block_product.h"

namespace fm {

namespace block {

namespace tiles {

constexpr int kTile = 256, kSlice = kBlock, kThreads = 256, kWaves = 4;
constexpr int kBlocks = 4;  // of 32, per wavefront and axis
constexpr int kOperandBytes = kTile * kSlice, kSlotBytes = 2 * kOperandBytes, kSlots = 2;
// Scales of a slice: a load per wavefront, of the rows of one half of the tile or of its weight rows, from an address of any alignment in pieces of
// 16.
constexpr int kScaleBytes = 1024, kScaleSlots = 3, kScaleSlotBytes = kWaves * kScaleBytes, kScalePieces = 128 / 16 + 1;
constexpr int kPlaceBytes = 3 * 1024 * 4;  // see Places
constexpr int kLdsBytes = kSlots * kSlotBytes + kScaleSlots * kScaleSlotBytes + kPlaceBytes;
static_assert(kLdsBytes <= 160 * 1024, "LDS of a CU");
constexpr int kLoads = kOperandBytes / 1024 / kWaves;  // of a wavefront, per operand and slice
constexpr int kResident = 256;                         // workgroups: one per CU
// The loads of scales run this many slices ahead; a tile has no fewer, so that they are at most one tile ahead. (What is behind a tile's last slice
// is zero.)
constexpr int kMinSlices = kSlots + 1;

template <int kFirst, int kLast, typename F>
__device__ __forceinline__ void for_each(const F &f) {
    if constexpr (kFirst < kLast) {
        f(std::integral_constant<int, kFirst>{});
        for_each<kFirst + 1, kLast>(f);
    }
}

__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer_of(const uint8_t *base, uint32_t bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<char *>(uniform_pointer(reinterpret_cast<const char *>(base))), 0,
                                             __builtin_amdgcn_readfirstlane(static_cast<int>(bytes)), kBufferResourceFlags);
}

// 16 bytes of each lane -> LDS at `target` + kMore + 16 * lane; zeros for offsets out of range. (M0 is not handed out by the register allocator and
// nothing else in this file uses it. Where the compiler has spilled the resource, it brings it back by vector instructions, maybe right in front of
// this: five wait states up to the load that reads it, which are more than M0's.)
template <int kMore>
__device__ __forceinline__ void load_to_lds(__amdgpu_buffer_rsrc_t resource, uint32_t offset, int target) {
    asm volatile("s_add_i32 m0, %0, %3\n\ts_nop 3\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
                 :
                 : "s"(__builtin_amdgcn_readfirstlane(target)), "v"(offset), "s"(resource), "n"(kMore)
                 : "memory", "scc");
}

// The products before this are done when it is over. (The compiler counts a product's 16 passes up to the instructions that it knows to read its
// sums, and does not look into assembly.)
__device__ __forceinline__ void wait_for_products() { asm volatile("s_nop 15\n\ts_nop 7"); }

// A block of sums, in accumulation registers up to here. (One by one: the compiler would copy a block that is handed over whole.) After
// `wait_for_products`.
__device__ __forceinline__ f32x16_t settled(const f32x16_t &sums) {
    f32x16_t values;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        float value;
        asm volatile("v_accvgpr_read_b32 %0, %1" : "=v"(value) : "a"(sums[i]));
        values[i] = value;
    }
    return values;
}

// Returns once at most `kNewest` of the loads and stores that this wavefront has issued are on their way, and all that it has asked LDS for is there.
template <int kNewest>
__device__ __forceinline__ void wait_for_memory() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(kNewest) : "memory");
    __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0), for the compiler, which does not look into assembly and would wait for later reads with the earlier ones
}

__device__ __forceinline__ u32x4_t read_lds(int address, int offset) {
    return *(FM_LDS(u32x4_t) *)((FM_LDS(char) *)static_cast<uintptr_t>(address) + offset);
}

// Where a tile lies. Wave-uniform.
struct Tile {
    int expert, tile_n, row0, rows_valid;
    int first_slice, slices;  // of the reduction
};

// Which tile: by rows as `locate_tile`, by the reduction expert after expert. Where the experts lie is looked up once and kept in LDS.
constexpr int kMaxExperts = 1024;
static_assert(kPlaceBytes == 3 * kMaxExperts * 4, "room for the tables");
template <bool kByInner>
struct Places {
    int at;         // in LDS: of every expert where its rows (or slices of the reduction) begin and end, and by rows the row tiles up to and with its own
    int row_tiles;  // of all experts

    __device__ __forceinline__ FM_LDS(int) * table(int which) const { return (FM_LDS(int) *)static_cast<uintptr_t>(at + which * kMaxExperts * 4); }
    // (Without a map all of them.)
    static __device__ __forceinline__ void range_of_expert(const GemmArgs &args, int expert, int64_t &first, int64_t &past) {
        first = 0, past = args.rows;
        if (args.expert_ends != nullptr) rows_of_expert(args, expert, first, past);
        first = max(first, static_cast<int64_t>(0)), past = max(past, first);
    }
    // All threads of the workgroup take part.
    __device__ __forceinline__ void load(const GemmArgs &args) {
        if (threadIdx.x < 64) {
            const int lane = threadIdx.x;
            int before = 0;
            for (int base = 0; base < args.num_experts; base += 64) {
                const int e = base + lane;
                int64_t first = 0, past = 0;
                if (e < args.num_experts) range_of_expert(args, e, first, past);
                if constexpr (kByInner) {
                    // In whole slices: an expert's part begins at one.
                    if (e < args.num_experts) table(0)[e] = static_cast<int>(first / kSlice), table(1)[e] = past > first ? static_cast<int>((past + kSlice - 1) / kSlice) : static_cast<int>(first / kSlice);
                } else {
                    int sum = static_cast<int>((past - first + kTile - 1) / kTile);
#pragma unroll
                    for (int offset = 1; offset < 64; offset <<= 1) {
                        const int other = __shfl_up(sum, offset, 64);
                        if (lane >= offset) sum += other;
                    }
                    sum += before;
                    before = __builtin_amdgcn_readlane(sum, 63);
                    if (e < args.num_experts) table(0)[e] = static_cast<int>(first), table(1)[e] = static_cast<int>(past), table(2)[e] = sum;
                }
            }
        }
        __syncthreads();
        if constexpr (!kByInner) row_tiles = __builtin_amdgcn_readfirstlane(table(2)[args.num_experts - 1]);
    }
    __device__ __forceinline__ bool locate(const GemmArgs &args, int logical, int slices, Tile &tile) const {
        int row_tile;
        if constexpr (kByInner) {
            const int per_expert = args.tiles_m * args.tiles_n, expert = logical / per_expert;
            if (expert >= args.num_experts) return false;
            place_in_expert(logical - expert * per_expert, args.tiles_m, args.tiles_n, row_tile, tile.tile_n);
            const int first = __builtin_amdgcn_readfirstlane(table(0)[expert]), past = __builtin_amdgcn_readfirstlane(table(1)[expert]);
            tile.expert = expert, tile.row0 = row_tile * kTile;
            tile.rows_valid = min(kTile, static_cast<int>(args.sparse_size) - tile.row0);
            tile.first_slice = first, tile.slices = past - first;
            return true;
        }
        // Where half of the workgroups or fewer have a tile in the last round, they have the halves of one each.
        const int total = row_tiles * args.tiles_n, last_round = total & ~(kResident - 1);
        const bool halved = total - last_round <= kResident / 2 && logical >= last_round;
        const bool second = halved && (logical & 1);
        if (halved) logical = last_round + (logical - last_round) / 2;
        if (logical >= total) return false;
        int expert = 0;  // of the first one whose tiles reach past this
        for (int base = 0;; base += 64) {
            const int e = min(base + static_cast<int>(threadIdx.x & 63), args.num_experts - 1);
            const uint64_t owners = __ballot(table(2)[e] * args.tiles_n > logical);
            if (owners == 0) continue;
            expert = base + __ffsll(static_cast<unsigned long long>(owners)) - 1;
            break;
        }
        const int past_tiles = __builtin_amdgcn_readfirstlane(table(2)[expert]), first_tile = expert > 0 ? __builtin_amdgcn_readfirstlane(table(2)[expert - 1]) : 0;
        const int first = __builtin_amdgcn_readfirstlane(table(0)[expert]), past = __builtin_amdgcn_readfirstlane(table(1)[expert]);
        place_in_expert(logical - first_tile * args.tiles_n, past_tiles - first_tile, args.tiles_n, row_tile, tile.tile_n);
        tile.expert = expert;
        tile.row0 = first + row_tile * kTile + (second ? kTile / 2 : 0);
        tile.rows_valid = min(halved ? kTile / 2 : kTile, past - tile.row0);
        tile.first_slice = 0, tile.slices = slices;
        return tile.rows_valid > 0;  // (a workgroup whose second half is empty has nothing after it)
    }
};

template <bool kByInner, bool kAccumulate, bool kWide, typename Result>
__global__ __launch_bounds__(kThreads, 1) void tile_kernel(ProductArgs args, GemmArgs placement) {
    extern __shared__ __attribute__((aligned(1024))) char lds_generic[];
    const int lds = static_cast<int>(reinterpret_cast<uintptr_t>((FM_LDS(char) *)lds_generic));
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5;
    const int wave_n = wave & 1, wave_m = wave >> 1;
    const int inner_slices = static_cast<int>(args.inner / kSlice), columns = static_cast<int>(args.columns);

    // The 32 workgroups of an XCD take consecutive tiles.
    int logical = (blockIdx.x % 8) * (kResident / 8) + blockIdx.x / 8;
    Places<kByInner> places;
    places.at = lds + kSlots * kSlotBytes + kScaleSlots * kScaleSlotBytes;
    places.load(placement);
    Tile tile, upcoming;
    if (!places.locate(placement, logical, inner_slices, upcoming)) return;

    // ---- loading: the slices of the workgroup's tiles one after the other, the last tile's followed by zeros -----------
    // `upcoming` is the tile that is loaded. Wavefronts 2 m and 2 m + 1 take turns with 8 rows of the tile's half m, so that a lane has the same unit
    // in all its rows. In two groups: first the blocks of weight rows but the last of each half, and the first 64 rows of each half of the rows; then
    // the others. (A tile of up to 128 rows, which both halves of the workgroup share, has 32 rows in place of each 64.)
    const uint32_t x_stride = static_cast<uint32_t>(args.x_stride), weight_stride = static_cast<uint32_t>(args.weight_stride);
    const int load_row = (wave & 1) * 8 + (lane >> 3), load_unit = (lane & 7) ^ ((load_row >> 1) & 7);
    const uint32_t x_offset = static_cast<uint32_t>(load_row) * x_stride + load_unit * 16;
    // LDS row 32 c + 8 a + 4 h + b is row 32 c + 16 h + 4 a + b.
    const uint32_t weight_offset = static_cast<uint32_t>((wave >> 1) * 128 + (lane >> 5) * 16 + (wave & 1) * 4 + (lane >> 3 & 3)) * weight_stride + load_unit * 16;
    const auto slices_of = [](const Tile &of) { return max(of.slices, kMinSlices); };
    const auto blocks_of = [](const Tile &of) { return of.rows_valid <= kTile / 2 ? kBlocks / 2 : kBlocks; };
    const auto weight_row_of = [&](const Tile &of) { return (kByInner ? 0 : static_cast<int64_t>(of.expert) * columns) + of.tile_n * kTile; };
    const auto weight_rows_of = [&](const Tile &of) { return min(kTile, columns - of.tile_n * kTile); };
    bool more = true;
    const uint8_t *x_from[2] = {}, *weight_from = nullptr;
    uint32_t x_bytes[2] = {}, weight_bytes = 0;  // of a slice; none behind the tile's last one
    int load_slice = 0, load_slices = 0, real_slices = 0, load_target = lds;
    const auto begin_loads = [&]() {
        const int64_t first = static_cast<int64_t>(upcoming.first_slice) * kSlice;
        weight_from = args.weight + weight_row_of(upcoming) * args.weight_stride + first;
        load_slice = 0, load_slices = slices_of(upcoming), real_slices = more ? upcoming.slices : 0;
        const bool whole = blocks_of(upcoming) == kBlocks;
#pragma unroll
        for (int group = 0; group < 2; ++group) {
            const int row = (wave >> 1) * (whole ? 128 : 64) + group * (whole ? 64 : 32), rows = min(upcoming.rows_valid - row, whole ? 64 : 32);
            x_from[group] = args.x + (upcoming.row0 + row) * args.x_stride + first;
            x_bytes[group] = real_slices > 0 && rows > 0 ? (rows - 1) * x_stride + kSlice : 0;
        }
        weight_bytes = real_slices > 0 ? (weight_rows_of(upcoming) - 1) * weight_stride + kSlice : 0;
    };
    const auto advance = [&]() {
        ++load_slice;
        weight_from += kSlice, weight_bytes = load_slice < real_slices ? weight_bytes : 0;
#pragma unroll
        for (int group = 0; group < 2; ++group) x_from[group] += kSlice, x_bytes[group] = load_slice < real_slices ? x_bytes[group] : 0;
        load_target = load_target == lds ? lds + kSlotBytes : lds;
    };
    // Scales, a slice further ahead: they come from as many places of memory as there are slices, and are the last to arrive. (As far ahead as the
    // slice itself, 14336 -> 4096 with 16384 rows of 8 experts took 937 us for 800; as bytes for each block of 32 rows, straight to the lanes that
    // hold them, 998.) The first two wavefronts bring those of the halves of the tile's rows, the others those of the halves of its weight rows.
    const bool of_weights = wave >= 2;
    const int64_t scale_stride = of_weights ? args.weight_scale_stride : args.x_scale_stride;
    const uint32_t scale_offset = lane < kScalePieces ? lane * 16 : 0x80000000u;
    const uint8_t *scale_from = nullptr;
    uint32_t scale_bytes = 0;
    const int scales_at = lds + kSlots * kSlotBytes;
    int scale_slice = 0, scale_target = scales_at;
    const auto first_x_row = [&](const Tile &of, int half_of_tile) { return of.row0 + half_of_tile * blocks_of(of) * 32; };
    const auto begin_scales = [&]() {
        const int64_t weight_row = weight_row_of(upcoming);
        const int64_t row = of_weights ? weight_row + (wave - 2) * 128 : first_x_row(upcoming, wave);
        const int64_t past = of_weights ? weight_row + weight_rows_of(upcoming) : upcoming.row0 + upcoming.rows_valid;
        const int64_t from = row & ~int64_t(15);
        scale_from = (of_weights ? args.weight_scales : args.x_scales) + static_cast<int64_t>(upcoming.first_slice) * scale_stride + from;
        // Whole pieces: rows of scales are padded to them.
        scale_bytes = more && upcoming.slices > 0 && past > row ? static_cast<uint32_t>((past - from + 15) & ~int64_t(15)) : 0;
        scale_slice = 0;
    };
    const auto load_scales = [&]() {
        load_to_lds<0>(buffer_of(scale_from, scale_bytes), scale_offset, scale_target + wave * kScaleBytes);
        ++scale_slice;
        scale_from += scale_stride;
        scale_bytes = scale_slice < upcoming.slices ? scale_bytes : 0;
        scale_target = scale_target == scales_at + (kScaleSlots - 1) * kScaleSlotBytes ? scales_at : scale_target + kScaleSlotBytes;
    };
    constexpr int kItems = 2 * kLoads, kFirstWeights = kLoads / kBlocks * (kBlocks - 1), kFirstItems = kFirstWeights + kLoads / 2;
    const auto load = [&](auto constant) {
        constexpr int item = decltype(constant)::value, group = item < kFirstItems ? 0 : 1;
        constexpr bool weights = item < kFirstWeights || item >= kItems - (kLoads - kFirstWeights);
        const int target = load_target + (wave >> 1) * (128 * kSlice) + (wave & 1) * (8 * kSlice);
        if constexpr (weights) {
            constexpr int j = group == 0 ? item : item - (kItems - kLoads);
            load_to_lds<kOperandBytes + j * 16 * kSlice>(buffer_of(weight_from, weight_bytes), weight_offset + (j / 2 * 32 + j % 2 * 8) * here(weight_stride), target);
        } else {
            constexpr int j = (item - kFirstWeights) % (kLoads / 2);
            load_to_lds<(group * 64 + j * 16) * kSlice>(buffer_of(x_from[group], x_bytes[group]), x_offset + j * 16 * x_stride, target);
        }
    };

    // ---- multiplying ---------------------------------------------------------------------------------------------------
    u32x4_t weight_part[2][kBlocks][2], x_part[2][kBlocks][2];
    uint32_t scales[2 * kBlocks], next_scales[2 * kBlocks];
    constexpr int kScales = 2 * kBlocks;
    int scale_slot = scales_at, x_scales_at[2] = {}, weight_scales_at = 0;  // of the slice whose scales are read, and a lane's places in it
    const auto begin_scale_reads = [&](const Tile &of) {
        x_scales_at[0] = wave_m * kScaleBytes + (first_x_row(of, wave_m) & 15) + (lane & 31);
        x_scales_at[1] = x_scales_at[0] + blocks_of(of) * 16;
        // (The weight row of LDS row `lane % 32`.)
        weight_scales_at = (2 + wave_n) * kScaleBytes + static_cast<int>((weight_row_of(of) + wave_n * 128) & 15) + (lane >> 2 & 1) * 16 + (lane >> 3 & 3) * 4 + (lane & 3);
    };
    const auto read_scale = [&](auto constant) {
        constexpr int item = decltype(constant)::value, block = item % kBlocks;
        if constexpr (item < kBlocks) next_scales[item] = *(FM_LDS(uint8_t) *)((FM_LDS(char) *)static_cast<uintptr_t>(weight_scales_at + scale_slot) + block * 32);
        else next_scales[item] = *(FM_LDS(uint8_t) *)((FM_LDS(char) *)static_cast<uintptr_t>(x_scales_at[block / 2] + scale_slot) + block % 2 * 32);
    };
    const auto next_scale_slot = [&]() { scale_slot = scale_slot == scales_at + (kScaleSlots - 1) * kScaleSlotBytes ? scales_at : scale_slot + kScaleSlotBytes; };
    int address[2][2];  // of a lane in a row block, by step and part
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int p = 0; p < 2; ++p) address[i][p] = (lane & 31) * kSlice + ((4 * i + 2 * p + half) ^ ((lane >> 1) & 7)) * 16;
    int slot = lds;  // of the slice that is read
    constexpr int kReads = 4 * kBlocks;
    constexpr std::integral_constant<int, 0> kFirst{};
    constexpr std::integral_constant<int, 1> kSecond{};
    // Where the reads of a step start, and by number the reads: the fragments of the wavefront's weight rows, then of its rows.
    int weight_from_lds[2][2], x_from_lds[2][2];
    const auto begin_reads = [&](auto step_constant) {
        constexpr int i = decltype(step_constant)::value;
        const int weights_at = static_cast<int>(here(slot + wave_n * 128 * kSlice)), rows_at = static_cast<int>(here(slot + wave_m * 128 * kSlice));
#pragma unroll
        for (int p = 0; p < 2; ++p) weight_from_lds[i][p] = address[i][p] + weights_at, x_from_lds[i][p] = address[i][p] + rows_at;
    };
    const auto read = [&](auto constant, auto step_constant) {
        constexpr int item = decltype(constant)::value, i = decltype(step_constant)::value, p = item % 2, block = item / 2 % kBlocks;
        if constexpr (item < 2 * kBlocks) weight_part[i][block][p] = read_lds(weight_from_lds[i][p], kOperandBytes + block * 32 * kSlice);
        else x_part[i][block][p] = read_lds(x_from_lds[i][p], block * 32 * kSlice);
    };
    // The same by their use in the narrow loop: four reads are a block of weight rows, or of rows, over the whole slice.
    const auto read_block = [&](auto constant) {
        constexpr int item = decltype(constant)::value, block = item / 4, i = item / 2 % 2, p = item % 2;
        read(std::integral_constant<int, 2 * block + p>{}, std::integral_constant<int, i>{});
    };

    begin_scales();
    begin_loads();
#pragma unroll 1
    for (int s = 0; s < kMinSlices; ++s) {
        load_scales();
        if (s < kSlots) {
            for_each<0, kItems>(load);
            advance();
        }
    }
    wait_for_memory<0>();
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    begin_scale_reads(upcoming);
    for_each<0, kScales>(read_scale);
#pragma unroll
    for (int i = 0; i < kScales; ++i) scales[i] = kWide ? wide_scale(next_scales[i]) : next_scales[i];
    // kWide: a step of 64 is four of 16, and while one is multiplied the fragments of the next become bf16: by number four words of each, the weight
    // rows' first.
    constexpr int kParts = kWide ? 4 : 1, kConversions = kWide ? 2 * kBlocks * 4 : 0;
    u32x4_t wide_weight[kWide ? 2 : 1][kBlocks], wide_x[kWide ? 2 : 1][kBlocks];
    const auto widen = [&](auto constant, auto step_constant, auto part_constant, const uint32_t(&factors)[2 * kBlocks]) {
        constexpr int item = decltype(constant)::value, i = decltype(step_constant)::value, q = decltype(part_constant)::value, block = item / 4 % kBlocks, k = item % 4;
        constexpr int word = q % 2 * 2 + k / 2;
        if constexpr (item < 4 * kBlocks) wide_weight[q % 2][block][k] = widened<k % 2>(weight_part[i][block][q / 2][word], factors[block]);
        else wide_x[q % 2][block][k] = widened<k % 2>(x_part[i][block][q / 2][word], factors[kBlocks + block]);
    };
    begin_reads(kFirst);
    for_each<0, kReads>([&](auto item) { read(item, kFirst); });
    if constexpr (!kWide) {
        begin_reads(kSecond);
        for_each<0, kReads>([&](auto item) { read(item, kSecond); });
    }
    for_each<0, kConversions>([&](auto item) { widen(item, kFirst, kFirst, scales); });

    f32x16_t acc[kBlocks][kBlocks];
    while (true) {
        tile = upcoming;
        const int slices = slices_of(tile), blocks = blocks_of(tile);
#pragma unroll
        for (int n = 0; n < kBlocks; ++n)
#pragma unroll
            for (int m = 0; m < kBlocks; ++m)
#pragma unroll
                for (int i = 0; i < 16; ++i) acc[n][m][i] = 0.f;
        // In front of what comes next. (A product alone may move, within what has no branches to behind all of it.)
        const auto keep = [](f32x16_t &sums) { asm volatile("" : "+a"(sums)); };
        const auto multiply_tile = [&](auto blocks_constant) {
            constexpr int kRows = decltype(blocks_constant)::value, kProducts = kBlocks * kRows;
            const auto begin_slice = [&]() {
                if (load_slice == load_slices) begin_loads();
                if (scale_slice == slices_of(upcoming)) {
                    logical += kResident;
                    more = more && places.locate(placement, logical, inner_slices, upcoming);
                    begin_scales();
                }
            };
            const auto next_slot = [&](bool last) {
                slot = slot == lds ? lds + kSlotBytes : lds;
                next_scale_slot();
                if (last) begin_scale_reads(upcoming);
            };
            // Block m of the tile's rows is the wavefront's block `place_of(m)` in LDS.
            const auto place_of = [](int m) { return kRows == kBlocks ? m : 2 * m; };
            // Wide: steps of 64. Beside the first the reads of the second, beside the second the reads of the next slice and the loads of the one
            // behind it.
            constexpr int kSteps = kParts * kProducts;  // products of a step of 64
            // Reads are there before the step's last part, in which they are widened.
            constexpr int kReadsBusy = 2 * kProducts, kLoadsBusy = kSteps - 2;
            const auto wide_product = [&](auto constant, auto step_constant) {
                // Neighbouring products share an operand.
                constexpr int at = decltype(constant)::value, i = decltype(step_constant)::value, q = at / kProducts, j = at % kProducts;
                constexpr int n = j / kRows, m = n % 2 ? kRows - 1 - j % kRows : j % kRows;
                acc[n][m] = multiply_wide(wide_weight[q % 2][n], wide_x[q % 2][place_of(m)], acc[n][m]);
                // What the next part reads, in this step or the next one (of the next slice, with its scales).
                constexpr int first = j * kConversions / kProducts, past = (j + 1) * kConversions / kProducts;
                if constexpr (q + 1 < kParts) for_each<first, past>([&](auto item) { widen(item, step_constant, std::integral_constant<int, q + 1>{}, scales); });
                else if constexpr (i == 0) for_each<first, past>([&](auto item) { widen(item, kSecond, kFirst, scales); });
                else for_each<first, past>([&](auto item) { widen(item, kFirst, kFirst, next_scales); });
            };
            const auto wide_slice = [&](bool last) {
                begin_slice();
                __builtin_amdgcn_sched_barrier(0);
                for_each<0, kSteps>([&](auto j) {
                    wide_product(j, kFirst);
                    if constexpr (j == 0) begin_reads(kSecond);
                    if constexpr (j < kReadsBusy) for_each<j * kReads / kReadsBusy, (j + 1) * kReads / kReadsBusy>([&](auto item) { read(item, kSecond); });
                    __builtin_amdgcn_sched_barrier(0);
                });
                // Slice s + 1 is there when all wavefronts' loads of it are, and slice s has been read: slice s + 2 takes its slot.
                wide_product(kFirst, kSecond);
                __builtin_amdgcn_sched_barrier(0);
                wait_for_memory<1>();  // all but the scales of slice s + 3, which are asked for last
                __builtin_amdgcn_s_barrier();
                asm volatile("" ::: "memory");
                next_slot(last);
                __builtin_amdgcn_sched_barrier(0);
                for_each<1, kSteps>([&](auto j) {
                    // Of the next slice: its scales are there before the last part, in which its first fragments are widened.
                    if constexpr (j == kSteps - kProducts) {
#pragma unroll
                        for (int i = 0; i < kScales; ++i) next_scales[i] = wide_scale(next_scales[i]);
                    }
                    wide_product(j, kSecond);
                    if constexpr (j == 1) begin_reads(kFirst);
                    if constexpr (j <= kReadsBusy) {
                        for_each<(j - 1) * kReads / kReadsBusy, j * kReads / kReadsBusy>([&](auto item) { read(item, kFirst); });
                        for_each<(j - 1) * kScales / kReadsBusy, j * kScales / kReadsBusy>(read_scale);
                    }
                    if constexpr (j <= kLoadsBusy) for_each<(j - 1) * kItems / kLoadsBusy, j * kItems / kLoadsBusy>(load);
                    if constexpr (j == kLoadsBusy) load_scales();  // the last of the slice's loads
                    __builtin_amdgcn_sched_barrier(0);
                });
            };
            // Narrow: the first step multiplies the whole slice of half of the rows, the second one that of the others. A slice's first group of
            // loads has been read before its first step and the second group before its second one, and what takes their places is asked for at once,
            // two to three steps before it is read.
            constexpr int kHalf = kProducts, kPerWeight = kHalf / kBlocks;  // products of a step, and of a block of weight rows in it
            constexpr int kFirstBusy = kHalf - 2, kFirstReads = 12, kAwaited = kItems + 1;
            const auto narrow_product = [&](auto constant, auto group_constant) {
                constexpr int at = decltype(constant)::value, group = decltype(group_constant)::value, n = at / kPerWeight;
                constexpr int i = at % kPerWeight / (kPerWeight / 2), b = at % (kPerWeight / 2), place = 2 * group + b, m = kRows == kBlocks ? place : group;
                acc[n][m] = multiply(weight_part[i][n], x_part[i][place], scales[n], scales[kBlocks + place], acc[n][m]);
                keep(acc[n][m]);
            };
            const auto narrow_slice = [&](bool last) {
                narrow_product(kFirst, kFirst);
                begin_slice();
                __builtin_amdgcn_sched_barrier(0);
                narrow_product(kSecond, kFirst);
                __builtin_amdgcn_sched_barrier(0);
                // The second group of slice s is there (all that was asked for after it are two groups and scales), and all wavefronts have read the
                // first one.
                wait_for_memory<kAwaited>();
                __builtin_amdgcn_s_barrier();
                asm volatile("" ::: "memory");
                load_scales();  // of slice s + 3, where those of this one were
                __builtin_amdgcn_sched_barrier(0);
                for_each<2, kHalf>([&](auto j) {
                    narrow_product(j, kFirst);
                    // The last block of weight rows and the other half of the rows.
                    for_each<(j - 2) * kFirstReads / kFirstBusy, (j - 1) * kFirstReads / kFirstBusy>([&](auto item) {
                        read_block(std::integral_constant<int, item < 4 ? 4 * (kBlocks - 1) + item : 4 * (kBlocks + kBlocks / 2) + item - 4>{});
                    });
                    for_each<(j - 2) * kFirstItems / kFirstBusy, (j - 1) * kFirstItems / kFirstBusy>(load);
                    __builtin_amdgcn_sched_barrier(0);
                });
                narrow_product(kFirst, kSecond);
                next_slot(last);
                __builtin_amdgcn_sched_barrier(0);
                narrow_product(kSecond, kSecond);
                begin_reads(kFirst);
                begin_reads(kSecond);
                // The first group of slice s + 1 is there, and the second one of slice s has been read.
                wait_for_memory<kAwaited>();
                __builtin_amdgcn_s_barrier();
                asm volatile("" ::: "memory");
                __builtin_amdgcn_sched_barrier(0);
                for_each<2, kHalf>([&](auto j) {
                    narrow_product(j, kSecond);
                    // The first half of the rows, and each block of weight rows once the present one has been multiplied.
                    constexpr int kRowReads = 8, kLate = kPerWeight + kRows / 2, kWeightReads = 12;
                    if constexpr (j < kLate) for_each<4 * kBlocks + (j - 2) * kRowReads / (kLate - 2), 4 * kBlocks + (j - 1) * kRowReads / (kLate - 2)>(read_block);
                    else for_each<(j - kLate) * kWeightReads / (kHalf - kLate), (j - kLate + 1) * kWeightReads / (kHalf - kLate)>(read_block);
                    for_each<(j - 2) * kScales / (kHalf - 2), (j - 1) * kScales / (kHalf - 2)>(read_scale);
                    if constexpr (j < kHalf - 1) for_each<kFirstItems + (j - 2) * (kItems - kFirstItems) / (kHalf - 3), kFirstItems + (j - 1) * (kItems - kFirstItems) / (kHalf - 3)>(load);
                    if constexpr (j == kHalf - 2) advance();
                    __builtin_amdgcn_sched_barrier(0);
                });
            };
#pragma unroll 1
            for (int s = 0; s < slices; ++s) {
                if constexpr (kWide) wide_slice(s + 1 == slices);
                else narrow_slice(s + 1 == slices);
                // The compiler would move products past the branches above, away from what they are to overlap.
#pragma unroll
                for (int n = 0; n < kBlocks; ++n)
#pragma unroll
                    for (int m = 0; m < kRows; ++m) asm volatile("" : "+a"(acc[n][m]));
                if constexpr (kWide) advance();
#pragma unroll
                for (int i = 0; i < kScales; ++i) scales[i] = next_scales[i];
            }
        };
        if (blocks == kBlocks) multiply_tile(std::integral_constant<int, kBlocks>{});
        else multiply_tile(std::integral_constant<int, kBlocks / 2>{});
        const bool last_tile = !more;
        __builtin_amdgcn_sched_barrier(0);
        wait_for_products();
        __builtin_amdgcn_sched_barrier(0);

        // ---- the tile's results: of block (n, m) a lane has columns 16 half .. + 15 of one row ---------------------------
        const int row_start = wave_m * blocks * 32, col0 = tile.tile_n * kTile, out_lane = opaque(lane);
        const int64_t out_row = (kByInner ? tile.expert * args.rows : 0) + tile.row0;
        constexpr int N = Vec16<Result>::N, kVectors = 16 / N;
        bool stored = false;
        if constexpr (kAccumulate) {
            stored = args.out_vectors && columns % 16 == 0;
            if (stored) {
                // What is added to is asked for kAhead blocks ahead. Rows and columns that do not exist read the tile's first.
                constexpr int kAhead = 2;
                Vec16<Result> previous[kAhead][kVectors];
                const auto place = [&](int m, int n, bool &exists) {
                    const int row = row_start + m * 32 + (out_lane & 31), column = wave_n * 128 + n * 32 + 16 * (out_lane >> 5);
                    exists = m < blocks && row < tile.rows_valid && col0 + column < columns;
                    return static_cast<Result *>(args.out) + out_row * args.out_stride + col0 + (exists ? row * args.out_stride + column : 0);
                };
                const auto load_previous = [&](auto constant) {
                    constexpr int at = decltype(constant)::value;
                    bool exists;
                    const Result *out = place(at / kBlocks, at % kBlocks, exists);
#pragma unroll
                    for (int part = 0; part < kVectors; ++part) previous[at % kAhead][part] = load16(out + part * N);
                };
                for_each<0, kAhead>(load_previous);
                for_each<0, kBlocks * kBlocks>([&](auto constant) {
                    constexpr int at = decltype(constant)::value, m = at / kBlocks, n = at % kBlocks;
                    __builtin_amdgcn_sched_barrier(0);
                    f32x16_t values = settled(acc[n][m]);
                    Vec16<Result> vectors[kVectors];
#pragma unroll
                    for (int part = 0; part < kVectors; ++part)
#pragma unroll
                        for (int c = 0; c < N; ++c) vectors[part].v[c] = from_float<Result>(values[part * N + c] + to_float(previous[at % kAhead][part].v[c]));
                    if constexpr (at + kAhead < kBlocks * kBlocks) load_previous(std::integral_constant<int, at + kAhead>{});
                    bool exists;
                    Result *out = place(m, n, exists);
                    if (exists) {
#pragma unroll
                        for (int part = 0; part < kVectors; ++part) store16(out + part * N, vectors[part]);
                    }
                });
                // For the compiler, which would otherwise take one of these loads to be on its way in every slice of the next tile, and wait for all.
                __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0)
            }
        }
        if (!stored) {
#pragma unroll
            for (int m = 0; m < kBlocks; ++m) {
                const int row = row_start + m * 32 + (out_lane & 31);
                if (m >= blocks || row >= tile.rows_valid) continue;
#pragma unroll
                for (int n = 0; n < kBlocks; ++n) {
                    __builtin_amdgcn_sched_barrier(0);
                    f32x16_t values = settled(acc[n][m]);
                    const int column = col0 + wave_n * 128 + n * 32 + 16 * (out_lane >> 5);
                    Result *out = static_cast<Result *>(args.out) + (out_row + row) * args.out_stride + column;
                    if (!kAccumulate && args.out_vectors && column + 15 < columns) {
#pragma unroll
                        for (int part = 0; part < 16 / N; ++part) {
                            Vec16<Result> vector;
#pragma unroll
                            for (int c = 0; c < N; ++c) vector.v[c] = from_float<Result>(values[part * N + c]);
                            store16(out + part * N, vector);
                        }
                    } else {
#pragma unroll
                        for (int c = 0; c < 16; ++c)
                            if (column + c < columns) out[c] = from_float<Result>(values[c] + (kAccumulate ? to_float(out[c]) : 0.f));
                    }
                }
            }
        }
        if (last_tile) break;
    }
    wait_for_memory<0>();  // zeros behind the last tile
}

template <bool kByInner, bool kAccumulate, bool kWide, typename Result>
static int launch(const ProductArgs &args, hipStream_t stream) {
    const auto kernel = tile_kernel<kByInner, kAccumulate, kWide, Result>;
    static std::atomic<uint64_t> configured{0};
    if (int status = allow_lds(reinterpret_cast<const void *>(kernel), kLdsBytes, configured)) return status;
    GemmArgs placement{};
    placement.expert_ends = args.expert_ends, placement.expert_pad_begins = args.expert_pad_begins, placement.index_dtype = args.index_dtype;
    placement.rows = kByInner ? args.inner : args.rows, placement.sparse_size = args.rows, placement.num_experts = static_cast<int>(args.experts);
    placement.tiles_m = static_cast<int>((args.rows + kTile - 1) / kTile);
    placement.tiles_n = static_cast<int>((args.columns + kTile - 1) / kTile);
    kernel<<<kResident, kThreads, kLdsBytes, stream>>>(args, placement);
    return FM_OK;
}

template <bool kWide>
static int launch_rows(const ProductArgs &args, hipStream_t stream) {
    return args.out_dtype == FM_DTYPE_BF16 ? launch<false, false, kWide, bf16_t>(args, stream) : launch<false, false, kWide, f16_t>(args, stream);
}

// Gradients in fp16 are summed as exactly as those in fp32: micro-batches add up in them, and half a step of fp16 is no more than sixteen times what
// inexact sums are off.
template <bool kAccumulate>
static int launch_gradients(const ProductArgs &args, hipStream_t stream) {
    switch (args.out_dtype) {
        case FM_DTYPE_F32: return launch<true, kAccumulate, true, float>(args, stream);
        case FM_DTYPE_F16: return launch<true, kAccumulate, true, f16_t>(args, stream);
        default: return launch<true, kAccumulate, false, bf16_t>(args, stream);
    }
}

}  // namespace tiles

bool tile_product_takes(const ProductArgs &args) {
    // Offsets from a tile's first row are counted in 32 bits; rows and tiles in 31.
    const int64_t row_tiles = (args.rows / tiles::kTile + 1) * (args.by_inner ? args.experts : 1) + args.experts;
    return std::max(args.x_stride, args.weight_stride) * tiles::kTile < (int64_t(1) << 31) &&
           row_tiles * ((args.columns + tiles::kTile - 1) / tiles::kTile) < (int64_t(1) << 30);
}

int tile_product(const ProductArgs &args, hipStream_t stream) {
    using namespace tiles;
    if (args.by_inner) return args.accumulate ? launch_gradients<true>(args, stream) : launch_gradients<false>(args, stream);
    if (args.out_dtype == FM_DTYPE_F32) return launch<false, false, true, float>(args, stream);
    return args.exact ? launch_rows<true>(args, stream) : launch_rows<false>(args, stream);
}

}  // namespace block

}  // namespace fm
