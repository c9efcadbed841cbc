// Products of many microscaled rows per expert with e2m1 expert weights, on tiles of 256 rows x 256 weight rows.
//
// One workgroup per CU walks over its tiles. Its four wavefronts, one per SIMD, multiply 128 rows x 128 weight rows each (4 x 4 blocks of
// v_mfma_scale_f32_32x32x64_f8f6f4; D's rows are weight rows, so that a lane has neighbouring columns of one row). K passes in slices of 128
// through three or four LDS slots. A slice's bytes go straight from memory into LDS, as many slices ahead of the multiplications and on into the
// next tile; the fragments of a step of 64 are read while the step before is multiplied. What a slice needs of memory instructions is spread over its
// MFMAs in a fixed order. Scales, 16 bytes of a row for four slices, take the same way.
//
// A row's slice is 128 bytes (e4m3) or 64 (e2m1), in LDS XOR-swizzled in units of 16 bytes so that 16 lanes that read the same unit of
// neighbouring rows hit all 64 banks. Of every 32 weight rows, LDS row 8 a + 4 h + b holds row 16 h + 4 a + b: a lane (h: its half of the
// wavefront) then has 16 neighbouring columns of its row, and results leave without a way through LDS, which is full of the next tile's slices.
//
// Measured on two cards, 16384 rows of 8 experts: 4096 -> 2 x 14336 with the gated activation 1534 and 1604 us (e4m3, 2.5 and 2.4 PFLOP/s), 14336 -> 4096
// 742 and 774 us (2.6 and 2.5) and in e2m1 545 and 565 us (3.5 and 3.4); a loop of the instruction in registers on random data reaches 3.94 and 6.14 on the
// second. Two bounds: the clock under the power of random data (1.7 to 1.8 GHz of 2.4; in e2m1 1.9; with zeros for data the products take 76 to 84 % of the
// time), and the one wavefront of a SIMD, which issues loads and reads beside its products (matrix units busy 65 % of the cycles, in e2m1 44 %; without
// the loads 3.1 and 4.5 PFLOP/s, without reads too 3.2 and 5.0). 30006 rows of 64 experts, 2048 -> 2 x 1408: 172 us, busy 48 %, the results' way out 22 %.
#include "fm_activation_math.h"
#include "fm_mx_product.h"

namespace fm {

namespace mx {

namespace tiles {

constexpr int kTile = 256, kSlice = 128, kThreads = 256, kWaves = 4;
constexpr int kBlocks = 4;  // of 32, per wavefront and axis
constexpr int kWeightBytes = kTile * kSlice / 2, kScaleBytes = 2 * kTile * 16;
template <int kFormat>
constexpr int kRowBytes = kFormat == FM_MX_E4M3 ? kSlice : kSlice / 2;
template <int kFormat>
constexpr int kSlotBytes = kTile * kRowBytes<kFormat> + kWeightBytes;
// Rows in e2m1 are multiplied in half the time, and a slice is less: one more.
template <int kFormat>
constexpr int kSlots = kFormat == FM_MX_E4M3 ? 3 : 4;
template <int kFormat>
constexpr int kScaleSlots = kSlots<kFormat> - 1;
template <int kFormat>
constexpr int kLdsBytes = kSlots<kFormat> * kSlotBytes<kFormat> + kScaleSlots<kFormat> * kScaleBytes;
static_assert(kLdsBytes<FM_MX_E4M3> <= 160 * 1024 && kLdsBytes<FM_MX_E2M1> <= 160 * 1024, "LDS of a CU");

constexpr uint32_t kOutOfRange = 0x80000000u, kRange = 0x7fffffffu;
constexpr int kResident = 256;  // workgroups: one per CU

template <int kFirst, int kLast, typename F>
__device__ __forceinline__ void for_each(const F &f) {
    if constexpr (kFirst < kLast) {
        f(std::integral_constant<int, kFirst>{});
        for_each<kFirst + 1, kLast>(f);
    }
}

__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer_of(const uint8_t *base) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<char *>(uniform_pointer(reinterpret_cast<const char *>(base))), 0, static_cast<int>(kRange),
                                             kBufferResourceFlags);
}

// 16 bytes of each lane -> LDS at `target` + kMore + 16 * lane; zeros for offsets out of range. (M0 is not handed out by the register allocator and
// nothing else in this file uses it. Where the compiler has spilled the resource or the position, it brings them back by vector instructions, maybe right in
// front of this: five wait states up to the load that reads them, which are more than M0's. With M0's only, 0.5 to 2 % faster, three loads of the kernels for
// e4m3 rows would come too early.)
template <int kMore>
__device__ __forceinline__ void load_to_lds(__amdgpu_buffer_rsrc_t resource, uint32_t offset, int position, int target) {
    asm volatile("s_add_i32 m0, %0, %4\n\ts_nop 3\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds"
                 :
                 : "s"(__builtin_amdgcn_readfirstlane(target)), "v"(offset), "s"(resource), "s"(__builtin_amdgcn_readfirstlane(position)), "n"(kMore)
                 : "memory", "scc");
}

// The same where `lanes` is ~0, and nothing where it is 0: without a branch, past which the compiler would move what is around it.
template <int kMore>
__device__ __forceinline__ void load_to_lds_if(uint32_t lanes, __amdgpu_buffer_rsrc_t resource, uint32_t offset, int position, int target) {
    asm volatile("s_add_i32 m0, %0, %5\n\ts_mov_b32 exec_lo, %4\n\ts_mov_b32 exec_hi, %4\n\ts_nop 1\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds\n\ts_mov_b64 exec, -1"
                 :
                 : "s"(__builtin_amdgcn_readfirstlane(target)), "v"(offset), "s"(resource), "s"(__builtin_amdgcn_readfirstlane(position)),
                   "s"(__builtin_amdgcn_readfirstlane(lanes)), "n"(kMore)
                 : "memory", "scc");
}

// The products before this are done when it is over. (The compiler counts a product's 16 passes up to the instructions that it knows to read its sums,
// and does not look into assembly.)
__device__ __forceinline__ void wait_for_products() { asm volatile("s_nop 15\n\ts_nop 7"); }

// A block of sums, in accumulation registers up to here. (One by one: the compiler would copy a block that is handed over whole.) After `wait_for_products`.
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

// The same value, computed no earlier than where this stands.
__device__ __forceinline__ int here(int value) {
    asm volatile("" : "+s"(value));
    return value;
}

// Returns once at most `kNewest` of the loads this wavefront has issued are on their way, and all that it has asked LDS for is there.
template <int kNewest>
__device__ __forceinline__ void wait_for_loads() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(kNewest) : "memory");
}

template <typename T>
__device__ __forceinline__ T read_lds(int address, int offset) {
    return *(FM_LDS(T) *)((FM_LDS(char) *)static_cast<uintptr_t>(address) + offset);
}

// Which tile: as `locate_tile`, with the experts' rows in registers, two experts per lane.
constexpr int kMaxInRegisters = 128;
struct Experts {
    int begin[2], count[2], last[2];  // first row, row tiles, row tiles up to and with this expert's
    int end[2];
    int before[3];  // row tiles in front of each 64 experts, and of all

    __device__ __forceinline__ void load(const GemmArgs &args, int lane) {
        before[0] = 0;
#pragma unroll
        for (int part = 0; part < 2; ++part) {
            const int e = part * 64 + lane;
            int64_t first = 0, past = 0;
            if (e < args.num_experts) rows_of_expert(args, e, first, past);
            count[part] = first >= 0 && past > first ? static_cast<int>((past - first + kTile - 1) / kTile) : 0;
            begin[part] = static_cast<int>(first), end[part] = static_cast<int>(past);
            int sum = count[part];
#pragma unroll
            for (int offset = 1; offset < 64; offset <<= 1) {
                const int other = __shfl_up(sum, offset, 64);
                if (lane >= offset) sum += other;
            }
            last[part] = sum + before[part];
            before[part + 1] = __builtin_amdgcn_readlane(last[part], 63);
        }
    }
    __device__ __forceinline__ bool locate(const GemmArgs &args, int logical, RowTile &tile) const {
        if (args.num_experts > kMaxInRegisters) {
            // (Without halves in the last round.) The same in all lanes, which the compiler cannot know.
            RowTile found{};
            const bool exists = locate_tile<kTile>(args, logical, found);
            tile.expert = __builtin_amdgcn_readfirstlane(found.expert), tile.tile_n = __builtin_amdgcn_readfirstlane(found.tile_n);
            tile.rows_valid = __builtin_amdgcn_readfirstlane(found.rows_valid);
            tile.row0 = __builtin_amdgcn_readfirstlane(static_cast<int>(found.row0));  // rows are counted in 31 bits
            return __builtin_amdgcn_readfirstlane(static_cast<int>(exists)) != 0;
        }
        // Where half of the workgroups or fewer have a tile in the last round, they have the halves of one each: 14336 -> 4096, 16384 rows of 8 experts (1104
        // tiles, 80 in the last round) in e4m3 757 -> 724 us, in e2m1 548 -> 533.
        const int total = before[2] * args.tiles_n, last_round = total & ~(kResident - 1);
        const bool halved = total - last_round <= kResident / 2 && logical >= last_round;
        const bool second = halved && (logical & 1);
        if (halved) logical = last_round + (logical - last_round) / 2;
        if (logical >= total) return false;
        const int part = logical >= before[1] * args.tiles_n;
        const int lasts = part ? last[1] : last[0], counts = part ? count[1] : count[0];
        const uint64_t owners = __ballot(lasts * args.tiles_n > logical);
        const int owner = __ffsll(static_cast<unsigned long long>(owners)) - 1;
        const int owner_count = __builtin_amdgcn_readlane(counts, owner), owner_last = __builtin_amdgcn_readlane(lasts, owner);
        const int first = __builtin_amdgcn_readlane(part ? begin[1] : begin[0], owner), past = __builtin_amdgcn_readlane(part ? end[1] : end[0], owner);
        int row_tile;
        place_in_expert(logical - (owner_last - owner_count) * args.tiles_n, owner_count, args.tiles_n, row_tile, tile.tile_n);
        tile.expert = part * 64 + owner;
        tile.row0 = first + row_tile * kTile + (second ? kTile / 2 : 0);
        tile.rows_valid = min(halved ? kTile / 2 : kTile, past - static_cast<int>(tile.row0));
        return tile.rows_valid > 0;  // (a workgroup whose second half is empty has nothing after it)
    }
};

template <int kFormat, bool kGated, typename Result>
__global__ __launch_bounds__(kThreads, 1) void tile_kernel(ProductArgs args, GemmArgs placement) {
    constexpr bool kQuantized = std::is_same<Result, uint8_t>::value;
    constexpr int kUnits = kRowBytes<kFormat> / 16, kXBytes = kTile * kRowBytes<kFormat>;
    constexpr int kXLoads = kXBytes / 1024 / kWaves, kWeightLoads = kWeightBytes / 1024 / kWaves, kLoads = kXLoads + kWeightLoads;
    constexpr int kScaleLoads = kScaleBytes / 1024 / kWaves;
    constexpr int kParts = kFormat == FM_MX_E4M3 ? 2 : 1;
    constexpr int kColumns = kGated ? kTile / 2 : kTile;  // of the result
    extern __shared__ __attribute__((aligned(1024))) char lds_generic[];
    const int lds = static_cast<int>(reinterpret_cast<uintptr_t>((FM_LDS(char) *)lds_generic));
    constexpr int kSlots = tiles::kSlots<kFormat>;
    const int scales_at = lds + kSlots * kSlotBytes<kFormat>;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5;
    const int wave_n = wave & 1, wave_m = wave >> 1;
    const int slices = static_cast<int>(args.inner) / kSlice, columns = static_cast<int>(args.columns);

    // The 32 workgroups of an XCD take consecutive tiles.
    int logical = (blockIdx.x % 8) * (kResident / 8) + blockIdx.x / 8;
    Experts experts;
    experts.load(placement, lane);
    RowTile tile, upcoming;
    if (!experts.locate(placement, logical, upcoming)) return;

    // ---- loading: the slices of the workgroup's tiles one after the other, the last tile's followed by zeros -----------
    // The loads of a slice are in two parts: those of its scales and most of its rows in the second step after which its slot is free, the others
    // in the step after that one. Each part has its own registers, so that the next tile's are there when the first part needs them.
    constexpr int kLate = kLoads / 2, kLateRows = kLate - kWeightLoads, kEarlyRows = kXLoads - kLateRows, kEarly = kScaleLoads + kEarlyRows;
    static_assert(kLateRows >= 0, "all loads of weights are in the second part");
    __amdgpu_buffer_rsrc_t x_buffer, scale_buffer, late_x_buffer, late_weight_buffer;
    uint32_t x_offset[kEarlyRows], scale_offset[kScaleLoads], late_offset[kLate];
    int load_slice = 0, load_slot = lds, load_group = 0, load_scales = scales_at;
    int x_position = 0, target = 0, scale_position = 0, scale_target = 0, late_x_position = 0, late_weight_position = 0, late_target = 0;
    uint32_t scale_lanes = 0;
    bool more = true;
    // `upcoming` is the tile that is loaded from here on.
    const auto columns_valid = [&]() { return more ? columns - upcoming.tile_n * kColumns : 0; };
    const auto first_weight_row = [&]() { return static_cast<int64_t>(upcoming.expert) * columns * (kGated ? 2 : 1) + upcoming.tile_n * kColumns; };
    // Row of LDS row `t` from the tile's first weight row; -1: there is none. Gated: a wavefront's 64 gates, then their ups.
    const auto weight_row_of = [&](int t) {
        const int in_block = (t >> 2 & 1) * 16 + (t >> 3 & 3) * 4 + (t & 3), block = t / 32;
        const int column = (kGated ? block / 4 * 64 + block % 2 * 32 : block * 32) + in_block;
        return column >= columns_valid() ? -1 : kGated && block % 4 >= 2 ? column + columns : column;
    };
    const auto row_offset = [&](int j) {
        const int at = (wave * kXLoads + j) * 64 + lane, row = at / kUnits;
        const int unit = kUnits == 8 ? at % 8 ^ ((row >> 1) & 7) : at % 4 ^ ((row >> 2) & 3);
        return more && row < upcoming.rows_valid ? static_cast<uint32_t>(row * static_cast<int>(args.x_stride) + unit * 16) : kOutOfRange;
    };
    const auto set_up_early = [&]() {
        x_buffer = buffer_of(args.x + upcoming.row0 * args.x_stride);
#pragma unroll
        for (int j = 0; j < kEarlyRows; ++j) x_offset[j] = row_offset(j);
        // The lower wavefronts load the scales of the rows, the upper ones those of the weight rows.
        const bool of_rows = wave < kWaves / 2;
        scale_buffer = buffer_of(of_rows ? args.x_scales + upcoming.row0 * args.x_scale_stride : args.weight_scales + first_weight_row() * args.weight_scale_stride);
#pragma unroll
        for (int j = 0; j < kScaleLoads; ++j) {
            const int t = (wave * kScaleLoads + j) * 64 + lane;
            const int row = of_rows ? more && t < upcoming.rows_valid ? t : -1 : weight_row_of(t - kTile);
            scale_offset[j] = row >= 0 ? static_cast<uint32_t>(row * static_cast<int>(of_rows ? args.x_scale_stride : args.weight_scale_stride)) : kOutOfRange;
        }
    };
    const auto set_up_late = [&]() {
        late_x_buffer = x_buffer;
        late_weight_buffer = buffer_of(args.weight + first_weight_row() * args.weight_stride);
#pragma unroll
        for (int j = 0; j < kLate; ++j) {
            if (j < kLateRows) {
                late_offset[j] = row_offset(kEarlyRows + j);
            } else {
                const int at = (wave * kWeightLoads + j - kLateRows) * 64 + lane, t = at / 4, unit = at % 4 ^ ((t >> 2) & 3), row = weight_row_of(t);
                late_offset[j] = row >= 0 ? static_cast<uint32_t>(row * static_cast<int>(args.weight_stride) + unit * 16) : kOutOfRange;
            }
        }
    };
    // The scales of four slices come together; the last slices of a tile are in groups of two at least: while a group is read, the space of the one
    // before it takes one that begins kSlots slices further on, and a group of two (two such, where there are more slots) lies in between. A group's 16 bytes end with the row.
    const auto next_group = [&](int first) { return first + 4 - (slices - first - 4 == 1); };
    const auto first_scales = [&](int first) { return min(first, slices - 4); };
    const auto next_slot_of = [&](int at) { return at == lds + (kSlots - 1) * kSlotBytes<kFormat> ? lds : at + kSlotBytes<kFormat>; };
    const auto next_scales = [&](int at) { return at == scales_at + (kScaleSlots<kFormat> - 1) * kScaleBytes ? scales_at : at + kScaleBytes; };
    const auto begin_late = [&]() { late_x_position = x_position, late_weight_position = x_position / kRowBytes<kFormat> * (kSlice / 2), late_target = target; };
    // In parts, for the shadows of products.
    bool begins_load_group = false;
    const auto begin_early = [&](auto part_constant) {
        constexpr int part = decltype(part_constant)::value;
        if constexpr (part == 0) {
            const int first = here(load_group);
            begins_load_group = load_slice == first;
            scale_lanes = begins_load_group ? ~0u : 0;
            scale_position = first_scales(first) * 4;
        } else if constexpr (part == 1) {
            const int first = here(load_group);
            load_group = begins_load_group ? next_group(first) : first;
        } else if constexpr (part == 2) {
            const int at = here(load_scales);
            scale_target = at + wave * (kScaleLoads * 1024);
            load_scales = begins_load_group ? next_scales(at) : at;
        } else {
            const int slice = here(load_slice);
            x_position = slice * kRowBytes<kFormat>;
            load_slice = slice + 1;
            target = load_slot;
            load_slot = next_slot_of(load_slot);
        }
    };
    constexpr int kEarlyParts = 4;
    const auto load_early = [&](auto constant) {
        constexpr int j = decltype(constant)::value, at = j - kScaleLoads;
        if constexpr (j < kScaleLoads) load_to_lds_if<j * 1024>(scale_lanes, scale_buffer, scale_offset[j], scale_position, scale_target);
        else load_to_lds<at * 1024>(x_buffer, x_offset[at], x_position, target + wave * (kXLoads * 1024));
    };
    const auto load_late = [&](auto constant) {
        constexpr int j = decltype(constant)::value;
        if constexpr (j < kLateRows)
            load_to_lds<(kEarlyRows + j) * 1024>(late_x_buffer, late_offset[j], late_x_position, late_target + wave * (kXLoads * 1024));
        else
            load_to_lds<kXBytes + (j - kLateRows) * 1024>(late_weight_buffer, late_offset[j], late_weight_position, late_target + wave * (kWeightLoads * 1024));
    };

    // ---- multiplying ---------------------------------------------------------------------------------------------------
    u32x4_t weight_part[2][kBlocks], x_part[2][kBlocks][kParts];
    uint32_t weight_scales[kBlocks], x_scales[kBlocks], next_weight_scales[kBlocks], next_x_scales[kBlocks];
    // Lane addresses in a slot, one per unit of a slice; blocks, slots and the wavefront's rows are added.
    int x_address[2][kParts], weight_address[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int row = lane & 31;
#pragma unroll
        for (int p = 0; p < kParts; ++p) {
            const int unit = kParts == 2 ? 4 * i + 2 * p + half : 2 * i + half;
            x_address[i][p] = row * kRowBytes<kFormat> + (kUnits == 8 ? unit ^ ((row >> 1) & 7) : unit ^ ((row >> 2) & 3)) * 16;
        }
        weight_address[i] = kXBytes + wave_n * 128 * (kSlice / 2) + row * (kSlice / 2) + ((2 * i + half) ^ ((row >> 2) & 3)) * 16;
    }
    const int weight_scale_address = (kTile + wave_n * 128 + (lane & 31)) * 16, x_scale_address = (lane & 31) * 16;
    // Rows of a wavefront: as many blocks of 32 for both halves of the workgroup as the tile's rows need.
    const auto blocks_of = [&](const RowTile &of) { return of.rows_valid <= kTile / 2 ? kBlocks / 2 : kBlocks; };
    int slot = lds, group = 0, group_scales = scales_at;  // of the slice that is read
    int first_row = wave_m * blocks_of(upcoming) * 32;    // of the wavefront, in the tile that is read
    // Where a step's reads start, and by number the reads: of the scales (with the first step of a slice), then of the fragments.
    int x_from[kParts], weight_from, x_scales_from, weight_scales_from;
    const auto begin_reads = [&](auto step_constant) {
        constexpr int i = decltype(step_constant)::value;
        const int rows_at = here(slot + first_row * kRowBytes<kFormat>);
#pragma unroll
        for (int p = 0; p < kParts; ++p) x_from[p] = x_address[i][p] + rows_at;
        weight_from = weight_address[i] + slot;
    };
    constexpr int kReads = kBlocks * (1 + kParts), kScaleReads = 2 * kBlocks;
    const auto read = [&](auto constant, auto step_constant) {
        constexpr int item = decltype(constant)::value, i = decltype(step_constant)::value, at = i == 0 ? item - kScaleReads : item;
        if constexpr (at < 0) {
            if constexpr (item < kBlocks) next_weight_scales[item] = read_lds<uint32_t>(weight_scales_from, item * 512);
            else next_x_scales[item - kBlocks] = read_lds<uint32_t>(x_scales_from, (item - kBlocks) * 512);
        } else if constexpr (at < kBlocks) {
            weight_part[i][at] = read_lds<u32x4_t>(weight_from, at * 32 * (kSlice / 2));
        } else {
            constexpr int m = (at - kBlocks) / kParts, p = (at - kBlocks) % kParts;
            x_part[i][m][p] = read_lds<u32x4_t>(x_from[p], m * 32 * kRowBytes<kFormat>);
        }
    };
    const auto begin_scale_reads = [&](int first_slice_of_word, int next) {
        const int word = here(group_scales + (next - first_slice_of_word) * 4);
        weight_scales_from = weight_scale_address + word, x_scales_from = x_scale_address + word + first_row * 16;
    };
    // Byte 2 i of the word is then that of the lane's block in step i.
    const auto take_weight_scales = [&](int n) { weight_scales[n] = next_weight_scales[n] >> (8 * half); };
    const auto take_x_scales = [&]() {
#pragma unroll
        for (int m = 0; m < kBlocks; ++m) x_scales[m] = next_x_scales[m] >> (8 * half);
    };
    constexpr std::integral_constant<int, 0> kFirst{};
    constexpr std::integral_constant<int, 1> kSecond{};

    set_up_early();
    set_up_late();
#pragma unroll 1
    for (int s = 0; s < kSlots; ++s) {
        if (s > 0) for_each<0, kLate>(load_late);
        for_each<0, kEarlyParts>(begin_early);
        for_each<0, kEarly>(load_early);
        begin_late();
    }
    wait_for_loads<(kSlots - 2) * kLoads + kEarlyRows>();
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    begin_reads(kFirst);
    begin_scale_reads(0, 0);
    for_each<0, kReads + kScaleReads>([&](auto item) { read(item, kFirst); });
#pragma unroll
    for (int n = 0; n < kBlocks; ++n) take_weight_scales(n);
    take_x_scales();

    f32x16_t acc[kBlocks][kBlocks];
    while (true) {
        tile = upcoming;
#pragma unroll
        for (int n = 0; n < kBlocks; ++n)
#pragma unroll
            for (int m = 0; m < kBlocks; ++m)
#pragma unroll
                for (int i = 0; i < 16; ++i) acc[n][m][i] = 0.f;
        const auto multiply_tile = [&](auto blocks_constant) {
            constexpr int kRows = decltype(blocks_constant)::value, kProducts = kBlocks * kRows;
            const auto product = [&](auto constant, auto step_constant) {
                // Neighbouring MFMAs share an operand.
                constexpr int j = decltype(constant)::value, i = decltype(step_constant)::value, n = j / kRows, m = n % 2 ? kRows - 1 - j % kRows : j % kRows;
                acc[n][m] = multiply<kFormat, 2 * i, 2 * i>(weight_part[i][n], x_part[i][m], weight_scales[n], x_scales[m], acc[n][m]);
            };
            group = 0;
#pragma unroll 1
            for (int s = 0; s < slices; ++s) {
                if (load_slice == slices) {
                    logical += kResident;
                    more = more && experts.locate(placement, logical, upcoming);
                    set_up_early();
                    load_slice = load_group = 0;
                }
                if (load_slice == 1) set_up_late();
                int next = 0, next_slot = 0;
                bool begins_group = false;
                __builtin_amdgcn_sched_barrier(0);
                // First step; beside it the reads of the second, the rest of the loads of slice s + kSlots - 1, and what the second step needs to know.
                for_each<0, kProducts>([&](auto j) {
                    product(j, kFirst);
                    if constexpr (j == 0) begin_reads(kSecond);
                    constexpr int kBusy = kProducts - 2;
                    if constexpr (j < kBusy) {
                        for_each<j * kReads / kBusy, (j + 1) * kReads / kBusy>([&](auto item) { read(item, kSecond); });
                        for_each<j * kLate / kBusy, (j + 1) * kLate / kBusy>(load_late);
                    }
                    // A part of the state of the next load beside every other product, and then that of the slice that is read next.
                    constexpr int kApart = kProducts == 16 ? 2 : 1, part = (j - 1) / kApart;
                    if constexpr ((j - 1) % kApart == 0 && j > 0 && part < kEarlyParts) begin_early(std::integral_constant<int, part>{});
                    if constexpr (j > 0 && (j - 1) % kApart == 0 && part == kEarlyParts) {
                        const int following = here(s) + 1;
                        next = following == slices ? 0 : following;
                        begins_group = (next == 0) | (next == next_group(group));
                    }
                    if constexpr (j > 0 && (j - 1) % kApart == 0 && part == kEarlyParts + 1) {
                        const int first = here(group), at = here(slot);
                        group = begins_group ? next : first;
                        group_scales = begins_group ? next_scales(group_scales) : group_scales;
                        next_slot = next_slot_of(at);
                    }
                    __builtin_amdgcn_sched_barrier(0);
                });
                // Second step. Slice s + 1 is there when all wavefronts' loads of it are, and slice s has been read: slice s + kSlots takes its slot.
                product(kFirst, kSecond);
                __builtin_amdgcn_sched_barrier(0);
                wait_for_loads<(kSlots - 2) * kLoads>();  // all but those of the slices from s + 2 on (their scales are asked for first)
                __builtin_amdgcn_s_barrier();
                asm volatile("" ::: "memory");
                __builtin_amdgcn_sched_barrier(0);
                slot = next_slot;
                first_row = next == 0 ? wave_m * blocks_of(upcoming) * 32 : first_row;
                for_each<1, kProducts>([&](auto j) {
                    product(j, kSecond);
                    if constexpr (j == 1) begin_scale_reads(first_scales(group), next), begin_reads(kFirst);
                    constexpr int kItems = kReads + kScaleReads, kBusy = kProducts - 2;
                    if constexpr (j <= kBusy) {
                        for_each<(j - 1) * kItems / kBusy, j * kItems / kBusy>([&](auto item) { read(item, kFirst); });
                        for_each<(j - 1) * kEarly / kBusy, j * kEarly / kBusy>(load_early);
                    }
                    // (The products of weight block n are behind.)
                    if constexpr (kRows == kBlocks && j % kRows == kRows - 1 && j / kRows + 1 < kBlocks) take_weight_scales(j / kRows);
                    if constexpr (j == kProducts - 1) begin_late();
                    __builtin_amdgcn_sched_barrier(0);
                });
#pragma unroll
                for (int n = kRows == kBlocks ? kBlocks - 1 : 0; n < kBlocks; ++n) take_weight_scales(n);
                take_x_scales();
                // The compiler would move products past the branches above, away from what they are to overlap.
#pragma unroll
                for (int n = 0; n < kBlocks; ++n)
#pragma unroll
                    for (int m = 0; m < kRows; ++m) asm volatile("" : "+a"(acc[n][m]));
            }
        };
        const int blocks = blocks_of(tile);
        if (blocks == kBlocks) multiply_tile(std::integral_constant<int, kBlocks>{});
        else multiply_tile(std::integral_constant<int, kBlocks / 2>{});
        const bool last_tile = !more;
        __builtin_amdgcn_sched_barrier(0);
        wait_for_products();
        __builtin_amdgcn_sched_barrier(0);

        // ---- the tile's results: of block (n, m) a lane has columns 16 half .. + 15 of one row ---------------------------
        const int row_start = wave_m * blocks * 32, col0 = tile.tile_n * kColumns, out_lane = opaque(lane);
        if constexpr (kQuantized) {
            const auto store = [&](auto activate) {
#pragma unroll
                for (int n = 0; n < (kGated ? 2 : 4); ++n)
#pragma unroll
                    for (int m = 0; m < kBlocks; ++m) {
                        __builtin_amdgcn_sched_barrier(0);  // one block's values at a time: registers
                        if (m >= blocks) continue;
                        f32x16_t gates = settled(acc[n][m]), ups = settled(acc[kGated ? n + 2 : n][m]);
                        float values[16];
                        uint32_t largest = 0;
#pragma unroll
                        for (int i = 0; i < 16; ++i) {
                            values[i] = activate(gates[i]);
                            if constexpr (kGated) values[i] *= ups[i];
                            largest = max(largest, magnitude_bits(values[i]));
                        }
                        largest = max(largest, static_cast<uint32_t>(__shfl_xor(static_cast<int>(largest), 32, 64)));
                        const uint32_t byte = scale_byte(kFormat, largest);
                        const float inverse = inverse_scale(byte);
                        const int row = row_start + m * 32 + (out_lane & 31), column = col0 + wave_n * (kGated ? 64 : 128) + n * 32;
                        if (row >= tile.rows_valid || column >= args.out_columns) continue;
                        const int64_t out_row = tile.row0 + row;
                        uint8_t *out = static_cast<uint8_t *>(args.out) + out_row * args.out_stride;
                        uint32_t packed[4];
#pragma unroll
                        for (int q = 0; q < 4; ++q) packed[q] = pack_four(kFormat, values[4 * q], values[4 * q + 1], values[4 * q + 2], values[4 * q + 3], inverse);
                        if (kFormat == FM_MX_E4M3) *reinterpret_cast<u32x4_t *>(out + column + 16 * (out_lane >> 5)) = u32x4_t{packed[0], packed[1], packed[2], packed[3]};
                        else *reinterpret_cast<u32x2_t *>(out + (column + 16 * (out_lane >> 5)) / 2) = u32x2_t{packed[0] | packed[1] << 16, packed[2] | packed[3] << 16};
                        if (out_lane < 32) args.out_scales[out_row * args.out_scale_stride + column / 32] = static_cast<uint8_t>(byte);
                    }
            };
            FM_DISPATCH_ACTIVATION(args.activation, kActivation, store([](float value) { return activation_forward<kActivation>(value); }));
        } else {
#pragma unroll
            for (int m = 0; m < kBlocks; ++m) {
                const int row = row_start + m * 32 + (out_lane & 31);
                if (m >= blocks || row >= tile.rows_valid) continue;
#pragma unroll
                for (int n = 0; n < kBlocks; ++n) {
                    __builtin_amdgcn_sched_barrier(0);
                    const f32x16_t values = settled(acc[n][m]);
                    const int column = col0 + wave_n * 128 + n * 32 + 16 * (out_lane >> 5);
                    Result *out = static_cast<Result *>(args.out) + (tile.row0 + row) * args.out_stride + column;
                    constexpr int N = Vec16<Result>::N;
                    if (args.out_vectors && column + 15 < columns) {
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
                            if (column + c < columns) out[c] = from_float<Result>(values[c]);
                    }
                }
            }
        }
        if (last_tile) break;
    }
    wait_for_loads<0>();  // zeros behind the last tile
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
    // Scales of four slices are loaded at once; offsets from a tile's first row are counted in 31 bits, rows and tiles too.
    const int64_t weight_rows = args.gated ? args.columns + kTile : kTile;
    const int64_t x_stride = max(args.x_stride, args.x_scale_stride), weight_stride = max(args.weight_stride, args.weight_scale_stride);
    return args.inner >= 4 * kSlice && x_stride * kTile < (int64_t(1) << 31) && weight_stride * weight_rows < (int64_t(1) << 31) &&
           (args.rows / kTile + args.experts + 1) * ((args.out_columns + 127) / 128) < (int64_t(1) << 30);
}

int tile_product(const ProductArgs &args, hipStream_t stream) {
    using namespace tiles;
    if (args.out_scales != nullptr) return args.gated ? launch<true, uint8_t>(args, stream) : launch<false, uint8_t>(args, stream);
    switch (args.out_dtype) {
        case FM_DTYPE_F32: return launch<false, float>(args, stream);
        case FM_DTYPE_BF16: return launch<false, bf16_t>(args, stream);
        default: return launch<false, f16_t>(args, stream);
    }
}

}  // namespace mx

}  // namespace fm
