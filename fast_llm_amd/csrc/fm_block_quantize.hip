// Rows to values of 8 bits with a scale per block of 128, along the rows, along the columns (transposed) or both, and back; their dispatch to the
// sparse layout.
//
// All are bound by memory. Rows alone: a lane takes sixteen neighbours, eight lanes a block, so that the block's maximum is three steps across lanes.
// With the columns: a workgroup takes a square of 128 x 128, in registers from its one read to the last write, eight rows x four columns a lane: of
// each row the maximum over 32 lanes, of each column over the lane's rows, two lanes and the eight wavefronts (by way of LDS). The transposed
// elements pass LDS, so that lines leave whole. In both forms 16384 x 4096 of bf16 take 50 us, 8 x 28672 x 4096 712, at 5.3 TB/s of the 6.5 that a
// copy reaches: the transposed form leaves as 128 lines of as many rows.
#include "fm_block_rows.h"

namespace fm {

namespace block {

// Rows of an input. `load`: eight rows x four columns of a lane in the square that begins at (`row0`, `column0`).
template <typename T>
struct Source {
    const T *input;
    int64_t stride;
    __device__ __forceinline__ void load(int64_t row0, int64_t column0, int exist, int count, int columns, float (&values)[kLaneRows][kLaneColumns]) const {
        Raw<T, kLaneColumns> raw[kLaneRows];
        load_block<kLaneRows, 1>(input + row0 * stride + column0, static_cast<uint32_t>(stride), threadIdx.x / 32 * kLaneRows, threadIdx.x % 32 * kLaneColumns, exist, count,
                                 columns, raw);
#pragma unroll
        for (int r = 0; r < kLaneRows; ++r)
#pragma unroll
            for (int c = 0; c < kLaneColumns; ++c) values[r][c] = to_float(raw[r].v[c]);
    }
};
// ... of 8 bits: with padding, so that columns are whole.
struct QuantizedSource {
    const uint8_t *input, *scales;
    int64_t stride, scale_stride;
    __device__ __forceinline__ void load(int64_t row0, int64_t column0, int exist, int count, int, float (&values)[kLaneRows][kLaneColumns]) const {
        const uint32_t first_row = threadIdx.x / 32 * kLaneRows, column = threadIdx.x % 32 * kLaneColumns;
        const uint8_t *block = input + row0 * stride + column0, *block_scales = scales + column0 / kBlock * scale_stride + row0;
        uint32_t words[kLaneRows], bytes[kLaneRows];
#pragma unroll
        for (int r = 0; r < kLaneRows; ++r) {
            const uint32_t row = min(static_cast<int>(first_row) + r, exist - 1);
            words[r] = *reinterpret_cast<const uint32_t *>(block + (row * static_cast<uint32_t>(stride) + column)), bytes[r] = block_scales[row];
        }
#pragma unroll
        for (int r = 0; r < kLaneRows; ++r) {
            const bool counts = static_cast<int>(first_row) + r < count;
            const uint32_t byte = counts ? bytes[r] : 0u;
            unpack_four(counts ? words[r] : 0u, scale_value(byte), values[r]);
            // 2^128, to which the largest values of fp32 were rounded, is not one: the largest takes its place and is rounded to it again.
            constexpr float kLargest = 3.40282346638528859812e+38f;
#pragma unroll
            for (int i = 0; i < kLaneColumns; ++i) values[r][i] = byte == 255u ? values[r][i] : __builtin_amdgcn_fmed3f(values[r][i], -kLargest, kLargest);
        }
    }
};

struct SquareArgs {
    uint8_t *values, *scales;          // null: the transposed form alone
    uint8_t *t_values, *t_scales;
    int64_t rows, columns;             // of a group
    int64_t value_stride, scale_stride, t_value_stride, t_scale_stride;
    uint32_t row_blocks, column_blocks;
    RowMap map;
};

template <typename Input, bool kRows>
__global__ __launch_bounds__(kSquareThreads) void square_kernel(Input input, SquareArgs args) {
    __shared__ __attribute__((aligned(16))) Square shared;
    const uint32_t column_block = blockIdx.x % args.column_blocks, rest = blockIdx.x / args.column_blocks;
    const int64_t group = rest / args.row_blocks, row_block = rest % args.row_blocks;
    const int64_t row0 = row_block * kBlock, column0 = static_cast<int64_t>(column_block) * kBlock;
    const int exist = static_cast<int>(min(args.rows - row0, static_cast<int64_t>(kBlock))), count = rows_in_block(args.map, row0, args.rows);
    const int64_t first = group * args.rows + row0;
    const int columns = static_cast<int>(min(args.columns - column0, static_cast<int64_t>(kBlock)));
    float values[kLaneRows][kLaneColumns];
    input.load(first, column0, exist, count, columns, values);
    const int64_t t_row = group * args.columns + column0;
    store_square<kRows>(values, shared, args.values + first * args.value_stride + column0, static_cast<uint32_t>(args.value_stride), args.scales + column_block * args.scale_stride + first, exist,
                        args.t_values + t_row * args.t_value_stride + row0, args.t_value_stride, args.t_scales + row_block * args.t_scale_stride + t_row,
                        columns);
}

template <typename T>
__global__ __launch_bounds__(kRowThreads) void row_kernel(const T *input, uint8_t *values, uint8_t *scales, int64_t rows, int64_t columns, int64_t input_stride,
                                                          int64_t value_stride, int64_t scale_stride, uint32_t column_blocks) {
    const uint32_t column_block = blockIdx.x % column_blocks;
    const int64_t row0 = static_cast<int64_t>(blockIdx.x / column_blocks) * kBlock, column0 = static_cast<int64_t>(column_block) * kBlock;
    const int first_row = threadIdx.x / 8, column = threadIdx.x % 8 * 16, exist = static_cast<int>(min(rows - row0, static_cast<int64_t>(kBlock)));
    Raw<T, 16> raw[kRowSteps];
    load_block<kRowSteps, kRowThreads / 8>(input + row0 * input_stride + column0, static_cast<uint32_t>(input_stride), first_row, column, exist, exist,
                                           static_cast<int>(min(columns - column0, static_cast<int64_t>(kBlock))), raw);
#pragma unroll
    for (int step = 0; step < kRowSteps; ++step) {
        float loaded[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) loaded[i] = to_float(raw[step].v[i]);
        const int row = first_row + step * (kRowThreads / 8);
        store_row(loaded, values + row0 * value_stride + column0 + (static_cast<uint32_t>(row) * static_cast<uint32_t>(value_stride) + column),
                  scales + column_block * scale_stride + row0 + row, row < exist);
    }
}

template <typename T>
__global__ __launch_bounds__(kRowThreads) void dequantize_kernel(const uint8_t *values, const uint8_t *scales, T *output, int64_t rows, int64_t columns,
                                                                 int64_t value_stride, int64_t scale_stride, uint32_t column_blocks, int vectors) {
    const uint32_t column_block = blockIdx.x % column_blocks;
    const int64_t row0 = static_cast<int64_t>(blockIdx.x / column_blocks) * kBlock, column = static_cast<int64_t>(column_block) * kBlock + threadIdx.x % 8 * 16;
#pragma unroll
    for (int step = 0; step < kRowSteps; ++step) {
        const int64_t row = row0 + step * (kRowThreads / 8) + threadIdx.x / 8;
        if (row >= rows || column >= columns) continue;
        const u32x4_t words = *reinterpret_cast<const u32x4_t *>(values + row * value_stride + column);
        const float scale = scale_value(scales[column_block * scale_stride + row]);
        T *out = output + row * columns + column;
        float result[16];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            float four[4];
            unpack_four(words[q], scale, four);
#pragma unroll
            for (int i = 0; i < 4; ++i) result[4 * q + i] = four[i];
        }
        constexpr int N = Vec16<T>::N;
        if (vectors && column + 16 <= columns) {
#pragma unroll
            for (int part = 0; part < 16 / N; ++part) {
                Vec16<T> vector;
#pragma unroll
                for (int i = 0; i < N; ++i) vector.v[i] = from_float<T>(result[part * N + i]);
                store16(out + part * N, vector);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 16; ++i)
                if (column + i < columns) out[i] = from_float<T>(result[i]);
        }
    }
}

// A workgroup per token: its bytes go to the token's rows of the sparse layout.
__global__ __launch_bounds__(kRowThreads) void dispatch_kernel(const uint8_t *values, const uint8_t *scales, uint8_t *out_values, uint8_t *out_scales,
                                                               const void *sparse_rows, int slots, int64_t sparse_row_count, int64_t value_stride,
                                                               int64_t scale_stride, int64_t out_stride, int64_t out_scale_stride, int blocks, int index_dtype) {
    const int64_t token = blockIdx.x;
    const int vectors = blocks * (kBlock / 16);
    for (int i = threadIdx.x; i < vectors + blocks; i += kRowThreads) {
        const bool is_value = i < vectors;
        u32x4_t vector = {};
        uint8_t scale = 0;
        if (is_value) vector = reinterpret_cast<const u32x4_t *>(values + token * value_stride)[i];
        else scale = scales[(i - vectors) * scale_stride + token];
        for (int j = 0; j < slots; ++j) {
            const int64_t row = load_index(sparse_rows, index_dtype, token * slots + j);
            if (row < 0 || row >= sparse_row_count) continue;
            if (is_value) reinterpret_cast<u32x4_t *>(out_values + row * out_stride)[i] = vector;
            else out_scales[(i - vectors) * out_scale_stride + row] = scale;
        }
    }
}

constexpr int64_t kMaxThreads = int64_t(1) << 32;

}  // namespace block

// What the entry points ask of a tensor in blocks; `rows` and padded `columns` of it.
int block::check_tensor(const char *name, const char *what, const void *values, const void *scales, int64_t rows, int64_t columns, int64_t value_stride,
                        int64_t scale_stride) {
    FM_REQUIRE(values && scales, "%s: null %s", name, what);
    FM_REQUIRE(value_stride >= columns && scale_stride >= padded_rows(rows), "%s: rows of %s overlap", name, what);
    FM_REQUIRE(aligned16(values) && value_stride % 16 == 0, "%s: rows of %s are 16-byte aligned", name, what);
    FM_REQUIRE(aligned16(scales) && scale_stride % 16 == 0, "%s: blocks of scales of %s are 16-byte aligned", name, what);
    return FM_OK;
}

int block::check_map(const char *name, RowMap &map, const void *expert_ends, const void *expert_pad_begins, int64_t num_experts, int index_dtype) {
    map = RowMap{};
    if (expert_ends == nullptr && expert_pad_begins == nullptr) return FM_OK;
    FM_REQUIRE(expert_ends && expert_pad_begins, "%s: half a map", name);
    FM_REQUIRE(num_experts > 0 && num_experts <= 1024, "%s: num_experts = %lld is not in 1 .. 1024", name, static_cast<long long>(num_experts));
    FM_REQUIRE(valid_index_dtype(index_dtype), "%s: bad index dtype %d", name, index_dtype);
    map = RowMap{expert_ends, expert_pad_begins, static_cast<int>(num_experts), index_dtype};
    return FM_OK;
}

}  // namespace fm

using namespace fm;

extern "C" int fm_block_quantize(const void *input, void *values, void *scales, void *transposed_values, void *transposed_scales, const void *expert_ends,
                                 const void *expert_pad_begins, int64_t groups, int64_t rows, int64_t columns, int64_t num_experts, int64_t input_row_stride,
                                 int64_t scale_stride, int64_t transposed_scale_stride, int dtype, int index_dtype, void *stream) {
    const char *name = "fm_block_quantize";
    FM_REQUIRE(valid_dtype(dtype), "%s: bad dtype %d", name, dtype);
    FM_REQUIRE(groups >= 0 && rows >= 0 && columns > 0 && columns <= block::kMaxColumns && rows < (int64_t(1) << 31) && groups < (int64_t(1) << 31) &&
                   groups * rows < (int64_t(1) << 31), "%s: bad sizes", name);
    block::SquareArgs args{};
    if (int status = block::check_map(name, args.map, expert_ends, expert_pad_begins, num_experts, index_dtype)) return status;
    FM_REQUIRE(args.map.expert_ends == nullptr || groups == 1, "%s: a map is of one group", name);
    const bool along_rows = values != nullptr || scales != nullptr, along_columns = transposed_values != nullptr || transposed_scales != nullptr;
    FM_REQUIRE(along_columns || args.map.expert_ends == nullptr, "%s: rows alone are quantised without a map", name);
    const int64_t all_rows = groups * rows, padded = block::padded_columns(columns), padded_rows = block::padded_columns(rows);
    if (all_rows == 0) return FM_OK;
    FM_REQUIRE(input && (along_rows || along_columns), "%s: null tensor", name);
    FM_REQUIRE(all_rows <= 1 || input_row_stride >= 0, "%s: negative stride", name);
    FM_REQUIRE(reinterpret_cast<uintptr_t>(input) % dtype_size(dtype) == 0, "%s: misaligned input", name);
    if (along_rows)
        if (int status = block::check_tensor(name, "the result", values, scales, all_rows, padded, padded, scale_stride)) return status;
    const int64_t row_blocks = padded_rows / block::kBlock, column_blocks = padded / block::kBlock;
    const auto hip_stream = static_cast<hipStream_t>(stream);
    if (padded > block::kMaxSquareStride || (all_rows > 1 && input_row_stride > block::kMaxSquareStride / dtype_size(dtype))) return fail(FM_ERR_UNSUPPORTED, "%s: too large", name);
    if (!along_columns) {
        const int64_t workgroups = (all_rows + block::kBlock - 1) / block::kBlock * column_blocks;
        if (workgroups >= block::kMaxThreads / block::kRowThreads) return fail(FM_ERR_UNSUPPORTED, "%s: too large", name);
        FM_DISPATCH_DTYPE(dtype, T, {
            block::row_kernel<T><<<static_cast<uint32_t>(workgroups), block::kRowThreads, 0, hip_stream>>>(
                static_cast<const T *>(input), static_cast<uint8_t *>(values), static_cast<uint8_t *>(scales), all_rows, columns, input_row_stride, padded,
                scale_stride, static_cast<uint32_t>(column_blocks));
        });
        return check_launch(name);
    }
    FM_REQUIRE(groups * columns < (int64_t(1) << 31), "%s: bad sizes", name);
    if (int status = block::check_tensor(name, "the transposed result", transposed_values, transposed_scales, groups * columns, padded_rows, padded_rows,
                                         transposed_scale_stride)) return status;
    if (groups * row_blocks * column_blocks >= block::kMaxThreads / block::kSquareThreads) return fail(FM_ERR_UNSUPPORTED, "%s: too large", name);
    args.values = static_cast<uint8_t *>(values), args.scales = static_cast<uint8_t *>(scales);
    args.t_values = static_cast<uint8_t *>(transposed_values), args.t_scales = static_cast<uint8_t *>(transposed_scales);
    args.rows = rows, args.columns = columns, args.value_stride = padded, args.scale_stride = scale_stride;
    args.t_value_stride = padded_rows, args.t_scale_stride = transposed_scale_stride;
    args.row_blocks = static_cast<uint32_t>(row_blocks), args.column_blocks = static_cast<uint32_t>(column_blocks);
    const uint32_t grid = static_cast<uint32_t>(groups * row_blocks * column_blocks);
    FM_DISPATCH_DTYPE(dtype, T, {
        const block::Source<T> source{static_cast<const T *>(input), input_row_stride};
        if (along_rows) block::square_kernel<block::Source<T>, true><<<grid, block::kSquareThreads, 0, hip_stream>>>(source, args);
        else block::square_kernel<block::Source<T>, false><<<grid, block::kSquareThreads, 0, hip_stream>>>(source, args);
    });
    return check_launch(name);
}

extern "C" int fm_block_transpose(const void *values, const void *scales, void *transposed_values, void *transposed_scales, const void *expert_ends,
                                  const void *expert_pad_begins, int64_t groups, int64_t rows, int64_t columns, int64_t num_experts, int64_t value_stride,
                                  int64_t scale_stride, int64_t transposed_scale_stride, int index_dtype, void *stream) {
    const char *name = "fm_block_transpose";
    FM_REQUIRE(groups >= 0 && rows >= 0 && columns > 0 && columns <= block::kMaxColumns && rows < (int64_t(1) << 31) && groups < (int64_t(1) << 31) &&
                   groups * rows < (int64_t(1) << 31) && groups * columns < (int64_t(1) << 31), "%s: bad sizes", name);
    block::SquareArgs args{};
    if (int status = block::check_map(name, args.map, expert_ends, expert_pad_begins, num_experts, index_dtype)) return status;
    FM_REQUIRE(args.map.expert_ends == nullptr || groups == 1, "%s: a map is of one group", name);
    const int64_t padded = block::padded_columns(columns), padded_rows = block::padded_columns(rows);
    if (groups * rows == 0) return FM_OK;
    if (int status = block::check_tensor(name, "the input", values, scales, groups * rows, padded, value_stride, scale_stride)) return status;
    if (int status = block::check_tensor(name, "the result", transposed_values, transposed_scales, groups * columns, padded_rows, padded_rows,
                                         transposed_scale_stride)) return status;
    const int64_t row_blocks = padded_rows / block::kBlock, column_blocks = padded / block::kBlock;
    if (value_stride > block::kMaxSquareStride || groups * row_blocks * column_blocks >= block::kMaxThreads / block::kSquareThreads)
        return fail(FM_ERR_UNSUPPORTED, "%s: too large", name);
    args.t_values = static_cast<uint8_t *>(transposed_values), args.t_scales = static_cast<uint8_t *>(transposed_scales);
    args.rows = rows, args.columns = columns, args.t_value_stride = padded_rows, args.t_scale_stride = transposed_scale_stride;
    args.row_blocks = static_cast<uint32_t>(row_blocks), args.column_blocks = static_cast<uint32_t>(column_blocks);
    const block::QuantizedSource source{static_cast<const uint8_t *>(values), static_cast<const uint8_t *>(scales), value_stride, scale_stride};
    block::square_kernel<block::QuantizedSource, false>
        <<<static_cast<uint32_t>(groups * row_blocks * column_blocks), block::kSquareThreads, 0, static_cast<hipStream_t>(stream)>>>(source, args);
    return check_launch(name);
}

extern "C" int fm_block_dequantize(const void *values, const void *scales, void *output, int64_t rows, int64_t columns, int64_t value_stride,
                                   int64_t scale_stride, int dtype, void *stream) {
    const char *name = "fm_block_dequantize";
    FM_REQUIRE(valid_dtype(dtype), "%s: bad dtype %d", name, dtype);
    FM_REQUIRE(rows >= 0 && rows < (int64_t(1) << 31) && columns > 0 && columns <= block::kMaxColumns, "%s: bad sizes", name);
    if (rows == 0) return FM_OK;
    const int64_t padded = block::padded_columns(columns), column_blocks = padded / block::kBlock;
    if (int status = block::check_tensor(name, "the input", values, scales, rows, padded, value_stride, scale_stride)) return status;
    FM_REQUIRE(output && reinterpret_cast<uintptr_t>(output) % dtype_size(dtype) == 0, "%s: null or misaligned output", name);
    const int64_t workgroups = (rows + block::kBlock - 1) / block::kBlock * column_blocks;
    if (workgroups >= block::kMaxThreads / block::kRowThreads) return fail(FM_ERR_UNSUPPORTED, "%s: too large", name);
    FM_DISPATCH_DTYPE(dtype, T, {
        block::dequantize_kernel<T><<<static_cast<uint32_t>(workgroups), block::kRowThreads, 0, static_cast<hipStream_t>(stream)>>>(
            static_cast<const uint8_t *>(values), static_cast<const uint8_t *>(scales), static_cast<T *>(output), rows, columns, value_stride, scale_stride,
            static_cast<uint32_t>(column_blocks), aligned16(output) && columns * dtype_size(dtype) % 16 == 0);
    });
    return check_launch(name);
}

extern "C" int fm_block_copy_dense_to_sparse(const void *values, const void *scales, const void *sparse_rows, void *out_values, void *out_scales,
                                             int64_t num_rows_dense, int64_t columns, int64_t num_experts_per_token, int64_t num_rows_sparse,
                                             int64_t value_stride, int64_t scale_stride, int64_t out_scale_stride, int index_dtype, void *stream) {
    const char *name = "fm_block_copy_dense_to_sparse";
    FM_REQUIRE(valid_index_dtype(index_dtype), "%s: bad index dtype %d", name, index_dtype);
    FM_REQUIRE(num_rows_dense >= 0 && num_rows_dense < (int64_t(1) << 31) && columns > 0 && columns <= block::kMaxColumns && num_experts_per_token > 0 &&
                   num_experts_per_token < (int64_t(1) << 31) && num_rows_sparse >= 0 && num_rows_sparse < (int64_t(1) << 31), "%s: bad sizes", name);
    if (num_rows_dense == 0 || num_rows_sparse == 0) return FM_OK;
    const int64_t padded = block::padded_columns(columns);
    if (int status = block::check_tensor(name, "the input", values, scales, num_rows_dense, padded, value_stride, scale_stride)) return status;
    if (int status = block::check_tensor(name, "the result", out_values, out_scales, num_rows_sparse, padded, padded, out_scale_stride)) return status;
    FM_REQUIRE(sparse_rows, "%s: null tensor", name);
    if (num_rows_dense >= block::kMaxThreads / block::kRowThreads) return fail(FM_ERR_UNSUPPORTED, "%s: too large", name);
    block::dispatch_kernel<<<static_cast<uint32_t>(num_rows_dense), block::kRowThreads, 0, static_cast<hipStream_t>(stream)>>>(
        static_cast<const uint8_t *>(values), static_cast<const uint8_t *>(scales), static_cast<uint8_t *>(out_values), static_cast<uint8_t *>(out_scales),
        sparse_rows, static_cast<int>(num_experts_per_token), num_rows_sparse, value_stride, scale_stride, padded, out_scale_stride,
        static_cast<int>(padded / block::kBlock), index_dtype);
    return check_launch(name);
}
