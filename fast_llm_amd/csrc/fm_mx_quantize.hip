// Rows to microscaled values and back, and their dispatch to the sparse layout. All three are bound by memory.
//
// A wavefront takes pieces of 512 columns of a row, eight columns a lane. The rows are buffers with their length as the bound: what is read behind it
// is zero, as the padding is to be, and what is written behind it is dropped, so that there is no branch and the loads of kUnroll pieces
// are under way at once. (At 1.5 to 2 bytes moved per element the arithmetic counts too: with 64-bit addresses and a division per lane, and the
// loads behind branches, 12001 x 3416 bf16 to e4m3 took 28.0 us, 32768 x 14336 bf16 to e2m1 219 and back 399.) Measured at these sizes: 22.5 us
// (126 MB, 5.6 TB/s), 180 and 177 us (1.20 GB each, 6.7 TB/s).
#include "fm_mx.h"

namespace fm {

namespace mx {

constexpr int kThreads = 256, kUnroll = 4;
constexpr int64_t kMaxWorkgroups = (int64_t(1) << 32) / kThreads;

constexpr int kPiece = 64 * 8, kNonTemporal = 2;

__device__ __forceinline__ __amdgpu_buffer_rsrc_t row_buffer(const void *start, int64_t bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<char *>(uniform_pointer(static_cast<const char *>(start))), 0,
                                             __builtin_amdgcn_readfirstlane(static_cast<int>(bytes)), kBufferResourceFlags);
}

// Which pieces a wavefront has: kUnroll in a row, counted along the rows.
struct Pieces {
    int64_t row;
    int part, per_row;
    __device__ __forceinline__ explicit Pieces(int columns) : per_row((columns + kPiece - 1) / kPiece) {
        const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), first = (blockIdx.x * (kThreads / 64) + wave) * kUnroll;
        row = first / static_cast<uint32_t>(per_row);
        part = static_cast<int>(first % static_cast<uint32_t>(per_row));
    }
    __device__ __forceinline__ void next() {
        if (++part == per_row) part = 0, ++row;
    }
};

template <typename T>
__device__ __forceinline__ void load_eight(__amdgpu_buffer_rsrc_t row, int offset, float (&values)[8]) {
    constexpr int N = Vec16<T>::N;
#pragma unroll
    for (int part = 0; part < 8 / N; ++part) {
        const auto vector = __builtin_bit_cast(Vec16<T>, __builtin_amdgcn_raw_buffer_load_b128(row, offset + part * 16, 0, kNonTemporal));
#pragma unroll
        for (int i = 0; i < N; ++i) values[part * N + i] = to_float(vector.v[i]);
    }
}

// Four neighbouring lanes have a block, sixteen the 128 columns whose four scales make a word. kWhole: the rows are whole vectors of eight, aligned to 16
// bytes; otherwise (from 8 columns on) loads are aligned as the values are, and the last lane of a row reads its last eight columns.
template <typename T, int kFormat, bool kWhole>
__global__ __launch_bounds__(kThreads) void quantize_kernel(const T *input, uint8_t *values, uint8_t *scales, int64_t rows, int64_t columns,
                                                            int64_t input_stride, int padded) {
    const int lane = threadIdx.x & 63;
    float loaded[kUnroll][8];
    Pieces pieces(padded);
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
        const int column = pieces.part * kPiece + lane * 8, size = static_cast<int>(sizeof(T)), count = static_cast<int>(columns);
        load_eight<T>(row_buffer(input + pieces.row * input_stride, pieces.row < rows ? columns * static_cast<int64_t>(sizeof(T)) : 0),
                      kWhole ? column * size : column < count ? window(column, count) * size : kNowhere, loaded[u]);
        pieces.next();
    }
    pieces = Pieces(padded);
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
        const bool exists = pieces.row < rows;
        const __amdgpu_buffer_rsrc_t value_row = row_buffer(values + pieces.row * value_bytes(kFormat, padded), exists ? value_bytes(kFormat, padded) : 0);
        const __amdgpu_buffer_rsrc_t scale_row = row_buffer(scales + pieces.row * scale_bytes(padded), exists ? scale_bytes(padded) : 0);
        const int column = pieces.part * kPiece + lane * 8;
        pieces.next();
        if constexpr (!kWhole) shift_down(loaded[u], max(column - window(column, static_cast<int>(columns)), 0) & 7);
        uint32_t largest = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) largest = max(largest, magnitude_bits(loaded[u][i]));
        const uint32_t byte = scale_byte(kFormat, max_of_neighbours<4>(largest));
        const float inverse = inverse_scale(byte);
        const uint32_t low = pack_four(kFormat, loaded[u][0], loaded[u][1], loaded[u][2], loaded[u][3], inverse);
        const uint32_t high = pack_four(kFormat, loaded[u][4], loaded[u][5], loaded[u][6], loaded[u][7], inverse);
        if constexpr (kFormat == FM_MX_E4M3) __builtin_amdgcn_raw_buffer_store_b64(u32x2_t{low, high}, value_row, column, 0, 0);
        else __builtin_amdgcn_raw_buffer_store_b32(low | high << 16, value_row, column / 2, 0, 0);
        uint32_t word = byte << (lane / 4 % 4 * 8);
        word |= static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(word), 0x141, 0xf, 0xf, true));  // the eight mirrored
        word |= static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(word), 0x140, 0xf, 0xf, true));  // the sixteen mirrored
        if (lane % 16 == 0) __builtin_amdgcn_raw_buffer_store_b32(word, scale_row, column / kBlock, 0, 0);
    }
}

// Rows of less than eight columns: a value per lane.
template <typename T>
__global__ __launch_bounds__(kThreads) void quantize_any_kernel(const T *input, uint8_t *values, uint8_t *scales, int64_t rows, int64_t columns,
                                                                int64_t input_stride, int padded, int format) {
    const int parts = (padded + kThreads - 1) / kThreads;
    for (int64_t part = blockIdx.x; part < rows * parts; part += gridDim.x) {
        const int64_t row = part / parts, column = (part - row * parts) * kThreads + threadIdx.x;
        const float value = column < columns ? to_float(input[row * input_stride + column]) : 0.f;
        store_one(format, value, values + row * value_bytes(format, padded), scales + row * scale_bytes(padded), column, column < padded);
    }
}

__device__ __forceinline__ float scale_value(uint32_t byte) {
    // 2^-127 is a subnormal number; 255 stands for NaN.
    return byte == 255u ? __builtin_nanf("") : byte == 0u ? __builtin_bit_cast(float, 0x00400000u) : __builtin_bit_cast(float, byte << 23);
}

// Eight elements, exact in fp32.
template <int kFormat>
__device__ __forceinline__ void elements(u32x2_t words, float (&result)[8]) {
    const auto pair = [&](auto position) {
        constexpr int kPair = decltype(position)::value;
        if constexpr (kFormat == FM_MX_E4M3) {
            result[2 * kPair] = __builtin_amdgcn_cvt_f32_fp8(static_cast<int>(words[kPair / 2]), kPair % 2 * 2);
            result[2 * kPair + 1] = __builtin_amdgcn_cvt_f32_fp8(static_cast<int>(words[kPair / 2]), kPair % 2 * 2 + 1);
        } else {
            const auto two = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(words[0], 1.f, kPair);
            result[2 * kPair] = two[0], result[2 * kPair + 1] = two[1];
        }
    };
    pair(std::integral_constant<int, 0>{});
    pair(std::integral_constant<int, 1>{});
    pair(std::integral_constant<int, 2>{});
    pair(std::integral_constant<int, 3>{});
}

template <typename T, int kFormat>
__global__ __launch_bounds__(kThreads) void dequantize_kernel(const uint8_t *values, const uint8_t *scales, T *output, int64_t rows, int64_t columns,
                                                              int64_t value_stride, int64_t scale_stride, int vectors) {
    const int lane = threadIdx.x & 63;
    const int64_t padded = padded_columns(columns);
    u32x2_t words[kUnroll];
    uint32_t scale[kUnroll];
    Pieces pieces(static_cast<int>(columns));
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
        const bool exists = pieces.row < rows;
        const __amdgpu_buffer_rsrc_t value_row = row_buffer(values + pieces.row * value_stride, exists ? value_bytes(kFormat, padded) : 0);
        const __amdgpu_buffer_rsrc_t scale_row = row_buffer(scales + pieces.row * scale_stride, exists ? scale_bytes(padded) : 0);
        const int column = pieces.part * kPiece + lane * 8;
        pieces.next();
        if constexpr (kFormat == FM_MX_E4M3) words[u] = __builtin_bit_cast(u32x2_t, __builtin_amdgcn_raw_buffer_load_b64(value_row, column, 0, kNonTemporal));
        else words[u] = u32x2_t{static_cast<uint32_t>(__builtin_amdgcn_raw_buffer_load_b32(value_row, column / 2, 0, kNonTemporal)), 0u};
        scale[u] = static_cast<uint8_t>(__builtin_amdgcn_raw_buffer_load_b8(scale_row, column / kBlock, 0, 0));
    }
    pieces = Pieces(static_cast<int>(columns));
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
        float result[8];
        elements<kFormat>(words[u], result);
        const float factor = scale_value(scale[u]);
#pragma unroll
        for (int i = 0; i < 8; ++i) result[i] *= factor;
        const __amdgpu_buffer_rsrc_t row = row_buffer(output + pieces.row * columns, pieces.row < rows ? columns * static_cast<int64_t>(sizeof(T)) : 0);
        const int column = pieces.part * kPiece + lane * 8, at = column * static_cast<int>(sizeof(T));
        pieces.next();
        if (vectors || column + 8 <= columns) {
            constexpr int N = Vec16<T>::N;
#pragma unroll
            for (int part = 0; part < 8 / N; ++part) {
                Vec16<T> vector;
#pragma unroll
                for (int i = 0; i < N; ++i) vector.v[i] = from_float<T>(result[part * N + i]);
                __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4_t, vector), row, at + part * 16, 0, kNonTemporal);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                if (column + i >= columns) break;
                if constexpr (sizeof(T) == 4) __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(uint32_t, result[i]), row, at + 4 * i, 0, 0);
                else __builtin_amdgcn_raw_buffer_store_b16(__builtin_bit_cast(uint16_t, from_float<T>(result[i])), row, at + 2 * i, 0, 0);
            }
        }
    }
}

// Workgroups for rows of so many columns, 0: too many for a launch, which counts its threads in 32 bits.
static int64_t piece_workgroups(int64_t rows, int64_t columns) {
    const int64_t per_workgroup = kUnroll * (kThreads / 64), per_row = (columns + kPiece - 1) / kPiece;
    const int64_t workgroups = (rows * per_row + per_workgroup - 1) / per_workgroup;
    return workgroups < kMaxWorkgroups ? workgroups : 0;
}

// A workgroup per token: its bytes go to the token's rows of the sparse layout.
__global__ __launch_bounds__(kThreads) void dispatch_kernel(const uint8_t *values, const uint8_t *scales, uint8_t *out_values, uint8_t *out_scales,
                                                            const void *sparse_rows, int slots, int64_t sparse_row_count, int64_t value_stride,
                                                            int64_t scale_stride, int vectors, int scale_words, int index_dtype) {
    const int64_t token = blockIdx.x;
    const u32x4_t *from = reinterpret_cast<const u32x4_t *>(values + token * value_stride);
    const uint32_t *from_scales = reinterpret_cast<const uint32_t *>(scales + token * scale_stride);
    for (int i = threadIdx.x; i < vectors + scale_words; i += kThreads) {
        const bool is_value = i < vectors;
        u32x4_t vector = {};
        uint32_t word = 0;
        if (is_value) vector = from[i];
        else word = from_scales[i - vectors];
        for (int j = 0; j < slots; ++j) {
            const int64_t row = load_index(sparse_rows, index_dtype, token * slots + j);
            if (row < 0 || row >= sparse_row_count) continue;
            if (is_value) reinterpret_cast<u32x4_t *>(out_values + row * vectors * 16)[i] = vector;
            else reinterpret_cast<uint32_t *>(out_scales + row * scale_words * 4)[i - vectors] = word;
        }
    }
}

// Rows of up to this many padded columns (and so many bytes of values) are addressed in 32 bits.
constexpr int64_t kMaxColumns = int64_t(1) << 28;

}  // namespace mx

}  // namespace fm

using namespace fm;

extern "C" int fm_mx_quantize(const void *input, void *values, void *scales, int64_t rows, int64_t columns, int64_t input_row_stride, int dtype,
                              int format, void *stream) {
    const char *name = "fm_mx_quantize";
    FM_REQUIRE(valid_dtype(dtype), "%s: bad dtype %d", name, dtype);
    FM_REQUIRE(mx::valid_format(format), "%s: bad format %d", name, format);
    FM_REQUIRE(rows >= 0 && columns > 0 && columns <= mx::kMaxColumns, "%s: bad sizes %lld x %lld", name, static_cast<long long>(rows), static_cast<long long>(columns));
    FM_REQUIRE(rows <= 1 || input_row_stride >= 0, "%s: negative stride", name);
    if (rows == 0) return FM_OK;
    FM_REQUIRE(input && values && scales, "%s: null tensor", name);
    FM_REQUIRE(aligned16(values) && aligned16(scales), "%s: results are 16-byte aligned", name);
    const int64_t padded = mx::padded_columns(columns);
    FM_REQUIRE(reinterpret_cast<uintptr_t>(input) % dtype_size(dtype) == 0, "%s: misaligned input", name);
    const bool whole = columns % 8 == 0 && aligned16(input) && (rows == 1 || input_row_stride * dtype_size(dtype) % 16 == 0);
    if (rows >= (int64_t(1) << 31) || mx::piece_workgroups(rows, padded) == 0) return fail(FM_ERR_UNSUPPORTED, "%s: too large", name);
    FM_DISPATCH_DTYPE(dtype, T, {
        const T *typed = static_cast<const T *>(input);
        uint8_t *value_pointer = static_cast<uint8_t *>(values), *scale_pointer = static_cast<uint8_t *>(scales);
        if (columns >= 8) {
            const auto launch = [&](auto kernel) {
                kernel<<<static_cast<uint32_t>(mx::piece_workgroups(rows, padded)), mx::kThreads, 0, static_cast<hipStream_t>(stream)>>>(
                    typed, value_pointer, scale_pointer, rows, columns, input_row_stride, static_cast<int>(padded));
            };
            if (whole && format == FM_MX_E4M3) launch(mx::quantize_kernel<T, FM_MX_E4M3, true>);
            else if (whole) launch(mx::quantize_kernel<T, FM_MX_E2M1, true>);
            else if (format == FM_MX_E4M3) launch(mx::quantize_kernel<T, FM_MX_E4M3, false>);
            else launch(mx::quantize_kernel<T, FM_MX_E2M1, false>);
        } else {
            const int64_t workgroups = min(rows * ((padded + mx::kThreads - 1) / mx::kThreads), mx::kMaxWorkgroups - 1);
            mx::quantize_any_kernel<T><<<static_cast<uint32_t>(workgroups), mx::kThreads, 0, static_cast<hipStream_t>(stream)>>>(
                typed, value_pointer, scale_pointer, rows, columns, input_row_stride, static_cast<int>(padded), format);
        }
    });
    return check_launch(name);
}

extern "C" int fm_mx_dequantize(const void *values, const void *scales, void *output, int64_t rows, int64_t columns, int64_t value_row_stride,
                                int64_t scale_row_stride, int dtype, int format, void *stream) {
    const char *name = "fm_mx_dequantize";
    FM_REQUIRE(valid_dtype(dtype), "%s: bad dtype %d", name, dtype);
    FM_REQUIRE(mx::valid_format(format), "%s: bad format %d", name, format);
    FM_REQUIRE(rows >= 0 && columns > 0 && columns <= mx::kMaxColumns, "%s: bad sizes %lld x %lld", name, static_cast<long long>(rows), static_cast<long long>(columns));
    if (rows == 0) return FM_OK;
    FM_REQUIRE(values && scales && output, "%s: null tensor", name);
    const int64_t padded = mx::padded_columns(columns);
    FM_REQUIRE(rows == 1 || (value_row_stride >= mx::value_bytes(format, padded) && scale_row_stride >= mx::scale_bytes(padded)), "%s: rows overlap", name);
    FM_REQUIRE(aligned16(values) && (rows == 1 || value_row_stride % 16 == 0), "%s: rows of values are 16-byte aligned", name);
    FM_REQUIRE(reinterpret_cast<uintptr_t>(output) % dtype_size(dtype) == 0, "%s: misaligned output", name);
    const int64_t workgroups = mx::piece_workgroups(rows, columns);
    if (rows >= (int64_t(1) << 31) || workgroups == 0) return fail(FM_ERR_UNSUPPORTED, "%s: too large", name);
    FM_DISPATCH_DTYPE(dtype, T, {
        const auto launch = [&](auto kernel) {
            kernel<<<static_cast<uint32_t>(workgroups), mx::kThreads, 0, static_cast<hipStream_t>(stream)>>>(
                static_cast<const uint8_t *>(values), static_cast<const uint8_t *>(scales), static_cast<T *>(output), rows, columns, value_row_stride,
                scale_row_stride, columns % 8 == 0 && aligned16(output));
        };
        if (format == FM_MX_E4M3) launch(mx::dequantize_kernel<T, FM_MX_E4M3>);
        else launch(mx::dequantize_kernel<T, FM_MX_E2M1>);
    });
    return check_launch(name);
}

extern "C" int fm_mx_copy_dense_to_sparse(const void *values, const void *scales, const void *sparse_rows, void *out_values, void *out_scales,
                                          int64_t num_rows_dense, int64_t columns, int64_t num_experts_per_token, int64_t num_rows_sparse,
                                          int64_t value_row_stride, int64_t scale_row_stride, int format, int index_dtype, void *stream) {
    const char *name = "fm_mx_copy_dense_to_sparse";
    FM_REQUIRE(mx::valid_format(format), "%s: bad format %d", name, format);
    FM_REQUIRE(valid_index_dtype(index_dtype), "%s: bad index dtype %d", name, index_dtype);
    FM_REQUIRE(num_rows_dense >= 0 && num_rows_dense < (int64_t(1) << 31) && columns > 0 && columns <= mx::kMaxColumns && num_experts_per_token > 0 &&
                   num_experts_per_token < (int64_t(1) << 31) && num_rows_sparse >= 0, "%s: bad sizes", name);
    if (num_rows_dense == 0) return FM_OK;
    FM_REQUIRE(values && scales && sparse_rows && ((out_values && out_scales) || num_rows_sparse == 0), "%s: null tensor", name);
    const int64_t padded = mx::padded_columns(columns);
    FM_REQUIRE(num_rows_dense == 1 || (value_row_stride >= mx::value_bytes(format, padded) && scale_row_stride >= mx::scale_bytes(padded)), "%s: rows overlap", name);
    FM_REQUIRE(aligned16(values) && value_row_stride % 16 == 0 && aligned16(out_values), "%s: rows of values are 16-byte aligned", name);
    FM_REQUIRE(reinterpret_cast<uintptr_t>(scales) % 4 == 0 && scale_row_stride % 4 == 0 && aligned16(out_scales), "%s: rows of scales are 4-byte aligned", name);
    if (num_rows_dense >= mx::kMaxWorkgroups) return fail(FM_ERR_UNSUPPORTED, "%s: too large", name);
    mx::dispatch_kernel<<<static_cast<uint32_t>(num_rows_dense), mx::kThreads, 0, static_cast<hipStream_t>(stream)>>>(
        static_cast<const uint8_t *>(values), static_cast<const uint8_t *>(scales), static_cast<uint8_t *>(out_values), static_cast<uint8_t *>(out_scales),
        sparse_rows, static_cast<int>(num_experts_per_token), num_rows_sparse, value_row_stride, scale_row_stride,
        static_cast<int>(mx::value_bytes(format, padded) / 16), static_cast<int>(mx::scale_bytes(padded) / 4), index_dtype);
    return check_launch(name);
}
