// Rows to microscaled values and back, and their dispatch to the sparse layout. All three are bound by memory: nothing is computed
// that does not hide behind it.
#include "fm_mx.h"

namespace fm {

namespace mx {

constexpr int kThreads = 256, kUnroll = 4;

template <typename T>
__device__ __forceinline__ void load_eight(const T *pointer, float (&values)[8]) {
    constexpr int N = Vec16<T>::N;
#pragma unroll
    for (int part = 0; part < 8 / N; ++part) {
        const Vec16<T> vector = load16_stream(pointer + part * N);
#pragma unroll
        for (int i = 0; i < N; ++i) values[part * N + i] = to_float(vector.v[i]);
    }
}

// Eight values per lane: a workgroup takes kUnroll * kThreads consecutive groups of eight of the padded rows.
template <typename T>
__global__ __launch_bounds__(kThreads) void quantize_kernel(const T *input, uint8_t *values, uint8_t *scales, int64_t rows, int64_t columns,
                                                            int64_t input_stride, int padded, int format) {
    const int per_row = padded / 8;
    const int64_t first = static_cast<int64_t>(blockIdx.x) * (kUnroll * kThreads);
    const int64_t first_row = first / per_row;
    const int within = static_cast<int>(first - first_row * per_row);
    float loaded[kUnroll][8];
    int64_t row[kUnroll], column[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
        const uint32_t group = within + u * kThreads + threadIdx.x;
        const uint32_t rows_on = group / static_cast<uint32_t>(per_row);
        row[u] = first_row + rows_on;
        column[u] = static_cast<int64_t>(group - rows_on * per_row) * 8;
#pragma unroll
        for (int i = 0; i < 8; ++i) loaded[u][i] = 0.f;
        if (row[u] < rows && column[u] < columns) load_eight(input + row[u] * input_stride + column[u], loaded[u]);
    }
    const int64_t value_stride = value_bytes(format, padded), scale_stride = scale_bytes(padded);
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
        store_eight(format, loaded[u], values + row[u] * value_stride, scales + row[u] * scale_stride, column[u], row[u] < rows);
}

// Rows whose length or alignment does not allow loads of eight values: a workgroup per row and 256 columns.
template <typename T>
__global__ __launch_bounds__(kThreads) void quantize_any_kernel(const T *input, uint8_t *values, uint8_t *scales, int64_t columns,
                                                                int64_t input_stride, int padded, int format) {
    const int parts = (padded + kThreads - 1) / kThreads;
    const int64_t row = blockIdx.x / parts, column = static_cast<int64_t>(blockIdx.x % parts) * kThreads + threadIdx.x;
    const float value = column < columns ? to_float(input[row * input_stride + column]) : 0.f;
    store_one(format, value, values + row * value_bytes(format, padded), scales + row * scale_bytes(padded), column, column < padded);
}

// The value of an element, exact in fp32.
__device__ __forceinline__ float e2m1_value(uint32_t code) {
    // Magnitude 0 .. 7: e = m >> 1: 0 is subnormal (m / 2), otherwise (1 + (m & 1) / 2) 2^(e - 1).
    const uint32_t m = code & 7u;
    const float size = m < 2u ? 0.5f * static_cast<float>(m) : __builtin_bit_cast(float, (126u + (m >> 1)) << 23 | (m & 1u) << 22);
    return code & 8u ? -size : size;
}

__device__ __forceinline__ float scale_value(uint32_t byte) {
    // 2^-127 is a subnormal number; 255 stands for NaN.
    return byte == 255u ? __builtin_nanf("") : byte == 0u ? __builtin_bit_cast(float, 0x00400000u) : __builtin_bit_cast(float, byte << 23);
}

// Eight values per lane.
template <typename T>
__global__ __launch_bounds__(kThreads) void dequantize_kernel(const uint8_t *values, const uint8_t *scales, T *output, int64_t rows, int64_t columns,
                                                              int64_t value_stride, int64_t scale_stride, int format, int vectors) {
    const int per_row = static_cast<int>((columns + 7) / 8);
    const int64_t first = static_cast<int64_t>(blockIdx.x) * kThreads;
    const int64_t first_row = first / per_row;
    const uint32_t group = static_cast<uint32_t>(first - first_row * per_row) + threadIdx.x, rows_on = group / static_cast<uint32_t>(per_row);
    const int64_t row = first_row + rows_on, column = static_cast<int64_t>(group - rows_on * per_row) * 8;
    if (row >= rows) return;
    const float scale = scale_value(scales[row * scale_stride + column / kBlock]);
    float result[8];
    if (format == FM_MX_E4M3) {
        const u32x2_t words = *reinterpret_cast<const u32x2_t *>(values + row * value_stride + column);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            result[4 * i] = __builtin_amdgcn_cvt_f32_fp8(static_cast<int>(words[i]), 0) * scale;
            result[4 * i + 1] = __builtin_amdgcn_cvt_f32_fp8(static_cast<int>(words[i]), 1) * scale;
            result[4 * i + 2] = __builtin_amdgcn_cvt_f32_fp8(static_cast<int>(words[i]), 2) * scale;
            result[4 * i + 3] = __builtin_amdgcn_cvt_f32_fp8(static_cast<int>(words[i]), 3) * scale;
        }
    } else {
        const uint32_t word = *reinterpret_cast<const uint32_t *>(values + row * value_stride + column / 2);
#pragma unroll
        for (int i = 0; i < 8; ++i) result[i] = e2m1_value(word >> (4 * i)) * scale;
    }
    T *target = output + row * columns + column;
    if (vectors) {
        constexpr int N = Vec16<T>::N;
#pragma unroll
        for (int part = 0; part < 8 / N; ++part) {
            Vec16<T> vector;
#pragma unroll
            for (int i = 0; i < N; ++i) vector.v[i] = from_float<T>(result[part * N + i]);
            store16_stream(target + part * N, vector);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (column + i < columns) target[i] = from_float<T>(result[i]);
    }
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
    const bool vectors = columns % 8 == 0 && aligned16(input) && (rows == 1 || input_row_stride * dtype_size(dtype) % 16 == 0);
    const int64_t parts = (padded + mx::kThreads - 1) / mx::kThreads;
    const int64_t workgroups = vectors ? (rows * (padded / 8) + mx::kUnroll * mx::kThreads - 1) / (mx::kUnroll * mx::kThreads) : rows * parts;
    if (rows >= (int64_t(1) << 40) || workgroups >= (int64_t(1) << 31)) return fail(FM_ERR_UNSUPPORTED, "%s: too large", name);
    FM_DISPATCH_DTYPE(dtype, T, {
        const T *typed = static_cast<const T *>(input);
        uint8_t *value_pointer = static_cast<uint8_t *>(values), *scale_pointer = static_cast<uint8_t *>(scales);
        if (vectors)
            mx::quantize_kernel<T><<<static_cast<uint32_t>(workgroups), mx::kThreads, 0, static_cast<hipStream_t>(stream)>>>(
                typed, value_pointer, scale_pointer, rows, columns, input_row_stride, static_cast<int>(padded), format);
        else
            mx::quantize_any_kernel<T><<<static_cast<uint32_t>(workgroups), mx::kThreads, 0, static_cast<hipStream_t>(stream)>>>(
                typed, value_pointer, scale_pointer, columns, input_row_stride, static_cast<int>(padded), format);
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
    const int64_t workgroups = (rows * ((columns + 7) / 8) + mx::kThreads - 1) / mx::kThreads;
    if (rows >= (int64_t(1) << 40) || workgroups >= (int64_t(1) << 31)) return fail(FM_ERR_UNSUPPORTED, "%s: too large", name);
    FM_DISPATCH_DTYPE(dtype, T, {
        mx::dequantize_kernel<T><<<static_cast<uint32_t>(workgroups), mx::kThreads, 0, static_cast<hipStream_t>(stream)>>>(
            static_cast<const uint8_t *>(values), static_cast<const uint8_t *>(scales), static_cast<T *>(output), rows, columns, value_row_stride,
            scale_row_stride, format, columns % 8 == 0 && aligned16(output));
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
    mx::dispatch_kernel<<<static_cast<uint32_t>(num_rows_dense), mx::kThreads, 0, static_cast<hipStream_t>(stream)>>>(
        static_cast<const uint8_t *>(values), static_cast<const uint8_t *>(scales), static_cast<uint8_t *>(out_values), static_cast<uint8_t *>(out_scales),
        sparse_rows, static_cast<int>(num_experts_per_token), num_rows_sparse, value_row_stride, scale_row_stride,
        static_cast<int>(mx::value_bytes(format, padded) / 16), static_cast<int>(mx::scale_bytes(padded) / 4), index_dtype);
    return check_launch(name);
}
