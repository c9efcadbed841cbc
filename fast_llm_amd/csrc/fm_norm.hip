// Root-mean-square norm with the residual's addition, forward (with its result in microscaled values beside it, for a product with
// quantised weights) and backward.
//
//   s = round(x + r) (the stream that goes on; s = x without a residual),  n = round(s * v * w),  v = 1 / sqrt(mean(s^2) + eps)
//   backward, of the gradients g of n and h of s:  ds = v (g w - s v^2 mean(g w s)) + h  (of x and of r alike),  dw = sum over rows of g s v
//
// What is normalised is the rounded stream, so that the backward needs nothing but it: v is computed again from the row that is in
// registers anyway. All of a row is in the registers of one wavefront (up to 2048 columns), of four or of sixteen (8192, 32768), so each tensor
// passes once: memory is the bound. Sums are in fp32: a lane's own values, then lanes, then wavefronts, in a fixed order. (No row is scaled first, so a sum of
// squares over 3.4e38 gives v = 0: values from 1.8e19 / sqrt(columns) on.)
// Rows whose length is no multiple of 8 or that are not aligned to 16 bytes: the same loads, aligned as the values are, with a last lane that takes the
// row's last eight columns. Rows of less than 8 columns and longer ones: a value per lane and load, the stream read a second time.
//
// Measured at 16384 x 2048 bf16 with a residual: forward 268 MB in 43.1 us (6.2 TB/s), backward 268 MB in 44.3 us and 4.2 us for the sum of 512
// shares of the weight's gradient; with 2047 columns the same within 2 us (a value per lane took 80 and 306 us). (With the loads behind branches, the
// backward without the next row's: 51 and 89 us.) 5001 x 2048 fp16 with e4m3 beside it: 92 MB in 16.3 us.
#include "fm_mx.h"

namespace fm {

namespace norm {

struct Args {
    const void *input, *residual, *weight;
    void *stream, *normalized;
    uint8_t *values, *scales;  // null: no microscaled result
    const void *grad_normalized, *grad_stream;
    void *grad_input;
    float *partials;  // [parts][columns] of the weight's gradient, or null
    int64_t rows;
    int columns, padded, format, weight_f32;
    float eps, inverse_columns;
};

template <typename T>
struct Eight {
    Vec16<T> part[8 / Vec16<T>::N];
    __device__ __forceinline__ float operator[](int i) const { return to_float(part[i / Vec16<T>::N].v[i % Vec16<T>::N]); }
    __device__ __forceinline__ void set(int i, float value) { part[i / Vec16<T>::N].v[i % Vec16<T>::N] = from_float<T>(value); }
};

// The same values, but the compiler cannot tell: it computes them once, as they are stored. (Otherwise it may round a product of fp32 straight to fp16
// for the store and by way of fp32 for what goes on with it.)
template <typename T>
__device__ __forceinline__ void settle(Eight<T> &eight) {
#pragma unroll
    for (int part = 0; part < 8 / Vec16<T>::N; ++part) {
        RawVec16 raw = __builtin_bit_cast(RawVec16, eight.part[part]);
        asm volatile("" : "+v"(raw));
        eight.part[part] = __builtin_bit_cast(Vec16<T>, raw);
    }
}
template <typename T>
__device__ __forceinline__ T settled(T value) {
    asm volatile("" : "+v"(value));
    return value;
}

// A row as a buffer: what is read past its end, or of a row (or a tensor) that does not exist, is zero, without a branch. (Behind
// branches the compiler cannot count which loads are under way and waits for all.)
template <typename T>
__device__ __forceinline__ __amdgpu_buffer_rsrc_t row_of(const void *base, int64_t row, const Args &args) {
    const char *start = static_cast<const char *>(base) + row * args.columns * static_cast<int64_t>(sizeof(T));
    const int bytes = base != nullptr && row < args.rows ? args.columns * static_cast<int>(sizeof(T)) : 0;  // up to 128 KiB
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<char *>(uniform_pointer(start)), 0, __builtin_amdgcn_readfirstlane(bytes), kBufferResourceFlags);
}
template <typename T>
__device__ __forceinline__ Eight<T> load_eight(__amdgpu_buffer_rsrc_t row, int column) {
    Eight<T> eight;
#pragma unroll
    for (int part = 0; part < 8 / Vec16<T>::N; ++part)
        eight.part[part] = __builtin_bit_cast(
            Vec16<T>, __builtin_amdgcn_raw_buffer_load_b128(row, column * static_cast<int>(sizeof(T)) + part * 16, 0, 0));
    return eight;
}
template <typename T>
__device__ __forceinline__ void store_eight(__amdgpu_buffer_rsrc_t row, int column, const Eight<T> &eight) {
    typedef __attribute__((__vector_size__(4 * sizeof(uint32_t)))) uint32_t u32x4_t;
#pragma unroll
    for (int part = 0; part < 8 / Vec16<T>::N; ++part)
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4_t, eight.part[part]), row, column * static_cast<int>(sizeof(T)) + part * 16, 0, 0);
}

// Where the eight columns that a lane has from `column` on are read and written, and how many of them are in front of `column`. Rows that are not
// kWhole, multiples of 8 and aligned to 16 bytes, have a last lane that takes the row's last eight: of what it shares with the lane before it computes and
// writes the same, and counts it in no sum.
constexpr int kNowhere = mx::kNowhere / 4;
template <bool kWhole>
__device__ __forceinline__ int place(int column, int columns) {
    return kWhole ? column : column < columns ? mx::window(column, columns) : kNowhere;
}
template <bool kWhole>
__device__ __forceinline__ int shared(int column, int columns) {
    return kWhole ? 0 : column < columns ? column - mx::window(column, columns) : 0;
}

// The weight, a row of the input's type or fp32, and eight of its columns.
template <typename T>
__device__ __forceinline__ __amdgpu_buffer_rsrc_t weight_row(const Args &args) {
    Args one = args;
    one.rows = 1;
    return args.weight_f32 ? row_of<float>(args.weight, 0, one) : row_of<T>(args.weight, 0, one);
}
template <typename T>
__device__ __forceinline__ void load_weight(const Args &args, __amdgpu_buffer_rsrc_t row, int column, float (&weight)[8]) {
    if (args.weight_f32) {
        const Eight<float> eight = load_eight<float>(row, column);
#pragma unroll
        for (int i = 0; i < 8; ++i) weight[i] = eight[i];
    } else {
        const Eight<T> eight = load_eight<T>(row, column);
#pragma unroll
        for (int i = 0; i < 8; ++i) weight[i] = eight[i];
    }
}

// The sum over a wavefront's lanes in all of them, without LDS: within four, eight, sixteen, then the rows of sixteen and the halves, both
// of which a swap with itself puts side by side.
__device__ __forceinline__ float lane_sum(float value) {
    const auto with = [&](auto control) {
        value += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, value), decltype(control)::value, 0xf, 0xf, true));
    };
    with(std::integral_constant<int, 0xb1>{});   // lanes 1 0 3 2 of every four
    with(std::integral_constant<int, 0x4e>{});   // 2 3 0 1
    with(std::integral_constant<int, 0x141>{});  // the eight mirrored
    with(std::integral_constant<int, 0x140>{});  // the sixteen mirrored
    const uint32_t bits = __builtin_bit_cast(uint32_t, value);
    const auto rows = __builtin_amdgcn_permlane16_swap(bits, bits, false, false);
    value = __builtin_bit_cast(float, static_cast<uint32_t>(rows[0])) + __builtin_bit_cast(float, static_cast<uint32_t>(rows[1]));
    const uint32_t bits_16 = __builtin_bit_cast(uint32_t, value);
    const auto halves = __builtin_amdgcn_permlane32_swap(bits_16, bits_16, false, false);
    return __builtin_bit_cast(float, static_cast<uint32_t>(halves[0])) + __builtin_bit_cast(float, static_cast<uint32_t>(halves[1]));
}

// Sums of kCount values over the kLanes threads of a row, in all of them.
template <int kLanes, int kCount>
__device__ __forceinline__ void row_sum(float (&values)[kCount]) {
#pragma unroll
    for (int c = 0; c < kCount; ++c) values[c] = lane_sum(values[c]);
    if constexpr (kLanes > 64) {
        __shared__ float sums[kCount][kLanes / 64];
        __syncthreads();  // the sums of the row before have been read
        if ((threadIdx.x & 63) == 0)
#pragma unroll
            for (int c = 0; c < kCount; ++c) sums[c][threadIdx.x >> 6] = values[c];
        __syncthreads();
#pragma unroll
        for (int c = 0; c < kCount; ++c) {
            values[c] = sums[c][0];
#pragma unroll
            for (int w = 1; w < kLanes / 64; ++w) values[c] += sums[c][w];
        }
    }
}

__device__ __forceinline__ float inverse_root(const Args &args, float sum_of_squares) {
    return 1.f / sqrtf(sum_of_squares * args.inverse_columns + args.eps);
}

template <int kLanes>
constexpr int kThreads = kLanes < 256 ? 256 : kLanes;

// kLanes threads a row, kVectors times eight columns each: vector v of lane l is the columns 8 (v kLanes + l) .. + 7.
template <typename T, int kLanes, int kVectors, bool kWhole>
__global__ __launch_bounds__(kThreads<kLanes>) void forward_kernel(Args args) {
    const int lane = threadIdx.x % kLanes;
    const int64_t row = static_cast<int64_t>(blockIdx.x) * (kThreads<kLanes> / kLanes) + __builtin_amdgcn_readfirstlane(threadIdx.x / kLanes);
    if (row >= args.rows) return;  // whole wavefronts
    const auto column_of = [&](int v) { return (v * kLanes + lane) * 8; };
    const auto place_of = [&](int v) { return place<kWhole>(column_of(v), args.columns); };
    const auto shared_of = [&](int v) { return shared<kWhole>(column_of(v), args.columns); };
    Eight<T> stream[kVectors];
    const __amdgpu_buffer_rsrc_t input = row_of<T>(args.input, row, args);
#pragma unroll
    for (int v = 0; v < kVectors; ++v) stream[v] = load_eight<T>(input, place_of(v));
    if (args.residual != nullptr) {
        Eight<T> residual[kVectors];
        const __amdgpu_buffer_rsrc_t residual_row = row_of<T>(args.residual, row, args), out = row_of<T>(args.stream, row, args);
#pragma unroll
        for (int v = 0; v < kVectors; ++v) residual[v] = load_eight<T>(residual_row, place_of(v));
#pragma unroll
        for (int v = 0; v < kVectors; ++v) {
#pragma unroll
            for (int i = 0; i < 8; ++i) stream[v].set(i, stream[v][i] + residual[v][i]);
            settle(stream[v]);
            store_eight(out, place_of(v), stream[v]);
        }
    }
    float sum[1] = {0.f};
#pragma unroll
    for (int v = 0; v < kVectors; ++v)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float value = kWhole || i >= shared_of(v) ? stream[v][i] : 0.f;
            sum[0] += value * value;
        }
    row_sum<kLanes>(sum);
    const float inverse = inverse_root(args, sum[0]);
    const __amdgpu_buffer_rsrc_t weights = weight_row<T>(args), out = row_of<T>(args.normalized, row, args);
#pragma unroll
    for (int v = 0; v < kVectors; ++v) {
        float weight[8];
        load_weight<T>(args, weights, place_of(v), weight);
        Eight<T> result;
#pragma unroll
        for (int i = 0; i < 8; ++i) result.set(i, stream[v][i] * inverse * weight[i]);
        settle(result);
        store_eight(out, place_of(v), result);
        if (args.values != nullptr) {
            // Of the rounded result, as its quantisation by itself would be; zeros (not what an infinite root makes of them) behind the row.
            float values[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) values[i] = column_of(v) < args.columns ? result[i] : 0.f;
            if constexpr (!kWhole) mx::shift_down(values, shared_of(v));
            mx::store_eight(args.format, values, args.values + row * mx::value_bytes(args.format, args.padded),
                            args.scales + row * mx::scale_bytes(args.padded), column_of(v), column_of(v) < args.padded);
        }
    }
}

// Rows of less than eight columns and the longest: a workgroup a row, a value a thread.
constexpr int kAnyThreads = 256;

template <typename T>
__global__ __launch_bounds__(kAnyThreads) void forward_any_kernel(Args args) {
    const int64_t row = blockIdx.x, start = row * args.columns;
    const T *input = static_cast<const T *>(args.input) + start, *residual = static_cast<const T *>(args.residual) + start;
    T *stream = static_cast<T *>(args.stream) + start;
    float sum[1] = {0.f};
    for (int column = threadIdx.x; column < args.columns; column += kAnyThreads) {
        float value = to_float(input[column]);
        if (args.residual != nullptr) {
            const T rounded = settled(from_float<T>(value + to_float(residual[column])));
            stream[column] = rounded;
            value = to_float(rounded);
        }
        sum[0] += value * value;
    }
    row_sum<kAnyThreads>(sum);
    const float inverse = inverse_root(args, sum[0]);
    const int end = args.values != nullptr ? (args.padded + kAnyThreads - 1) / kAnyThreads * kAnyThreads : args.columns;
    for (int column = threadIdx.x; column < end; column += kAnyThreads) {
        T result = from_float<T>(0.f);
        if (column < args.columns) {
            // Each thread reads what it has written itself.
            const float value = to_float(args.residual != nullptr ? stream[column] : input[column]);
            const float weight = args.weight_f32 ? static_cast<const float *>(args.weight)[column] : to_float(static_cast<const T *>(args.weight)[column]);
            result = settled(from_float<T>(value * inverse * weight));
            static_cast<T *>(args.normalized)[start + column] = result;
        }
        if (args.values != nullptr)
            mx::store_one(args.format, to_float(result), args.values + row * mx::value_bytes(args.format, args.padded),
                          args.scales + row * mx::scale_bytes(args.padded), column, column < args.padded);
    }
}

// What a row's backward reads.
template <typename T, int kLanes, int kVectors, bool kWhole, bool kGradStream>
struct BackwardRow {
    Eight<T> stream[kVectors], grad[kVectors], grad_stream[kGradStream ? kVectors : 1];
    __device__ __forceinline__ void load(const Args &args, int64_t row, int lane) {
        const __amdgpu_buffer_rsrc_t stream_row = row_of<T>(args.stream, row, args), grad_row = row_of<T>(args.grad_normalized, row, args);
        const __amdgpu_buffer_rsrc_t grad_stream_row = row_of<T>(args.grad_stream, row, args);
#pragma unroll
        for (int v = 0; v < kVectors; ++v) {
            const int column = place<kWhole>((v * kLanes + lane) * 8, args.columns);
            stream[v] = load_eight<T>(stream_row, column);
            grad[v] = load_eight<T>(grad_row, column);
            if constexpr (kGradStream) grad_stream[v] = load_eight<T>(grad_stream_row, column);
        }
    }
};

// A group of kLanes threads walks over rows and keeps its share of the weight's gradient in registers; the groups of a workgroup add
// theirs up in LDS, the workgroups theirs in `weight_gradient_kernel`.
template <typename T, int kLanes, int kVectors, bool kWhole>
__global__ __launch_bounds__(kThreads<kLanes>, kLanes < 1024 ? 2 : 1) void backward_kernel(Args args) {
    constexpr int kGroups = kThreads<kLanes> / kLanes;
    // The next row is asked for before this one is worked on and the weight stays in registers, but where the registers do not hold that (rows of
    // over 1024 or 4096 columns of fp32; 16 wavefronts on a CU): there the weight and the stream's gradient are read when they are needed.
    constexpr bool kAhead = kLanes < 1024 && kVectors * sizeof(T) <= 8;
    using Row = BackwardRow<T, kLanes, kVectors, kWhole, kAhead>;
    const int lane = threadIdx.x % kLanes, group = __builtin_amdgcn_readfirstlane(threadIdx.x / kLanes);
    const int64_t step = static_cast<int64_t>(gridDim.x) * kGroups;
    const auto place_of = [&](int v) { return place<kWhole>((v * kLanes + lane) * 8, args.columns); };
    const auto shared_of = [&](int v) { return shared<kWhole>((v * kLanes + lane) * 8, args.columns); };
    const __amdgpu_buffer_rsrc_t weight_buffer = weight_row<T>(args);
    float weight_grad[kVectors][8], weights[kAhead ? kVectors : 1][8];
#pragma unroll
    for (int v = 0; v < kVectors; ++v)
#pragma unroll
        for (int i = 0; i < 8; ++i) weight_grad[v][i] = 0.f;
    int64_t row = static_cast<int64_t>(blockIdx.x) * kGroups + group;
    Row current, next;
    if constexpr (kAhead) {
        current.load(args, row, lane);
#pragma unroll
        for (int v = 0; v < kVectors; ++v) {
            load_weight<T>(args, weight_buffer, place_of(v), weights[v]);
        }
    }
    for (; row < args.rows; row += step) {
        if constexpr (kAhead) next.load(args, row + step, lane);
        else current.load(args, row, lane);
        auto &stream = current.stream;
        auto &grad = current.grad;
        const __amdgpu_buffer_rsrc_t out = row_of<T>(args.grad_input, row, args);
        float sums[2] = {0.f, 0.f};  // of s^2 and of g w s
#pragma unroll
        for (int v = 0; v < kVectors; ++v) {
            float read[8];
            if constexpr (!kAhead) load_weight<T>(args, weight_buffer, place_of(v), read);
            const float(&weight)[8] = kAhead ? weights[kAhead ? v : 0] : read;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const bool counts = kWhole || i >= shared_of(v);
                sums[0] += counts ? stream[v][i] * stream[v][i] : 0.f;
                sums[1] += counts ? grad[v][i] * weight[i] * stream[v][i] : 0.f;
            }
        }
        row_sum<kLanes>(sums);
        const float inverse = inverse_root(args, sums[0]), factor = inverse * inverse * sums[1] * args.inverse_columns;
        // Kept in their own type meanwhile, not widened.
#pragma unroll
        for (int v = 0; v < kVectors; ++v) settle(stream[v]), settle(grad[v]);
#pragma unroll
        for (int v = 0; v < kVectors; ++v) {
            float read[8];
            if constexpr (!kAhead) {
                load_weight<T>(args, weight_buffer, place_of(v), read);
                current.grad_stream[0] = load_eight<T>(row_of<T>(args.grad_stream, row, args), place_of(v));
            }
            const float(&weight)[8] = kAhead ? weights[kAhead ? v : 0] : read;
            Eight<T> result;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                result.set(i, inverse * (grad[v][i] * weight[i] - stream[v][i] * factor) + current.grad_stream[kAhead ? v : 0][i]);
                weight_grad[v][i] += grad[v][i] * (stream[v][i] * inverse);
            }
            store_eight(out, place_of(v), result);
        }
        if constexpr (kAhead) current = next;
    }
    if (args.partials == nullptr) return;
    float *target = args.partials + static_cast<int64_t>(blockIdx.x) * args.columns;
    if constexpr (!kWhole)
#pragma unroll
        for (int v = 0; v < kVectors; ++v) mx::shift_down(weight_grad[v], shared_of(v));
    if constexpr (kGroups == 1) {
#pragma unroll
        for (int v = 0; v < kVectors; ++v) {
            const int column = (v * kLanes + lane) * 8;
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (kWhole ? column < args.columns : column + i < args.columns) target[column + i] = weight_grad[v][i];
        }
    } else {
        __shared__ float shared[kGroups][kLanes * 8];
#pragma unroll
        for (int v = 0; v < kVectors; ++v) {
            __syncthreads();
#pragma unroll
            for (int i = 0; i < 8; ++i) shared[group][i * kLanes + lane] = weight_grad[v][i];
            __syncthreads();
            for (int at = threadIdx.x; at < kLanes * 8; at += kThreads<kLanes>) {
                const int column = v * kLanes * 8 + at, from = at % 8 * kLanes + at / 8;
                float sum = shared[0][from];
#pragma unroll
                for (int g = 1; g < kGroups; ++g) sum += shared[g][from];
                if (column < args.columns) target[column] = sum;
            }
        }
    }
}

// Rows of less than eight columns and the longest. The weight's gradient: a workgroup's share is in its row of `partials` from the first row on, each value
// written and read by one thread.
template <typename T>
__global__ __launch_bounds__(kAnyThreads) void backward_any_kernel(Args args) {
    float *target = args.partials + static_cast<int64_t>(blockIdx.x) * args.columns;
    bool first = true;
    for (int64_t row = blockIdx.x; row < args.rows; row += gridDim.x) {
        const int64_t start = row * args.columns;
        const T *stream = static_cast<const T *>(args.stream) + start, *grad = static_cast<const T *>(args.grad_normalized) + start;
        const T *grad_stream = static_cast<const T *>(args.grad_stream) + start;
        const auto weight_at = [&](int column) {
            return args.weight_f32 ? static_cast<const float *>(args.weight)[column] : to_float(static_cast<const T *>(args.weight)[column]);
        };
        float sums[2] = {0.f, 0.f};
        for (int column = threadIdx.x; column < args.columns; column += kAnyThreads) {
            const float s = to_float(stream[column]);
            sums[0] += s * s;
            sums[1] += to_float(grad[column]) * weight_at(column) * s;
        }
        row_sum<kAnyThreads>(sums);
        const float inverse = inverse_root(args, sums[0]), factor = inverse * inverse * sums[1] * args.inverse_columns;
        for (int column = threadIdx.x; column < args.columns; column += kAnyThreads) {
            const float s = to_float(stream[column]), g = to_float(grad[column]);
            const float more = args.grad_stream != nullptr ? to_float(grad_stream[column]) : 0.f;
            static_cast<T *>(args.grad_input)[start + column] = from_float<T>(inverse * (g * weight_at(column) - s * factor) + more);
            if (args.partials != nullptr) target[column] = (first ? 0.f : target[column]) + g * (s * inverse);
        }
        first = false;
    }
}

// 16 columns a workgroup, 64 threads each that take every 64th part.
constexpr int kReduceColumns = 16, kReduceThreads = 1024;

template <typename T>
__global__ __launch_bounds__(kReduceThreads) void weight_gradient_kernel(const float *partials, T *out, int columns, int parts) {
    __shared__ float sums[kReduceThreads / kReduceColumns][kReduceColumns + 1];
    const int within = threadIdx.x % kReduceColumns, part = threadIdx.x / kReduceColumns, column = blockIdx.x * kReduceColumns + within;
    float sum = 0.f;
    if (column < columns)
        for (int p = part; p < parts; p += kReduceThreads / kReduceColumns) sum += partials[static_cast<int64_t>(p) * columns + column];
    sums[part][within] = sum;
#pragma unroll
    for (int width = kReduceThreads / kReduceColumns / 2; width > 0; width /= 2) {
        __syncthreads();
        if (part < width) sums[part][within] += sums[part + width][within];
    }
    if (part == 0 && column < columns) out[column] = from_float<T>(sums[0][within]);
}

constexpr int64_t kMaxColumns = int64_t(1) << 28;
constexpr int kMaxParts = 512;

// Threads of a row, 0: `..._any_kernel`.
static int lanes_of(int64_t columns) {
    if (columns < 8 || columns > 32768) return 0;
    return columns <= 2048 ? 64 : columns <= 8192 ? 256 : 1024;
}

// Workgroups of a backward: what two per CU hold, walking over the rows.
static int64_t parts_of(int64_t rows, int64_t columns) {
    const int64_t at_once = columns <= 2048 ? 4 : 1;
    return min((rows + at_once - 1) / at_once, static_cast<int64_t>(kMaxParts));
}

template <typename Launch>
static void for_shape(int columns, int lanes, bool whole, Launch launch) {
    const auto with = [&](auto lanes_constant, auto vectors) {
        if (whole) launch(lanes_constant, vectors, std::true_type{});
        else launch(lanes_constant, vectors, std::false_type{});
    };
    if (lanes == 64 && columns <= 512) with(std::integral_constant<int, 64>{}, std::integral_constant<int, 1>{});
    else if (lanes == 64 && columns <= 1024) with(std::integral_constant<int, 64>{}, std::integral_constant<int, 2>{});
    else if (lanes == 64) with(std::integral_constant<int, 64>{}, std::integral_constant<int, 4>{});
    else if (lanes == 256 && columns <= 4096) with(std::integral_constant<int, 256>{}, std::integral_constant<int, 2>{});
    else if (lanes == 256) with(std::integral_constant<int, 256>{}, std::integral_constant<int, 4>{});
    else with(std::integral_constant<int, 1024>{}, std::integral_constant<int, 4>{});
}

}  // namespace norm

}  // namespace fm

using namespace fm;

static int check_norm(const char *name, int64_t rows, int64_t columns, double eps, int dtype, int weight_dtype) {
    FM_REQUIRE(valid_dtype(dtype), "%s: bad dtype %d", name, dtype);
    FM_REQUIRE(weight_dtype == dtype || weight_dtype == FM_DTYPE_F32, "%s: bad weight dtype %d: the input's or fp32", name, weight_dtype);
    FM_REQUIRE(rows >= 0 && rows < (int64_t(1) << 31) && columns > 0 && columns <= norm::kMaxColumns, "%s: bad sizes %lld x %lld", name,
               static_cast<long long>(rows), static_cast<long long>(columns));
    FM_REQUIRE(eps >= 0., "%s: negative eps", name);
    return FM_OK;
}

extern "C" int fm_rms_norm_forward(const void *input, const void *residual, const void *weight, void *stream_out, void *normalized, void *values,
                                   void *scales, int64_t rows, int64_t columns, double eps, int dtype, int weight_dtype, int format, void *stream) {
    const char *name = "fm_rms_norm_forward";
    if (int status = check_norm(name, rows, columns, eps, dtype, weight_dtype)) return status;
    FM_REQUIRE((values == nullptr) == (scales == nullptr), "%s: microscaled values and scales come together", name);
    FM_REQUIRE(values == nullptr || mx::valid_format(format), "%s: bad format %d", name, format);
    if (rows == 0) return FM_OK;
    FM_REQUIRE(input && weight && normalized, "%s: null tensor", name);
    FM_REQUIRE((residual == nullptr) == (stream_out == nullptr), "%s: the residual and the stream that goes on come together", name);
    FM_REQUIRE(normalized != input && normalized != residual && stream_out != input && (stream_out == nullptr || stream_out != residual) && normalized != stream_out,
               "%s: a result in place of an input", name);
    FM_REQUIRE(values == nullptr || (aligned16(values) && aligned16(scales)), "%s: microscaled results are 16-byte aligned", name);
    const bool whole = columns % 8 == 0 && aligned16(input) && aligned16(residual) && aligned16(weight) && aligned16(stream_out) && aligned16(normalized);
    const int lanes = norm::lanes_of(columns);
    norm::Args args{};
    args.weight = weight, args.columns = static_cast<int>(columns), args.padded = static_cast<int>(mx::padded_columns(columns)), args.format = format;
    args.weight_f32 = weight_dtype == FM_DTYPE_F32 && dtype != FM_DTYPE_F32;
    args.eps = static_cast<float>(eps), args.inverse_columns = static_cast<float>(1. / static_cast<double>(columns));
    // A launch counts its threads in 32 bits: up to 1024 per row.
    constexpr int64_t kRowsAtOnce = (int64_t(1) << 22) - 4;
    const auto past = [](const void *pointer, int64_t bytes) { return pointer == nullptr ? nullptr : const_cast<char *>(static_cast<const char *>(pointer)) + bytes; };
    for (int64_t row = 0; row < rows; row += kRowsAtOnce) {
        const int64_t bytes = row * columns * dtype_size(dtype);
        args.input = past(input, bytes), args.residual = past(residual, bytes), args.stream = past(stream_out, bytes), args.normalized = past(normalized, bytes);
        args.values = reinterpret_cast<uint8_t *>(past(values, row * mx::value_bytes(format, args.padded)));
        args.scales = reinterpret_cast<uint8_t *>(past(scales, row * mx::scale_bytes(args.padded)));
        args.rows = min(rows - row, kRowsAtOnce);
        FM_DISPATCH_DTYPE(dtype, T, {
            if (lanes == 0) {
                norm::forward_any_kernel<T><<<static_cast<uint32_t>(args.rows), norm::kAnyThreads, 0, static_cast<hipStream_t>(stream)>>>(args);
            } else {
                norm::for_shape(static_cast<int>(columns), lanes, whole, [&](auto lanes_constant, auto vectors, auto whole_constant) {
                    constexpr int kLanes = decltype(lanes_constant)::value, kRows = norm::kThreads<kLanes> / kLanes;
                    norm::forward_kernel<T, kLanes, decltype(vectors)::value, decltype(whole_constant)::value>
                        <<<static_cast<uint32_t>((args.rows + kRows - 1) / kRows), norm::kThreads<kLanes>, 0, static_cast<hipStream_t>(stream)>>>(args);
                });
            }
        });
    }
    return check_launch(name);
}

extern "C" size_t fm_rms_norm_backward_workspace_size(int64_t rows, int64_t columns) {
    if (rows <= 0 || columns <= 0 || columns > norm::kMaxColumns) return 0;
    return static_cast<size_t>(norm::parts_of(rows, columns)) * columns * sizeof(float);
}

extern "C" int fm_rms_norm_backward(const void *grad_normalized, const void *grad_stream, const void *stream_in, const void *weight, void *grad_input,
                                    void *grad_weight, int64_t rows, int64_t columns, double eps, int dtype, int weight_dtype, void *workspace,
                                    size_t workspace_size, void *stream) {
    const char *name = "fm_rms_norm_backward";
    if (int status = check_norm(name, rows, columns, eps, dtype, weight_dtype)) return status;
    const size_t needed = fm_rms_norm_backward_workspace_size(rows, columns);
    if (rows > 0) {
        FM_REQUIRE(grad_normalized && stream_in && weight && grad_input, "%s: null tensor", name);
        FM_REQUIRE(grad_input != grad_normalized && grad_input != grad_stream && grad_input != stream_in, "%s: a result in place of an input", name);
        FM_REQUIRE(grad_weight == nullptr || (workspace && aligned16(workspace) && workspace_size >= needed),
                   "%s: workspace of %zu bytes (16-byte aligned) needed, got %zu", name, needed, workspace_size);
    }
    norm::Args args{};
    args.stream = const_cast<void *>(stream_in), args.weight = weight, args.grad_normalized = grad_normalized, args.grad_stream = grad_stream;
    args.grad_input = grad_input, args.partials = grad_weight != nullptr ? static_cast<float *>(workspace) : nullptr;
    args.rows = rows, args.columns = static_cast<int>(columns);
    args.weight_f32 = weight_dtype == FM_DTYPE_F32 && dtype != FM_DTYPE_F32;
    args.eps = static_cast<float>(eps), args.inverse_columns = static_cast<float>(1. / static_cast<double>(columns));
    const bool whole = columns % 8 == 0 && aligned16(grad_normalized) && aligned16(grad_stream) && aligned16(stream_in) && aligned16(weight) && aligned16(grad_input);
    const int lanes = norm::lanes_of(columns);
    // Without rows the weight's gradient is the sum of nothing.
    const uint32_t parts = rows > 0 ? static_cast<uint32_t>(norm::parts_of(rows, columns)) : 0;
    if (rows > 0) {
        FM_DISPATCH_DTYPE(dtype, T, {
            if (lanes == 0) {
                norm::backward_any_kernel<T><<<parts, norm::kAnyThreads, 0, static_cast<hipStream_t>(stream)>>>(args);
            } else {
                norm::for_shape(static_cast<int>(columns), lanes, whole, [&](auto lanes_constant, auto vectors, auto whole_constant) {
                    constexpr int kLanes = decltype(lanes_constant)::value;
                    norm::backward_kernel<T, kLanes, decltype(vectors)::value, decltype(whole_constant)::value>
                        <<<parts, norm::kThreads<kLanes>, 0, static_cast<hipStream_t>(stream)>>>(args);
                });
            }
        });
    }
    if (grad_weight != nullptr) {
        const uint32_t workgroups = static_cast<uint32_t>((columns + norm::kReduceColumns - 1) / norm::kReduceColumns);
        FM_DISPATCH_DTYPE(weight_dtype, W, {
            norm::weight_gradient_kernel<W><<<workgroups, norm::kReduceThreads, 0, static_cast<hipStream_t>(stream)>>>(
                args.partials, static_cast<W *>(grad_weight), static_cast<int>(columns), static_cast<int>(parts));
        });
    }
    return check_launch(name);
}
