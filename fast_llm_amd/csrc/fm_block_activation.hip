// The MLP's activation between products of 8 bits: forward into the second layer's rows and a checkpoint of the input, both of 8 bits; backward from
// that checkpoint into what the remaining products read: the input's gradient along its rows and its columns, and the forward's result along its
// columns.
//
// Both are one pass over their operands and no 16-bit copy leaves them. 98304 rows of 2 x 1408 in bf16: forward 204 us at 4.9 TB/s, backward 360 at
// 3.6 (two workgroups per CU; with one 540). The forward is bound by memory. Of the backward every element has four conversions and the slope of the
// activation, so that memory and arithmetic weigh about the same; a lane keeps its three results (gate's and up's gradient, output) in registers
// between the two directions of quantisation, eight rows x four columns of each.
#include "fm_activation_math.h"
#include "fm_block_rows.h"

namespace fm {

namespace block {

// What values of a type are activated in. A step in fp32 is 2^-24 of a value, and it is a border of e4m3 that decides: fp32 goes by fp64, and of 1.5
// million values none is off, where hardware functions in fp32 leave four and library functions in fp32 forty. Silu of 98304 rows of 2 x 1408:
// forward 305 us for 290, backward 740 for 385. What was rounded to 16 bits has hardware exponentials and reciprocals of fp32.
template <typename T>
struct ActivatedIn { typedef float Real; };
template <>
struct ActivatedIn<float> { typedef double Real; };

// sigma(x) and 1 - sigma(x). Where gelu's argument is, a third power, the complement is e^-x of sigma, of which nothing is lost beside 1, and the
// exponent's own rounding, up to 2^-24 of as many units as it has, is made good: without that 1200 bf16 rows of 2 x 1408 have 150 gradients on the
// other side of a border, with it 110 (of fp32 in library functions 180). For silu it makes no difference, and 98304 such rows take 602 us there and
// back instead of 566.
template <bool kFine>
__device__ __forceinline__ float sigmoid(float x, float &complement) {
    if constexpr (!kFine) {
        const float sigma = fast_rcp(1.f + fast_exp(-x));
        complement = 1.f - sigma;
        return sigma;
    }
    const float bounded = fmaxf(x, -88.f), exponent = bounded * -1.44269502f;
    const float rest = fmaf(bounded, -1.925963033e-8f, fmaf(bounded, -1.44269502f, -exponent));
    float power = __builtin_amdgcn_exp2f(exponent);
    power = fmaf(power, rest * 0.693147182f, power);
    const float sigma = x < -88.f ? 0.f : fast_rcp(1.f + power);
    complement = power * sigma;
    return sigma;
}
// In fp64, to 2^-36 of itself: e^-x = 2^n e^g with |g| <= ln(2) / 2 by Taylor's series up to g^9, and a step of Newton's from the hardware's
// reciprocal. (Beyond 2^+-1000 nothing changes in fp32.)
template <bool kFine>
__device__ __forceinline__ double sigmoid(double x, double &complement) {
    double t = x * -1.4426950408889634;
    t = t > 1000. ? 1000. : t < -1000. ? -1000. : t;
    const double n = rint(t), g = (t - n) * 0.69314718055994531;
    double power = 1. / 362880;
#pragma unroll
    for (int k = 9; k > 0; --k) {
        constexpr double kInverse[] = {1., 1., 1. / 2, 1. / 6, 1. / 24, 1. / 120, 1. / 720, 1. / 5040, 1. / 40320};
        power = fma(power, g, kInverse[k - 1]);
    }
    power = ldexp(power, static_cast<int>(n));
    const double inverse = 1. + power, guess = __builtin_amdgcn_rcp(inverse), sigma = guess * fma(-inverse, guess, 2.);
    complement = power * sigma;
    return sigma;
}

// act(x), and act'(x) for the backward. Gelu (in its tanh form) and silu are x times a sigmoid, which has no cancellation where it is small: x
// sigma(z), with the slope sigma + x sigma (1 - sigma) z'.
template <int kActivation, typename Real>
__device__ __forceinline__ Real activate(Real x, Real &slope) {
    if constexpr (kActivation == FM_ACT_GELU || kActivation == FM_ACT_SILU) {
        Real z = x, z_slope = 1;
        if constexpr (kActivation == FM_ACT_GELU) {
            // (Beyond 100 it is x or 0, whose powers would overflow.)
            const Real bounded = x > 100 ? static_cast<Real>(100) : x < -100 ? static_cast<Real>(-100) : x;
            const Real square = bounded * bounded, linear = static_cast<Real>(1.5957691216057308), cubic = static_cast<Real>(0.071354816272600254);
            z = bounded * (linear + cubic * square);
            z_slope = linear + 3 * cubic * square;
        }
        Real complement, sigma = sigmoid<kActivation == FM_ACT_GELU>(z, complement);
        // Gelu is that of the other activation kernels, x / 2 times 1 + tanh in fp32: zero from where this sum is, which a block with no larger value
        // shows. (Above, where the sum has few bits left, a sigmoid has all of them.)
        if constexpr (kActivation == FM_ACT_GELU) sigma = sigma < static_cast<Real>(0x1p-26) ? 0 : sigma;
        const Real out = x * sigma;
        slope = sigma + out * complement * z_slope;
        return out;
    }
    // NaN is no number that either comparison lets go: it stays, in the slope as well.
    const Real positive = kActivation != FM_ACT_IDENTITY && x <= 0 ? 0 : x;
    slope = kActivation == FM_ACT_SQUARED_RELU ? 2 * positive : kActivation == FM_ACT_IDENTITY || x > 0 ? 1 : positive;
    return kActivation == FM_ACT_SQUARED_RELU ? positive * positive : positive;
}

// As fp32 in front of a rounding to fewer bits: what fp32 does not have leaves its last bit odd, so that no value comes to lie on a border that it is
// next to.
__device__ __forceinline__ float before_rounding(float value) { return value; }
__device__ __forceinline__ float before_rounding(double value) {
    const float nearest = static_cast<float>(value);
    const double rest = value - static_cast<double>(nearest);
    const uint32_t bits = __builtin_bit_cast(uint32_t, nearest);
    const bool between = rest != 0. && (bits & 1) == 0 && (bits & 0x7f800000u) != 0x7f800000u;
    // (Away from zero where the rest has the value's sign.)
    return __builtin_bit_cast(float, between ? ((rest < 0.) == ((bits >> 31) != 0) ? bits + 1 : bits - 1) : bits);
}

struct ActivationArgs {
    const void *input;                    // forward
    const void *grad_output;              // backward
    uint8_t *checkpoint, *checkpoint_scales;
    uint8_t *output, *output_scales;      // backward: transposed
    uint8_t *grad, *grad_scales, *grad_transposed, *grad_transposed_scales;
    int64_t rows, columns;                // of the result
    int64_t input_stride, grad_output_stride, checkpoint_stride, checkpoint_scale_stride, output_stride, output_scale_stride, grad_stride, grad_scale_stride,
        transposed_stride, transposed_scale_stride;
    uint32_t column_blocks;
    RowMap map;
};

template <typename T, int kActivation, bool kGated>
__global__ __launch_bounds__(kRowThreads) void activation_forward_kernel(ActivationArgs args) {
    typedef typename ActivatedIn<T>::Real Real;
    const uint32_t column_block = blockIdx.x % args.column_blocks;
    const int64_t row0 = static_cast<int64_t>(blockIdx.x / args.column_blocks) * kBlock, column0 = static_cast<int64_t>(column_block) * kBlock;
    const int count = rows_in_block(args.map, row0, args.rows), exist = static_cast<int>(min(args.rows - row0, static_cast<int64_t>(kBlock)));
    const int columns = static_cast<int>(min(args.columns - column0, static_cast<int64_t>(kBlock))), first_row = threadIdx.x / 8, column = threadIdx.x % 8 * 16;
    const T *input = static_cast<const T *>(args.input) + row0 * args.input_stride + column0;
    uint8_t *output = args.output + row0 * args.output_stride + column0, *output_scales = args.output_scales + column_block * args.output_scale_stride + row0;
    uint8_t *checkpoint = args.checkpoint + row0 * args.checkpoint_stride + column0, *scales = args.checkpoint_scales + column_block * args.checkpoint_scale_stride + row0;
    // Two rows of a lane at a time.
#pragma unroll 1
    for (int begin = 0; begin < kBlock; begin += kRowThreads / 4) {
        Raw<T, 16> gates[2], ups[2];
        const uint32_t stride = static_cast<uint32_t>(args.input_stride);
        load_block<2, kRowThreads / 8>(input, stride, begin + first_row, column, exist, count, columns, gates);
        if constexpr (kGated) load_block<2, kRowThreads / 8>(input + args.columns, stride, begin + first_row, column, exist, count, columns, ups);
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const uint32_t row = begin + first_row + r * (kRowThreads / 8);
            const bool exists = static_cast<int>(row) < exist;
            float gate[16], up[16], result[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                gate[i] = to_float(gates[r].v[i]);
                Real slope, out = activate<kActivation, Real>(gate[i], slope);
                if constexpr (kGated) up[i] = to_float(ups[r].v[i]), out *= up[i];
                result[i] = before_rounding(out);
            }
            const uint32_t at = row * static_cast<uint32_t>(args.checkpoint_stride) + column;
            store_row(gate, checkpoint + at, scales + row, exists);
            // (Gated: whole blocks of columns.)
            if constexpr (kGated) store_row(up, checkpoint + args.columns + at, scales + args.column_blocks * args.checkpoint_scale_stride + row, exists);
            store_row(result, output + (row * static_cast<uint32_t>(args.output_stride) + column), output_scales + row, exists);
        }
    }
}

// The same values, but the compiler cannot tell.
template <typename T>
__device__ __forceinline__ void kept_apart(Raw<T, 4> &four) {
    typedef __attribute__((__vector_size__(4 * sizeof(T)))) uint32_t Words;
    Words words = __builtin_bit_cast(Words, four);
    asm volatile("" : "+v"(words));
    four = __builtin_bit_cast(Raw<T, 4>, words);
}

// At most 128 registers, for two workgroups on a CU: gates, ups and gradients stay as they were read, and the results are made one after the other.
template <typename T, int kActivation, bool kGated>
__global__ __launch_bounds__(kSquareThreads, sizeof(T) == 4 ? 2 : 4) void activation_backward_kernel(ActivationArgs args) {
    typedef typename ActivatedIn<T>::Real Real;
    __shared__ __attribute__((aligned(16))) Square shared;
    const uint32_t column_block = blockIdx.x % args.column_blocks;
    const int64_t row_block = blockIdx.x / args.column_blocks, row0 = row_block * kBlock, column0 = static_cast<int64_t>(column_block) * kBlock;
    const int cg = threadIdx.x & 31, row_group = threadIdx.x >> 5;
    const int exist = static_cast<int>(min(args.rows - row0, static_cast<int64_t>(kBlock))), count = rows_in_block(args.map, row0, args.rows);
    const int columns = static_cast<int>(min(args.columns - column0, static_cast<int64_t>(kBlock)));
    const T *grad_output = static_cast<const T *>(args.grad_output) + row0 * args.grad_output_stride + column0;
    const uint8_t *gate_from = args.checkpoint + row0 * args.checkpoint_stride + column0, *up_from = gate_from + args.columns;
    const uint8_t *gate_scales_from = args.checkpoint_scales + column_block * args.checkpoint_scale_stride + row0;
    const uint8_t *up_scales_from = gate_scales_from + args.column_blocks * args.checkpoint_scale_stride;
    const uint32_t grad_stride = static_cast<uint32_t>(args.grad_output_stride), checkpoint_stride = static_cast<uint32_t>(args.checkpoint_stride);
    const int first_row = row_group * kLaneRows, first_column = cg * kLaneColumns;
    Raw<T, kLaneColumns> grad[kLaneRows];
    load_block<kLaneRows, 1>(grad_output, grad_stride, first_row, first_column, exist, count, columns, grad);
    // In fp64 it is arithmetic that counts: the ups' gradients are kept from the first time.
    constexpr bool kOnce = sizeof(T) == 4;
    float values[kLaneRows][kLaneColumns], output[kLaneRows][kLaneColumns], up_grad[kOnce ? kLaneRows : 1][kLaneColumns];
    uint32_t gates[kLaneRows], ups[kLaneRows];
#pragma unroll
    for (int r = 0; r < kLaneRows; ++r) {
        const uint32_t at = min(first_row + r, exist - 1) * checkpoint_stride + first_column;
        gates[r] = *reinterpret_cast<const uint32_t *>(gate_from + at);
        if constexpr (kGated) ups[r] = *reinterpret_cast<const uint32_t *>(up_from + at);
    }
    // A byte for each row. (Scales are padded to whole pieces of sixteen rows.)
    const int scale_row = min(first_row, (exist - 1) & ~7);
    uint64_t gate_scales = *reinterpret_cast<const uint64_t *>(gate_scales_from + scale_row), up_scales = 0;
    if constexpr (kGated) up_scales = *reinterpret_cast<const uint64_t *>(up_scales_from + scale_row);
    if (count < kBlock) {
        // Zeros, whatever the checkpoint holds for rows that do not count.
        const int counting = min(max(count - first_row, 0), kLaneRows);
        const uint64_t bytes = counting > 0 ? ~uint64_t(0) >> (kLaneRows - counting) * 8 : 0;
        gate_scales &= bytes, up_scales &= bytes;
#pragma unroll
        for (int r = 0; r < kLaneRows; ++r) {
            gates[r] = r < counting ? gates[r] : 0u;
            if constexpr (kGated) ups[r] = r < counting ? ups[r] : 0u;
        }
    }
    const auto scale_of = [](uint64_t scales, int r) { return scale_value(static_cast<uint32_t>(scales >> r * 8) & 255u); };
#pragma unroll
    for (int r = 0; r < kLaneRows; ++r) {
        __builtin_amdgcn_sched_barrier(0);  // one row's values at a time: registers
        float gate[kLaneColumns], up[kLaneColumns];
        unpack_four(gates[r], scale_of(gate_scales, r), gate);
        if constexpr (kGated) unpack_four(ups[r], scale_of(up_scales, r), up);
#pragma unroll
        for (int c = 0; c < kLaneColumns; ++c) {
            Real slope;
            const Real out = activate<kActivation, Real>(gate[c], slope);
            const Real of_result = to_float(grad[r].v[c]);
            if constexpr (!kGated) output[r][c] = before_rounding(out);
            else if constexpr (kOnce) output[r][c] = before_rounding(out * up[c]), up_grad[r][c] = before_rounding(out * of_result);
            // (The product of an up, of 4 bits, and a gradient of 16 is exact in fp32.)
            values[r][c] = before_rounding(slope * (kGated ? up[c] * of_result : of_result));
        }
    }
    __builtin_amdgcn_sched_barrier(0);
    const int64_t t_scales = row_block * args.transposed_scale_stride;
    const auto store_gradient = [&](int part) {
        const int64_t from_column = column0 + part * args.columns;
        store_square<true>(values, shared, args.grad + row0 * args.grad_stride + from_column, static_cast<uint32_t>(args.grad_stride),
                           args.grad_scales + (column_block + part * args.column_blocks) * args.grad_scale_stride + row0, exist,
                           args.grad_transposed + from_column * args.transposed_stride + row0, args.transposed_stride, args.grad_transposed_scales + t_scales + from_column, columns);
    };
    store_gradient(0);
    if constexpr (kGated) {
#pragma unroll
        for (int r = 0; r < kLaneRows; ++r) {
            __builtin_amdgcn_sched_barrier(0);
            if constexpr (kOnce) {
#pragma unroll
                for (int c = 0; c < kLaneColumns; ++c) values[r][c] = up_grad[r][c];
                continue;
            }
            // (Activated again: what there was above would not fit the registers until here.)
            float gate[kLaneColumns], up[kLaneColumns];
            asm volatile("" : "+v"(gates[r]), "+v"(ups[r]));
            unpack_four(gates[r], scale_of(gate_scales, r), gate);
            unpack_four(ups[r], scale_of(up_scales, r), up);
            kept_apart(grad[r]);
#pragma unroll
            for (int c = 0; c < kLaneColumns; ++c) {
                Real slope;
                const Real out = activate<kActivation, Real>(gate[c], slope);
                values[r][c] = before_rounding(out * to_float(grad[r].v[c])), output[r][c] = before_rounding(out * up[c]);
            }
        }
        store_gradient(1);
    }
    store_square<false>(output, shared, nullptr, 0, nullptr, 0, args.output + column0 * args.output_stride + row0, args.output_stride,
                        args.output_scales + row_block * args.output_scale_stride + column0, columns);
}

template <typename T, bool kGated>
static void launch_activation(bool forward, int activation, const ActivationArgs &args, uint32_t grid, hipStream_t stream) {
    FM_DISPATCH_ACTIVATION(activation, kActivation, {
        if (forward) activation_forward_kernel<T, kActivation, kGated><<<grid, kRowThreads, 0, stream>>>(args);
        else activation_backward_kernel<T, kActivation, kGated><<<grid, kSquareThreads, 0, stream>>>(args);
    });
}

// Checks and launch of both directions; `args` without what is computed here.
static int run_activation(const char *name, bool forward, ActivationArgs args, const void *expert_ends, const void *expert_pad_begins, int64_t num_experts, int gated,
                          int activation, int dtype, int index_dtype, void *stream) {
    FM_REQUIRE(valid_dtype(dtype), "%s: bad dtype %d", name, dtype);
    FM_REQUIRE(activation >= FM_ACT_GELU && activation <= FM_ACT_IDENTITY, "%s: bad activation %d", name, activation);
    FM_REQUIRE(args.rows >= 0 && args.rows < (int64_t(1) << 31) && args.columns > 0 && args.columns <= kMaxColumns / 2, "%s: bad sizes", name);
    if (int status = check_map(name, args.map, expert_ends, expert_pad_begins, num_experts, index_dtype)) return status;
    if (gated && args.columns % kBlock != 0) return fail(FM_ERR_UNSUPPORTED, "%s: a gated activation has whole blocks of %d columns", name, kBlock);
    if (args.rows == 0) return FM_OK;
    const int64_t parts = gated ? 2 : 1, input_columns = parts * args.columns, padded = padded_columns(args.columns), padded_input = padded_columns(input_columns);
    const int64_t row_padding = padded_columns(args.rows);
    const void *plain = forward ? args.input : args.grad_output;
    FM_REQUIRE(plain && reinterpret_cast<uintptr_t>(plain) % dtype_size(dtype) == 0, "%s: null or misaligned tensor", name);
    FM_REQUIRE(args.rows <= 1 || (forward ? args.input_stride >= input_columns : args.grad_output_stride >= args.columns), "%s: rows overlap", name);
    args.column_blocks = static_cast<uint32_t>(padded / kBlock);
    if (forward) args.checkpoint_stride = padded_input, args.output_stride = padded;
    else args.grad_stride = padded_input, args.transposed_stride = args.output_stride = row_padding;
    if (int status = check_tensor(name, "the checkpoint", args.checkpoint, args.checkpoint_scales, args.rows, padded_input, args.checkpoint_stride,
                                  args.checkpoint_scale_stride)) return status;
    if (int status = check_tensor(name, "the output", args.output, args.output_scales, forward ? args.rows : args.columns, args.output_stride, args.output_stride,
                                  args.output_scale_stride)) return status;
    if (!forward) {
        if (int status = check_tensor(name, "the gradient", args.grad, args.grad_scales, args.rows, padded_input, padded_input, args.grad_scale_stride)) return status;
        if (int status = check_tensor(name, "the transposed gradient", args.grad_transposed, args.grad_transposed_scales, input_columns, row_padding, row_padding,
                                      args.transposed_scale_stride)) return status;
    }
    const int64_t grid = row_padding / kBlock * args.column_blocks;
    if ((forward && args.rows > 1 && args.input_stride > kMaxSquareStride / dtype_size(dtype)) || padded_input > kMaxSquareStride ||
        (!forward && ((args.rows > 1 && args.grad_output_stride > kMaxSquareStride / dtype_size(dtype)) || args.checkpoint_stride > kMaxSquareStride)))
        return fail(FM_ERR_UNSUPPORTED, "%s: too large", name);
    if (grid >= (int64_t(1) << 32) / kSquareThreads) return fail(FM_ERR_UNSUPPORTED, "%s: too large", name);
    FM_DISPATCH_DTYPE(dtype, T, {
        if (gated) launch_activation<T, true>(forward, activation, args, static_cast<uint32_t>(grid), static_cast<hipStream_t>(stream));
        else launch_activation<T, false>(forward, activation, args, static_cast<uint32_t>(grid), static_cast<hipStream_t>(stream));
    });
    return check_launch(name);
}

}  // namespace block

}  // namespace fm

using namespace fm;

extern "C" int fm_block_activation_forward(const void *input, void *output, void *output_scales, void *checkpoint, void *checkpoint_scales,
                                           const void *expert_ends, const void *expert_pad_begins, int64_t rows, int64_t columns, int64_t num_experts,
                                           int64_t input_stride, int64_t output_scale_stride, int64_t checkpoint_scale_stride, int gated, int activation,
                                           int dtype, int index_dtype, void *stream) {
    block::ActivationArgs args{};
    args.input = input, args.output = static_cast<uint8_t *>(output), args.output_scales = static_cast<uint8_t *>(output_scales);
    args.checkpoint = static_cast<uint8_t *>(checkpoint), args.checkpoint_scales = static_cast<uint8_t *>(checkpoint_scales);
    args.rows = rows, args.columns = columns, args.input_stride = input_stride;
    args.output_scale_stride = output_scale_stride, args.checkpoint_scale_stride = checkpoint_scale_stride;
    return block::run_activation("fm_block_activation_forward", true, args, expert_ends, expert_pad_begins, num_experts, gated, activation, dtype, index_dtype, stream);
}

extern "C" int fm_block_activation_backward(const void *grad_output, const void *checkpoint, const void *checkpoint_scales, void *grad, void *grad_scales,
                                            void *grad_transposed, void *grad_transposed_scales, void *output_transposed, void *output_transposed_scales,
                                            const void *expert_ends, const void *expert_pad_begins, int64_t rows, int64_t columns, int64_t num_experts,
                                            int64_t grad_output_stride, int64_t checkpoint_stride, int64_t checkpoint_scale_stride, int64_t grad_scale_stride,
                                            int64_t grad_transposed_scale_stride, int64_t output_transposed_scale_stride, int gated, int activation, int dtype,
                                            int index_dtype, void *stream) {
    block::ActivationArgs args{};
    args.grad_output = grad_output;
    args.checkpoint = static_cast<uint8_t *>(const_cast<void *>(checkpoint)), args.checkpoint_scales = static_cast<uint8_t *>(const_cast<void *>(checkpoint_scales));
    args.grad = static_cast<uint8_t *>(grad), args.grad_scales = static_cast<uint8_t *>(grad_scales);
    args.grad_transposed = static_cast<uint8_t *>(grad_transposed), args.grad_transposed_scales = static_cast<uint8_t *>(grad_transposed_scales);
    args.output = static_cast<uint8_t *>(output_transposed), args.output_scales = static_cast<uint8_t *>(output_transposed_scales);
    args.rows = rows, args.columns = columns, args.grad_output_stride = grad_output_stride;
    args.checkpoint_stride = checkpoint_stride, args.checkpoint_scale_stride = checkpoint_scale_stride, args.grad_scale_stride = grad_scale_stride;
    args.transposed_scale_stride = grad_transposed_scale_stride, args.output_scale_stride = output_transposed_scale_stride;
    return block::run_activation("fm_block_activation_backward", false, args, expert_ends, expert_pad_begins, num_experts, gated, activation, dtype, index_dtype, stream);
}
