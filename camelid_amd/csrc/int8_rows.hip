// Rows to 8 bits with one scale each: the activation side of the int8 product (matmul_i8.hip).
//
//   h = rnd(x + residual)                 the residual stream, rounded to its own type: what the next layer reads is what is normalised
//   y = h * inv * weight, inv = 1 / sqrt(mean(h^2) + eps)
//   scale = max|y| / 127, q = round(y / scale), ties to even
//
// A row stays in registers between its one read and its writes.  The quotient y / scale is h * weight * (127 / max|h * weight|): inv cancels, so
// the sum of squares and the maximum are reduced together, behind one barrier.  Sums (of up to 32 squares a thread; longer rows in 64 bits) and products are f32; the only roundings to
// fewer bits are the stream's type and the 8 bits themselves.
//
// Memory's rate bounds long prompts: 8192 x 4096 bf16 in 45 us (5.2 TB/s; a large copy 5.2), read back in 18 (5.5); the quantizer alone 21 (4.8).  One token: 2.7 us, a launch.
#include "typed_rows.hpp"

#include <algorithm>

#pragma clang fp contract(off)

namespace cml {

struct NormRows {
    const void *x, *residual;
    const float *weight;
    void *sum;
    float *normed;
    int8_t *q;
    float *scales;
    int64_t x_stride, residual_stride, sum_stride, q_stride;  // elements
    int64_t n_rows;
    int cols;
    float eps;
};

// What a row's sum of squares and largest |h * weight| (as bits) make of it.
struct RowScale {
    float most, inv, scale, lift, to_q;
    bool live;
    __device__ __forceinline__ int quant(float hw) const { return live ? static_cast<int>(fminf(fmaxf(rintf(hw * lift * to_q), -127.0f), 127.0f)) : 0; }
    // v (inv or scale) as it is told: squares past the largest f32, whose inverse root would be 0, make it NaN, and a row of zeros is one whatever eps says (0 / 0 is none).
    // (Only where it is written: two instructions more for every lane are 2 % of 8192 x 4096 bf16.)
    __device__ __forceinline__ float told(float v) const { return most == 0.0f ? 0.0f : inv > 0.0f ? v : __builtin_nanf(""); }
};
template <bool NORM>
__device__ __forceinline__ RowScale row_scale(const NormRows &a, float sum, uint32_t top) {
    RowScale f;
    f.most = __builtin_bit_cast(float, top);
    f.inv = NORM ? 1.0f / sqrtf(sum / static_cast<float>(a.cols) + a.eps) : 1.0f;
    f.scale = f.most * f.inv / 127.0f;
    f.lift = f.most < 1e-30f ? 18446744073709551616.0f : 1.0f;              // 127 / most of a row of tiny values would be infinite: such a row is lifted by 2^64 first
    f.live = f.most > 0.0f && f.inv > 0.0f && fabsf(f.scale) < INFINITY;  // a row of zeros, or one that leaves f32 (its scale is NaN or infinite): no quants
    f.to_q = f.live ? 127.0f / (f.most * f.lift) : 0.0f;
    return f;
}

// A row by THREADS threads that hold CH times eight values each; workgroups of 256 threads at least, so rows of one wave go four to a workgroup.
// NORM: the norm above; otherwise y = x.  ONCE: x and residual are read past the caches.
template <class T, bool NORM, int THREADS, int CH, bool ONCE>
__global__ __launch_bounds__(THREADS < 256 ? 256 : THREADS) void rows_to_i8_kernel(NormRows a) {
    typedef typename T::Bits Bits;
    constexpr int kWaves = THREADS / 64, kRows = THREADS < 256 ? 256 / THREADS : 1;
    __shared__ float s_sum[kWaves];
    __shared__ uint32_t s_max[kWaves];
    const int tid = threadIdx.x & (THREADS - 1), wave = tid >> 6, lane = tid & 63;
    const int64_t row = static_cast<int64_t>(blockIdx.x) * kRows + (kRows > 1 ? threadIdx.x / THREADS : 0);
    if (kRows > 1 && row >= a.n_rows) return;  // (such rows meet no barrier)
    const Bits *x = static_cast<const Bits *>(a.x) + row * a.x_stride;
    const Bits *r = NORM && a.residual ? static_cast<const Bits *>(a.residual) + row * a.residual_stride : nullptr;
    float h[CH][8], hw[CH][8];
    float sum = 0.0f;
    uint32_t top = 0;  // |h * weight| as bits: they order like the values, and a NaN is above all
    auto weigh = [&](int c, float (&out)[8]) __attribute__((always_inline)) {
        const int i = (c * THREADS + tid) * 8;
        if (!NORM) {
#pragma unroll
            for (int j = 0; j < 8; j++) out[j] = h[c][j];
        } else {
            if (i + 8 <= a.cols) {
                load8<TypeF32>(a.weight + i, out);
            } else {
#pragma unroll
                for (int j = 0; j < 8; j++) out[j] = i + j < a.cols ? a.weight[i + j] : 0.0f;
            }
#pragma unroll
            for (int j = 0; j < 8; j++) out[j] = h[c][j] * out[j];
        }
    };
#pragma unroll
    for (int c = 0; c < CH; c++) {
        const int i = (c * THREADS + tid) * 8;
        if (i + 8 <= a.cols) {
            load8<T, ONCE>(x + i, h[c]);
            if (NORM && r) {
                float add[8];
                load8<T, ONCE>(r + i, add);
#pragma unroll
                for (int j = 0; j < 8; j++) h[c][j] = rounded<T>(h[c][j] + add[j]);
            }
        } else {
#pragma unroll
            for (int j = 0; j < 8; j++) {
                h[c][j] = 0.0f;
                if (i + j < a.cols) {
                    h[c][j] = load_value<T>(x + i + j);
                    if (NORM && r) h[c][j] = rounded<T>(h[c][j] + load_value<T>(r + i + j));
                }
            }
        }
        weigh(c, hw[c]);
#pragma unroll
        for (int j = 0; j < 8; j++) {
            if (NORM) sum = fmaf(h[c][j], h[c][j], sum);
            top = max(top, __builtin_bit_cast(uint32_t, hw[c][j]) & 0x7fffffffu);
        }
    }
    if (NORM && a.sum) {
        Bits *out = static_cast<Bits *>(a.sum) + row * a.sum_stride;
#pragma unroll
        for (int c = 0; c < CH; c++) {
            const int i = (c * THREADS + tid) * 8;
            if (i + 8 <= a.cols) {
                store8<T>(out + i, h[c]);
            } else {
#pragma unroll
                for (int j = 0; j < 8; j++)
                    if (i + j < a.cols) store_value<T>(out + i + j, h[c][j]);
            }
        }
    }
    if (NORM) sum = wave_allsum(sum);
    top = static_cast<uint32_t>(wave_allmax_i32(static_cast<int>(top)));
    if constexpr (kWaves > 1) {
        if (lane == 0) {
            s_sum[wave] = sum;
            s_max[wave] = top;
        }
        __syncthreads();
        sum = 0.0f;
#pragma unroll
        for (int w = 0; w < kWaves; w++) {
            sum = sum + s_sum[w];
            top = max(top, s_max[w]);
        }
    }
    const RowScale f = row_scale<NORM>(a, sum, top);
    if (tid == 0) a.scales[row] = f.told(f.scale);
    int8_t *q = a.q + row * a.q_stride;
    float *normed = NORM && a.normed ? a.normed + row * a.cols : nullptr;
    const float inv = normed ? f.told(f.inv) : 0.0f;
#pragma unroll
    for (int c = 0; c < CH; c++) {
        const int i = (c * THREADS + tid) * 8;
        int v[8];
#pragma unroll
        for (int j = 0; j < 8; j++) v[j] = f.quant(hw[c][j]);
        if (i + 8 <= a.cols) {
            typedef uint32_t v2u __attribute__((ext_vector_type(2), aligned(1)));
            *reinterpret_cast<v2u *>(q + i) = v2u{pack4(v[0], v[1], v[2], v[3]), pack4(v[4], v[5], v[6], v[7])};
        } else {
#pragma unroll
            for (int j = 0; j < 8; j++)
                if (i + j < a.cols) q[i + j] = static_cast<int8_t>(v[j]);
        }
        if (!normed) continue;
        float y[8];
#pragma unroll
        for (int j = 0; j < 8; j++) y[j] = hw[c][j] * inv;
        if (i + 8 <= a.cols) {
            store8<TypeF32>(normed + i, y);
        } else {
#pragma unroll
            for (int j = 0; j < 8; j++)
                if (i + j < a.cols) normed[i + j] = y[j];
        }
    }
}

// Rows that the registers do not hold: read twice, the second time from `sum` where it is written (which may be x or residual).  A thread adds up to 16384 squares, one
// after the other: in 64 bits, because in 32 their roundings, which all go one way where values are alike, come to 1e-4 of the inverse root.
// One value a lane and load, one workgroup a row, and x twice: the quantizer takes 17 us for one row of 53248 bf16 and 200 for 2048 (1.6 TB/s of input and output), the norm 29 and 318.
template <class T, bool NORM>
__global__ __launch_bounds__(1024) void long_rows_to_i8_kernel(NormRows a) {
    typedef typename T::Bits Bits;
    __shared__ float s_sum[16];
    __shared__ uint32_t s_max[16];
    const int tid = threadIdx.x;
    const int64_t row = blockIdx.x;
    const Bits *x = static_cast<const Bits *>(a.x) + row * a.x_stride;
    const Bits *r = NORM && a.residual ? static_cast<const Bits *>(a.residual) + row * a.residual_stride : nullptr;
    Bits *out = NORM && a.sum ? static_cast<Bits *>(a.sum) + row * a.sum_stride : nullptr;
    auto value = [&](int i) __attribute__((always_inline)) {
        const float v = load_value<T>(x + i);
        return r ? rounded<T>(v + load_value<T>(r + i)) : v;
    };
    double squares = 0.0;
    uint32_t top = 0;
    for (int i = tid; i < a.cols; i += 1024) {
        const float h = value(i);
        if (out) store_value<T>(out + i, h);
        if (NORM) squares = fma(static_cast<double>(h), static_cast<double>(h), squares);
        top = max(top, __builtin_bit_cast(uint32_t, NORM ? h * a.weight[i] : h) & 0x7fffffffu);
    }
    float sum = wave_allsum(static_cast<float>(squares));
    top = static_cast<uint32_t>(wave_allmax_i32(static_cast<int>(top)));
    if ((tid & 63) == 0) {
        s_sum[tid >> 6] = sum;
        s_max[tid >> 6] = top;
    }
    __syncthreads();
    sum = 0.0f;
#pragma unroll
    for (int w = 0; w < 16; w++) {
        sum = sum + s_sum[w];
        top = max(top, s_max[w]);
    }
    const RowScale f = row_scale<NORM>(a, sum, top);
    if (tid == 0) a.scales[row] = f.told(f.scale);
    for (int i = tid; i < a.cols; i += 1024) {
        const float h = out ? load_value<T>(out + i) : value(i), hw = NORM ? h * a.weight[i] : h;
        a.q[row * a.q_stride + i] = static_cast<int8_t>(f.quant(hw));
        if (NORM && a.normed) a.normed[row * a.cols + i] = hw * f.told(f.inv);
    }
}

template <class T, bool NORM, int THREADS, int CH>
static int launch_rows(const NormRows &a, hipStream_t st) {
    constexpr int kThreads = THREADS < 256 ? 256 : THREADS, kRows = kThreads / THREADS;
    const dim3 grid(static_cast<unsigned>((a.n_rows + kRows - 1) / kRows));
    // Rows of 16-bit values that no cache holds go past them, and leave them to the quants, which are read next (us with cml_dequantize_i8 behind it, plain / so: 8192 x 4096
    // bf16 64.6 / 63.2, 4096 x 8192 67.6 / 60.1, 8192 x 8192 128.6 / 115.1; 512 x 4096 8.9 / 10.0; f32 4096 x 4096 51.5 / 53.9).
    if (sizeof(typename T::Bits) == 2 && a.n_rows * a.cols >= 16ll << 20) hipLaunchKernelGGL((rows_to_i8_kernel<T, NORM, THREADS, CH, true>), grid, dim3(kThreads), 0, st, a);
    else hipLaunchKernelGGL((rows_to_i8_kernel<T, NORM, THREADS, CH, false>), grid, dim3(kThreads), 0, st, a);
    CML_HIP_TRY(hipGetLastError());
    return CML_OK;
}

template <class T, bool NORM>
static int launch_rows_typed(const NormRows &a, hipStream_t st) {
    // Most threads that still have 16 bytes of a 16-bit row each, up to 8192 values (us with cml_dequantize_i8 behind it, 256 / 512 / 1024 threads: 1 x 4096 4.8 / 4.2 / 4.9, 512 x 8192
    // 16.0 / 13.9 / 14.3, 8192 x 4096 61.6 / 63.2 / 85.9, 8192 x 8192 120 / 115 / 118); 1 x 16384 with 512 / 1024 7.1 / 6.7, 2048 x 16384 66.3 / 63.1.
    if (a.cols <= 512) return launch_rows<T, NORM, 64, 1>(a, st);
    if (a.cols <= 2048) return launch_rows<T, NORM, 256, 1>(a, st);
    if (a.cols <= 4096) return launch_rows<T, NORM, 512, 1>(a, st);
    if (a.cols <= 8192) return launch_rows<T, NORM, 512, 2>(a, st);
    if (a.cols <= 16384) return launch_rows<T, NORM, 1024, 2>(a, st);
    if (a.cols <= 32768) return launch_rows<T, NORM, 1024, 4>(a, st);
    hipLaunchKernelGGL((long_rows_to_i8_kernel<T, NORM>), dim3(static_cast<unsigned>(a.n_rows)), dim3(1024), 0, st, a);
    CML_HIP_TRY(hipGetLastError());
    return CML_OK;
}

// Rows in as many launches as workgroups of 1024, the largest, allow.
template <bool NORM>
static int launch_all_rows(int dtype, const NormRows &a, hipStream_t st) {
    const int64_t most = most_workgroups(1024);
    return with_type(dtype, [&](auto t) {
        typedef decltype(t) T;
        typedef typename T::Bits Bits;
        for (int64_t first = 0; first < a.n_rows; first += most) {
            NormRows part = a;
            part.x = static_cast<const Bits *>(a.x) + first * a.x_stride;
            if (a.residual) part.residual = static_cast<const Bits *>(a.residual) + first * a.residual_stride;
            if (a.sum) part.sum = static_cast<Bits *>(a.sum) + first * a.sum_stride;
            if (a.normed) part.normed = a.normed + first * a.cols;
            part.q = a.q + first * a.q_stride;
            part.scales = a.scales + first;
            part.n_rows = std::min(most, a.n_rows - first);
            if (NORM) CML_COUNT_LAUNCH("i8.add_rms_norm");
            else CML_COUNT_LAUNCH("i8.quantize");
            if (int rc = launch_rows_typed<T, NORM>(part, st)) return rc;
        }
        return CML_OK;
    });
}

int launch_add_rms_norm_i8(int dtype, const void *x, int64_t x_stride, const void *residual, int64_t residual_stride, const float *weight, float eps, int64_t n_tokens, int64_t cols,
                           void *sum, int64_t sum_stride, float *normed, int8_t *q, int64_t q_stride, float *scales, hipStream_t st) {
    const NormRows a{x, residual, weight, sum, normed, q, scales, x_stride, residual_stride, sum_stride, q_stride, n_tokens, static_cast<int>(cols), eps};
    return launch_all_rows<true>(dtype, a, st);
}

int launch_quantize_i8(int dtype, const void *x, int64_t x_stride, int64_t n_rows, int64_t cols, int8_t *q, int64_t q_stride, float *scales, hipStream_t st) {
    const NormRows a{x, nullptr, nullptr, nullptr, nullptr, q, scales, x_stride, 0, 0, q_stride, n_rows, static_cast<int>(cols), 0.0f};
    return launch_all_rows<false>(dtype, a, st);
}

// out = q * scale, sixteen values a thread.
template <class T>
__global__ __launch_bounds__(256) void dequantize_i8_kernel(const int8_t *__restrict__ q, int64_t q_stride, const float *__restrict__ scales, int cols, int chunks,
                                                            typename T::Bits *__restrict__ out, int64_t out_stride) {
    const int64_t row = blockIdx.x / static_cast<unsigned>(chunks);
    const int i = (static_cast<int>(blockIdx.x - row * chunks) * 256 + threadIdx.x) * 16;
    if (i >= cols) return;
    const int8_t *from = q + row * q_stride + i;
    typename T::Bits *to = out + row * out_stride + i;
    const float s = scales[row];
    if (i + 16 <= cols) {
        typedef uint32_t v4u __attribute__((ext_vector_type(4), aligned(1)));
        const v4u p = *reinterpret_cast<const v4u *>(from);
#pragma unroll
        for (int k = 0; k < 2; k++) {
            float v[8];
#pragma unroll
            for (int j = 0; j < 8; j++) v[j] = static_cast<float>(static_cast<int8_t>(p[2 * k + j / 4] >> (8 * (j % 4)))) * s;
            store8<T>(to + 8 * k, v);
        }
    } else {
        for (int j = 0; i + j < cols; j++) store_value<T>(to + j, static_cast<float>(from[j]) * s);
    }
}

int launch_dequantize_i8(const int8_t *q, int64_t q_stride, const float *scales, int64_t n_rows, int64_t cols, int dtype, void *out, int64_t out_stride, hipStream_t st) {
    const int chunks = static_cast<int>((cols + 4095) / 4096);
    const int64_t most = std::max<int64_t>(1, most_workgroups(256) / chunks);
    return with_type(dtype, [&](auto t) {
        typedef decltype(t) T;
        for (int64_t first = 0; first < n_rows; first += most) {
            CML_COUNT_LAUNCH("i8.dequantize");
            hipLaunchKernelGGL(dequantize_i8_kernel<T>, dim3(static_cast<unsigned>(std::min(most, n_rows - first) * chunks)), dim3(256), 0, st, q + first * q_stride, q_stride, scales + first,
                               static_cast<int>(cols), chunks, static_cast<typename T::Bits *>(out) + first * out_stride, out_stride);
            CML_HIP_TRY(hipGetLastError());
        }
        return CML_OK;
    });
}

}  // namespace cml
