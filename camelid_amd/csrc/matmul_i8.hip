// The int8 product with a scale for every token and every weight row:
//   out[t][r] = rnd((sum_c q[t][c] * w[r][c]) * scales[t] * w_scales[r] + bias[r])
// The sum is an exact 32-bit integer (rows of up to 131071 values: 2^14 * 131071 < 2^31), so no split of the contraction changes a bit.  It is
// widened to f32 (24 bits), scaled in f32 and rounded once to the output's type.
#include "typed_rows.hpp"

#pragma clang fp contract(off)

namespace cml {

typedef int v4i_i8 __attribute__((ext_vector_type(4)));

struct MatmulI8 {
    const int8_t *q, *w;
    const float *scales, *w_scales, *bias;
    void *out;
    int64_t q_stride, w_stride, out_stride;
    int n_tokens, rows, cols;
};

// Four neighbouring weight rows of one token.
template <class T>
__device__ __forceinline__ void store_cells(const MatmulI8 &a, int t, int r, const v4i_i8 &acc) {
    if (t >= a.n_tokens) return;
    typename T::Bits *out = static_cast<typename T::Bits *>(a.out) + t * a.out_stride + r;
    const float s = a.scales[t];
#pragma unroll
    for (int i = 0; i < 4; i++)
        if (r + i < a.rows) {
            const float v = static_cast<float>(acc[i]) * s * a.w_scales[r + i];
            store_value<T>(out + i, a.bias ? v + a.bias[r + i] : v);
        }
}

// Any alignment and size: 64 rows x 64 tokens a workgroup of four waves, 64 values of the contraction a step, staged through registers.
template <class T>
__global__ __launch_bounds__(256) void matmul_i8_kernel(MatmulI8 a) {
    constexpr int kPitch = 80;  // bytes
    __shared__ __align__(16) int8_t sw[64 * kPitch], sq[64 * kPitch];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int r0 = blockIdx.x * 64, t0 = blockIdx.y * 64;
    const int row = tid >> 2, k_at = (tid & 3) * 16;
    const int8_t *w = a.w + min(r0 + row, a.rows - 1) * a.w_stride, *q = a.q + min(t0 + row, a.n_tokens - 1) * a.q_stride;
    auto piece = [&](const int8_t *p, int k) {
        typedef uint32_t v4u __attribute__((ext_vector_type(4), aligned(1)));
        if (k + 16 <= a.cols) {
            const v4u v = *reinterpret_cast<const v4u *>(p + k);
            return make_uint4(v.x, v.y, v.z, v.w);
        }
        uint32_t v[4] = {0, 0, 0, 0};
        for (int j = 0; j < 16; j++)
            if (k + j < a.cols) v[j >> 2] |= static_cast<uint32_t>(static_cast<uint8_t>(p[k + j])) << (8 * (j & 3));
        return make_uint4(v[0], v[1], v[2], v[3]);
    };
    v4i_i8 acc[2][2] = {};
    const int wr = (wave & 1) * 32, wt = (wave >> 1) * 32, n = lane & 15, kq = (lane >> 4) * 16;
    for (int k = 0; k < a.cols; k += 64) {
        const uint4 pw = piece(w, k + k_at), pq = piece(q, k + k_at);
        __syncthreads();
        *reinterpret_cast<uint4 *>(sw + row * kPitch + k_at) = pw;
        *reinterpret_cast<uint4 *>(sq + row * kPitch + k_at) = pq;
        __syncthreads();
        v4i_i8 fw[2], fq[2];
#pragma unroll
        for (int i = 0; i < 2; i++) {
            fw[i] = *reinterpret_cast<const v4i_i8 *>(sw + (wr + 16 * i + n) * kPitch + kq);
            fq[i] = *reinterpret_cast<const v4i_i8 *>(sq + (wt + 16 * i + n) * kPitch + kq);
        }
#pragma unroll
        for (int i = 0; i < 2; i++)
#pragma unroll
            for (int j = 0; j < 2; j++) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(fw[i], fq[j], acc[i][j], 0, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < 2; i++)
#pragma unroll
        for (int j = 0; j < 2; j++) store_cells<T>(a, t0 + wt + 16 * j + n, r0 + wr + 16 * i + 4 * (lane >> 4), acc[i][j]);
}

int launch_matmul_i8(const int8_t *q, int64_t q_stride, const float *scales, int64_t n_tokens, const int8_t *w, int64_t w_stride, const float *w_scales, int64_t rows, int64_t cols,
                     const float *bias, int dtype, void *out, int64_t out_stride, hipStream_t st) {
    const MatmulI8 a{q, w, scales, w_scales, bias, out, q_stride, w_stride, out_stride, static_cast<int>(n_tokens), static_cast<int>(rows), static_cast<int>(cols)};
    CML_COUNT_LAUNCH("i8.matmul.staged");
    return with_type(dtype, [&](auto t) {
        const dim3 grid(static_cast<unsigned>((rows + 63) / 64), static_cast<unsigned>((n_tokens + 63) / 64));
        hipLaunchKernelGGL(matmul_i8_kernel<decltype(t)>, grid, dim3(256), 0, st, a);
        CML_HIP_TRY(hipGetLastError());
        return CML_OK;
    });
}

}  // namespace cml
