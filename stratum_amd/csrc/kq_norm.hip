// kq_norm.hip -- RMS norm of rows with the residual's addition before it, to
// binary32 or int8 rows (gfx950).
//
//   s = fl(x + r),  m = (1 / K) sum s^2,  y = fl(s (m + eps)^-1/2 w)
//
// One workgroup per row.  The squares, their sum and the product are binary64
// and y is rounded once: squares of binary32 values above 1.8e19 do not
// overflow, and an int8 step is taken from the correctly rounded y.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "kq_launch.h"

#pragma clang fp contract(off)

namespace {

__device__ __forceinline__ double wg_sum(double v, double* sm) {
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) v += __shfl_xor(v, off);
    if ((threadIdx.x & 63) == 0) sm[threadIdx.x >> 6] = v;
    __syncthreads();
    v = sm[0];
    for (int i = 1; i < (int)blockDim.x / 64; i++) v += sm[i];
    return v;
}

// The int8 group of G values that G consecutive lanes hold (one each):
// kq_quantize_kernel's arithmetic.
template <int G>
__device__ __forceinline__ void store_group(const kq_rmsnorm& a, long row, int i, float y) {
    float amax = fabsf(y);
#pragma unroll
    for (int off = 1; off < G; off <<= 1) amax = fmaxf(amax, __shfl_xor(amax, off));
    const float scale = __fdiv_rn(amax, 127.0f);
    const float inv = scale > 0.0f ? __fdiv_rn(1.0f, scale) : 0.0f;
    const int q = min(127, max(-128, __float2int_rn(y * inv)));
    int sum = q;
#pragma unroll
    for (int off = 1; off < G; off <<= 1) sum += __shfl_xor(sum, off);
    if (i >= a.K) return;
    a.xq[row * a.K + i] = (int8_t)q;
    if (i % G == 0) {
        a.xscale[row * (a.K / G) + i / G] = scale;
        if (a.xsum) a.xsum[row * (a.K / G) + i / G] = sum;
    }
}

__global__ __launch_bounds__(256) void kq_rmsnorm_kernel(kq_rmsnorm a) {
    __shared__ double sm[4];
    const long row = blockIdx.x;
    const float* x = a.x + row * a.x_stride;
    const float* r = a.resid ? a.resid + row * a.resid_stride : nullptr;
    float* s = a.sum ? a.sum + row * a.sum_stride : nullptr;
    float* y = a.y ? a.y + row * a.y_stride : nullptr;
    double sq = 0.0;
    for (int i = threadIdx.x; i < a.K; i += 256) {
        const float v = r ? x[i] + r[i] : x[i];
        if (s) s[i] = v;
        sq = sq + (double)v * (double)v;
    }
    sq = wg_sum(sq, sm);
    const double inv = 1.0 / sqrt(sq / (double)a.K + (double)a.eps);
    for (int i0 = 0; i0 < a.K; i0 += 256) {
        const int i = i0 + threadIdx.x;
        float v = 0.0f;
        if (i < a.K) {
            v = s ? s[i] : r ? x[i] + r[i] : x[i];
            const double n = (double)v * inv;
            v = (float)(a.weight ? n * (double)a.weight[i] : n);
            if (y) y[i] = v;
        }
        if (a.group == 32) store_group<32>(a, row, i, v);
        if (a.group == 16) store_group<16>(a, row, i, v);
    }
}

}  // namespace

extern "C" int kqk_launch_rmsnorm(const kq_rmsnorm* a, hipStream_t st) {
    if (a->B < 1 || a->K < 1) return (int)hipErrorInvalidValue;
    hipLaunchKernelGGL(kq_rmsnorm_kernel, dim3((unsigned)a->B), dim3(256), 0, st, *a);
    return (int)hipGetLastError();
}
