// kq_norm.hip -- RMS norm of rows with the residual's addition before it, to
// binary32 or int8 rows (gfx950).
//
//   s = fl(x + r),  m = (1 / K) sum s^2,  y = fl(s (m + eps)^-1/2 w)
//
// One workgroup per row, which it reads once.  The squares, their sum and the
// product are binary64 and y is rounded once: squares of binary32 values above
// 1.8e19 do not overflow, and an int8 step is taken from the correctly rounded y.
// Memory bounds many rows (4096 of 5120, residual, to int8: 60 us, 4.6 TB/s; a copy
// reaches 5.1), the chain load, sum, product a few (one of 5120: 3.3 us, eight
// with residual to int8 5.0).
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

template <int V> struct Vec;
template <> struct Vec<1> { typedef float f __attribute__((ext_vector_type(1))); };
template <> struct Vec<4> { typedef float f __attribute__((ext_vector_type(4))); };

// The int8 group of G values that G / V consecutive lanes hold (lane t's
// first is value i): kq_quantize_kernel's arithmetic.
template <int G, int V>
__device__ __forceinline__ void store_group(const kq_rmsnorm& a, long row, int i,
                                            const typename Vec<V>::f y) {
    float amax = fabsf(y[0]);
#pragma unroll
    for (int e = 1; e < V; e++) amax = fmaxf(amax, fabsf(y[e]));
#pragma unroll
    for (int off = 1; off < G / V; off <<= 1) amax = fmaxf(amax, __shfl_xor(amax, off));
    const float scale = __fdiv_rn(amax, 127.0f);
    const float inv = scale > 0.0f ? __fdiv_rn(1.0f, scale) : 0.0f;
    int sum = 0;
    uint32_t w = 0;
#pragma unroll
    for (int e = 0; e < V; e++) {
        const int q = min(127, max(-128, __float2int_rn(y[e] * inv)));
        sum += q;
        w |= ((uint32_t)q & 0xffu) << (8 * e);
    }
    if (a.xsum) {
#pragma unroll
        for (int off = 1; off < G / V; off <<= 1) sum += __shfl_xor(sum, off);
    }
    if (i >= a.K) return;
    if (V == 4)
        *reinterpret_cast<uint32_t*>(a.xq + row * a.K + i) = w;
    else
        a.xq[row * a.K + i] = (int8_t)w;
    if (i % G == 0) {
        const long g = row * (a.K / G) + i / G;
        a.xscale[g] = scale;
        if (a.xsum) a.xsum[g] = sum;
    }
}

template <int V>
__device__ __forceinline__ void store_rows(const kq_rmsnorm& a, long row, int i,
                                           const typename Vec<V>::f y) {
    if (a.y && i < a.K)
        *reinterpret_cast<typename Vec<V>::f*>(a.y + row * a.y_stride + i) = y;
    if (a.group == 32) store_group<32, V>(a, row, i, y);
    if (a.group == 16) store_group<16, V>(a, row, i, y);
}

// V consecutive values a lane and step; NV steps hold the row in registers
// (NV V blockDim >= K), so that it is read once.  NV = 0: rows of any length,
// read a second time (from `sum`, when that is written: it may be x's rows).
template <int V, int NV>
__global__ __launch_bounds__(1024) void kq_rmsnorm_kernel(kq_rmsnorm a) {
    using F = typename Vec<V>::f;
    __shared__ double sm[16];
    const long row = blockIdx.x;
    const int T = blockDim.x, i0 = V * threadIdx.x, K = a.K;
    const float* x = a.x + row * a.x_stride;
    const float* r = a.resid ? a.resid + row * a.resid_stride : nullptr;
    float* s = a.sum ? a.sum + row * a.sum_stride : nullptr;
    const F zero = (F)0.0f;
    F v[NV ? NV : 1], w[NV ? NV : 1];
    double sq = 0.0;
    auto take = [&](F t, int i) {
        if (s) *reinterpret_cast<F*>(s + i) = t;
#pragma unroll
        for (int e = 0; e < V; e++) sq = fma((double)t[e], (double)t[e], sq);
    };
    if constexpr (NV > 0) {
#pragma unroll
        for (int j = 0; j < NV; j++) {
            const int i = i0 + j * V * T;
            v[j] = i < K ? *reinterpret_cast<const F*>(x + i) : zero;
        }
        if (r) {
#pragma unroll
            for (int j = 0; j < NV; j++) {
                const int i = i0 + j * V * T;
                if (i < K) v[j] = v[j] + *reinterpret_cast<const F*>(r + i);
            }
        }
#pragma unroll
        for (int j = 0; j < NV; j++) {
            const int i = i0 + j * V * T;
            // (the weights are asked for before the sum)
            if (a.weight) w[j] = i < K ? *reinterpret_cast<const F*>(a.weight + i) : zero;
            if (i < K) take(v[j], i);
        }
    } else {
        for (int i = i0; i < K; i += V * T) {
            F t = *reinterpret_cast<const F*>(x + i);
            if (r) t = t + *reinterpret_cast<const F*>(r + i);
            take(t, i);
        }
    }
    sq = wg_sum(sq, sm);
    const double inv = 1.0 / sqrt(sq / (double)K + (double)a.eps);
    auto finish = [&](F t, F g, int i) {
#pragma unroll
        for (int e = 0; e < V; e++) {
            const double n = (double)t[e] * inv;
            t[e] = (float)(a.weight ? n * (double)g[e] : n);
        }
        store_rows<V>(a, row, i, t);
    };
    if constexpr (NV > 0) {
#pragma unroll
        for (int j = 0; j < NV; j++) {
            const int i = i0 + j * V * T;
            finish(v[j], a.weight ? w[j] : zero, i);
        }
    } else {
        for (int j = 0; j < K; j += V * T) {
            const int i = i0 + j;
            F t = zero, g = zero;
            if (i < K) {
                t = *reinterpret_cast<const F*>((s ? s : x) + i);
                if (!s && r) t = t + *reinterpret_cast<const F*>(r + i);
                if (a.weight) g = *reinterpret_cast<const F*>(a.weight + i);
            }
            finish(t, g, i);
        }
    }
}

template <int V>
int launch(const kq_rmsnorm& a, hipStream_t st) {
    const int nv = (a.K + V - 1) / V;
    // As few steps as 1024 lanes allow (one up to 1024 loads a row) while the device's
    // lanes (2048 on each of 256 CUs) hold all rows; four steps in fewer lanes, which
    // keep more loads in flight, when they do not.  One step / four, us: rows of 1024
    // to int8, one 2.5 / 4.1, 2048 rows 8.2 / 8.5, 4096 14.2 / 13.8.  Two steps (of 1280
    // or 1153 loads) / four: rows of 5120 to binary32, one 3.1 / 3.4, 512 rows 7.8 / 7.4,
    // 1024 13.5 / 11.2, 4096 36.2 / 33.5; to int8 4.2 / 5.3, 10.0 / 10.5, 19.0 / 17.1,
    // 53.7 / 52.4; rows of 1153 single values, one 2.7 / 2.8, 512 rows 4.6 / 4.2, 4096
    // 23.0 / 17.1.
    constexpr int MOST = V == 4 ? 4 : 8;       // (8 steps of 4 spill registers)
    int steps = (long)a.B * nv <= 1 << 19 ? 1 : 4;
    while (steps <= MOST && nv > 1024 * steps) steps *= 2;
    const int per = steps <= MOST ? (nv + steps - 1) / steps : 1024;
    const dim3 wg((unsigned)((per + 63) / 64 * 64));
    auto* const k = steps == 1 ? kq_rmsnorm_kernel<V, 1> : steps == 2 ? kq_rmsnorm_kernel<V, 2>
                  : steps == 4 ? kq_rmsnorm_kernel<V, 4> : steps == MOST ? kq_rmsnorm_kernel<V, MOST>
                                                                         : kq_rmsnorm_kernel<V, 0>;
    // A launch of 2^32 lanes or more is cut to their number modulo that without an
    // error: more rows (2^26 where each takes 64) go in parts.
    const int most = (int)(0xffffffffu / wg.x);
    kq_rmsnorm b = a;
    for (int left = a.B; left > 0; left -= most) {
        b.B = left < most ? left : most;
        hipLaunchKernelGGL(k, dim3((unsigned)b.B), wg, 0, st, b);
        const int e = (int)hipGetLastError();
        if (e) return e;
        b.x += most * b.x_stride;
        if (b.resid) b.resid += most * b.resid_stride;
        if (b.sum) b.sum += most * b.sum_stride;
        if (b.y) b.y += most * b.y_stride;
        if (b.group) {
            const int64_t groups = (int64_t)most * (b.K / b.group);
            b.xq += (int64_t)most * b.K;
            b.xscale += groups;
            if (b.xsum) b.xsum += groups;
        }
    }
    return 0;
}

}  // namespace

extern "C" int kqk_launch_rmsnorm(const kq_rmsnorm* a, hipStream_t st) {
    if (a->B < 1 || a->K < 1) return (int)hipErrorInvalidValue;
    // four values a load where every row allows it
    const uintptr_t p = (uintptr_t)a->x | (uintptr_t)a->resid | (uintptr_t)a->weight |
                        (uintptr_t)a->sum | (uintptr_t)a->y;
    const int64_t n = a->K | a->x_stride | (a->resid ? a->resid_stride : 0) |
                      (a->sum ? a->sum_stride : 0) | (a->y ? a->y_stride : 0);
    return (p & 15) == 0 && (n & 3) == 0 ? launch<4>(*a, st) : launch<1>(*a, st);
}
