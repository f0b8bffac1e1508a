// kq_w4.hip -- products with 4-bit weights and group scales (gfx950).
//
//   y[b][n] = add[b][n] + sum over groups g of
//             s[n][g] * sum over k in g of (q[n][k] - z[n][g]) x[b][k]
//
// Weights are planes, not blocks: a row is K / 2 bytes of nibbles (weight 2j
// in byte j's low half), its scales and zero points lie in planes of their own.
#include <hip/hip_runtime.h>
#include <hip/hip_fp16.h>
#include <stdint.h>

#include "kq_launch.h"

#pragma clang fp contract(off)

namespace {

__device__ __forceinline__ float w4_scale(const void* s, int type, long i) {
    if (type == KQ_TYPE_F16) return __half2float(static_cast<const __half*>(s)[i]);
    if (type == KQ_TYPE_F32) return static_cast<const float*>(s)[i];
    return __uint_as_float((uint32_t)static_cast<const uint16_t*>(s)[i] << 16);
}

// One wave per row, a lane per 32 weights, up to 4 streams a pass.
template <bool Q8>
__global__ __launch_bounds__(256) void kq_w4_kernel(kq_w4 w, const float* x, const int8_t* xq,
                                                    const float* xs, const float* add, float* y,
                                                    int B) {
    const int row = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
    if (row >= w.N) return;
    const int b0 = blockIdx.y * 4, nb = min(4, B - b0), nblk = w.K / 32;
    const uint4* q = reinterpret_cast<const uint4*>(w.q + (long)row * (w.K / 2));
    float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int c = lane; c < nblk; c += 64) {
        const uint4 v = q[c];
        const long g = (long)row * (w.K / w.group) + (long)c * 32 / w.group;
        const float s = w4_scale(w.scales, w.scale_type, g);
        const int z = w.zeros ? w.zeros[g] : 8;
        const uint32_t d[4] = {v.x, v.y, v.z, v.w};
        for (int b = 0; b < nb; b++) {
            float t = 0.0f;
#pragma unroll
            for (int i = 0; i < 32; i++) {
                const float n = (float)((int)((d[i / 8] >> (4 * (i % 8))) & 15) - z);
                const long at = (long)(b0 + b) * w.K + 32 * c + i;
                t = fmaf(n, Q8 ? (float)xq[at] : x[at], t);
            }
            if (Q8) t = t * xs[(long)(b0 + b) * nblk + c];
            acc[b] = fmaf(s, t, acc[b]);
        }
    }
    for (int b = 0; b < nb; b++) {
        float t = acc[b];
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) t += __shfl_xor(t, off);
        const long o = (long)(b0 + b) * w.N + row;
        if (lane == 0) y[o] = add ? add[o] + t : t;
    }
}

}  // namespace

extern "C" {

int64_t kqk_w4_workspace(const kq_w4* w, int B, int q8, int n_cu) { return 0; }

int kqk_launch_w4(const kq_w4* w, const float* x, const int8_t* xq, const float* xs,
                  const float* add, float* y, int B, void* work, int n_cu, hipStream_t st) {
    if (w->N < 1 || w->K < 32 || w->K % 32 || B < 1) return (int)hipErrorInvalidValue;
    const dim3 grid((unsigned)((w->N + 3) / 4), (unsigned)((B + 3) / 4));
    if (xq)
        hipLaunchKernelGGL(kq_w4_kernel<true>, grid, dim3(256), 0, st, *w, x, xq, xs, add, y, B);
    else
        hipLaunchKernelGGL(kq_w4_kernel<false>, grid, dim3(256), 0, st, *w, x, xq, xs, add, y, B);
    return (int)hipGetLastError();
}

}
