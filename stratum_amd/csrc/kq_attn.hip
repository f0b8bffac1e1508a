// kq_attn.hip -- attention of a few new tokens over a paged cache (gfx950).
//
//   out = sum_j p_j v_j,  p = softmax over the keys j that a token sees of scale q . k_j
//
// One wave per token and query head: 64 keys at a time, a key's product in each
// lane, then the values, D / 64 of them in each lane.
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "kq_launch.h"

#pragma clang fp contract(off)

namespace {

template <int TYPE>
__device__ __forceinline__ float value(const void* p, long i) {
    if constexpr (TYPE == KQ_TYPE_F16) return __half2float(static_cast<const __half*>(p)[i]);
    if constexpr (TYPE == KQ_TYPE_BF16)
        return __uint_as_float((uint32_t)static_cast<const uint16_t*>(p)[i] << 16);
    return (float)static_cast<const int8_t*>(p)[i];
}

template <int TYPE>
__global__ __launch_bounds__(64) void kq_attn_kernel(kq_paged_attn a) {
    const kq_kv_cache& c = a.cache;
    const int s = blockIdx.x, h = blockIdx.y, t = blockIdx.z, lane = threadIdx.x, D = c.D;
    const int hk = h / (a.shape.n_q / a.shape.n_kv);
    const int row0 = a.start ? a.start[s] : s, n = a.start ? a.start[s + 1] - row0 : 1;
    const long row = (long)row0 + t;
    if (n < 1 || n > a.shape.T || t >= n || row < 0 || row >= a.N) return;
    const int last = a.lens[s] - n + t;                   // the last key it sees
    const int from = a.shape.window ? max(0, last + 1 - a.shape.window) : 0;
    const int end = (int)min((long)last + 1, (long)a.table_stride * c.page);
    __shared__ float q[KQ_KV_MAX_D];
    __shared__ float ps[64];
    __shared__ long at[64];
    for (int d = lane; d < D; d += 64) q[d] = a.q[row * a.q_stride + (long)h * D + d] * a.scale;
    __syncthreads();
    float m = -INFINITY, l = 0.0f, o[KQ_KV_MAX_D / 64] = {};
    for (int j0 = from; j0 < end; j0 += 64) {
        const int j = j0 + lane;
        long where = -1, sc = 0;
        if (j < end) {
            const int page = a.table[(long)s * a.table_stride + j / c.page], i = j % c.page;
            if (page >= 0 && page < c.n_pages) {
                where = page * c.page_stride + hk * c.head_stride + i * c.token_stride;
                sc = ((long)page * c.n_kv + hk) * c.page + i;
            }
        }
        float x = -INFINITY;
        if (where >= 0) {
            x = 0.0f;
            for (int d = 0; d < D; d++) x = fmaf(q[d], value<TYPE>(c.k, where + d), x);
            if (TYPE == KQ_TYPE_I8) x *= c.k_scale[sc];
        }
        float top = x;
        for (int off = 1; off < 64; off <<= 1) top = fmaxf(top, __shfl_xor(top, off));
        const float nm = fmaxf(m, top);
        float p = where >= 0 ? expf(x - nm) : 0.0f, sum = p;
        for (int off = 1; off < 64; off <<= 1) sum += __shfl_xor(sum, off);
        const float f = nm == m ? 1.0f : expf(m - nm);
        l = l * f + sum;
        m = nm;
        if (TYPE == KQ_TYPE_I8 && where >= 0) p *= c.v_scale[sc];
        ps[lane] = p;
        at[lane] = where;
        __syncthreads();
        for (int e = 0; e < KQ_KV_MAX_D / 64; e++) {
            const int d = lane + 64 * e;
            if (d >= D) break;
            o[e] *= f;
            for (int k = 0; k < 64; k++)
                if (at[k] >= 0) o[e] = fmaf(ps[k], value<TYPE>(c.v, at[k] + d), o[e]);
        }
        __syncthreads();
    }
    for (int e = 0; e < KQ_KV_MAX_D / 64; e++) {
        const int d = lane + 64 * e;
        if (d < D) a.out[row * a.out_stride + (long)h * D + d] = l == 0.0f ? 0.0f : o[e] / l;
    }
}

}  // namespace

extern "C" {

void kqk_attn_plan(const kq_attn_shape* s, int n_cu, kqk_attn_sizes* z) {
    z->blocks = 1;
    const int per = s->n_kv * z->blocks;
    z->budget = (4 * n_cu + per - 1) / per;
    z->cap = s->S + z->budget;
    z->parts = 2 * z->budget;
    z->counters = (int64_t)s->S * per;
}

int64_t kqk_attn_workspace(const kq_attn_shape* s, int n_cu) { return 0; }

int kqk_launch_attn(const kq_paged_attn* a, const kqk_attn_sizes* z, void* work, hipStream_t st) {
    auto* const k = a->cache.type == KQ_TYPE_F16    ? kq_attn_kernel<KQ_TYPE_F16>
                    : a->cache.type == KQ_TYPE_BF16 ? kq_attn_kernel<KQ_TYPE_BF16>
                                                    : kq_attn_kernel<KQ_TYPE_I8>;
    hipLaunchKernelGGL(k, dim3((unsigned)a->shape.S, (unsigned)a->shape.n_q, (unsigned)a->shape.T),
                       dim3(64), 0, st, *a);
    return (int)hipGetLastError();
}

}
