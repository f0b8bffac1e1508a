// kq_kv.hip -- a paged cache of keys and values (gfx950): block tables and slots of
// a step's new tokens, and the rotation of queries and keys with the store into the
// cache.
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "kq_launch.h"

#pragma clang fp contract(off)

namespace {

// ------------------------------------------------------------------ plan

constexpr int PT = 1024;            // lanes of the plan's one workgroup
constexpr int MOST = (1 << 30) - 1; // of a length

struct PlanArg {
    kq_kv_plan p;
    int budget, cap;
    long long counters;
    int* items;                     // KQK_ITEM each
    int* count;
    int* counter;
};

struct Seq {
    int cached, fresh, held, from, end;  // keys [from, end) are read by its new tokens
    long long need;                      // pages
    bool narrow;
};

__device__ __forceinline__ int clamped(int v, int most) { return min(max(v, 0), most); }

__device__ __forceinline__ Seq load_seq(const kq_kv_plan& p, int s) {
    Seq q = {};
    if (s >= p.S) return q;
    q.cached = clamped(p.cached[s], MOST);
    q.fresh = p.n_new ? clamped(p.n_new[s], MOST) : 1;
    q.end = q.cached + q.fresh;
    if (p.table) {
        const int pages = (q.end + p.page - 1) / p.page;
        q.held = p.held ? clamped(p.held[s], p.table_stride)
                        : min((q.cached + p.page - 1) / p.page, p.table_stride);
        q.narrow = pages > p.table_stride;
        q.need = q.narrow ? 0 : max(0, pages - q.held);
    }
    const int w = p.shape.window;
    q.from = w ? max(0, q.cached + 1 - w) & ~31 : 0;
    return q;
}

__device__ __forceinline__ bool attended(const PlanArg& a, const Seq& q) {
    return a.items && q.fresh >= 1 && q.fresh <= a.p.shape.T;
}

// The sum before each lane's value over the workgroup, and all of it.
__device__ __forceinline__ long long wg_scan(long long v, long long* sm, long long* total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    long long in = v;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const long long o = __shfl_up(in, off);
        if (lane >= off) in += o;
    }
    __syncthreads();                      // (the last scan's sums have been read)
    if (lane == 63) sm[wave] = in;
    __syncthreads();
    long long before = 0, all = 0;
    for (int i = 0; i < PT / 64; i++) {
        if (i < wave) before += sm[i];
        all += sm[i];
    }
    *total = all;
    return before + in - v;
}

// The last i < n with first[i] <= v (first[0] is 0, the values ascend).
__device__ __forceinline__ int owner(const int* first, int n, int v) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (first[mid] <= v) lo = mid;
        else hi = mid;
    }
    return lo;
}

__device__ __forceinline__ int items_of(int keys, int share) {
    if (keys <= share) return 1;
    const int n = (keys + share - 1) / share;
    const int per = ((keys + n - 1) / n + 31) & ~31;
    return (keys + per - 1) / per;
}

__global__ __launch_bounds__(PT) void kq_kv_plan_kernel(PlanArg a) {
    __shared__ long long sm[PT / 64];
    __shared__ int first_tok[PT], first_page[PT], first_item[PT], first_part[PT];
    __shared__ int s_cached[PT], s_held[PT], s_from[PT], s_end[PT], s_fresh[PT];
    __shared__ bool s_ok[PT];
    const kq_kv_plan& p = a.p;
    const int tid = threadIdx.x;
    const long long room = p.table ? max(0, *p.n_free) : 0;
    for (long long i = tid; i < a.counters; i += PT) a.counter[i] = 0;
    int share = 0x7fffffc0;
    if (a.items && a.budget) {
        long long keys = 0, all;
        for (int s0 = 0; s0 < p.S; s0 += PT) {
            const Seq q = load_seq(p, s0 + tid);
            if (s0 + tid < p.S && attended(a, q)) keys += q.end - q.from;
        }
        wg_scan(keys, sm, &all);
        share = (int)min((long long)share, max(64ll, ((all + a.budget - 1) / a.budget + 31) & ~31ll));
    }
    long long tok0 = 0, page0 = 0, taken = 0, shorts = 0;
    int item0 = 0, part0 = 0;
    for (int s0 = 0; s0 < p.S; s0 += PT) {
        const int s = s0 + tid, n = min(PT, p.S - s0);
        const Seq q = load_seq(p, s);
        long long ntok, npage, nitem, npart, nshort, last;
        const long long tok = wg_scan(s < p.S ? q.fresh : 0, sm, &ntok);
        const long long pg = wg_scan(q.need, sm, &npage);
        const bool ok = !q.narrow && (q.need == 0 || page0 + pg + q.need <= room);
        const int from = ok ? q.from : 0, end = ok ? q.end : 0;
        const int items = s < p.S && attended(a, q) ? items_of(end - from, share) : 0;
        const int item = (int)wg_scan(items, sm, &nitem);
        const int parts = items > 1 ? items : 0;
        const int part = (int)wg_scan(parts, sm, &npart);
        wg_scan(s < p.S && !ok, sm, &nshort);
        wg_scan(ok ? q.need : 0, sm, &last);
        // (pages run out once: those who get theirs are the first that need any)
        taken += last;
        shorts += nshort;
        first_tok[tid] = (int)min(tok, 0x7fffffffll);
        first_page[tid] = (int)min(pg, 0x7fffffffll);
        first_item[tid] = item;
        first_part[tid] = part;
        s_cached[tid] = q.cached;
        s_held[tid] = q.held;
        s_from[tid] = from;
        s_end[tid] = end;
        s_fresh[tid] = q.fresh;
        s_ok[tid] = ok;
        if (s < p.S) {
            if (p.start) p.start[s] = (int)(tok0 + tok);
            if (p.lens) p.lens[s] = ok ? q.end : 0;
            if (p.held_out) p.held_out[s] = q.held + (ok ? (int)q.need : 0);
        }
        __syncthreads();
        // new pages, from the end of the free ones
        if (p.table)
            for (long long e = tid; e < npage && page0 + e < room; e += PT) {
                const int i = owner(first_page, n, (int)e);
                if (s_ok[i])
                    p.table[(long long)(s0 + i) * p.table_stride + s_held[i] + (int)(e - first_page[i])] =
                        p.free_pages[room - 1 - (page0 + e)];
            }
        // new tokens
        if (p.pos || p.slot)
            for (long long t = tid; t < ntok && tok0 + t < p.N; t += PT) {
                const int i = owner(first_tok, n, (int)t);
                const int pos = s_cached[i] + (int)(t - first_tok[i]);
                if (p.pos) p.pos[tok0 + t] = pos;
                if (!p.slot) continue;
                int slot = -1;
                if (s_ok[i]) {
                    const int b = pos / p.page, more = b - s_held[i];
                    const int page = more < 0 ? p.table[(long long)(s0 + i) * p.table_stride + b]
                                              : p.free_pages[room - 1 - (page0 + first_page[i] + more)];
                    if (page >= 0 && page < p.n_pages) slot = page * p.page + (pos - b * p.page);
                }
                p.slot[tok0 + t] = slot;
            }
        // the attention's items
        for (long long e = tid; e < nitem && item0 + e < a.cap; e += PT) {
            const int i = owner(first_item, n, (int)e), idx = (int)e - first_item[i];
            const int keys = s_end[i] - s_from[i], num = items_of(keys, share);
            const int per = ((keys + num - 1) / num + 31) & ~31;
            int* const o = a.items + (item0 + e) * KQK_ITEM;
            o[0] = s0 + i;
            o[1] = s_from[i] + idx * per;
            o[2] = min(s_end[i], s_from[i] + (idx + 1) * per);
            o[3] = num << 16 | idx;
            o[4] = part0 + first_part[i];
            o[5] = (int)(tok0 + first_tok[i]);
            o[6] = s_fresh[i];
            o[7] = s_end[i];
        }
        tok0 += ntok;
        page0 += npage;
        item0 += (int)nitem;
        part0 += (int)npart;
        __syncthreads();
    }
    if (tid == 0) {
        if (p.start) p.start[p.S] = (int)tok0;
        if (p.n_free_out) *p.n_free_out = (int)(room - taken);
        if (p.n_short) *p.n_short = (int)shorts;
        if (a.items) *a.count = min(item0, a.cap);
    }
}

// ----------------------------------------------------------------- store

typedef float f32x4 __attribute__((ext_vector_type(4)));

template <int TYPE>
__global__ __launch_bounds__(256) void kq_kv_store_kernel(kq_kv_store a, int lanes) {
    __shared__ double cs[KQ_KV_MAX_D / 2], sn[KQ_KV_MAX_D / 2];
    const kq_kv_cache& c = a.cache;
    const long tok = blockIdx.x;
    if (a.n_tokens && tok >= *a.n_tokens) return;
    const int half = a.rot / 2, D = c.D;
    if ((int)threadIdx.x < half) {
        const double angle = (double)a.pos[tok] * (double)a.freq[threadIdx.x];
        sincos(angle, &sn[threadIdx.x], &cs[threadIdx.x]);
    }
    __syncthreads();
    const long slot = a.slot[tok];
    const bool live = slot >= 0 && slot < (long)c.n_pages * c.page;
    const long page = live ? slot / c.page : 0, at = live ? slot - page * c.page : 0;
    const int rows = a.n_q + 2 * c.n_kv, per = 64 / lanes * 4;
    const int j0 = (threadIdx.x & (lanes - 1)) * 4;
    for (int r0 = blockIdx.y * per; r0 < rows; r0 += gridDim.y * per) {
        const int r = r0 + (int)threadIdx.x / lanes;
        const bool on = r < rows && j0 < D;
        const int head = r < a.n_q ? r : r < a.n_q + c.n_kv ? r - a.n_q : r - a.n_q - c.n_kv;
        const bool is_q = r < a.n_q, is_v = r >= a.n_q + c.n_kv;
        const float* const x = is_q ? a.q + tok * a.q_stride + (long)head * D
                             : is_v ? a.v + tok * a.v_stride + (long)head * D
                                    : a.k + tok * a.k_stride + (long)head * D;
        f32x4 y = (f32x4)0.0f;
        if (on) y = *reinterpret_cast<const f32x4*>(x + j0);
        // (q_out may be q: a row is one wave's, which reads it before it writes)
        f32x4 o = y;
        if (on && !is_v && j0 < a.rot) {
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int j = j0 + e;
                if (j >= a.rot) continue;
                const int other = a.interleaved ? j ^ 1 : j < half ? j + half : j - half;
                o[e] = x[other];
            }
        }
        if (on && !is_v && j0 < a.rot) {
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int j = j0 + e;
                if (j >= a.rot) continue;
                const int i = a.interleaved ? j >> 1 : j < half ? j : j - half;
                const bool lead = a.interleaved ? !(j & 1) : j < half;
                const double m = (double)y[e] * cs[i], n = (double)o[e] * sn[i];
                y[e] = (float)(lead ? m - n : m + n);
            }
        }
        if (is_q) {
            if (on) *reinterpret_cast<f32x4*>(a.q_out + tok * a.q_out_stride + (long)head * D + j0) = y;
            continue;
        }
        const long row = page * c.page_stride + head * c.head_stride + at * c.token_stride + j0;
        if constexpr (TYPE == KQ_TYPE_I8) {
            float amax = fmaxf(fmaxf(fabsf(y[0]), fabsf(y[1])), fmaxf(fabsf(y[2]), fabsf(y[3])));
            for (int off = 1; off < lanes; off <<= 1) amax = fmaxf(amax, __shfl_xor(amax, off));
            const float scale = __fdiv_rn(amax, 127.0f);
            const float inv = scale > 0.0f ? __fdiv_rn(1.0f, scale) : 0.0f;
            uint32_t w = 0;
#pragma unroll
            for (int e = 0; e < 4; e++)
                w |= ((uint32_t)min(127, max(-128, __float2int_rn(y[e] * inv))) & 0xffu) << (8 * e);
            if (on && live) {
                *reinterpret_cast<uint32_t*>((int8_t*)(is_v ? c.v : c.k) + row) = w;
                if (j0 == 0)
                    (is_v ? c.v_scale : c.k_scale)[(page * c.n_kv + head) * c.page + at] = scale;
            }
        } else if (on && live) {
            uint16_t h[4];
#pragma unroll
            for (int e = 0; e < 4; e++)
                h[e] = TYPE == KQ_TYPE_F16 ? __half_as_ushort(__float2half_rn(y[e]))
                                           : __bfloat16_as_ushort(__float2bfloat16(y[e]));
            *reinterpret_cast<uint2*>((uint16_t*)(is_v ? c.v : c.k) + row) =
                make_uint2(h[0] | (uint32_t)h[1] << 16, h[2] | (uint32_t)h[3] << 16);
        }
    }
}

}  // namespace

extern "C" int kqk_launch_kv_plan(const kq_kv_plan* p, const kqk_attn_sizes* z, hipStream_t st) {
    PlanArg a = {};
    a.p = *p;
    if (p->list) {
        a.budget = z->budget;
        a.cap = z->cap;
        a.counters = z->counters;
        a.count = (int*)p->list;
        a.items = a.count + KQK_LIST_HEAD;
        a.counter = a.items + (long)z->cap * KQK_ITEM;
    }
    hipLaunchKernelGGL(kq_kv_plan_kernel, dim3(1), dim3(PT), 0, st, a);
    return (int)hipGetLastError();
}

extern "C" int kqk_launch_kv_store(const kq_kv_store* a, int n_cu, hipStream_t st) {
    int lanes = 2;
    while (4 * lanes < a->cache.D) lanes *= 2;
    const int per = 64 / lanes * 4, rows = a->n_q + 2 * a->cache.n_kv;
    const int parts = a->N < n_cu ? (rows + per - 1) / per : 1;
    auto* const k = a->cache.type == KQ_TYPE_F16    ? kq_kv_store_kernel<KQ_TYPE_F16>
                    : a->cache.type == KQ_TYPE_BF16 ? kq_kv_store_kernel<KQ_TYPE_BF16>
                                                    : kq_kv_store_kernel<KQ_TYPE_I8>;
    hipLaunchKernelGGL(k, dim3((unsigned)a->N, (unsigned)parts), dim3(256), 0, st, *a, lanes);
    return (int)hipGetLastError();
}
