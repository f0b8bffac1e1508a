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
//
// One workgroup, or up to 16 for the slots of more than 4096 new tokens: a sequence a
// lane (more in rounds), sums over them by lanes' shifts, then new pages, new tokens and the
// attention's items over all lanes, each of which finds its sequence by bisection in LDS.
// A chain of latencies bounds it: lengths, sums, the pages that slots lie on (one
// sequence 5.0 us, 256 of up to four new tokens 8.6, with a list; 1.7 of it the launch).

constexpr int PT = 1024;            // lanes at most
constexpr int MOST = (1 << 30) - 1; // of a length

struct PlanArg {
    kq_kv_plan p;
    int cap, few;                   // (kqk_attn_sizes)
    int counters;
    int* items;                     // KQK_ITEM each
    int* count;
    int* counter;
};

struct Seq {
    uint32_t cached, fresh, held, need, from, end;   // keys [from, end) are read by its new tokens
    bool narrow, attended;
};

__device__ __forceinline__ uint32_t clamped(int v, int most) { return (uint32_t)min(max(v, 0), most); }
__device__ __forceinline__ uint32_t plus(uint32_t a, uint32_t b) { return __builtin_elementwise_add_sat(a, b); }

__device__ __forceinline__ Seq load_seq(const PlanArg& a, int s) {
    const kq_kv_plan& p = a.p;
    Seq q = {};
    if (s >= p.S) return q;
    const int cached = p.cached[s], fresh = p.n_new ? p.n_new[s] : 1, held = p.held ? p.held[s] : 0;
    q.cached = clamped(cached, MOST);
    q.fresh = clamped(fresh, MOST);
    q.end = q.cached + q.fresh;
    if (p.table) {
        const uint32_t page = (uint32_t)p.page, pages = (q.end + page - 1) / page;
        q.held = p.held ? clamped(held, p.table_stride)
                        : min((q.cached + page - 1) / page, (uint32_t)p.table_stride);
        q.narrow = pages > (uint32_t)p.table_stride;
        q.need = q.narrow || pages <= q.held ? 0 : pages - q.held;
    }
    const int w = p.shape.window;
    q.from = w && (int)q.cached + 1 > w ? (q.cached + 1 - w) & ~31u : 0;
    q.attended = a.items && q.fresh >= 1 && q.fresh <= (uint32_t)p.shape.T;
    return q;
}

// A step of a sum over the lanes before: DPP row_shr by 1 to 8, then a row's last lane
// to the next row and the second row's to the upper half.
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t scan_step(uint32_t x) {
    return plus(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, ROWS, 0xf, false));
}
__device__ __forceinline__ uint32_t wave_scan(uint32_t x) {
    x = scan_step<0x111, 0xf>(x);
    x = scan_step<0x112, 0xf>(x);
    x = scan_step<0x114, 0xf>(x);
    x = scan_step<0x118, 0xf>(x);
    x = scan_step<0x142, 0xa>(x);
    return scan_step<0x143, 0xc>(x);
}

// N sums (that stay at 2^32 - 1 from there on) over the lanes before each and over all.
template <int N>
__device__ __forceinline__ void wg_scan(const uint32_t (&v)[N], uint32_t (*sm)[PT / 64], uint32_t (&before)[N],
                                        uint32_t (&all)[N]) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int waves = blockDim.x >> 6;
    uint32_t in[N];
#pragma unroll
    for (int i = 0; i < N; i++) in[i] = wave_scan(v[i]);
    if (lane == 63)
#pragma unroll
        for (int i = 0; i < N; i++) sm[i][wave] = in[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; i++) {
        // the waves' sums, one a lane, summed in their turn
        const uint32_t w = wave_scan(lane < waves ? sm[i][lane] : 0);
        all[i] = (uint32_t)__builtin_amdgcn_readlane((int)w, 63);
        const uint32_t mine = wave ? (uint32_t)__builtin_amdgcn_readlane((int)w, wave - 1) : 0;
        // (the lane before's inclusive sum: exact also where sums stay at their most)
        const uint32_t prev = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)in[i], 0x138, 0xf, 0xf, false);
        before[i] = plus(mine, prev);
    }
}

// The last i < n with first[i] <= v (first[0] is 0, the values ascend), of K values at
// once, whose steps wait for LDS together.
template <int K>
__device__ __forceinline__ void owners(const uint32_t* first, int n, const uint32_t (&v)[K], int (&at)[K]) {
#pragma unroll
    for (int k = 0; k < K; k++) at[k] = 0;
    for (int step = n > 1 ? 1 << (31 - __clz(n - 1)) : 0; step; step >>= 1) {
#pragma unroll
        for (int k = 0; k < K; k++) {
            const int mid = at[k] + step;
            const uint32_t f = first[min(mid, n - 1)];
            at[k] = mid < n && f <= v[k] ? mid : at[k];
        }
    }
}
__device__ __forceinline__ int owner(const uint32_t* first, int n, uint32_t v) {
    const uint32_t w[1] = {v};
    int at[1];
    owners<1>(first, n, w, at);
    return at[0];
}

// An item's keys are a multiple of 128 (a step of 32 for each of four waves), but for a
// sequence's last.
constexpr uint32_t ROUND = 128;

// How many items keys take where one has at most `share`, and the keys of each.
__device__ __forceinline__ uint32_t items_of(uint32_t keys, uint32_t share, uint32_t* per) {
    *per = max(keys, 1u);
    if (keys <= share) return 1;
    const uint32_t n = (keys + share - 1) / share;
    *per = ((keys + n - 1) / n + ROUND - 1) / ROUND * ROUND;
    return (keys + *per - 1) / *per;
}

__device__ __forceinline__ void put_item(const PlanArg& a, uint32_t at, int s, uint32_t from, uint32_t to, uint32_t num,
                                         uint32_t idx, uint32_t part, uint32_t row, uint32_t fresh, uint32_t len) {
    int4* const o = reinterpret_cast<int4*>(a.items + (int64_t)at * KQK_ITEM);
    o[0] = make_int4(s, (int)from, (int)to, (int)(num << 16 | idx));
    o[1] = make_int4((int)part, (int)row, (int)fresh, (int)len);
}

__global__ __launch_bounds__(PT) void kq_kv_plan_kernel(const PlanArg a) {
    __shared__ uint32_t sm[8][4][PT / 64];
    __shared__ uint32_t first_tok[PT], first_page[PT], first_item[PT], s_cached[PT], s_held[PT], s_from[PT],
        s_end[PT], s_fresh[PT], s_part[PT];
    __shared__ bool s_ok[PT];
    const kq_kv_plan& p = a.p;
    const int tid = threadIdx.x, T = blockDim.x;
    const uint32_t many = T * gridDim.x;
    const bool head = blockIdx.x == 0;          // (the others only help with the tokens)
    const uint32_t room = p.table ? (uint32_t)max(0, *p.n_free) : 0;
    Seq q = load_seq(a, tid);
    for (int i = tid; head && i < a.counters; i += T) a.counter[i] = 0;
    uint32_t share = 0;
    if (head && a.items) {
        // The most keys that an item has: with keys / extra or more there are no more than
        // `extra` items beyond one a sequence.  Keys in units of ROUND, their lower and
        // upper 16 bits:
        uint32_t units[3] = {0, 0, 0}, before[3], all[3];
        for (int s0 = 0; s0 < p.S; s0 += T) {
            const Seq r = s0 ? load_seq(a, s0 + tid) : q;
            const uint32_t n = r.attended ? (r.end - r.from + ROUND - 1) / ROUND : 0;
            units[0] += n & 0xffff;
            units[1] += n >> 16;
            units[2] += r.attended;
        }
        wg_scan<3>(units, sm[0], before, all);
        const uint64_t total = ((uint64_t)all[1] << 16) + all[0];
        const uint32_t extra = a.cap - p.S, cap = all[2] + extra;
        // x / n rounded up, or a little more (x past 2^24), and 2^26 where it is above, which
        // is more units than a sequence has
        auto over = [](uint64_t x, uint32_t n) {
            if (x >= (uint64_t)n << 26) return 1u << 26;
            uint32_t y = (uint32_t)((float)x / (float)n);
            while ((uint64_t)y * n < x) y++;
            return y;
        };
        const uint32_t least = total * ROUND <= (uint64_t)a.few ? 1 : 2;
        uint32_t most = max(least, over(total, extra));
        if (p.S <= 64) {
            // Fewer, where that gives no more items either, by bisection (0.6 us a step where
            // there are several waves, and with many sequences little to gain; 64 ragged
            // streams' attention takes 103 us for 108 with it).
            const uint32_t mine = q.attended ? (q.end - q.from + ROUND - 1) / ROUND : 0;
            uint32_t lo = max(least, min(over(total, cap), most));
#pragma unroll 1
            for (int i = 0; i < 5 && lo < most; i++) {
                const uint32_t mid = (lo + most) / 2;
                uint32_t v[1] = {q.attended ? max(1u, over(mine, mid)) : 0}, b1[1], n1[1];
                wg_scan<1>(v, sm[3 + i], b1, n1);
                if (n1[0] <= cap) most = mid;
                else lo = mid + 1;
            }
        }
        share = min(most, 0x1ffffffu) * ROUND;
    }
    uint32_t tok0 = 0, page0 = 0, taken = 0, shorts = 0, item0 = 0, part0 = 0;
    for (int s0 = 0; s0 < p.S; s0 += T) {
        const int s = s0 + tid, n = min(T, p.S - s0);
        if (s0) q = load_seq(a, s);
        uint32_t b1[2], n1[2], b2[4], n2[4], per;
        const uint32_t v1[2] = {q.fresh, q.need};
        wg_scan<2>(v1, sm[1], b1, n1);
        const bool ok = !q.narrow && (q.need == 0 || plus(plus(page0, b1[1]), q.need) <= room);
        const uint32_t from = ok ? q.from : 0, end = ok ? q.end : 0;
        const uint32_t items = head && q.attended ? items_of(end - from, share, &per) : 0, parts = items > 1 ? items : 0;
        // (pages run out once: those who get theirs are the first that need any)
        const uint32_t v2[4] = {items, parts, s < p.S && !ok ? 1u : 0u, ok ? q.need : 0u};
        wg_scan<4>(v2, sm[2], b2, n2);
        first_tok[tid] = b1[0];
        first_page[tid] = b1[1];
        // (items: first those of sequences with several, which are the longer ones)
        const uint32_t single = items == 1 ? 1 : 0;
        first_item[tid] = b2[1];
        s_part[tid] = b2[1];
        if (single) {
            const uint32_t e = item0 + n2[1] + (b2[0] - b2[1]);
            if (e < (uint32_t)a.cap) put_item(a, e, s, from, end, 1, 0, 0, tok0 + b1[0], q.fresh, end);
        }
        s_cached[tid] = q.cached;
        s_held[tid] = q.held;
        s_from[tid] = from;
        s_end[tid] = end;
        s_fresh[tid] = q.fresh;
        s_ok[tid] = ok;
        if (head && s < p.S) {
            if (p.start) p.start[s] = (int)(tok0 + b1[0]);
            if (p.lens) p.lens[s] = ok ? (int)q.end : 0;
            if (p.held_out) p.held_out[s] = (int)(q.held + (ok ? q.need : 0));
        }
        __syncthreads();
        // new pages, from the end of the free ones
        if (head && p.table)
            for (uint32_t e = tid; e < n1[1] && plus(page0, e) < room; e += T) {
                const int i = owner(first_page, n, e);
                if (s_ok[i])
                    p.table[(int64_t)(s0 + i) * p.table_stride + s_held[i] + (e - first_page[i])] =
                        p.free_pages[room - 1 - (page0 + e)];
            }
        // new tokens, four a lane at a time, as their pages are a memory's latency away
        if (p.pos || p.slot)
            for (uint32_t t0 = tid + blockIdx.x * T; t0 < n1[0] && plus(tok0, t0) < (uint32_t)p.N; t0 += 4 * many) {
                uint32_t tok[4], pos[4], b[4];
                int page[4], at[4];
#pragma unroll
                for (int u = 0; u < 4; u++) tok[u] = min(t0 + u * many, n1[0] - 1);
                owners<4>(first_tok, n, tok, at);
#pragma unroll
                for (int u = 0; u < 4; u++) {
                    if (t0 + u * many >= n1[0]) break;
                    const int i = at[u];
                    pos[u] = s_cached[i] + (tok[u] - first_tok[i]);
                    b[u] = pos[u] / (uint32_t)p.page;
                    page[u] = -1;
                    if (p.slot && s_ok[i])
                        page[u] = b[u] < s_held[i] ? p.table[(int64_t)(s0 + i) * p.table_stride + b[u]]
                                                   : p.free_pages[room - 1 - (page0 + first_page[i] + (b[u] - s_held[i]))];
                }
#pragma unroll
                for (int u = 0; u < 4; u++) {
                    const uint32_t t = t0 + u * many;
                    if (t >= n1[0] || plus(tok0, t) >= (uint32_t)p.N) break;
                    if (p.pos) p.pos[tok0 + t] = (int)pos[u];
                    const bool ok = (uint32_t)page[u] < (uint32_t)p.n_pages;
                    if (p.slot) p.slot[tok0 + t] = ok ? page[u] * p.page + (int)(pos[u] - b[u] * (uint32_t)p.page) : -1;
                }
            }
        // the attention's items
        for (uint32_t e = tid; e < n2[1] && item0 + e < (uint32_t)a.cap; e += T) {
            const int i = owner(first_item, n, e);
            const uint32_t idx = e - first_item[i], num = items_of(s_end[i] - s_from[i], share, &per);
            put_item(a, item0 + e, s0 + i, s_from[i] + idx * per, min(s_end[i], s_from[i] + (idx + 1) * per), num, idx,
                     part0 + s_part[i], tok0 + first_tok[i], s_fresh[i], s_end[i]);
        }
        tok0 = plus(tok0, n1[0]);
        page0 = plus(page0, n1[1]);
        item0 += n2[0];
        part0 += n2[1];
        shorts += n2[2];
        taken += n2[3];
        __syncthreads();
    }
    if (head && tid == 0) {
        if (p.start) p.start[p.S] = (int)tok0;
        if (p.n_free_out) *p.n_free_out = (int)(room - taken);
        if (p.n_short) *p.n_short = (int)shorts;
        if (a.items) *a.count = min((int)item0, a.cap);
    }
}

// ----------------------------------------------------------------- store

typedef float f32x4 __attribute__((ext_vector_type(4)));

// One workgroup a token (several, where tokens are few): its angles' cosines and sines
// once in LDS, then its heads' rows, `lanes` lanes of four values each, U rows a lane
// in flight.  The partners of a rotation are read a second time, from the cache.
// Memory bounds many tokens (4096 of 16 + 2 x 8 heads of 128 to bfloat16: 26 us, 4.5 TB/s;
// a SIMD's binary64 products, sums and conversions are 1152 of 7400 instructions, at 8 clocks a sixth of
// the time), one launch few (one of 24 + 2 x 4 heads of 256: 3.9 us).
constexpr int U = 4;

template <int TYPE>
__global__ __launch_bounds__(256) void kq_kv_store_kernel(kq_kv_store a, int lanes) {
    __shared__ double cs[KQ_KV_MAX_D / 2], sn[KQ_KV_MAX_D / 2];
    const kq_kv_cache& c = a.cache;
    const long tok = blockIdx.x;
    if (a.n_tokens && tok >= *a.n_tokens) return;
    const int half = a.rot / 2, D = c.D;
    const long slot = a.slot[tok];
    const bool live = slot >= 0 && slot < (long)c.n_pages * c.page;
    const long page = live ? slot / c.page : 0, at = live ? slot - page * c.page : 0;
    const int rows = a.n_q + 2 * c.n_kv, per = 256 / lanes;
    const int j0 = (threadIdx.x & (lanes - 1)) * 4, r1 = threadIdx.x / lanes;
    // four partners in a row, or four pairs of neighbours, at 16-byte addresses
    const bool even = a.interleaved ? a.rot % 4 == 0 : half % 4 == 0;
    bool first = true;
    for (int r0 = blockIdx.y * per; r0 < rows; r0 += gridDim.y * per * U) {
        f32x4 y[U], o[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int r = r0 + u * gridDim.y * per + r1;
            y[u] = o[u] = (f32x4)0.0f;
            if (r >= rows || j0 >= D) continue;
            const float* const x = r < a.n_q           ? a.q + tok * a.q_stride + (long)r * D
                                   : r < a.n_q + c.n_kv ? a.k + tok * a.k_stride + (long)(r - a.n_q) * D
                                                        : a.v + tok * a.v_stride + (long)(r - a.n_q - c.n_kv) * D;
            y[u] = *reinterpret_cast<const f32x4*>(x + j0);
            if (r >= a.n_q + c.n_kv || j0 >= a.rot) continue;
            if (a.interleaved) {
                o[u] = (f32x4){y[u][1], y[u][0], y[u][3], y[u][2]};
            } else if (even) {
                o[u] = *reinterpret_cast<const f32x4*>(x + (j0 < half ? j0 + half : j0 - half));
            } else {
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const int j = j0 + e;
                    if (j < a.rot) o[u][e] = x[j < half ? j + half : j - half];
                }
            }
        }
        if (first) {
            if ((int)threadIdx.x < half) {
                const double angle = (double)a.pos[tok] * (double)a.freq[threadIdx.x];
                sincos(angle, &sn[threadIdx.x], &cs[threadIdx.x]);
            }
            __syncthreads();
            first = false;
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int r = r0 + u * gridDim.y * per + r1;
            const bool on = r < rows && j0 < D;
            const bool is_q = r < a.n_q, is_v = r >= a.n_q + c.n_kv;
            const int head = is_q ? r : is_v ? r - a.n_q - c.n_kv : r - a.n_q;
            if (on && !is_v && j0 < a.rot) {
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const int j = j0 + e;
                    if (j >= a.rot) continue;
                    const int i = a.interleaved ? j >> 1 : j < half ? j : j - half;
                    const bool lead = a.interleaved ? !(j & 1) : j < half;
                    const double m = (double)y[u][e] * cs[i], n = (double)o[u][e] * sn[i];
                    y[u][e] = (float)(lead ? m - n : m + n);
                }
            }
            if (is_q) {
                if (on) *reinterpret_cast<f32x4*>(a.q_out + tok * a.q_out_stride + (long)head * D + j0) = y[u];
                continue;
            }
            const long row = page * c.page_stride + head * c.head_stride + at * c.token_stride + j0;
            if constexpr (TYPE == KQ_TYPE_I8) {
                float amax = fmaxf(fmaxf(fabsf(y[u][0]), fabsf(y[u][1])), fmaxf(fabsf(y[u][2]), fabsf(y[u][3])));
                for (int off = 1; off < lanes; off <<= 1) amax = fmaxf(amax, __shfl_xor(amax, off));
                const float scale = __fdiv_rn(amax, 127.0f);
                const float inv = scale > 0.0f ? __fdiv_rn(1.0f, scale) : 0.0f;
                uint32_t w = 0;
#pragma unroll
                for (int e = 0; e < 4; e++)
                    w |= ((uint32_t)min(127, max(-128, __float2int_rn(y[u][e] * inv))) & 0xffu) << (8 * e);
                if (on && live) {
                    *reinterpret_cast<uint32_t*>((int8_t*)(is_v ? c.v : c.k) + row) = w;
                    if (j0 == 0) (is_v ? c.v_scale : c.k_scale)[(page * c.n_kv + head) * c.page + at] = scale;
                }
            } else if (on && live) {
                uint16_t h[4];
#pragma unroll
                for (int e = 0; e < 4; e++)
                    h[e] = TYPE == KQ_TYPE_F16 ? __half_as_ushort(__float2half_rn(y[u][e]))
                                               : __bfloat16_as_ushort(__float2bfloat16(y[u][e]));
                *reinterpret_cast<uint2*>((uint16_t*)(is_v ? c.v : c.k) + row) =
                    make_uint2(h[0] | (uint32_t)h[1] << 16, h[2] | (uint32_t)h[3] << 16);
            }
        }
    }
}

}  // namespace

extern "C" int kqk_launch_kv_plan(const kq_kv_plan* p, const kqk_attn_sizes* z, hipStream_t st) {
    PlanArg a = {};
    a.p = *p;
    if (p->list) {
        a.cap = z->cap;
        a.few = z->few;
        a.counters = (int)z->counters;
        a.count = (int*)p->list;
        a.items = a.count + KQK_LIST_HEAD;
        a.counter = a.items + (long)z->cap * KQK_ITEM;
    }
    // A lane for each sequence, and for each new token that there may be; of many
    // tokens (14119: one workgroup 17 us, this 8.6) several workgroups, each of
    // which takes the sums for itself, unless the first writes over what they read
    // (`held` and n_free in place: 17 us).
    int lanes = p->S > p->N ? p->S : p->N;
    lanes = lanes > PT ? PT : (lanes + 63) / 64 * 64;
    const bool apart = (!p->held_out || p->held_out != p->held) && (!p->n_free_out || p->n_free_out != p->n_free);
    const int groups = !apart || p->N <= 4096 ? 1 : p->N >= 16 * 2048 ? 16 : p->N / 2048;
    hipLaunchKernelGGL(kq_kv_plan_kernel, dim3((unsigned)groups), dim3((unsigned)lanes), 0, st, a);
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
