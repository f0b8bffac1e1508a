// kq_attn.hip -- attention of a few new tokens over a paged cache (gfx950).
//
//   out = sum_j p_j v_j,  p = softmax over the keys j that a token sees of scale q . k_j
//
// The rows of a sequence and a head of keys are its new tokens' queries of the G =
// n_q / n_kv heads that read it; a workgroup takes 16 of them and an item of the list
// (a share of the sequence's keys), each of its waves every fourth step of 32 keys.  One
// pass, with a running maximum m and sum l of each row:
//   S^T = K Q^T   16 keys x 16 rows a matrix instruction, K as it lies in the cache
//                 (a lane has 8 values of one key), Q^T from LDS
//   p = 2^(S - m), in the layout that S^T has: 8 keys of a row a lane, which is that
//                 of the second product's right operand if the keys of a step are
//                 taken in the order 4 g + j, 16 + 4 g + j (lane group g)
//   O^T = V^T P^T a lane loads 8 (or 4) neighbouring values of those 8 keys; an
//                 operand for value t of each is one byte permutation a register
// so that keys and values go from memory to registers and matrix cores without LDS.
// Queries and weights are rounded to two binary16 numbers (22 bits: queries with a power
// of two a row, weights times 2^9, with int8 weights times their values' scales and a
// power of two a row) where keys are binary16 or int8, to three bfloat16 numbers (24
// bits) where they are bfloat16.  Matrix work is far from full, so that the further
// products are free.
// Long caches are bound by memory (16 / 8 heads of 128, binary16, 16 sequences of 8192:
// 101 us, 5.3 TB/s; 24 / 4 of 256, bfloat16, 64 of 8192: 375 us, 5.7), short ones by a
// chain of latencies: item, pages, keys, a step, the join of waves (one sequence of 32:
// 5.9 us, heads of 256 7.8), and 4 to 5 us for a join of items.  Two tiles of 16 rows a
// wave share a step's operands but take all of a SIMD's registers: 8 sequences of 8 new
// tokens, 24 / 4 heads of 256, of 32 / 1000 to 4000 / 4096 keys took 14 / 64 / 57 us, which
// one takes in 9.5 / 43 / 56 to 60 (with 32 keys a step; 9 / 50 / 71 before).  8 waves a
// workgroup took 96 us for 82 with 200 sequences of 500 keys, and no less with few.
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "kq_launch.h"

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef u32x4 u32x4a __attribute__((aligned(8)));
struct __attribute__((aligned(4))) F4 { float v[4]; };    // four floats at any 4-byte address

struct AttnArg {
    const uint8_t* k;
    const uint8_t* v;
    const float* ks;
    const float* vs;
    const float* q;
    float* out;
    const int* table;
    const int* start;
    const int* lens;
    const int* items;           // NULL: workgroup x is sequence x
    const int* count;
    int* counter;
    float* part;                // partial results: parts x n_kv x R rows of D
    float2* ml;                 // and their maximum and sum
    int64_t q_stride, out_stride;
    int64_t page_b, head_b;     // cache strides in bytes
    uint32_t tok_b, page_s;     // (page_s: scales of a page)
    uint64_t div, kv_div, blocks_div;    // page / 16, n_kv and 8 blocks by multiplication
    float qscale;               // scale log2 e
    int div_shift, S, T, G, R, n_kv, D, window, N, page, n_pages, table_stride, cap, parts, blocks;
};

__device__ __forceinline__ uint32_t perm(uint32_t hi, uint32_t lo, uint32_t sel) {
    return __builtin_amdgcn_perm(hi, lo, sel);
}

// Maximum (sum) over the four lanes of a row: lanes c, 16 + c, 32 + c, 48 + c.
__device__ __forceinline__ float max4(float x) {
    auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
}
__device__ __forceinline__ float sum4(float x) {
    auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(a[0]) + __uint_as_float(a[1]);
}

// Two binary32 values as 16-bit ones in NP registers whose sum they are.
template <int NP>
__device__ __forceinline__ void split(float a, float b, uint32_t* o) {
    if constexpr (NP == 2) {
        const f16x2 h = {(_Float16)a, (_Float16)b};
        const f16x2 l = {(_Float16)(a - (float)h[0]), (_Float16)(b - (float)h[1])};
        o[0] = __builtin_bit_cast(uint32_t, h);
        o[1] = __builtin_bit_cast(uint32_t, l);
    } else {
        // by truncation: 8 bits each, nothing is left over
        const uint32_t top = 0xffff0000u;
        o[0] = perm(__float_as_uint(b), __float_as_uint(a), 0x07060302);
        a -= __uint_as_float(__float_as_uint(a) & top);
        b -= __uint_as_float(__float_as_uint(b) & top);
        o[1] = perm(__float_as_uint(b), __float_as_uint(a), 0x07060302);
        a -= __uint_as_float(__float_as_uint(a) & top);
        b -= __uint_as_float(__float_as_uint(b) & top);
        o[2] = perm(__float_as_uint(b), __float_as_uint(a), 0x07060302);
    }
}

// Two int8 values, in the lower bytes of a register's halves, as binary16 numbers: 1024
// + 128 + the value by its bits, less 1152.
__device__ __forceinline__ uint32_t halves(uint32_t u) {
    const f16x2 off = {(_Float16)1152.0f, (_Float16)1152.0f};
    return __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2, u ^ 0x64806480u) - off);
}

template <int NP>
__device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
    if constexpr (NP == 2)
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a),
                                                      __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a),
                                                       __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

constexpr int NW = 4;           // waves of a workgroup

__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }

// DM: values of a head at most (D itself where EXACT); TILED: the page is a multiple
// of 16 tokens, so that 16 keys lie on one page.
template <int TYPE, int DM, bool EXACT, bool TILED>
__global__ __launch_bounds__(64 * NW) __attribute__((amdgpu_waves_per_eu(2)))
void kq_attn_kernel(const AttnArg a) {
    constexpr int NP = TYPE == KQ_TYPE_BF16 ? 3 : 2;      // numbers for a query or weight
    constexpr int ES = TYPE == KQ_TYPE_I8 ? 1 : 2;
    constexpr int NCH = DM / 32;                          // steps of 32 values of the first product
    constexpr bool WIDE = TYPE == KQ_TYPE_I8 && EXACT;    // int8 keys in loads of 16
    constexpr int W = DM >= 128 ? 8 : 4;                  // values a lane of a key in the second
    constexpr int NB = DM / (16 * W);
    constexpr int VW = W * ES / 4;                        // registers of W values
    constexpr int OS = DM + 4;                            // a row of sums in LDS
    constexpr int QB = NP * 16 * DM * 2, OB = NW * 16 * OS * 4;
    __shared__ __attribute__((aligned(16))) uint8_t lds[QB > OB ? QB : OB];
    __shared__ float2 s_ml[NW][16], s_all[16];
    __shared__ float s_inv[16];
    __shared__ int s_last, s_odd[NW][2];
    __shared__ uint32_t s_inf[ES == 2 ? DM : 1];

    const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
    const int c = lane & 15, g = lane >> 4, D = EXACT ? DM : a.D, G = a.G;
    // Item after item, of each all heads and blocks of rows: those beyond the list's come
    // last (head after head instead, 64 workgroups with 64 more in front of each other's
    // took 22.6 us for 17.3).  Blocks of rows of one item and head are eight workgroups
    // apart, which puts them on one XCD, in whose L2 the keys are.
    const int eight = (int)((uint64_t)blockIdx.x * a.blocks_div >> 40), rest = blockIdx.x - 8 * a.blocks * eight;
    const int z = rest >> 3, pair = 8 * eight + (rest & 7);
    int s = (int)((uint64_t)(uint32_t)pair * a.kv_div >> 40);
    const int h = pair - s * a.n_kv;
    int k0 = 0, k1, num = 1, idx = 0, part = 0, row0, n, len;
    if (a.items) {
        // (the item is read with the number of items, not after it: the list reaches to cap)
        const int* const it = a.items + min(s, a.cap - 1) * KQK_ITEM;
        const int at = s;
        s = it[0];
        k0 = it[1];
        k1 = it[2];
        num = it[3] >> 16;
        idx = it[3] & 0xffff;
        part = it[4];
        row0 = it[5];
        n = it[6];
        len = it[7];
        if ((at >= min(a.cap, *a.count)) | (s < 0) | (s >= a.S) | (k0 < 0) | (num < 1) |
            ((num > 1) & ((part < 0) | (idx >= num) | (part > a.parts - num))))
            return;
    } else {
        if (s >= a.S) return;
        row0 = a.start ? a.start[s] : s;
        n = a.start ? a.start[s + 1] - row0 : 1;
        k1 = len = a.lens[s];
        if (a.window) k0 = max(0, len - n + 1 - a.window);
    }
    if (n < 1 || n > a.T) return;
    const int first = 16 * z, live = min(16, n * G - first);      // rows of this workgroup
    if (live <= 0) return;
    const int* const table = a.table + (int64_t)s * a.table_stride;
    k0 &= ~31;
    k1 = (int)min((int64_t)min(k1, 0x7fff0000), (int64_t)a.table_stride * a.page);
    const uint8_t* const kh = a.k + h * a.head_b;
    const uint8_t* const vh = a.v + h * a.head_b;

    int lo, hi;                             // the keys that a lane's row sees
    float m, l;
    f32x4 acc[NB][W];
    constexpr int VE0 = 11;                 // int8: the sums are acc 2^(ve - 137), of one ve a row
    int ve;
    // An infinity or NaN among the values would reach rows that do not see its key, and
    // an infinity as NaN those that do, as 0 times itself.  Where a sum ends as no
    // number all are taken again without such values, which are then added alone.
    // So are sums past 2^96, of large bfloat16 values, and rows in which they are that still
    // once more, with weights (and their sum) times 2^-40: 2^30 values of any size stay
    // finite, where the result is.  (Rows of other sums keep theirs, as 2^-40 costs small
    // values bits.)
    // Rows whose weights' sum is no number stay as they are: so are all of their sums.
    int pass = 0;
    float less = 0.0f;
    int odd0 = 0x7fffffff, odd1 = 0;        // keys among which are this wave's with such values
#pragma unroll 1
    while (true) {
        // ---- queries: as 16-bit numbers in LDS, in the right operand's layout
        constexpr int QO = (DM / 8 + 15) / 16;
        const int qr = tid >> 4;            // 16 lanes a row
        f32x4 qv[QO][2];
        {
            const int64_t tok = (int64_t)row0 + (first + qr) / G;
            const bool on = qr < live && tok >= 0 && tok < a.N;
            const float* const q = a.q + tok * a.q_stride + (int64_t)(h * G + (first + qr) % G) * D;
#pragma unroll
            for (int o = 0; o < QO; o++) {
                const int d = 8 * (c + 16 * o);
                qv[o][0] = qv[o][1] = (f32x4)0.0f;
                if (on && d < D) {
                    qv[o][0] = *reinterpret_cast<const f32x4*>(q + d);
                    qv[o][1] = *reinterpret_cast<const f32x4*>(q + d + 4);
                }
            }
        }

        // ---- where a step's keys lie
        int pg[2];                     // pages of the next step's keys
        auto fetch = [&](int kb) {
#pragma unroll
            for (int t = 0; t < 2; t++) {
                uint32_t b;
                if constexpr (TILED) b = (uint32_t)(((uint64_t)(uint32_t)(kb / 16 + t) * a.div) >> a.div_shift);
                else b = (uint32_t)(kb + 16 * t + c) / (uint32_t)a.page;
                pg[t] = b < (uint32_t)a.table_stride ? table[b] : -1;
            }
        };
        u32x4 kr[2][WIDE ? NCH / 2 : NCH], vr[8][NB];
        float ksr[8], vsr[8];
        bool have[2];                  // the keys' pages are pages
        const uint8_t* vp[8];
        int64_t sp[2];
        const uint32_t klane = (TILED ? c * a.tok_b : 0u) + (WIDE ? 16 : 8 * ES) * g;
        const uint32_t vlane = (TILED ? 4 * g * a.tok_b : 0u) + W * ES * c;
        auto octet = [&](int ch) { return EXACT || 32 * ch + 8 * g < D; };
        auto load_k = [&](int kb) {
#pragma unroll
            for (int t = 0; t < 2; t++) {
                // (a key that is not there is read as the first one of the first page)
                int page = TILED ? uniform(pg[t]) : pg[t], at;
                have[t] = (uint32_t)page < (uint32_t)a.n_pages;
                page = have[t] ? page : 0;
                if constexpr (TILED) {
                    const uint32_t b = (uint32_t)(((uint64_t)(uint32_t)(kb / 16 + t) * a.div) >> a.div_shift);
                    at = kb + 16 * t - (int)(b * (uint32_t)a.page);
                } else {
                    at = (int)((uint32_t)(kb + 16 * t + c) % (uint32_t)a.page);
                }
                at = have[t] ? at : 0;
                const int64_t o = (uint32_t)page * a.page_b + (int64_t)((uint64_t)(uint32_t)at * a.tok_b);
#pragma unroll
                for (int j = 0; j < 4; j++)
                    vp[4 * t + j] = vh + (TILED ? o + j * a.tok_b : (int64_t)__shfl(o, 4 * g + j));
                sp[t] = (int64_t)((uint64_t)(uint32_t)page * a.page_s) + (h * a.page + at);
#pragma unroll
                for (int ch = 0; ch < NCH; ch++) {
                    if (!EXACT && 32 * ch >= D) continue;
                    const uint8_t* const x = kh + o + (klane + (WIDE || octet(ch) ? 32 * ES * ch : -8 * ES * g));
                    if constexpr (WIDE) {
                        if (ch % 2 == 0) kr[t][ch / 2] = *reinterpret_cast<const u32x4a*>(x);
                    } else if constexpr (ES == 2) {
                        kr[t][ch] = *reinterpret_cast<const u32x4*>(x);
                    } else {
                        const u32x2 y = *reinterpret_cast<const u32x2*>(x);
                        kr[t][ch][0] = y[0];
                        kr[t][ch][1] = y[1];
                    }
                }
                if constexpr (TYPE == KQ_TYPE_I8 && TILED) {
                    const F4 x = *reinterpret_cast<const F4*>(a.ks + sp[t] + 4 * g);
#pragma unroll
                    for (int j = 0; j < 4; j++) ksr[4 * t + j] = x.v[j];
                } else if constexpr (TYPE == KQ_TYPE_I8) {
                    ksr[t] = a.ks[sp[t]];
                }
            }
        };
        auto load_v = [&]() {
#pragma unroll
            for (int j = 0; j < 8; j++)
#pragma unroll
                for (int b = 0; b < NB; b++) {
                    const uint8_t* const x = vp[j] + (EXACT || W * c + 16 * W * b < D ? vlane + 16 * W * ES * b
                                                                                     : vlane - W * ES * c);
                    if constexpr (VW == 4) {
                        vr[j][b] = *reinterpret_cast<const u32x4*>(x);
                    } else if constexpr (VW == 2) {
                        const u32x2 y = *reinterpret_cast<const u32x2*>(x);
                        vr[j][b][0] = y[0];
                        vr[j][b][1] = y[1];
                    } else {
                        vr[j][b][0] = *reinterpret_cast<const uint32_t*>(x);
                    }
                }
            if constexpr (TYPE == KQ_TYPE_I8) {
#pragma unroll
                for (int t = 0; t < 2; t++) {
                    if constexpr (TILED) {
                        const F4 x = *reinterpret_cast<const F4*>(a.vs + sp[t] + 4 * g);
#pragma unroll
                        for (int j = 0; j < 4; j++) vsr[4 * t + j] = x.v[j];
                    } else {
                        vsr[t] = a.vs[sp[t]];
                    }
                }
            }
        };

        int kb = k0 + 32 * wave;
        if (kb < k1) {
            fetch(kb);
            load_k(kb);
            load_v();
            if (kb + 32 * NW < k1) fetch(kb + 32 * NW);
        }

        u32x4* const ql = reinterpret_cast<u32x4*>(lds);
        {
            float inv = 1.0f, f = 1.0f, top = 0.0f;
#pragma unroll
            for (int o = 0; o < QO; o++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    qv[o][0][e] *= a.qscale;
                    qv[o][1][e] *= a.qscale;
                    top = fmaxf(top, fmaxf(fabsf(qv[o][0][e]), fabsf(qv[o][1][e])));
                }
            if constexpr (NP == 2) {
                // the row times a power of two, its largest value from 2^13 to 2^14
#pragma unroll
                for (int off = 1; off < 16; off <<= 1) top = fmaxf(top, __shfl_xor(top, off));
                if (top > 0.0f && top < INFINITY) {
                    const int e = min(126, 140 - (int)(__float_as_uint(top) >> 23));
                    f = __uint_as_float((uint32_t)(127 + e) << 23);
                    inv = __uint_as_float((uint32_t)(127 - e) << 23);
                }
                if (c == 0) s_inv[qr] = inv;
            }
#pragma unroll
            for (int o = 0; o < QO; o++) {
                if (DM % 128 && c + 16 * o >= DM / 8) continue;
                u32x4 w[NP];
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    uint32_t p[NP];
                    split<NP>(qv[o][e >> 1][2 * (e & 1)] * f, qv[o][e >> 1][2 * (e & 1) + 1] * f, p);
#pragma unroll
                    for (int j = 0; j < NP; j++) w[j][e] = p[j];
                }
#pragma unroll
                for (int j = 0; j < NP; j++) ql[(j * (DM / 8) + c + 16 * o) * 16 + qr] = w[j];
            }
        }
        __syncthreads();

        // ---- the lane's row (those behind the last see everything: their sums are nobody's)
        {
            const int last = len - n + (first + c) / G;
            lo = c < live && a.window ? last + 1 - a.window : 0;
            hi = c < live ? min(last + 1, k1) : k1;
        }
        const float inv = NP == 2 ? s_inv[c] : 1.0f;
        m = -INFINITY;
        l = 0.0f;
        ve = VE0;
#pragma unroll
        for (int b = 0; b < NB; b++)
#pragma unroll
            for (int t = 0; t < W; t++) acc[b][t] = (f32x4)0.0f;
        // keys within [all_lo, all_hi) are seen by all rows
        const int all_hi = min(k1, len - n + first / G + 1);
        const int all_lo = a.window ? len - n + (first + live - 1) / G + 1 - a.window : 0;

        // ---- steps
#pragma unroll 1
        for (; kb < k1; kb += 32 * NW) {
            bool ok[2], all_ok = true;
#pragma unroll
            for (int t = 0; t < 2; t++) {
                ok[t] = have[t];
                all_ok &= ok[t];
            }
            const bool full = kb >= all_lo && kb + 32 <= all_hi && (TILED ? all_ok : __all(all_ok));
            // (queries are read in each step: the compiler would keep them in registers)
            uint32_t qat = WIDE ? 32 * g + c : lane;
            asm volatile("" : "+v"(qat));
            f32x4 sc[2];
#pragma unroll
            for (int t = 0; t < 2; t++) sc[t] = (f32x4)0.0f;
#pragma unroll
            for (int ch = 0; ch < NCH; ch++) {
                if (!EXACT && 32 * ch >= D) continue;
                u32x4 x[2];
#pragma unroll
                for (int t = 0; t < 2; t++) {
                    if constexpr (TYPE == KQ_TYPE_I8) {
                        const uint32_t y0 = WIDE ? kr[t][ch / 2][2 * (ch & 1)] : kr[t][ch][0];
                        const uint32_t y1 = WIDE ? kr[t][ch / 2][2 * (ch & 1) + 1] : kr[t][ch][1];
                        x[t][0] = halves(perm(0, y0, 0x0c010c00));
                        x[t][1] = halves(perm(0, y0, 0x0c030c02));
                        x[t][2] = halves(perm(0, y1, 0x0c010c00));
                        x[t][3] = halves(perm(0, y1, 0x0c030c02));
                    } else {
                        x[t] = kr[t][ch];
                    }
                    if (!EXACT && !octet(ch)) x[t] = (u32x4)0u;
                }
                // (a lane's 8 values of chunk ch are the (4 ch + g)th of the row, WIDE: the
                // (8 (ch / 2) + 2 g + ch % 2)th)
#pragma unroll
                for (int j = 0; j < NP; j++) {
                    const u32x4 y = ql[(j * (DM / 8) + (WIDE ? 8 * (ch / 2) + (ch & 1) : 4 * ch)) * 16 + qat];
#pragma unroll
                    for (int t = 0; t < 2; t++) sc[t] = mfma<NP>(x[t], y, sc[t]);
                }
            }
            __builtin_amdgcn_sched_barrier(0);
            float kscale[8], vscale[8];
            if constexpr (TYPE == KQ_TYPE_I8) {
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    kscale[j] = TILED ? ksr[j] : __shfl(ksr[j >> 2], 4 * g + (j & 3));
                    vscale[j] = TILED ? vsr[j] : __shfl(vsr[j >> 2], 4 * g + (j & 3));
                }
            }
            // which of the lane's keys are there at all, bit j: key 16 (j / 4) + 4 g + j % 4
            uint32_t there = 0xff;
            if (!full) {
                uint32_t p = 0;
#pragma unroll
                for (int t = 0; t < 2; t++)
                    p |= (TILED ? (ok[t] ? 15u : 0u) : (uint32_t)(__ballot(ok[t]) >> (4 * g)) & 15u) << (4 * t);
                there = 0;
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const int key = kb + 16 * (j >> 2) + 4 * g + (j & 3);
                    if (key < k1 && (p >> j & 1)) there |= 1u << j;
                }
                if constexpr (TYPE == KQ_TYPE_I8) {
#pragma unroll
                    for (int j = 0; j < 8; j++) vscale[j] = there >> j & 1 ? vscale[j] : 0.0f;
                }
            }
            // the next step's keys are asked for as soon as this one's are used
            const int nb = kb + 32 * NW;
            if (nb < k1) {
                load_k(nb);
                if (nb + 32 * NW < k1) fetch(nb + 32 * NW);
            }
            // weights
            float x[8];
#pragma unroll
            for (int j = 0; j < 8; j++) {
                x[j] = sc[j >> 2][j & 3];
                if constexpr (NP == 2) x[j] *= inv;
                if constexpr (TYPE == KQ_TYPE_I8) x[j] *= kscale[j];
            }
            if (!full) {
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const int key = kb + 16 * (j >> 2) + 4 * g + (j & 3);
                    x[j] = key >= lo && key < hi && (there >> j & 1) ? x[j] : -INFINITY;
                }
            }
            float top = x[0];
#pragma unroll
            for (int j = 1; j < 8; j++) top = fmaxf(top, x[j]);
            top = max4(top);
            // (2^5 above the maximum that the weights are taken from before that is moved; int8: by
            // whole steps, which the exponent takes)
            if (__any(top > m + 5.0f)) {
                const float nm = fmaxf(m, TYPE == KQ_TYPE_I8 ? ceilf(top) : top);
                float f = nm == -INFINITY ? 1.0f : exp2_(m - nm);
                l *= f;
                if constexpr (TYPE == KQ_TYPE_I8) {
                    const int e = ve - (int)fminf(nm - m, 1000.0f);
                    ve = max(e, VE0);
                    f = __uint_as_float((uint32_t)max(0, 127 + e - ve) << 23);
                }
                m = nm;
#pragma unroll
                for (int b = 0; b < NB; b++)
#pragma unroll
                    for (int t = 0; t < W; t++) acc[b][t] *= f;
            }
            // binary16: times 2^9, which leaves with the division by the sum; int8: times 2^-6, so
            // that weights up to 2^5 times their values' scales stay finite
            const float base =
                (m == -INFINITY ? 0.0f : m) - (TYPE == KQ_TYPE_I8 ? -6.0f : NP == 2 ? 9.0f : -less);
            float p[8];
#pragma unroll
            for (int j = 0; j < 8; j += 2) {
                p[j] = exp2_(x[j] - base);
                p[j + 1] = exp2_(x[j + 1] - base);
                l += p[j] + p[j + 1];
            }
            if constexpr (TYPE == KQ_TYPE_I8) {
                // A row's sums are those of weights times scales, in units of a power of two that
                // puts the largest of these so far (of the keys that the row sees) from 2^10 to
                // 2^15.  (A hidden key's scale may be no number.)
                float big = 0.0f;
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    p[j] = full || x[j] != -INFINITY ? p[j] * vscale[j] : 0.0f;
                    big = fmaxf(big, fabsf(p[j]));
                }
                const int e = min(253, (int)(__float_as_uint(max4(big)) >> 23));
                if (__any(e > ve + 4)) {
                    const int top = e > ve + 4 ? e : ve;
                    const float f = __uint_as_float((uint32_t)max(0, 127 + ve - top) << 23);
                    ve = top;
#pragma unroll
                    for (int b = 0; b < NB; b++)
#pragma unroll
                        for (int t = 0; t < W; t++) acc[b][t] *= f;
                }
                const float f = __uint_as_float((uint32_t)(264 - ve) << 23);
#pragma unroll
                for (int j = 0; j < 8; j++) p[j] *= f;
            }
            u32x4 w[NP];
#pragma unroll
            for (int j = 0; j < 8; j += 2) {
                uint32_t o[NP];
                split<NP>(p[j], p[j + 1], o);
#pragma unroll
                for (int e = 0; e < NP; e++) w[e][j >> 1] = o[e];
            }
            __builtin_amdgcn_sched_barrier(0);
            // values
            if (!full) {
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const uint32_t keep = there >> j & 1 ? 0xffffffffu : 0u;
#pragma unroll
                    for (int b = 0; b < NB; b++)
#pragma unroll
                        for (int e = 0; e < VW; e++) vr[j][b][e] &= keep;
                }
            }
            if (ES == 2 && pass) {
                // (an exponent of ones plus one is the sign's bit)
                constexpr uint32_t NONE = TYPE == KQ_TYPE_F16 ? 0x7c00 : 0x7f80, ONE = 0x8000 - NONE;
                uint32_t sum = 0;
#pragma unroll
                for (int j = 0; j < 8; j++)
#pragma unroll
                    for (int b = 0; b < NB; b++)
#pragma unroll
                        for (int e = 0; e < VW; e++) sum |= (vr[j][b][e] & 0x7fff7fffu) + ONE * 0x10001u;
                if (__any((sum & 0x80008000u) != 0)) {
                    odd0 = min(odd0, kb);
                    odd1 = kb + 32;
#pragma unroll
                    for (int j = 0; j < 8; j++)
#pragma unroll
                        for (int b = 0; b < NB; b++)
#pragma unroll
                            for (int e = 0; e < VW; e++) {
                                const uint32_t v = vr[j][b][e];
                                if ((v & 0x7fff) >= NONE) vr[j][b][e] &= 0xffff0000u;
                                if ((v >> 16 & 0x7fff) >= NONE) vr[j][b][e] &= 0xffffu;
                            }
                }
            }
#pragma unroll
            for (int b = 0; b < NB; b++) {
                if (!EXACT && 16 * W * b >= D) continue;
#pragma unroll
                for (int t = 0; t < W; t++) {
                    u32x4 v;
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const u32x4 v0 = vr[2 * j][b], v1 = vr[2 * j + 1][b];
                        if constexpr (ES == 2)
                            v[j] = perm(v1[t >> 1], v0[t >> 1], t & 1 ? 0x07060302 : 0x05040100);
                        else
                            v[j] = halves(perm(v1[t >> 2], v0[t >> 2], 0x0c000c00u | (t & 3) | (4 + (t & 3)) << 16));
                    }
#pragma unroll
                    for (int j = 0; j < NP; j++) acc[b][t] = mfma<NP>(v, w[j], acc[b][t]);
                    // (in few registers: the compiler would make all operands first)
                    if (t % 4 == 3) __builtin_amdgcn_sched_barrier(0);
                }
            }
            if (nb < k1) load_v();
        }

        float none = 0.0f;
        if constexpr (ES == 2) {
#pragma unroll
            for (int b = 0; b < NB; b++)
#pragma unroll
                for (int t = 0; t < W; t++)
#pragma unroll
                    for (int i = 0; i < 4; i++) none = fmaf(acc[b][t][i], 0x1p32f, none);
        }
        const float sum = sum4(l);
        const bool bad = c < live && __builtin_isfinite(sum) && !__builtin_isfinite(none);
        // (a barrier: queries have been read)
        if (!__syncthreads_or(bad) || pass == NP - 1) break;
        if (++pass == 2) less = max4(bad ? 40.0f : 0.0f);
    }
    if (NP == 3 && m != -INFINITY) m += less;               // (what the weights were taken from)

    // ---- the waves' sums
    l = sum4(l);
    if constexpr (TYPE == KQ_TYPE_I8) {
        // (where products pass 2^33, sums of them and of weights times 2^-64: 2^30 values of any
        // scale stay finite, where the result is)
        if (ve > 160) {
            ve -= 64;
            l *= 0x1p-64f;
            m += 64.0f;
        }
    }
    if (g == 0) s_ml[wave][c] = make_float2(m, l);
    if (ES == 2 && pass) {
        if (lane == 0) {
            s_odd[wave][0] = odd0;
            s_odd[wave][1] = odd1;
        }
        if (tid < D) s_inf[tid] = 0;
    }
    __syncthreads();
    float* const ol = reinterpret_cast<float*>(lds);
    const int quads = D / 4;
    {
        float top = s_ml[0][c].x, sum = 0.0f;
#pragma unroll
        for (int i = 1; i < NW; i++) top = fmaxf(top, s_ml[i][c].x);
        const float base = top == -INFINITY ? 0.0f : top;
        if (tid < 16) {
#pragma unroll
            for (int i = 0; i < NW; i++) sum += s_ml[i][c].y * exp2_(s_ml[i][c].x - base);
            s_all[c] = make_float2(top, sum);
        }
        float f = exp2_(m - base);
        if constexpr (TYPE == KQ_TYPE_I8) f *= __uint_as_float((uint32_t)(ve - 10) << 23);
        if (c < live) {
#pragma unroll
            for (int b = 0; b < NB; b++)
#pragma unroll
                for (int i = 0; i < 4; i++)
#pragma unroll
                    for (int t = 0; t < W; t += 4)
                        *reinterpret_cast<f32x4*>(ol + (wave * 16 + c) * OS + 16 * W * b + W * (4 * g + i) + t) =
                            (f32x4){acc[b][t][i], acc[b][t + 1][i], acc[b][t + 2][i], acc[b][t + 3][i]} * f;
        }
    }
    if (ES == 2 && pass) {
        // Which rows see infinities and NaN of a place in a row of values: bit r of s_inf for +inf,
        // 16 + r for -inf, both for NaN.  A lane has eight places of every (2048 / D)th key, eight of them
        // in flight (a lane's keys one by one: one sequence of 32768, heads of 256, with NaN in one
        // key's values took 372 us for 52, 31 ms for 1.6 without a list).
        int from = 0x7fffffff, to = 0;
#pragma unroll
        for (int i = 0; i < NW; i++) {
            from = min(from, s_odd[i][0]);
            to = max(to, s_odd[i][1]);
        }
        to = min(to, k1);
        constexpr int KU = 8;
        constexpr uint32_t NONE = TYPE == KQ_TYPE_F16 ? 0x7c00 : 0x7f80;
        const int pieces = D / 8, by = 64 * NW / pieces, piece = tid % pieces, old = len - n;
        uint32_t inf[8];
#pragma unroll
        for (int e = 0; e < 8; e++) inf[e] = 0;
#pragma unroll 1
        for (int64_t key0 = (int64_t)from + tid / pieces; key0 < to && tid < pieces * by; key0 += KU * by) {
            int page[KU];
            u32x4 v[KU];
#pragma unroll
            for (int u = 0; u < KU; u++) page[u] = table[(uint32_t)min(key0 + u * by, (int64_t)to - 1) / (uint32_t)a.page];
#pragma unroll
            for (int u = 0; u < KU; u++) {
                const uint32_t key = (uint32_t)min(key0 + u * by, (int64_t)to - 1);
                const bool there = (uint32_t)page[u] < (uint32_t)a.n_pages;
                v[u] = *reinterpret_cast<const u32x4*>(vh + (there ? page[u] : 0) * a.page_b +
                                                       (int64_t)((uint64_t)(key % (uint32_t)a.page) * a.tok_b) + 16 * piece);
                if (!there) v[u] = (u32x4)0u;
            }
#pragma unroll
            for (int u = 0; u < KU; u++) {
                uint32_t sum = 0;
#pragma unroll
                for (int e = 0; e < 4; e++) sum |= (v[u][e] & 0x7fff7fffu) + (0x8000 - NONE) * 0x10001u;
                if (!(sum & 0x80008000u)) continue;
                // rows lo..hi - 1 see the key (the last one again, where there are fewer)
                const int rel = (int)min(key0 + u * by, (int64_t)to - 1) - old;
                const int lo = min(max(rel <= 0 ? 0 : rel * G - first, 0), 16);
                const int hi = !a.window || rel + a.window >= n ? 16 : min(max(max(rel + a.window, 0) * G - first, 0), 16);
                const uint32_t rows = (1u << max(hi, lo)) - (1u << lo);
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const uint32_t x = v[u][e >> 1] >> 16 * (e & 1) & 0xffff, y = x & 0x7fff;
                    if (y == NONE) inf[e] |= rows << (x == y ? 0 : 16);
                    if (y > NONE) inf[e] |= rows * 0x10001u;
                }
            }
        }
#pragma unroll
        for (int e = 0; e < 8; e++)
            if (inf[e]) atomicOr(&s_inf[8 * piece + e], inf[e]);
    }
    __syncthreads();
    auto store_out = [&](int r, int d, f32x4 y) {
        const int64_t tok = (int64_t)row0 + (first + r) / G;
        if (tok >= 0 && tok < a.N)
            *reinterpret_cast<f32x4*>(a.out + tok * a.out_stride + (int64_t)(h * G + (first + r) % G) * D + d) = y;
    };
    // (row of the partial results)
    auto put = [](void* p, float lo, float hi) {
        __hip_atomic_store(static_cast<uint64_t*>(p), (uint64_t)__float_as_uint(lo) | (uint64_t)__float_as_uint(hi) << 32,
                           __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    };
    auto store_part = [&](int64_t row, int d, f32x4 y) {
        put(a.part + row * D + d, y[0], y[1]);
        put(a.part + row * D + d + 2, y[2], y[3]);
    };
    const int64_t prow = ((int64_t)(part + idx) * a.n_kv + h) * a.R + first;
    for (int e = tid; e < live * quads; e += 64 * NW) {
        const int r = e / quads, d = e % quads * 4;
        f32x4 y = *reinterpret_cast<const f32x4*>(ol + r * OS + d);
#pragma unroll
        for (int i = 1; i < NW; i++) y += *reinterpret_cast<const f32x4*>(ol + (i * 16 + r) * OS + d);
        if (ES == 2 && pass) {
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const uint32_t x = s_inf[d + i] >> r;
                if (x & 1) y[i] += INFINITY;
                if (x & 0x10000) y[i] -= INFINITY;
            }
        }
        const float2 all = s_all[r];
        if (num == 1) {
            store_out(r, d, all.y == 0.0f ? (f32x4)0.0f : y / all.y);
        } else {
            store_part(prow + r, d, y);
            if (d == 0) put(a.ml + prow + r, all.x, all.y);
        }
    }
    if (num == 1) return;

    // ---- Partial results are joined by the last workgroup, or, where that would be long, by
    // the last of each eight and theirs by the last of these.  Results and counts are
    // device-scope atomics, which go past the caches that another XCD does not see: once
    // a wave's stores are acknowledged they are there for all, and the barrier puts every
    // wave's before the count.  (A release fence instead writes back the L2, in each of
    // hundreds of workgroups: 64 ragged streams took 233 us with it, 124 without.)
    auto last_of = [&](int slot, int of) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        if (tid == 0) {
            int* const p = a.counter + ((int64_t)(part + slot) * a.n_kv + h) * a.blocks + z;
            s_last = __hip_atomic_fetch_add(p, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == of - 1;
            if (s_last) __hip_atomic_store(p, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
        __syncthreads();
        return s_last != 0;
    };
    auto get = [](const void* p) {
        const uint64_t x = __hip_atomic_load(static_cast<const uint64_t*>(p), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        return make_float2(__uint_as_float((uint32_t)x), __uint_as_float((uint32_t)(x >> 32)));
    };
    // JU quads of JN results that a lane has in flight.  By eights where there are more than
    // FLAT quads (of 6 rows of 256, 16 parts: all at once 18 us a call, by eights 24; 64
    // parts: 46 and 40).
    constexpr int JU = 2, JN = 8, FLAT = 12288;
    // n results, `by` apart from slot `from` on, to the first's place or, `end`, to out
    auto join = [&](int from, int by, int of, bool end) {
        const int64_t row1 = ((int64_t)(part + from) * a.n_kv + h) * a.R + first, step = (int64_t)by * a.n_kv * a.R;
        for (int e0 = tid; e0 < live * quads; e0 += 64 * NW * JU) {
            f32x4 y[JU];
            float top[JU], sum[JU];
#pragma unroll
            for (int u = 0; u < JU; u++) {
                y[u] = (f32x4)0.0f;
                top[u] = -INFINITY;
                sum[u] = 0.0f;
            }
#pragma unroll 1
            for (int i0 = 0; i0 < of; i0 += JN) {
                float2 t[JU][JN], o[JU][JN][2];
#pragma unroll
                for (int u = 0; u < JU; u++) {
                    const int e = min(e0 + 64 * NW * u, live * quads - 1), r = e / quads, d = e % quads * 4;
#pragma unroll
                    for (int i = 0; i < JN; i++) {
                        const int64_t at = row1 + r + min(i0 + i, of - 1) * step;
                        t[u][i] = get(a.ml + at);
                        o[u][i][0] = get(a.part + at * D + d);
                        o[u][i][1] = get(a.part + at * D + d + 2);
                    }
                }
#pragma unroll
                for (int u = 0; u < JU; u++) {
                    float nm = top[u];
#pragma unroll
                    for (int i = 0; i < JN; i++) nm = fmaxf(nm, t[u][i].x);
                    const float base = nm == -INFINITY ? 0.0f : nm, f = exp2_(top[u] - base);
                    top[u] = nm;
                    y[u] *= f;
                    sum[u] *= f;
#pragma unroll
                    for (int i = 0; i < JN; i++) {
                        const float w = exp2_(t[u][i].x - base);
                        if (i0 + i < of) {
                            y[u] += (f32x4){o[u][i][0].x, o[u][i][0].y, o[u][i][1].x, o[u][i][1].y} * w;
                            sum[u] += t[u][i].y * w;
                        }
                    }
                }
            }
#pragma unroll
            for (int u = 0; u < JU; u++) {
                const int e = e0 + 64 * NW * u, r = e / quads, d = e % quads * 4;
                if (e >= live * quads) continue;
                if (end) {
                    store_out(r, d, sum[u] == 0.0f ? (f32x4)0.0f : y[u] / sum[u]);
                } else {
                    store_part(row1 + r, d, y[u]);
                    if (d == 0) s_all[r] = make_float2(top[u], sum[u]);
                }
            }
        }
        if (end) return;
        __syncthreads();                    // (all lanes have read the maximum and sum of their row)
        if (tid < live) put(a.ml + row1 + tid, s_all[tid].x, s_all[tid].y);
    };
    const bool flat = num <= 8 || live * quads * num <= FLAT;
    const int group = flat ? 0 : idx & ~7, of = flat ? num : min(8, num - group);
    if (!last_of(group, of)) return;
    join(group, 1, of, flat);
    if (!flat && last_of(1, (num + 7) / 8)) join(0, 8, (num + 7) / 8, true);
}

typedef void (*Kernel)(AttnArg);

template <int TYPE>
Kernel pick(int D, bool tiled) {
    if (!tiled) return D <= 128 ? kq_attn_kernel<TYPE, 128, false, false> : kq_attn_kernel<TYPE, 256, false, false>;
    if (D == 64) return kq_attn_kernel<TYPE, 64, true, true>;
    if (D == 128) return kq_attn_kernel<TYPE, 128, true, true>;
    if (D == 256) return kq_attn_kernel<TYPE, 256, true, true>;
    return D < 128 ? kq_attn_kernel<TYPE, 128, false, true> : kq_attn_kernel<TYPE, 256, false, true>;
}

int64_t up256(int64_t n) { return (n + 255) & ~(int64_t)255; }

}  // namespace

extern "C" {

void kqk_attn_plan(const kq_attn_shape* s, int n_cu, kqk_attn_sizes* z) {
    z->blocks = (s->T * (s->n_q / s->n_kv) + 15) / 16;
    const int per = s->n_kv * z->blocks;
    // Two workgroups on each CU, in one round, where sequences are few (8 of 8192 keys, 16 / 8
    // heads of 128, 320 / 448 / 512 / 576 workgroups: 65 / 56 / 55 / 63 us), one with heads
    // past 128 values, of which the join of more is longer (heads of 256, 256 / 512
    // workgroups: one of 32768 39 / 43.6, 8 of 8192 59 / 65, 8 of 500 to 20000 51 / 56; int8
    // heads of 128 are the other way, 46 / 34); beyond, one on each more than there are
    // sequences (64 ragged ones, 400 / 500 / 756: 114 / 100 / 103).  128 keys an item where
    // that is a workgroup on every fourth CU at most, 256 otherwise (one sequence, heads of
    // 256, of 1024: 13.2 / 17.1, of 4096: 20.0 / 18.3).
    const int one = (n_cu + per - 1) / per;       // items for a workgroup on each CU
    z->few = 32 * n_cu / per;
    const int few = s->D > 128 && 8 * s->S <= one ? one : 2 * one;
    const int extra = few - s->S > one || few == one ? few - s->S : one;
    z->cap = s->S + extra;
    z->parts = 2 * extra;                         // (a split sequence has two items or more)
    z->counters = (int64_t)z->parts * per;
}

int64_t kqk_attn_workspace(const kq_attn_shape* s, int n_cu) {
    kqk_attn_sizes z;
    kqk_attn_plan(s, n_cu, &z);
    const int64_t rows = (int64_t)z.parts * s->n_kv * s->T * (s->n_q / s->n_kv);
    return up256(rows * s->D * 4) + up256(rows * 8);
}

int kqk_launch_attn(const kq_paged_attn* p, const kqk_attn_sizes* z, void* work, hipStream_t st) {
    const kq_kv_cache& c = p->cache;
    const kq_attn_shape& s = p->shape;
    const int es = c.type == KQ_TYPE_I8 ? 1 : 2;
    AttnArg a = {};
    a.k = (const uint8_t*)c.k;
    a.v = (const uint8_t*)c.v;
    a.ks = c.k_scale;
    a.vs = c.v_scale;
    a.q = p->q;
    a.out = p->out;
    a.table = p->table;
    a.start = p->start;
    a.lens = p->lens;
    a.page_b = c.page_stride * es;
    a.head_b = c.head_stride * es;
    a.tok_b = (uint32_t)c.token_stride * es;
    a.page_s = (uint32_t)c.n_kv * c.page;
    a.q_stride = p->q_stride;
    a.out_stride = p->out_stride;
    a.qscale = (float)(p->scale * 1.4426950408889634);
    a.S = s.S;
    a.T = s.T;
    a.G = s.n_q / s.n_kv;
    a.R = s.T * a.G;
    a.n_kv = s.n_kv;
    a.D = s.D;
    a.window = s.window;
    a.N = p->N;
    a.page = c.page;
    a.n_pages = c.n_pages;
    a.table_stride = p->table_stride;
    a.cap = z->cap;
    a.parts = z->parts;
    const bool tiled = c.page % 16 == 0;
    if (tiled) {
        // div d = 2^shift + e with e < d = page / 16 and 2^27 d <= 2^shift < 2^28 d: tiles below
        // 2^27 (keys below 2^31) are divided exactly, their products below 2^56
        const uint64_t d = c.page / 16;
        a.div_shift = 27;
        while ((uint64_t)1 << (a.div_shift - 27) < d) a.div_shift++;
        a.div = (((uint64_t)1 << a.div_shift) + d - 1) / d;
    }
    if (p->list) {
        a.count = (const int*)p->list;
        a.items = a.count + KQK_LIST_HEAD;
        a.counter = (int*)p->list + KQK_LIST_HEAD + (int64_t)z->cap * KQK_ITEM;
        const int64_t rows = (int64_t)z->parts * s.n_kv * a.R;
        a.part = (float*)work;
        a.ml = (float2*)((uint8_t*)work + up256(rows * s.D * 4));
    }
    const Kernel k = c.type == KQ_TYPE_F16    ? pick<KQ_TYPE_F16>(s.D, tiled)
                     : c.type == KQ_TYPE_BF16 ? pick<KQ_TYPE_BF16>(s.D, tiled)
                                              : pick<KQ_TYPE_I8>(s.D, tiled);
    // A number x divided by d as x ceil(2^40 / d) 2^-40 is exact where x d < 2^40: here d = n_kv is at most
    // 2^10, or 8 blocks at most 2^15 (64 tokens of 1024 heads are 2^12 blocks), and x below 2^23.
    a.blocks = z->blocks;
    a.kv_div = (((uint64_t)1 << 40) + s.n_kv - 1) / s.n_kv;
    a.blocks_div = (((uint64_t)1 << 40) + 8 * z->blocks - 1) / (8 * z->blocks);
    const int64_t pairs = (int64_t)(p->list ? z->cap : s.S) * s.n_kv;
    const dim3 grid((unsigned)((pairs + 7) / 8 * 8 * z->blocks));
    hipLaunchKernelGGL(k, grid, dim3(64 * NW), 0, st, a);
    return (int)hipGetLastError();
}

}
