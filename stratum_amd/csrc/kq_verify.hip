// kq_verify.hip -- drafted tokens against the target's distributions, from
// given random numbers (gfx950).
//
// Row i of a sequence holds the target's distribution p_i at drafted token
// t_i; q_i is the draft's.  Token i is accepted iff u_i q_i(t_i) < p_i(t_i)
// and all before it were.  The token that follows the n accepted ones is drawn
// from max(p_n - q_n, 0), or from p_n when nothing was refused: the first v
// whose running sum of weights is above u times their total.
//
// All of it is binary64: a running sum over 150 K tokens has as many borders,
// and a token changes where one of them moves past u.  Of logits the weights are
// good to 6e-12 (pow2() below), which moves borders by a ten-thousandth of a
// binary32 u's step (2^-24).
//
// Launches: the rows' maxima and sums of exponentials per chunk of CH tokens
// (logits and greedy form); then the weights' sums per chunk of the row drawn
// from, and, by the workgroup that ends a sequence's last, the token.  (The
// count of ended ones is cleared by the first launch; probabilities, which need
// no first launch, draw in a launch of their own instead.)  Binary64 instructions
// bound the first (240 rows of 151936 31 us, 4.7 TB/s), a chain of waits the second
// (one sequence 9.2 us, sixteen 20).
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "kq_launch.h"

#pragma clang fp contract(off)

namespace {

constexpr int TH = 256, NJ = 4, CH = 4 * NJ * TH;    // lanes; steps of 4 tokens a lane; tokens of a chunk
constexpr int SUB = 256, NSUB = CH / SUB;            // a chunk's parts: a wave's step
constexpr double LOG2E = 1.4426950408889634;

struct VfArg {
    kq_spec_verify v;
    int nch, cpw;           // chunks of a row; of a workgroup of the second launch
    float* pmax;            // [rows][nch]
    double* psum;           // [rows][nch]
    int* parg;              // [rows][nch]
    int nsum;               // nch + nch * NSUB
    double* wsum;           // [S][nsum]: weights' sums per chunk, then per part of 256 tokens
    int* ended;             // [S]: workgroups of the second launch that are done
    double c, far;          // inv_temp / ln 2; 2^(d c) is taken for nothing from d = far = -1000 / c down
};

// 2^(d c) for d <= 0, nothing for NaN and below 2^-1000: d c = k + r, |r| <= 1/2,
// and the polynomial of degree 8 that meets 2^r at the nine Chebyshev points of
// that interval, within 1.1e-12 of it.  d is the difference of two logits, so it
// is 0 at the maximum whatever that is (a row of the type's lowest value is a
// uniform one).  k comes as the low bits of d c + 1.5 * 2^52 and goes into the
// exponent as an integer.  A weight has five of them on its way: its own, and four
// in its row's sum, to the maximum of a wave, a chunk, a lane's chunks and the row (one
// more per 64 chunks after the first).  These 18 binary64 instructions a value bound the first
// launch (sixteen sequences of seven, 240 rows of 151936, both launches: 57 us,
// with the library's exp2() 76; one of four, 15 and 18).
__device__ __forceinline__ double pow2(double d, double c, double far) {
    constexpr double C[9] = {
        0x1.0000000000000p+0, 0x1.62e42fef84ceap-1, 0x1.ebfbdff823dddp-3,
        0x1.c6b08dd6fdf85p-5, 0x1.3b2ab71805844p-7, 0x1.5d8745a62da0ep-10,
        0x1.4308acadc0000p-13, 0x1.00dc4af70e38ep-16, 0x1.63d109578e38ep-20};
    constexpr double MAGIC = 0x1.8p52;
    const double t = fma(d, c, MAGIC), r = fma(d, c, -(t - MAGIC));
    double p = C[8];
#pragma unroll
    for (int i = 7; i >= 0; i--) p = fma(p, r, C[i]);
    const int hi = __double2hiint(p) + (__double2loint(t) << 20);
    return d > far ? __hiloint2double(hi, __double2loint(p)) : 0.0;
}

// 4 values at any 4-byte alignment
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

// rows of the chunk tables: target rows first, then the draft's
__device__ __forceinline__ int trow(const VfArg& a, int s, int i) { return s * (a.v.T + 1) + i; }
__device__ __forceinline__ int drow(const VfArg& a, int s, int i) {
    return a.v.S * (a.v.T + 1) + s * a.v.T + i;
}
__device__ __forceinline__ int drafted(const VfArg& a, int s) {
    return a.v.n_draft ? min(max(a.v.n_draft[s], 0), a.v.T) : a.v.T;
}
__device__ __forceinline__ const float* target_row(const VfArg& a, int s, int i) {
    return a.v.target + s * a.v.target_seq + i * a.v.target_row;
}
__device__ __forceinline__ const float* draft_row(const VfArg& a, int s, int i) {
    return a.v.draft + s * a.v.draft_seq + i * a.v.draft_row;
}

// 4 tokens from k on, `fill` behind the end
__device__ __forceinline__ f32x4 load4(const float* row, int k, int V, float fill) {
    f32x4 x;
    if (k + 4 <= V) {
        x = *reinterpret_cast<const f32x4u*>(row + k);
    } else {
#pragma unroll
        for (int e = 0; e < 4; e++) x[e] = k + e < V ? row[k + e] : fill;
    }
    return x;
}

// a lane's NJ times 4 tokens of a chunk: base + 4 (TH j + tid) .. + 3
struct Chunk {
    f32x4 v[NJ];
    __device__ __forceinline__ void load(const float* row, int base, int V, float fill) {
#pragma unroll
        for (int j = 0; j < NJ; j++) v[j] = load4(row, base + 4 * (TH * j + (int)threadIdx.x), V, fill);
    }
    // the first four; the others move up: for loops over j that stay loops (the
    // code of long unrolled ones is read from memory in every launch)
    __device__ __forceinline__ f32x4 next() {
        const f32x4 f = v[0];
#pragma unroll
        for (int j = 0; j < NJ - 1; j++) v[j] = v[j + 1];
        return f;
    }
};

template <int CTRL>
__device__ __forceinline__ double dpp(double v) {
    const int lo = __builtin_amdgcn_mov_dpp(__double2loint(v), CTRL, 0xf, 0xf, false);
    const int hi = __builtin_amdgcn_mov_dpp(__double2hiint(v), CTRL, 0xf, 0xf, false);
    return __hiloint2double(hi, lo);
}
// sums over 16 lanes and over a wave, in every lane
__device__ __forceinline__ double sum16(double v) {
    v = v + dpp<0xB1>(v);                   // quad_perm [1, 0, 3, 2]
    v = v + dpp<0x4E>(v);                   // quad_perm [2, 3, 0, 1]
    v = v + dpp<0x141>(v);                  // row_half_mirror
    return v + dpp<0x140>(v);               // row_mirror
}
__device__ __forceinline__ double wave_sum(double v) {
    v = sum16(v);
    const uint32_t l = (uint32_t)__double2loint(v), h = (uint32_t)__double2hiint(v);
    const auto l1 = __builtin_amdgcn_permlane16_swap(l, l, false, false);    // rows 0, 0, 2, 2 and 1, 1, 3, 3
    const auto h1 = __builtin_amdgcn_permlane16_swap(h, h, false, false);
    v = __hiloint2double((int)h1[0], (int)l1[0]) + __hiloint2double((int)h1[1], (int)l1[1]);
    const uint32_t m = (uint32_t)__double2loint(v), g = (uint32_t)__double2hiint(v);
    const auto l2 = __builtin_amdgcn_permlane32_swap(m, m, false, false);
    const auto h2 = __builtin_amdgcn_permlane32_swap(g, g, false, false);
    return __hiloint2double((int)h2[0], (int)l2[0]) + __hiloint2double((int)h2[1], (int)l2[1]);
}
// what `v` of another lane is, 0 where there is none or the row is not in `ROWS`
template <int CTRL, int ROWS>
__device__ __forceinline__ double from(double v) {
    return __hiloint2double(__builtin_amdgcn_update_dpp(0, __double2hiint(v), CTRL, ROWS, 0xf, false),
                            __builtin_amdgcn_update_dpp(0, __double2loint(v), CTRL, ROWS, 0xf, false));
}
template <int CTRL>
__device__ __forceinline__ float dpp_max(float v) {
    return fmaxf(v, __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), CTRL, 0xf, 0xf, false)));
}
__device__ __forceinline__ float max16(float v) {
    return dpp_max<0x140>(dpp_max<0x141>(dpp_max<0x4E>(dpp_max<0xB1>(v))));
}

// A chunk's maximum, its first place, and the sum of exp((l - max) inv_temp).
template <bool GREEDY>
__global__ __launch_bounds__(TH) void kq_vf_stats_kernel(VfArg a) {
    __shared__ float sm[TH / 64];
    __shared__ int si[TH / 64];
    __shared__ double sd[TH / 64];
    const int T = a.v.T, row = blockIdx.y, nt = a.v.S * (T + 1), tid = threadIdx.x;
    if (!GREEDY && blockIdx.x == 0 && row < a.v.S && tid == 0) a.ended[row] = 0;
    const bool isd = row >= nt;
    const int s = isd ? (row - nt) / T : row / (T + 1), i = isd ? (row - nt) % T : row % (T + 1);
    if (isd ? i >= drafted(a, s) : i > drafted(a, s)) return;
    const int base = blockIdx.x * CH;
    Chunk v;
    v.load(isd ? draft_row(a, s, i) : target_row(a, s, i), base, a.v.V, -INFINITY);
    float m = -INFINITY;
#pragma unroll
    for (int j = 0; j < NJ; j++)                                // (a NaN is never the maximum)
        m = fmaxf(m, fmaxf(fmaxf(v.v[j][0], v.v[j][1]), fmaxf(v.v[j][2], v.v[j][3])));
    const float mine = m;
    m = max16(m);
    m = fmaxf(m, __shfl_xor(m, 16));
    m = fmaxf(m, __shfl_xor(m, 32));
    const long o = (long)row * a.nch + blockIdx.x;
    if (GREEDY) {
        int at = 0x7fffffff;
        if (mine == m && m > -INFINITY) {
#pragma unroll
            for (int k = 4 * NJ - 1; k >= 0; k--)
                if (v.v[k / 4][k % 4] == m) at = base + 4 * (TH * (k / 4) + tid) + k % 4;
        }
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) at = min(at, __shfl_xor(at, off));
        if ((tid & 63) == 0) { sm[tid >> 6] = m; si[tid >> 6] = at; }
        __syncthreads();
        m = sm[0]; at = si[0];
        for (int k = 1; k < TH / 64; k++)
            if (sm[k] > m || (sm[k] == m && si[k] < at)) { m = sm[k]; at = si[k]; }
        if (tid == 0) { a.pmax[o] = m; a.parg[o] = at; }
        return;
    }
    const double top = m;
    double z = 0.0;
#pragma unroll
    for (int j = 0; j < NJ; j++)
#pragma unroll
        for (int e = 0; e < 4; e++) z = z + pow2((double)v.v[j][e] - top, a.c, a.far);
    z = wave_sum(z);
    if ((tid & 63) == 0) { sm[tid >> 6] = m; sd[tid >> 6] = z; }
    __syncthreads();
    if (tid < 4) {                          // the waves' sums on one maximum
        const float mm = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3]));
        z = pow2((double)sm[tid] - (double)mm, a.c, a.far) * sd[tid];
        z = z + dpp<0xB1>(z);
        z = z + dpp<0x4E>(z);
        if (tid == 0) {
            a.pmax[o] = mm;
            a.psum[o] = z;
        }
    }
}

// 16 lanes: a row's maximum and sum from its chunks
__device__ __forceinline__ void row_stats(const VfArg& a, int row, float* m, double* z) {
    const int lane = threadIdx.x & 15;
    const long o = (long)row * a.nch;
    float mm = -INFINITY;
    double t = 0.0;
#pragma unroll 1
    for (int k0 = lane; k0 < a.nch; k0 += 64) {
        float pm[4], was = mm;
        double ps[4];
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const bool in = k0 + 16 * k < a.nch;
            pm[k] = in ? a.pmax[o + k0 + 16 * k] : -INFINITY;
            ps[k] = in ? a.psum[o + k0 + 16 * k] : 0.0;
        }
        mm = fmaxf(fmaxf(fmaxf(mm, pm[0]), pm[1]), fmaxf(pm[2], pm[3]));
        t = t * pow2((double)was - (double)mm, a.c, a.far);
#pragma unroll
        for (int k = 0; k < 4; k++) t = fma(pow2((double)pm[k] - (double)mm, a.c, a.far), ps[k], t);
    }
    const float top = max16(mm);
    *z = sum16(t * pow2((double)mm - (double)top, a.c, a.far));
    *m = top;
}

// The weight of a token at the row drawn from.
struct Drawn {
    const float* p;
    const float* q;         // NULL: one-hot, or nothing refused
    int hot;                // one-hot draft's token, or -1
    bool logits;
    double pm, qm;
    double pz, qz, c, far;  // 1 / sums
    __device__ __forceinline__ double at(int k, float pk, float qk) const {
        double pv = pk, qv = qk;
        if (logits) {
            pv = pow2(pv - pm, c, far) * pz;
            if (q) qv = pow2(qv - qm, c, far) * qz;
        }
        pv = fmax(pv, 0.0);                 // (NaN: nothing)
        return k == hot ? 0.0 : q ? fmax(pv - fmax(qv, 0.0), 0.0) : pv;
    }
};

// Every thread of the workgroup: tokens accepted, and what is drawn from.
__device__ __forceinline__ Drawn decide(const VfArg& a, int s, int* nacc) {
    __shared__ float mx[2 * KQ_VERIFY_MAX_DRAFT + 2];
    __shared__ double zs[2 * KQ_VERIFY_MAX_DRAFT + 2];
    __shared__ int sn;
    const int T = a.v.T, nd = drafted(a, s), tid = threadIdx.x;
    const bool lg = a.v.flags & KQ_VERIFY_LOGITS, dr = a.v.draft != nullptr;
    // the drafted tokens' own values, asked for before the sums are known
    int tok = -1;
    float pt = 0.0f, qt = 0.0f, ut = 0.0f;
    if (tid < nd) {
        tok = a.v.tokens[s * T + tid];
        ut = a.v.u[s * (T + 1) + tid];
        if (tok >= 0 && tok < a.v.V) {
            pt = target_row(a, s, tid)[tok];
            if (dr) qt = draft_row(a, s, tid)[tok];
        }
    }
    if (lg) {
        for (int j = tid >> 4; j < 2 * T + 1; j += (int)blockDim.x / 16) {
            const bool isd = j > T;
            const int i = isd ? j - T - 1 : j;
            if (isd ? !dr || i >= nd : i > nd) continue;
            float m;
            double z;
            row_stats(a, isd ? drow(a, s, i) : trow(a, s, i), &m, &z);
            mx[j] = m;
            zs[j] = 1.0 / z;
        }
        __syncthreads();
    }
    if (tid < 64) {
        bool no = tid >= nd || tok < 0 || tok >= a.v.V;
        if (!no) {
            double p = pt, q = dr ? qt : 1.0;
            if (lg) {
                p = pow2(p - (double)mx[tid], a.c, a.far) * zs[tid];
                if (dr) q = pow2(q - (double)mx[T + 1 + tid], a.c, a.far) * zs[T + 1 + tid];
            }
            no = !((double)ut * q < p);
        }
        const unsigned long long b = __ballot(no);
        if (tid == 0) sn = b ? __ffsll(b) - 1 : 64;
    }
    __syncthreads();
    const int n = min(sn, nd);
    Drawn d;
    d.p = target_row(a, s, n);
    d.q = n < nd && dr ? draft_row(a, s, n) : nullptr;
    d.hot = n < nd && !dr ? a.v.tokens[s * T + n] : -1;
    d.logits = lg;
    d.c = a.c;
    d.far = a.far;
    d.pm = lg ? mx[n] : 0.0f;
    d.pz = lg ? zs[n] : 0.0;
    d.qm = lg && d.q ? mx[T + 1 + n] : 0.0f;
    d.qz = lg && d.q ? zs[T + 1 + n] : 0.0;
    *nacc = n;
    return d;
}

__device__ __forceinline__ void draw(const VfArg& a, int s, int n, Drawn d);

// DRAW: the sequence's last workgroup draws
template <bool DRAW>
__global__ __launch_bounds__(TH) void kq_vf_weights_kernel(VfArg a) {
    __shared__ double sd[TH / 64], ps[NSUB];
    __shared__ int last;
    const int s = blockIdx.y, tid = threadIdx.x;
    int n;
    const Drawn d = decide(a, s, &n);
    const float none = d.logits ? -INFINITY : 0.0f;
    double* const sums = a.wsum + (long)s * a.nsum;
    const int end = min(a.nch, ((int)blockIdx.x + 1) * a.cpw);
    Chunk p, q, pn, qn;
    pn.load(d.p, blockIdx.x * a.cpw * CH, a.v.V, none);
    if (d.q) qn.load(d.q, blockIdx.x * a.cpw * CH, a.v.V, none);
#pragma unroll 1
    for (int ch = blockIdx.x * a.cpw; ch < end; ch++) {
        const int base = ch * CH;
        p = pn;
        q = qn;
        if (ch + 1 < end) {                 // the next, while this one is used
            pn.load(d.p, base + CH, a.v.V, none);
            if (d.q) qn.load(d.q, base + CH, a.v.V, none);
        }
        double w = 0.0;
#pragma unroll 1
        for (int j = 0; j < NJ; j++) {
            const f32x4 pv = p.next(), qv = d.q ? q.next() : pv;
            double wj = 0.0;
#pragma unroll
            for (int e = 0; e < 4; e++) wj = wj + d.at(base + 4 * (TH * j + tid) + e, pv[e], qv[e]);
            wj = wave_sum(wj);
            if ((tid & 63) == 0) ps[4 * j + (tid >> 6)] = wj;
            w = w + wj;
        }
        if ((tid & 63) == 0) sd[tid >> 6] = w;
        __syncthreads();
        // Stores past this XCD's L2, where the last workgroup does not look; all by the
        // wave that counts, as its release waits for no other wave's.
        static_assert(NSUB < 64);
        if (tid <= NSUB)
            __hip_atomic_store(tid < NSUB ? sums + a.nch + (long)ch * NSUB + tid : sums + ch,
                               tid < NSUB ? ps[tid] : (sd[0] + sd[1]) + (sd[2] + sd[3]), __ATOMIC_RELAXED,
                               __HIP_MEMORY_SCOPE_AGENT);
        if (ch + 1 < end) __syncthreads();
    }
    __builtin_amdgcn_wave_barrier();
    if (DRAW && tid == 0)
        last = __hip_atomic_fetch_add(a.ended + s, 1, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT) == (int)gridDim.x - 1;
    if (!DRAW) return;
    __syncthreads();
    if (last && tid < 64) draw(a, s, n, d);
}

// inclusive running sum over a wave's lanes
__device__ __forceinline__ double wave_scan(double v) {
    v = v + from<0x111, 0xf>(v);            // row_shr 1, 2, 4, 8
    v = v + from<0x112, 0xf>(v);
    v = v + from<0x114, 0xf>(v);
    v = v + from<0x118, 0xf>(v);
    v = v + from<0x142, 0xa>(v);            // row_bcast 15: a row's end to the next, to rows 1 and 3
    return v + from<0x143, 0xc>(v);         // row_bcast 31: to rows 2 and 3
}

// One step of looking for what a running sum passes `target` in: 64 values, one a
// lane, after `sum`.  The lane of the first at which it is above the target, else
// of the last that is not nothing (and `found` stays false); -1 if all are.
// `base`: the sum before that one.
__device__ __forceinline__ int passed(double v, double target, double& sum, double& base, bool& found) {
    const int lane = threadIdx.x & 63;
    const double in = sum + wave_scan(v);
    const double prev = from<0x138, 0xf>(in);                  // wave_shr 1, by every lane
    const double ex = lane ? prev : sum;
    const unsigned long long over = __ballot(v > 0.0 && in > target), some = __ballot(v > 0.0);
    sum = __shfl(in, 63);
    found = over != 0;
    if (!some) return -1;
    const int j = over ? __ffsll(over) - 1 : 63 - __clzll(some);
    base = __shfl(ex, j);
    return j;
}

// One wave: the chunk, its part and the token in which the running sum passes u
// times the total.
__device__ __forceinline__ void draw(const VfArg& a, int s, int n, Drawn d) {
    const int T = a.v.T, lane = threadIdx.x & 63;
    const double* const ws = a.wsum + (long)s * a.nsum;
    auto sum = [&](int k, int end) {
        return k < end ? __hip_atomic_load(ws + k, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : 0.0;
    };
    const float u = a.v.u[s * (T + 1) + T], none = d.logits ? -INFINITY : 0.0f;
    // the first 64 chunks' sums stay in registers (most vocabularies have fewer)
    const double v0 = sum(lane, a.nch);
    double total = wave_sum(v0);
#pragma unroll 1
    for (int c0 = 64; c0 < a.nch; c0 += 64) total = total + wave_sum(sum(c0 + lane, a.nch));
    double target = (double)u * total, run = 0.0, base = 0.0;
    bool found = false;
    int token = -1, k0 = 0, end = 0;         // 256 tokens at a time, [k0, end)
    if (total > 0.0) {
        int chunk = passed(v0, target, run, base, found);
#pragma unroll 1
        for (int c0 = 64; c0 < a.nch && !found; c0 += 64) {
            const int j = passed(sum(c0 + lane, a.nch), target, run, base, found);
            if (j >= 0) chunk = c0 + j;
        }
        run = base;
        const int first = a.nch + chunk * NSUB;
        const int part = max(0, passed(lane < NSUB ? sum(first + lane, a.nsum) : 0.0, target, run, base, found));
        k0 = chunk * CH + part * SUB;
        end = k0 + 1;
    } else if (d.q || d.hot >= 0) {
        // Nothing is left of p - q: a token refused though p and q are equal (u =
        // 1, or values that are no distributions).  From p itself then, by this
        // wave alone: its sum, and the token.
        d.q = nullptr;
        d.hot = -1;
        end = a.v.V;
#pragma unroll 1
        for (int k = 4 * lane; k - 4 * lane < end; k += 256) {
            const f32x4 pv = load4(d.p, k, a.v.V, none);
            total = total + wave_sum((d.at(k, pv[0], 0.0f) + d.at(k + 1, pv[1], 0.0f)) +
                                     (d.at(k + 2, pv[2], 0.0f) + d.at(k + 3, pv[3], 0.0f)));
        }
        target = (double)u * total;
    }
    run = base;
    found = false;
#pragma unroll 1
    for (; k0 < end && !found; k0 += 256) {
        const int k = k0 + 4 * lane;         // 4 tokens a lane
        const f32x4 pv = load4(d.p, k, a.v.V, none), qv = d.q ? load4(d.q, k, a.v.V, none) : pv;
        double w4[4], w = 0.0;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            w4[e] = d.at(k + e, pv[e], qv[e]);
            w = w + w4[e];
        }
        const int who = passed(w, target, run, base, found);
        // that lane's token: until the sum is past the target, its first with any weight
        // where the sum before it is already (a negative u; or a last bit, as lanes'
        // running sums are added up in orders of their own)
        int at = -1;
        double cum = base;
#pragma unroll
        for (int e = 0; e < 4; e++)
            if (w4[e] > 0.0 && (at < 0 || !(cum > target))) {
                cum = cum + w4[e];
                at = k + e;
            }
        if (who >= 0) token = __shfl(at, who);
    }
    int* const out = a.v.out + (long)s * (T + 1);
    if (lane < n) out[lane] = a.v.tokens[s * T + lane];
    if (lane >= n && lane <= T) out[lane] = lane == n ? token : -1;
    if (lane == 0) a.v.n_accept[s] = n;
}

__global__ __launch_bounds__(64) void kq_vf_draw_kernel(VfArg a) {
    int n;
    const Drawn d = decide(a, blockIdx.x, &n);
    draw(a, blockIdx.x, n, d);
}

// The greedy form: a token is accepted iff it is its row's first maximum.  All
// rows at once, 16 lanes each (row after row until the first refusal, one sequence
// of 4 drafts, all accepted, took 10.8 us against 6.1, of 63 63.8 against 14.1).
__global__ __launch_bounds__(TH) void kq_vf_greedy_kernel(VfArg a) {
    __shared__ int best[KQ_VERIFY_MAX_DRAFT + 1];
    const int s = blockIdx.x, T = a.v.T, tid = threadIdx.x, nd = drafted(a, s);
    const int tok = tid < nd ? a.v.tokens[s * T + tid] : -1;
    for (int i = tid >> 4; i <= nd; i += TH / 16) {
        const long o = (long)trow(a, s, i) * a.nch;
        float m = -INFINITY;
        int at = 0x7fffffff;
#pragma unroll 1
        for (int c = tid & 15; c < a.nch; c += 64) {
            float pm[4];
            int pa[4];
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const bool in = c + 16 * k < a.nch;
                pm[k] = in ? a.pmax[o + c + 16 * k] : -INFINITY;
                pa[k] = in ? a.parg[o + c + 16 * k] : 0;
            }
#pragma unroll
            for (int k = 0; k < 4; k++)
                if (pm[k] > m) { m = pm[k]; at = pa[k]; }
        }
#pragma unroll
        for (int off = 1; off < 16; off <<= 1) {
            const float om = __shfl_xor(m, off);
            const int oa = __shfl_xor(at, off);
            if (om > m || (om == m && oa < at)) { m = om; at = oa; }
        }
        if ((tid & 15) == 0) best[i] = at == 0x7fffffff ? -1 : at;
    }
    __syncthreads();
    if (tid >= 64) return;
    const unsigned long long no = __ballot(tid >= nd || best[tid] < 0 || tok != best[tid]);
    const int n = __ffsll(no) - 1;                     // (nd <= 63: that lane refuses)
    int* const out = a.v.out + (long)s * (T + 1);
    if (tid < n) out[tid] = tok;
    if (tid >= n && tid <= T) out[tid] = tid == n ? best[n] : -1;
    if (tid == 0) a.v.n_accept[s] = n;
}

int64_t up256(int64_t n) { return (n + 255) & ~(int64_t)255; }

int64_t layout(const kq_spec_verify* v, VfArg* a, uint8_t* w) {
    const int64_t nch = ((int64_t)v->V + CH - 1) / CH;
    const bool stats = v->flags & (KQ_VERIFY_LOGITS | KQ_VERIFY_GREEDY);
    const int64_t rows = stats ? (int64_t)v->S * (v->T + 1) + (v->draft ? (int64_t)v->S * v->T : 0) : 0;
    int64_t o[6] = {0};
    o[1] = o[0] + up256(rows * nch * 8);              // psum
    o[2] = o[1] + up256(rows * nch * 4);              // pmax
    o[3] = o[2] + up256(rows * nch * 4);              // parg
    o[4] = o[3] + up256((int64_t)v->S * nch * (1 + NSUB) * 8);   // wsum
    if (a) {
        a->v = *v;
        a->nch = (int)nch;
        a->nsum = (int)nch * (1 + NSUB);
        a->psum = (double*)(w + o[0]);
        a->pmax = (float*)(w + o[1]);
        a->parg = (int*)(w + o[2]);
        a->wsum = (double*)(w + o[3]);
        a->ended = (int*)(w + o[4]);
        a->c = v->inv_temp * LOG2E;
        a->far = -1000.0 / a->c;
    }
    o[5] = o[4] + up256((int64_t)v->S * 4);           // ended
    return o[5];
}

}  // namespace

extern "C" {

int64_t kqk_verify_workspace(const kq_spec_verify* v) { return layout(v, nullptr, nullptr); }

int kqk_launch_verify(const kq_spec_verify* v, void* work, hipStream_t st) {
    if (v->S < 1 || v->T < 0 || v->T > KQ_VERIFY_MAX_DRAFT || v->V < 1)
        return (int)hipErrorInvalidValue;
    VfArg a;
    layout(v, &a, static_cast<uint8_t*>(work));
    const bool greedy = v->flags & KQ_VERIFY_GREEDY, logits = v->flags & KQ_VERIFY_LOGITS;
    // Where there are many sequences, a workgroup takes several chunks after it has
    // decided, which each does for itself, and counts itself once (us, 151936 tokens,
    // one chunk each / this: 32 sequences of 7 111 / 96, 64 of 3 140 / 112, 128 of 2
    // 280 / 168; 256 of 4 over 32000 135 / 108); few, one, as a chunk more is 3 us more
    // (one sequence of 4 15.3 / 19.1 with two, sixteen of 7 56.9 / 58.2).
    const long per = (long)v->S * a.nch / 512;
    a.cpw = per < 1 ? 1 : per > 6 ? 6 : (int)per;
    const dim3 chunks((unsigned)((a.nch + a.cpw - 1) / a.cpw), (unsigned)v->S), wg(TH), seqs((unsigned)v->S);
    if (greedy || logits) {
        const dim3 grid((unsigned)a.nch, (unsigned)(v->S * (v->T + 1) + (v->draft && !greedy ? v->S * v->T : 0)));
        if (greedy) hipLaunchKernelGGL(kq_vf_stats_kernel<true>, grid, wg, 0, st, a);
        else hipLaunchKernelGGL(kq_vf_stats_kernel<false>, grid, wg, 0, st, a);
    }
    if (greedy) {
        hipLaunchKernelGGL(kq_vf_greedy_kernel, seqs, wg, 0, st, a);
    } else if (logits) {
        hipLaunchKernelGGL(kq_vf_weights_kernel<true>, chunks, wg, 0, st, a);
    } else {
        hipLaunchKernelGGL(kq_vf_weights_kernel<false>, chunks, wg, 0, st, a);
        hipLaunchKernelGGL(kq_vf_draw_kernel, seqs, dim3(64), 0, st, a);
    }
    return (int)hipGetLastError();
}

}
