// kq_w4.hip -- products with 4-bit weights and group scales (gfx950).
//
//   y[b][n] = add[b][n] + sum over groups g of
//             s[n][g] * sum over k in g of (q[n][k] - z[n][g]) x[b][k]
//
// Weights are planes, not blocks: a row is K / 2 bytes of nibbles (weight 2j
// in byte j's low half), its scales and zero points lie in planes of their own.
//
// All products are integer.  A nibble becomes a byte with one AND (a shift
// and an AND for the other half), so x is brought to bytes too: per block of
// 32 values, x = xs * v with v an integer in P signed base-256 digits.  int8
// rows are P = 1 as they come.  Binary32 rows are P = 3: xs is the power of
// two that puts the block's largest |v| in (2^21, 2^22], so v is off by half a
// unit, 2^-22 of that largest value, as x's own last bits are from the value
// it was computed from.  Per block, sum q v (at most 480 * 2^22 < 2^31) is
// exact; blocks are scaled and added in binary32.
#include <hip/hip_runtime.h>
#include <hip/hip_fp16.h>
#include <stdint.h>

#include "kq_launch.h"

#pragma clang fp contract(off)

namespace {

struct W4Arg {
    kq_w4 w;
    const float* x;
    const int8_t* xq;
    const float* xs;
    const float* add;
    float* y;
    int nblk, ngrp;          // blocks of 32, groups of a row
    unsigned gmagic;         // block -> group (group_of)
    int rs, rpw;             // rows of a step, of a workgroup
    int pass, tstride, red;  // steps of a pass; floats of a row of terms; lanes that add them up
};

// c / (group / 32), with gmagic = floor(2^31 / (group / 32)) + 1: exact while
// (2 c + 1) (group / 32) < 2^31, which K <= 2^20 keeps
__device__ __forceinline__ int group_of(const W4Arg& a, int c) {
    return (int)__umulhi(2u * (unsigned)c + 1u, a.gmagic);
}

__device__ __forceinline__ float w4_scale(const kq_w4& w, long i) {
    if (w.scale_type == KQ_TYPE_F16) return __half2float(static_cast<const __half*>(w.scales)[i]);
    if (w.scale_type == KQ_TYPE_F32) return static_cast<const float*>(w.scales)[i];
    return __uint_as_float((uint32_t)static_cast<const uint16_t*>(w.scales)[i] << 16);
}

// What a step loads per 32 weights beside them.  A kernel is compiled for each
// MODE, because a branch around a load makes every later wait for loads wait
// for all of them.
constexpr int M_16 = 0, M_16Z = 1, M_32Z = 2;   // 16-bit scales; with zeros; binary32, with or without

// Bytes [at, end) of a plane as a buffer: what is asked for behind its end
// reads as zero and touches nothing.  (Offsets go in the address register: the
// scalar offset is not in the range check.)
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ __amdgpu_buffer_rsrc_t plane(const void* p, long at, long end) {
    return __builtin_amdgcn_make_buffer_rsrc(
        const_cast<uint8_t*>(static_cast<const uint8_t*>(p)) + at, 0, (int)(end - at), 0x00027000);
}

template <int MODE>
struct RawScale {
    static constexpr int SB = MODE == M_32Z ? 4 : 2;      // bytes of a scale
    uint32_t s, z;
    __device__ __forceinline__ void load(__amdgpu_buffer_rsrc_t sp, __amdgpu_buffer_rsrc_t zp, int e) {
        if (MODE == M_32Z) s = __builtin_amdgcn_raw_buffer_load_b32(sp, SB * e, 0, 0);
        else s = __builtin_amdgcn_raw_buffer_load_b16(sp, SB * e, 0, 0);
        if (MODE != M_16) z = __builtin_amdgcn_raw_buffer_load_b8(zp, e, 0, 0);
    }
    __device__ __forceinline__ float scale(bool half) const {
        if (MODE == M_32Z) return __uint_as_float(s);
        const float h = __half2float(__ushort_as_half((unsigned short)s));
        return half ? h : __uint_as_float(s << 16);
    }
    __device__ __forceinline__ float zero(bool zeros) const {
        return MODE == M_16 || (MODE == M_32Z && !zeros) ? 8.0f : (float)(z & 15);
    }
};

// bytes `sel` of the pair {hi, lo}: lo's are 0..3
__device__ __forceinline__ uint32_t perm(uint32_t hi, uint32_t lo, uint32_t sel) {
    return __builtin_amdgcn_perm(hi, lo, sel);
}

// 8 consecutive binary32 x of one stream as 3 digits: by plane, the even values'
// bytes and the odd ones' (as the weights' low and high nibbles come).  4
// neighbouring lanes hold a block and agree on its scale and sum.
struct X8 {
    uint32_t even[3], odd[3];
    float scale, sum;        // xs; xs * sum of v over the block
};

template <int CTRL>
__device__ __forceinline__ int dpp(int v) {
    return __builtin_amdgcn_mov_dpp(v, CTRL, 0xf, 0xf, false);
}
constexpr int QUAD_1 = 0xB1, QUAD_2 = 0x4E;    // lane ^ 1 and lane ^ 2 of 4
constexpr int HALF_MIRROR = 0x141, MIRROR = 0x140;   // the other 4 of 8, the other 8 of 16

__device__ __forceinline__ X8 split_x(const uint4 lo, const uint4 hi) {
    X8 o;
    const uint32_t b[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
    uint32_t am = 0;                    // as integers: infinity and NaN are above all
#pragma unroll
    for (int i = 0; i < 8; i++) am = max(am, b[i] & 0x7fffffffu);
    am = max(am, (uint32_t)dpp<QUAD_1>((int)am));
    am = max(am, (uint32_t)dpp<QUAD_2>((int)am));
    const bool fine = am < 0x7f800000u;
    const int ex = max(1, (int)(am >> 23));              // |x| < 2^(ex - 126)
    o.scale = fine ? ldexpf(1.0f, ex - 148) : NAN;
    // v = x 2^(148 - ex), to the nearest: the low bits of v + 1.5 * 2^23.  The
    // factor in two parts, as it may lie past the binary32 range.
    const float f1 = ex < 64 ? 0x1p64f : 1.0f, f2 = ldexpf(1.0f, (ex < 64 ? 84 : 148) - ex);
    const uint32_t base = 0x4b400000;
    uint32_t sum8 = 0;
    uint32_t u[8];
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const uint32_t t = __float_as_uint(fmaf(__uint_as_float(b[i]) * f1, f2, 0x1.8p23f));
        sum8 += t;
        u[i] = (t + (0x8080u - base)) ^ 0x8080u;     // bytes: the signed digits
    }
    int sum = (int)(sum8 - 8u * base);
#pragma unroll
    for (int p = 0; p < 3; p++) {
        const uint32_t s2 = 0x0c0c0400u + 0x0101u * p;   // byte p of both, zeros above
        o.even[p] = perm(u[2], u[0], s2) | perm(u[6], u[4], s2) << 16;
        o.odd[p] = perm(u[3], u[1], s2) | perm(u[7], u[5], s2) << 16;
    }
    sum += dpp<QUAD_1>(sum);
    sum += dpp<QUAD_2>(sum);
    o.sum = o.scale * (float)sum;
    return o;
}

// A barrier for LDS only: __syncthreads would wait for the weights that are
// on their way.
__device__ __forceinline__ void lds_barrier() {
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

// Steps of weights in flight, and the waves a SIMD has to hold, of the walk
// below: 8 NB P registers hold x, 5 or 6 each step.  (2 and 5 steps, 4 to 8
// waves: within 5 % of each other.)
constexpr int WALK_D = 3;
constexpr int walk_waves(int P, int NB) { return P * NB <= 3 ? 5 : P * NB <= 6 ? 4 : 3; }

// Few streams, on the vector ALU.  A workgroup has rs rows' worth of lanes, a
// lane per block of 32 weights, and walks down its rows rs at a time: a lane
// stays at its block of the row, so it holds that block of x (of NB streams) in
// registers, and a step's weights are rs neighbouring rows in address order.
// A lane's term of a row goes to LDS; after a pass of steps a few lanes add up
// each row's terms, while the next pass goes on with the other half of the buffer.
template <int P, int NB, int MODE>
__global__ __launch_bounds__(1024, walk_waves(P, NB)) void kq_w4_walk_kernel(W4Arg a) {
    extern __shared__ __align__(16) uint8_t smem[];
    constexpr int D = WALK_D;
    const int nblk = a.nblk, tid = threadIdx.x, T = blockDim.x, rs = a.rs;
    const bool half = a.w.scale_type == KQ_TYPE_F16, zeros = a.w.zeros != nullptr;
    const long r0 = (long)blockIdx.x * a.rpw;
    const int rows = (int)min((long)a.rpw, a.w.N - r0);
    const int u = min(tid, rs * nblk - 1), sub = u / nblk, c = u - sub * nblk;
    const bool mine = tid < rs * nblk;

    // x is asked for before the weights: loads return in order
    constexpr int XT = 4;               // binary32: up to 4 pieces of 8 values a lane at once
    uint4 xr[P == 1 ? 2 * NB : 2 * XT];
    float xs[NB], xz[NB];
    const int xn = NB * nblk * 4;
    if constexpr (P == 1) {
#pragma unroll
        for (int s = 0; s < NB; s++) {
            const uint4* src = reinterpret_cast<const uint4*>(a.xq + (long)s * a.w.K + 32 * c);
            xr[2 * s] = src[0];
            xr[2 * s + 1] = src[1];
            xs[s] = a.xs[(long)s * nblk + c];
        }
    } else {
#pragma unroll
        for (int j = 0; j < XT; j++) {
            const int i = min(tid + j * T, xn - 4 + (tid & 3));
            if (j * T < xn) {
                const uint4* src = reinterpret_cast<const uint4*>(a.x + 8L * i);
                xr[2 * j] = src[0];
                xr[2 * j + 1] = src[1];
            }
        }
    }

    struct Raw { uint4 q; RawScale<MODE> s; };
    const long rowb = 16L * nblk, rowsb = (long)a.ngrp * RawScale<MODE>::SB;
    const auto qp = plane(a.w.q, r0 * rowb, (r0 + rows) * rowb);
    const auto sp = plane(a.w.scales, r0 * rowsb, (r0 + rows) * rowsb);
    const auto zp = plane(zeros ? a.w.zeros : a.w.scales, zeros ? r0 * a.ngrp : 0,
                          zeros ? (r0 + rows) * a.ngrp : 0);
    uint32_t vq = 16u * u;
    int ve = sub * a.ngrp + group_of(a, c);
    auto load = [&](Raw& t) {
        const u32x4 v = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(qp, (int)vq, 0, 0));
        t.q = make_uint4(v.x, v.y, v.z, v.w);
        t.s.load(sp, zp, ve);
        vq += (uint32_t)rs * (uint32_t)rowb;
        ve += rs * a.ngrp;
    };
    Raw ring[D];
#pragma unroll
    for (int d = 0; d < D - 1; d++) load(ring[d]);

    uint32_t xe[NB][P][4], xo[NB][P][4];
    if constexpr (P == 1) {
#pragma unroll
        for (int s = 0; s < NB; s++) {
            const uint32_t w[8] = {xr[2 * s].x, xr[2 * s].y, xr[2 * s].z, xr[2 * s].w,
                                   xr[2 * s + 1].x, xr[2 * s + 1].y, xr[2 * s + 1].z, xr[2 * s + 1].w};
            int sum = 0;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                xe[s][0][i] = perm(w[2 * i + 1], w[2 * i], 0x06040200);
                xo[s][0][i] = perm(w[2 * i + 1], w[2 * i], 0x07050301);
                sum = __builtin_amdgcn_sdot4((int)xe[s][0][i], 0x01010101, sum, false);
                sum = __builtin_amdgcn_sdot4((int)xo[s][0][i], 0x01010101, sum, false);
            }
            xz[s] = xs[s] * (float)sum;
        }
    } else {
        // [stream][plane][even, odd][block] of 16 bytes, then {xs, xs sum}
        uint32_t* const xp = reinterpret_cast<uint32_t*>(smem);
        float2* const meta = reinterpret_cast<float2*>(smem + (size_t)NB * P * nblk * 32);
        auto put = [&](int i, const uint4 lo, const uint4 hi) {
            const X8 v = split_x(lo, hi);
            const int s = i / (nblk * 4), e8 = i - s * nblk * 4;
            uint32_t* d = xp + s * P * 2 * nblk * 4 + e8;
#pragma unroll
            for (int p = 0; p < P; p++) {
                d[2 * p * nblk * 4] = v.even[p];
                d[(2 * p + 1) * nblk * 4] = v.odd[p];
            }
            if ((e8 & 3) == 0) meta[s * nblk + (e8 >> 2)] = make_float2(v.scale, v.sum);
        };
#pragma unroll
        for (int j = 0; j < XT; j++)
            if (tid + j * T < xn) put(tid + j * T, xr[2 * j], xr[2 * j + 1]);
        for (int i = tid + XT * T; i < xn; i += T) {
            const uint4* src = reinterpret_cast<const uint4*>(a.x + 8L * i);
            put(i, src[0], src[1]);
        }
        lds_barrier();
        const uint4* const xv = reinterpret_cast<const uint4*>(smem);
#pragma unroll
        for (int s = 0; s < NB; s++) {
#pragma unroll
            for (int p = 0; p < P; p++) {
                const uint4 e = xv[((s * P + p) * 2) * nblk + c], o = xv[((s * P + p) * 2 + 1) * nblk + c];
                xe[s][p][0] = e.x; xe[s][p][1] = e.y; xe[s][p][2] = e.z; xe[s][p][3] = e.w;
                xo[s][p][0] = o.x; xo[s][p][1] = o.y; xo[s][p][2] = o.z; xo[s][p][3] = o.w;
            }
            const float2 m = meta[s * nblk + c];
            xs[s] = m.x;
            xz[s] = m.y;
        }
        lds_barrier();
    }

    float* const terms = reinterpret_cast<float*>(smem);
    const int prow = a.pass * rs, tsize = prow * a.tstride;      // rows of a pass; a stream's terms
    const int steps = (rows + rs - 1) / rs;
    int half_at = 0;                                              // the half of the buffer in use
    for (int k0 = 0; k0 < steps; k0 += a.pass) {
        float* t = terms + half_at + sub * a.tstride + c;
        const int kn = min(a.pass, steps - k0);
        for (int k = 0; k < kn; k += D) {                         // (a.pass is a multiple of D)
#pragma unroll
            for (int j = 0; j < D; j++) {
                load(ring[(j + D - 1) % D]);
                if (k + j < kn) {
                    const Raw& cur = ring[j];
                    const uint32_t d[4] = {cur.q.x, cur.q.y, cur.q.z, cur.q.w};
                    uint32_t lo[4], hi[4];
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        lo[i] = d[i] & 0x0f0f0f0fu;
                        hi[i] = (d[i] >> 4) & 0x0f0f0f0fu;
                    }
                    const float sc = cur.s.scale(half), ze = cur.s.zero(zeros);
#pragma unroll
                    for (int s = 0; s < NB; s++) {
                        int dot = 0;
#pragma unroll
                        for (int p = P - 1; p >= 0; p--) {
                            if (p < P - 1) dot = dot << 8;
#pragma unroll
                            for (int i = 0; i < 4; i++) {
                                dot = __builtin_amdgcn_sdot4((int)lo[i], (int)xe[s][p][i], dot, false);
                                dot = __builtin_amdgcn_sdot4((int)hi[i], (int)xo[s][p][i], dot, false);
                            }
                        }
                        if (mine) t[s * tsize] = sc * fmaf(-ze, xz[s], xs[s] * (float)dot);
                    }
                    t += rs * a.tstride;
                }
            }
        }
        lds_barrier();
        // LR lanes a row: lane j takes terms j, j + LR, ...
        const int n = min(kn * rs, rows - k0 * rs), LR = a.red, j0 = tid & (LR - 1);
        const int rstep = T >> (LR == 4 ? 2 : 4);
#pragma unroll
        for (int s = 0; s < NB; s++)
            for (int r = tid >> (LR == 4 ? 2 : 4); r < n; r += rstep) {
                const float* v = terms + half_at + s * tsize + r * a.tstride;
                float sum = 0.0f;
                int j = j0;
                for (; j + 3 * LR < nblk; j += 4 * LR) {
                    const float v0 = v[j], v1 = v[j + LR], v2 = v[j + 2 * LR], v3 = v[j + 3 * LR];
                    sum = sum + ((v0 + v1) + (v2 + v3));
                }
                for (; j < nblk; j += LR) sum = sum + v[j];
                sum = sum + __int_as_float(dpp<QUAD_1>(__float_as_int(sum)));
                sum = sum + __int_as_float(dpp<QUAD_2>(__float_as_int(sum)));
                if (LR == 16) {
                    sum = sum + __int_as_float(dpp<HALF_MIRROR>(__float_as_int(sum)));
                    sum = sum + __int_as_float(dpp<MIRROR>(__float_as_int(sum)));
                }
                const long o = (long)s * a.w.N + r0 + k0 * rs + r;
                if (j0 == 0) a.y[o] = a.add ? a.add[o] + sum : sum;
            }
        half_at = NB * tsize - half_at;
    }
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
        const float s = w4_scale(w, g);
        const int z = w.zeros ? w.zeros[g] & 15 : 8;
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

// ------------------------------------------------------------- the plan

constexpr int WALK_MAX_BLK = 1024;
constexpr int walk_max_b(int P) { return P == 1 ? 4 : 3; }     // (more spill registers)
int g_lds_max = 65536;

// Rows of a step and of a workgroup, steps of a pass, LDS bytes (-1: not
// taken).  Two workgroups a CU, of as many waves as the registers allow,
// where the row is short enough; one where the matrix is a step's work of
// one (1024 x 1024: 3.1 us against 3.5, 17408 x 5120 11.6 against 11.5).
long walk_plan(W4Arg& a, int P, int NB, int n_cu) {
    const int nblk = a.nblk, waves = 4 * walk_waves(P, NB), D = WALK_D;
    const long N = a.w.N, rowb = 16L * nblk;
    const bool small = (N + n_cu - 1) / n_cu * nblk <= 512;
    const int per_cu = nblk <= 32 * waves && !small ? 2 : 1, lanes = 64 * waves / per_cu;
    const long slots = (long)per_cu * n_cu;
    const long fair = (N + slots - 1) / slots;         // rows of a workgroup, were they cut evenly
    const long fits = (lanes < 1024 ? lanes : 1024) / nblk;
    if (fits < 1) return -1;
    a.rs = (int)(fair < fits ? fair : fits);
    const long steps = (fair + a.rs - 1) / a.rs;
    long rpw = steps * a.rs;
    const long most = (1L << 30) / rowb / a.rs * a.rs;  // 32-bit offsets
    if (rpw > most) rpw = most;
    a.rpw = (int)rpw;
    // no bank conflicts: 16 rows of 4 lanes each, 4 apart, or 4 rows of 16
    a.red = nblk <= 64 ? 4 : 16;
    a.tstride = a.red == 4 ? (nblk + 3) / 8 * 8 + 4 : (nblk + 15) / 32 * 32 + 16;
    const long stage = P == 1 ? 0 : (long)NB * nblk * (32 * P + 8), budget = g_lds_max / per_cu;
    const long step = 4L * NB * a.rs * a.tstride, all = rpw / a.rs;
    const long once = (all + D - 1) / D * D;
    a.pass = (int)(once * step <= budget ? once : budget / (2 * step) / D * D);
    if (a.pass < D || stage > budget) return -1;
    const long terms = a.pass >= all ? a.pass * step : 2 * a.pass * step;
    return stage > terms ? stage : terms;
}

template <int P, int NB, int MODE>
int launch_walk_m(const W4Arg& a, long lds, hipStream_t st) {
    const dim3 grid((unsigned)((a.w.N + a.rpw - 1) / a.rpw)), wg((unsigned)((a.rs * a.nblk + 63) & ~63));
    hipLaunchKernelGGL((kq_w4_walk_kernel<P, NB, MODE>), grid, wg, (size_t)lds, st, a);
    return (int)hipGetLastError();
}

template <int P, int NB>
int launch_walk(const W4Arg& a, long lds, hipStream_t st) {
    if (a.w.scale_type == KQ_TYPE_F32) return launch_walk_m<P, NB, M_32Z>(a, lds, st);
    return a.w.zeros ? launch_walk_m<P, NB, M_16Z>(a, lds, st) : launch_walk_m<P, NB, M_16>(a, lds, st);
}

template <int P>
int launch_walk_b(const W4Arg& a, int B, long lds, hipStream_t st) {
    if (B == 1) return launch_walk<P, 1>(a, lds, st);
    if (B == 2) return launch_walk<P, 2>(a, lds, st);
    if constexpr (walk_max_b(P) > 3)
        if (B == 4) return launch_walk<P, 4>(a, lds, st);
    return launch_walk<P, 3>(a, lds, st);
}

template <int P, int NB, int MODE>
int raise_lds_m(int bytes) {
    return (int)hipFuncSetAttribute((const void*)kq_w4_walk_kernel<P, NB, MODE>,
                                    hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
}

template <int P, int NB>
int raise_lds(int bytes) {
    const int e = raise_lds_m<P, NB, M_16>(bytes), f = raise_lds_m<P, NB, M_16Z>(bytes),
              g = raise_lds_m<P, NB, M_32Z>(bytes);
    return e ? e : f ? f : g;
}

}  // namespace

extern "C" {

int kqk_w4_set_max_lds(int bytes) {
    g_lds_max = bytes;
    const int e[7] = {raise_lds<1, 1>(bytes), raise_lds<1, 2>(bytes), raise_lds<1, 3>(bytes),
                      raise_lds<1, 4>(bytes), raise_lds<3, 1>(bytes), raise_lds<3, 2>(bytes),
                      raise_lds<3, 3>(bytes)};
    for (int i = 0; i < 7; i++)
        if (e[i]) return e[i];
    return 0;
}

int64_t kqk_w4_workspace(const kq_w4* w, int B, int q8, int n_cu) { return 0; }

int kqk_launch_w4(const kq_w4* w, const float* x, const int8_t* xq, const float* xs,
                  const float* add, float* y, int B, void* work, int n_cu, hipStream_t st) {
    if (w->N < 1 || w->K < 32 || w->K % 32 || B < 1) return (int)hipErrorInvalidValue;
    W4Arg a;
    a.w = *w;
    a.x = x; a.xq = xq; a.xs = xs; a.add = add; a.y = y;
    a.nblk = w->K / 32;
    a.ngrp = w->K / w->group;
    a.gmagic = (1u << 31) / (unsigned)(w->group / 32) + 1;
    if (B <= walk_max_b(xq ? 1 : 3) && a.nblk <= WALK_MAX_BLK) {
        const long lds = walk_plan(a, xq ? 1 : 3, B, n_cu);
        if (lds > 0) return xq ? launch_walk_b<1>(a, B, lds, st) : launch_walk_b<3>(a, B, lds, st);
    }
    const dim3 grid((unsigned)((w->N + 3) / 4), (unsigned)((B + 3) / 4));
    if (xq)
        hipLaunchKernelGGL(kq_w4_kernel<true>, grid, dim3(256), 0, st, *w, x, xq, xs, add, y, B);
    else
        hipLaunchKernelGGL(kq_w4_kernel<false>, grid, dim3(256), 0, st, *w, x, xq, xs, add, y, B);
    return (int)hipGetLastError();
}

}
