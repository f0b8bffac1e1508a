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
    int isum;                // that sum of v
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
    o.isum = sum;
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

// ---------------------------------------------------- 4 and more streams
// On the int8 matrix cores: one v_mfma_i32_16x16x32_i8 takes a block of 32 of
// 16 streams (one digit) against the same block of 16 rows; D[stream 4 (l / 16)
// + i][row l % 16] in lane l.
//
// A wave stays at M windows of 128 weights of the row and walks down the rows
// 16 at a time, so its streams' x stays in registers in the operand's layout
// (8 bytes a lane, block and digit).  A lane's 16 bytes of a window are one
// block of one row; four lane-group swaps bring its four dwords to the four
// lanes that the operand wants them in.  The digits share an accumulator: what
// the higher ones gave is shifted by 8 in between.  C0 = -8 sum v makes it sum
// (q - 8) v; zero points other than 8 are taken off per block with xz.
// The waves' sums of a step meet in LDS.

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

// x of one tile of 16 streams as the kernel reads it, per block: P digits of
// 64 lanes' 8 bytes (lane 16 q + s: stream s, positions 8 q .. 8 q + 7, the even
// ones' bytes first), then xs[16], C0[16] and xz[16].
constexpr int mm_xbytes(int P) { return P * 512; }
constexpr int MM_META = 192;

// One lane per 8 values: binary32 rows (P = 3) or int8 rows (P = 1) to the layout
// above, streams past B and blocks past the row's end as zeros.
template <int P>
__global__ __launch_bounds__(256) void kq_w4_split_kernel(W4Arg a, int B, int nblkp, uint8_t* xop,
                                                          uint8_t* meta) {
    const int i = blockIdx.x * 256 + threadIdx.x;        // [block][stream][4]
    const int q = i & 3, s = (i >> 2) & 15, b = i >> 6, tile = blockIdx.y, st = tile * 16 + s;
    if (b >= nblkp) return;
    const bool on = st < B && b < a.nblk;
    uint2 o[P];
    float scale, xz;
    int sum;
    if constexpr (P == 3) {
        uint4 lo = make_uint4(0, 0, 0, 0), hi = lo;
        if (on) {
            const uint4* src = reinterpret_cast<const uint4*>(a.x + (long)st * a.w.K + 32L * b + 8 * q);
            lo = src[0];
            hi = src[1];
        }
        const X8 v = split_x(lo, hi);
#pragma unroll
        for (int p = 0; p < P; p++) o[p] = make_uint2(v.even[p], v.odd[p]);
        scale = v.scale;
        xz = v.sum;
        sum = v.isum;
    } else {
        uint2 v = make_uint2(0, 0);
        if (on) v = *reinterpret_cast<const uint2*>(a.xq + (long)st * a.w.K + 32L * b + 8 * q);
        o[0] = make_uint2(perm(v.y, v.x, 0x06040200), perm(v.y, v.x, 0x07050301));
        sum = __builtin_amdgcn_sdot4((int)v.x, 0x01010101, 0, false);
        sum = __builtin_amdgcn_sdot4((int)v.y, 0x01010101, sum, false);
        sum += dpp<QUAD_1>(sum);
        sum += dpp<QUAD_2>(sum);
        scale = on ? a.xs[(long)st * a.nblk + b] : 0.0f;
        xz = scale * (float)sum;
    }
    uint2* const x = reinterpret_cast<uint2*>(xop + ((long)tile * nblkp + b) * mm_xbytes(P));
#pragma unroll
    for (int p = 0; p < P; p++) x[p * 64 + 16 * q + s] = o[p];
    uint32_t* const m = reinterpret_cast<uint32_t*>(meta + ((long)tile * nblkp + b) * MM_META);
    if (q == 0) m[s] = __float_as_uint(scale);
    if (q == 1) m[16 + s] = (uint32_t)(-8 * sum);
    if (q == 2) m[32 + s] = __float_as_uint(xz);
}

struct MmArg {
    W4Arg a;
    int B, ntile;            // streams, tiles of 16
    int nblkp, nwin;         // blocks and windows of a padded row
    int nw, ks;              // windows of a workgroup, parts of a row
    int steps;               // steps of 16 rows of a workgroup
    const uint8_t* xop;
    const uint8_t* meta;
    float* part;             // ks > 1: [ks][B][N]
};

constexpr int MM_PASS = 2;   // steps between barriers
constexpr int MM_ROW = 17;   // floats of a row's 16 streams in LDS

constexpr int mm_waves(int P, int M) { return P == 3 ? (M <= 1 ? 4 : M <= 2 ? 3 : 2) : M <= 2 ? 4 : M <= 4 ? 3 : 2; }

// ONE: a window lies in one group (group % 128 == 0)
template <int P, int M, int MODE, bool ONE>
__global__ __launch_bounds__(512, mm_waves(P, M)) void kq_w4_mm_kernel(MmArg g) {
    extern __shared__ __align__(16) uint8_t smem[];
    const W4Arg& a = g.a;
    const int tid = threadIdx.x, T = blockDim.x, lane = tid & 63, n = lane & 15, q = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), W = T >> 6;
    // workgroups of the same rows next to each other: tile, then part of the row
    const int tile = blockIdx.x % g.ntile, rest = blockIdx.x / g.ntile;
    const int part = rest % g.ks, w0 = part * g.nw + wave * M;       // first window
    const long r0 = (long)(rest / g.ks) * g.steps * 16;
    const int rows = (int)min((long)g.steps * 16, a.w.N - r0);
    const bool half = a.w.scale_type == KQ_TYPE_F16, zeros = a.w.zeros != nullptr;
    const int wend = min(g.nwin, (part + 1) * g.nw);                 // windows of this part end here

    const long rowb = 16L * a.nblk, rowsb = (long)a.ngrp * RawScale<MODE>::SB;
    const auto qp = plane(a.w.q, r0 * rowb, (r0 + rows) * rowb);
    const auto sp = plane(a.w.scales, r0 * rowsb, (r0 + rows) * rowsb);
    const auto zp = plane(zeros ? a.w.zeros : a.w.scales, zeros ? r0 * a.ngrp : 0,
                          zeros ? (r0 + rows) * a.ngrp : 0);

    // scales: lane group q loads window (ONE) or block (else) 4 k + q's
    constexpr int NS = ONE ? (M + 3) / 4 : M;
    struct Raw { uint4 q[M]; RawScale<MODE> s[NS]; };
    uint32_t vq = (uint32_t)n * (uint32_t)rowb + 64u * w0 + 16u * q;
    int ve[NS];
#pragma unroll
    for (int k = 0; k < NS; k++) {
        const int blk = ONE ? 4 * (w0 + 4 * k + q) : 4 * (w0 + k) + q;
        ve[k] = n * a.ngrp + min(group_of(a, min(blk, a.nblk - 1)), a.ngrp - 1);
    }
    auto load = [&](Raw& t) {
#pragma unroll
        for (int j = 0; j < M; j++) {
            const u32x4 v = __builtin_bit_cast(
                u32x4, __builtin_amdgcn_raw_buffer_load_b128(qp, (int)(vq + 64u * j), 0, 0));
            t.q[j] = make_uint4(v.x, v.y, v.z, v.w);
        }
#pragma unroll
        for (int k = 0; k < NS; k++) {
            t.s[k].load(sp, zp, ve[k]);
            ve[k] += 16 * a.ngrp;
        }
        vq += 16u * (uint32_t)rowb;
    };
    Raw cur, nxt;
    load(cur);

    // this wave's x, and the workgroup's block data to LDS
    uint2 x[M][4][P];
#pragma unroll
    for (int j = 0; j < M; j++)
#pragma unroll
        for (int b = 0; b < 4; b++)
#pragma unroll
            for (int p = 0; p < P; p++) {
                x[j][b][p] = make_uint2(0, 0);
                if (w0 + j < wend)
                    x[j][b][p] = reinterpret_cast<const uint2*>(
                        g.xop + ((long)tile * g.nblkp + 4 * (w0 + j) + b) * mm_xbytes(P))[64 * p + lane];
            }
    const int mblk = 4 * W * M;                                       // blocks in LDS
    float* const xsum = reinterpret_cast<float*>(smem + (size_t)mblk * MM_META);
    for (int i = tid; i < mblk * (MM_META / 16); i += T) {
        const int b = i / (MM_META / 16), blk = 4 * part * g.nw + b;
        uint4 v = make_uint4(0, 0, 0, 0);
        if (blk < 4 * wend)
            v = reinterpret_cast<const uint4*>(g.meta + ((long)tile * g.nblkp + blk) * MM_META)[i % (MM_META / 16)];
        reinterpret_cast<uint4*>(smem)[i] = v;
    }
    lds_barrier();

    const int half_floats = MM_PASS * W * 16 * MM_ROW;
    int at = 0;
    for (int k0 = 0; k0 < g.steps; k0 += MM_PASS) {
#pragma unroll 1
        for (int k = 0; k < MM_PASS; k++) {
            load(nxt);
            f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int j = 0; j < M; j++) {
                // dword k of block b, from register k of lane group b to register b of group k
                const auto p02 = __builtin_amdgcn_permlane32_swap(cur.q[j].x, cur.q[j].z, false, false);
                const auto p13 = __builtin_amdgcn_permlane32_swap(cur.q[j].y, cur.q[j].w, false, false);
                const auto b01 = __builtin_amdgcn_permlane16_swap(p02[0], p13[0], false, false);
                const auto b23 = __builtin_amdgcn_permlane16_swap(p02[1], p13[1], false, false);
                const uint32_t d[4] = {b01[0], b01[1], b23[0], b23[1]};
                // the scales of the window or its blocks, to all lane groups
                const RawScale<MODE>& rs = cur.s[ONE ? j / 4 : j];
                float sc[4], ze[4];
                {
                    const float s = rs.scale(half);
                    const auto e = __builtin_amdgcn_permlane16_swap(__float_as_uint(s), __float_as_uint(s), false, false);
                    const auto lo = __builtin_amdgcn_permlane32_swap(e[0], e[0], false, false);
                    const auto hi = __builtin_amdgcn_permlane32_swap(e[1], e[1], false, false);
                    sc[0] = __uint_as_float(lo[0]); sc[1] = __uint_as_float(hi[0]);
                    sc[2] = __uint_as_float(lo[1]); sc[3] = __uint_as_float(hi[1]);
                }
                if (MODE != M_16) {
                    const float z = rs.zero(zeros) - 8.0f;
                    const auto e = __builtin_amdgcn_permlane16_swap(__float_as_uint(z), __float_as_uint(z), false, false);
                    const auto lo = __builtin_amdgcn_permlane32_swap(e[0], e[0], false, false);
                    const auto hi = __builtin_amdgcn_permlane32_swap(e[1], e[1], false, false);
                    ze[0] = __uint_as_float(lo[0]); ze[1] = __uint_as_float(hi[0]);
                    ze[2] = __uint_as_float(lo[1]); ze[3] = __uint_as_float(hi[1]);
                }
                f32x4 t = {0.0f, 0.0f, 0.0f, 0.0f};
                const uint8_t* mb = smem + (size_t)(4 * (wave * M + j)) * MM_META + 16 * q;
#pragma unroll
                for (int b = 0; b < 4; b++) {
                    const long w = (long)(((uint64_t)((d[b] >> 4) & 0x0f0f0f0fu) << 32) | (d[b] & 0x0f0f0f0fu));
                    const f32x4 xs = *reinterpret_cast<const f32x4*>(mb + b * MM_META);
                    const i32x4 c0 = *reinterpret_cast<const i32x4*>(mb + b * MM_META + 64);
                    i32x4 D;
                    if constexpr (P == 1) {
                        D = __builtin_amdgcn_mfma_i32_16x16x32_i8(__builtin_bit_cast(long, x[j][b][0]), w, c0, 0, 0, 0);
                    } else {
                        D = i32x4{0, 0, 0, 0};
                        D = __builtin_amdgcn_mfma_i32_16x16x32_i8(__builtin_bit_cast(long, x[j][b][2]), w, D, 0, 0, 0);
                        D = D << 8;
                        D = __builtin_amdgcn_mfma_i32_16x16x32_i8(__builtin_bit_cast(long, x[j][b][1]), w, D, 0, 0, 0);
                        D = (D << 8) + c0;
                        D = __builtin_amdgcn_mfma_i32_16x16x32_i8(__builtin_bit_cast(long, x[j][b][0]), w, D, 0, 0, 0);
                    }
                    f32x4 xz;
                    if (MODE != M_16) xz = *reinterpret_cast<const f32x4*>(mb + b * MM_META + 128);
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        if (ONE) {
                            t[i] = fmaf(xs[i], (float)D[i], t[i]);
                            if (MODE != M_16) t[i] = fmaf(-ze[j & 3], xz[i], t[i]);
                        } else {
                            float v = xs[i] * (float)D[i];
                            if (MODE != M_16) v = fmaf(-ze[b], xz[i], v);
                            acc[i] = fmaf(sc[b], v, acc[i]);
                        }
                    }
                }
                if (ONE) {
#pragma unroll
                    for (int i = 0; i < 4; i++) acc[i] = fmaf(sc[j & 3], t[i], acc[i]);
                }
            }
            float* o = xsum + at + ((k * W + wave) * 16 + n) * MM_ROW + 4 * q;
#pragma unroll
            for (int i = 0; i < 4; i++) o[i] = acc[i];
            cur = nxt;
        }
        lds_barrier();
        // outputs of the pass: rows next to each other
        const int nr = min(MM_PASS * 16, rows - k0 * 16);
        for (int i = tid; i < MM_PASS * 256; i += T) {
            const int r = i & (MM_PASS * 16 - 1), s = i / (MM_PASS * 16), st = tile * 16 + s;
            if (r >= nr || st >= g.B) continue;
            const float* v = xsum + at + ((r >> 4) * W * 16 + (r & 15)) * MM_ROW + s;
            float sum = v[0];
            for (int w = 1; w < W; w++) sum = sum + v[w * 16 * MM_ROW];
            const long o = (long)st * a.w.N + r0 + k0 * 16 + r;
            if (g.ks > 1) g.part[(long)part * g.B * a.w.N + o] = sum;
            else a.y[o] = a.add ? a.add[o] + sum : sum;
        }
        at = half_floats - at;
    }
}

// the parts of rows that were cut, in their order
__global__ __launch_bounds__(256) void kq_w4_join_kernel(const float* part, const float* add, float* y,
                                                         long n, int ks) {
    const long i = (long)blockIdx.x * 256 + threadIdx.x;
    if (i >= n) return;
    float sum = part[i];
    for (int k = 1; k < ks; k++) sum = sum + part[k * n + i];
    y[i] = add ? add[i] + sum : sum;
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

// ------------------------------------------------------- matrix-core plan

constexpr int MM_M = 5, MM_W = 8;        // windows of a wave, waves of a workgroup at most

struct MmPlan { int M, W; long lds, grid, xop, meta, part; };

void mm_plan(MmArg& g, int P, int n_cu, MmPlan* p) {
    const W4Arg& a = g.a;
    g.ntile = (g.B + 15) / 16;
    g.nwin = (a.nblk + 3) / 4;
    g.nblkp = 4 * g.nwin;
    g.ks = (g.nwin + MM_M * MM_W - 1) / (MM_M * MM_W);
    g.nw = (g.nwin + g.ks - 1) / g.ks;
    g.ks = (g.nwin + g.nw - 1) / g.nw;
    p->M = (g.nw + MM_W - 1) / MM_W;
    p->W = (g.nw + p->M - 1) / p->M;
    const long rows16 = (a.w.N + 15) / 16;
    const long slots = (long)n_cu * mm_waves(P, p->M) * 4 / p->W;
    long steps = (rows16 * g.ntile * g.ks + slots - 1) / slots;
    const long most = (1L << 30) / (16L * a.nblk) / 16;        // 32-bit offsets
    if (steps > most) steps = most;
    if (steps > rows16) steps = rows16;
    g.steps = (int)steps;
    p->grid = (rows16 + steps - 1) / steps * g.ks * g.ntile;
    p->lds = 4L * p->W * p->M * MM_META + 2L * MM_PASS * p->W * 16 * MM_ROW * 4;
    p->xop = ((long)g.ntile * g.nblkp * mm_xbytes(P) + 255) & ~255L;
    p->meta = ((long)g.ntile * g.nblkp * MM_META + 255) & ~255L;
    p->part = g.ks > 1 ? ((long)g.ks * g.B * a.w.N * 4 + 255) & ~255L : 0;
}

template <int P, int M, int MODE>
int launch_mm_m(const MmArg& g, const MmPlan& p, hipStream_t st) {
    const dim3 grid((unsigned)p.grid), wg((unsigned)(64 * p.W));
    if (g.a.w.group % 128 == 0)
        hipLaunchKernelGGL((kq_w4_mm_kernel<P, M, MODE, true>), grid, wg, (size_t)p.lds, st, g);
    else
        hipLaunchKernelGGL((kq_w4_mm_kernel<P, M, MODE, false>), grid, wg, (size_t)p.lds, st, g);
    return (int)hipGetLastError();
}

template <int P, int M>
int launch_mm(const MmArg& g, const MmPlan& p, hipStream_t st) {
    if (g.a.w.scale_type == KQ_TYPE_F32) return launch_mm_m<P, M, M_32Z>(g, p, st);
    return g.a.w.zeros ? launch_mm_m<P, M, M_16Z>(g, p, st) : launch_mm_m<P, M, M_16>(g, p, st);
}

template <int P>
int launch_mm_all(MmArg& g, const MmPlan& p, uint8_t* work, hipStream_t st) {
    g.xop = work;
    g.meta = work + p.xop;
    g.part = reinterpret_cast<float*>(work + p.xop + p.meta);
    hipLaunchKernelGGL((kq_w4_split_kernel<P>), dim3((unsigned)((g.nblkp * 64 + 255) / 256), (unsigned)g.ntile),
                       dim3(256), 0, st, g.a, g.B, g.nblkp, work, work + p.xop);
    int e = (int)hipGetLastError();
    if (e) return e;
    switch (p.M) {
    case 1: e = launch_mm<P, 1>(g, p, st); break;
    case 2: e = launch_mm<P, 2>(g, p, st); break;
    case 3: e = launch_mm<P, 3>(g, p, st); break;
    case 4: e = launch_mm<P, 4>(g, p, st); break;
    default: e = launch_mm<P, 5>(g, p, st); break;
    }
    if (e || g.ks == 1) return e;
    const long n = (long)g.B * g.a.w.N;
    hipLaunchKernelGGL(kq_w4_join_kernel, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, st, g.part, g.a.add,
                       g.a.y, n, g.ks);
    return (int)hipGetLastError();
}

bool fill(W4Arg& a, const kq_w4* w) {
    a.w = *w;
    a.x = nullptr; a.xq = nullptr; a.xs = nullptr; a.add = nullptr; a.y = nullptr;
    a.nblk = w->K / 32;
    a.ngrp = w->K / w->group;
    a.gmagic = (1u << 31) / (unsigned)(w->group / 32) + 1;
    a.rs = a.rpw = a.pass = a.tstride = a.red = 0;
    return w->N >= 1 && w->K >= 32 && w->K % 32 == 0;
}

// LDS bytes of the walk kernel where it takes the call, else -1.
long walk_takes(W4Arg& a, int P, int B, int n_cu) {
    return B <= walk_max_b(P) && a.nblk <= WALK_MAX_BLK ? walk_plan(a, P, B, n_cu) : -1;
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

int64_t kqk_w4_workspace(const kq_w4* w, int B, int q8, int n_cu) {
    MmArg g;
    MmPlan p;
    fill(g.a, w);
    if (walk_takes(g.a, q8 ? 1 : 3, B, n_cu) > 0) return 0;
    g.B = B;
    mm_plan(g, q8 ? 1 : 3, n_cu, &p);
    return p.xop + p.meta + p.part;
}

int kqk_launch_w4(const kq_w4* w, const float* x, const int8_t* xq, const float* xs,
                  const float* add, float* y, int B, void* work, int n_cu, hipStream_t st) {
    MmArg g;
    MmPlan p;
    W4Arg& a = g.a;
    if (!fill(a, w) || B < 1) return (int)hipErrorInvalidValue;
    a.x = x; a.xq = xq; a.xs = xs; a.add = add; a.y = y;
    const long lds = walk_takes(a, xq ? 1 : 3, B, n_cu);
    if (lds > 0) return xq ? launch_walk_b<1>(a, B, lds, st) : launch_walk_b<3>(a, B, lds, st);
    g.B = B;
    mm_plan(g, xq ? 1 : 3, n_cu, &p);
    uint8_t* const ws = static_cast<uint8_t*>(work);
    return xq ? launch_mm_all<1>(g, p, ws, st) : launch_mm_all<3>(g, p, ws, st);
}

}
