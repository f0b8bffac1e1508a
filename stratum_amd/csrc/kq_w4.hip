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
// it was computed from.  Per block, sum (q - z) v is exact, as is sum q v on its
// way (at most 480 * 2^22 < 2^31): zero points are taken off in integers, so that
// weights at theirs give nothing, whatever x is.  Blocks are scaled and added in
// binary32, by the weights' scale first: sum (q - z) x passes binary32's range from
// |x| of 7e35 on, s sum (q - z) v stays in it for scales below 2^96.
#include <hip/hip_runtime.h>
#include <hip/hip_fp16.h>
#include <stdint.h>
#include <type_traits>

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
    // (as loaded: widening them would wait for them)
    std::conditional_t<MODE == M_32Z, uint32_t, uint16_t> s;
    uint8_t z;
    __device__ __forceinline__ void load(__amdgpu_buffer_rsrc_t sp, __amdgpu_buffer_rsrc_t zp, int e) {
        if (MODE == M_32Z) s = __builtin_amdgcn_raw_buffer_load_b32(sp, SB * e, 0, 0);
        else s = __builtin_amdgcn_raw_buffer_load_b16(sp, SB * e, 0, 0);
        if (MODE != M_16) z = __builtin_amdgcn_raw_buffer_load_b8(zp, e, 0, 0);
    }
    __device__ __forceinline__ float scale(bool half) const {
        if (MODE == M_32Z) return __uint_as_float(s);
        const float h = __half2float(__ushort_as_half((unsigned short)s));
        return half ? h : __uint_as_float((uint32_t)s << 16);
    }
    __device__ __forceinline__ int zero(bool zeros) const {
        return MODE == M_16 || (MODE == M_32Z && !zeros) ? 8 : z & 15;
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
    float scale;
    int sum;                 // of v over the block
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
    o.sum = sum + dpp<QUAD_2>(sum);
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
// The zero point: -8 sum v, kept, where it is 8 for all; else z times sum v, in 24
// bits (binary32 x in two parts, as its sum v has 28).
// The stream of weights bounds it: 17408 x 5120, one stream, 10.7 us, 4.3 TB/s (a plain
// read of these bytes: 9); 5120 x 17408 of int8 rows 10.6 us, 4.6 TB/s; the vector
// ALU is busy for half of that.
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
    float xs[NB];
    int xz[NB], xh[NB];                 // sum v, less 4096 xh of it (P > 1); M_16: -8 sum v
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
            xz[s] = MODE == M_16 ? -8 * sum : sum;
        }
    } else {
        // [stream][plane][even, odd][block] of 16 bytes, then {xs, sum v}
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
            if ((e8 & 3) == 0) meta[s * nblk + (e8 >> 2)] = make_float2(v.scale, __int_as_float(v.sum));
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
            const int sum = __float_as_int(m.y);
            xs[s] = m.x;
            xz[s] = MODE == M_16 ? -8 * sum : sum & 4095;
            xh[s] = sum >> 12;
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
                    const float sc = cur.s.scale(half);
                    const int nz = -cur.s.zero(zeros);
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
                        if (MODE == M_16) {
                            dot += xz[s];
                        } else {
                            dot += __mul24(nz, xz[s]);
                            if (P > 1) dot += __mul24(nz, xh[s]) * 4096;
                        }
                        if (mine) t[s * tsize] = sc * (float)dot * xs[s];
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

// ------------------------------------------------- more streams
// On the int8 matrix cores: one v_mfma_i32_16x16x32_i8 takes a block of 32 of 16
// operand rows against the same block of 16 rows of weights; D[4 (l / 16) +
// i][weight row l % 16] in register i of lane l.  Streams are laid over the
// operand rows so that lane group q holds streams q, q + 4, ... (G of them) and
// nothing else: int8 rows, operand row 4 q + i is stream q + 4 i; binary32 rows,
// one product per 4 streams, operand row 4 q + i is digit i of stream q + 4 g, so
// that a lane has the digits it adds up (the fourth row is not read).
//
// A workgroup has a part of the row (nw windows of 128 weights), whose x it
// brings to digits in LDS, and a run of rows.  Its (tile of 16 rows, window)
// pairs are cut evenly among the waves, wherever that falls: a wave adds up a
// tile's windows in registers and writes the tile out, or, of a tile that it
// shares with other waves, leaves its sum in LDS to be joined behind a barrier.
//
// A window's weights are loaded in address order (lane 4 r + b: block b of row r;
// a row to a lane, as the operand wants them, makes every lane of a load a cache
// access of its own) and change lanes in LDS, in the wave's own 1.5 KB, together
// with their scales.  A nibble becomes q - z on its way to the operand: (q - 8) 16,
// which is the nibble in the byte's high half with its top bit turned (the 16 goes
// with the digits' joining, or with the scale), or, by a zero point of its row,
// q + (128 - z), no byte of which carries, with its top bit turned back.
//
// No unit is full: 17408 x 5120, sixteen int8 streams, 17.7 us (2.7 TB/s of weights),
// the vector ALU and the LDS busy for half of it each, the matrix cores for 0.1; a
// workgroup's 68 rows are five tiles (15 % of whose rows are not there), 100 pairs on 16
// waves, and every workgroup brings x to LDS.  151936 x 1024, five of binary32, 24.9 us
// (3.6 TB/s), 0.6, 0.55 and 0.2.  (Tiles of 32 rows, two operands of weights for one of
// x, when these took 19.1 and 27.6 us: 20.6 us the former, the latter the same.)

typedef int i32x4 __attribute__((ext_vector_type(4)));

// A window's x in LDS: 8 places of P * 4 G entries of 16 bytes, for two blocks
// (pair b2 of the window's) and a lane group each (8 values of either block: the
// even positions' bytes, then the odd ones'); then xs of its blocks, [block][q][G].
// Lane groups q and q ^ 1 are 4 places apart, a multiple of 256 bytes: a read of 16 bytes a lane takes lanes of
// both at once, and so finds them in different banks.
constexpr int mm_place(int b2, int q) { return (q & 1) * 4 + (q >> 1) * 2 + b2; }
constexpr int mm_xbytes(int P, int G) { return 512 * P * G; }
constexpr int mm_window(int P, int G) { return mm_xbytes(P, G) + 64 * G; }

struct MmArg {
    W4Arg a;
    int B, bt, ntile;        // streams, of a tile of streams; those tiles
    int nwin, nw, ks;        // windows of a row, of a part; parts
    int rows;                // of a workgroup
    int xwaves, xmagic;      // waves that bring a stream's x to LDS; w / xwaves = w * xmagic >> 16
    float* part;             // ks > 1: [ks][B][N]
};

constexpr int MM_W = 16;     // waves
constexpr int mm_slot(int G) { return 16 * (4 * G + 1); }   // floats of a tile's sums in LDS
// A wave's own LDS: the sums of the tile that it began with, if others share
// it; 16 rows of a window, 64 bytes each, and their scales and zeros.  What it
// ends with takes the place of the rows.
constexpr int MM_STAGE = 16 * 64 + 64 * 8;
constexpr int mm_wave(int G) { return 4 * mm_slot(G) + MM_STAGE; }
static_assert(4 * mm_slot(4) <= MM_STAGE);
constexpr uint32_t FAR = 0x80000000u;    // an offset behind every buffer's end

// ONE: a window lies in one group (group % 128 == 0)
// ADD: there is something to add (a load of it in the loop makes waits for
// weights wait for all of them)
template <int P, int G, int MODE, bool ONE, bool ADD>
__global__ __launch_bounds__(64 * MM_W) void kq_w4_mm_kernel(MmArg g) {
    extern __shared__ __align__(16) uint8_t smem[];
    constexpr int T = 64 * MM_W, WB = mm_window(P, G), XB = mm_xbytes(P, G), E = P * 4 * G;
    const W4Arg& a = g.a;
    const int tid = threadIdx.x, lane = tid & 63, n = lane & 15, q = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    // workgroups of the same weights next to each other
    const int tile = blockIdx.x, part = blockIdx.y, w0 = part * g.nw, nw = min(g.nw, g.nwin - w0);
    const long r0 = (long)blockIdx.z * g.rows;
    const int rows = (int)min((long)g.rows, a.w.N - r0), tiles = (rows + 15) / 16;
    const bool half = a.w.scale_type == KQ_TYPE_F16, zeros = a.w.zeros != nullptr;
    const int s0 = tile * g.bt, ns = min(g.bt, g.B - s0);          // streams of this tile

    // x: g.xwaves waves to a stream, a lane 8 values a step.  (What lies in LDS
    // for streams that are not there only reaches sums that are not theirs.)
    constexpr int XL = P == 1 ? 1 : 2;
    const int s = min(wave * g.xmagic >> 16, ns - 1), xstep = g.xwaves * 64;   // (waves left over repeat the last's)
    const int np = (nw + 1) >> 1, per = np * 32, e0 = w0 * 16;     // (pairs of windows)
    const int elast = min(a.nblk * 4, e0 + nw * 16) - 1;
    int e = (wave * g.xmagic >> 16 == s ? (wave - s * g.xwaves) * 64 : 0) + lane;
    const long st = s0 + s;
    struct X { uint4 v[XL]; float s; };
    auto get = [&](int e) {
        X r;
        e = min(e0 + e, elast - 3 + (e & 3));
        if constexpr (P == 1) {
            const uint2 v = *reinterpret_cast<const uint2*>(a.xq + st * a.w.K + 8L * e);
            r.v[0] = make_uint4(v.x, v.y, 0, 0);
            r.s = a.xs[st * a.nblk + (e >> 2)];
        } else {
            const uint4* src = reinterpret_cast<const uint4*>(a.x + st * a.w.K + 8L * e);
            r.v[0] = src[0];
            r.v[1] = src[1];
            r.s = 0.0f;
        }
        return r;
    };
    auto put = [&](int e, X r) {
        const int b = e >> 2, kq = e & 3;
        const bool on = e0 + e <= elast, in = e < per;
#pragma unroll
        for (int k = 0; k < XL; k++) r.v[k] = on ? r.v[k] : make_uint4(0, 0, 0, 0);
        uint2 d[P];
        float scale;
        if constexpr (P == 1) {
            const uint32_t x = r.v[0].x, y = r.v[0].y;
            d[0] = make_uint2(perm(y, x, 0x06040200), perm(y, x, 0x07050301));
            scale = on ? r.s : 0.0f;
        } else {
            const X8 v = split_x(r.v[0], r.v[XL - 1]);
#pragma unroll
            for (int p = 0; p < P; p++) d[p] = make_uint2(v.even[p], v.odd[p]);
            scale = v.scale;
        }
        uint8_t* const w = smem + (size_t)(b >> 2) * WB;
        const int at = mm_place((b >> 1) & 1, kq) * E + s * P;
        if (in) {
#pragma unroll
            for (int p = 0; p < P; p++) reinterpret_cast<uint2*>(w)[(at + p) * 2 + (b & 1)] = d[p];
        }
        if (in && kq == 0) reinterpret_cast<float*>(w + XB)[((b & 3) * 4 + (s & 3)) * G + (s >> 2)] = scale;
    };
    // on its way before the weights, as loads return in order
    X x0 = get(e), x1 = get(e + xstep);
    __builtin_amdgcn_sched_barrier(0);

    const long rowb = 16L * a.nblk, rowsb = (long)a.ngrp * RawScale<MODE>::SB;
    const auto qp = plane(a.w.q, r0 * rowb, (r0 + rows) * rowb);
    const auto sp = plane(a.w.scales, r0 * rowsb, (r0 + rows) * rowsb);
    const auto zp = plane(zeros ? a.w.zeros : a.w.scales, zeros ? r0 * a.ngrp : 0,
                          zeros ? (r0 + rows) * a.ngrp : 0);

    // this wave's share: [i0, i1) of tiles x pairs of windows, those fastest
    const int items = tiles * np, ipw = (items + MM_W - 1) / MM_W;
    const int i0 = min(wave * ipw, items), i1 = min(i0 + ipw, items);
    constexpr int NS = ONE ? 1 : 2;
    struct Raw { uint4 q[2]; RawScale<MODE> s[NS]; };
    int li = i0, lt = i0 / np, lp = i0 - lt * np;         // the next to load
    const int ldr = lane >> 2, lb = lane & 3;             // row and block of a lane's load
    const uint32_t vq = (uint32_t)ldr * (uint32_t)rowb + 16u * lb;
    const int vs = ldr * a.ngrp;
    auto load = [&](Raw& t) {
        const uint32_t off = li < i1 ? 0 : FAR;
        const uint32_t at = (uint32_t)lt * 16u * (uint32_t)rowb + 64u * (uint32_t)(w0 + 2 * lp);
        const int es = lt * 16 * a.ngrp;
#pragma unroll
        for (int j = 0; j < 2; j++) {
            const uint32_t o = j && 2 * lp + 1 == nw ? FAR : off;     // (a pair's second may be missing)
            const u32x4 v = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(
                qp, (int)(vq + (o | (at + 64u * j))), 0, 0));
            t.q[j] = make_uint4(v.x, v.y, v.z, v.w);
        }
        // scales: the windows' by the first two lanes of their row, or the blocks'
#pragma unroll
        for (int j = 0; j < NS; j++) {
            const int blk = min(4 * (w0 + 2 * lp + j) + (ONE ? 4 * lb : lb), a.nblk - 1);
            t.s[j].load(sp, zp, ONE && lb > 1 ? (int)(FAR / 4) : (int)((off / 4) | (uint32_t)(vs + es + group_of(a, blk))));
        }
        li++;
        if (++lp == np) { lp = 0; lt++; }
    };
    Raw cur;
    load(cur);

    __builtin_amdgcn_sched_barrier(0);
    do {                                                  // (once whatever the length, lest the loads be moved here)
        put(e, x0);
        x0 = get(e + 2 * xstep);
        put(e + xstep, x1);
        x1 = get(e + 3 * xstep);
        e += 2 * xstep;
    } while (e < per);
    lds_barrier();
    uint8_t* const own = smem + (size_t)(2 * np) * WB + (size_t)wave * mm_wave(G);
    uint8_t* const stage = own + 4 * mm_slot(G);
    // (a row's four pieces change places every four rows: no bank conflicts either way)
    const int put_at = ldr * 64 + 16 * (lb ^ ((ldr >> 2) & 3)), take_at = n * 64 + 4 * q + 16 * ((n >> 2) & 3);

    float* const dst = g.ks > 1 ? g.part + (long)part * g.B * a.w.N : a.y;
    auto out = [&](int s, int r, float v) {               // stream s of the tile, row r of the workgroup
        if (r >= rows || s >= ns) return;
        const long o = (long)(s0 + s) * a.w.N + r0 + r;
        dst[o] = ADD ? a.add[o] + v : v;
    };

    // this lane's entry of an operand: row n = 4 qs + i
    const int qs = n >> 2, ni = n & 3;
    const int entry = P == 1 ? qs + 4 * min(ni, G - 1) : qs * P + min(ni, P - 1);
    const int xoff = (mm_place(0, q) * E + entry) * 16, moff = XB + q * G * 4;

    float acc[G];
#pragma unroll
    for (int k = 0; k < G; k++) acc[k] = 0.0f;
    int t = i0 / np, w = i0 - t * np, from = w;           // `from`: the tile's first pair here
    float* const sl = reinterpret_cast<float*>(stage + 16 * 64);
    for (int i = i0; i < i1; i++) {
        uint32_t d[2][4];
        float sc[2][4];
        uint32_t zb[2][4];                             // 128 - z in every byte
#pragma unroll
        for (int j = 0; j < 2; j++) {
            // A wave's LDS accesses are in order; the fences keep the compiler's order of what
            // its lanes write and others of them read, both ways.
            *reinterpret_cast<uint4*>(stage + put_at) = cur.q[j];
            if (j < NS) {
                const RawScale<MODE>& r = cur.s[j];
                if (MODE == M_16) sl[lane] = r.scale(half) * (P == 1 ? 0.0625f : 1.0f);
                else reinterpret_cast<uint2*>(sl)[lane] =
                    make_uint2(__float_as_uint(r.scale(half)), 0x80808080u - 0x01010101u * (uint32_t)r.zero(zeros));
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
            for (int b = 0; b < 4; b++) d[j][b] = *reinterpret_cast<const uint32_t*>(stage + (take_at ^ (16 * b)));
#pragma unroll
            for (int b = 0; b < (ONE ? 1 : 4); b++) {
                const int at = 4 * n + (ONE ? j : b);
                if (MODE == M_16) {
                    sc[j][b] = sl[at];
                } else {
                    const uint2 v = reinterpret_cast<const uint2*>(sl)[at];
                    sc[j][b] = __uint_as_float(v.x);
                    zb[j][b] = v.y;
                }
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        }
        load(cur);                                     // the next pair's, while this one's are used
#pragma unroll
        for (int j = 0; j < 2; j++) {
            const uint8_t* const xb = smem + (2 * w + j) * WB;
            const float* const m = reinterpret_cast<const float*>(xb + moff);
#pragma unroll
            for (int b2 = 0; b2 < 2; b2++) {
                constexpr int NX = P == 1 ? 1 : G;
                uint4 x[NX];
#pragma unroll
                for (int c = 0; c < NX; c++)
                    x[c] = *reinterpret_cast<const uint4*>(xb + xoff + (mm_place(b2, 0) * E + 4 * P * c) * 16);
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const int b = 2 * b2 + h;
                    const uint32_t db = d[j][b];
                    uint32_t lo, hi;
                    if (MODE == M_16) {
                        lo = ((db << 4) & 0xf0f0f0f0u) ^ 0x80808080u;
                        hi = (db & 0xf0f0f0f0u) ^ 0x80808080u;
                    } else {
                        const uint32_t z = zb[j][ONE ? 0 : b];
                        lo = ((db & 0x0f0f0f0fu) + z) ^ 0x80808080u;
                        hi = (((db >> 4) & 0x0f0f0f0fu) + z) ^ 0x80808080u;
                    }
                    const long wv = (long)(((uint64_t)hi << 32) | lo);
                    int dot[G];
#pragma unroll
                    for (int c = 0; c < NX; c++) {
                        const uint2 xv = h ? make_uint2(x[c].z, x[c].w) : make_uint2(x[c].x, x[c].y);
                        const i32x4 D = __builtin_amdgcn_mfma_i32_16x16x32_i8(
                            __builtin_bit_cast(long, xv), wv, i32x4{0, 0, 0, 0}, 0, 0, 0);
                        if constexpr (P == 1) {
#pragma unroll
                            for (int e = 0; e < G; e++) dot[e] = D[e];
                        } else {
                            int top = D[2] * 256 + D[1];
                            asm("" : "+v"(top));       // (else two shifts and a sum of three)
                            dot[c] = MODE == M_16 ? top * 16 + (D[0] >> 4) : top * 256 + D[0];
                        }
                    }
#pragma unroll
                    for (int c = 0; c < G; c++) {
                        const float xs = m[4 * G * b + c];
                        acc[c] = fmaf(sc[j][ONE ? 0 : b] * (float)dot[c], xs, acc[c]);
                    }
                }
            }
        }
        w++;
        if (w == np || i + 1 == i1) {                  // the tile's end, or this wave's
            if (from == 0 && w == np) {
#pragma unroll
                for (int c = 0; c < G; c++) out(4 * c + q, t * 16 + n, acc[c]);
            } else {
                // the first slot for what began with this wave's first pair
                float* o = reinterpret_cast<float*>(t * np + from == i0 ? own : stage) + n * (4 * G + 1) + q;
#pragma unroll
                for (int c = 0; c < G; c++) o[4 * c] = acc[c];
            }
#pragma unroll
            for (int c = 0; c < G; c++) acc[c] = 0.0f;
            w = from = 0;
            t++;
        }
    }
    __syncthreads();
    // shared tiles: their waves' sums in order
    for (int k = tid / (64 * G); k < tiles; k += T / (64 * G)) {
        const int wa = k * np / ipw, wb = (k * np + np - 1) / ipw;
        if (wa == wb) continue;
        const int r = tid & 15, s = (tid >> 4) % (4 * G);
        const float* v = reinterpret_cast<const float*>(smem + (size_t)(2 * np) * WB) + r * (4 * G + 1) + s;
        constexpr int WF = mm_wave(G) / 4;
        float sum = v[wa * WF + (k * np != wa * ipw ? mm_slot(G) : 0)];
        for (int x = wa + 1; x <= wb; x++) sum = sum + v[x * WF];
        out(s, k * 16 + r, sum);
    }
}

// the parts of rows that were cut, in their order (a launch of 2^32 lanes or more is
// cut to their number modulo that without an error, so the lanes step over the rest)
constexpr long JOIN_WGS = 1L << 22;
__global__ __launch_bounds__(256) void kq_w4_join_kernel(const float* part, const float* add, float* y,
                                                         long n, int ks) {
    for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long)gridDim.x * 256) {
        float sum = part[i];
        for (int k = 1; k < ks; k++) sum = sum + part[k * n + i];
        y[i] = add ? add[i] + sum : sum;
    }
}

// ------------------------------------------------------------- the plan

constexpr int WALK_MAX_BLK = 1024;
constexpr int walk_max_b(int P) { return P == 1 ? 4 : 3; }     // (more spill registers)
int g_lds_max = 65536;

// a matrix of which a CU's share is one step of 512 lanes
bool small_matrix(const W4Arg& a, int n_cu) { return ((long)a.w.N + n_cu - 1) / n_cu * a.nblk <= 512; }

// Rows of a step and of a workgroup, steps of a pass, LDS bytes (-1: not
// taken).  Two workgroups a CU, of as many waves as the registers allow,
// where the row is short enough; one where the matrix is a step's work of
// one (1024 x 1024: 3.1 us against 3.5, 17408 x 5120 11.6 against 11.5).
long walk_plan(W4Arg& a, int P, int NB, int n_cu) {
    const int nblk = a.nblk, waves = 4 * walk_waves(P, NB), D = WALK_D;
    const long N = a.w.N, rowb = 16L * nblk;
    const int per_cu = nblk <= 32 * waves && !small_matrix(a, n_cu) ? 2 : 1, lanes = 64 * waves / per_cu;
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

struct MmPlan { int G; long lds, runs, part; };

void mm_plan(MmArg& g, int P, int n_cu, MmPlan* p) {
    const W4Arg& a = g.a;
    g.ntile = (g.B + 15) / 16;
    g.bt = (g.B + g.ntile - 1) / g.ntile;
    p->G = (g.bt + 3) / 4;
    if (p->G == 3) p->G = 4;
    g.nwin = (a.nblk + 3) / 4;
    const long own = (long)MM_W * mm_wave(p->G), wb = mm_window(P, p->G);
    const int most_w = (int)((g_lds_max - own) / wb) & ~1;                  // windows that LDS takes, in pairs
    // as few parts as x needs.  Eight streams of binary32 in one part / in two, us: 11008
    // rows of 4096 12.5 / 13.3, of 5120 15.1 / 15.6; 65536 rows of 5120 44.9 / 48.6, 17408
    // 19.6 / 19.2, 5120 12.7 / 12.0 (what two gain where a CU has few rows, x's way to LDS,
    // is less than the join's launch costs elsewhere); int8 rows in one / four, 17408 x
    // 5120, four streams 13.4 / 15.6, sixteen 18.0 / 19.3
    g.ks = (g.nwin + most_w - 1) / most_w;
    g.nw = (g.nwin + g.ks - 1) / g.ks;
    g.ks = (g.nwin + g.nw - 1) / g.nw;
    long runs = (long)n_cu / ((long)g.ks * g.ntile);                  // one workgroup a CU
    if (runs < 1) runs = 1;
    long rows = (a.w.N + runs - 1) / runs;
    const long most = (1L << 30) / (16L * a.nblk) - 16;               // 32-bit offsets
    if (rows > most) rows = most;
    g.rows = (int)rows;
    p->runs = (a.w.N + rows - 1) / rows;
    g.xwaves = MM_W / g.bt;
    g.xmagic = 65536 / g.xwaves + 1;
    p->lds = (g.nw + 1) / 2 * 2 * wb + own;
    p->part = g.ks > 1 ? ((long)g.ks * g.B * a.w.N * 4 + 255) & ~255L : 0;
}

template <int P, int G, int MODE>
int launch_mm_m(const MmArg& g, const MmPlan& p, hipStream_t st) {
    if (p.runs > 65535 || g.ks > 65535) return (int)hipErrorInvalidValue;
    const dim3 grid((unsigned)g.ntile, (unsigned)g.ks, (unsigned)p.runs), wg(64 * MM_W);
    const bool one = g.a.w.group % 128 == 0, add = g.a.add && g.ks == 1;
    auto* const k = one ? (add ? kq_w4_mm_kernel<P, G, MODE, true, true> : kq_w4_mm_kernel<P, G, MODE, true, false>)
                        : (add ? kq_w4_mm_kernel<P, G, MODE, false, true> : kq_w4_mm_kernel<P, G, MODE, false, false>);
    hipLaunchKernelGGL(k, grid, wg, (size_t)p.lds, st, g);
    return (int)hipGetLastError();
}

template <int P, int G>
int launch_mm_g(const MmArg& g, const MmPlan& p, hipStream_t st) {
    if (g.a.w.scale_type == KQ_TYPE_F32) return launch_mm_m<P, G, M_32Z>(g, p, st);
    return g.a.w.zeros ? launch_mm_m<P, G, M_16Z>(g, p, st) : launch_mm_m<P, G, M_16>(g, p, st);
}

template <int P>
int launch_mm(MmArg& g, const MmPlan& p, void* work, hipStream_t st) {
    g.part = static_cast<float*>(work);
    const int e = p.G == 1 ? launch_mm_g<P, 1>(g, p, st) : p.G == 2 ? launch_mm_g<P, 2>(g, p, st)
                                                                    : launch_mm_g<P, 4>(g, p, st);
    if (e || g.ks == 1) return e;
    const long n = (long)g.B * g.a.w.N;
    const long wgs = (n + 255) / 256;
    hipLaunchKernelGGL(kq_w4_join_kernel, dim3((unsigned)(wgs < JOIN_WGS ? wgs : JOIN_WGS)), dim3(256), 0, st,
                       g.part, g.a.add, g.a.y, n, g.ks);
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

// LDS bytes of the walk kernel where it takes the call, else -1.  It is ahead of
// the matrix cores
// - with one stream (17408 x 5120 11.3 us against 13.9, int8 rows 11.1 / 12.8) and
//   with two of int8 rows (12.0 / 12.9; 5120 x 17408 12.7 / 14.4);
// - with three of int8 rows, where a CU has few rows for x, whose way to LDS is
//   what the other kernel waits for (5120 x 17408 14.4 / 15.2, 5120 x 9216 9.9 / 10.5,
//   1024 x 5120 4.8 / 5.8; but 5120 x 5120 7.8 / 7.5, 17408 x 17408 39.5 / 37.4);
// - with as many as it takes, where the matrix is one step of its workgroups and a
//   launch's latency is what counts (1024 x 1024: four of int8 rows 4.0 / 4.5, three of
//   binary32 4.7 / 4.9);
// and behind with more (17408 x 5120: two of binary32 16.4 / 14.2, 5120 x 17408 20.6 /
// 16.1; four of int8 rows 17.3 / 13.4).
long walk_takes(W4Arg& a, int P, int B, int n_cu) {
    const long rows = ((long)a.w.N + n_cu - 1) / n_cu;
    const bool few = B <= (P == 1 ? 2 : 1) || (P == 1 && B == 3 && a.nblk > 8 * rows) ||
                     (B <= walk_max_b(P) && small_matrix(a, n_cu));
    return few && a.nblk <= WALK_MAX_BLK ? walk_plan(a, P, B, n_cu) : -1;
}

template <int P, int G, int MODE>
int raise_mm_m(int bytes) {
    const void* k[4] = {(const void*)kq_w4_mm_kernel<P, G, MODE, true, true>,
                        (const void*)kq_w4_mm_kernel<P, G, MODE, true, false>,
                        (const void*)kq_w4_mm_kernel<P, G, MODE, false, true>,
                        (const void*)kq_w4_mm_kernel<P, G, MODE, false, false>};
    for (int i = 0; i < 4; i++) {
        const int e = (int)hipFuncSetAttribute(k[i], hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
        if (e) return e;
    }
    return 0;
}
template <int P, int G>
int raise_mm(int bytes) {
    const int e = raise_mm_m<P, G, M_16>(bytes), f = raise_mm_m<P, G, M_16Z>(bytes), g = raise_mm_m<P, G, M_32Z>(bytes);
    return e ? e : f ? f : g;
}

}  // namespace

extern "C" {

int kqk_w4_set_max_lds(int bytes) {
    g_lds_max = bytes;
    const int e[13] = {raise_lds<1, 1>(bytes), raise_lds<1, 2>(bytes), raise_lds<1, 3>(bytes),
                      raise_lds<1, 4>(bytes), raise_lds<3, 1>(bytes), raise_lds<3, 2>(bytes),
                      raise_lds<3, 3>(bytes), raise_mm<1, 1>(bytes), raise_mm<1, 2>(bytes),
                       raise_mm<1, 4>(bytes), raise_mm<3, 1>(bytes), raise_mm<3, 2>(bytes), raise_mm<3, 4>(bytes)};
    for (int i = 0; i < 13; i++)
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
    return p.part;
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
    return xq ? launch_mm<1>(g, p, work, st) : launch_mm<3>(g, p, work, st);
}

}
