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
// and a token changes where one of them moves past u.
//
// Launches: the rows' maxima and sums of exponentials per chunk of CH tokens
// (logits and greedy form); the weights' sums per chunk of the row drawn
// from; the token.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "kq_launch.h"

#pragma clang fp contract(off)

namespace {

constexpr int CH = 4096, TH = 256, PER = CH / TH;

struct VfArg {
    kq_spec_verify v;
    int nch;                // chunks of a row
    float* pmax;            // [rows][nch]
    double* psum;           // [rows][nch]
    int* parg;              // [rows][nch]
    double* wsum;           // [S][2][nch]: of max(p - q, 0); of p
};

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

// a chunk's maximum, its first place, and the sum of exp((l - max) inv_temp)
__global__ __launch_bounds__(TH) void kq_vf_stats_kernel(VfArg a) {
    __shared__ float sm[TH / 64];
    __shared__ int si[TH / 64];
    __shared__ double sd[TH / 64];
    const int T = a.v.T, row = blockIdx.y, nt = a.v.S * (T + 1), tid = threadIdx.x;
    const bool isd = row >= nt;
    const int s = isd ? (row - nt) / T : row / (T + 1), i = isd ? (row - nt) % T : row % (T + 1);
    if (isd ? i >= drafted(a, s) : i > drafted(a, s)) return;
    const float* l = isd ? draft_row(a, s, i) : target_row(a, s, i);
    const int lo = blockIdx.x * CH, hi = min(a.v.V - lo, CH) + lo;
    float m = -INFINITY;
    int at = 0x7fffffff;
    for (int k = lo + tid; k < hi; k += TH)
        if (l[k] > m) { m = l[k]; at = k; }
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const float om = __shfl_xor(m, off);
        const int oa = __shfl_xor(at, off);
        if (om > m || (om == m && oa < at)) { m = om; at = oa; }
    }
    if ((tid & 63) == 0) { sm[tid >> 6] = m; si[tid >> 6] = at; }
    __syncthreads();
    m = sm[0]; at = si[0];
    for (int k = 1; k < TH / 64; k++)
        if (sm[k] > m || (sm[k] == m && si[k] < at)) { m = sm[k]; at = si[k]; }
    const long o = (long)row * a.nch + blockIdx.x;
    if (tid == 0) { a.pmax[o] = m; a.parg[o] = at; }
    if (a.v.flags & KQ_VERIFY_GREEDY) return;
    double z = 0.0;
    for (int k = lo + tid; k < hi; k += TH) {
        const double e = exp(((double)l[k] - (double)m) * (double)a.v.inv_temp);
        if (e > 0.0) z = z + e;                     // a NaN weighs nothing
    }
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) z = z + __shfl_xor(z, off);
    if ((tid & 63) == 0) sd[tid >> 6] = z;
    __syncthreads();
    if (tid == 0) a.psum[o] = (sd[0] + sd[1]) + (sd[2] + sd[3]);
}

// one wave: a row's maximum and sum from its chunks
__device__ __forceinline__ void row_stats(const VfArg& a, int row, float* m, double* z) {
    const int lane = threadIdx.x & 63;
    const long o = (long)row * a.nch;
    float mm = -INFINITY;
    for (int c = lane; c < a.nch; c += 64) mm = fmaxf(mm, a.pmax[o + c]);
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) mm = fmaxf(mm, __shfl_xor(mm, off));
    double t = 0.0;
    for (int c = lane; c < a.nch; c += 64) {
        const double e = exp(((double)a.pmax[o + c] - (double)mm) * (double)a.v.inv_temp);
        if (e > 0.0) t = t + e * a.psum[o + c];
    }
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) t = t + __shfl_xor(t, off);
    *m = mm;
    *z = t;
}

// The weight of token k at the row drawn from, and its p.
struct Drawn {
    const float* p;
    const float* q;         // NULL: one-hot, or nothing refused
    int hot;                // one-hot draft's token, or -1
    bool logits;
    float pm, qm;
    double pz, qz, it;      // 1 / sums; inv_temp
    __device__ __forceinline__ void at(int k, double* r, double* w) const {
        double pv, qv = 0.0;
        if (logits) {
            pv = exp(((double)p[k] - (double)pm) * it) * pz;
            if (q) qv = exp(((double)q[k] - (double)qm) * it) * qz;
        } else {
            pv = (double)p[k];
            if (q) qv = (double)q[k];
        }
        pv = pv > 0.0 ? pv : 0.0;
        const double d = pv - (qv > 0.0 ? qv : 0.0);
        *w = pv;
        *r = k == hot || !(d > 0.0) ? 0.0 : d;
    }
};

// Every thread of the workgroup: tokens accepted, and what is drawn from.
__device__ __forceinline__ Drawn decide(const VfArg& a, int s, int* nacc) {
    __shared__ float mx[2 * KQ_VERIFY_MAX_DRAFT + 2];
    __shared__ double zs[2 * KQ_VERIFY_MAX_DRAFT + 2];
    __shared__ int sn;
    const int T = a.v.T, nd = drafted(a, s), tid = threadIdx.x;
    const bool lg = a.v.flags & KQ_VERIFY_LOGITS, dr = a.v.draft != nullptr;
    const double it = a.v.inv_temp;
    if (lg) {
        for (int j = tid >> 6; j < 2 * T + 1; j += TH / 64) {
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
        bool no = tid >= nd;
        if (tid < nd) {
            const int t = a.v.tokens[s * T + tid];
            if (t < 0 || t >= a.v.V) {
                no = true;
            } else {
                double p = target_row(a, s, tid)[t], q = dr ? draft_row(a, s, tid)[t] : 1.0;
                if (lg) {
                    p = exp((p - (double)mx[tid]) * it) * zs[tid];
                    if (dr) q = exp((q - (double)mx[T + 1 + tid]) * it) * zs[T + 1 + tid];
                }
                no = !((double)a.v.u[s * (T + 1) + tid] * q < p);
            }
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
    d.it = it;
    d.pm = lg ? mx[n] : 0.0f;
    d.pz = lg ? zs[n] : 0.0;
    d.qm = lg && d.q ? mx[T + 1 + n] : 0.0f;
    d.qz = lg && d.q ? zs[T + 1 + n] : 0.0;
    *nacc = n;
    return d;
}

__global__ __launch_bounds__(TH) void kq_vf_weights_kernel(VfArg a) {
    __shared__ double sd[2][TH / 64];
    const int s = blockIdx.y, tid = threadIdx.x;
    int n;
    const Drawn d = decide(a, s, &n);
    const int lo = blockIdx.x * CH, hi = min(a.v.V - lo, CH) + lo;
    double r = 0.0, w = 0.0;
    for (int k = lo + tid; k < hi; k += TH) {
        double rk, wk;
        d.at(k, &rk, &wk);
        r = r + rk;
        w = w + wk;
    }
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        r = r + __shfl_xor(r, off);
        w = w + __shfl_xor(w, off);
    }
    if ((tid & 63) == 0) { sd[0][tid >> 6] = r; sd[1][tid >> 6] = w; }
    __syncthreads();
    if (tid < 2)
        a.wsum[(2 * (long)s + tid) * a.nch + blockIdx.x] =
            (sd[tid][0] + sd[tid][1]) + (sd[tid][2] + sd[tid][3]);
}

// inclusive running sum over a wave's lanes
__device__ __forceinline__ double wave_scan(double v) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const double o = __shfl_up(v, off);
        if (lane >= off) v = v + o;
    }
    return v;
}

// One workgroup per sequence: the chunk in which the running sum passes u
// times the total, then the token in it.
__global__ __launch_bounds__(TH) void kq_vf_draw_kernel(VfArg a) {
    __shared__ double incl[TH];
    __shared__ double sbase, starget;
    __shared__ int schunk, sbest, slast;
    const int s = blockIdx.x, T = a.v.T, tid = threadIdx.x, lane = tid & 63;
    int n;
    const Drawn d = decide(a, s, &n);
    const double* ws = a.wsum + 2 * (long)s * a.nch;
    double tot = 0.0;
    for (int c0 = 0; c0 < a.nch; c0 += 64)
        tot = tot + __shfl(wave_scan(c0 + lane < a.nch ? ws[c0 + lane] : 0.0), 63);
    const bool left = tot > 0.0;             // else p itself: p and q are equal here
    if (!left) ws += a.nch;
    if (tid < 64) {
        double base = 0.0, cbase = 0.0, total = 0.0;
        for (int c0 = 0; c0 < a.nch; c0 += 64)
            total = total + __shfl(wave_scan(c0 + lane < a.nch ? ws[c0 + lane] : 0.0), 63);
        const double target = (double)a.v.u[s * (T + 1) + T] * total;
        int chunk = -1;
        for (int c0 = 0; c0 < a.nch; c0 += 64) {
            const double v = c0 + lane < a.nch ? ws[c0 + lane] : 0.0;
            const double in = base + wave_scan(v);
            double ex = __shfl_up(in, 1);
            if (lane == 0) ex = base;
            const unsigned long long over = __ballot(v > 0.0 && in > target);
            const unsigned long long some = __ballot(v > 0.0);
            if (over) {
                const int j = __ffsll(over) - 1;
                chunk = c0 + j;
                cbase = __shfl(ex, j);
                break;
            }
            if (some) {                      // the last one with any weight
                const int j = 63 - __clzll(some);
                chunk = c0 + j;
                cbase = __shfl(ex, j);
            }
            base = __shfl(in, 63);
        }
        if (tid == 0) {
            schunk = chunk;
            sbase = cbase;
            starget = target;
            sbest = TH;
            slast = -1;
        }
    }
    __syncthreads();
    int token = -1;
    if (schunk >= 0) {
        const int lo = schunk * CH + tid * PER, hi = min(a.v.V, lo + PER);
        double sum = 0.0, v[PER];
#pragma unroll
        for (int j = 0; j < PER; j++) {
            double rk = 0.0, wk = 0.0;
            if (lo + j < hi) d.at(lo + j, &rk, &wk);
            v[j] = left ? rk : wk;
            sum = sum + v[j];
        }
        const double ws1 = wave_scan(sum);
        if (lane == 63) incl[tid >> 6] = ws1;
        __syncthreads();
        double before = sbase;
        for (int k = 0; k < tid >> 6; k++) before = before + incl[k];
        const double in = before + ws1;
        __syncthreads();
        incl[tid] = in;
        if (sum > 0.0 && in > starget) atomicMin(&sbest, tid);
        if (sum > 0.0) atomicMax(&slast, tid);
        __syncthreads();
        const int who = sbest < TH ? sbest : slast;
        if (tid == who) {
            double cum = tid ? incl[tid - 1] : sbase;
#pragma unroll
            for (int j = 0; j < PER; j++)
                if (v[j] > 0.0 && !(cum > starget)) {
                    cum = cum + v[j];
                    token = lo + j;
                }
            a.v.out[s * (T + 1) + n] = token;
        }
    } else if (tid == 0) {
        a.v.out[s * (T + 1) + n] = -1;
    }
    if (tid < n) a.v.out[s * (T + 1) + tid] = a.v.tokens[s * T + tid];
    if (tid > n && tid <= T) a.v.out[s * (T + 1) + tid] = -1;
    if (tid == 0) a.v.n_accept[s] = n;
}

// The greedy form: a token is accepted iff it is its row's first maximum.
__global__ __launch_bounds__(64) void kq_vf_greedy_kernel(VfArg a) {
    const int s = blockIdx.x, T = a.v.T, lane = threadIdx.x, nd = drafted(a, s);
    int n = 0, best = -1;
    for (; n <= nd; n++) {
        const long o = (long)trow(a, s, n) * a.nch;
        float m = -INFINITY;
        int at = 0x7fffffff;
        for (int c = lane; c < a.nch; c += 64)
            if (a.pmax[o + c] > m) { m = a.pmax[o + c]; at = a.parg[o + c]; }
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
            const float om = __shfl_xor(m, off);
            const int oa = __shfl_xor(at, off);
            if (om > m || (om == m && oa < at)) { m = om; at = oa; }
        }
        best = at == 0x7fffffff ? -1 : at;
        if (n == nd || best < 0 || a.v.tokens[s * T + n] != best) break;
    }
    if (lane < n) a.v.out[s * (T + 1) + lane] = a.v.tokens[s * T + lane];
    if (lane >= n && lane <= T) a.v.out[s * (T + 1) + lane] = lane == n ? best : -1;
    if (lane == 0) a.v.n_accept[s] = n;
}

int64_t up256(int64_t n) { return (n + 255) & ~(int64_t)255; }

int64_t layout(const kq_spec_verify* v, VfArg* a, uint8_t* w) {
    const int64_t nch = ((int64_t)v->V + CH - 1) / CH;
    const bool stats = v->flags & (KQ_VERIFY_LOGITS | KQ_VERIFY_GREEDY);
    const int64_t rows = stats ? (int64_t)v->S * (v->T + 1) + (v->draft ? (int64_t)v->S * v->T : 0) : 0;
    int64_t o[5] = {0};
    o[1] = o[0] + up256(rows * nch * 8);              // psum
    o[2] = o[1] + up256(rows * nch * 4);              // pmax
    o[3] = o[2] + up256(rows * nch * 4);              // parg
    o[4] = o[3] + up256(2 * (int64_t)v->S * nch * 8); // wsum
    if (a) {
        a->v = *v;
        a->nch = (int)nch;
        a->psum = (double*)(w + o[0]);
        a->pmax = (float*)(w + o[1]);
        a->parg = (int*)(w + o[2]);
        a->wsum = (double*)(w + o[3]);
    }
    return o[4];
}

}  // namespace

extern "C" {

int64_t kqk_verify_workspace(const kq_spec_verify* v) { return layout(v, nullptr, nullptr); }

int kqk_launch_verify(const kq_spec_verify* v, void* work, hipStream_t st) {
    if (v->S < 1 || v->T < 0 || v->T > KQ_VERIFY_MAX_DRAFT || v->V < 1)
        return (int)hipErrorInvalidValue;
    VfArg a;
    layout(v, &a, static_cast<uint8_t*>(work));
    const bool greedy = v->flags & KQ_VERIFY_GREEDY;
    if (v->flags & (KQ_VERIFY_LOGITS | KQ_VERIFY_GREEDY)) {
        const int rows = v->S * (v->T + 1) + (v->draft && !greedy ? v->S * v->T : 0);
        hipLaunchKernelGGL(kq_vf_stats_kernel, dim3((unsigned)a.nch, (unsigned)rows), dim3(TH), 0, st, a);
    }
    if (greedy) {
        hipLaunchKernelGGL(kq_vf_greedy_kernel, dim3((unsigned)v->S), dim3(64), 0, st, a);
    } else {
        hipLaunchKernelGGL(kq_vf_weights_kernel, dim3((unsigned)a.nch, (unsigned)v->S), dim3(TH), 0, st, a);
        hipLaunchKernelGGL(kq_vf_draw_kernel, dim3((unsigned)v->S), dim3(TH), 0, st, a);
    }
    return (int)hipGetLastError();
}

}
