/*
 * kq_step.c -- host side of the row operators around the products (C11): the
 * RMS norm, the products with 4-bit weights and group scales, and the
 * verification of drafted tokens.  Each entry checks its arguments before
 * anything is enqueued (a kernel reads and writes only what the checked
 * descriptor covers), allocates nothing and launches on the caller's stream.
 */
#include <math.h>
#include <string.h>

#include "kq_launch.h"

/* kq_linear.c */
int kq_fail(const char* fmt, ...);
int kq_device(int* n_cu);

static int misaligned(const void* p, unsigned a) { return ((uintptr_t)p & (a - 1)) != 0; }

/* ---------------------------------------------------------------- norm */

#define NORM_MAX_K (1 << 28)

int kq_rmsnorm_dev(const kq_rmsnorm* in, kq_stream stream) {
    static const char who[] = "kq_rmsnorm_dev";
    int n_cu;
    if (!in) return kq_fail("%s: NULL descriptor", who);
    kq_rmsnorm a = *in;
    if (a.B < 1 || a.K < 1 || a.K > NORM_MAX_K) return kq_fail("%s: B=%d K=%d", who, a.B, a.K);
    if (!(a.eps >= 0.0f) || isinf(a.eps)) return kq_fail("%s: eps %g", who, (double)a.eps);
    if (a.group != 0 && a.group != 16 && a.group != 32)
        return kq_fail("%s: group %d (0, 16 or 32)", who, a.group);
    if (a.group && a.K % a.group) return kq_fail("%s: K=%d, group %d", who, a.K, a.group);
    if (!a.x) return kq_fail("%s: NULL x", who);
    if (a.group ? !a.xq || !a.xscale : !a.y || a.xq || a.xscale || a.xsum)
        return kq_fail("%s: group %d takes %s", who, a.group,
                       a.group ? "xq and xscale" : "y, and no int8 rows");
    if (misaligned(a.x, 4) || misaligned(a.resid, 4) || misaligned(a.weight, 4) ||
        misaligned(a.sum, 4) || misaligned(a.y, 4) || misaligned(a.xscale, 4) ||
        misaligned(a.xsum, 4) || misaligned(a.xq, 4))
        return kq_fail("%s: operands must be 4-byte aligned", who);
    int64_t* const st[4] = {&a.x_stride, &a.resid_stride, &a.sum_stride, &a.y_stride};
    for (int i = 0; i < 4; i++) {
        if (*st[i] == 0) *st[i] = a.K;
        if (*st[i] < a.K) return kq_fail("%s: row stride %lld, K=%d", who, (long long)*st[i], a.K);
    }
    if (a.y && a.y == a.sum) return kq_fail("%s: y and sum are one buffer", who);
    if ((a.sum && a.sum == a.x && a.sum_stride != a.x_stride) ||
        (a.sum && a.sum == a.resid && a.sum_stride != a.resid_stride) ||
        (a.y && a.y == a.x && a.y_stride != a.x_stride) ||
        (a.y && a.y == a.resid && a.y_stride != a.resid_stride))
        return kq_fail("%s: in place, but with another row stride", who);
    if (kq_device(&n_cu)) return -1;
    const int e = kqk_launch_rmsnorm(&a, (hipStream_t)stream);
    if (e) return kq_fail("rmsnorm launch: %s", hipGetErrorString((hipError_t)e));
    return 0;
}

/* ------------------------------------------- 4-bit weights, group scales */

#define W4_MAX_ROWS (1 << 28)
#define W4_MAX_BATCH 65535
#define W4_MAX_K (1 << 20)

static int w4_check(const kq_w4* w, int B, const char* who) {
    if (!w) return kq_fail("%s: NULL descriptor", who);
    if (w->N < 1 || w->N > W4_MAX_ROWS || w->K < 32 || w->K % 32 || w->K > W4_MAX_K)
        return kq_fail("%s: N=%d K=%d (K %% 32 must be 0)", who, w->N, w->K);
    if (w->group < 32 || w->group % 32 || w->K % w->group)
        return kq_fail("%s: group %d of K=%d (a multiple of 32 that divides K)", who, w->group, w->K);
    if (w->scale_type != KQ_TYPE_F16 && w->scale_type != KQ_TYPE_BF16 && w->scale_type != KQ_TYPE_F32)
        return kq_fail("%s: scale type %d", who, w->scale_type);
    if (B < 1 || B > W4_MAX_BATCH) return kq_fail("%s: B=%d (1..%d)", who, B, W4_MAX_BATCH);
    return 0;
}

int64_t kq_w4_workspace_bytes(const kq_w4* w, int B, int q8) {
    int n_cu;
    if (w4_check(w, B, "kq_w4_workspace_bytes") || kq_device(&n_cu)) return -1;
    return kqk_w4_workspace(w, B, q8 != 0, n_cu);
}

static int w4_gemv(const char* who, const kq_w4* w, const float* x, const int8_t* xq,
                   const float* xs, const float* add, float* y, int B, void* work,
                   int64_t work_bytes, kq_stream stream) {
    int n_cu;
    if (w4_check(w, B, who)) return -1;
    if (!w->q || !w->scales || !y || !(xq ? (const void*)xs : (const void*)x))
        return kq_fail("%s: NULL pointer", who);
    if (misaligned(w->q, 16) || misaligned(x, 16) || misaligned(xq, 16))
        return kq_fail("%s: q and x must be 16-byte aligned", who);
    if (misaligned(w->scales, w->scale_type == KQ_TYPE_F32 ? 4 : 2) || misaligned(xs, 4) ||
        misaligned(add, 4) || misaligned(y, 4))
        return kq_fail("%s: scales, add and y must be aligned to their elements", who);
    if (kq_device(&n_cu)) return -1;
    const int64_t need = kqk_w4_workspace(w, B, xq != NULL, n_cu);
    if (need > 0 && (!work || misaligned(work, 256) || work_bytes < need))
        return kq_fail("%s: workspace of %lld bytes, 256-byte aligned, needed", who, (long long)need);
    const int e = kqk_launch_w4(w, x, xq, xs, add, y, B, work, n_cu, (hipStream_t)stream);
    if (e) return kq_fail("w4 launch: %s", hipGetErrorString((hipError_t)e));
    return 0;
}

int kq_w4_gemv_dev(const kq_w4* w, const float* x, const float* add, float* y, int B, void* work,
                   int64_t work_bytes, kq_stream stream) {
    return w4_gemv("kq_w4_gemv_dev", w, x, NULL, NULL, add, y, B, work, work_bytes, stream);
}

int kq_w4_gemv_q8_dev(const kq_w4* w, const int8_t* xq, const float* xscale, const float* add,
                      float* y, int B, void* work, int64_t work_bytes, kq_stream stream) {
    if (!xq) return kq_fail("kq_w4_gemv_q8_dev: NULL pointer");
    return w4_gemv("kq_w4_gemv_q8_dev", w, NULL, xq, xscale, add, y, B, work, work_bytes, stream);
}

/* --------------------------------------------------------- verification */

static int verify_check(const kq_spec_verify* v, const char* who) {
    if (!v) return kq_fail("%s: NULL descriptor", who);
    if (v->S < 1 || v->T < 0 || v->T > KQ_VERIFY_MAX_DRAFT ||
        (int64_t)v->S * (2 * v->T + 1) > KQ_VERIFY_MAX_ROWS)
        return kq_fail("%s: S=%d T=%d", who, v->S, v->T);
    if (v->V < 1 || v->V > KQ_VERIFY_MAX_VOCAB) return kq_fail("%s: V=%d", who, v->V);
    if (v->flags & ~(KQ_VERIFY_LOGITS | KQ_VERIFY_GREEDY)) return kq_fail("%s: flags %d", who, v->flags);
    return 0;
}

int64_t kq_spec_verify_workspace_bytes(const kq_spec_verify* v) {
    if (verify_check(v, "kq_spec_verify_workspace_bytes")) return -1;
    return kqk_verify_workspace(v);
}

int kq_spec_verify_dev(const kq_spec_verify* in, void* work, int64_t work_bytes, kq_stream stream) {
    static const char who[] = "kq_spec_verify_dev";
    int n_cu;
    if (verify_check(in, who)) return -1;
    kq_spec_verify v = *in;
    const int greedy = (v.flags & KQ_VERIFY_GREEDY) != 0;
    if (greedy || v.T == 0) v.draft = NULL;
    if (!v.target || !v.n_accept || !v.out || (v.T && !v.tokens) || (!greedy && !v.u))
        return kq_fail("%s: NULL pointer", who);
    if ((v.flags & KQ_VERIFY_LOGITS) && !greedy && (!(v.inv_temp > 0.0f) || isinf(v.inv_temp)))
        return kq_fail("%s: inv_temp %g", who, (double)v.inv_temp);
    if (misaligned(v.target, 4) || misaligned(v.draft, 4) || misaligned(v.tokens, 4) ||
        misaligned(v.n_draft, 4) || misaligned(v.u, 4) || misaligned(v.n_accept, 4) ||
        misaligned(v.out, 4))
        return kq_fail("%s: operands must be 4-byte aligned", who);
    if (!v.target_row) v.target_row = v.V;
    if (!v.target_seq) v.target_seq = (v.T + 1) * v.target_row;
    if (!v.draft_row) v.draft_row = v.V;
    if (!v.draft_seq) v.draft_seq = v.T * v.draft_row;
    if (v.target_row < 0 || v.target_seq < 0 || v.draft_row < 0 || v.draft_seq < 0)
        return kq_fail("%s: negative stride", who);
    if (kq_device(&n_cu)) return -1;
    const int64_t need = kqk_verify_workspace(in);
    if (!work || misaligned(work, 256) || work_bytes < need)
        return kq_fail("%s: workspace of %lld bytes, 256-byte aligned, needed", who, (long long)need);
    const int e = kqk_launch_verify(&v, work, (hipStream_t)stream);
    if (e) return kq_fail("verify launch: %s", hipGetErrorString((hipError_t)e));
    return 0;
}
