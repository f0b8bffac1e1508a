/*
 * kq_kv.c -- host side of attention over a paged cache (C11): block tables and
 * slots, rotary embedding and store, attention.  Each entry checks its arguments
 * before anything is enqueued, allocates nothing and launches on the caller's
 * stream.
 */
#include <math.h>
#include <string.h>

#include "kq_launch.h"

/* kq_linear.c */
int kq_fail(const char* fmt, ...);
int kq_device(int* n_cu);

static int misaligned(const void* p, unsigned a) { return ((uintptr_t)p & (a - 1)) != 0; }

/* --------------------------------------------------------------- checks */

static int page_check(int n_pages, int page, const char* who) {
    if (page < 1 || page > KQ_KV_MAX_PAGE || n_pages < 1 || (int64_t)n_pages * page > 0x7fffffff)
        return kq_fail("%s: %d pages of %d tokens", who, n_pages, page);
    return 0;
}

static int cache_check(kq_kv_cache* c, const char* who) {
    if (c->type != KQ_TYPE_F16 && c->type != KQ_TYPE_BF16 && c->type != KQ_TYPE_I8)
        return kq_fail("%s: cache type %d", who, c->type);
    if (page_check(c->n_pages, c->page, who)) return -1;
    if (c->n_kv < 1 || c->n_kv > KQ_ATTN_MAX_HEADS || c->D < 8 || c->D > KQ_KV_MAX_D || c->D % 8)
        return kq_fail("%s: %d heads of D=%d (a multiple of 8 up to %d)", who, c->n_kv, c->D, KQ_KV_MAX_D);
    if (!c->k || !c->v) return kq_fail("%s: NULL cache", who);
    if (misaligned(c->k, 16) || misaligned(c->v, 16))
        return kq_fail("%s: k and v of the cache must be 16-byte aligned", who);
    if (c->type == KQ_TYPE_I8) {
        if (!c->k_scale || !c->v_scale || misaligned(c->k_scale, 4) || misaligned(c->v_scale, 4))
            return kq_fail("%s: an int8 cache has scales, 4-byte aligned", who);
    } else if (c->k_scale || c->v_scale) {
        return kq_fail("%s: scales of a cache that is not int8", who);
    }
    if (!c->token_stride) c->token_stride = c->D;
    if (!c->head_stride) c->head_stride = c->token_stride * c->page;
    if (!c->page_stride) c->page_stride = c->head_stride * c->n_kv;
    if (c->token_stride < c->D || c->head_stride < c->D || c->page_stride < c->D ||
        c->token_stride > KQ_KV_MAX_TOKEN_STRIDE || (c->token_stride | c->head_stride | c->page_stride) % 8)
        return kq_fail("%s: cache strides %lld, %lld, %lld", who, (long long)c->page_stride,
                       (long long)c->head_stride, (long long)c->token_stride);
    return 0;
}

static int shape_check(const kq_attn_shape* s, const char* who) {
    if (!s) return kq_fail("%s: NULL shape", who);
    if (s->S < 1 || s->S > KQ_ATTN_MAX_SEQS || s->T < 1 || s->T > KQ_ATTN_MAX_NEW)
        return kq_fail("%s: S=%d T=%d", who, s->S, s->T);
    if (s->n_q < 1 || s->n_q > KQ_ATTN_MAX_HEADS || s->n_kv < 1 || s->n_q % s->n_kv)
        return kq_fail("%s: %d heads of queries, %d of keys", who, s->n_q, s->n_kv);
    if (s->D < 8 || s->D > KQ_KV_MAX_D || s->D % 8)
        return kq_fail("%s: D=%d (a multiple of 8 up to %d)", who, s->D, KQ_KV_MAX_D);
    if (s->window < 0 || s->window > KQ_ATTN_MAX_WINDOW) return kq_fail("%s: window %d", who, s->window);
    return 0;
}

static int sizes(const kq_attn_shape* s, int listed, const char* who, kqk_attn_sizes* z) {
    int n_cu;
    if (kq_device(&n_cu)) return -1;
    kqk_attn_plan(s, n_cu, z);
    /* a launch's lanes are counted in 32 bits */
    if ((int64_t)(listed ? z->cap : s->S) * s->n_kv * z->blocks > 1 << 22)
        return kq_fail("%s: %d sequences x %d heads x %d rows are too many for one call", who, s->S,
                       s->n_kv, s->T * (s->n_q / s->n_kv));
    return 0;
}

static int64_t list_bytes(const kqk_attn_sizes* z) {
    return 4 * (KQK_LIST_HEAD + (int64_t)z->cap * KQK_ITEM + z->counters);
}

/* ----------------------------------------------------------------- plan */

int64_t kq_kv_list_bytes(const kq_attn_shape* s) {
    kqk_attn_sizes z;
    if (shape_check(s, "kq_kv_list_bytes") || sizes(s, 1, "kq_kv_list_bytes", &z)) return -1;
    return list_bytes(&z);
}

int kq_kv_plan_dev(const kq_kv_plan* in, kq_stream stream) {
    static const char who[] = "kq_kv_plan_dev";
    kqk_attn_sizes z;
    int n_cu;
    if (!in) return kq_fail("%s: NULL descriptor", who);
    kq_kv_plan p = *in;
    if (p.S < 1 || p.S > KQ_ATTN_MAX_SEQS) return kq_fail("%s: S=%d", who, p.S);
    if (page_check(p.n_pages, p.page, who)) return -1;
    if (!p.cached) return kq_fail("%s: NULL lengths", who);
    if (p.table) {
        if (p.table_stride < 1) return kq_fail("%s: table of %d pages", who, p.table_stride);
        if (!p.free_pages || !p.n_free) return kq_fail("%s: NULL free pages", who);
    } else if (p.free_pages || p.n_free || p.held || p.held_out || p.n_free_out || p.slot || p.n_short) {
        return kq_fail("%s: pages without a table", who);
    }
    if (p.N < 0 || ((p.pos || p.slot) && p.N < 1)) return kq_fail("%s: N=%d", who, p.N);
    const void* const ints[] = {p.cached, p.n_new, p.held, p.table, p.free_pages, p.n_free, p.held_out,
                                p.n_free_out, p.start, p.lens, p.pos, p.slot, p.n_short};
    for (unsigned i = 0; i < sizeof ints / sizeof *ints; i++)
        if (misaligned(ints[i], 4)) return kq_fail("%s: operands must be 4-byte aligned", who);
    /* inputs, then outputs, which may be held and n_free where they are held_out and n_free_out */
    const void* const in_out[] = {p.cached, p.n_new, p.free_pages, p.held, p.n_free, p.held_out, p.n_free_out,
                                  p.table, p.start, p.lens, p.pos, p.slot, p.n_short};
    for (unsigned i = 0; i < sizeof in_out / sizeof *in_out; i++)
        for (unsigned j = i < 5 ? 5 : i + 1; j < sizeof in_out / sizeof *in_out; j++)
            if (in_out[i] && in_out[i] == in_out[j] && !(i == 3 && j == 5) && !(i == 4 && j == 6))
                return kq_fail("%s: an output is another operand's buffer", who);
    memset(&z, 0, sizeof z);
    if (p.list) {
        if (shape_check(&p.shape, who)) return -1;
        if (p.shape.S != p.S) return kq_fail("%s: S=%d, shape of S=%d", who, p.S, p.shape.S);
        if (sizes(&p.shape, 1, who, &z)) return -1;
        if (misaligned(p.list, 256) || p.list_bytes < list_bytes(&z))
            return kq_fail("%s: list of %lld bytes, 256-byte aligned, needed", who, (long long)list_bytes(&z));
    }
    if (kq_device(&n_cu)) return -1;
    const int e = kqk_launch_kv_plan(&p, &z, (hipStream_t)stream);
    if (e) return kq_fail("kv plan launch: %s", hipGetErrorString((hipError_t)e));
    return 0;
}

/* ---------------------------------------------------------------- store */

int kq_kv_store_dev(const kq_kv_store* in, kq_stream stream) {
    static const char who[] = "kq_kv_store_dev";
    int n_cu;
    if (!in) return kq_fail("%s: NULL descriptor", who);
    kq_kv_store a = *in;
    if (cache_check(&a.cache, who)) return -1;
    if (a.N < 1 || a.N > KQ_KV_MAX_ROWS) return kq_fail("%s: N=%d", who, a.N);
    if (!a.k || !a.v || !a.slot) return kq_fail("%s: NULL pointer", who);
    if (a.rot < 0 || a.rot % 2 || a.rot > a.cache.D) return kq_fail("%s: rot %d of D=%d", who, a.rot, a.cache.D);
    if (a.rot && (!a.pos || !a.freq)) return kq_fail("%s: NULL pos or freq", who);
    if (a.q ? !a.q_out || a.n_q < 1 || a.n_q > KQ_ATTN_MAX_HEADS : a.q_out || a.n_q)
        return kq_fail("%s: q, q_out and n_q=%d go together", who, a.n_q);
    if (misaligned(a.k, 16) || misaligned(a.v, 16) || misaligned(a.q, 16) || misaligned(a.q_out, 16))
        return kq_fail("%s: rows must be 16-byte aligned", who);
    if (misaligned(a.slot, 4) || misaligned(a.pos, 4) || misaligned(a.freq, 4) || misaligned(a.n_tokens, 4))
        return kq_fail("%s: operands must be 4-byte aligned", who);
    int64_t* const st[4] = {&a.k_stride, &a.v_stride, &a.q_stride, &a.q_out_stride};
    for (int i = 0; i < 4; i++) {
        const int64_t n = (int64_t)a.cache.D * (i < 2 ? a.cache.n_kv : a.n_q);
        if (*st[i] == 0) *st[i] = n;
        if (*st[i] < n || *st[i] % 4) return kq_fail("%s: row stride %lld", who, (long long)*st[i]);
    }
    if (a.q && a.q == a.q_out && a.q_stride != a.q_out_stride)
        return kq_fail("%s: in place, but with another row stride", who);
    if (kq_device(&n_cu)) return -1;
    const int e = kqk_launch_kv_store(&a, n_cu, (hipStream_t)stream);
    if (e) return kq_fail("kv store launch: %s", hipGetErrorString((hipError_t)e));
    return 0;
}

/* ------------------------------------------------------------ attention */

int64_t kq_paged_attn_workspace_bytes(const kq_attn_shape* s) {
    static const char who[] = "kq_paged_attn_workspace_bytes";
    kqk_attn_sizes z;
    int n_cu;
    if (shape_check(s, who) || sizes(s, 1, who, &z) || kq_device(&n_cu)) return -1;
    return kqk_attn_workspace(s, n_cu);
}

int kq_paged_attn_dev(const kq_paged_attn* in, void* work, int64_t work_bytes, kq_stream stream) {
    static const char who[] = "kq_paged_attn_dev";
    kqk_attn_sizes z;
    int n_cu;
    if (!in) return kq_fail("%s: NULL descriptor", who);
    kq_paged_attn a = *in;
    if (shape_check(&a.shape, who) || cache_check(&a.cache, who)) return -1;
    if (a.shape.n_kv != a.cache.n_kv || a.shape.D != a.cache.D)
        return kq_fail("%s: shape of %d heads of %d, cache of %d of %d", who, a.shape.n_kv, a.shape.D,
                       a.cache.n_kv, a.cache.D);
    /* (the kernel's scores are powers of two) */
    if (!isfinite((float)(a.scale * 1.4426950408889634))) return kq_fail("%s: scale %g", who, (double)a.scale);
    if (a.N < 1) return kq_fail("%s: N=%d", who, a.N);
    if (!a.q || !a.out || !a.table || !a.lens) return kq_fail("%s: NULL pointer", who);
    if (a.q == a.out) return kq_fail("%s: q and out are one buffer", who);
    if (a.table_stride < 1) return kq_fail("%s: table of %d pages", who, a.table_stride);
    if (misaligned(a.q, 16) || misaligned(a.out, 16))
        return kq_fail("%s: q and out must be 16-byte aligned", who);
    if (misaligned(a.table, 4) || misaligned(a.start, 4) || misaligned(a.lens, 4))
        return kq_fail("%s: operands must be 4-byte aligned", who);
    const int64_t n = (int64_t)a.shape.n_q * a.shape.D;
    if (!a.q_stride) a.q_stride = n;
    if (!a.out_stride) a.out_stride = n;
    if (a.q_stride < n || a.out_stride < n || (a.q_stride | a.out_stride) % 4)
        return kq_fail("%s: row strides %lld, %lld", who, (long long)a.q_stride, (long long)a.out_stride);
    if (sizes(&a.shape, a.list != NULL, who, &z) || kq_device(&n_cu)) return -1;
    if (a.list) {
        if (misaligned(a.list, 256) || a.list_bytes < list_bytes(&z))
            return kq_fail("%s: list of %lld bytes, 256-byte aligned, needed", who, (long long)list_bytes(&z));
        const int64_t need = kqk_attn_workspace(&a.shape, n_cu);
        if (need > 0 && (!work || misaligned(work, 256) || work_bytes < need))
            return kq_fail("%s: workspace of %lld bytes, 256-byte aligned, needed", who, (long long)need);
    }
    const int e = kqk_launch_attn(&a, &z, work, (hipStream_t)stream);
    if (e) return kq_fail("attention launch: %s", hipGetErrorString((hipError_t)e));
    return 0;
}
