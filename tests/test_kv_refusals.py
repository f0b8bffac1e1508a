"""Block tables, the store into the cache and attention over it refuse bad
arguments with -1 and a message before anything is enqueued (no GPU needed: each
check comes before the device is looked at, and the addresses here are never read)."""
import ctypes

import pytest

import stratum_amd as K

P = 1 << 20          # an aligned address; nothing is read from it


def refused(rc, word):
    assert rc == -1
    msg = K.lib().kq_last_error().decode()
    assert word in msg, msg


def test_null_descriptors():
    L = K.lib()
    refused(L.kq_kv_plan_dev(None, None), "NULL")
    refused(L.kq_kv_store_dev(None, None), "NULL")
    refused(L.kq_paged_attn_dev(None, None, 0, None), "NULL")
    refused(L.kq_kv_list_bytes(None), "NULL")
    refused(L.kq_paged_attn_workspace_bytes(None), "NULL")


def shape(**kw):
    a = dict(S=2, T=4, n_q=8, n_kv=2, D=64, window=0)
    a.update(kw)
    return K.attn_shape(**a)


SHAPES = [(dict(S=0), "S=0"), (dict(S=65536), "S=65536"), (dict(T=0), "T=0"), (dict(T=65), "T=65"),
          (dict(n_q=0), "0 heads"), (dict(n_kv=0), "0 of keys"), (dict(n_kv=3), "3 of keys"), (dict(n_q=2048), "2048"),
          (dict(n_kv=-2), "-2 of keys"), (dict(D=0), "D=0"), (dict(D=60), "D=60"), (dict(D=264), "D=264"),
          (dict(window=-1), "window"), (dict(window=(1 << 30) + 1), "window")]


@pytest.mark.parametrize("kw,word", SHAPES)
def test_shapes(kw, word):
    L, s = K.lib(), shape(**kw)
    refused(L.kq_kv_list_bytes(ctypes.byref(s)), word)
    refused(L.kq_paged_attn_workspace_bytes(ctypes.byref(s)), word)
    if kw.get("S", 2) in (2, 0):
        S = kw.get("S", 2) or 2
        p = K.kv_plan(S, 16, 10, P, shape=s, list_ptr=P, list_bytes=1 << 40)
        refused(L.kq_kv_plan_dev(ctypes.byref(p), None), word)
    refused(L.kq_paged_attn_dev(ctypes.byref(attn(shape=s)), P, 1 << 40, None), word)


def plan(**kw):
    at = [P * i for i in range(1, 10)]
    a = dict(S=2, page=16, n_pages=100, cached_ptr=at[0], new_ptr=at[1], table_ptr=at[2], table_stride=10, free_ptr=at[3],
             n_free_ptr=at[4], lens_ptr=at[5], start_ptr=at[6], N=8, pos_ptr=at[7], slot_ptr=at[8])
    a.update(kw)
    return K.kv_plan(**a)


@pytest.mark.parametrize("kw,word", [
    (dict(S=0), "S=0"), (dict(S=-1), "S=-1"), (dict(S=65536), "S=65536"), (dict(page=0), "0 tokens"),
    (dict(page=65537), "65537 tokens"), (dict(n_pages=0), "0 pages"), (dict(n_pages=1 << 27), "pages of"),
    (dict(cached_ptr=None), "NULL lengths"), (dict(table_stride=0), "table of 0"), (dict(free_ptr=None), "NULL free"),
    (dict(n_free_ptr=None), "NULL free"), (dict(table_ptr=None), "without a table"),
    (dict(table_ptr=None, free_ptr=None, n_free_ptr=None), "without a table"),
    (dict(table_ptr=None, free_ptr=None, n_free_ptr=None, slot_ptr=None, held_ptr=P), "without a table"),
    (dict(table_ptr=None, free_ptr=None, n_free_ptr=None, slot_ptr=None, short_ptr=P), "without a table"),
    (dict(N=0), "N=0"), (dict(N=-1), "N=-1"), (dict(cached_ptr=P + 2), "aligned"), (dict(slot_ptr=P + 1), "aligned"),
    (dict(n_free_ptr=P + 2), "aligned"), (dict(short_ptr=P + 2), "aligned"),
    (dict(list_ptr=P, list_bytes=1 << 40, shape=shape(S=3)), "shape of S=3"),
    (dict(lens_ptr=P), "another operand"), (dict(held_out_ptr=P), "another operand"), (dict(n_free_out_ptr=4 * P), "another operand"),
    (dict(held_ptr=10 * P, held_out_ptr=5 * P), "another operand"), (dict(slot_ptr=8 * P), "another operand"),
    (dict(short_ptr=3 * P), "another operand"), (dict(start_ptr=2 * P), "another operand"),
])
def test_plan_refuses(kw, word):
    refused(K.lib().kq_kv_plan_dev(ctypes.byref(plan(**kw)), None), word)


def cache(**kw):
    a = dict(qtype=K.TYPE_F16, n_pages=100, page=16, n_kv=2, D=64, k_ptr=P, v_ptr=P)
    a.update(kw)
    return K.kv_cache(**a)


CACHES = [(dict(qtype=K.TYPE_F32), "cache type 0"), (dict(qtype=12), "cache type 12"), (dict(n_pages=0), "0 pages"),
          (dict(page=0), "0 tokens"), (dict(n_pages=1 << 28, page=16), "pages of"), (dict(n_kv=0), "0 heads"),
          (dict(D=4), "D=4"), (dict(D=68), "D=68"), (dict(D=512), "D=512"), (dict(k_ptr=None), "NULL cache"),
          (dict(v_ptr=None), "NULL cache"), (dict(k_ptr=P + 8), "16-byte"), (dict(v_ptr=P + 2), "16-byte"),
          (dict(qtype=K.TYPE_I8), "scales"), (dict(qtype=K.TYPE_I8, k_scale_ptr=P), "scales"),
          (dict(qtype=K.TYPE_I8, k_scale_ptr=P, v_scale_ptr=P + 2), "scales"), (dict(k_scale_ptr=P), "not int8"),
          (dict(token_stride=56), "strides"), (dict(token_stride=68), "strides"), (dict(head_stride=-64), "strides"),
          (dict(page_stride=100), "strides"), (dict(token_stride=(1 << 24) + 8), "strides")]


@pytest.mark.parametrize("kw,word", CACHES)
def test_caches(kw, word):
    L = K.lib()
    refused(L.kq_kv_store_dev(ctypes.byref(store(cache=cache(**kw))), None), word)
    refused(L.kq_paged_attn_dev(ctypes.byref(attn(cache=cache(**kw))), P, 1 << 40, None), word)


def store(**kw):
    a = dict(cache=cache(), N=3, slot_ptr=P, k_ptr=P, v_ptr=P, pos_ptr=P, rot=64, freq_ptr=P, n_q=8, q_ptr=P, q_out_ptr=P)
    a.update(kw)
    return K.kv_store(**a)


@pytest.mark.parametrize("kw,word", [
    (dict(N=0), "N=0"), (dict(N=(1 << 22) + 1), "N="), (dict(slot_ptr=None), "NULL"), (dict(k_ptr=None), "NULL"),
    (dict(v_ptr=None), "NULL"), (dict(rot=63), "rot 63"), (dict(rot=66), "rot 66"), (dict(rot=-2), "rot -2"),
    (dict(pos_ptr=None), "pos or freq"), (dict(freq_ptr=None), "pos or freq"), (dict(q_out_ptr=None), "go together"),
    (dict(n_q=0), "go together"), (dict(q_ptr=None), "go together"), (dict(n_q=1025), "go together"),
    (dict(k_ptr=P + 4), "16-byte"), (dict(q_ptr=P + 8), "16-byte"), (dict(slot_ptr=P + 2), "aligned"),
    (dict(freq_ptr=P + 1), "aligned"), (dict(n_tokens_ptr=P + 1), "aligned"), (dict(k_stride=127), "stride"),
    (dict(v_stride=130), "stride"), (dict(q_stride=-512), "stride"), (dict(q_out_stride=516), "in place"),
])
def test_store_refuses(kw, word):
    refused(K.lib().kq_kv_store_dev(ctypes.byref(store(**kw)), None), word)


def attn(**kw):
    a = dict(shape=shape(), cache=cache(), q_ptr=P, out_ptr=2 * P, N=8, table_ptr=P, table_stride=10, start_ptr=P,
             lens_ptr=P, scale=0.125)
    a.update(kw)
    return K.paged_attn(**a)


@pytest.mark.parametrize("kw,word", [
    (dict(shape=shape(n_kv=4)), "cache of 2"), (dict(shape=shape(D=128)), "cache of 2"),
    (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale"), (dict(N=0), "N=0"),
    (dict(q_ptr=None), "NULL"), (dict(out_ptr=None), "NULL"), (dict(table_ptr=None), "NULL"), (dict(lens_ptr=None), "NULL"),
    (dict(out_ptr=P), "one buffer"), (dict(table_stride=0), "table of 0"), (dict(q_ptr=P + 4), "16-byte"),
    (dict(out_ptr=P + 8), "16-byte"), (dict(table_ptr=P + 2), "aligned"), (dict(start_ptr=P + 1), "aligned"),
    (dict(lens_ptr=P + 2), "aligned"), (dict(q_stride=508), "strides"), (dict(out_stride=513), "strides"),
    (dict(q_stride=-512), "strides"),
])
def test_attn_refuses(kw, word):
    refused(K.lib().kq_paged_attn_dev(ctypes.byref(attn(**kw)), None, 0, None), word)


@pytest.mark.parametrize("scale", [2.5e38, -3e38, 3.4028234e38])
def test_attn_refuses_scales_that_pass_the_range_times_log2_e(scale):
    refused(K.lib().kq_paged_attn_dev(ctypes.byref(attn(scale=scale)), None, 0, None), "scale")
