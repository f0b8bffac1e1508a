"""The row operators around the products refuse bad arguments with -1 and a
message before anything is enqueued (no GPU needed: each check comes before
the device is looked at, and the addresses here are never read)."""
import ctypes

import pytest

import stratum_amd as K

P = 1 << 20          # an aligned address; nothing is read from it


def refused(rc, word):
    assert rc == -1
    msg = K.lib().kq_last_error().decode()
    assert word in msg, msg


def norm(**kw):
    a = dict(B=2, K=64, eps=1e-6, x_ptr=P, y_ptr=P + 4096)
    a.update(kw)
    return K.rmsnorm(**a)


@pytest.mark.parametrize("kw,word", [
    (dict(B=0), "B=0"), (dict(K=0), "K=0"), (dict(K=-5), "K=-5"),
    (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"), (dict(eps=float("inf")), "eps"),
    (dict(x_ptr=None), "NULL x"), (dict(y_ptr=None), "group 0 takes y"),
    (dict(xq_ptr=P), "group 0 takes y"), (dict(xscale_ptr=P), "group 0 takes y"),
    (dict(group=8), "group 8"), (dict(group=64), "group 64"),
    (dict(group=32, K=48, xq_ptr=P, xscale_ptr=P), "K=48"),
    (dict(group=32), "xq and xscale"), (dict(group=16, xq_ptr=P), "xq and xscale"),
    (dict(x_ptr=P + 2), "aligned"), (dict(resid_ptr=P + 1), "aligned"),
    (dict(group=32, xq_ptr=P + 2, xscale_ptr=P), "aligned"),
    (dict(x_stride=63), "stride"), (dict(y_stride=-64), "stride"), (dict(sum_ptr=P, sum_stride=8), "stride"),
    (dict(sum_ptr=P + 4096), "one buffer"),
    (dict(sum_ptr=P, sum_stride=128), "another row stride"),
    (dict(y_ptr=P, x_stride=128), "another row stride"),
])
def test_rmsnorm_refuses(kw, word):
    refused(K.lib().kq_rmsnorm_dev(ctypes.byref(norm(**kw)), None), word)


def test_null_descriptors():
    L = K.lib()
    refused(L.kq_rmsnorm_dev(None, None), "NULL")
    refused(L.kq_w4_gemv_dev(None, P, None, P, 1, None, 0, None), "NULL")
    refused(L.kq_w4_gemv_q8_dev(None, P, P, None, P, 1, None, 0, None), "NULL")
    refused(L.kq_w4_workspace_bytes(None, 1, 0), "NULL")
    refused(L.kq_spec_verify_dev(None, P, 0, None), "NULL")
    refused(L.kq_spec_verify_workspace_bytes(None), "NULL")


def w4(**kw):
    a = dict(N=16, K=128, group=32, scale_type=K.TYPE_F16, q_ptr=P, scales_ptr=P)
    a.update(kw)
    return K.w4(**a)


@pytest.mark.parametrize("kw,word", [
    (dict(N=0), "N=0"), (dict(N=(1 << 28) + 1), "N="), (dict(K=0), "K=0"), (dict(K=48), "K=48"),
    (dict(group=16), "group 16"), (dict(group=48), "group 48"), (dict(group=96), "group 96"),
    (dict(group=0), "group 0"), (dict(group=-32), "group -32"), (dict(group=256), "group 256"),
    (dict(scale_type=12), "scale type"), (dict(q_ptr=None), "NULL"), (dict(scales_ptr=None), "NULL"),
    (dict(q_ptr=P + 8), "16-byte"), (dict(scales_ptr=P + 1), "aligned"),
    (dict(scale_type=K.TYPE_F32, scales_ptr=P + 2), "aligned"),
])
def test_w4_refuses(kw, word):
    L, w = K.lib(), w4(**kw)
    refused(L.kq_w4_gemv_dev(ctypes.byref(w), P, None, P, 1, None, 0, None), word)
    refused(L.kq_w4_gemv_q8_dev(ctypes.byref(w), P, P, None, P, 1, None, 0, None), word)
    if word not in ("NULL", "16-byte", "aligned"):
        refused(L.kq_w4_workspace_bytes(ctypes.byref(w), 1, 0), word)


def test_w4_refuses_operands():
    L, w = K.lib(), ctypes.byref(w4())
    for B in (0, -1, 65536):
        refused(L.kq_w4_gemv_dev(w, P, None, P, B, None, 0, None), "B=")
        refused(L.kq_w4_workspace_bytes(w, B, 1), "B=")
    refused(L.kq_w4_gemv_dev(w, None, None, P, 1, None, 0, None), "NULL")
    refused(L.kq_w4_gemv_dev(w, P, None, None, 1, None, 0, None), "NULL")
    refused(L.kq_w4_gemv_dev(w, P + 4, None, P, 1, None, 0, None), "16-byte")
    refused(L.kq_w4_gemv_dev(w, P, P + 2, P, 1, None, 0, None), "aligned")
    refused(L.kq_w4_gemv_dev(w, P, None, P + 1, 1, None, 0, None), "aligned")
    refused(L.kq_w4_gemv_q8_dev(w, None, P, None, P, 1, None, 0, None), "NULL")
    refused(L.kq_w4_gemv_q8_dev(w, P, None, None, P, 1, None, 0, None), "NULL")
    refused(L.kq_w4_gemv_q8_dev(w, P + 8, P, None, P, 1, None, 0, None), "16-byte")
    refused(L.kq_w4_gemv_q8_dev(w, P, P + 2, None, P, 1, None, 0, None), "aligned")


def verify(**kw):
    a = dict(S=2, T=3, V=100, flags=K.VERIFY_LOGITS, target_ptr=P, tokens_ptr=P, u_ptr=P,
             n_accept_ptr=P, out_ptr=P)
    a.update(kw)
    return K.spec_verify(**a)


@pytest.mark.parametrize("kw,word", [
    (dict(S=0), "S=0"), (dict(T=-1), "T=-1"), (dict(T=64), "T=64"), (dict(S=10000, T=3), "S=10000"),
    (dict(V=0), "V=0"), (dict(V=(1 << 28) + 1), "V="), (dict(flags=4), "flags"),
    (dict(target_ptr=None), "NULL"), (dict(tokens_ptr=None), "NULL"), (dict(u_ptr=None), "NULL"),
    (dict(n_accept_ptr=None), "NULL"), (dict(out_ptr=None), "NULL"),
    (dict(inv_temp=0.0), "inv_temp"), (dict(inv_temp=-1.0), "inv_temp"),
    (dict(inv_temp=float("inf")), "inv_temp"), (dict(inv_temp=float("nan")), "inv_temp"),
    (dict(target_ptr=P + 2), "aligned"), (dict(u_ptr=P + 1), "aligned"), (dict(out_ptr=P + 2), "aligned"),
    (dict(draft_ptr=P + 2), "aligned"), (dict(n_draft_ptr=P + 2), "aligned"),
    (dict(target_row=-100), "stride"), (dict(draft_ptr=P, draft_seq=-1), "stride"),
])
def test_verify_refuses(kw, word):
    v = verify(**kw)
    refused(K.lib().kq_spec_verify_dev(ctypes.byref(v), P, 1 << 40, None), word)


def test_verify_workspace_bytes():
    """Refuses what the call refuses by shape; grows with the rows that are read."""
    L = K.lib()
    for kw, word in ((dict(S=0), "S=0"), (dict(T=64), "T=64"), (dict(V=0), "V=0"), (dict(flags=8), "flags")):
        refused(L.kq_spec_verify_workspace_bytes(ctypes.byref(verify(**kw))), word)
    n = [K.spec_verify_workspace_bytes(verify(**kw)) for kw in
         (dict(flags=0), dict(), dict(draft_ptr=P), dict(draft_ptr=P, V=100000))]
    assert 0 < n[0] < n[1] <= n[2] < n[3]
