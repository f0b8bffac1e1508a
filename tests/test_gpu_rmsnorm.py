"""kq_rmsnorm_dev against the formula in 64 bits.

Bounds: s = fl(x + r) exactly.  y is the binary64 value rounded once: within
half a step, 2^-24 |y| (2^-150 below the normal range), of the exact one, but
for the binary64 value's own error, at most (K + 8) 2^-53 |y| (a sum of K
squares of one sign, its root, two products).  The int8 rows are
kq_quantize_x_q8_dev's of the written y, bit for bit."""
import numpy as np
import pytest

import stratum_amd as K

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module", autouse=True)
def device():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    K.lib()
    yield
    torch.cuda.synchronize()


def st():
    return torch.cuda.current_stream().cuda_stream


def rows(seed, B, n, stride, off=0, scale=1.0):
    """B rows of n values, `stride` apart, `off` floats past a 256-byte border; the rest NaN."""
    g = np.random.default_rng(seed)
    buf = torch.full((B * stride + off + 8,), float("nan"), device="cuda")
    v = buf[off:off + B * stride].view(B, stride)
    x = (g.standard_normal((B, n)) * scale).astype(np.float32)
    x[:, g.random(n) < 0.01] *= 8
    v[:, :n] = torch.from_numpy(x).cuda()
    return buf, v, x


def want(x, r, w, eps):
    s = x + r if r is not None else x
    assert s.dtype == np.float32
    d = s.astype(np.float64)
    y = d / np.sqrt((d * d).sum(1, keepdims=True) / d.shape[1] + np.float64(np.float32(eps)))
    return s, y * w.astype(np.float64) if w is not None else y


def check_y(got, exact):
    n = exact.shape[1]
    tol = np.abs(exact) * (2.0 ** -24 * (1 + 2.0 ** -20) + (n + 8) * 2.0 ** -53) + 2.0 ** -149
    assert (np.abs(got.astype(np.float64) - exact) <= tol).all()


def quantized(y, B, n, G):
    q, sc, su = (torch.empty(B * n, dtype=torch.int8, device="cuda"), torch.empty(B * n // G, device="cuda"),
                 torch.empty(B * n // G, dtype=torch.int32, device="cuda"))
    K.quantize_x_q8_dev(y.contiguous().data_ptr(), B * n, G, q.data_ptr(), sc.data_ptr(), su.data_ptr(), st())
    return q, sc, su


@pytest.mark.parametrize("resid,weight", [(False, False), (False, True), (True, False), (True, True)])
@pytest.mark.parametrize("B,n,stride,off", [
    (1, 1, 1, 0), (3, 2, 5, 1), (1, 63, 63, 0), (5, 64, 64, 0), (2, 100, 101, 3), (7, 256, 260, 0),
    (4, 1027, 1027, 2), (3, 1028, 1028, 0), (1, 5120, 5120, 0), (9, 5120, 5121, 0), (2, 8192, 8192, 4),
    (2, 8196, 8200, 0), (3, 16384, 16384, 0), (2, 20001, 20001, 0), (2, 40000, 40000, 0), (1, 70001, 70001, 1),
    (1, 150000, 150000, 0), (700, 130, 132, 0), (300, 4096, 4096, 0)])
def test_rows(B, n, stride, off, resid, weight):
    xb, xv, x = rows(1 + n, B, n, stride, off)
    rb, rv, r = rows(2 + n, B, n, stride, off, 2.0)
    wb, wv, w = rows(3 + n, 1, n, n, off)
    sb, sv, _ = rows(4, B, n, stride, off)
    yb, yv, _ = rows(5, B, n, stride, off)
    sv[:], yv[:] = float("nan"), float("nan")
    r, w = r if resid else None, w[0] if weight else None
    s_exact, y_exact = want(x, r, w, 1e-6)
    K.rmsnorm_dev(K.rmsnorm(B, n, 1e-6, xv.data_ptr(), resid_ptr=rv.data_ptr() if resid else None,
                            sum_ptr=sv.data_ptr() if resid else None,
                            weight_ptr=wv.data_ptr() if weight else None, y_ptr=yv.data_ptr(),
                            x_stride=stride, resid_stride=stride, sum_stride=stride, y_stride=stride), st())
    torch.cuda.synchronize()
    got = yv[:, :n].cpu().numpy()
    check_y(got, y_exact)
    if resid:
        assert np.array_equal(sv[:, :n].cpu().numpy().view(np.uint32), s_exact.view(np.uint32))
    # nothing between or behind the rows is written
    assert torch.isnan(yv[:, n:]).all() and torch.isnan(yb[:off]).all() and torch.isnan(yb[-8:]).all()
    assert torch.isnan(sv[:, n:]).all() and torch.isnan(sb[-8:]).all()


@pytest.mark.parametrize("G", [16, 32])
@pytest.mark.parametrize("keep_y", [False, True])
@pytest.mark.parametrize("B,n,stride,off", [
    (1, 32, 32, 0), (3, 64, 65, 1), (5, 96, 96, 0), (2, 1024, 1024, 0), (1, 5120, 5120, 0), (13, 5120, 5124, 0),
    (2, 5152, 5152, 3), (600, 2080, 2080, 0), (2, 20000, 20000, 0), (2, 17408, 17408, 0), (1, 66048, 66048, 0),
    (1, 66080, 66081, 1)])
def test_int8_rows(B, n, stride, off, G, keep_y):
    n -= n % G
    xb, xv, x = rows(10 + n, B, n, stride, off)
    rb, rv, r = rows(11 + n, B, n, stride, off)
    w = (1 + 0.2 * np.random.default_rng(12).standard_normal(n)).astype(np.float32)
    dw = torch.from_numpy(w).cuda()
    sm = torch.empty(B, n, device="cuda")
    y = torch.empty(B, n, device="cuda")
    q = torch.full((B * n + 64,), 77, dtype=torch.int8, device="cuda")
    sc = torch.full((B * n // G + 8,), float("nan"), device="cuda")
    su = torch.full((B * n // G + 8,), 12345, dtype=torch.int32, device="cuda")

    def call(yp, sup):
        K.rmsnorm_dev(K.rmsnorm(B, n, 1e-5, xv.data_ptr(), resid_ptr=rv.data_ptr(), sum_ptr=sm.data_ptr(),
                                weight_ptr=dw.data_ptr(), y_ptr=yp, group=G, xq_ptr=q.data_ptr(),
                                xscale_ptr=sc.data_ptr(), xsum_ptr=sup, x_stride=stride, resid_stride=stride), st())
    s_exact, y_exact = want(x, r, w, 1e-5)
    # the binary32 rows of the same call without int8 rows
    K.rmsnorm_dev(K.rmsnorm(B, n, 1e-5, xv.data_ptr(), resid_ptr=rv.data_ptr(), weight_ptr=dw.data_ptr(),
                            y_ptr=y.data_ptr(), x_stride=stride, resid_stride=stride), st())
    torch.cuda.synchronize()
    check_y(y.cpu().numpy(), y_exact)
    y2 = torch.full((B, n), float("nan"), device="cuda")
    call(y2.data_ptr() if keep_y else None, su.data_ptr() if keep_y else None)
    wq, ws, wu = quantized(y, B, n, G)
    torch.cuda.synchronize()
    assert torch.equal(q[:B * n], wq) and (q[B * n:] == 77).all()
    assert torch.equal(sc[:B * n // G].view(torch.int32), ws.view(torch.int32)) and torch.isnan(sc[B * n // G:]).all()
    if keep_y:
        assert torch.equal(y2.view(torch.int32), y.view(torch.int32))
        assert torch.equal(su[:B * n // G], wu) and (su[B * n // G:] == 12345).all()
    else:
        assert torch.isnan(y2).all() and (su == 12345).all()
    assert np.array_equal(sm.cpu().numpy().view(np.uint32), s_exact.view(np.uint32))


@pytest.mark.parametrize("B,n", [(3, 200), (2, 5120), (2, 40001)])
def test_in_place(B, n):
    """sum over x with y over the residual, the other way round, and y over x."""
    _, xv, x = rows(20, B, n, n)
    _, rv, r = rows(21, B, n, n)
    s_exact, y_exact = want(x, r, None, 1e-6)
    for s_at, y_at in (("x", "r"), ("r", "x")):
        bx, br = xv.clone(), rv.clone()
        at = {"x": bx, "r": br}
        K.rmsnorm_dev(K.rmsnorm(B, n, 1e-6, bx.data_ptr(), resid_ptr=br.data_ptr(), sum_ptr=at[s_at].data_ptr(),
                                y_ptr=at[y_at].data_ptr()), st())
        torch.cuda.synchronize()
        assert np.array_equal(at[s_at].cpu().numpy(), s_exact)
        check_y(at[y_at].cpu().numpy(), y_exact)
    bx = xv.clone()
    K.rmsnorm_dev(K.rmsnorm(B, n, 1e-6, bx.data_ptr(), y_ptr=bx.data_ptr()), st())
    torch.cuda.synchronize()
    check_y(bx.cpu().numpy(), want(x, None, None, 1e-6)[1])


def test_far_values():
    """Squares past the binary32 range on both sides, a zero row, and eps = 0."""
    n = 512
    g = np.random.default_rng(30)
    x = g.standard_normal((5, n)).astype(np.float32)
    x[0] *= np.float32(1e30)
    x[1] *= np.float32(1e-30)
    x[2] = 0
    x[3, 1:] = 0
    dx = torch.from_numpy(x).cuda()
    for eps in (0.0, 1e-6):
        y = torch.empty_like(dx)
        K.rmsnorm_dev(K.rmsnorm(5, n, eps, dx.data_ptr(), y_ptr=y.data_ptr()), st())
        torch.cuda.synchronize()
        got = y.cpu().numpy()
        with np.errstate(invalid="ignore", divide="ignore"):
            exact = want(x, None, None, eps)[1]
        live = [0, 1, 3, 4] if eps == 0 else [0, 1, 2, 3, 4]
        check_y(got[live], exact[live])
        if eps == 0:
            assert np.isnan(got[2]).all()


def test_infinite_and_nan_values_stay_in_their_row():
    x = np.random.default_rng(31).standard_normal((4, 1000)).astype(np.float32)
    exact = want(x, None, None, 1e-6)[1]
    x[1, 5], x[2, 7] = np.inf, np.nan
    dx = torch.from_numpy(x).cuda()
    y = torch.empty_like(dx)
    K.rmsnorm_dev(K.rmsnorm(4, 1000, 1e-6, dx.data_ptr(), y_ptr=y.data_ptr()), st())
    torch.cuda.synchronize()
    got = y.cpu().numpy()
    check_y(got[[0, 3]], exact[[0, 3]])
    assert np.isnan(got[2]).all() and np.isnan(got[1, 5]) and (got[1, :5] == 0).all()


def test_captured_and_on_another_stream():
    """A replayed graph of the call follows its inputs; a call on a side stream gives the same bits."""
    B, n = 6, 2048
    _, xv, x = rows(40, B, n, n)
    _, rv, r = rows(41, B, n, n)
    q, sc = torch.empty(B, n, dtype=torch.int8, device="cuda"), torch.empty(B, n // 32, device="cuda")
    sm = torch.empty(B, n, device="cuda")
    a = K.rmsnorm(B, n, 1e-6, xv.data_ptr(), resid_ptr=rv.data_ptr(), sum_ptr=sm.data_ptr(), group=32,
                  xq_ptr=q.data_ptr(), xscale_ptr=sc.data_ptr())
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        K.rmsnorm_dev(a, st())
    for i in range(3):
        xv.copy_(torch.from_numpy(x * (i + 1)))
        q.zero_(), sc.zero_()
        graph.replay()
        torch.cuda.synchronize()
        got = q.clone(), sc.clone(), sm.clone()
        with torch.cuda.stream(side):
            q.zero_(), sc.zero_()
            K.rmsnorm_dev(a, side.cuda_stream)
        torch.cuda.synchronize()
        assert torch.equal(got[0], q) and torch.equal(got[1], sc) and torch.equal(got[2], sm)
        assert np.array_equal(sm.cpu().numpy(), (x * np.float32(i + 1) + r))


def test_rows_past_32_bits():
    """Row strides that put the second row past 2^32 bytes, and the fourth past 2^32 elements."""
    n, stride = 1000, (1 << 30) + 4
    buf = torch.empty(4 * stride, device="cuda")
    rows4 = buf.view(4, stride)[:, :n]
    x = np.random.default_rng(50).standard_normal((4, n)).astype(np.float32)
    rows4.copy_(torch.from_numpy(x))
    y = torch.empty(4, n, device="cuda")
    K.rmsnorm_dev(K.rmsnorm(4, n, 1e-6, buf.data_ptr(), y_ptr=y.data_ptr(), x_stride=stride), st())
    K.rmsnorm_dev(K.rmsnorm(4, n, 1e-6, buf.data_ptr(), y_ptr=buf.data_ptr(), x_stride=stride, y_stride=stride), st())
    torch.cuda.synchronize()
    check_y(y.cpu().numpy(), want(x, None, None, 1e-6)[1])
    assert torch.equal(rows4, y)


@pytest.mark.parametrize("group", [0, 16])
def test_more_rows_than_a_launch_takes(group):
    """Rows times lanes past 2^32: 64 lanes a row are the fewest, so 2^26 rows and some."""
    B, n = (1 << 26) + 77, 16 if group else 1
    x = torch.empty(B, n, device="cuda").uniform_(0.5, 2.0)
    x[:, ::3] *= -1
    q, sc = (torch.zeros(B, n, dtype=torch.int8, device="cuda"), torch.zeros(B, device="cuda")) if group else (None, None)
    y = torch.full((B, n), float("nan"), device="cuda")
    K.rmsnorm_dev(K.rmsnorm(B, n, 1e-6, x.data_ptr(), y_ptr=y.data_ptr(), group=group,
                            xq_ptr=q.data_ptr() if group else None, xscale_ptr=sc.data_ptr() if group else None), st())
    torch.cuda.synchronize()
    for a in range(0, B, 1 << 24):
        d = x[a:a + (1 << 24)].double()
        want = d / torch.sqrt((d * d).mean(1, keepdim=True) + np.float64(np.float32(1e-6)))
        got = y[a:a + (1 << 24)].double()
        assert ((got - want).abs() <= want.abs() * (2.0 ** -24 * (1 + 2.0 ** -20) + 24 * 2.0 ** -53)).all()
        if group:
            s = sc[a:a + (1 << 24), None].double()
            assert ((q[a:a + (1 << 24)].double() * s - got).abs() <= s * (0.5 + 2.0 ** -16)).all()
