"""kq_w4_gemv_dev and kq_w4_gemv_q8_dev against the products in 64 bits.

Bounds, per output, with a = sum_k |s| |q - z| amax_k (amax_k: the largest |x|
of the 32 values that k lies in): a binary32 x enters with an error of at most
2^-22 amax (half a unit of 2^-22 of the power of two above amax); a block of 32
products is an integer sum, rounded at most 5 times on its way (its planes'
sum, the zero point's part, the scales); the blocks' sums are added in any
order, at most K / 32 additions, then `add`: in all
(K / 32 + 8) 2^-24 a + 2^-24 |y|."""
import ctypes

import numpy as np
import pytest

import stratum_amd as K

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

TYPES = {"f16": (K.TYPE_F16, torch.float16), "bf16": (K.TYPE_BF16, torch.bfloat16), "f32": (K.TYPE_F32, torch.float32)}


@pytest.fixture(scope="module", autouse=True)
def device():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    K.lib()
    yield
    torch.cuda.synchronize()


def st():
    return torch.cuda.current_stream().cuda_stream


class Case:
    """A matrix, B rows of x, and the exact products (binary64, on the CPU)."""

    def __init__(self, N, Kd, B, g, scale="f16", zeros=False, q8=False, seed=0, xscale=1.0):
        r = np.random.default_rng(1000 * seed + N + 7 * Kd + 13 * B + g)
        self.N, self.K, self.B, self.g, self.q8 = N, Kd, B, g, q8
        q = r.integers(0, 256, (N, Kd // 2), dtype=np.uint8)
        s = torch.from_numpy((0.004 * np.exp(0.5 * r.standard_normal((N, Kd // g)))).astype(np.float32))
        s[r.random((N, Kd // g)) < 0.05] *= -1
        s = s.to(TYPES[scale][1])
        z = r.integers(0, 16, (N, Kd // g), dtype=np.uint8) if zeros else None
        x = (r.standard_normal((B, Kd)) * xscale).astype(np.float32)
        x[:, r.random(Kd) < 0.01] *= 30
        if Kd > 64:
            x[:, 32:64] = 0                      # a block of zeros
        self.dq, self.ds = torch.from_numpy(q).cuda(), s.cuda()
        self.dz = torch.from_numpy(z).cuda() if zeros else None
        n = np.stack([q & 15, q >> 4], -1).reshape(N, Kd // g, g).astype(np.float64)
        n -= 8.0 if z is None else z[:, :, None]
        self.W = (n * s.double().numpy()[:, :, None]).reshape(N, Kd)
        amax = np.abs(x).reshape(B, -1, 32).max(-1)
        if q8:
            sc = (amax / np.float32(127)).astype(np.float32)
            xq = np.where(sc[:, :, None] > 0, np.rint(x.reshape(B, -1, 32) / np.where(sc > 0, sc, 1)[:, :, None]), 0)
            xq = np.clip(xq, -128, 127).astype(np.int8).reshape(B, Kd)
            if Kd > 64:
                xq[:, :32] = np.where(r.random((B, 32)) < 0.5, -128, 127)    # the ends of the type
            x = xq.astype(np.float64) * np.repeat(sc, 32, 1).astype(np.float64)
            amax = sc * 128.0
            self.dxq, self.dxs = torch.from_numpy(xq).cuda(), torch.from_numpy(sc).cuda()
        else:
            self.dx = torch.from_numpy(x).cuda()
        self.exact = x.astype(np.float64) @ self.W.T
        self.a = np.repeat(amax, 32, 1).astype(np.float64) @ np.abs(self.W).T
        self.desc = K.w4(N, Kd, g, TYPES[scale][0], self.dq.data_ptr(), self.ds.data_ptr(),
                         self.dz.data_ptr() if zeros else None)
        self.nb = K.w4_workspace_bytes(self.desc, B, q8)
        self.work = torch.full((self.nb + 256,), 0xA5, dtype=torch.uint8, device="cuda")

    def call(self, y, add=None, stream=None, work=None):
        args = (y.data_ptr(), self.B, (self.work if work is None else work).data_ptr(), self.nb,
                add.data_ptr() if add is not None else None, st() if stream is None else stream)
        if self.q8:
            K.w4_gemv_q8_dev(self.desc, self.dxq.data_ptr(), self.dxs.data_ptr(), *args)
        else:
            K.w4_gemv_dev(self.desc, self.dx.data_ptr(), *args)

    def tol(self, y):
        return (self.K / 32 + 8) * 2.0 ** -24 * self.a + 2.0 ** -24 * np.abs(y) + 1e-40

    def check(self, add=None):
        y = torch.full((self.B * self.N + 32,), float("nan"), device="cuda")
        self.call(y, add)
        torch.cuda.synchronize()
        got = y[:self.B * self.N].cpu().numpy().reshape(self.B, self.N).astype(np.float64)
        want = self.exact if add is None else self.exact + add.cpu().numpy().reshape(self.B, self.N)
        bad = ~(np.abs(got - want) <= self.tol(want))
        assert not bad.any(), (np.argwhere(bad)[:5], got[bad][:5], want[bad][:5])
        assert torch.isnan(y[self.B * self.N:]).all()
        assert (self.work[self.nb:] == 0xA5).all()
        return y


SHAPES = [(1, 32, 32), (1, 64, 64), (5, 96, 32), (16, 128, 128), (17, 160, 160), (33, 256, 64), (64, 1024, 32),
          (100, 1056, 352), (257, 2048, 128), (31, 4096, 4096), (1000, 640, 64), (130, 5120, 128), (40, 17408, 64),
          (19, 2720, 32), (3000, 512, 256)]


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("N,Kd,g", SHAPES)
@pytest.mark.parametrize("B", [1, 2, 3, 4, 5, 8])
def test_products(N, Kd, g, B, q8):
    Case(N, Kd, B, g, zeros=(N + B) % 2 == 0, q8=q8).check()


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("B", [6, 7, 9, 12, 15, 16, 17, 31, 32, 33, 48, 63, 64, 65, 130])
@pytest.mark.parametrize("N,Kd,g", [(77, 352, 32), (208, 1280, 128), (19, 3104, 3104)])
def test_many_rows(N, Kd, g, B, q8):
    Case(N, Kd, B, g, zeros=B % 2 == 1, q8=q8).check()


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("scale", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("g", [32, 64, 96, 128, 192, 256, 384])
@pytest.mark.parametrize("B", [1, 3, 11])
def test_groups_and_scale_types(B, g, zeros, scale, q8):
    Case(53, 2304, B, g, scale, zeros, q8).check()


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("N,Kd,B", [(151, 57344, 1), (50, 65536, 3), (20, 90112, 9), (7, 131072 + 32, 2), (6, 131072, 20)])
def test_long_rows(N, Kd, B, q8):
    Case(N, Kd, B, 32, q8=q8).check()


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("B", [1, 2, 5, 16])
def test_many_rows_of_weights(B, q8):
    """More rows than any grid has waves, the last ones cut off mid-tile."""
    Case(70001, 64, B, 32, zeros=True, q8=q8).check()


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("B", [1, 3, 20])
def test_add(B, q8):
    c = Case(300, 768, B, 128, q8=q8)
    add = torch.from_numpy(np.random.default_rng(5).standard_normal(B * 300).astype(np.float32)).cuda()
    y = c.check(add)
    over = add.clone()                           # in place
    c.call(over, over)
    torch.cuda.synchronize()
    assert torch.equal(over, y[:B * 300])


@pytest.mark.parametrize("xscale", [1e-30, 1e-3, 1e4, 1e30])
@pytest.mark.parametrize("B", [1, 6])
def test_far_x(B, xscale):
    """x far from 1, each block with its own power of two."""
    Case(64, 1024, B, 64, "f32", xscale=xscale).check()


@pytest.mark.parametrize("B", [1, 6])
def test_wide_blocks(B):
    """Values of one block of 32 that lie 2^20 apart: the bound counts the largest."""
    c = Case(64, 512, B, 32)
    x = c.dx.cpu().numpy()
    x[:, ::3] *= np.float32(2.0 ** -20)
    c.dx = torch.from_numpy(x).cuda()
    c.exact = x.astype(np.float64) @ c.W.T
    c.a = np.repeat(np.abs(x).reshape(B, -1, 32).max(-1), 32, 1).astype(np.float64) @ np.abs(c.W).T
    c.check()


@pytest.mark.parametrize("q8", [False, True])
def test_rows_do_not_depend_on_each_other(q8):
    """A non-finite row of x leaves the others' bits alone (within one B)."""
    for B in (2, 4, 12):
        c = Case(90, 640, B, 64, q8=q8)
        y = c.check()[:B * 90].view(B, 90).clone()
        if q8:
            c.dxs[1, 3] = float("nan")
        else:
            c.dx[1, 100] = float("inf")
        y2 = torch.empty(B, 90, device="cuda")
        c.call(y2)
        torch.cuda.synchronize()
        keep = [b for b in range(B) if b != 1]
        assert torch.equal(y[keep].view(torch.int32), y2[keep].view(torch.int32))
        assert not torch.isfinite(y2[1]).any()


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("B", [1, 4, 16])
def test_same_bits_again_captured_and_on_two_streams(B, q8):
    """Repeated calls, replays of a graph and overlapping calls on two streams
    with workspaces of their own give the same bits."""
    c = [Case(500, 2048, B, 128, q8=q8, seed=i) for i in range(2)]
    n = B * 500
    first = [k.check()[:n].clone() for k in c]
    side = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    outs = []
    for rnd in range(4):
        for i in range(2):
            with torch.cuda.stream(side[i]):
                y = torch.full((n,), float("nan"), device="cuda")
                c[i].call(y, stream=side[i].cuda_stream)
                outs.append((i, y))
    torch.cuda.synchronize()
    for i, y in outs:
        assert torch.equal(y, first[i])
    graph, ys = torch.cuda.CUDAGraph(), [torch.empty(n, device="cuda") for _ in c]
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        for k, y in zip(c, ys):
            k.call(y)
    for rnd in range(3):
        for k, y in zip(c, ys):
            y.fill_(float("nan"))
            k.work.fill_(rnd)
        graph.replay()
        torch.cuda.synchronize()
        for i, y in enumerate(ys):
            assert torch.equal(y, first[i])
            z = torch.empty(n, device="cuda")      # eager work between the replays
            c[i].call(z)
            assert torch.equal(z, first[i])


def test_norm_to_product():
    """The norm's int8 rows go to the product as they are."""
    N, Kd, B = 200, 1024, 5
    c = Case(N, Kd, B, 128, q8=True)
    x = torch.randn(B, Kd, device="cuda")
    K.rmsnorm_dev(K.rmsnorm(B, Kd, 1e-6, x.data_ptr(), group=32, xq_ptr=c.dxq.data_ptr(),
                            xscale_ptr=c.dxs.data_ptr()), st())
    torch.cuda.synchronize()
    sc = c.dxs.cpu().numpy()
    xv = c.dxq.cpu().numpy().astype(np.float64) * np.repeat(sc, 32, 1)
    c.exact, c.a = xv @ c.W.T, np.repeat(sc * 128.0, 32, 1) @ np.abs(c.W).T
    c.check()


def test_refuses_a_short_workspace():
    for B in (1, 8, 16, 64):
        for q8 in (False, True):
            c = Case(64, 1024, B, 128, q8=q8)
            if not c.nb:
                continue
            y = torch.full((B, 64), 3.0, device="cuda")
            for work, nb in ((None, c.nb), (c.work.data_ptr(), c.nb - 1), (c.work.data_ptr() + 16, c.nb)):
                d = ctypes.byref(c.desc)
                L = K.lib()
                rc = (L.kq_w4_gemv_q8_dev(d, c.dxq.data_ptr(), c.dxs.data_ptr(), None, y.data_ptr(), B, work, nb, st())
                      if q8 else L.kq_w4_gemv_dev(d, c.dx.data_ptr(), None, y.data_ptr(), B, work, nb, st()))
                assert rc == -1 and b"workspace" in L.kq_last_error()
            torch.cuda.synchronize()
            assert (y == 3.0).all()


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("N,Kd,B", [(3, 64, 4097), (1, 32, 65535), (300, 6400, 250)])
def test_very_many_rows(N, Kd, B, q8):
    Case(N, Kd, B, 32, zeros=True, q8=q8).check()


@pytest.mark.parametrize("q8", [False, True])
def test_refuses_a_short_workspace_for_cut_rows(q8):
    """Rows that are cut into parts need workspace: without it, with less, unaligned."""
    for Kd, B in ((40960, 8), (65536, 16)):
        c = Case(20, Kd, B, 128, q8=q8)
        assert c.nb >= (2 if not q8 else 0) * 4 * 20 * B and c.nb % 256 == 0
        if not c.nb:
            continue
        y = torch.full((B, 20), 3.0, device="cuda")
        for work, nb in ((None, c.nb), (c.work.data_ptr(), c.nb - 1), (c.work.data_ptr() + 16, c.nb)):
            L, d = K.lib(), ctypes.byref(c.desc)
            rc = (L.kq_w4_gemv_q8_dev(d, c.dxq.data_ptr(), c.dxs.data_ptr(), None, y.data_ptr(), B, work, nb, st())
                  if q8 else L.kq_w4_gemv_dev(d, c.dx.data_ptr(), None, y.data_ptr(), B, work, nb, st()))
            assert rc == -1 and b"workspace" in L.kq_last_error()
        torch.cuda.synchronize()
        assert (y == 3.0).all()
        c.check()


@pytest.mark.parametrize("B", [1, 2, 6])
def test_subnormal_x(B):
    """Blocks of x below 2^-126: half a unit of x's integers is 2^-148 then, as at 2^-126; and per block
    the three roundings to multiples of 2^-149, the scale (below 1 / 8) and the zero (15) on them."""
    c = Case(70, 640, B, 64, zeros=True, xscale=1e-40)
    y = torch.empty(B, 70, device="cuda")
    c.call(y)
    torch.cuda.synchronize()
    xmax = np.maximum(c.dx.cpu().numpy().reshape(B, -1, 32).__abs__().max(-1), 2.0 ** -126)
    a = np.repeat(xmax, 32, 1).astype(np.float64) @ np.abs(c.W).T
    tol = (640 / 32 + 8) * 2.0 ** -24 * a + (640 / 32 + 8) * 4 * 2.0 ** -150
    assert (np.abs(y.cpu().numpy().astype(np.float64) - c.exact) <= tol).all()
    assert (y != 0).any()


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("B", [1, 3, 8])
def test_matrices_past_4_gib(B, q8):
    """Offsets past 32 bits: 2.2 M rows of 4096 weights, 4.5 GB.  Repeats of one small matrix, so that
    every repeat has to give the same bits."""
    n, Kd, g, reps = 1103, 4096, 128, 2000
    c = Case(n, Kd, B, g, zeros=True, q8=q8)
    first = c.check()[:B * n].view(B, n).clone()
    N = n * reps
    q, s, z = c.dq.repeat(reps, 1), c.ds.repeat(reps, 1), c.dz.repeat(reps, 1)
    assert q.numel() > 1 << 32
    w = K.w4(N, Kd, g, K.TYPE_F16, q.data_ptr(), s.data_ptr(), z.data_ptr())
    nb = K.w4_workspace_bytes(w, B, q8)
    work = torch.empty(max(256, nb), dtype=torch.uint8, device="cuda")
    y = torch.full((B, N), float("nan"), device="cuda")
    args = (y.data_ptr(), B, work.data_ptr(), nb)
    if q8:
        K.w4_gemv_q8_dev(w, c.dxq.data_ptr(), c.dxs.data_ptr(), *args, stream=st())
    else:
        K.w4_gemv_dev(w, c.dx.data_ptr(), *args, stream=st())
    torch.cuda.synchronize()
    got = y.view(B, reps, n)
    # (where a matrix is cut depends on its size, and with it the order of a row's sums)
    want, tol = torch.from_numpy(c.exact).cuda().view(B, 1, n), torch.from_numpy(c.tol(c.exact)).cuda().view(B, 1, n)
    assert ((got.double() - want).abs() <= tol).all()
    if B == 1:
        assert (got == first.view(B, 1, n)).all()


def given(c, x=None, nib=None):
    """The case with other x and other nibbles (N rows of K), and its exact products."""
    if x is not None:
        amax = np.abs(x).reshape(c.B, -1, 32).max(-1)
        if c.q8:
            sc = (amax / np.float32(127)).astype(np.float32)
            xq = np.rint(x.reshape(c.B, -1, 32).astype(np.float64) / sc[:, :, None])
            c.dxq, c.dxs = torch.from_numpy(xq.astype(np.int8).reshape(c.B, c.K)).cuda(), torch.from_numpy(sc).cuda()
        else:
            c.dx = torch.from_numpy(x).cuda()
    if nib is not None:
        c.dq.copy_(torch.from_numpy((nib[:, ::2] | nib[:, 1::2] << 4).astype(np.uint8)))
    q = c.dq.cpu().numpy()
    n = np.stack([q & 15, q >> 4], -1).reshape(c.N, -1, c.g).astype(np.float64)
    n -= 8.0 if c.dz is None else c.dz.cpu().numpy()[:, :, None]
    c.W = (n * c.ds.cpu().double().numpy()[:, :, None]).reshape(c.N, c.K)
    if c.q8:
        sc = c.dxs.cpu().numpy().astype(np.float64)
        x, amax = c.dxq.cpu().numpy().astype(np.float64) * np.repeat(sc, 32, 1), sc * 128
    else:
        x = c.dx.cpu().numpy().astype(np.float64)
        amax = np.abs(x).reshape(c.B, -1, 32).max(-1)
    c.exact, c.a = x @ c.W.T, np.repeat(amax, 32, 1) @ np.abs(c.W).T
    return c


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("B", [1, 2, 3, 4, 6, 16])
@pytest.mark.parametrize("g", [32, 128])
@pytest.mark.parametrize("scale", ["f16", "f32"])
def test_weights_at_their_zero_point(scale, g, B, q8):
    """Padded and pruned rows, x of one sign: the bound goes with |q - z|, so rows of which every
    weight is at its zero point give 0, and one weight in 128 gives no more error than its own."""
    r = np.random.default_rng(B + g)
    x = (1 + 0.2 * r.standard_normal((B, 1024))).astype(np.float32) * np.float32(5)
    for z in (None, 7, 8, 11, 15):
        c = Case(80, 1024, B, g, scale, z is not None, q8)
        zero = 8 if z is None else z
        if z is not None:
            c.dz.fill_(z)
        nib = np.full((80, 1024), zero, np.uint8)
        y = given(c, x, nib).check()
        assert (y[:B * 80] == 0).all()
        for k in range(8):
            nib[np.arange(80), 128 * k + r.integers(0, 128, 80)] ^= 1
        given(c, nib=nib).check()
        # near the zero point, most of them on it
        near = np.clip(zero + np.rint(0.4 * r.standard_normal((80, 1024))), 0, 15).astype(np.uint8)
        given(c, nib=near).check()


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("B", [1, 2, 3, 6, 16])
@pytest.mark.parametrize("zeros", [False, True])
def test_x_near_the_largest(zeros, B, q8):
    """Finite results of x up to binary32's largest: sums of 15 |x| over a block or a window lie past it
    while those of |w x| (at most 0.3 * 3.4e38, and 0.03 * 256 * 1e37 in the mean) do not."""
    r = np.random.default_rng(B)
    for g in (32, 128):
        for scale in ("f16", "bf16", "f32"):
            c = Case(48, 256, B, g, scale, zeros, q8)
            x = (1e37 * r.standard_normal((B, 256))).astype(np.float32)
            assert np.isfinite(given(c, x).check()[:B * 48].cpu().numpy()).all()
            x = (1e30 * r.standard_normal((B, 256))).astype(np.float32)
            x[:, 70] = np.float32(3.4e38)
            assert np.isfinite(given(c, x).check()[:B * 48].cpu().numpy()).all()
            if scale != "f16":              # scales far from 1 on either side of x
                for p in (-90, 90):
                    c.ds.mul_(2.0 ** p)
                    given(c, (r.standard_normal((B, 256)) * 2.0 ** -p).astype(np.float32)).check()
                    c.ds.mul_(2.0 ** -p)


def test_more_outputs_of_cut_rows_than_a_launch_has_lanes():
    """2^32 and more outputs of rows in two parts, which a launch of its own joins (50 GB): seven rows of x
    over and over, so that every repeat has to give the same bits, the first of them the bound's."""
    n, Kd, g, m = 337, 2560, 128, 7
    reps, B = 195, 65534
    c = Case(n, Kd, m, g)
    N = n * reps
    assert N * B > 1 << 32
    q, s = c.dq.repeat(reps, 1), c.ds.repeat(reps, 1)
    x = c.dx.repeat(B // m, 1).contiguous()
    w = K.w4(N, Kd, g, K.TYPE_F16, q.data_ptr(), s.data_ptr())
    nb = K.w4_workspace_bytes(w, B)
    assert nb >= 2 * 4 * N * B
    work = torch.empty(nb, dtype=torch.uint8, device="cuda")
    y = torch.full((B, N), float("nan"), device="cuda")
    K.w4_gemv_dev(w, x.data_ptr(), y.data_ptr(), B, work.data_ptr(), nb, stream=st())
    torch.cuda.synchronize()
    del work
    got = y[:m].cpu().numpy().reshape(m, reps, n).astype(np.float64)
    assert (np.abs(got - c.exact[:, None]) <= c.tol(c.exact)[:, None]).all()
    for a in range(0, B, 700):
        part = y[a:a + 700].view(-1, m, N)
        assert (part == y[:m]).all()
    del y, part
    torch.cuda.empty_cache()


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("g", [32, 64, 128])
def test_workspace_only_where_x_does_not_fit(g, q8):
    """With eight rows the waves' own LDS is 33 KB and a window of 128 values 3200 bytes (int8 1152), so
    that 160 KB hold 40 windows of them; none of these needs a workspace."""
    for N in (5120, 17408, 65536):
        for Kd in (128, 4096, 4992, 5120):
            for B in (1, 2, 5, 8):
                assert K.w4_workspace_bytes(K.w4(N, Kd, g, K.TYPE_F16, 256, 256), B, q8) == 0
    assert K.w4_workspace_bytes(K.w4(5120, 40960, g, K.TYPE_F16, 256, 256), 8, q8) > 0
