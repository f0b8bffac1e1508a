"""kq_paged_attn_dev against softmax attention in 64 bits.

Bounds.  With u = 2^-24: a score's products are good to 2^-21 of |scale q_d k_d| and
their sum of D terms, its scaling and the step to powers of two add at most (D + 8) u
of the sum of magnitudes X, and 4 u of the largest score (the maximum that is taken off
is such a value, and the exponent's product is rounded): every score is within
e = X (2^-21 + (D + 8) u) + 4 u max|x|.  A weight exp(x - m) and the sum of weights
are then within factors of exp(+-e) and of the power's own error (2 u), so that p_j
is within 2 e + 4 u of its value; the products with the values are good to 2^-21, and
sums over L keys (and the joins, fewer than L) are off by at most (2 L + 64) u of the
sum of p|v|, as is the weights' sum of itself.  Together, times sum p|v|:
    2 e + 2^-20 + (4 L + 200) u.
With binary16 and int8 caches a weight is two binary16 numbers, of 2^9 times the weight
(and of its value's scale over the largest one's power of two), whose last step is 2^-24:
2^-25 / 2^9 = 2^-34 of the row's largest weight (the one that has not more than 2^5 on
the base they are taken from, so it is no less than the base's) and of the largest
scale go missing at most, times a value each: L 2^-34 max|v| in all.  Queries likewise: two
binary16 numbers of the row times a power of two that puts its largest from 2^13 on, so
2^-25 / 2^13 = 2^-38 of that one, times sum |scale k_d|, is added to e."""
import copy

import numpy as np
import pytest

import stratum_amd as K

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

DT = {K.TYPE_F16: torch.float16, K.TYPE_BF16: torch.bfloat16, K.TYPE_I8: torch.int8}
U = 2.0 ** -24


@pytest.fixture(scope="module", autouse=True)
def device():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    K.lib()
    yield
    torch.cuda.synchronize()


def st():
    return torch.cuda.current_stream().cuda_stream


def ints(a):
    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).cuda()


class Case:
    """A cache whose unused places are NaN (int8: garbage under NaN scales), queries, tables."""

    def __init__(self, seed, t, lens, new, n_q, n_kv, D, page=16, window=0, T=None, layout="pages", scale=None, qscale=1.5,
                 pad_rows=3, width=None, ps=None):
        g = np.random.default_rng(seed)
        self.t, self.n_q, self.n_kv, self.D, self.page, self.window = t, n_q, n_kv, D, page, window
        self.lens, self.new = np.asarray(lens), np.asarray(new)
        S = self.S = len(self.lens)
        self.T = int(T or max(1, self.new.max()))
        self.scale = D ** -0.5 if scale is None else scale
        used = -(-self.lens // page)
        self.n_pages = int(used.sum()) + 3
        order = g.permutation(self.n_pages)
        self.table = np.full((S, width or max(1, int(used.max()) + 1)), -1)
        at = 0
        for s in range(S):
            self.table[s, :used[s]] = order[at:at + used[s]]
            at += used[s]
        strides = {"pages": (0, 0, 0), "tokens": (page * n_kv * D, D, n_kv * D),
                   "gaps": (n_kv * page * (D + 8) + 16, page * (D + 8), D + 8)}[layout]
        if ps:
            strides = (ps, page * D, D)
        self.strides = strides
        self.ps, self.hs, self.ts = strides[0] or n_kv * page * D, strides[1] or page * D, strides[2] or D
        size = -(-self.n_pages * self.ps // 64) * 64 + 64
        if t == K.TYPE_I8:
            self.kv = torch.randint(-128, 128, (2, size), dtype=torch.int8, device="cuda")
            self.sc = torch.full((2, self.n_pages, n_kv, page), float("nan"), device="cuda")
        else:
            self.kv, self.sc = torch.full((2, size), float("nan"), dtype=DT[t], device="cuda"), None
        self.start = np.concatenate([[0], np.cumsum(self.new)])
        self.rows = []                # each sequence's keys and values in 64 bits: 2, n_kv, len, D
        gen = torch.Generator(device="cuda").manual_seed(seed)
        for s in range(S):
            L = int(self.lens[s])
            x = torch.randn(2, n_kv, L, D, generator=gen, device="cuda")
            x[0] += 2 * (torch.rand(D, generator=gen, device="cuda") < 0.05)
            self.put(s, x)
        self.N = int(self.start[-1]) + pad_rows
        self.q = qscale * torch.randn(self.N, n_q * D + 4, generator=gen, device="cuda")

    def places(self, s):
        L = int(self.lens[s])
        j = np.arange(L)
        return self.table[s][j // self.page], j % self.page

    def put(self, s, x):
        """x: 2 x n_kv x L x D becomes sequence s's keys and values."""
        page, at = self.places(s)
        idx = (page * self.ps + at * self.ts)[None, :, None] + (np.arange(self.n_kv) * self.hs)[:, None, None] + np.arange(self.D)
        idx = torch.from_numpy(idx.reshape(-1)).cuda()
        if self.t == K.TYPE_I8:
            sc = (x.abs().amax(-1) / 127).clamp(min=1e-30)
            qv = torch.round(x / sc.unsqueeze(-1)).clamp(-127, 127).to(torch.int8)
            p, a = torch.from_numpy(page).cuda(), torch.from_numpy(at).cuda()
            for j in range(2):
                self.kv[j][idx] = qv[j].reshape(-1)
                self.sc[j][p, :, a] = sc[j].transpose(0, 1)
            exact = qv.double() * sc.double().unsqueeze(-1)
        else:
            y = x.to(DT[self.t])
            for j in range(2):
                self.kv[j][idx] = y[j].reshape(-1)
            exact = y.double()
        if s < len(self.rows):
            self.rows[s] = exact
        else:
            self.rows.append(exact)

    def shape(self):
        return K.attn_shape(self.S, self.T, self.n_q, self.n_kv, self.D, self.window)

    def cache(self):
        sc = (None, None) if self.sc is None else (self.sc[0].data_ptr(), self.sc[1].data_ptr())
        return K.kv_cache(self.t, self.n_pages, self.page, self.n_kv, self.D, self.kv[0].data_ptr(), self.kv[1].data_ptr(),
                          *sc, *self.strides)

    def device(self):
        if not hasattr(self, "d"):
            self.d = {"table": ints(self.table), "start": ints(self.start), "lens": ints(self.lens),
                      "cached": ints(self.lens - self.new), "new": ints(self.new)}
        return self.d

    def make_list(self):
        d, shape = self.device(), self.shape()
        nb, wb = K.kv_list_bytes(shape), K.paged_attn_workspace_bytes(shape)
        self.list = torch.full((nb,), 123, dtype=torch.uint8, device="cuda")
        self.work = torch.full((max(256, wb),), 255, dtype=torch.uint8, device="cuda")       # NaN
        p = K.kv_plan(self.S, self.page, self.n_pages, d["cached"].data_ptr(), new_ptr=d["new"].data_ptr(), shape=shape,
                      list_ptr=self.list.data_ptr(), list_bytes=nb)
        return p, nb, wb

    def run(self, listed, start=True):
        d = self.device()
        out = torch.full((self.N, self.n_q * self.D + 8), float("nan"), device="cuda")
        nb = wb = 0
        if listed:
            p, nb, wb = self.make_list()
            K.kv_plan_dev(p, st())
        a = K.paged_attn(self.shape(), self.cache(), self.q.data_ptr(), out.data_ptr(), self.N, d["table"].data_ptr(),
                         self.table.shape[1], d["start"].data_ptr() if start else None, d["lens"].data_ptr(), self.scale,
                         list_ptr=self.list.data_ptr() if listed else None, list_bytes=nb, q_stride=self.n_q * self.D + 4,
                         out_stride=self.n_q * self.D + 8)
        K.paged_attn_dev(a, self.work.data_ptr() if listed else None, wb, st())
        torch.cuda.synchronize()
        return out

    def seen(self, s, i):
        """The keys that new token i of sequence s sees."""
        last = int(self.lens[s] - self.new[s]) + i
        lo = max(0, last + 1 - self.window) if self.window else 0
        keys = np.arange(lo, last + 1)
        page = self.table[s][keys // self.page] if len(keys) else keys
        return keys[(page >= 0) & (page < self.n_pages)]

    def check(self, out, skip=()):
        G, D = self.n_q // self.n_kv, self.D
        got = out[:, :self.n_q * D].double().view(self.N, self.n_q, D)
        live = np.zeros(self.N, bool)
        for s in range(self.S):
            if not 1 <= self.new[s] <= self.T:
                continue
            for i in range(int(self.new[s])):
                r = int(self.start[s]) + i
                live[r] = True
                if (s, i) in skip:
                    continue
                keys = torch.from_numpy(self.seen(s, i)).cuda()
                if len(keys) == 0:
                    assert (got[r] == 0).all(), (s, i)
                    continue
                k, v = self.rows[s][0][:, keys], self.rows[s][1][:, keys]
                q = self.q[r, :self.n_q * D].double().view(self.n_kv, G, D) * float(np.float32(self.scale))
                x = torch.matmul(q, k.transpose(1, 2).contiguous())
                X = torch.matmul(q.abs(), k.abs().transpose(1, 2).contiguous())
                p = torch.softmax(x, -1)
                want = torch.matmul(p, v).reshape(self.n_q, D)
                pv = torch.matmul(p, v.abs()).reshape(self.n_q, D)
                e = X.amax(-1) * (2.0 ** -21 + (D + 8) * U) + 4 * U * x.abs().amax(-1)
                tol = pv * (2 * e.reshape(self.n_q, 1) + 2.0 ** -20 + (4 * len(keys) + 200) * U) + 2.0 ** -126
                if self.t != K.TYPE_BF16:
                    e = e + 2.0 ** -38 * q.abs().amax(-1) * k.abs().sum(-1).amax(-1, keepdim=True)
                    top = v.abs().amax((1, 2)).repeat_interleave(G).reshape(self.n_q, 1)
                    tol = pv * (2 * e.reshape(self.n_q, 1) + 2.0 ** -20 + (4 * len(keys) + 200) * U) + \
                        len(keys) * 2.0 ** -34 * top + 2.0 ** -126
                bad = ~((got[r] - want).abs() <= tol)
                assert not bad.any(), (s, i, int(bad.sum()), float((got[r] - want).abs().max()), float(tol.max()))
        rest = out[:, self.n_q * D:]
        assert torch.isnan(rest).all() and torch.isnan(out[torch.from_numpy(~live).cuda()]).all()


def both(c, **kw):
    for listed in (False, True):
        c.check(c.run(listed), **kw)


@pytest.mark.parametrize("t", [K.TYPE_F16, K.TYPE_BF16, K.TYPE_I8])
@pytest.mark.parametrize("n_q,n_kv,D,page", [
    (1, 1, 8, 16), (16, 8, 128, 16), (24, 4, 256, 16), (15, 3, 80, 7), (6, 1, 64, 32), (12, 2, 96, 1), (8, 8, 192, 5),
    (32, 2, 128, 48), (40, 1, 72, 64), (4, 2, 248, 256), (20, 1, 136, 16)])
def test_shapes(t, n_q, n_kv, D, page):
    lens = [1, 2, 15, 16, 17, 31, 33, 64, 100, 129, 300, 1000]
    both(Case(D + page, t, lens, np.ones(len(lens), int), n_q, n_kv, D, page))


@pytest.mark.parametrize("t", [K.TYPE_F16, K.TYPE_BF16, K.TYPE_I8])
@pytest.mark.parametrize("n_q,n_kv,D,page,T", [(24, 4, 256, 16, 8), (16, 8, 128, 16, 5), (15, 3, 80, 7, 3), (8, 1, 64, 32, 64),
                                               (6, 1, 256, 5, 17), (2, 2, 128, 16, 33)])
def test_drafts(t, n_q, n_kv, D, page, T):
    """Several new tokens of a sequence, each seeing itself and what is before it; none, and too many."""
    g = np.random.default_rng(T)
    new = np.concatenate([[T, 1, 0, T], g.integers(1, T + 1, 6), [T + 1, 0]])
    lens = new + np.array([0, 0, 40, 1, 30, 31, 32, 500, 63, 700, 20, 0])
    both(Case(T, t, lens, new, n_q, n_kv, D, page, T=T))


@pytest.mark.parametrize("window", [1, 2, 16, 33, 100, 5000])
@pytest.mark.parametrize("t,D,page", [(K.TYPE_F16, 128, 16), (K.TYPE_BF16, 80, 7), (K.TYPE_I8, 256, 32)])
def test_windows(t, D, page, window):
    new = np.array([1, 4, 3, 1, 4, 2, 1])
    both(Case(window, t, np.array([1, 4, 90, 640, 333, 1500, 64]), new, 6, 2, D, page, window=window))


@pytest.mark.parametrize("t", [K.TYPE_F16, K.TYPE_I8])
@pytest.mark.parametrize("layout", ["tokens", "gaps"])
@pytest.mark.parametrize("page", [3, 16, 80])
def test_layouts(t, layout, page):
    both(Case(page, t, [70, 1, 200, 33], [1, 1, 3, 2], 12, 4, 128, page, layout=layout))


@pytest.mark.parametrize("t,n_q,n_kv,D,page", [(K.TYPE_F16, 24, 4, 256, 16), (K.TYPE_BF16, 16, 8, 128, 32),
                                               (K.TYPE_I8, 8, 1, 64, 16), (K.TYPE_BF16, 6, 2, 80, 7)])
def test_long(t, n_q, n_kv, D, page):
    """One long sequence, and a long one among short ones: split and joined."""
    both(Case(1, t, [20011], [1], n_q, n_kv, D, page))
    both(Case(2, t, [5, 9000, 1, 40, 17, 700], [1, 4, 1, 2, 3, 1], n_q, n_kv, D, page))


def test_many_sequences():
    g = np.random.default_rng(4)
    lens = np.exp(g.uniform(0, np.log(900), 700)).astype(int)
    both(Case(5, K.TYPE_F16, lens, np.ones(700, int), 8, 2, 64))


def test_more_sequences_than_the_plan_has_lanes():
    """Sums over sequences in rounds; short ones, and a few long ones that are split."""
    g = np.random.default_rng(40)
    lens = g.integers(1, 30, 2300)
    lens[[5, 1100, 2299]] = 5000, 3000, 700
    c = Case(41, K.TYPE_F16, lens, np.ones(2300, int), 2, 1, 64)
    c.check(c.run(True))


@pytest.mark.parametrize("lo,hi", [(1e-40, 2e-38), (3e-39, 1e-36), (1e-30, 1e30)])
def test_int8_scales_of_all_sizes(lo, hi):
    """Values' scales below the normal range, and far apart, in either order over the keys."""
    for s1, s2 in ((lo, hi), (hi, lo)):
        c = Case(42, K.TYPE_I8, [1000, 140], [1, 2], 4, 2, 128, qscale=0.3)
        for s in range(2):
            page, at = c.places(s)
            f = np.where(np.arange(len(at)) < len(at) // 2, s1, s2).astype(np.float32)
            p, a = torch.from_numpy(page).cuda(), torch.from_numpy(at).cuda()
            new = torch.from_numpy(f).cuda().unsqueeze(1) * c.sc[1][p, :, a]
            old = c.sc[1][p, :, a]
            c.rows[s][1] *= (new.double() / old.double()).t().unsqueeze(-1)
            c.sc[1][p, :, a] = new
        both(c)


def test_one_row_each_without_offsets():
    c = Case(6, K.TYPE_BF16, [3, 50, 64, 900], [1, 1, 1, 1], 8, 4, 128, pad_rows=0)
    for listed in (False, True):
        c.check(c.run(listed, start=False))


@pytest.mark.parametrize("t", [K.TYPE_F16, K.TYPE_BF16, K.TYPE_I8])
def test_bad_pages_and_short_tables(t):
    """Keys on pages that are none are left out, as those past the table; nothing but such gives zeros."""
    c = Case(7, t, [100, 64, 48, 31, 2000], [1, 3, 2, 1, 4], 6, 2, 128)
    c.table[0, 2] = -1
    c.table[0, 4] = c.n_pages
    c.table[1, 0] = 2 ** 31 - 1
    c.table[2, :] = -5
    c.table[4, 50] = -2 ** 31
    c.table[4, 124] = c.n_pages
    both(c)
    c = Case(8, t, [100, 64, 2000], [1, 1, 2], 6, 2, 128)
    wide = c.table
    c.table = np.ascontiguousarray(wide[:, :70])       # 1120 tokens
    c.seen = lambda s, i, seen=c.seen: (lambda k: k[k < 1120])(_all(c, wide, seen, s, i))
    both(c)


def _all(c, wide, seen, s, i):
    narrow, c.table = c.table, wide
    try:
        return seen(s, i)
    finally:
        c.table = narrow


def test_inconsistent_lengths_see_nothing():
    """A length of 0, or less than its new tokens: the tokens before the first key get zeros."""
    c = Case(9, K.TYPE_F16, [40, 40, 40], [4, 1, 3], 4, 2, 64)
    c.device()["lens"].copy_(ints([2, 0, 40]))
    c.lens = np.array([2, 0, 40])
    c.check(c.run(False))


def test_lengths_of_zero_in_the_list():
    """Sequences whose pages are missing (length 0): zeros."""
    c = Case(10, K.TYPE_F16, [40, 40, 900], [2, 1, 3], 4, 2, 64)
    d = c.device()
    # as a plan without free pages leaves it: no pages held
    d["lens"].copy_(ints([0, 40, 900]))
    c.lens = np.array([0, 40, 900])
    shape = c.shape()
    nb, wb = K.kv_list_bytes(shape), K.paged_attn_workspace_bytes(shape)
    lst, work = torch.empty(nb, dtype=torch.uint8, device="cuda"), torch.empty(max(256, wb), dtype=torch.uint8, device="cuda")
    held, free, n_free, table = ints([0, 3, 57]), ints([0]), ints([0]), d["table"].clone()
    K.kv_plan_dev(K.kv_plan(3, 16, c.n_pages, d["cached"].data_ptr(), new_ptr=d["new"].data_ptr(), held_ptr=held.data_ptr(),
                            table_ptr=table.data_ptr(), table_stride=c.table.shape[1], free_ptr=free.data_ptr(),
                            n_free_ptr=n_free.data_ptr(), shape=shape, list_ptr=lst.data_ptr(), list_bytes=nb), st())
    out = torch.full((c.N, 4 * 64 + 8), float("nan"), device="cuda")
    K.paged_attn_dev(K.paged_attn(shape, c.cache(), c.q.data_ptr(), out.data_ptr(), c.N, table.data_ptr(), c.table.shape[1],
                                  d["start"].data_ptr(), d["lens"].data_ptr(), c.scale, list_ptr=lst.data_ptr(),
                                  list_bytes=nb, q_stride=260, out_stride=264), work.data_ptr(), wb, st())
    torch.cuda.synchronize()
    c.check(out)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("t", [K.TYPE_F16, K.TYPE_BF16])
@pytest.mark.parametrize("n_q", [4, 12])
def test_what_a_token_does_not_see_does_not_reach_it(t, bad, n_q):
    """NaN and infinities in later tokens' keys and values, and before a window."""
    c = Case(11, t, [50, 400], [6, 5], n_q, 2, 128, window=100)
    for s, places in ((0, (46, 48)), (1, (397, 290, 299, 60))):
        x = c.rows[s].float()
        x[:, :, list(places)] = bad
        c.put(s, x)
    # tokens 44.. of 50 and 395.. of 400; the windows start at 0 and 296..300
    skip = {(0, i) for i in range(2, 6)} | {(1, i) for i in (0, 1, 2, 3, 4) if i >= 2 or 296 + i <= 299}
    for listed in (False, True):
        out = c.run(listed)
        c.check(out, skip=skip)
        got = out[:, :n_q * 128]
        if bad != bad:
            for s, i in skip:
                assert torch.isnan(got[c.start[s] + i]).all()


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_scales_of_hidden_keys_do_not_reach_a_token(bad):
    """The same of an int8 cache's scales, of keys, of values and of both."""
    for which in ((0,), (1,), (0, 1)):
        c = Case(24, K.TYPE_I8, [50, 400], [6, 5], 4, 2, 128, window=100)
        for s, places in ((0, (46, 48)), (1, (397, 290, 299, 60))):
            page, at = c.places(s)
            for j in which:
                for e in places:
                    c.sc[j][int(page[e]), :, int(at[e])] = bad
        skip = {(0, i) for i in range(2, 6)} | {(1, i) for i in (0, 1, 2, 3, 4) if i >= 2 or 296 + i <= 299}
        both(c, skip=skip)


def test_infinite_values_that_are_seen():
    """An infinite value gives an infinity in its place; others stay finite."""
    c = Case(12, K.TYPE_F16, [40], [1], 2, 1, 64)
    x = c.rows[0].float()
    x[1, 0, 7, 5] = float("inf")
    x[1, 0, 9, 6] = float("-inf")
    c.put(0, x)
    for listed in (False, True):
        got = c.run(listed)[0, :128].view(2, 64)
        assert (got[:, 5] == float("inf")).all() and (got[:, 6] == float("-inf")).all()
        assert torch.isfinite(got[:, [i for i in range(64) if i not in (5, 6)]]).all()


@pytest.mark.parametrize("t", [K.TYPE_F16, K.TYPE_BF16, K.TYPE_I8])
def test_sizes_of_values(t):
    """Scores of hundreds, scores of one value, a scale of 0 and a negative one, small and large queries."""
    lens, new = [200, 33, 1500], [2, 1, 1]
    both(Case(13, t, lens, new, 8, 2, 128, qscale=60.0))
    both(Case(14, t, lens, new, 8, 2, 128, scale=0.0))
    both(Case(15, t, lens, new, 8, 2, 128, scale=-0.3))
    both(Case(16, t, lens, new, 8, 2, 64, qscale=1e-6))
    both(Case(17, t, lens, new, 8, 2, 64, qscale=1e-6, scale=1e6))
    both(Case(18, t, lens, new, 8, 2, 64, qscale=3e5, scale=1e-5))
    c = Case(19, t, lens, new, 8, 2, 64)
    c.q.zero_()
    c.q[1, :3] = 1e-20                    # a row of few values
    both(c)
    c = Case(20, t, lens, new, 8, 2, 64)
    for s in range(3):
        x = c.rows[s].float()
        x[1] *= 1e-5 if t == K.TYPE_F16 else 1e-30
        c.put(s, x)
    c.q[:, ::7] *= 1e-9
    both(c)


def test_past_32_bits():
    """Pages past 2^32 bytes and 2^32 elements of the cache."""
    c = Case(21, K.TYPE_F16, [40, 17], [1, 2], 4, 1, 128, ps=(1 << 30) + 64)
    both(c)


@pytest.mark.parametrize("lens,new", [([200, 33, 9000], [2, 1, 1]), ([20000, 5], [1, 3])])
@pytest.mark.parametrize("size", [1e27, 3e33, 7e37])
def test_large_bfloat16_values(lens, new, size):
    """Sums of weights up to 2^5 and values near the type's largest pass binary32's range; their quotient does
    not.  One sequence has large values in the last keys only, so that its shares differ in how they are summed."""
    c = Case(25, K.TYPE_BF16, lens, new, 8, 2, 64)
    for s in range(len(lens)):
        x = c.rows[s].float()
        x[1] = (x[1].clamp(-4, 4) * size)
        if s == 0:
            x[1, :, :lens[0] // 2] /= 1e20
        c.put(s, x)
    both(c)


@pytest.mark.parametrize("page", [16, 32, 48, 112, 128])
@pytest.mark.parametrize("t", [K.TYPE_F16, K.TYPE_I8])
def test_long_tables(t, page):
    """Keys past the first 2^24 pages of a table, of which a window hides those before: the same bits as of
    a table of the last pages, with as many keys fewer."""
    c = Case(24, t, [5 * page + 3], [2], 4, 2, 64, page=page, window=2 * page + 5)
    want = c.run(False)
    c.check(want)
    before = (2 ** 31 - 2 ** 17 - 8 * page) // page // 32 * 32 if page > 112 else 2 ** 24
    tail = c.table
    c.table = np.zeros((1, before + tail.shape[1]), np.int32)
    c.table[0, before:] = tail
    c.lens = c.lens + before * page
    del c.d
    assert torch.equal(torch.nan_to_num(want), torch.nan_to_num(c.run(False)))


def test_repeatable_and_equal_in_a_batch():
    """The same bits from call to call, also where sequences are split."""
    c = Case(22, K.TYPE_F16, [9000, 300, 40], [1, 2, 1], 24, 4, 256)
    a = c.run(True)
    for _ in range(3):
        assert torch.equal(torch.nan_to_num(a), torch.nan_to_num(c.run(True)))


def test_captured_and_two_streams():
    """A replayed graph of plan and attention follows lengths and queries; two streams with a list and a
    workspace each give the same bits."""
    c = Case(23, K.TYPE_BF16, [6000, 130, 77, 1], [1, 2, 1, 1], 16, 4, 128)
    full = c.lens.copy()
    d = c.device()
    d["cached"], d["lens_out"] = ints(c.lens - c.new), ints(c.lens)
    p, nb, wb = c.make_list()
    p.lens = d["lens_out"].data_ptr()
    out = torch.full((c.N, 16 * 128 + 8), float("nan"), device="cuda")

    def desc(o, lst):
        return K.paged_attn(c.shape(), c.cache(), c.q.data_ptr(), o.data_ptr(), c.N, d["table"].data_ptr(), c.table.shape[1],
                            d["start"].data_ptr(), d["lens_out"].data_ptr(), c.scale, list_ptr=lst.data_ptr(), list_bytes=nb,
                            q_stride=16 * 128 + 4, out_stride=16 * 128 + 8)
    a = desc(out, c.list)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        K.kv_plan_dev(p, st())
        for _ in range(3):
            K.paged_attn_dev(a, c.work.data_ptr(), wb, st())
    rows = c.rows
    for i in range(4):
        c.lens = np.maximum(c.new, full - i * np.array([997, 31, 20, 0]))
        c.rows = [r[:, :, :n] for r, n in zip(rows, c.lens)]
        d["cached"].copy_(ints(c.lens - c.new))
        c.q.mul_(-1.1)
        out.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        c.check(out)
        eager = torch.full_like(out, float("nan"))
        K.kv_plan_dev(p, st())
        K.paged_attn_dev(desc(eager, c.list), c.work.data_ptr(), wb, st())
        torch.cuda.synchronize()
        assert torch.equal(torch.nan_to_num(eager), torch.nan_to_num(out))
    # two streams at once
    outs, lists, works = ([torch.full_like(out, float("nan")) for _ in range(2)], [c.list.clone() for _ in range(2)],
                          [torch.empty_like(c.work) for _ in range(2)])
    side = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(10):
        for j in range(2):
            K.paged_attn_dev(desc(outs[j], lists[j]), works[j].data_ptr(), wb, side[j].cuda_stream)
    torch.cuda.synchronize()
    for o in outs:
        assert torch.equal(torch.nan_to_num(o), torch.nan_to_num(eager))


@pytest.mark.parametrize("t,listed", [(K.TYPE_F16, True), (K.TYPE_BF16, False), (K.TYPE_I8, True)])
def test_decode_steps(t, listed):
    """Plan, store and attention together as one captured step, replayed while the sequences grow: prompt
    chunks first, then drafted tokens of which some are taken back, against attention over all rows so far."""
    S, T, n_q, n_kv, D, page, width, steps = 5, 4, 6, 2, 64, 8, 40, 14
    N, wide, n_pages = S * T, (n_q + 2 * n_kv) * D, 90
    g = np.random.default_rng(30)
    kv = torch.full((2, n_pages, n_kv, page, D), 9 if t == K.TYPE_I8 else float("nan"), dtype=DT[t], device="cuda")
    sc = torch.full((2, n_pages, n_kv, page), float("nan"), device="cuda") if t == K.TYPE_I8 else None
    i = {k: ints(np.zeros(n)) for k, n in (("cached", S), ("new", S), ("held", S), ("n_free", 1), ("start", S + 1),
                                          ("lens", S), ("pos", N), ("slot", N), ("short", 1))}
    table, free = ints(np.full((S, width), -1)), ints(g.permutation(n_pages))
    i["n_free"].fill_(n_pages)
    x, q, out = (torch.zeros(N, wide, device="cuda"), torch.zeros(N, n_q * D, device="cuda"),
                 torch.zeros(N, n_q * D, device="cuda"))
    freq = torch.from_numpy((1e4 ** (-np.arange(D // 2) / (D // 2))).astype(np.float32)).cuda()
    shape = K.attn_shape(S, T, n_q, n_kv, D)
    nb, wb = K.kv_list_bytes(shape), K.paged_attn_workspace_bytes(shape)
    lst, work = torch.empty(nb, dtype=torch.uint8, device="cuda"), torch.empty(max(256, wb), dtype=torch.uint8, device="cuda")
    p = K.kv_plan(S, page, n_pages, i["cached"].data_ptr(), new_ptr=i["new"].data_ptr(), held_ptr=i["held"].data_ptr(),
                  table_ptr=table.data_ptr(), table_stride=width, free_ptr=free.data_ptr(), n_free_ptr=i["n_free"].data_ptr(),
                  held_out_ptr=i["held"].data_ptr(), n_free_out_ptr=i["n_free"].data_ptr(), start_ptr=i["start"].data_ptr(),
                  lens_ptr=i["lens"].data_ptr(), N=N, pos_ptr=i["pos"].data_ptr(), slot_ptr=i["slot"].data_ptr(),
                  short_ptr=i["short"].data_ptr(), shape=shape if listed else None,
                  list_ptr=lst.data_ptr() if listed else None, list_bytes=nb if listed else 0)
    cache = K.kv_cache(t, n_pages, page, n_kv, D, kv[0].data_ptr(), kv[1].data_ptr(),
                       None if sc is None else sc[0].data_ptr(), None if sc is None else sc[1].data_ptr())
    a = K.kv_store(cache, N, i["slot"].data_ptr(), x.data_ptr() + 4 * n_q * D, x.data_ptr() + 4 * (n_q + n_kv) * D,
                   k_stride=wide, v_stride=wide, n_tokens_ptr=i["start"].data_ptr() + 4 * S, pos_ptr=i["pos"].data_ptr(),
                   rot=D, freq_ptr=freq.data_ptr(), n_q=n_q, q_ptr=x.data_ptr(), q_stride=wide, q_out_ptr=q.data_ptr())
    b = K.paged_attn(shape, cache, q.data_ptr(), out.data_ptr(), N, table.data_ptr(), width, i["start"].data_ptr(),
                     i["lens"].data_ptr(), D ** -0.5, list_ptr=lst.data_ptr() if listed else None, list_bytes=nb)

    def step():
        K.kv_plan_dev(p, st())
        K.kv_store_dev(a, st())
        K.paged_attn_dev(b, work.data_ptr() if listed else None, wb, st())
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        step()
    cached = np.zeros(S, int)
    past = [np.zeros((0, 2 * n_kv, D)) for _ in range(S)]        # rotated keys and values of each sequence
    for n in range(steps):
        new = g.integers(0, T + 1, S) if n else np.full(S, T)
        i["cached"].copy_(ints(cached))
        i["new"].copy_(ints(new))
        rows = g.standard_normal((N, wide)).astype(np.float32)
        x.copy_(torch.from_numpy(rows))
        out.fill_(float("nan"))
        torch.cuda.synchronize()
        if n % 4 == 3:
            step()
        else:
            graph.replay()
        torch.cuda.synchronize()
        assert i["short"].item() == 0 and np.array_equal(i["lens"].cpu().numpy(), cached + new)
        got, r = out.cpu().numpy().reshape(N, n_q, D), 0
        for s in range(S):
            for e in range(new[s]):
                y = rows[r].reshape(n_q + 2 * n_kv, D).astype(np.float64)
                ang = (cached[s] + e) * freq.cpu().numpy().astype(np.float64)
                u, v = y[:n_q + n_kv, :D // 2].copy(), y[:n_q + n_kv, D // 2:].copy()
                y[:n_q + n_kv, :D // 2], y[:n_q + n_kv, D // 2:] = (u * np.cos(ang) - v * np.sin(ang),
                                                                 v * np.cos(ang) + u * np.sin(ang))
                past[s] = np.concatenate([past[s], y[n_q:][None]])
                k, val = past[s][:, :n_kv].repeat(n_q // n_kv, 1), past[s][:, n_kv:].repeat(n_q // n_kv, 1)
                sco = np.einsum("hd,lhd->hl", y[:n_q], k) * D ** -0.5
                w = np.exp(sco - sco.max(1, keepdims=True))
                w /= w.sum(1, keepdims=True)
                want = np.einsum("hl,lhd->hd", w, val)
                # a rounding of the cache, h of a key's and a value's magnitude (half a step of the type;
                # of int8, of the row's largest), moves a score by h X, and the result by 2 h X + h of p|v|
                h = {K.TYPE_F16: 2.0 ** -11, K.TYPE_BF16: 2.0 ** -8, K.TYPE_I8: 0.51 / 127}[t]
                if t == K.TYPE_I8:
                    X = np.abs(y[:n_q]).sum(1)[:, None] * np.abs(k).max(2).max(0) [:, None] * D ** -0.5
                    V = np.abs(val).max(2).max(0)[:, None]
                else:
                    X = (np.einsum("hd,lhd->hl", np.abs(y[:n_q]), np.abs(k)) * D ** -0.5).max(1)[:, None]
                    V = np.einsum("hl,lhd->hd", w, np.abs(val))
                tol = h * V + np.einsum("hl,lhd->hd", w, np.abs(val)) * np.expm1(2 * h * X) + 1e-4 * V
                assert (np.abs(got[r] - want) <= tol).all(), (n, s, e)
                r += 1
        assert np.isnan(got[r:]).all()
        # of the drafted tokens some are taken back
        keep = np.where(new > 0, new - (g.random(S) < 0.5) * (new > 1), 0)
        for s in range(S):
            past[s] = past[s][:cached[s] + keep[s]]
        cached = cached + keep


def scale_values(c, s, keys, f):
    """The value scales of these keys of sequence s times f (one factor, or one a key)."""
    page, at = c.places(s)
    for e, x in zip(keys, np.broadcast_to(f, len(keys))):
        old = c.sc[1][int(page[e]), :, int(at[e])].clone()
        new = old * float(x)
        c.sc[1][int(page[e]), :, int(at[e])] = new
        c.rows[s][1][:, e] *= (new.double() / old.double()).unsqueeze(-1)


@pytest.mark.parametrize("size", [1e5, 1e10, 1e30])
@pytest.mark.parametrize("n_q,n_kv,D,page", [(4, 2, 128, 16), (12, 2, 80, 7), (2, 1, 256, 32)])
def test_finite_scales_of_hidden_keys_do_not_reach_a_token(n_q, n_kv, D, page, size):
    """Large value scales of later tokens and of tokens before a window: the bound knows only those that are seen."""
    c = Case(26, K.TYPE_I8, [50, 400], [6, 5], n_q, n_kv, D, page, window=100)
    for s, places in ((0, (46, 48)), (1, (397, 290, 299, 60))):
        scale_values(c, s, places, size)
    both(c)


def check_int8(c, out):
    """The module's bound with the loss of an int8 cache's weights taken at what they multiply.  A weight times
    its value's scale is two binary16 numbers of a power of two that puts the row's largest such product from
    2^10 on, so that 2^-25 / 2^10 = 2^-35 of that one goes missing at most, times 128: L 2^-28 max p s in all."""
    G, D = c.n_q // c.n_kv, c.D
    got = out[:, :c.n_q * D].double().view(c.N, c.n_q, D)
    for s in range(c.S):
        page, at = c.places(s)
        p_, a_ = torch.from_numpy(page).cuda(), torch.from_numpy(at).cuda()
        scales = c.sc[1][p_, :, a_].double().t().abs()
        for i in range(int(c.new[s])):
            r = int(c.start[s]) + i
            keys = torch.from_numpy(c.seen(s, i)).cuda()
            k, v = c.rows[s][0][:, keys], c.rows[s][1][:, keys]
            q = c.q[r, :c.n_q * D].double().view(c.n_kv, G, D) * float(np.float32(c.scale))
            x = torch.matmul(q, k.transpose(1, 2).contiguous())
            X = torch.matmul(q.abs(), k.abs().transpose(1, 2).contiguous())
            p = torch.softmax(x, -1)
            want, pv = torch.matmul(p, v).reshape(c.n_q, D), torch.matmul(p, v.abs()).reshape(c.n_q, D)
            e = X.amax(-1) * (2.0 ** -21 + (D + 8) * U) + 4 * U * x.abs().amax(-1) + \
                2.0 ** -38 * q.abs().amax(-1) * k.abs().sum(-1).amax(-1, keepdim=True)
            ps = (p * scales[:, keys].unsqueeze(1)).amax(-1).reshape(c.n_q, 1)
            tol = pv * (2 * e.reshape(c.n_q, 1) + 2.0 ** -20 + (4 * len(keys) + 200) * U) + len(keys) * 2.0 ** -28 * ps + 2.0 ** -126
            bad = ~((got[r] - want).abs() <= tol)
            assert not bad.any(), (s, i, int(bad.sum()), float((got[r] - want).abs().max()), float(tol.max()))


def steer(c, scores):
    """Keys become multiples of one vector, queries all ones, so that sequence s's scores are those given."""
    c.q.fill_(1.0)
    g = torch.Generator(device="cuda").manual_seed(27)
    for s, x in enumerate(scores):
        L = int(c.lens[s])
        y = torch.randn(2, c.n_kv, L, c.D, generator=g, device="cuda")
        y[0] = (torch.from_numpy(np.asarray(x, dtype=np.float32)).cuda() / (c.D * c.scale)).view(1, L, 1)
        c.put(s, y)


@pytest.mark.parametrize("size", [2.0 ** 30, 2.0 ** 40, 2.0 ** 70, 2.0 ** 100])
@pytest.mark.parametrize("D,page", [(128, 16), (80, 7), (256, 32), (64, 16)])
def test_int8_scales_under_small_weights(D, page, size):
    """Values of large scales whose keys have scores of -50 beside others of about 0: first, last, a step of keys
    at once, and before a window, where the maximum moves past them."""
    lens = [40, 700, 300, 3000]
    at = [[3], [0, 699], list(range(32)), list(range(64, 96)) + [2999]]
    c = Case(28, K.TYPE_I8, lens, [1, 2, 1, 3], 6, 2, D, page)
    g = np.random.default_rng(29)
    scores = [0.3 * g.standard_normal(n) for n in lens]
    for x, j in zip(scores, at):
        x[j] = -50.0
    steer(c, scores)
    for s in range(4):
        scale_values(c, s, at[s], size)
    for listed in (False, True):
        check_int8(c, c.run(listed))


@pytest.mark.parametrize("T", [1, 5])
@pytest.mark.parametrize("D,page", [(128, 16), (72, 5), (256, 16)])
def test_int8_scales_of_any_size_under_any_weight(D, page, T):
    """Scores of -40 to 40 and scales from 2^-50 to 2^50, in any order, rising and falling against each other."""
    lens = [90, 33, 500, 6000, 400, 400]
    c = Case(30, K.TYPE_I8, lens, [1, 1, T, T, T, T], 4, 2, D, page, window=350)
    g = np.random.default_rng(31)
    scores, scales = [g.uniform(-40, 40, n) for n in lens], [2.0 ** g.uniform(-50, 50, n) for n in lens]
    scores[4], scales[4] = np.linspace(-60, 60, 400), 2.0 ** np.linspace(80, -80, 400)
    scores[5], scales[5] = np.linspace(60, -60, 400), 2.0 ** np.linspace(-80, 80, 400)
    steer(c, scores)
    for s, n in enumerate(lens):
        scale_values(c, s, range(n), scales[s])
    for listed in (False, True):
        check_int8(c, c.run(listed))


@pytest.mark.parametrize("lens,new", [([200, 33, 9000], [2, 1, 1]), ([20000, 5], [1, 3])])
@pytest.mark.parametrize("size", [1e27, 3e33, 7e37])
def test_large_int8_scales(lens, new, size):
    """Sums of weights and values of scales near binary32's largest pass its range; their quotient does not.  One
    sequence has large values in the last keys only, so that its shares differ in how they are summed."""
    c = Case(32, K.TYPE_I8, lens, new, 8, 2, 64)
    for s in range(len(lens)):
        x = c.rows[s].float()
        x[1] = x[1].clamp(-4, 4) * size
        if s == 0:
            x[1, :, :lens[0] // 2] /= 1e20
        c.put(s, x)
    for listed in (False, True):
        out = c.run(listed)
        c.check(out)
        check_int8(c, out)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf"), 3e38])
@pytest.mark.parametrize("n_q,D,page", [(4, 128, 16), (12, 80, 7), (2, 256, 16)])
def test_hidden_values_do_not_cost_small_ones_bits(n_q, D, page, bad):
    """bfloat16 values of 1e-30 beside infinities, NaN and values near the largest that tokens do not see."""
    c = Case(33, K.TYPE_BF16, [50, 400], [6, 5], n_q, 2, D, page, window=100)
    for s, places in ((0, (46, 48)), (1, (397, 290, 299, 60))):
        x = c.rows[s].float()
        x[1] *= 1e-30
        x[1][:, list(places)] = bad
        c.put(s, x)
    # tokens 44.. of 50 and 395.. of 400; the windows start at 0 and 296..300
    skip = {(0, i) for i in range(2, 6)} | {(1, i) for i in (0, 1, 2, 3, 4) if i >= 2 or 296 + i <= 299}
    both(c, skip=skip if not bad == 3e38 else ())


@pytest.mark.parametrize("t", [K.TYPE_F16, K.TYPE_BF16])
@pytest.mark.parametrize("n_q,n_kv,D,page,T,window", [(4, 2, 128, 16, 4, 0), (24, 2, 256, 16, 5, 90), (15, 3, 80, 7, 3, 40),
                                                      (2, 2, 64, 32, 1, 0), (33, 1, 72, 5, 9, 500), (6, 1, 248, 48, 7, 1)])
def test_infinities_and_nan_anywhere(t, n_q, n_kv, D, page, T, window):
    """Values that are no numbers in places far apart: those that a token sees give an infinity, or NaN of NaN or of
    both signs, in their place of the row; the others are within the bound."""
    lens = [T, 33 + T, 260, 5000]
    c = Case(34, t, lens, [T] * 4, n_q, n_kv, D, page, window=window)
    g = np.random.default_rng(35)
    for s, n in enumerate(lens):
        x = c.rows[s].float()
        for e in range(12):
            x[1, g.integers(n_kv), g.choice([0, n // 3, n - 1, n - 1 - g.integers(T), g.integers(n)]), g.integers(D)] = float(
                g.choice(["inf", "-inf", "nan"]))
        c.put(s, x)
    special = [r[1].clone() for r in c.rows]
    for r in c.rows:
        r[1] = torch.nan_to_num(r[1], 0.0, 0.0, 0.0)
    for listed in (False, True):
        out = c.run(listed)
        for s, n in enumerate(lens):
            for i in range(T):
                keys, r = torch.from_numpy(c.seen(s, i)).cuda(), int(c.start[s]) + i
                v = special[s][:, keys]
                y = torch.where(torch.isfinite(v), torch.zeros_like(v), v).sum(1)         # inf - inf and NaN: NaN
                y = y.repeat_interleave(n_q // n_kv, 0).reshape(-1)
                got, odd = out[r, :n_q * D], y != 0
                assert torch.equal(torch.nan_to_num(got[odd].double(), 1e300), torch.nan_to_num(y[odd], 1e300)), (s, i)
                # (in the others the sums of finite values: here those take the places of these as well)
                q = c.q[r, :n_q * D].double().view(n_kv, n_q // n_kv, D) * float(np.float32(c.scale))
                x = torch.matmul(q, c.rows[s][0][:, keys].transpose(1, 2).contiguous())
                got[odd] = torch.matmul(torch.softmax(x, -1), c.rows[s][1][:, keys]).reshape(-1)[odd].float()
        c.check(out)


def test_as_many_blocks_of_rows_as_a_launch_takes():
    """2^22 workgroups are a call without a list; the list of as many sequences would have one item more."""
    c = Case(37, K.TYPE_F16, np.arange(1024) % 40 + 1, np.ones(1024, int), 1024, 1, 8, T=64)
    c.check(c.run(False))
    with pytest.raises(RuntimeError, match="too many"):
        K.kv_list_bytes(c.shape())
    c.T, c.S = 64, 1025
    with pytest.raises(RuntimeError, match="too many"):
        c.run(False)


@pytest.mark.parametrize("t,S,T,n_q,n_kv,D,page", [(K.TYPE_F16, 2, 64, 1024, 1, 8, 16), (K.TYPE_I8, 3, 64, 300, 1, 64, 16),
                                                   (K.TYPE_BF16, 2, 50, 700, 2, 16, 7)])
def test_thousands_of_rows_of_one_head(t, S, T, n_q, n_kv, D, page):
    """64 new tokens of many heads over one head of keys: up to 4096 blocks of rows."""
    both(Case(36, t, [90, 700, 64][:S], [T, T - 1, 1][:S], n_q, n_kv, D, page, T=T))


def test_a_sequence_alone_and_in_a_batch():
    """The same keys and queries, whose shares are others alone than in a batch: within the bound both ways."""
    c = Case(38, K.TYPE_F16, [9000, 300, 40], [1, 2, 1], 24, 4, 256)
    c.check(c.run(True))
    for s in range(3):
        one, r = copy.copy(c), int(c.start[s])
        del one.d
        one.S, one.N, one.rows = 1, int(c.new[s]), c.rows[s:s + 1]
        one.lens, one.new, one.table = c.lens[s:s + 1], c.new[s:s + 1], c.table[s:s + 1]
        one.start, one.q = np.array([0, c.new[s]]), c.q[r:r + one.N].clone()
        both(one)
