"""Block tables and slots against a sequential restatement, rotation and store
against the formula in 64 bits.

Bounds of the rotation: binary64 products and a sum rounded once to binary32, so
half a step, 2^-24 |y|, and the binary64 errors of angle, sine, cosine, products
and sum: at most 2^-50 (|a| + |b|) for |angle| < 2^21 (the angle is rounded once, off by
2^-53 of its value, which is below 2^-32 of a turn's sine there: 2^-32 (|a| + |b|) at
2^21, and 2^-53 |angle| (|a| + |b|) in general).  The rounding to the cache's type of
that binary32 value: half a step of the type more, from the exact value."""
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


def ints(a):
    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).cuda()


# ------------------------------------------------------------------ plan

def planned(cached, new, held, table, free, n_free, page, n_pages):
    """Sequence after sequence."""
    table, width, free = table.copy(), table.shape[1], list(free[:max(0, n_free)])
    out = {"start": [0], "lens": [], "held": [], "pos": [], "slot": [], "short": 0}
    wanted, room = 0, len(free)
    for s in range(len(cached)):
        c, n = max(0, int(cached[s])), max(0, int(new[s]))
        pages = -(-(c + n) // page)
        h = min(-(-c // page), width) if held is None else min(max(0, int(held[s])), width)
        need = max(0, pages - h) if pages <= width else 0
        wanted += need
        ok = pages <= width and (need == 0 or wanted <= room)
        if ok:
            for b in range(h, h + need):
                table[s, b] = free.pop()
            h += need
        for p in range(c, c + n):
            out["pos"].append(p)
            b = table[s, p // page] if ok else -1
            out["slot"].append(b * page + p % page if 0 <= b < n_pages else -1)
        out["start"].append(out["start"][-1] + n)
        out["lens"].append(c + n if ok else 0)
        out["held"].append(h)
        out["short"] += not ok
    return dict(out, table=table, n_free=len(free))


def run_plan(cached, new, held, table, free, n_free, page, n_pages, N=None, in_place=False, shape=None):
    S, total = len(cached), int(np.maximum(new, 0).sum())
    N = total if N is None else N
    d = {"cached": ints(cached), "new": ints(new), "held": None if held is None else ints(held), "table": ints(table),
         "free": ints(free), "n_free": ints([n_free])}
    o = {"held": torch.full((S + 2,), -7, dtype=torch.int32, device="cuda"), "n_free": ints([-7, -7]),
         "start": torch.full((S + 3,), -7, dtype=torch.int32, device="cuda"),
         "lens": torch.full((S + 2,), -7, dtype=torch.int32, device="cuda"),
         "pos": torch.full((N + 5,), -7, dtype=torch.int32, device="cuda"),
         "slot": torch.full((N + 5,), -7, dtype=torch.int32, device="cuda"), "short": ints([-7, -7])}
    if in_place:
        o["n_free"], o["held"] = d["n_free"], d["held"]
    nb = 0 if shape is None else K.kv_list_bytes(shape)
    lst = None if shape is None else torch.full((nb // 4 + 8,), -7, dtype=torch.int32, device="cuda")
    p = K.kv_plan(S, page, n_pages, d["cached"].data_ptr(), new_ptr=d["new"].data_ptr(),
                  held_ptr=None if held is None else d["held"].data_ptr(), table_ptr=d["table"].data_ptr(),
                  table_stride=table.shape[1], free_ptr=d["free"].data_ptr(), n_free_ptr=d["n_free"].data_ptr(),
                  held_out_ptr=o["held"].data_ptr(), n_free_out_ptr=o["n_free"].data_ptr(),
                  start_ptr=o["start"].data_ptr(), lens_ptr=o["lens"].data_ptr(), N=N,
                  pos_ptr=o["pos"].data_ptr() if N else None, slot_ptr=o["slot"].data_ptr() if N else None,
                  short_ptr=o["short"].data_ptr(), shape=shape, list_ptr=None if lst is None else lst.data_ptr(),
                  list_bytes=nb)
    K.kv_plan_dev(p, st())
    torch.cuda.synchronize()
    return d, {k: v.cpu().numpy() for k, v in o.items()}, lst


def check_plan(d, o, w, S, N, in_place=False):
    total = w["start"][-1]
    N = min(N, total)
    assert np.array_equal(d["table"].cpu().numpy(), w["table"])
    assert o["n_free"][0] == w["n_free"] and o["short"][0] == w["short"] and o["short"][1] == -7
    assert np.array_equal(o["start"][:S + 1], w["start"]) and (o["start"][S + 1:] == -7).all()
    for k, n in (("lens", S), ("held", S), ("pos", N), ("slot", N)):
        assert np.array_equal(o[k][:n], np.array(w[k])[:n]), k
        if not (in_place and k == "held"):
            assert (o[k][n:] == -7).all(), k


def setup(seed, S, page, longest, most_new, spare=1.0, held_mode="given", narrow=False):
    g = np.random.default_rng(seed)
    new = g.integers(0, most_new + 1, S)
    cached = g.integers(0, longest + 1, S) * (g.random(S) < 0.9)
    held = -(-cached // page)
    if held_mode == "given":
        held = held + (g.random(S) < 0.3) * g.integers(0, 4, S)
    pages = -(-(cached + new) // page)
    width = max(1, int(max(held.max(), pages.max())) + (0 if narrow else 2))
    if narrow:
        width = max(1, width * 3 // 4)
    held = np.minimum(held, width)
    need = np.maximum(0, pages - held)
    n_pages = int(held.sum() + need.sum()) + 9
    order = g.permutation(n_pages)
    table, at = np.full((S, width), -1), 0
    for s in range(S):
        table[s, :held[s]] = order[at:at + held[s]]
        at += held[s]
    free = order[at:]
    return cached, new, held if held_mode == "given" else None, table, free, int(min(len(free), need.sum() * spare)), n_pages


@pytest.mark.parametrize("spare", [0.0, 0.5, 1.0])
@pytest.mark.parametrize("S,page,longest,new", [
    (1, 16, 0, 1), (1, 16, 15, 1), (1, 1, 40, 3), (2, 7, 100, 0), (3, 16, 300, 33), (64, 16, 5000, 8), (65, 32, 500, 1),
    (1000, 16, 900, 2), (1024, 5, 60, 3), (1025, 16, 60, 3), (3000, 16, 200, 4), (8, 16, 100, 4096), (2, 65536, 200000, 9)])
def test_plan(S, page, longest, new, spare):
    for mode in ("given", "none"):
        cached, n, held, table, free, n_free, n_pages = setup(S + page, S, page, longest, new, spare, mode)
        w = planned(cached, n, held, table, free, n_free, page, n_pages)
        d, o, _ = run_plan(cached, n, held, table, free, n_free, page, n_pages)
        check_plan(d, o, w, S, 1 << 30)


def test_plan_in_place_and_few_rows():
    """held_out over held, n_free_out over n_free; pos and slot for less than all tokens."""
    a = setup(5, 200, 16, 700, 5, 0.8)
    w = planned(*a[:6], 16, a[6])
    d, o, _ = run_plan(*a[:6], 16, a[6], in_place=True)
    check_plan(d, o, w, 200, 1 << 30, in_place=True)
    d, o, _ = run_plan(*a[:6], 16, a[6], N=131)
    check_plan(d, o, w, 200, 131)


def test_plan_of_narrow_tables():
    a = setup(6, 150, 16, 2000, 40, 1.0, narrow=True)
    w = planned(*a[:6], 16, a[6])
    assert w["short"] > 0
    d, o, _ = run_plan(*a[:6], 16, a[6])
    check_plan(d, o, w, 150, 1 << 30)


def test_plan_of_wrong_numbers():
    """Lengths below 0 count as 0; pages that are none give no slot; no free pages below 0."""
    cached, new = np.array([-5, 3, 40, 16, 20, 31]), np.array([2, -1, 1, 1, 1, 3])
    held = np.array([0, 1, -3, 1, 90, 2])
    table = np.array([[-1] * 4, [5, -1, -1, -1], [-1] * 4, [-9, -1, -1, -1], [3, 1 << 30, 2, 1], [7, 12, -1, -1]])
    free = np.array([0, 1, 2, 3, 4, 99, 6, 8, 9])
    w = planned(cached, new, held, table, free, 9, 16, 12)
    d, o, _ = run_plan(cached, new, held, table, free, 9, 16, 12)
    check_plan(d, o, w, 6, 1 << 30)
    assert (o["slot"][:8] < 12 * 16).all()
    w = planned(cached, new, held, table, free, -4, 16, 12)
    d, o, _ = run_plan(cached, new, held, table, free, -4, 16, 12)
    check_plan(d, o, w, 6, 1 << 30)


def test_plan_without_pages():
    """Only lengths, offsets and positions; one new token each without n_new."""
    S = 300
    cached = np.arange(S) * 3
    d, lens, start, pos = ints(cached), ints(np.zeros(S)), ints(np.zeros(S + 1)), ints(np.zeros(S))
    K.kv_plan_dev(K.kv_plan(S, 16, 1, d.data_ptr(), start_ptr=start.data_ptr(), lens_ptr=lens.data_ptr(), N=S,
                            pos_ptr=pos.data_ptr()), st())
    torch.cuda.synchronize()
    assert np.array_equal(lens.cpu().numpy(), cached + 1) and np.array_equal(pos.cpu().numpy(), cached)
    assert np.array_equal(start.cpu().numpy(), np.arange(S + 1))


@pytest.mark.parametrize("S,T,n_kv,window,longest,new", [
    (1, 1, 8, 0, 40000, 1), (5, 4, 2, 0, 3000, 6), (64, 8, 4, 0, 9000, 8), (64, 8, 4, 700, 9000, 8), (1500, 2, 1, 0, 600, 3),
    (3, 64, 1, 1, 500, 64), (7, 1, 4, 0, 0, 1)])
def test_list(S, T, n_kv, window, longest, new):
    """Each sequence's keys lie in its items, once, in order; nothing is written behind the list."""
    a = setup(S + T, S, 16, longest, new, 0.9)
    shape = K.attn_shape(S, T, n_kv * 2, n_kv, 128, window)
    d, o, lst = run_plan(*a[:6], 16, a[6], shape=shape)
    lst = lst.cpu().numpy()
    assert (lst[-8:] == -7).all()
    count, items = lst[0], lst[8:8 + 8 * lst[0]].reshape(-1, 8)
    n, lens = np.maximum(a[1], 0), o["lens"][:S]
    want = [s for s in range(S) if 1 <= n[s] <= T]
    parts = []
    for s in want:
        lo = max(0, lens[s] - n[s] + 1 - window) & ~31 if window and lens[s] else 0
        mine = items[items[:, 0] == s]
        num = len(mine)
        assert num >= 1
        if num > 1:
            parts += range(mine[0][4], mine[0][4] + num)
        for i, it in enumerate(mine):
            assert it[1] == lo and it[3] == num << 16 | i and (num == 1 or it[4] == mine[0][4])
            assert it[5] == o["start"][s] and it[6] == n[s] and it[7] == lens[s]
            assert it[1] <= it[2] and (it[2] == lens[s]) == (i == num - 1) and it[1] % 32 == 0
            assert num == 1 or it[2] > it[1]
            lo = it[2]
    assert sorted(parts) == list(range(len(parts))) and sum(np.isin(items[:, 0], want)) == count
    if S <= 1024:            # the longer ones first
        assert (np.diff(((items[:, 3] >> 16) > 1).astype(int)) <= 0).all()
    used = 8 + 8 * count
    assert (lst[used:-8] >= -7).all() and ((lst[used:-8] == 0) | (lst[used:-8] == -7)).all()


@pytest.mark.parametrize("S", [3, 1000])
def test_list_of_the_longest_lengths(S):
    """Lengths above 2^30 - 1 count as that; as many keys as a list may have to share out."""
    shape = K.attn_shape(S, 1, 1024, 1024, 128)
    nb = K.kv_list_bytes(shape)
    lst, cached, lens = torch.empty(nb // 4, dtype=torch.int32, device="cuda"), ints(np.full(S, 2 ** 31 - 1)), ints(np.zeros(S))
    K.kv_plan_dev(K.kv_plan(S, 16, 1, cached.data_ptr(), lens_ptr=lens.data_ptr(), shape=shape, list_ptr=lst.data_ptr(),
                            list_bytes=nb), st())
    torch.cuda.synchronize()
    assert (lens == 2 ** 30).all()
    lst = lst.cpu().numpy()
    items = lst[8:8 + 8 * lst[0]].reshape(-1, 8).astype(np.int64)
    assert lst[0] <= S + 1 and sorted(set(items[:, 0])) == list(range(S))
    assert (items[:, 2] - items[:, 1]).sum() == S * 2 ** 30


def test_plan_captured():
    """A replayed graph of the call follows its lengths."""
    S, page = 70, 16
    a = setup(9, S, page, 400, 4)
    cached, new, held, table, free, n_free, n_pages = a
    d = {k: ints(v) for k, v in zip(("cached", "new", "held", "table", "free"), a[:5])}
    n = ints([n_free])
    o = {k: ints(np.zeros(m)) for k, m in (("held", S), ("n_free", 1), ("start", S + 1), ("lens", S), ("pos", 400),
                                          ("slot", 400), ("short", 1))}
    p = K.kv_plan(S, page, n_pages, d["cached"].data_ptr(), new_ptr=d["new"].data_ptr(), held_ptr=d["held"].data_ptr(),
                  table_ptr=d["table"].data_ptr(), table_stride=table.shape[1], free_ptr=d["free"].data_ptr(),
                  n_free_ptr=n.data_ptr(), held_out_ptr=o["held"].data_ptr(), n_free_out_ptr=o["n_free"].data_ptr(),
                  start_ptr=o["start"].data_ptr(), lens_ptr=o["lens"].data_ptr(), N=400, pos_ptr=o["pos"].data_ptr(),
                  slot_ptr=o["slot"].data_ptr(), short_ptr=o["short"].data_ptr())
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        K.kv_plan_dev(p, st())
    for i in range(3):
        now = np.where(np.arange(S) % (i + 2) == 0, 0, new)
        d["new"].copy_(ints(now))
        d["table"].copy_(ints(table))
        w = planned(cached, now, held, table, free, n_free, page, n_pages)
        for v in o.values():
            v.fill_(-7)
        graph.replay()
        torch.cuda.synchronize()
        check_plan(d, {k: np.append(v.cpu().numpy(), -7) for k, v in o.items()}, w, S, 400)


# ----------------------------------------------------------------- store

DT = {K.TYPE_F16: torch.float16, K.TYPE_BF16: torch.bfloat16, K.TYPE_I8: torch.int8}
HALF = {K.TYPE_F16: 2.0 ** -11, K.TYPE_BF16: 2.0 ** -8}


def rotated(x, pos, freq, rot, inter):
    """N x heads x D in 64 bits, and the bound of the binary32 value's error."""
    y = x.astype(np.float64)
    tol = np.zeros_like(y)
    if rot:
        h = rot // 2
        ang = pos.astype(np.float64)[:, None, None] * freq.astype(np.float64)[None, None, :]
        i = np.arange(0, rot, 2) if inter else np.arange(h)
        j = i + (1 if inter else h)
        a, b = y[:, :, i].copy(), y[:, :, j].copy()
        y[:, :, i], y[:, :, j] = a * np.cos(ang) - b * np.sin(ang), b * np.cos(ang) + a * np.sin(ang)
        e = (np.abs(a) + np.abs(b)) * (2.0 ** -50 + 2.0 ** -53 * np.abs(ang))
        tol[:, :, i] = tol[:, :, j] = e
    return y, tol + np.abs(y) * 2.0 ** -24 * (rot > 0)


def store_case(seed, t, N, n_q, n_kv, D, rot, inter, page=16, far=40000, layout="pages", q=True, in_place=False,
               n_tokens=None, dead=True):
    g = np.random.default_rng(seed)
    pad = 4 * int(g.integers(0, 3))
    wide = (n_q + 2 * n_kv) * D + pad
    rows = g.standard_normal((N, wide)).astype(np.float32)
    rows[:, g.random(wide) < 0.02] *= 20
    n_pages = -(-N // page) + 2
    slot = g.permutation(n_pages * page)[:N]
    if dead:
        slot = np.where(g.random(N) < 0.1, g.choice([-1, n_pages * page, -2 ** 31, 2 ** 31 - 1], N), slot)
    pos = g.integers(0, far, N)
    freq = (1e4 ** (-np.arange(max(1, rot // 2)) / max(1, rot // 2))).astype(np.float32)
    strides = {"pages": (0, 0, 0), "tokens": (page * n_kv * D, D, n_kv * D),
               "gaps": (n_kv * page * (D + 8) + 16, page * (D + 8), D + 8)}[layout]
    ps = strides[0] or n_kv * page * D
    fill = 3 if t == K.TYPE_I8 else float("nan")
    kv = torch.full((2, -(-n_pages * ps // 64) * 64 + 64), fill, dtype=DT[t], device="cuda")
    sc = torch.full((2, n_pages, n_kv, page), float("nan"), device="cuda") if t == K.TYPE_I8 else None
    dr, dp, ds, df = torch.from_numpy(rows).cuda(), ints(pos), ints(slot), torch.from_numpy(freq).cuda()
    qo = dr if in_place else torch.full((N, n_q * D + 4), float("nan"), device="cuda")
    nt = None if n_tokens is None else ints([n_tokens])
    c = K.kv_cache(t, n_pages, page, n_kv, D, kv[0].data_ptr(), kv[1].data_ptr(),
                   sc[0].data_ptr() if sc is not None else None, sc[1].data_ptr() if sc is not None else None, *strides)
    a = K.kv_store(c, N, ds.data_ptr(), dr.data_ptr() + 4 * n_q * D, dr.data_ptr() + 4 * (n_q + n_kv) * D, k_stride=wide,
                   v_stride=wide, n_tokens_ptr=None if nt is None else nt.data_ptr(), pos_ptr=dp.data_ptr(), rot=rot,
                   interleaved=inter, freq_ptr=df.data_ptr(), n_q=n_q if q else 0, q_ptr=dr.data_ptr() if q else None,
                   q_stride=wide if q else 0, q_out_ptr=qo.data_ptr() if q else None,
                   q_out_stride=(wide if in_place else n_q * D + 4) if q else 0)
    K.kv_store_dev(a, st())
    torch.cuda.synchronize()
    live = N if n_tokens is None else n_tokens
    x = rows[:, :(n_q + 2 * n_kv) * D].reshape(N, -1, D)
    y, tol = rotated(x[:, :n_q + n_kv], pos, freq, rot, inter)
    # queries
    got = qo.cpu().numpy()
    if q:
        e = np.abs(got[:live, :n_q * D].reshape(live, n_q, D) - y[:live, :n_q])
        assert (e <= tol[:live, :n_q]).all()
        if not in_place:
            assert np.isnan(got[live:]).all() and np.isnan(got[:, n_q * D:]).all()
    if in_place:
        assert np.array_equal(got[:, n_q * D:], rows[:, n_q * D:])
        assert np.array_equal(got[live:], rows[live:])
    # the cache: rows at their slots, everything else as it was
    hs, ts = strides[1] or page * D, strides[2] or D
    want = torch.full_like(kv, fill)
    exact = np.concatenate([y[:, n_q:], x[:, n_q + n_kv:].astype(np.float64)], 1)
    etol = np.concatenate([tol[:, n_q:], 0 * tol[:, n_q:]], 1)
    where = np.nonzero((slot >= 0) & (slot < n_pages * page) & (np.arange(N) < live))[0]
    s = slot[where]
    at = ((s // page) * ps)[:, None, None] + np.arange(n_kv)[None, :, None] * hs + ((s % page) * ts)[:, None, None] + np.arange(D)
    at = torch.from_numpy(at).cuda()
    for j in range(2):
        w = exact[where, j * n_kv:(j + 1) * n_kv]
        wt = etol[where, j * n_kv:(j + 1) * n_kv]
        have = kv[j][at.reshape(-1)].view(at.shape)
        if t == K.TYPE_I8:
            hsc = sc[j].cpu().numpy()[s // page, :, s % page]
            top = np.abs(w).max(-1)
            assert (np.abs(hsc - top / 127) <= top / 127 * 2.0 ** -22 + wt.max(-1)).all()
            # half a step, and what the binary32 value, its scale and their product are off by
            assert (np.abs(have.cpu().numpy() * hsc[..., None].astype(np.float64) - w) <=
                    hsc[..., None] * (0.5 + 2.0 ** -14) + wt).all()
        else:
            e = np.abs(have.double().cpu().numpy() - w)
            assert (e <= np.abs(w) * HALF[t] * (1 + 2.0 ** -10) + wt + 2.0 ** -25).all()
        want[j][at.reshape(-1)] = have.reshape(-1)
    a1, b1 = (kv, want) if t == K.TYPE_I8 else (kv.view(torch.int16), want.view(torch.int16))
    assert torch.equal(a1, b1)
    if sc is not None:
        m = torch.ones(n_pages * page, dtype=torch.bool)
        m[torch.from_numpy(s)] = False
        rest = sc.cpu().permute(0, 1, 3, 2).reshape(2, n_pages * page, n_kv)[:, m]
        assert torch.isnan(rest).all()
    return kv, sc, got


@pytest.mark.parametrize("t", [K.TYPE_F16, K.TYPE_BF16, K.TYPE_I8])
@pytest.mark.parametrize("N,n_q,n_kv,D,rot,inter", [
    (1, 16, 8, 128, 128, False), (1, 24, 4, 256, 64, False), (3, 1, 1, 8, 8, True), (5, 4, 2, 8, 2, False),
    (7, 6, 3, 80, 80, True), (7, 6, 3, 80, 46, False), (64, 16, 8, 128, 128, True), (33, 5, 1, 192, 190, True),
    (33, 5, 1, 192, 96, False), (300, 8, 2, 64, 64, False), (700, 4, 4, 256, 256, True), (20, 3, 3, 96, 0, False),
    (2, 40, 40, 104, 104, False)])
def test_store(t, N, n_q, n_kv, D, rot, inter):
    store_case(N + D + rot, t, N, n_q, n_kv, D, rot, inter)


@pytest.mark.parametrize("t", [K.TYPE_F16, K.TYPE_I8])
@pytest.mark.parametrize("layout", ["tokens", "gaps"])
@pytest.mark.parametrize("page", [1, 5, 48])
def test_store_layouts(t, layout, page):
    store_case(page, t, 61, 6, 3, 72, 40, False, page=page, layout=layout)


def test_store_far_positions_in_place_and_part_of_the_rows():
    store_case(1, K.TYPE_BF16, 50, 8, 2, 128, 128, False, far=2 ** 31 - 1)
    store_case(2, K.TYPE_F16, 50, 8, 2, 128, 128, True, in_place=True)
    store_case(3, K.TYPE_F16, 50, 8, 2, 128, 90, False, in_place=True)
    store_case(4, K.TYPE_I8, 50, 8, 2, 128, 128, False, n_tokens=17)
    store_case(5, K.TYPE_F16, 50, 8, 2, 128, 128, False, n_tokens=0)
    store_case(6, K.TYPE_F16, 50, 0, 2, 128, 64, False, q=False)
    store_case(7, K.TYPE_F16, 600, 4, 2, 64, 64, False, in_place=True)


def test_store_int8_rows_are_the_quantizers():
    """Rows without rotation, bit for bit kq_quantize_x_q8_dev's with a group of the row."""
    N, D = 40, 32
    g = np.random.default_rng(3)
    rows = g.standard_normal((N, 2 * D)).astype(np.float32)
    rows[3, :D] = 0
    rows[4, :D] *= np.float32(1e-40)
    rows[5, D:] *= np.float32(1e30)
    d = torch.from_numpy(rows).cuda()
    kv, sc = torch.zeros(2, 4, 1, 16, D, dtype=torch.int8, device="cuda"), torch.zeros(2, 4, 1, 16, device="cuda")
    slot = ints(np.arange(N))
    c = K.kv_cache(K.TYPE_I8, 4, 16, 1, D, kv[0].data_ptr(), kv[1].data_ptr(), sc[0].data_ptr(), sc[1].data_ptr())
    K.kv_store_dev(K.kv_store(c, N, slot.data_ptr(), d.data_ptr(), d.data_ptr() + 4 * D, k_stride=2 * D, v_stride=2 * D), st())
    for j in range(2):
        x = d[:, j * D:(j + 1) * D].contiguous()
        q, s = torch.empty(N * D, dtype=torch.int8, device="cuda"), torch.empty(N, device="cuda")
        K.quantize_x_q8_dev(x.data_ptr(), N * D, 32, q.data_ptr(), s.data_ptr(), None, st())
        torch.cuda.synchronize()
        assert torch.equal(kv[j].view(-1, D)[:N].reshape(-1), q)
        assert torch.equal(sc[j].view(-1)[:N].view(torch.int32), s.view(torch.int32))


def test_store_special_values():
    """Infinities, NaN, values past binary16 and below its normal range."""
    x = np.zeros((2, 16), np.float32)
    x[0] = [np.inf, -np.inf, np.nan, 65504, 65519, 65520, 1e-8, 6e-8, 3e-8, -0.0, 1e30, -1e30, 1, 2 ** -14, 2 ** -24, 0]
    x[1] = x[0][::-1]
    d = torch.from_numpy(x).cuda()
    for t in (K.TYPE_F16, K.TYPE_BF16):
        kv = torch.zeros(2, 1, 1, 16, 8, dtype=DT[t], device="cuda")
        c = K.kv_cache(t, 1, 16, 1, 8, kv[0].data_ptr(), kv[1].data_ptr())
        slot = ints([2, 5])
        K.kv_store_dev(K.kv_store(c, 2, slot.data_ptr(), d.data_ptr(), d.data_ptr() + 32, k_stride=16, v_stride=16), st())
        torch.cuda.synchronize()
        got = torch.stack([torch.cat([kv[0, 0, 0, i], kv[1, 0, 0, i]]) for i in (2, 5)]).cpu()
        want = torch.from_numpy(x).to(DT[t])
        assert torch.equal(torch.isnan(got), torch.isnan(want))
        assert torch.equal(torch.nan_to_num(got.float()), torch.nan_to_num(want.float()))


def test_store_past_32_bits():
    """Pages whose rows lie past 2^32 bytes and 2^32 elements of the cache."""
    D, page, n_pages, ps = 64, 16, 3, (1 << 31) + 64
    kv = torch.zeros(2, n_pages * ps, dtype=torch.float16, device="cuda")
    g = np.random.default_rng(8)
    x = g.standard_normal((6, 2, D)).astype(np.float32)
    d, slot = torch.from_numpy(x).cuda(), ints([0, 15, 17, 30, 33, 47])
    c = K.kv_cache(K.TYPE_F16, n_pages, page, 1, D, kv[0].data_ptr(), kv[1].data_ptr(), page_stride=ps)
    K.kv_store_dev(K.kv_store(c, 6, slot.data_ptr(), d.data_ptr(), d.data_ptr() + 4 * D, k_stride=2 * D, v_stride=2 * D), st())
    torch.cuda.synchronize()
    for i, s in enumerate(slot.tolist()):
        o = (s // page) * ps + (s % page) * D
        assert torch.equal(kv[:, o:o + D].cpu(), torch.from_numpy(x[i]).half())


def test_store_captured_and_on_another_stream():
    N, n_q, n_kv, D = 24, 8, 2, 128
    g = np.random.default_rng(11)
    x = torch.from_numpy(g.standard_normal((N, (n_q + 2 * n_kv) * D)).astype(np.float32)).cuda()
    kv, q = torch.zeros(2, 3, n_kv, 16, D, dtype=torch.bfloat16, device="cuda"), torch.empty(N, n_q * D, device="cuda")
    pos, slot = ints(np.arange(N) * 37), ints(g.permutation(48)[:N])
    freq = torch.from_numpy((1e4 ** (-np.arange(64) / 64)).astype(np.float32)).cuda()
    wide = (n_q + 2 * n_kv) * D
    c = K.kv_cache(K.TYPE_BF16, 3, 16, n_kv, D, kv[0].data_ptr(), kv[1].data_ptr())
    a = K.kv_store(c, N, slot.data_ptr(), x.data_ptr() + 4 * n_q * D, x.data_ptr() + 4 * (n_q + n_kv) * D, k_stride=wide,
                   v_stride=wide, pos_ptr=pos.data_ptr(), rot=D, freq_ptr=freq.data_ptr(), n_q=n_q, q_ptr=x.data_ptr(),
                   q_stride=wide, q_out_ptr=q.data_ptr())
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        K.kv_store_dev(a, st())
    for i in range(3):
        x.mul_(-1.5)
        kv.zero_(), q.zero_()
        graph.replay()
        torch.cuda.synchronize()
        got = kv.clone(), q.clone()
        kv.zero_(), q.zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            K.kv_store_dev(a, side.cuda_stream)
        torch.cuda.synchronize()
        assert torch.equal(got[0], kv) and torch.equal(got[1], q) and bool((q != 0).any())
