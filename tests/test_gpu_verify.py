"""kq_spec_verify_dev against the rule in 64 bits (numpy, on the CPU): the
tokens are whole numbers and have to be equal.  A binary64 running sum over V
weights is off by at most V 2^-53 of its total; the random u of these seeds lie
further than that from every border (checked, not assumed)."""
import ctypes

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


def softmax(l, it):
    l = l.astype(np.float64)
    with np.errstate(invalid="ignore"):
        e = np.exp((l - np.nanmax(l)) * np.float64(np.float32(it)))
    e = np.where(e > 0, e, 0.0)
    return e / e.sum()


def draw_from(w, u):
    w = np.where(w > 0, w, 0.0)
    if not w.any():
        return -1
    cum = np.cumsum(w)
    at = np.float64(u) * cum[-1]
    over = np.flatnonzero(cum > at)
    if len(over):
        # a border may not lie as near as the running sum's own error
        assert np.abs(cum - at).min() > len(w) * 2.0 ** -52 * cum[-1] or at == 0.0
        return int(over[0])
    return int(np.flatnonzero(w)[-1])


def rule(target, draft, tokens, nd, u, form, it):
    """One sequence."""
    T, V = len(tokens), target.shape[-1]
    n = 0
    if form == "greedy":
        def best(i):
            row = np.where(np.isnan(target[i]), -np.inf, target[i])
            return int(row.argmax()) if (row > -np.inf).any() else -1
        while n < nd and best(n) == tokens[n] >= 0:
            n += 1
        return n, tokens[:n].tolist() + [best(n)] + [-1] * (T - n)

    def dist(row):
        return softmax(row, it) if form == "logits" else np.where(row > 0, row, 0).astype(np.float64)
    while n < nd:
        t, p = tokens[n], dist(target[n])
        if draft is None:
            q = np.zeros(V)
            if 0 <= t < V:
                q[t] = 1.0
        else:
            q = dist(draft[n])
        if not (0 <= t < V and np.float64(u[n]) * q[t] < p[t]):
            r = np.maximum(p - q, 0)
            if draft is None and 0 <= t < V:
                r[t] = 0
            return n, tokens[:n].tolist() + [draw_from(r if (r > 0).any() else p, u[T])] + [-1] * (T - n)
        n += 1
    return n, tokens[:n].tolist() + [draw_from(dist(target[n]), u[T])] + [-1] * (T - n)


def make(S, T, V, form, draft, seed, spread=2.5):
    r = np.random.default_rng(seed + 31 * V + T)
    target = (spread * r.standard_normal((S, T + 1, V))).astype(np.float32)
    d = (target[:, :T] + 0.7 * r.standard_normal((S, T, V))).astype(np.float32)
    tokens = np.zeros((S, T), np.int32)
    for s in range(S):
        for i in range(T):
            tokens[s, i] = r.choice(V, p=softmax(d[s, i], 1.0)) if draft or r.random() < 0.5 else target[s, i].argmax()
    if form == "probs":
        target = np.stack([[softmax(v, 1.0) for v in row] for row in target]).astype(np.float32)
        d = np.stack([[softmax(v, 1.0) for v in row] for row in d]).astype(np.float32).reshape(S, T, V)
    if form == "greedy":
        tokens = np.where(r.random((S, T)) < 0.8, target[:, :T].argmax(-1), tokens).astype(np.int32)
    u = r.random((S, T + 1)).astype(np.float32)
    u[:, :T] *= np.float32(0.7)
    nd = r.integers(0, T + 1, S).astype(np.int32)
    nd[0] = T
    return target, d if draft else None, tokens, nd, u


FLAGS = {"logits": K.VERIFY_LOGITS, "probs": 0, "greedy": K.VERIFY_GREEDY}


def run(target, draft, tokens, nd, u, form, it=1.0, stream=None, row=0):
    """The call on rows `row` elements apart (0: dense), guards around the outputs."""
    S, T = tokens.shape
    V = target.shape[-1]
    row = row or V

    def rows(a, n):
        b = np.full((S, n, row), np.nan, np.float32)
        b[:, :, :V] = a
        return torch.from_numpy(b).cuda()
    dt = rows(target, T + 1)
    dd = rows(draft, T) if draft is not None and T else None
    tk, du = torch.from_numpy(tokens).cuda(), torch.from_numpy(u).cuda()
    dn = torch.from_numpy(nd).cuda() if nd is not None else None
    na = torch.full((S + 4,), -9, dtype=torch.int32, device="cuda")
    out = torch.full((S * (T + 1) + 4,), -9, dtype=torch.int32, device="cuda")
    v = K.spec_verify(S, T, V, FLAGS[form], dt.data_ptr(), tk.data_ptr() if T else None, du.data_ptr(), na.data_ptr(),
                      out.data_ptr(), draft_ptr=dd.data_ptr() if dd is not None else None,
                      n_draft_ptr=dn.data_ptr() if dn is not None else None, inv_temp=it, target_row=row,
                      draft_row=row)
    nb = K.spec_verify_workspace_bytes(v)
    work = torch.full((nb + 256,), 0xA5, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    K.spec_verify_dev(v, work.data_ptr(), nb, st() if stream is None else stream)
    torch.cuda.synchronize()
    assert (na[S:] == -9).all() and (out[S * (T + 1):] == -9).all() and (work[nb:] == 0xA5).all()
    return na[:S].cpu().numpy(), out[:S * (T + 1)].cpu().numpy().reshape(S, T + 1)


def check(target, draft, tokens, nd, u, form, it=1.0, row=0):
    na, out = run(target, draft, tokens, nd, u, form, it, row=row)
    S, T = tokens.shape
    for s in range(S):
        k = T if nd is None else min(max(int(nd[s]), 0), T)
        n, want = rule(target[s], None if draft is None else draft[s], tokens[s], k, u[s], form, it)
        assert na[s] == n and out[s].tolist() == want, (s, k, na[s], n, out[s], want)
    return na


@pytest.mark.parametrize("form", ["logits", "probs", "greedy"])
@pytest.mark.parametrize("draft", [False, True])
@pytest.mark.parametrize("S,T,V", [(1, 0, 1), (1, 1, 1), (2, 1, 2), (3, 0, 50), (4, 4, 63), (5, 3, 1000), (8, 7, 4095),
                                   (3, 2, 4096), (3, 2, 4097), (2, 5, 20001), (2, 3, 151936), (1, 63, 300),
                                   (40, 2, 700)])
def test_rule(S, T, V, form, draft):
    seen = set()
    for seed in range(3):
        na = check(*make(S, T, V, form, draft, seed), form, it=1.25 if seed else 1.0)
        seen |= set(na.tolist())
    print(form, draft, S, T, V, "accepted", sorted(seen), flush=True)


@pytest.mark.parametrize("form", ["logits", "probs", "greedy"])
def test_strides_and_no_lengths(form):
    target, draft, tokens, nd, u = make(3, 4, 777, form, form != "greedy", 7)
    check(target, draft, tokens, None, u, form, row=1001)
    nd[:] = [-5, 99, 2]                       # clamped to 0..T
    check(target, draft, tokens, nd, u, form, row=780)


@pytest.mark.parametrize("draft", [False, True])
@pytest.mark.parametrize("form", ["logits", "probs"])
def test_ends_of_u(form, draft):
    """u = 0 takes the first token with any weight, the largest u below 1 the last ones, u >= 1 and NaN the very last."""
    target, d, tokens, nd, u = make(4, 2, 5000, form, draft, 9)
    nd[:] = 0
    lo = -np.inf if form == "logits" else 0.0
    target[:, :, :3], target[:, :, 4990:] = lo, lo
    u[:, 2] = [0.0, 1.0, 7.0, np.nan]
    na, out = run(target, d, tokens, nd, u, form)
    assert na.tolist() == [0] * 4 and out[:, 0].tolist() == [3, 4989, 4989, 4989]
    u[:, 2] = np.float32(1) - np.float32(2) ** -24
    assert (run(target, d, tokens, nd, u, form)[1][:, 0] >= 4900).all()


@pytest.mark.parametrize("form", ["logits", "probs", "greedy"])
def test_masked_and_odd_rows(form):
    """Rows of which nothing is left, NaN among the values, an infinite logit,
    equal distributions, tokens outside the vocabulary."""
    V = 6000
    target, draft, tokens, nd, u = make(7, 2, V, form, form != "greedy", 11)
    nd[:] = 2
    lo = 0.0 if form == "probs" else -np.inf
    target[0] = lo                            # nothing anywhere
    target[1, :, 100:5000] = np.nan
    target[1, :, 5000:] = lo
    tokens[2] = [V, -1]                       # both outside
    tokens[3] = [-7, V + 100]
    if draft is not None:
        target[4, 0] = draft[4, 0]            # p equals q: everything is accepted below u = 1
        u[4, 0] = np.float32(0.999)
    target[5, 1] = lo
    if form != "probs":
        target[6, 0, 17] = np.inf
    na, out = run(target, draft, tokens, nd, u, form)
    assert na[0] == 0 and out[0].tolist() == [-1, -1, -1]
    assert na[2] == 0 and na[3] == 0 and out[2, 0] >= 0 and out[3, 0] >= 0
    assert (out[1][out[1] >= 0] < 100).all() or na[1] > 0
    if form == "logits":
        assert na[6] == 0 and out[6].tolist() == [-1, -1, -1]
    skip = {6} if form == "logits" else set()
    for s in range(7):
        if s in skip:
            continue
        n, want = rule(target[s], None if draft is None else draft[s], tokens[s], 2, u[s], form, 1.0) \
            if s not in (0, 5) or form != "logits" else (na[s], out[s].tolist())
        assert na[s] == n and out[s].tolist() == want, (s, na[s], n, out[s], want)


@pytest.mark.parametrize("form,draft", [("logits", False), ("logits", True), ("probs", True)])
@pytest.mark.parametrize("S,V", [(300, 20001), (700, 21000)])
def test_many_sequences(form, draft, S, V):
    """Workgroups of two and of six chunks, the last of a row with fewer."""
    check(*make(S, 1, V, form, draft, 17), form)


def test_nothing_left_of_the_difference():
    """u = 1 refuses a token although p equals q: the draw is from p itself."""
    target, draft, tokens, nd, u = make(2, 1, 3000, "probs", True, 12)
    target[:, 0] = draft[:, 0]
    nd[:] = 1
    u[:, 0] = 1.0
    check(target, draft, tokens, nd, u, "probs")
    # a one-hot draft's own token with all the weight
    target[:] = 0
    target[0, 0, 7], target[1, 0, 9] = 1.0, 1.0
    tokens[:, 0] = [7, 9]
    na, out = run(target, None, tokens, nd, u, "probs")
    assert na.tolist() == [0, 0] and out[:, 0].tolist() == [7, 9]


def test_nothing_left_of_the_difference_of_logits():
    """The same with logits: equal rows, and a draft on the only token that has any weight."""
    target, draft, tokens, nd, u = make(2, 1, 3000, "logits", True, 14)
    target[:, 0] = draft[:, 0]
    nd[:] = 1
    u[:, 0] = 1.0
    check(target, draft, tokens, nd, u, "logits")
    target[:, 0] = -np.inf
    target[0, 0, 7], target[1, 0, 2999] = -3.0, 400.0
    tokens[:, 0] = [7, 2999]
    na, out = run(target, None, tokens, nd, u, "logits")
    assert na.tolist() == [0, 0] and out[:, 0].tolist() == [7, 2999]


@pytest.mark.parametrize("draft", [False, True])
@pytest.mark.parametrize("it", [1.0, 0.7, 1e-30, 1e30])
def test_logits_of_any_size(it, draft):
    """Rows of the type's lowest value alone (uniform), rows masked with it, logits
    of which neighbours are far apart, large and tiny factors."""
    V = 5000
    target, d, tokens, nd, u = make(6, 2, V, "logits", draft, 15)
    low = np.finfo(np.float32).min
    nd[:] = 2
    target[0] = low
    target[1, :, 5:] = low
    target[2] = np.float32(1e20)
    target[2, :, 100:] = np.nextafter(np.float32(1e20), np.float32(0))
    target[3, :, 10:4990] = low
    target[3, :, :10] = target[3, :, 4990:] = -low
    target[4] += np.float32(1e6)
    if draft:
        d[1, :, 5:] = low
        d[5] = low
    check(target, d, tokens, nd, u, "logits", it=it)


def test_greedy_ties():
    """Equal maxima, also across chunks and lanes: the lowest token."""
    V = 9000
    target = np.zeros((3, 2, V), np.float32)
    target[0, :, [8999, 4096, 5000]] = 2.0
    target[1, :, [70, 69, 8000]] = 2.0
    tokens = np.array([[4096], [70], [0]], np.int32)
    nd = np.ones(3, np.int32)
    na, out = run(target, None, tokens, nd, np.zeros((3, 2), np.float32), "greedy")
    assert na.tolist() == [1, 0, 1] and out.tolist() == [[4096, 4096], [69, -1], [0, 0]]


def test_distribution_of_the_output():
    """Rejection sampling keeps the target's distribution: the first token of
    65536 / (2 T + 1) independent sequences, chi-squared below its 1 - 1e-9 quantile."""
    from scipy import stats
    V, S = 12, 20000
    r = np.random.default_rng(13)
    p1, q1 = softmax(1.5 * r.standard_normal(V), 1.0), softmax(1.5 * r.standard_normal(V), 1.0)
    target = np.tile(p1.astype(np.float32), (S, 2, 1))
    draft = np.tile(q1.astype(np.float32), (S, 1, 1))
    tokens = r.choice(V, (S, 1), p=q1).astype(np.int32)
    u = r.random((S, 2)).astype(np.float32)
    na, out = run(target, draft, tokens, None, u, "probs")
    got = np.bincount(out[:, 0], minlength=V)
    chi = ((got - S * p1) ** 2 / (S * p1)).sum()
    assert chi < stats.chi2.ppf(1 - 1e-9, V - 1), (chi, got, S * p1)
    assert 0 < na.sum() < S


@pytest.mark.parametrize("form", ["logits", "probs", "greedy"])
def test_captured_and_replayed(form):
    """A graph's replays follow its inputs, with eager calls of other sizes between."""
    S, T, V = 3, 3, 10000
    a = [make(S, T, V, form, form != "greedy", 20 + i) for i in range(3)]
    dev = [torch.from_numpy(v).cuda() if v is not None else None for v in a[0]]
    na = torch.empty(S, dtype=torch.int32, device="cuda")
    out = torch.empty(S, T + 1, dtype=torch.int32, device="cuda")
    v = K.spec_verify(S, T, V, FLAGS[form], dev[0].data_ptr(), dev[2].data_ptr(), dev[4].data_ptr(), na.data_ptr(),
                      out.data_ptr(), draft_ptr=dev[1].data_ptr() if dev[1] is not None else None,
                      n_draft_ptr=dev[3].data_ptr())
    nb = K.spec_verify_workspace_bytes(v)
    work = torch.empty(nb, dtype=torch.uint8, device="cuda")
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        K.spec_verify_dev(v, work.data_ptr(), nb, st())
    for i in (1, 2, 0, 1):
        for d, h in zip(dev, a[i]):
            if d is not None:
                d.copy_(torch.from_numpy(h))
        work.fill_(0xFF if i % 2 else 0)      # nothing is kept there between calls
        graph.replay()
        torch.cuda.synchronize()
        want = run(*a[i], form)
        assert np.array_equal(na.cpu().numpy(), want[0]) and np.array_equal(out.cpu().numpy(), want[1])


def test_two_streams():
    a = [make(4, 3, 30000, "logits", True, 30 + i) for i in range(2)]
    alone = [run(*k, "logits") for k in a]
    side = [torch.cuda.Stream(), torch.cuda.Stream()]
    keep, got = [], []
    for i in (0, 1):
        dev = [torch.from_numpy(v).cuda() for v in a[i]]
        na, out = torch.empty(4, dtype=torch.int32, device="cuda"), torch.empty(4, 4, dtype=torch.int32, device="cuda")
        v = K.spec_verify(4, 3, 30000, K.VERIFY_LOGITS, dev[0].data_ptr(), dev[2].data_ptr(), dev[4].data_ptr(),
                          na.data_ptr(), out.data_ptr(), draft_ptr=dev[1].data_ptr(), n_draft_ptr=dev[3].data_ptr())
        nb = K.spec_verify_workspace_bytes(v)
        keep.append((dev, v, torch.empty(nb, dtype=torch.uint8, device="cuda"), nb))
        got.append((na, out))
    torch.cuda.synchronize()
    for rnd in range(5):
        for i in (0, 1):
            _, v, work, nb = keep[i]
            K.spec_verify_dev(v, work.data_ptr(), nb, side[i].cuda_stream)
    torch.cuda.synchronize()
    for i in (0, 1):
        assert np.array_equal(got[i][0].cpu().numpy(), alone[i][0])
        assert np.array_equal(got[i][1].cpu().numpy(), alone[i][1])


def test_refuses_a_short_workspace():
    target, _, tokens, nd, u = make(2, 2, 100, "logits", False, 1)
    d = [torch.from_numpy(v).cuda() for v in (target, tokens, u)]
    na = torch.full((2,), 5, dtype=torch.int32, device="cuda")
    out = torch.full((2, 3), 5, dtype=torch.int32, device="cuda")
    v = K.spec_verify(2, 2, 100, K.VERIFY_LOGITS, d[0].data_ptr(), d[1].data_ptr(), d[2].data_ptr(), na.data_ptr(),
                      out.data_ptr())
    nb = K.spec_verify_workspace_bytes(v)
    work = torch.empty(nb + 256, dtype=torch.uint8, device="cuda")
    for p, n in ((None, nb), (work.data_ptr(), nb - 1), (work.data_ptr() + 4, nb)):
        assert K.lib().kq_spec_verify_dev(ctypes.byref(v), p, n, st()) == -1
        assert b"workspace" in K.lib().kq_last_error()
    torch.cuda.synchronize()
    assert (na == 5).all() and (out == 5).all()


def test_decode_step():
    """Residual and norm to int8 rows, the 4-bit LM head on them, verification
    of its logits: the whole chain on one stream, against the same in numpy from
    the head's own logits."""
    S, T, H, V, g = 2, 3, 512, 4500, 64
    B = S * (T + 1)
    gen = torch.Generator(device="cuda").manual_seed(3)
    x, r = torch.randn(B, H, generator=gen, device="cuda"), torch.randn(B, H, generator=gen, device="cuda")
    wn = 1 + 0.1 * torch.randn(H, generator=gen, device="cuda")
    q = torch.randint(0, 256, (V, H // 2), generator=gen, device="cuda", dtype=torch.uint8)
    sc = (0.03 + 0.01 * torch.rand(V, H // g, generator=gen, device="cuda")).half()
    xq, xs = torch.empty(B, H, dtype=torch.int8, device="cuda"), torch.empty(B, H // 32, device="cuda")
    sm, logits = torch.empty(B, H, device="cuda"), torch.empty(B, V, device="cuda")
    u = torch.rand(S, T + 1, generator=gen, device="cuda")
    tokens = torch.zeros(S, T, dtype=torch.int32, device="cuda")
    na, out = torch.empty(S, dtype=torch.int32, device="cuda"), torch.empty(S, T + 1, dtype=torch.int32, device="cuda")
    head = K.w4(V, H, g, K.TYPE_F16, q.data_ptr(), sc.data_ptr())
    nb = K.w4_workspace_bytes(head, B, True)
    v = K.spec_verify(S, T, V, K.VERIFY_LOGITS, logits.data_ptr(), tokens.data_ptr(), u.data_ptr(), na.data_ptr(),
                      out.data_ptr())
    vb = K.spec_verify_workspace_bytes(v)
    work = torch.empty(max(nb, vb), dtype=torch.uint8, device="cuda")

    def step():
        K.rmsnorm_dev(K.rmsnorm(B, H, 1e-6, x.data_ptr(), resid_ptr=r.data_ptr(), sum_ptr=sm.data_ptr(),
                                weight_ptr=wn.data_ptr(), group=32, xq_ptr=xq.data_ptr(), xscale_ptr=xs.data_ptr()), st())
        K.w4_gemv_q8_dev(head, xq.data_ptr(), xs.data_ptr(), logits.data_ptr(), B, work.data_ptr(), nb, stream=st())
        K.spec_verify_dev(v, work.data_ptr(), vb, st())
    step()
    torch.cuda.synchronize()
    # the drafts: the likeliest token of some rows, so that some are accepted
    tokens.copy_(logits.view(S, T + 1, V)[:, :T].argmax(-1).to(torch.int32))
    tokens[1, 1] = 5
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        step()
    for i in range(3):
        u.copy_(torch.rand(S, T + 1, generator=gen, device="cuda") * 0.5)
        graph.replay()
        torch.cuda.synchronize()
        l, tk, uu = logits.view(S, T + 1, V).cpu().numpy(), tokens.cpu().numpy(), u.cpu().numpy()
        s = (x + r).double()
        y = s * torch.rsqrt((s * s).mean(1, keepdim=True) + 1e-6) * wn.double()
        w = torch.stack([q & 15, q >> 4], -1).reshape(V, H // g, g).double() - 8
        plain = (y @ (w * sc.double().unsqueeze(-1)).reshape(V, H).t()).view(S, T + 1, V).cpu().numpy()
        # int8 activations: half a step of amax / 127 each, 512 of them, as independent errors
        assert np.sqrt(((l - plain) ** 2).mean()) < 0.02 * np.sqrt((plain ** 2).mean())
        for k in range(S):
            n, want = rule(l[k], None, tk[k], T, uu[k], "logits", 1.0)
            assert na[k].item() == n and out[k].tolist() == want


@pytest.mark.parametrize("form", ["logits", "probs", "greedy"])
def test_rows_past_32_bits(form):
    """Sequences 2^31 elements apart (8 GiB), the draft's rows 2^30."""
    S, T, V = 2, 1, 5000
    target, draft, tokens, nd, u = make(S, T, V, form, form != "greedy", 41)
    nd[:] = T
    far, row = (1 << 31) + 8, 1 << 30
    buf = torch.empty(far + 2 * V, device="cuda")
    for s in range(S):
        for i in range(T + 1):
            buf[s * far + i * V:s * far + (i + 1) * V] = torch.from_numpy(target[s, i]).cuda()
    dbuf = torch.empty(row + V, device="cuda")
    if draft is not None:
        for s in range(S):
            dbuf[s * row:s * row + V] = torch.from_numpy(draft[s, 0]).cuda()
    tk, du = torch.from_numpy(tokens).cuda(), torch.from_numpy(u).cuda()
    na, out = torch.empty(S, dtype=torch.int32, device="cuda"), torch.empty(S, T + 1, dtype=torch.int32, device="cuda")
    v = K.spec_verify(S, T, V, FLAGS[form], buf.data_ptr(), tk.data_ptr(), du.data_ptr(), na.data_ptr(), out.data_ptr(),
                      draft_ptr=dbuf.data_ptr() if draft is not None else None, target_seq=far, draft_seq=row)
    nb = K.spec_verify_workspace_bytes(v)
    work = torch.empty(nb, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    K.spec_verify_dev(v, work.data_ptr(), nb, st())
    torch.cuda.synchronize()
    for s in range(S):
        n, want = rule(target[s], None if draft is None else draft[s], tokens[s], T, u[s], form, 1.0)
        assert na[s].item() == n and out[s].tolist() == want


@pytest.mark.parametrize("form", ["logits", "probs"])
@pytest.mark.parametrize("draft", [False, True])
def test_vocabulary_of_many_chunks(form, draft):
    """More chunks than a wave has lanes: the draw goes over them 64 at a time."""
    r = np.random.default_rng(42)
    S, T, V = 3, 2, 700001
    target = (1.5 * r.standard_normal((S, T + 1, V))).astype(np.float32)
    d = (target[:, :T] + 0.5 * r.standard_normal((S, T, V))).astype(np.float32)
    if form == "probs":
        target = np.stack([[softmax(v, 1.0) for v in row] for row in target]).astype(np.float32)
        d = np.stack([[softmax(v, 1.0) for v in row] for row in d]).astype(np.float32)
    tokens = r.integers(0, V, (S, T)).astype(np.int32)
    u = np.array([[0.9, 0.1, 0.02], [0.5, 0.9, 0.55], [0.9, 0.9, 0.999]], np.float32)
    check(target, d if draft else None, tokens, np.array([2, 0, 1], np.int32), u, form)


@pytest.mark.parametrize("form", ["logits", "probs"])
@pytest.mark.parametrize("draft", [False, True])
def test_u_below_zero(form, draft):
    """u below zero draws the first token with any weight, as u = 0 does."""
    target, d, tokens, nd, u = make(4, 2, 9000, form, draft, 51)
    nd[:] = [0, 2, 0, 2]
    u[:, :2] = [[0, 0], [0, 0], [0, 0], [2, 2]]          # the last refuses its first token
    target[:, :, :4100] = -np.inf if form == "logits" else 0.0
    tokens[:] = [4100, 8000]
    u[:, 2] = [-0.0, -1e-30, -3.0, -np.inf]
    na, out = run(target, d, tokens, nd, u, form)
    assert na.tolist() == [0, 2, 0, 0] if not draft else na[0] == na[2] == na[3] == 0
    for s in range(4):
        n = na[s]
        if form == "logits":
            p = softmax(target[s, n], 1.0)
            q = softmax(d[s, n], 1.0) if draft and n < nd[s] else 0.0
        else:
            p, q = target[s, n].astype(np.float64), d[s, n].astype(np.float64) if draft and n < nd[s] else 0.0
        w = np.maximum(p - q, 0)
        if not draft and n < nd[s]:
            w[tokens[s, n]] = 0
        assert out[s, n] == np.flatnonzero(w)[0]


@pytest.mark.parametrize("draft", [False, True])
def test_empty_row_after_accepted_tokens(draft):
    """Logits of -inf everywhere at the second drafted token, and in the row after the last:
    what lies before is accepted (u = 0), nothing can be drawn there."""
    target, d, tokens, nd, u = make(3, 2, 6000, "logits", draft, 52)
    u[:], nd[:] = 0.0, 2
    u[:, 2] = 0.5
    target[0, 1], target[1, 2], target[2, 1, :] = -np.inf, -np.inf, np.nan
    na, out = run(target, d, tokens, nd, u, "logits")
    assert na.tolist() == [1, 2, 1]
    assert out.tolist() == [[tokens[0, 0], -1, -1], [*tokens[1], -1], [tokens[2, 0], -1, -1]]


@pytest.mark.parametrize("draft", [False, True])
@pytest.mark.parametrize("S,T,V", [(6, 2, 50), (6, 5, 1000), (4, 3, 20001)])
def test_logits_with_their_error(S, T, V, draft):
    """A weight is within 6e-12 of p's (five exponentials of 1.1e-12 on its way, include/kq_gemv.h), so p - q
    within 6e-12 (p + q), and a running sum of it within 1.2e-11, and V 2^-52 of the total: u lies further from
    every border that decides something, and then the tokens are equal."""
    for seed in range(4):
        target, d, tokens, nd, u = make(S, T, V, "logits", draft, 60 + seed)
        for s in range(S):
            n = 0
            while True:
                p = softmax(target[s, n], 1.25)
                if n == nd[s]:
                    w = p
                    break
                t = tokens[s, n]
                q = softmax(d[s, n], 1.25) if draft else np.eye(1, V, t)[0]
                a = np.float64(u[s, n]) * q[t]
                assert abs(a - p[t]) > 6e-12 * (a + p[t])
                if not a < p[t]:
                    w = np.maximum(p - q, 0)
                    break
                n += 1
            cum = np.cumsum(w)
            assert np.abs(cum - np.float64(u[s, T]) * cum[-1]).min() > 2 * 1.2e-11 + V * 2.0 ** -52 * cum[-1]
        check(target, d, tokens, nd, u, "logits", it=1.25)
