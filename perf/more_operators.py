"""Attention over a paged cache of keys and values, as timed cases.

Kinds:

  plan    the block tables, slots and positions of a step's new tokens, from the
          requests' lengths and a list of free pages
  store   rotary embedding of a step's queries and keys, and keys and values into
          their slots of the cache, as binary16, bfloat16, or int8 with a scale per
          token and head
  attn    the attention of one or a few new tokens of each sequence over the cached
          ones, with the list of work that a step makes once for its layers; a pass
          goes over `n` layers' caches, as a decode step does

Sequences' lengths are spread evenly over their logarithm from `lo` to `hi` (the
new tokens included) and come in an order that the seed decides.

`run` computes the operators from elementary torch operations, or, where `own` is
set, calls the library.
"""
import math
import random

import numpy as np
import torch

own = False

DEV = "cuda"
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "i8": torch.int8}


# ------------------------------------------------------------------- cases

def _attn(name, S, n_q, n_kv, D, page, type, lo, hi, T=1, window=0, n=1):
    return {"name": name, "kind": "attn", "S": S, "n_q": n_q, "n_kv": n_kv, "D": D, "page": page, "type": type,
            "lo": lo, "hi": hi, "T": T, "window": window, "n": n}


def _store(name, N, n_q, n_kv, D, rot, inter, page, type, far):
    return {"name": name, "kind": "store", "N": N, "n_q": n_q, "n_kv": n_kv, "D": D, "rot": rot, "inter": inter,
            "page": page, "type": type, "far": far}


def _plan(name, S, page, lo, hi, T, spare=1.0):
    return {"name": name, "kind": "plan", "S": S, "page": page, "lo": lo, "hi": hi, "T": T, "spare": spare}


def listed():
    return [
        # a conversation's first tokens, one stream of a small model: latency
        _attn("attn_s1_40", 1, 16, 8, 128, 16, "f16", 40, 40, n=4),
        # one stream with a long document before it, a 27B-class layer
        _attn("attn_s1_32768", 1, 24, 4, 256, 16, "f16", 32768, 32768, n=2),
        # many streams of all lengths, the largest call
        _attn("attn_s64_ragged", 64, 24, 4, 256, 32, "bf16", 200, 6000),
        # up to eight tokens a stream: drafted ones before they are verified
        _attn("attn_drafts_s8_t8", 8, 24, 4, 256, 16, "f16", 1000, 4000, T=8, n=2),
        # the int8 cache, sixteen streams
        _attn("attn_i8_s16", 16, 16, 8, 128, 16, "i8", 100, 8000, n=4),
        # a sliding window, odd page and head sizes, five queries to a key's head
        _attn("attn_window_odd", 5, 15, 3, 80, 7, "bf16", 90, 5000, T=3, window=1000, n=2),
        # one token of a 27B-class layer, a quarter of each head rotated: latency
        _store("store_n1", 1, 24, 4, 256, 64, False, 16, "f16", 40000),
        # 64 streams into an int8 cache
        _store("store_i8_n64", 64, 16, 8, 128, 128, False, 16, "i8", 40000),
        # a prompt's chunk, neighbouring values in pairs, far positions
        _store("store_n4096", 4096, 16, 8, 128, 128, True, 32, "bf16", 1000000),
        # one stream, one token
        _plan("plan_s1", 1, 16, 1000, 1000, 1),
        # 256 streams with up to four tokens
        _plan("plan_s256_t4", 256, 16, 50, 30000, 4),
        # eight prompts
        _plan("plan_prompts", 8, 16, 500, 4000, 4000),
    ]


MOST_BYTES, MOST_FLOPS = 4.4e8, 3.5e9      # of a drawn case: no more than the largest listed one


def _log(rng, lo, hi):
    return int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))


def _draw(rng):
    kind = rng.choice(["attn", "attn", "attn", "store", "store", "plan"])
    type = rng.choice(["f16", "f16", "bf16", "bf16", "i8"])
    page = rng.choice([1, 5, 7, 16, 16, 16, 32, 32, 48, 64, 256])
    D = rng.choice([64, 64, 80, 96, 128, 128, 128, 192, 256, 256])
    n_kv = rng.choice([1, 2, 3, 4, 4, 8, 8])
    n_q = n_kv * rng.choice([1, 2, 3, 4, 5, 6, 8])
    if kind == "attn":
        hi = _log(rng, 1, 40000)
        return _attn("", _log(rng, 1, 64), n_q, n_kv, D, page, type, _log(rng, 1, hi), hi,
                     T=rng.choice([1, 1, 1, rng.randint(2, 9)]), window=rng.choice([0, 0, 0, _log(rng, 16, 8000)]),
                     n=rng.randint(1, 4))
    if kind == "store":
        rot = rng.choice([0, D, D, D, 2 * rng.randint(1, D // 2), D // 4])
        return _store("", _log(rng, 1, 4096), n_q, n_kv, D, rot, rng.random() < 0.4, page, type, _log(rng, 100, 1000000))
    hi = _log(rng, 1, 30000)
    return _plan("", _log(rng, 1, 300), page, _log(rng, 1, hi), hi, rng.choice([1, 1, rng.randint(2, 9), 1000]),
                 rng.choice([1.0, 1.0, 1.0, 0.5]))


def draw(rng):
    while True:
        c = _draw(rng)
        w = work(c)
        if w["bytes"] <= MOST_BYTES and w["flops"] <= MOST_FLOPS and (c["kind"] != "plan" or _tokens(c) <= 20000):
            # the keys as a padded batch, in 32 bits, have to fit as well
            if c["kind"] != "attn" or 8 * c["S"] * max(_lens(c)[0]) * c["n_kv"] * c["D"] <= 6e9:
                del c["name"]
                return c


def _lens(c):
    """Each sequence's length and how many of its tokens are new."""
    S, T = c["S"], c["T"]
    lens = [round(c["lo"] * (c["hi"] / c["lo"]) ** (i / max(1, S - 1))) for i in range(S)]
    new = [min(n, 1 + (5 * i + T - 1) % T) for i, n in enumerate(lens)]
    if c["kind"] == "plan" and T >= 1000:             # prompts: all of a sequence is new
        new = [min(n, T) for n in lens]
    return lens, new


def _tokens(c):
    return sum(_lens(c)[1])


# ------------------------------------------------------------------- inputs

def _gen(seed, salt):
    return torch.Generator(device=DEV).manual_seed(seed * 1000003 + salt)


def _order(c, seed):
    lens, new = _lens(c)
    at = list(range(c["S"]))
    random.Random(seed * 31 + 7).shuffle(at)
    return np.array([lens[i] for i in at]), np.array([new[i] for i in at])


def _ints(a):
    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).to(DEV)


def _to_cache(x, type):
    """Rows of values as a cache holds them: the type's values, and a scale each for int8."""
    if type != "i8":
        return x.to(TYPES[type]), None
    a = x.abs().amax(-1)
    s = a / torch.full_like(a, 127.0)                 # by a tensor: a scalar divisor becomes a product
    inv = torch.where(s > 0, 1.0 / s, torch.zeros_like(s))
    return torch.clamp(torch.round(x * inv.unsqueeze(-1)), -128, 127).to(torch.int8), s


def _data(c, seed):
    """The case's inputs, from the seed alone."""
    g = np.random.default_rng(seed * 7919 + 3)
    if c["kind"] == "plan":
        lens, new = _order(c, seed)
        S, page = c["S"], c["page"]
        held = -(-(lens - new) // page)
        # some sequences hold a page or two more: tokens that were taken back
        held = held + np.where(g.random(S) < 0.2, g.integers(1, 3, S), 0)
        need = np.maximum(0, -(-lens // page) - held)
        width = int(max(held.max(), (-(-lens // page)).max())) + 2
        pages = g.permutation(int(held.sum() + need.sum()) + 40)
        table = np.full((S, width), -1)
        at = 0
        for s in range(S):
            table[s, :held[s]] = pages[at:at + held[s]]
            at += held[s]
        free = pages[at:]
        n_free = len(free) if c["spare"] >= 1 else int(need.sum() * c["spare"])
        return {"cached": _ints(lens - new), "new": _ints(new), "held": _ints(held), "table": _ints(table),
                "free": _ints(free), "n_free": _ints([n_free]), "n_pages": len(pages), "N": int(new.sum())}
    n_kv, n_q, D, page, type = c["n_kv"], c["n_q"], c["D"], c["page"], c["type"]
    gen = _gen(seed, 1)
    if c["kind"] == "store":
        N = c["N"]
        pages = -(-N // page) + 3 + N // (8 * page)
        slot = g.permutation(pages * page)[:N]
        slot = np.where(g.random(N) < 0.02, -1, slot)          # padding of a batch
        rows = torch.randn(N, (n_q + 2 * n_kv) * D, generator=gen, device=DEV)
        freq = (1e6 ** (-np.arange(max(1, c["rot"] // 2)) * 2.0 / max(2, c["rot"]))).astype(np.float32)
        kv, scale = _to_cache(torch.randn(2, pages, n_kv, page, D, generator=gen, device=DEV), type)
        return {"rows": rows, "pos": _ints(g.integers(0, c["far"], N)), "slot": _ints(slot), "kv": kv, "scale": scale,
                "freq": torch.from_numpy(freq).to(DEV), "pages": pages,
                "live": torch.from_numpy(np.nonzero(slot >= 0)[0]).to(DEV)}
    lens, new = _order(c, seed)
    S, n = c["S"], c["n"]
    used = -(-lens // page)
    pages = int(used.sum()) + 5
    order = g.permutation(pages)
    table, at = np.full((S, int(used.max()) + 1), -1), 0
    for s in range(S):
        table[s, :used[s]] = order[at:at + used[s]]
        at += used[s]
    kv, scale = [], []
    for _ in range(n):
        # keys with a few strong channels that all tokens share
        x = torch.randn(2, pages, n_kv, page, D, generator=gen, device=DEV)
        x[0] += 2 * torch.randn(n_kv, 1, D, generator=gen, device=DEV) * (torch.rand(D, generator=gen, device=DEV) < 0.05)
        x, s = _to_cache(x, type)
        kv.append(x)
        scale.append(s)
    N = int(new.sum())
    q = 1.7 * torch.randn(n, N, n_q, D, generator=gen, device=DEV)
    return {"cached": _ints(lens - new), "new": _ints(new), "table": _ints(table), "kv": kv, "scale": scale, "q": q,
            "most": int(lens.max()), "pages": pages, "N": N}


def prepare(case, seed):
    st = _data(case, seed)
    st["case"] = dict(case)
    if own:
        _bind(st)
    return st


# ------------------------------------------------------------ the plain form

def _run_plan(st):
    c = st["case"]
    page, table = c["page"], st["table"]
    S, width = table.shape
    cached, new, held = st["cached"].long(), st["new"].long(), st["held"].long()
    lens, seqs = cached + new, torch.arange(S, device=DEV)
    need = torch.clamp((lens + page - 1) // page - held, min=0)
    upto = torch.cumsum(need, 0)
    n_free = st["n_free"].long()
    fits = (need == 0) | (upto <= n_free)
    got = torch.where(fits, need, torch.zeros_like(need))
    block = torch.arange(width, device=DEV) - held.unsqueeze(1)
    fresh = (block >= 0) & (block < got.unsqueeze(1))
    at = n_free - 1 - (upto - need).unsqueeze(1) - block
    free = st["free"].long()
    out = torch.where(fresh, free[at.clamp(0, free.numel() - 1)], table.long())
    end = torch.cumsum(new, 0)
    start = torch.cat([torch.zeros_like(end[:1]), end])
    seq = torch.repeat_interleave(seqs, new, output_size=st["N"])
    pos = torch.arange(st["N"], device=DEV) - start[seq] + cached[seq]
    slot = out[seq, pos // page] * page + pos % page
    slot = torch.where(fits[seq], slot, torch.full_like(slot, -1))
    taken = torch.where(fits & (need > 0), upto, torch.zeros_like(upto)).amax()
    return {k: v.to(torch.int32) for k, v in
            {"table": out, "held": held + got, "n_free": n_free - taken, "start": start,
             "lens": torch.where(fits, lens, torch.zeros_like(lens)), "pos": pos, "slot": slot,
             "short": (~fits).sum().reshape(1)}.items()}


def _rotated(x, c, s, rot, inter):
    """x: N rows of heads of D values, the first `rot` rotated in pairs; in 64 bits, rounded once."""
    if rot == 0:
        return x
    d = x[..., :rot].double()
    a, b = (d[..., 0::2], d[..., 1::2]) if inter else (d[..., :rot // 2], d[..., rot // 2:])
    a, b = a * c - b * s, b * c + a * s
    y = torch.stack([a, b], -1).reshape(d.shape) if inter else torch.cat([a, b], -1)
    return torch.cat([y.float(), x[..., rot:]], -1)


def _run_store(st):
    c = st["case"]
    N, n_q, n_kv, D, page = c["N"], c["n_q"], c["n_kv"], c["D"], c["page"]
    x = st["rows"].view(N, n_q + 2 * n_kv, D)
    angle = (st["pos"].double().unsqueeze(1) * st["freq"].double()).unsqueeze(1)
    qk = _rotated(x[:, :n_q + n_kv], torch.cos(angle), torch.sin(angle), c["rot"], c["inter"])
    kv, scale = _to_cache(torch.stack([qk[:, n_q:], x[:, n_q + n_kv:]]), c["type"])
    slot = st["slot"].long()[st["live"]]
    st["kv"][:, slot // page, :, slot % page] = kv[:, st["live"]].transpose(0, 1)
    if scale is None:
        return {"q": qk[:, :n_q], "kv": st["kv"]}
    st["scale"][:, slot // page, :, slot % page] = scale[:, st["live"]].transpose(0, 1)
    return {"q": qk[:, :n_q], "kv": st["kv"] * st["scale"].unsqueeze(-1)}


def _run_attn(st):
    c = st["case"]
    S, T, n_q, n_kv, D, page, L = c["S"], c["T"], c["n_q"], c["n_kv"], c["D"], c["page"], st["most"]
    G = n_q // n_kv
    cached, new = st["cached"].long(), st["new"].long()
    start = torch.cumsum(new, 0) - new
    blocks = st["table"].long().clamp(min=0)[:, :(L + page - 1) // page]
    steps = torch.arange(T, device=DEV)
    row = (start.unsqueeze(1) + steps).clamp(max=st["N"] - 1)
    last = cached.unsqueeze(1) + torch.minimum(steps, new.unsqueeze(1) - 1)      # the last key that a token sees
    keys = torch.arange(L, device=DEV)
    seen = keys <= last.unsqueeze(2)
    if c["window"]:
        seen = seen & (keys > last.unsqueeze(2) - c["window"])
    seen = seen.repeat_interleave(G, 1).unsqueeze(1)                             # S, 1, T G, L
    seq = torch.repeat_interleave(torch.arange(S, device=DEV), new, output_size=st["N"])
    step = torch.arange(st["N"], device=DEV) - start[seq]
    out = []
    for i in range(c["n"]):
        def cached_rows(j):
            x = st["kv"][i][j][blocks].float()
            if c["type"] == "i8":
                x = x * st["scale"][i][j][blocks].unsqueeze(-1)
            return x.permute(0, 2, 1, 3, 4).reshape(S * n_kv, -1, D)[:, :L].contiguous()
        q = st["q"][i][row].view(S, T, n_kv, G, D).permute(0, 2, 1, 3, 4).reshape(S * n_kv, T * G, D)
        x = torch.bmm(q, cached_rows(0).transpose(1, 2).contiguous()) * D ** -0.5
        x = torch.where(seen, x.view(S, n_kv, T * G, L), torch.full_like(x[:1, :1, :1], -math.inf))
        x = torch.exp(x - x.amax(-1, keepdim=True)).view(S * n_kv, T * G, L)
        y = torch.bmm(x, cached_rows(1)) / x.sum(-1, keepdim=True)
        y = y.view(S, n_kv, T, G, D).permute(0, 2, 1, 3, 4).reshape(S, T, n_q, D)
        out.append(y[seq, step])
    return torch.stack(out)


# --------------------------------------------------------- the library's calls

def _bind(st):
    """Output buffers, descriptors, workspaces and the calls' arguments, as a program keeps them."""
    import ctypes

    import stratum_amd as KQ
    c, lib = st["case"], KQ.lib()
    stream = torch.cuda.current_stream().cuda_stream
    st["error"] = lib.kq_last_error

    def at(t):
        return None if t is None else t.data_ptr()

    def ints(*shape):
        return torch.empty(*shape, dtype=torch.int32, device=DEV)

    def cache(kv, scale, pages):
        t = {"f16": KQ.TYPE_F16, "bf16": KQ.TYPE_BF16, "i8": KQ.TYPE_I8}[c["type"]]
        return KQ.kv_cache(t, pages, c["page"], c["n_kv"], c["D"], at(kv[0]), at(kv[1]),
                           None if scale is None else at(scale[0]), None if scale is None else at(scale[1]))
    if c["kind"] == "plan":
        S, N = c["S"], st["N"]
        out = st["outputs"] = {"table": st["table"].clone(), "held": ints(S), "n_free": ints(1), "start": ints(S + 1),
                               "lens": ints(S), "pos": ints(N), "slot": ints(N), "short": ints(1)}
        shape = KQ.attn_shape(S, min(c["T"], 8), 24, 4, 256)
        nb = KQ.kv_list_bytes(shape)
        st["list"] = torch.empty(nb, dtype=torch.uint8, device=DEV)
        st["desc"] = KQ.kv_plan(S, c["page"], st["n_pages"], at(st["cached"]), new_ptr=at(st["new"]),
                                held_ptr=at(st["held"]), table_ptr=at(out["table"]), table_stride=out["table"].shape[1],
                                free_ptr=at(st["free"]), n_free_ptr=at(st["n_free"]), held_out_ptr=at(out["held"]),
                                n_free_out_ptr=at(out["n_free"]), start_ptr=at(out["start"]), lens_ptr=at(out["lens"]),
                                N=N, pos_ptr=at(out["pos"]), slot_ptr=at(out["slot"]), short_ptr=at(out["short"]),
                                shape=shape, list_ptr=at(st["list"]), list_bytes=nb)
        st["calls"] = [(lib.kq_kv_plan_dev, (ctypes.byref(st["desc"]), stream))]
    elif c["kind"] == "store":
        N, n_q, n_kv, D = c["N"], c["n_q"], c["n_kv"], c["D"]
        wide = (n_q + 2 * n_kv) * D
        q = torch.empty(N, n_q, D, device=DEV)
        st["outputs"] = {"q": q, "kv": st["kv"]}
        st["cache"] = cache(st["kv"], st["scale"], st["pages"])
        rows = at(st["rows"])
        st["desc"] = KQ.kv_store(st["cache"], N, at(st["slot"]), rows + 4 * n_q * D, rows + 4 * (n_q + n_kv) * D,
                                 k_stride=wide, v_stride=wide, pos_ptr=at(st["pos"]), rot=c["rot"],
                                 interleaved=c["inter"], freq_ptr=at(st["freq"]) if c["rot"] else None, n_q=n_q,
                                 q_ptr=rows, q_stride=wide, q_out_ptr=at(q))
        st["calls"] = [(lib.kq_kv_store_dev, (ctypes.byref(st["desc"]), stream))]
    else:
        S, N, n_q, D = c["S"], st["N"], c["n_q"], c["D"]
        out = st["outputs"] = torch.zeros(c["n"], N, n_q, D, device=DEV)
        st["start"], st["lens"] = ints(S + 1), ints(S)
        shape = KQ.attn_shape(S, c["T"], n_q, c["n_kv"], D, window=c["window"])
        nb, wb = KQ.kv_list_bytes(shape), KQ.paged_attn_workspace_bytes(shape)
        st["list"] = torch.empty(nb, dtype=torch.uint8, device=DEV)
        st["work"] = torch.empty(max(256, wb), dtype=torch.uint8, device=DEV)
        # the lengths and the list of work: once a step, for all of its layers
        plan = KQ.kv_plan(S, c["page"], st["pages"], at(st["cached"]), new_ptr=at(st["new"]), start_ptr=at(st["start"]),
                          lens_ptr=at(st["lens"]), shape=shape, list_ptr=at(st["list"]), list_bytes=nb)
        st["cache"] = [cache(st["kv"][i], st["scale"][i], st["pages"]) for i in range(c["n"])]
        st["desc"] = [plan] + [KQ.paged_attn(shape, st["cache"][i], at(st["q"][i]), at(out[i]), N, at(st["table"]),
                                             st["table"].shape[1], at(st["start"]), at(st["lens"]), D ** -0.5,
                                             list_ptr=at(st["list"]), list_bytes=nb) for i in range(c["n"])]
        st["calls"] = [(lib.kq_kv_plan_dev, (ctypes.byref(plan), stream))] + [
            (lib.kq_paged_attn_dev, (ctypes.byref(d), at(st["work"]), wb, stream)) for d in st["desc"][1:]]


def _call(st):
    for call, args in st["calls"]:
        if call(*args) != 0:
            raise RuntimeError(st["error"]().decode(errors="replace"))
    if st["case"]["kind"] == "store" and st["scale"] is not None:      # the int8 rows as the values they stand for
        return dict(st["outputs"], kv=st["kv"] * st["scale"].unsqueeze(-1))
    return st["outputs"]


def run(st):
    if own:
        return _call(st)
    return {"plan": _run_plan, "store": _run_store, "attn": _run_attn}[st["case"]["kind"]](st)


# ------------------------------------------------------------ floor of a pass

def work(case):
    """Inputs and outputs once; two operations per weight of a sum."""
    c = case
    if c["kind"] == "plan":
        lens, new = _lens(c)
        fresh = sum(-(-n // c["page"]) - -(-(n - k) // c["page"]) for n, k in zip(lens, new))
        return {"bytes": 4.0 * (5 * c["S"] + 2 * fresh + 2 * sum(new) + 4), "flops": 4.0 * c["S"] + 2.0 * sum(new)}
    size = {"f16": 2, "bf16": 2, "i8": 1}[c["type"]]
    row = c["D"] * size + (4 if c["type"] == "i8" else 0)
    if c["kind"] == "store":
        N, n_q, n_kv, D = c["N"], c["n_q"], c["n_kv"], c["D"]
        return {"bytes": float(N * (4 * D * (2 * n_q + 2 * n_kv) + 2 * n_kv * row + 8)),
                "flops": 3.0 * N * (n_q + n_kv) * c["rot"]}
    lens, new = _lens(c)
    w = c["window"]
    keys = [min(n, w + k - 1) if w else n for n, k in zip(lens, new)]
    b = sum(keys) * c["n_kv"] * 2 * row + 8 * sum(new) * c["n_q"] * c["D"]
    return {"bytes": float(c["n"] * b),
            "flops": 4.0 * c["n"] * c["n_q"] * c["D"] * sum(a * k for a, k in zip(keys, new))}


# -------------------------------------------------- the same results, 64 bits

def exact(case, seed):
    d, c = _data(case, seed), case
    if c["kind"] == "plan":
        page, table, free = c["page"], d["table"].cpu().numpy().copy(), d["free"].tolist()[:int(d["n_free"][0])]
        held, start, lens, pos, slot, short = d["held"].tolist(), [0], [], [], [], 0
        wanted, room = 0, len(free)
        for s, (old, k) in enumerate(zip(d["cached"].tolist(), d["new"].tolist())):
            more = max(0, math.ceil((old + k) / page) - held[s])
            wanted += more
            ok = more == 0 or wanted <= room
            for _ in range(more if ok else 0):
                table[s, held[s]] = free.pop()
                held[s] += 1
            for p in range(old, old + k):
                pos.append(p)
                slot.append(int(table[s, p // page]) * page + p % page if ok else -1)
            start.append(start[-1] + k)
            lens.append(old + k if ok else 0)
            short += not ok
        return {k: torch.from_numpy(np.asarray(v, dtype=np.int32)) for k, v in
                {"table": table, "held": held, "n_free": [len(free)], "start": start, "lens": lens, "pos": pos,
                 "slot": slot, "short": [short]}.items()}
    n_q, n_kv, D, page = c["n_q"], c["n_kv"], c["D"], c["page"]
    if c["kind"] == "store":
        N, rot = c["N"], c["rot"]
        x = d["rows"].double().view(N, n_q + 2 * n_kv, D)
        if rot:
            turn = torch.polar(torch.ones(N, 1, rot // 2, dtype=torch.float64, device=DEV),
                               torch.outer(d["pos"].double(), d["freq"].double()).unsqueeze(1))
            first = torch.arange(0, rot, 2, device=DEV) if c["inter"] else torch.arange(rot // 2, device=DEV)
            second = first + (1 if c["inter"] else rot // 2)
            z = torch.complex(x[:, :n_q + n_kv, first], x[:, :n_q + n_kv, second]) * turn
            x[:, :n_q + n_kv, first], x[:, :n_q + n_kv, second] = z.real, z.imag
        kv = d["kv"].double() if d["scale"] is None else d["kv"].double() * d["scale"].double().unsqueeze(-1)
        rows = torch.stack([x[:, n_q:n_q + n_kv], x[:, n_q + n_kv:]])
        if d["scale"] is not None:
            # the int8 step takes the binary32 values; its scale and reciprocal are binary32
            r = rows.float().double()
            scale = (r.abs().amax(-1, keepdim=True) / 127.0).float()
            recip = torch.where(scale > 0, (1.0 / scale.double()).float(), scale)
            rows = (r * recip.double()).float().round().clamp(-128, 127).double() * scale.double()
        for i, s in enumerate(d["slot"].tolist()):
            if s >= 0:
                kv[:, s // page, :, s % page] = rows[:, i]
        return {"q": x[:, :n_q].clone(), "kv": kv}
    G, out, at = n_q // n_kv, torch.zeros(c["n"], d["N"], n_q, D, dtype=torch.float64, device=DEV), 0
    for s, (old, k) in enumerate(zip(d["cached"].tolist(), d["new"].tolist())):
        blocks = d["table"][s, :-(-(old + k) // page)].long()
        for i in range(c["n"]):
            kv = d["kv"][i][:, blocks].double()
            if d["scale"][i] is not None:
                kv = kv * d["scale"][i][:, blocks].double().unsqueeze(-1)
            kv = kv.transpose(1, 2).reshape(2, n_kv, -1, D)
            for t in range(k):
                end = old + t + 1
                first = max(0, end - c["window"]) if c["window"] else 0
                q = d["q"][i][at + t].double().view(n_kv, G, D)
                x = torch.matmul(q, kv[0][:, first:end].transpose(1, 2).contiguous()) / math.sqrt(D)
                p = torch.softmax(x, -1)
                out[i, at + t] = torch.matmul(p, kv[1][:, first:end].contiguous()).reshape(n_q, D)
        at += k
    return out
