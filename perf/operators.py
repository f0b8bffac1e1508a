"""The operators around the quantized products of a decode step, as timed cases.

Kinds:

  norm    RMS norm of rows with the residual's addition before it; the normed
          rows as binary32, or as int8 with a scale per group
  w4      B rows times a matrix of 4-bit weights with group scales; x binary32,
          or int8 rows with a scale per 32 as the norm writes them
  verify  drafted tokens against the target's distributions, from given random
          numbers: how many are accepted, and the token that follows them

Hidden states are N(0, 1) with a few channels several times larger, weights have
|w| around 0.02, logits a spread of a few units.  A pass of the w4 cases goes over
`n` matrices, as a decode step goes from layer to layer: over the states that a
timing loop rotates they do not stay in the 256 MB cache in front of HBM.

`run` computes the operators from elementary torch operations, or, where `own` is
set, calls the library.
"""
import math

import torch

own = False

DEV = "cuda"
EPS = 1e-6


# ------------------------------------------------------------------- cases

def listed():
    return [
        # the norm before a matvec of one token, the smallest call: latency
        {"name": "norm_b1_5120", "kind": "norm", "B": 1, "K": 5120, "resid": True, "weight": True, "group": 0},
        # eight token streams, straight to the int8 rows that a product reads
        {"name": "norm_q8_b8_5120", "kind": "norm", "B": 8, "K": 5120, "resid": True, "weight": True, "group": 32},
        # rows of an odd length, no residual (a norm over a projection's output)
        {"name": "norm_b517_1153", "kind": "norm", "B": 517, "K": 1153, "resid": False, "weight": True, "group": 0},
        # a prompt's chunk, normed and quantized
        {"name": "norm_q8_b4096_5120", "kind": "norm", "B": 4096, "K": 5120, "resid": True, "weight": True, "group": 32},
        # the smallest product: one token, one small matrix
        {"name": "w4_b1_1024x1024", "kind": "w4", "N": 1024, "K": 1024, "n": 1, "B": 1, "g": 32, "scale": "f16",
         "zeros": False, "q8": False},
        # gate and up of a 27B-class layer, one token
        {"name": "w4_b1_17408x5120", "kind": "w4", "N": 17408, "K": 5120, "n": 2, "B": 1, "g": 128, "scale": "f16",
         "zeros": False, "q8": False},
        # its down projection: long rows, int8 activations, zero points
        {"name": "w4_q8_b1_5120x17408", "kind": "w4", "N": 5120, "K": 17408, "n": 2, "B": 1, "g": 64, "scale": "f16",
         "zeros": True, "q8": True},
        # a few drafted tokens through an LM head: many short rows
        {"name": "w4_b5_151936x1024", "kind": "w4", "N": 151936, "K": 1024, "n": 1, "B": 5, "g": 32, "scale": "f16",
         "zeros": False, "q8": False},
        # a row count that divides nothing, three tokens, bf16 scales and zero points
        {"name": "w4_b3_11007x4096", "kind": "w4", "N": 11007, "K": 4096, "n": 4, "B": 3, "g": 128, "scale": "bf16",
         "zeros": True, "q8": False},
        # batched decode, sixteen streams with int8 activations
        {"name": "w4_q8_b16_17408x5120", "kind": "w4", "N": 17408, "K": 5120, "n": 2, "B": 16, "g": 128, "scale": "f16",
         "zeros": False, "q8": True},
        # one sequence, four tokens drafted from an n-gram table (no draft distribution)
        {"name": "verify_s1_t4", "kind": "verify", "S": 1, "T": 4, "V": 151936, "form": "logits", "draft": False},
        # sixteen sequences with up to seven tokens from a draft model's logits
        {"name": "verify_s16_t7", "kind": "verify", "S": 16, "T": 7, "V": 151936, "form": "logits", "draft": True},
    ]


MOST_BYTES, MOST_FLOPS = 1.5e8, 6e9     # of a drawn case: no larger than the largest listed one


def _log(rng, lo, hi):
    return math.exp(rng.uniform(math.log(lo), math.log(hi)))


def _draw(rng):
    kind = rng.choice(["norm", "w4", "w4", "w4", "verify", "verify"])
    if kind == "norm":
        group = rng.choice([0, 0, 16, 32, 32])
        K = int(_log(rng, 100, 20000))
        K = group * max(1, round(K / group)) if group else K
        return {"kind": kind, "B": int(_log(rng, 1, 4097)), "K": K, "resid": rng.random() < 0.7,
                "weight": rng.random() < 0.8, "group": group}
    if kind == "w4":
        g = rng.choice([32, 64, 128, 128, 256])
        N, K = int(_log(rng, 100, 152000)), g * max(1, round(_log(rng, 256, 17409) / g))
        n = max(1, min(4, int(1.8e8 / (N * K))))
        return {"kind": kind, "N": N, "K": K, "n": n, "B": int(_log(rng, 1, 33)), "g": g,
                "scale": rng.choice(["f16", "f16", "bf16", "f32"]), "zeros": rng.random() < 0.4,
                "q8": rng.random() < 0.5}
    form = rng.choice(["logits", "logits", "probs", "greedy"])
    return {"kind": kind, "S": int(_log(rng, 1, 17)), "T": rng.randint(0, 8), "V": int(_log(rng, 1000, 152000)),
            "form": form, "draft": form != "greedy" and rng.random() < 0.6}


def draw(rng):
    while True:
        c = _draw(rng)
        w = work(c)
        if w["bytes"] <= MOST_BYTES and w["flops"] <= MOST_FLOPS:
            return c


# ------------------------------------------------------------------- inputs

def _gen(seed, salt):
    return torch.Generator(device=DEV).manual_seed(seed * 1000003 + salt)


def _hidden(seed, salt, *shape):
    """Hidden states: N(0, 1), one channel in about 200 several times larger."""
    g = _gen(seed, salt)
    x = torch.randn(*shape, generator=g, device=DEV)
    big = torch.rand(shape[-1], generator=g, device=DEV) < 0.005
    return torch.where(big, x * 8, x).contiguous()


SCALES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


def _data(c, seed):
    """The case's inputs, from the seed alone."""
    kind = c["kind"]
    if kind == "norm":
        B, K = c["B"], c["K"]
        return {"x": _hidden(seed, 1, B, K), "r": _hidden(seed, 2, B, K) * 2 if c["resid"] else None,
                "w": 1 + 0.2 * torch.randn(K, generator=_gen(seed, 3), device=DEV) if c["weight"] else None}
    if kind == "w4":
        N, K, n, B, g = c["N"], c["K"], c["n"], c["B"], c["g"]
        gen = _gen(seed, 1)
        q = torch.randint(0, 256, (n, N, K // 2), generator=gen, device=DEV, dtype=torch.uint8)
        s = (0.0043 * torch.exp(0.3 * torch.randn(n, N, K // g, generator=gen, device=DEV))).to(SCALES[c["scale"]])
        z = torch.randint(5, 11, (n, N, K // g), generator=gen, device=DEV, dtype=torch.uint8) if c["zeros"] else None
        d = {"q": q, "s": s, "z": z, "x": _hidden(seed, 2, B, K), "xq": None, "xs": None}
        if c["q8"]:
            v = d["x"].reshape(B, K // 32, 32)
            a = v.abs().amax(-1) / 127.0
            d["xq"] = torch.round(v / a.unsqueeze(-1)).clamp(-127, 127).to(torch.int8).reshape(B, K)
            d["xs"], d["x"] = a, None
        return d
    S, T, V = c["S"], c["T"], c["V"]
    gen = _gen(seed, 1)
    target = 2.5 * torch.randn(S, T + 1, V, generator=gen, device=DEV)
    # the likely tokens of a row, some ten units above the rest
    hot = torch.randint(0, V, (S, T + 1, 6), generator=gen, device=DEV)
    target.scatter_reduce_(2, hot, 12 + 2 * torch.randn(S, T + 1, 6, generator=gen, device=DEV), "amax")
    draft = target[:, :T] + 0.7 * torch.randn(S, T, V, generator=gen, device=DEV)
    # the drafted tokens, drawn from the draft's distribution
    noise = -torch.log(-torch.log(torch.rand(S, T, V, generator=gen, device=DEV).clamp(1e-12, 1 - 1e-7)))
    tokens = torch.argmax(draft * 1.25 + noise, -1).to(torch.int32)
    if c["form"] == "probs":
        target = torch.softmax(target.double() * 1.25, -1).float()
        draft = torch.softmax(draft.double() * 1.25, -1).float()
    n_draft = torch.randint((T + 1) // 2, T + 1, (S,), generator=gen, device=DEV, dtype=torch.int32)
    return {"target": target, "draft": draft.contiguous() if c["draft"] else None, "tokens": tokens.contiguous(),
            "n_draft": n_draft, "u": torch.rand(S, T + 1, generator=gen, device=DEV), "inv_temp": 1.25}


def prepare(case, seed):
    st = _data(case, seed)
    st["case"] = dict(case)
    if own:
        _bind(st)
    return st


# ------------------------------------------------------------ the plain form

def _quantize(y, G):
    """y as int8 per group of G, and the values that stands for."""
    v = y.reshape(*y.shape[:-1], -1, G)
    s = v.abs().amax(-1, keepdim=True)
    s = s / torch.full_like(s, 127.0)          # by a tensor: a scalar divisor becomes a product
    inv = torch.where(s > 0, 1.0 / s, torch.zeros_like(s))
    q = torch.clamp(torch.round(v * inv), -128, 127)
    return (q * s).reshape(y.shape), s.squeeze(-1)


def _norm(st):
    c = st["case"]
    s = st["x"] if st["r"] is None else st["x"] + st["r"]
    # in 64 bits where the result is rounded to int8: a value next to a step's border
    v = s.double() if c["group"] else s
    y = v * torch.rsqrt((v * v).mean(-1, keepdim=True) + EPS)
    if st["w"] is not None:
        y = y * st["w"]
    y = y.float()
    out = {"sum": s} if st["r"] is not None else {}
    if c["group"]:
        out["values"], out["scales"] = _quantize(y, c["group"])
    else:
        out["y"] = y
    return out


def _w4(st):
    c, out = st["case"], []
    x = st["x"]
    if c["q8"]:
        x = (st["xq"].reshape(c["B"], -1, 32) * st["xs"].unsqueeze(-1)).reshape(c["B"], c["K"])
    for i in range(c["n"]):
        q = torch.stack([st["q"][i] & 15, st["q"][i] >> 4], -1).reshape(c["N"], -1, c["g"]).float()
        z = 8.0 if st["z"] is None else st["z"][i].float().unsqueeze(-1)
        w = ((q - z) * st["s"][i].float().unsqueeze(-1)).reshape(c["N"], c["K"])
        out.append(x @ w.t())
    return torch.stack(out)


def _verify(st):
    c = st["case"]
    S, T = c["S"], c["T"]
    tok, nd, u = st["tokens"].long(), st["n_draft"].long(), st["u"].double()
    steps = torch.arange(T, device=DEV)
    last = torch.arange(T + 1, device=DEV)
    if c["form"] == "greedy":
        best = torch.argmax(st["target"], -1)
        ok = (tok == best[:, :T]) & (steps < nd.unsqueeze(1))
        n = torch.cumprod(ok.long(), 1).sum(1)
        nxt = torch.gather(best, 1, n.unsqueeze(1)).squeeze(1)
    else:
        # in 64 bits: where the running sum passes u decides the token
        def dist(a):
            if c["form"] == "probs":
                return a.double()
            a = a.double() * st["inv_temp"]
            e = torch.exp(a - a.amax(-1, keepdim=True))
            return e / e.sum(-1, keepdim=True)
        p = dist(st["target"])
        pt = torch.gather(p[:, :T], 2, tok.unsqueeze(2)).squeeze(2)
        q = None if st["draft"] is None else dist(st["draft"])
        qt = 1.0 if q is None else torch.gather(q, 2, tok.unsqueeze(2)).squeeze(2)
        ok = (u[:, :T] * qt < pt) & (steps < nd.unsqueeze(1))
        n = torch.cumprod(ok.long(), 1).sum(1)
        seqs = torch.arange(S, device=DEV)
        r = p[seqs, n]
        if T:
            at = n.clamp(max=T - 1)
            sub = torch.zeros_like(r)
            if q is None:
                sub.scatter_(1, tok[seqs, at].unsqueeze(1), math.inf)
            else:
                sub = q[seqs, at]
            left = torch.clamp(r - sub, min=0.0)
            left = torch.where(left.sum(1, keepdim=True) > 0, left, r)
            r = torch.where((n < nd).unsqueeze(1), left, r)
        cum = torch.cumsum(r, 1)
        over = (cum > u[:, T:] * cum[:, -1:]) & (r > 0)
        nxt = torch.argmax(over.to(torch.uint8), 1)
    nxt = nxt.unsqueeze(1)
    pad = torch.cat([tok, torch.zeros_like(nxt)], 1)
    out = torch.where(last < n.unsqueeze(1), pad, torch.where(last == n.unsqueeze(1), nxt, torch.full_like(pad, -1)))
    return {"n_accept": n.to(torch.int32), "out": out.to(torch.int32)}


# --------------------------------------------------------- the library's calls

def _bind(st):
    """Output buffers, descriptors, workspaces and the calls' arguments, as a program keeps them."""
    import ctypes

    import stratum_amd as KQ
    c, kind, lib = st["case"], st["case"]["kind"], KQ.lib()
    stream = torch.cuda.current_stream().cuda_stream
    st["error"] = lib.kq_last_error

    def at(t):
        return None if t is None else t.data_ptr()
    if kind == "norm":
        B, K, G = c["B"], c["K"], c["group"]
        out = st["outputs"] = {"sum": torch.empty(B, K, device=DEV)} if c["resid"] else {}
        if G:
            st["xq"] = torch.empty(B, K // G, G, dtype=torch.int8, device=DEV)
            out["scales"] = torch.empty(B, K // G, device=DEV)
            st["steps"] = out["scales"].unsqueeze(-1)
        else:
            out["y"] = torch.empty(B, K, device=DEV)
        st["desc"] = KQ.rmsnorm(B, K, EPS, at(st["x"]), resid_ptr=at(st["r"]), sum_ptr=at(out.get("sum")),
                                weight_ptr=at(st["w"]), y_ptr=at(out.get("y")), group=G, xq_ptr=at(st.get("xq")),
                                xscale_ptr=at(out.get("scales")))
        st["calls"] = [(lib.kq_rmsnorm_dev, (ctypes.byref(st["desc"]), stream))]
    elif kind == "w4":
        N, K, B = c["N"], c["K"], c["B"]
        t = {"f16": KQ.TYPE_F16, "bf16": KQ.TYPE_BF16, "f32": KQ.TYPE_F32}[c["scale"]]
        st["desc"] = [KQ.w4(N, K, c["g"], t, at(st["q"][i]), at(st["s"][i]), None if st["z"] is None else at(st["z"][i]))
                      for i in range(c["n"])]
        y = st["outputs"] = torch.empty(c["n"], B, N, device=DEV)
        nb = KQ.w4_workspace_bytes(st["desc"][0], B, c["q8"])
        st["work"] = torch.empty(max(16, nb), dtype=torch.uint8, device=DEV)
        tail = (B, at(st["work"]), nb, stream)
        if c["q8"]:
            st["calls"] = [(lib.kq_w4_gemv_q8_dev, (ctypes.byref(d), at(st["xq"]), at(st["xs"]), None, at(y[i])) + tail)
                           for i, d in enumerate(st["desc"])]
        else:
            st["calls"] = [(lib.kq_w4_gemv_dev, (ctypes.byref(d), at(st["x"]), None, at(y[i])) + tail)
                           for i, d in enumerate(st["desc"])]
    else:
        S, T, V = c["S"], c["T"], c["V"]
        flags = {"logits": KQ.VERIFY_LOGITS, "probs": 0, "greedy": KQ.VERIFY_GREEDY}[c["form"]]
        out = st["outputs"] = {"n_accept": torch.empty(S, dtype=torch.int32, device=DEV),
                               "out": torch.empty(S, T + 1, dtype=torch.int32, device=DEV)}
        st["desc"] = KQ.spec_verify(S, T, V, flags, at(st["target"]), at(st["tokens"]), at(st["u"]), at(out["n_accept"]),
                                    at(out["out"]), draft_ptr=at(st["draft"]), n_draft_ptr=at(st["n_draft"]),
                                    inv_temp=st["inv_temp"])
        nb = KQ.spec_verify_workspace_bytes(st["desc"])
        st["work"] = torch.empty(max(16, nb), dtype=torch.uint8, device=DEV)
        st["calls"] = [(lib.kq_spec_verify_dev, (ctypes.byref(st["desc"]), at(st["work"]), nb, stream))]


def _call(st):
    for call, args in st["calls"]:
        if call(*args) != 0:
            raise RuntimeError(st["error"]().decode(errors="replace"))
    if "steps" in st:       # the int8 rows as the values they stand for
        values = (st["xq"] * st["steps"]).reshape(st["case"]["B"], st["case"]["K"])
        return dict(st["outputs"], values=values)
    return st["outputs"]


def run(st):
    if own:
        return _call(st)
    return {"norm": _norm, "w4": _w4, "verify": _verify}[st["case"]["kind"]](st)


# ------------------------------------------------------------ floor of a pass

def work(case):
    """Inputs and outputs once; two operations per weight and row."""
    c = case
    if c["kind"] == "norm":
        B, K, G = c["B"], c["K"], c["group"]
        n = B * K
        b = n * (4 + (8 if c["resid"] else 0)) + (4 * K if c["weight"] else 0) + (n + 4 * n // G if G else 4 * n)
        return {"bytes": float(b), "flops": 6.0 * n}
    if c["kind"] == "w4":
        N, K, B, g = c["N"], c["K"], c["B"], c["g"]
        groups = N * (K // g)
        b = N * K // 2 + groups * ((4 if c["scale"] == "f32" else 2) + (1 if c["zeros"] else 0)) + 4 * B * N
        x = B * K + 4 * B * (K // 32) if c["q8"] else 4 * B * K
        return {"bytes": float(c["n"] * b + x), "flops": 2.0 * c["n"] * N * K * B}
    S, T, V = c["S"], c["T"], c["V"]
    rows = S * (T + 1) + (S * T if c["draft"] else 0)
    if c["form"] == "probs":
        rows = S * (2 if c["draft"] and T else 1)     # the row drawn from, and the draft's
    return {"bytes": float(4 * rows * V + 4 * S * (3 * T + 4)), "flops": 4.0 * rows * V}


# -------------------------------------------------- the same results, 64 bits

def exact(case, seed):
    d = _data(case, seed)
    kind = case["kind"]
    if kind == "norm":
        B, K, G = case["B"], case["K"], case["group"]
        total = d["x"].double() + (0 if d["r"] is None else d["r"].double())
        total = total.float().double()               # the residual stream is binary32
        out = {"sum": total} if d["r"] is not None else {}
        y = total / torch.sqrt(total.square().sum(1, keepdim=True) / K + EPS)
        if d["w"] is not None:
            y = y * d["w"].double()
        if not G:
            out["y"] = y
            return out
        # the int8 step takes the binary32 values; its scale and reciprocal are binary32
        rows = y.float().reshape(B * (K // G), G)
        top = rows.abs().max(1).values
        scale = (top.double() / 127.0).float()
        recip = torch.where(scale > 0, (1.0 / scale.double()).float(), scale)
        steps = (rows.double() * recip.double().unsqueeze(1)).float().round().clamp(-128, 127)
        out["values"] = (steps.double() * scale.double().unsqueeze(1)).reshape(B, K)
        out["scales"] = scale.double().reshape(B, K // G)
        return out
    if kind == "w4":
        N, K, g, B = case["N"], case["K"], case["g"], case["B"]
        x = d["x"].double() if d["xq"] is None else d["xq"].double() * d["xs"].double().repeat_interleave(32, 1)
        even, odd = x[:, 0::2].t().contiguous(), x[:, 1::2].t().contiguous()
        sums = x.reshape(B, K // g, g).sum(2)
        y = torch.empty(case["n"], B, N, dtype=torch.float64, device=DEV)
        step = max(1, (1 << 25) // K)
        for i in range(case["n"]):
            for a in range(0, N, step):
                b = min(N, a + step)
                s = d["s"][i, a:b].double()
                wide = s.repeat_interleave(g // 2, 1)
                raw = d["q"][i, a:b]
                acc = ((raw % 16).double() * wide) @ even + ((raw // 16).double() * wide) @ odd
                z = s * (8.0 if d["z"] is None else d["z"][i, a:b].double())
                y[i, :, a:b] = (acc - z @ sums.t().contiguous()).t()
        return y
    S, T = case["S"], case["T"]
    ns, outs = [], []
    for s in range(S):
        def row(a, i):
            v = a[s, i].double()
            if case["form"] == "probs":
                return v
            v = v * d["inv_temp"]
            return torch.exp(v - torch.logsumexp(v, 0))
        nd, toks, u = int(d["n_draft"][s]), d["tokens"][s].tolist(), d["u"][s].double().tolist()
        n, nxt = 0, None
        if case["form"] == "greedy":
            while n < nd and int((d["target"][s, n] == d["target"][s, n].max()).nonzero()[0]) == toks[n]:
                n += 1
            nxt = int((d["target"][s, n] == d["target"][s, n].max()).nonzero()[0])
        else:
            left = None
            while n < nd:
                p = row(d["target"], n)
                q = torch.zeros_like(p)
                if d["draft"] is None:
                    q[toks[n]] = 1.0
                else:
                    q = row(d["draft"], n)
                if not u[n] * float(q[toks[n]]) < float(p[toks[n]]):
                    left = (p - q).clamp(min=0)
                    if d["draft"] is None:
                        left[toks[n]] = 0.0
                    if float(left.sum()) <= 0:
                        left = p
                    break
                n += 1
            if left is None:
                left = row(d["target"], n)
            cum = torch.cumsum(left, 0)
            nxt = int(torch.searchsorted(cum, (cum[-1] * u[T]).reshape(1), right=True))
        ns.append(n)
        outs.append(toks[:n] + [nxt] + [-1] * (T - n))
    return {"n_accept": torch.tensor(ns, dtype=torch.int32), "out": torch.tensor(outs, dtype=torch.int32)}
