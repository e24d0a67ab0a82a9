"""Timed calls of the token-step operators: appending rotated keys and values
to the paged 8-bit cache, attention over that cache, and sampling.

A case is a dict of plain values; ``prepare`` makes what a serving program
holds before the call (cache pages, page tables, lengths, rotation tables, new
rows, logits and random numbers), ``run`` makes one pass, through the
framework's entry points where ``own`` is true and otherwise as elementary
torch operations, and ``exact`` restates it in float64 from the definition.

The cache: pages of P tokens in E4M3, K as [pages][KVH][P][R] and V as
[pages][KVH][R][P] bytes (R: the head size padded), with a power-of-two scale
per page and head for each.  Sequence b's new tokens are the rows starts[b] ..
starts[b+1] - 1 of the packed inputs, at positions lens[b], lens[b] + 1, ...

Families (``kind``):
  append   rotate new queries and keys, quantise keys and values into pages
  attend   softmax(q K^T) V over each sequence's pages
  sample   temperature, top-k, top-p, min-p and a draw, one token a row
"""
import ctypes as C
import math

import numpy as np
import torch

own = False

DT = {"f32": torch.float32, "bf16": torch.bfloat16}
DCODE = {"f32": 0, "bf16": 1}
FP8_MAX, MIN_EXP = 448.0, -100


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # a token of a few sequences of the small language model (8 heads of 32): latency
        dict(name="append_step_small", kind="append", dtype="f32", B=4, heads=8, kvh=8, hd=32, page=16,
             new=1, past=120, ragged=False),
        # a token of every sequence of a busy server, grouped heads
        dict(name="append_step_batch", kind="append", dtype="bf16", B=256, heads=32, kvh=8, hd=128, page=64,
             new=1, past=500, ragged=True),
        # prompts of several requests at once
        dict(name="append_prompt", kind="append", dtype="bf16", B=6, heads=32, kvh=8, hd=128, page=64,
             new=2048, past=300, ragged=True),
        # odd sizes: an 80-wide head, short and empty requests among longer ones
        dict(name="append_ragged_f32", kind="append", dtype="f32", B=7, heads=12, kvh=4, hd=80, page=32,
             new=333, past=77, ragged=True),
        # a token of a few sequences of the small language model at its usual context
        dict(name="attend_step_small", kind="attend", dtype="f32", B=4, heads=8, kvh=8, hd=32, page=16,
             new=1, past=127, ragged=False),
        # one conversation with a long history: the work has to be split along it
        dict(name="attend_step_long", kind="attend", dtype="bf16", B=1, heads=32, kvh=8, hd=128, page=64,
             new=1, past=131071, ragged=False),
        # a token of every sequence of a busy server: the cache is read once
        dict(name="attend_step_batch", kind="attend", dtype="bf16", B=64, heads=32, kvh=8, hd=128, page=64,
             new=1, past=8191, ragged=True),
        # the next part of two long prompts, behind what is cached
        dict(name="attend_prompt", kind="attend", dtype="bf16", B=2, heads=32, kvh=8, hd=128, page=64,
             new=2048, past=2048, ragged=False),
        # prompts of odd lengths in float32, an 80-wide head, three queries a key head
        dict(name="attend_prompt_f32", kind="attend", dtype="f32", B=5, heads=12, kvh=4, hd=80, page=32,
             new=333, past=200, ragged=True),
        # the small language model's vocabulary, a few rows
        dict(name="sample_small", kind="sample", dtype="f32", B=4, V=8000, filters="all"),
        # one row of a larger vocabulary
        dict(name="sample_one", kind="sample", dtype="bf16", B=1, V=50257, filters="top_k"),
        # a busy server's step over a large vocabulary
        dict(name="sample_batch", kind="sample", dtype="f32", B=128, V=131072, filters="all"),
    ]


def _logint(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["append", "append", "attend", "attend", "attend", "sample", "sample"])
    dtype = rng.choice(["f32", "bf16"])
    if kind == "sample":
        return dict(kind=kind, dtype=dtype, B=_logint(rng, 1, 128), V=_logint(rng, 100, 131072),
                    filters=rng.choice(["all", "none", "top_k", "top_p", "min_p"]))
    while True:
        kvh = rng.choice([1, 2, 3, 4, 8])
        c = dict(kind=kind, dtype=dtype, B=_logint(rng, 1, 64), heads=kvh * rng.choice([1, 1, 2, 3, 4, 7, 8]), kvh=kvh,
                 hd=rng.choice([16, 32, 48, 64, 72, 80, 96, 128, 192, 256]), page=rng.choice([16, 32, 64, 128]),
                 new=1 if rng.random() < 0.55 else _logint(rng, 2, 2048), past=_logint(rng, 1, 16384),
                 ragged=rng.random() < 0.7)
        if c["heads"] > 32:
            continue
        w = work(c)
        cells = c["B"] * c["heads"] * c["new"] * (c["new"] + c["past"])
        rows = c["B"] * c["kvh"] * (c["new"] + c["past"] + 128)
        top = 1.0e11 if dtype == "bf16" else 3.0e10
        if kind == "append" and w["bytes"] <= 1.0e8 and rows * c["hd"] <= 1e8:
            return c
        if kind == "attend" and cells <= 5e8 and rows * c["hd"] <= 4e8 and w["flops"] <= top:
            return c


# ------------------------------------------------------------------ shapes
def _row(hd):
    return next(r for r in (32, 64, 96, 128, 192, 256) if r >= hd)


def _lengths(c):
    """(past, new) tokens of every sequence: whole numbers that go by the case
    alone.  Ragged: spread between none and the case's sizes, one sequence at
    the largest, one prompt of no tokens."""
    B, past, new = c["B"], c["past"], c["new"]
    if not c["ragged"]:
        return [past] * B, [new] * B
    r = np.random.RandomState(B * 7919 + past * 31 + new)
    p = [int(x) for x in r.randint(0, past + 1, B)]
    n = [int(x) for x in r.randint(1, new + 1, B)]
    p[0], n[0] = past, new
    if B > 2 and new > 1:
        n[1] = 0
    return p, n


# ------------------------------------------------------------------ what a program holds
def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda").manual_seed(int(seed) * 1000003 + 29)
    d = DT[c["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    if c["kind"] == "sample":
        return _prepare_sample(c, g, d, normal)
    B, heads, kvh, hd, P = c["B"], c["heads"], c["kvh"], c["hd"], c["page"]
    R = _row(hd)
    past, new = _lengths(c)
    N = sum(new)
    per = [-(-(a + b) // P) for a, b in zip(past, new)]
    max_pages, pages = max(1, max(per)), sum(per) + 3
    # pages are handed out in any order, as a server's free list gives them
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    at = torch.tensor([sum(per[:b]) for b in range(B)], device="cuda")[:, None] + torch.arange(max_pages, device="cuda")[None]
    table = order[at.clamp(max=pages - 1)].contiguous()
    starts = torch.tensor([sum(new[:b]) for b in range(B + 1)], dtype=torch.int32, device="cuda")
    lens = torch.tensor(past, dtype=torch.int32, device="cuda")

    def pool(shape):
        """Bytes of a used cache: every code but NaN, the padding of a head 0."""
        b = torch.empty(shape, dtype=torch.uint8, device="cuda")
        for i in range(0, shape[0], 1024):  # in parts: the float32 draw is four times the bytes
            part = b[i:i + 1024]
            part.copy_((normal(*part.shape) * 100).clamp_(-FP8_MAX, FP8_MAX).to(torch.float8_e4m3fn).view(torch.uint8))
        return b

    k, v = pool((pages, kvh, P, R)), pool((pages, kvh, R, P))
    k[..., hd:] = 0
    v[:, :, hd:] = 0
    ks = torch.exp2(torch.randint(-8, -5, (pages, kvh), generator=g, device="cuda").float())
    vs = torch.exp2(torch.randint(-8, -5, (pages, kvh), generator=g, device="cuda").float())
    s = dict(case=c, k=k, v=v, ks=ks, vs=vs, table=table, starts=starts, lens=lens, N=N, max_new=max(new),
             max_len=max(a + b for a, b in zip(past, new)), max_pages=max_pages, pages=pages)
    if c["kind"] == "append":
        # rows of one projection: queries, keys and values side by side
        s["qkv"] = (normal(N, (heads + 2 * kvh) * hd) * 1.5).to(d)
        s["q_out"] = torch.zeros(N, heads * hd, dtype=d, device="cuda")
        ang = torch.arange(max_pages * P, device="cuda").double()[:, None] \
            * torch.pow(10000.0, -2.0 * torch.arange(hd // 2, device="cuda").double() / hd)[None]
        s["cos"], s["sin"] = ang.cos().float(), ang.sin().float()
    else:
        s["q"] = normal(N, heads * hd).to(d)
        s["out"] = torch.zeros(N, heads * hd, dtype=d, device="cuda")
        s["scale"] = 1.0 / math.sqrt(hd)
    if own:
        _prepare_own(s)
    torch.cuda.synchronize()
    return s


def _prepare_sample(c, g, d, normal):
    B, V = c["B"], c["V"]
    # a few likely tokens above a long tail, as a trained model's rows are
    z = normal(B, V) * 2.0
    z += 6.0 * (torch.rand(B, V, generator=g, device="cuda") < 20.0 / V)
    f = c["filters"]

    def some(lo, hi):
        return torch.rand(B, generator=g, device="cuda") * (hi - lo) + lo

    s = dict(case=c, z=z.to(d), u=torch.rand(B, generator=g, device="cuda"), ids=torch.zeros(B, dtype=torch.int32, device="cuda"),
             temperature=some(0.6, 1.2), top_k=None, top_p=None, min_p=None)
    if f in ("all", "top_k"):
        s["top_k"] = torch.randint(1, max(2, min(V, 1000)), (B,), generator=g, device="cuda").to(torch.int32)
    if f in ("all", "top_p"):
        s["top_p"] = some(0.5, 0.99)
    if f in ("all", "min_p"):
        s["min_p"] = some(0.0, 0.1)
    if own:
        _prepare_own(s)
    torch.cuda.synchronize()
    return s


def _prepare_own(s):
    """The framework's handles: the device, the cache's description, workspaces."""
    import goneuron_amd as gn
    from goneuron_amd._lib import KVCache, check, lib
    c, L, n = s["case"], lib(), C.c_int64()
    s["dev"] = gn.GetDefaultDevice()
    if c["kind"] == "sample":
        check(None, L.gn_sample_workspace(c["B"], c["V"], C.byref(n)))
    else:
        s["kv"] = KVCache(k=s["k"].data_ptr(), v=s["v"].data_ptr(), k_scale=s["ks"].data_ptr(), v_scale=s["vs"].data_ptr(),
                          table=s["table"].data_ptr(), pages=s["pages"], page_size=c["page"], kv_heads=c["kvh"],
                          head_dim=c["hd"], max_pages=s["max_pages"])
        if c["kind"] == "attend":
            check(None, L.gn_kv_attention_workspace(c["B"], s["max_new"], s["max_len"], c["heads"], c["kvh"], c["hd"],
                                                    C.byref(n)))
    s["work"] = torch.empty(max(1, n.value), device="cuda")


# ------------------------------------------------------------------ one pass
def run(state):
    if own:
        return _run_own(state)
    return {"append": _append, "attend": _attend, "sample": _sample}[state["case"]["kind"]](state)


def _answer(s):
    f8 = torch.float8_e4m3fn
    return {"q": s["q_out"], "k": s["k"].view(f8), "v": s["v"].view(f8), "k_scale": s["ks"], "v_scale": s["vs"]}


def _run_own(s):
    from goneuron_amd._lib import check, lib
    c, L, h = s["case"], lib(), s["dev"].h

    def p(name):
        return s[name].data_ptr() if s[name] is not None else None

    if c["kind"] == "sample":
        check(h, L.gn_sample(h, p("z"), c["V"], DCODE[c["dtype"]], p("temperature"), p("top_k"), p("top_p"), p("min_p"),
                             p("u"), p("ids"), c["B"], c["V"], p("work")))
        return s["ids"]
    if c["kind"] == "append":
        e, w = s["qkv"].element_size(), (c["heads"] + 2 * c["kvh"]) * c["hd"]
        q = p("qkv")
        k = q + c["heads"] * c["hd"] * e
        v = k + c["kvh"] * c["hd"] * e
        check(h, L.gn_kv_append(h, C.byref(s["kv"]), q, k, v, p("q_out"), w, w, w, c["heads"] * c["hd"], p("cos"), p("sin"),
                                s["max_pages"] * c["page"], p("starts"), p("lens"), c["B"], s["N"], s["max_new"],
                                c["heads"], DCODE[c["dtype"]], None))
        return _answer(s)
    w = c["heads"] * c["hd"]
    check(h, L.gn_kv_attention(h, C.byref(s["kv"]), p("q"), p("out"), w, w, p("starts"), p("lens"), c["B"], s["N"],
                               s["max_new"], s["max_len"], c["heads"], s["scale"], 1, DCODE[c["dtype"]], p("work"), None))
    return s["out"]


# ------------------------------------------------------------------ the plain forms
def _tokens(s):
    """(sequence, position) of every packed row."""
    n = s["starts"][1:] - s["starts"][:-1]
    b = torch.repeat_interleave(torch.arange(n.numel(), device="cuda"), n, output_size=s["N"])
    return b, torch.arange(s["N"], device="cuda") - s["starts"][b] + s["lens"][b]


def _append(s):
    c = s["case"]
    heads, kvh, hd, P, N = c["heads"], c["kvh"], c["hd"], c["page"], s["N"]
    b, pos = _tokens(s)
    page, slot = s["table"][b, pos // P].long(), pos % P
    q, k, v = s["qkv"].split([heads * hd, kvh * hd, kvh * hd], 1)
    cs, sn, h = s["cos"][pos].double()[:, None], s["sin"][pos].double()[:, None], hd // 2

    def turned(x, nh):  # float64: values next to a quantisation border
        x = x.double().view(N, nh, hd)
        return torch.cat([x[..., :h] * cs - x[..., h:] * sn, x[..., :h] * sn + x[..., h:] * cs], 2)

    s["q_out"].copy_(turned(q, heads).view(N, heads * hd))
    part = (s["lens"] % P != 0) & (s["starts"][1:] > s["starts"][:-1])
    rows = torch.nonzero(part)[:, 0]
    first = s["table"][rows, s["lens"][rows] // P].long()
    held = torch.arange(P, device="cuda")[None] < (s["lens"][rows] % P)[:, None]  # tokens already in those pages
    for x, cache, scale, up in ((turned(k, kvh).float(), s["k"], s["ks"], False), (v.float().view(N, kvh, hd), s["v"], s["vs"], True)):
        most = torch.zeros(s["pages"], kvh, device="cuda").index_reduce_(0, page, x.abs().amax(2), "amax")
        frac, e = torch.frexp(most / FP8_MAX)
        e = torch.where(frac == 0.5, e - 1, e).clamp(min=MIN_EXP)
        e = torch.where(most == 0, torch.full_like(e, MIN_EXP), e)
        fresh = torch.ldexp(torch.ones_like(most), e)
        old = scale[first]
        grown = torch.maximum(old, fresh[first])
        touched = torch.zeros(s["pages"], dtype=torch.bool, device="cuda").index_fill_(0, page, True)
        scale.copy_(torch.where(touched[:, None], fresh, scale))
        scale[first] = grown
        was = cache[first].view(torch.float8_e4m3fn).float() * (old / grown)[:, :, None, None]
        was = was.to(torch.float8_e4m3fn).view(torch.uint8)
        keep = held[:, None, None, :] if up else held[:, None, :, None]
        cache[first] = torch.where(keep, was, cache[first])
        bytes_ = (x / scale[page][:, :, None]).to(torch.float8_e4m3fn).view(torch.uint8)
        if up:
            cache[page, :, :hd, slot] = bytes_
        else:
            cache[page, :, slot, :hd] = bytes_
            cache[page, :, slot, hd:] = 0
    return _answer(s)


def _attend(s):
    c = s["case"]
    B, heads, kvh, hd, P = c["B"], c["heads"], c["kvh"], c["hd"], c["page"]
    G, T, L = heads // kvh, s["max_new"], s["max_pages"] * P
    t = s["table"].long()
    f8 = torch.float8_e4m3fn
    k = s["k"][t][..., :hd].view(f8).float() * s["ks"][t][..., None, None]     # B, pages, KVH, P, hd
    k = k.permute(0, 2, 4, 1, 3).reshape(B, kvh, hd, L)
    v = s["v"][t][:, :, :, :hd].view(f8).float() * s["vs"][t][..., None, None]  # B, pages, KVH, hd, P
    v = v.permute(0, 2, 1, 4, 3).reshape(B, kvh, L, hd)
    n = s["starts"][1:] - s["starts"][:-1]
    step = torch.arange(T, device="cuda")
    real = step[None] < n[:, None]
    row = (s["starts"][:-1, None] + step[None]).clamp(max=s["N"] - 1)
    q = s["q"][row].float().view(B, T, kvh, G, hd).permute(0, 2, 3, 1, 4).reshape(B, kvh, G * T, hd)
    a = torch.matmul(q, k).view(B, kvh, G, T, L) * s["scale"]
    seen = torch.arange(L, device="cuda")[None, None] <= (s["lens"][:, None] + step[None])[:, :, None]
    a = torch.where(seen[:, None, None], a, torch.full((), -math.inf, device="cuda"))
    a = torch.exp(a - a.amax(4, keepdim=True))
    a = a / a.sum(4, keepdim=True)
    o = torch.matmul(a.view(B, kvh, G * T, L), v).view(B, kvh, G, T, hd).permute(0, 3, 1, 2, 4).reshape(B, T, heads * hd)
    s["out"][row[real]] = o[real].to(s["out"].dtype)
    return s["out"]


def _sample(s):
    z = s["z"].double()  # float64: long sums, values next to a border
    B, V = z.shape
    zs, order = z.sort(dim=1, descending=True, stable=True)  # ties: the lowest index first
    w = torch.exp((zs - zs[:, :1]) / s["temperature"].double()[:, None])
    rank = torch.arange(V, device="cuda")[None]
    keep = torch.ones(B, V, dtype=torch.bool, device="cuda")
    if s["top_k"] is not None:
        keep &= rank < s["top_k"][:, None]
    if s["top_p"] is not None:
        cum = torch.cumsum(w * keep, 1)
        before = cum - w * keep
        keep &= before < s["top_p"].double()[:, None] * cum[:, -1:]
    if s["min_p"] is not None:
        keep &= w >= s["min_p"].double()[:, None]
    cum = torch.cumsum(torch.zeros_like(w).scatter_(1, order, w * keep), 1)
    s["ids"].copy_((cum > s["u"].double()[:, None] * cum[:, -1:]).int().argmax(1))
    return s["ids"]


# ------------------------------------------------------------------ the cost
def work(case):
    """Bytes and operations one pass cannot do without: each input read once,
    each output written once, the products of the (query, key) pairs in sight."""
    c = case
    e = 4.0 if c["dtype"] == "f32" else 2.0
    if c["kind"] == "sample":
        return {"bytes": c["B"] * (c["V"] * e + 24.0), "flops": 4.0 * c["B"] * c["V"]}
    past, new = _lengths(c)
    N, hd = sum(new), c["hd"]
    if c["kind"] == "append":
        rows = N * hd
        return {"bytes": rows * (2 * e * c["heads"] + 2 * (e + 1.0) * c["kvh"]) + 4.0 * N * hd,
                "flops": rows * (3.0 * c["heads"] + 8.0 * c["kvh"])}
    pairs = sum(b * a + b * (b + 1) / 2 for a, b in zip(past, new))
    read = sum(a + b for a, b in zip(past, new) if b)
    return {"bytes": 2.0 * read * c["kvh"] * hd + 2 * e * N * c["heads"] * hd, "flops": 4.0 * pairs * c["heads"] * hd}


# ------------------------------------------------------------------ the definition in 64 bits
def exact(case, seed):
    global own
    mine, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = mine
    return {"append": _exact_append, "attend": _exact_attend, "sample": _exact_sample}[case["kind"]](s)


def _e4m3(x):
    """The nearest E4M3 value, ties to the even one, as float64."""
    m, e = np.frexp(np.abs(x))
    step = np.ldexp(1.0, np.maximum(e - 1, -6) - 3)
    return np.minimum(np.round(x / step) * step, FP8_MAX)


def _exact_append(s):
    c = s["case"]
    heads, kvh, hd, P = c["heads"], c["kvh"], c["hd"], c["page"]
    x = s["qkv"].double().cpu().numpy()
    N, h = x.shape[0], hd // 2
    cs, sn = s["cos"].double().cpu().numpy(), s["sin"].double().cpu().numpy()
    table, past, new = s["table"].cpu().numpy(), *_lengths(c)
    K = s["k"].view(torch.float8_e4m3fn).float().cpu().numpy().astype(np.float64)
    V = s["v"].view(torch.float8_e4m3fn).float().cpu().numpy().astype(np.float64).swapaxes(2, 3)
    KS, VS = s["ks"].double().cpu().numpy(), s["vs"].double().cpu().numpy()
    qs, at = np.zeros((N, heads, hd)), 0
    for b in range(c["B"]):
        if not new[b]:
            continue
        pos = np.arange(past[b], past[b] + new[b])
        rows = x[at:at + new[b]]
        q, k = (rows[:, i:j].reshape(new[b], -1, hd) for i, j in ((0, heads * hd), (heads * hd, (heads + kvh) * hd)))
        co, si = cs[pos][:, None], sn[pos][:, None]
        q, k = (np.concatenate([y[..., :h] * co - y[..., h:] * si, y[..., :h] * si + y[..., h:] * co], 2) for y in (q, k))
        qs[at:at + new[b]] = q
        k = k.astype(np.float32).astype(np.float64)  # a rotated key is a float32 number
        v = rows[:, (heads + kvh) * hd:].reshape(new[b], kvh, hd)
        at += new[b]
        for j in range(past[b] // P, -(-(past[b] + new[b]) // P)):
            page, lo, hi = table[b, j], max(past[b] - j * P, 0), min(past[b] + new[b] - j * P, P)
            i = j * P + lo - past[b]
            for X, S, y in ((K, KS, k), (V, VS, v)):
                part = y[i:i + hi - lo].swapaxes(0, 1)
                m = np.abs(part).max((1, 2))
                e = np.where(m > 0, np.ceil(np.log2(np.maximum(m, 1e-300) / FP8_MAX)), MIN_EXP)
                sc = np.exp2(np.maximum(e, MIN_EXP))
                if lo:
                    sc = np.maximum(sc, S[page])
                    X[page, :, :lo] = _e4m3(X[page, :, :lo] * (S[page] / sc)[:, None, None])
                S[page] = sc
                X[page, :, lo:hi, :hd] = _e4m3(part / sc[:, None, None])
                X[page, :, lo:hi, hd:] = 0
    V = np.ascontiguousarray(V.swapaxes(2, 3))
    return {"q": qs.reshape(N, heads * hd), "k": K, "v": V, "k_scale": KS, "v_scale": VS}


def _exact_attend(s):
    c = s["case"]
    kvh, hd, P = c["kvh"], c["hd"], c["page"]
    G = c["heads"] // kvh
    past, new = _lengths(c)
    out, at = [], 0
    for b in range(c["B"]):
        n, length = new[b], past[b] + new[b]
        if not n:
            continue
        pages = s["table"][b, :-(-length // P)].long()
        k = (s["k"][pages].view(torch.float8_e4m3fn).double() * s["ks"][pages].double()[..., None, None]).transpose(0, 1)
        v = (s["v"][pages].view(torch.float8_e4m3fn).double() * s["vs"][pages].double()[..., None, None]).permute(1, 0, 3, 2)
        k = k.reshape(kvh, -1, k.shape[-1])[:, :length, :hd]
        v = v.reshape(kvh, -1, v.shape[-1])[:, :length, :hd]
        q = s["q"][at:at + n].double().view(n, kvh, G, hd)
        o = torch.zeros(n, kvh, G, hd, dtype=torch.float64, device="cuda")
        later = torch.arange(length, device="cuda")[None] > torch.arange(past[b], length, device="cuda")[:, None]
        for h in range(kvh):
            for i in range(G):
                a = torch.mm(q[:, h, i], k[h].t().contiguous()) / math.sqrt(hd)
                o[:, h, i] = torch.mm(torch.softmax(a.masked_fill(later, -math.inf), 1), v[h].contiguous())
        out.append(o.view(n, -1))
        at += n
    return torch.cat(out)


def _exact_sample(s):
    z, u = s["z"].double().cpu().numpy(), s["u"].double().cpu().numpy()
    T = s["temperature"].double().cpu().numpy()
    ids = []
    for r in range(z.shape[0]):
        w = np.exp((z[r] - z[r].max()) / T[r])
        order = np.argsort(-z[r], kind="stable")
        if s["top_k"] is not None:
            order = order[:int(s["top_k"][r])]
        if s["top_p"] is not None:
            cum = np.cumsum(w[order])
            order = order[:int(np.searchsorted(cum, float(s["top_p"][r]) * cum[-1], "left")) + 1]
        if s["min_p"] is not None:
            order = order[w[order] >= float(s["min_p"][r])]
        at = np.sort(order)
        cum = np.cumsum(w[at])
        ids.append(int(at[int(np.searchsorted(cum, u[r] * cum[-1], "right"))]))
    return np.array(ids, np.int32)
