"""Timed calls of the operators for drafted tokens, long streams and steered
logits: attention with a sliding window and sinks, attention of a tree of
drafted tokens, the append of such a tree, the move of its accepted path, and
penalties, biases and grammar masks on logits.

A case is a dict of plain values; ``prepare`` makes what a serving program
holds before the call, ``run`` makes one pass, through the framework's entry
points where ``own`` is true and otherwise as elementary torch operations, and
``exact`` restates it in float64 from the definition.

The cache: pages of P tokens in E4M3, K as [pages][KVH][P][R] and V as
[pages][KVH][R][P] bytes (R: the head size padded), with a power-of-two scale
per page and head for each.  Sequence b's new tokens are the rows starts[b] ..
starts[b+1] - 1 of the packed inputs and stand at lens[b], lens[b] + 1, ... of
the sequence.

Families (``kind``):
  window   softmax(q K^T) V over the last `window` tokens and the first `sinks`
  tree     the same over all cached tokens and a drafted token's ancestors
  append   rotate a tree's tokens by their depth, quantise them into pages
  keep     move the accepted path of a tree behind what was cached
  adjust   logits with penalties, biases and a grammar's bit mask
"""
import ctypes as C
import math

import numpy as np
import torch

own = False

DT = {"f32": torch.float32, "bf16": torch.bfloat16}
DCODE = {"f32": 0, "bf16": 1}
FP8_MAX, MIN_EXP = 448.0, -100
F8 = torch.float8_e4m3fn


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # a token of a few sequences of the small language model (8 heads of 32) with half its context in sight
        dict(name="window_step_small", kind="window", dtype="f32", B=4, heads=8, kvh=8, hd=32, page=16,
             new=1, past=127, ragged=False, sinks=4, window=64),
        # a token of every sequence of a busy server, most of them far beyond their window
        dict(name="window_step_batch", kind="window", dtype="bf16", B=64, heads=32, kvh=8, hd=128, page=64,
             new=1, past=16383, ragged=True, sinks=4, window=4096),
        # the next part of two long prompts
        dict(name="window_prompt", kind="window", dtype="bf16", B=2, heads=32, kvh=8, hd=128, page=64,
             new=2048, past=2048, ragged=False, sinks=4, window=1024),
        # a few drafted tokens of the small language model: latency
        dict(name="tree_small", kind="tree", dtype="f32", B=4, heads=8, kvh=8, hd=32, page=16,
             new=16, past=120, ragged=False),
        # trees of every sequence of a server
        dict(name="tree_batch", kind="tree", dtype="bf16", B=16, heads=32, kvh=8, hd=128, page=64,
             new=64, past=8000, ragged=True),
        # odd sizes behind long histories: an 80-wide head, three queries a key head
        dict(name="tree_long_f32", kind="tree", dtype="f32", B=3, heads=12, kvh=4, hd=80, page=32,
             new=37, past=33333, ragged=True),
        # odd sizes: short and empty trees among longer ones
        dict(name="append_ragged_f32", kind="append", dtype="f32", B=7, heads=12, kvh=4, hd=80, page=32,
             new=37, past=77, ragged=True),
        # trees of every sequence of a busy server
        dict(name="append_batch", kind="append", dtype="bf16", B=64, heads=32, kvh=8, hd=128, page=64,
             new=64, past=2000, ragged=True),
        # the small language model's accepted tokens: latency
        dict(name="keep_small", kind="keep", B=4, kvh=8, hd=32, page=16, new=16, past=120, ragged=False),
        # those of a busy server
        dict(name="keep_batch", kind="keep", B=64, kvh=8, hd=128, page=64, new=64, past=2000, ragged=True),
        # a few rows of an odd vocabulary
        dict(name="adjust_small", kind="adjust", dtype="bf16", B=5, V=50257, history=300, rules="all"),
        # a busy server's step over a large vocabulary, with long histories
        dict(name="adjust_batch", kind="adjust", dtype="f32", B=128, V=131072, history=4096, rules="all"),
    ]


def _logint(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["window", "window", "window", "tree", "tree", "append", "keep", "adjust", "adjust"])
    dtype = rng.choice(["f32", "bf16"])
    if kind == "adjust":
        return dict(kind=kind, dtype=dtype, B=_logint(rng, 1, 128), V=_logint(rng, 100, 131072), history=_logint(rng, 1, 4096),
                    rules=rng.choice(["all", "penalties", "bias", "mask"]))
    while True:
        kvh = rng.choice([1, 2, 3, 4, 8])
        c = dict(kind=kind, dtype=dtype, B=_logint(rng, 1, 64), heads=kvh * rng.choice([1, 1, 2, 3, 4, 7, 8]), kvh=kvh,
                 hd=rng.choice([16, 32, 48, 64, 72, 80, 96, 128, 192, 256]), page=rng.choice([16, 32, 64, 128]),
                 new=_logint(rng, 2, 128), past=_logint(rng, 1, 16384), ragged=rng.random() < 0.7)
        if kind == "window":
            c.update(new=1 if rng.random() < 0.55 else _logint(rng, 2, 2048), sinks=rng.choice([0, 1, 4, 4, 16, 100]),
                     window=_logint(rng, 16, 8192))
        if kind == "keep":
            del c["dtype"], c["heads"]
        elif c["heads"] > 32:
            continue
        rows = c["B"] * c["kvh"] * (c["new"] + c["past"] + 128) * c["hd"]
        if kind in ("append", "keep"):
            if rows <= 3e8 and c["B"] * c["new"] * c["kvh"] * c["hd"] <= 4e6:
                return c
            continue
        seen = c["past"] + c["new"] if kind == "tree" else min(c["past"], c["window"] + c["sinks"]) + c["new"]
        cells = c["B"] * c["heads"] * c["new"] * seen
        top = 3.5e10 if dtype == "bf16" else 1.0e10
        if rows <= 4e8 and cells <= 2.5e8 and 4.0 * cells * c["hd"] <= top:
            return c


# ------------------------------------------------------------------ shapes
def _row(hd):
    return next(r for r in (32, 64, 96, 128, 192, 256) if r >= hd)


def _lengths(c):
    """(past, new) tokens of every sequence: whole numbers that go by the case
    alone.  Ragged: spread between none and the case's sizes, one sequence at
    the largest, one of several without new tokens."""
    B, past, new = c["B"], c["past"], c["new"]
    if not c["ragged"]:
        return [past] * B, [new] * B
    r = np.random.RandomState(B * 6151 + past * 37 + new)
    p = [int(x) for x in r.randint(0, past + 1, B)]
    n = [int(x) for x in r.randint(1, new + 1, B)]
    p[0], n[0] = past, new
    if B > 2 and new > 1:
        n[1] = 0
    return p, n


def _trees(c):
    """Each sequence's drafted tree, by the case alone: a token's parent (an
    earlier one, or -1: it follows the cached tokens).  Most tokens carry a
    branch on, some open another."""
    r = np.random.RandomState(c["new"] * 613 + c["B"] * 17 + c["past"])
    out = []
    for n in _lengths(c)[1]:
        p = [-1] * n
        for i in range(1, n):
            p[i] = i - 1 if r.rand() < 0.7 else int(r.randint(-1, i))
        out.append(p)
    return out


def _depths(parents):
    d = []
    for p in parents:
        d.append(d[p] + 1 if p >= 0 else 0)
    return d


def _ancestors(parents):
    n = len(parents)
    m = np.zeros((n, n), bool)
    for i, p in enumerate(parents):
        if p >= 0:
            m[i] = m[p]
        m[i, i] = True
    return m


def _path(parents, r):
    """An accepted path: from the root to a token of the tree, cut where one of
    its tokens would be overwritten by a later one (a second call on the same
    state then moves the same tokens)."""
    i, p = int(r.randint(len(parents))), []
    while i >= 0:
        p.append(i)
        i = parents[i]
    p = p[::-1]
    m = len(p)
    while any(p[k] != k and p[k] < m for k in range(m)):
        m -= 1
    return p[:m]


# ------------------------------------------------------------------ what a program holds
def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda").manual_seed(int(seed) * 1000003 + 41)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    s = _prepare_logits(c, g, normal, int(seed)) if c["kind"] == "adjust" else _prepare_cache(c, g, normal, int(seed))
    if own:
        _prepare_own(s)
    torch.cuda.synchronize()
    return s


def _prepare_cache(c, g, normal, seed):
    B, kvh, hd, P, R = c["B"], c["kvh"], c["hd"], c["page"], _row(c["hd"])
    past, new = _lengths(c)
    N, most = sum(new), max(new)
    per = [-(-(a + b) // P) for a, b in zip(past, new)]
    # the first pages that a query sees, and the first of the window: those between were given back
    near, far = [0] * B, [0] * B
    if c["kind"] == "window":
        far = [min(-(-c["sinks"] // P), n) for n in per]
        near = [max(f, max(0, a - c["window"] + 1) // P) for a, f in zip(past, far)]
    held = [f + n - m for f, n, m in zip(far, per, near)]
    max_pages, pages = max(1, max(per)), sum(held) + 3
    # pages are handed out in any order, as a server's free list gives them
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    j = torch.arange(max_pages, device="cuda")[None]
    base, far_, near_ = (torch.tensor(x, device="cuda")[:, None] for x in ([sum(held[:b]) for b in range(B)], far, near))
    table = order[(base + torch.where(j < far_, j, far_ + j - near_)).clamp(0, pages - 1)]
    table = torch.where((j >= far_) & (j < near_), torch.full_like(table, -1), table).contiguous()

    def pool(shape):
        """Bytes of a used cache: every code but NaN, the padding of a head 0."""
        b = torch.empty(shape, dtype=torch.uint8, device="cuda")
        for i in range(0, shape[0], 1024):  # in parts: the float32 draw is four times the bytes
            part = b[i:i + 1024]
            part.copy_((normal(*part.shape) * 100).clamp_(-FP8_MAX, FP8_MAX).to(F8).view(torch.uint8))
        return b

    k, v = pool((pages, kvh, P, R)), pool((pages, kvh, R, P))
    k[..., hd:] = 0
    v[:, :, hd:] = 0
    ks, vs = (torch.exp2(torch.randint(-8, -5, (pages, kvh), generator=g, device="cuda").float()) for _ in range(2))
    starts = torch.tensor([sum(new[:b]) for b in range(B + 1)], dtype=torch.int32, device="cuda")
    s = dict(case=c, k=k, v=v, ks=ks, vs=vs, table=table, starts=starts, N=N, max_new=most, max_pages=max_pages, pages=pages,
             lens=torch.tensor(past, dtype=torch.int32, device="cuda"), max_len=max(a + b for a, b in zip(past, new)))
    if c["kind"] in ("window", "tree"):
        s["q"] = normal(N, c["heads"] * hd).to(DT[c["dtype"]])
        s["out"] = torch.zeros_like(s["q"])
        s["scale"] = 1.0 / math.sqrt(hd)
    if c["kind"] == "tree":
        words = -(-most // 32)
        m = np.zeros((N, words * 32), bool)
        for at, p in zip(np.cumsum([0] + new), _trees(c)):
            m[at:at + len(p), :len(p)] = _ancestors(p)
        bits = np.packbits(m, axis=1, bitorder="little").reshape(N, words, 4).view("<i4").reshape(N, words)
        s["mask"] = torch.from_numpy(np.ascontiguousarray(bits)).cuda()
    if c["kind"] == "append":
        # rows of one projection: queries, keys and values side by side
        s["qkv"] = (normal(N, (c["heads"] + 2 * kvh) * hd) * 1.5).to(DT[c["dtype"]])
        s["q_out"] = torch.zeros(N, c["heads"] * hd, dtype=DT[c["dtype"]], device="cuda")
        at = [a + d for a, p in zip(past, _trees(c)) for d in _depths(p)]
        s["positions"] = torch.tensor(at, dtype=torch.int32, device="cuda")
        ang = torch.arange(max_pages * P, device="cuda").double()[:, None] \
            * torch.pow(10000.0, -2.0 * torch.arange(hd // 2, device="cuda").double() / hd)[None]
        s["cos"], s["sin"] = ang.cos().float(), ang.sin().float()
    if c["kind"] == "keep":
        r = np.random.RandomState(seed % (1 << 31))
        paths = [_path(p, r) if p else [] for p in _trees(c)]
        keep = np.zeros(N, np.int32)
        for at, p in zip(np.cumsum([0] + new), paths):
            keep[at:at + len(p)] = p
        s["keep"] = torch.from_numpy(keep).cuda()
        s["counts"] = torch.tensor([len(p) for p in paths], dtype=torch.int32, device="cuda")
    return s


def _prepare_logits(c, g, normal, seed):
    B, V, H, rules = c["B"], c["V"], c["history"], c["rules"]
    # a few likely tokens above a long tail, as a trained model's rows are
    z = normal(B, V) * 2.0
    z += 6.0 * (torch.rand(B, V, generator=g, device="cuda") < 20.0 / V)
    z = z.to(DT[c["dtype"]])

    def some(lo, hi):
        return torch.rand(B, generator=g, device="cuda") * (hi - lo) + lo

    def upto(n, *shape):
        return torch.randint(0, n, shape, generator=g, device="cuda").to(torch.int32)

    s = dict(case=c, z=z, out=torch.zeros_like(z), repetition=None, frequency=None, presence=None, tokens=None, token_lens=None,
             prompt_lens=None, bias_ids=None, bias=None, bias_lens=None, allowed=None, allowed_row=None)
    if rules in ("all", "penalties"):
        # text repeats itself: the square of a uniform number makes some tokens frequent
        s["tokens"] = (torch.rand(B, H, generator=g, device="cuda").square() * V).to(torch.int32).clamp(max=V - 1)
        s["token_lens"] = upto(H, B) + 1
        s["prompt_lens"] = (s["token_lens"] * torch.rand(B, generator=g, device="cuda")).to(torch.int32)
        s["repetition"], s["frequency"], s["presence"] = some(1.0, 1.3), some(0.0, 0.5), some(0.0, 0.5)
    if rules in ("all", "bias"):
        s["bias_ids"], s["bias"], s["bias_lens"] = upto(V, B, 64), normal(B, 64) * 4.0, upto(65, B)
    if rules in ("all", "mask"):
        words = -(-V // 32)
        rows = max(1, B // 2)
        # some grammars leave a few tokens, some nearly all; every second row has one
        share = torch.rand(rows, 1, generator=g, device="cuda").square()
        bits = (torch.rand(rows, words * 32, generator=g, device="cuda") < share).view(rows, words, 32).long()
        word = (bits << torch.arange(32, device="cuda")).sum(2)
        s["allowed"] = torch.where(word >= 1 << 31, word - (1 << 32), word).to(torch.int32)
        b = torch.arange(B, device="cuda", dtype=torch.int32)
        s["allowed_row"] = torch.where(b % 2 == 0, (b // 2) % rows, torch.full_like(b, -1))
    return s


def _prepare_own(s):
    """The framework's handles: the device, descriptions, workspaces."""
    import goneuron_amd as gn
    from goneuron_amd._lib import KVCache, LogitRules, check, lib
    c, L = s["case"], lib()
    s["dev"] = gn.GetDefaultDevice()

    def p(name):
        return s[name].data_ptr() if s[name] is not None else None

    if c["kind"] == "adjust":
        s["rules"] = LogitRules(
            repetition=p("repetition"), frequency=p("frequency"), presence=p("presence"), tokens=p("tokens"),
            token_lens=p("token_lens"), prompt_lens=p("prompt_lens"), tokens_stride=c["history"], bias_ids=p("bias_ids"),
            bias=p("bias"), bias_lens=p("bias_lens"), bias_stride=64 if s["bias"] is not None else 0, allowed=p("allowed"),
            allowed_row=p("allowed_row"), allowed_stride=-(-c["V"] // 32), allowed_rows=max(1, c["B"] // 2))
        return
    s["kv"] = KVCache(k=p("k"), v=p("v"), k_scale=p("ks"), v_scale=p("vs"), table=p("table"), pages=s["pages"],
                      page_size=c["page"], kv_heads=c["kvh"], head_dim=c["hd"], max_pages=s["max_pages"])
    if c["kind"] in ("window", "tree"):
        n = C.c_int64()
        check(None, L.gn_kv_attention_workspace(c["B"], s["max_new"], s["max_len"], c["heads"], c["kvh"], c["hd"], C.byref(n)))
        s["work"] = torch.empty(max(1, n.value), device="cuda")


# ------------------------------------------------------------------ one pass
def run(state):
    if own:
        return _run_own(state)
    return {"window": _window, "tree": _tree, "append": _append, "keep": _keep, "adjust": _adjust}[state["case"]["kind"]](state)


def _cache_of(s):
    return {"k": s["k"].view(F8), "v": s["v"].view(F8), "k_scale": s["ks"], "v_scale": s["vs"]}


def _run_own(s):
    from goneuron_amd._lib import check, lib
    c, L, h = s["case"], lib(), s["dev"].h

    def p(name):
        return s[name].data_ptr()

    if c["kind"] == "adjust":
        check(h, L.gn_logits_adjust(h, p("z"), c["V"], p("out"), c["V"], DCODE[c["dtype"]], C.byref(s["rules"]), c["B"], c["V"]))
        return s["out"]
    if c["kind"] == "keep":
        check(h, L.gn_kv_keep(h, C.byref(s["kv"]), p("keep"), p("counts"), p("starts"), p("lens"), c["B"], s["N"], s["max_new"],
                              None))
        return _cache_of(s)
    w = c["heads"] * c["hd"]
    if c["kind"] == "append":
        e, row = s["qkv"].element_size(), (c["heads"] + 2 * c["kvh"]) * c["hd"]
        q = p("qkv")
        k = q + w * e
        v = k + c["kvh"] * c["hd"] * e
        check(h, L.gn_kv_append_at(h, C.byref(s["kv"]), q, k, v, p("q_out"), row, row, row, w, p("cos"), p("sin"),
                                   s["max_pages"] * c["page"], p("positions"), p("starts"), p("lens"), c["B"], s["N"],
                                   s["max_new"], c["heads"], DCODE[c["dtype"]], None))
        return {"q": s["q_out"], **_cache_of(s)}
    if c["kind"] == "tree":
        check(h, L.gn_kv_attention_tree(h, C.byref(s["kv"]), p("q"), p("out"), w, w, p("mask"), s["mask"].shape[1], p("starts"),
                                        p("lens"), c["B"], s["N"], s["max_new"], s["max_len"], c["heads"], s["scale"],
                                        DCODE[c["dtype"]], p("work"), None))
    else:
        check(h, L.gn_kv_attention_window(h, C.byref(s["kv"]), p("q"), p("out"), w, w, p("starts"), p("lens"), c["B"], s["N"],
                                          s["max_new"], s["max_len"], c["heads"], s["scale"], c["sinks"], c["window"],
                                          DCODE[c["dtype"]], p("work"), None))
    return s["out"]


# ------------------------------------------------------------------ the plain forms
def _inf():
    return torch.full((), -math.inf, device="cuda")


def _rows_of(s):
    """Each sequence's new tokens, padded to the most: (row of the packed inputs, whether there is one)."""
    n, step = s["starts"][1:] - s["starts"][:-1], torch.arange(s["max_new"], device="cuda")
    return (s["starts"][:-1, None] + step[None]).clamp(max=max(s["N"] - 1, 0)), step[None] < n[:, None]


def _attend(s, pos, seen):
    """Attention of the new tokens to the keys at the positions pos [B, L], as far as seen [B, T, L] says."""
    c = s["case"]
    B, heads, kvh, hd, P, T, Lk = c["B"], c["heads"], c["kvh"], c["hd"], c["page"], s["max_new"], pos.shape[1]
    G = heads // kvh
    page = torch.gather(s["table"], 1, (pos // P).clamp(0, s["max_pages"] - 1)).long().clamp(min=0)
    slot = pos % P
    h = torch.arange(kvh, device="cuda")[None, :, None]
    k = s["k"].view(F8)[page[:, None], h, slot[:, None]][..., :hd].float() * s["ks"][page].transpose(1, 2)[..., None]
    v = s["v"][:, :, :hd].transpose(2, 3)[page[:, None], h, slot[:, None]].view(F8).float() * s["vs"][page].transpose(1, 2)[..., None]
    row, real = _rows_of(s)
    q = s["q"][row].float().view(B, T, kvh, G, hd).permute(0, 2, 3, 1, 4).reshape(B, kvh, G * T, hd)
    a = torch.matmul(q, k.transpose(2, 3).contiguous()).view(B, kvh, G, T, Lk) * s["scale"]
    a = torch.where(seen[:, None, None], a, _inf())
    a = torch.exp(a - a.amax(4, keepdim=True))
    a = a / a.sum(4, keepdim=True)
    o = torch.matmul(a.view(B, kvh, G * T, Lk), v).view(B, kvh, G, T, hd).permute(0, 3, 1, 2, 4).reshape(B, T, heads * hd)
    s["out"][row[real]] = o[real].to(s["out"].dtype)
    return s["out"]


def _window(s):
    c = s["case"]
    # the first tokens, then those of the sequence's whole window
    most = min(c["window"], s["max_len"])
    near = s["lens"].long()[:, None] - (most - 1) + torch.arange(most + s["max_new"] - 1, device="cuda")[None]
    first = torch.arange(c["sinks"], device="cuda")[None].expand(c["B"], -1)
    pos = torch.cat([first, near], 1)
    again = torch.cat([torch.zeros_like(first, dtype=torch.bool), near < c["sinks"]], 1)  # sinks inside the window, and nothing
    at = s["lens"].long()[:, None] + torch.arange(s["max_new"], device="cuda")[None]
    d = at[:, :, None] - pos[:, None]
    seen = (d >= 0) & ((d < c["window"]) | (pos < c["sinks"])[:, None]) & ~again[:, None]
    return _attend(s, pos.clamp(min=0), seen)


def _tree(s):
    T = s["max_new"]
    pos = torch.arange(s["max_len"], device="cuda")[None].expand(s["case"]["B"], -1)
    j = pos - s["lens"].long()[:, None]  # the new token's number
    row, _ = _rows_of(s)
    bits = (s["mask"][row][..., None] >> torch.arange(32, device="cuda", dtype=torch.int32) & 1).flatten(2).bool()  # B, T, words * 32
    bits = torch.gather(bits, 2, j.clamp(0, T - 1)[:, None].expand(-1, T, -1))
    return _attend(s, pos, (j < 0)[:, None] | (bits & (j < T)[:, None]))


def _tokens(s):
    """(sequence, place in it) of every packed row."""
    n = s["starts"][1:] - s["starts"][:-1]
    b = torch.repeat_interleave(torch.arange(n.numel(), device="cuda"), n, output_size=s["N"])
    return b, torch.arange(s["N"], device="cuda") - s["starts"][b] + s["lens"][b]


def _append(s):
    c = s["case"]
    heads, kvh, hd, P, N = c["heads"], c["kvh"], c["hd"], c["page"], s["N"]
    b, place = _tokens(s)
    page, slot = s["table"][b, place // P].long(), place % P
    pos = s["positions"].long()
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

    def store(x, cache, scale, up):
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
        was = (cache[first].view(F8).float() * (old / grown)[:, :, None, None]).to(F8).view(torch.uint8)
        cache[first] = torch.where(held[:, None, None, :] if up else held[:, None, :, None], was, cache[first])
        bytes_ = (x / scale[page][:, :, None]).to(F8).view(torch.uint8)
        if up:
            cache[page, :, :hd, slot] = bytes_
        else:
            cache[page, :, slot, :hd] = bytes_
            cache[page, :, slot, hd:] = 0

    store(turned(k, kvh).float(), s["k"], s["ks"], False)
    store(v.float().view(N, kvh, hd), s["v"], s["vs"], True)
    return {"q": s["q_out"], **_cache_of(s)}


def _keep(s):
    c = s["case"]
    kvh, P = c["kvh"], c["page"]
    b, place = _tokens(s)
    i = place - s["lens"][b]
    at = torch.nonzero(i < s["counts"][b])[:, 0]
    b, i, place = b[at], i[at], place[at]
    come = s["lens"][b] + s["keep"][at]
    to, from_ = s["table"][b, place // P].long(), s["table"][b, come // P].long()
    to_slot, from_slot = place % P, come % P

    def move(cache, scale, up):
        fresh = scale.clone().index_reduce_(0, to, scale[from_], "amax")
        moved = (cache[from_, :, :, from_slot] if up else cache[from_, :, from_slot]).view(F8).float()
        moved = (moved * (scale[from_] / fresh[to])[..., None]).to(F8).view(torch.uint8)
        cache[to] = (cache[to].view(F8).float() * (scale / fresh)[to][..., None, None]).to(F8).view(torch.uint8)
        if up:
            cache[to, :, :, to_slot] = moved
        else:
            cache[to, :, to_slot] = moved
        scale.copy_(fresh)

    move(s["k"], s["ks"], False)
    move(s["v"], s["vs"], True)
    return _cache_of(s)


def _adjust(s):
    z = s["z"].float()
    B, V = z.shape
    if s["tokens"] is not None:
        ids, j = s["tokens"].long(), torch.arange(s["tokens"].shape[1], device="cuda")[None]
        live = j < s["token_lens"][:, None]
        some = torch.zeros(B, V, device="cuda").scatter_add_(1, ids, live.float())
        later = torch.zeros(B, V, device="cuda").scatter_add_(1, ids, (live & (j >= s["prompt_lens"][:, None])).float())
        r = s["repetition"][:, None]
        z = torch.where(some > 0, torch.where(z > 0, z / r, z * r), z)
        z = z - s["frequency"][:, None] * later - s["presence"][:, None] * (later > 0)
    if s["bias"] is not None:  # of an id's several entries the last
        ids, j = s["bias_ids"].long(), torch.arange(s["bias"].shape[1], device="cuda")[None]
        j = torch.where(j < s["bias_lens"][:, None], j, torch.full_like(j, -1))
        last = torch.full((B, V), -1, device="cuda").scatter_reduce_(1, ids, j, "amax")
        z = torch.where(last >= 0, z + torch.gather(s["bias"], 1, last.clamp(min=0)), z)
    if s["allowed"] is not None:
        bits = (s["allowed"][s["allowed_row"].clamp(min=0).long()][..., None] >> torch.arange(32, device="cuda", dtype=torch.int32)) & 1
        z = torch.where((s["allowed_row"] < 0)[:, None] | bits.flatten(1)[:, :V].bool(), z, _inf())
    s["out"].copy_(z)
    return s["out"]


# ------------------------------------------------------------------ the cost
def work(case):
    """Bytes and operations one pass cannot do without: each input read once,
    each output written once, the products of the (query, key) pairs in sight."""
    c = case
    e = 4.0 if c.get("dtype") == "f32" else 2.0
    if c["kind"] == "adjust":
        more = {"all": 1, "penalties": 1}.get(c["rules"], 0) * 2.0 * c["history"]  # half of the history on average
        more += {"all": 1, "bias": 1}.get(c["rules"], 0) * 8.0 * 32
        mask = {"all": 1, "mask": 1}.get(c["rules"], 0) * max(1, c["B"] // 2) * c["V"] / 8.0
        return {"bytes": c["B"] * (2.0 * c["V"] * e + more) + mask, "flops": 6.0 * c["B"] * c["V"]}
    past, new = _lengths(c)
    N, hd = sum(new), c["hd"]
    if c["kind"] == "keep":
        r = np.random.RandomState(0)
        moved = sum(sum(k != i for i, k in enumerate(_path(p, r))) for p in _trees(c) if p)
        return {"bytes": 4.0 * moved * c["kvh"] * hd + 8.0 * N, "flops": 2.0 * moved * c["kvh"] * hd}
    if c["kind"] == "append":
        rows = N * hd
        return {"bytes": rows * (2 * e * c["heads"] + 2 * (e + 1.0) * c["kvh"]) + 4.0 * rows,
                "flops": rows * (3.0 * c["heads"] + 8.0 * c["kvh"])}
    if c["kind"] == "tree":
        pairs = sum(b * a for a, b in zip(past, new)) + sum(sum(_depths(p)) + len(p) for p in _trees(c))
        read = sum(a + b for a, b in zip(past, new) if b)
    else:
        pairs, read = 0, 0
        for a, b in zip(past, new):
            p = np.arange(a, a + b)
            low = np.maximum(p - c["window"] + 1, 0)
            pairs += int((p + 1 - low + np.minimum(low, c["sinks"])).sum())
            read += (a + b - int(low[0]) + min(int(low[0]), c["sinks"])) if b else 0
    return {"bytes": 2.0 * read * c["kvh"] * hd + 2 * e * N * c["heads"] * hd, "flops": 4.0 * pairs * c["heads"] * hd}


# ------------------------------------------------------------------ the definition in 64 bits
def exact(case, seed):
    global own
    mine, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = mine
    return {"window": _exact_attention, "tree": _exact_attention, "append": _exact_append, "keep": _exact_keep,
            "adjust": _exact_adjust}[case["kind"]](s)


def _exact_attention(s):
    c = s["case"]
    kvh, hd, P = c["kvh"], c["hd"], c["page"]
    G = c["heads"] // kvh
    past, new = _lengths(c)
    trees = _trees(c) if c["kind"] == "tree" else None
    out, at = [], 0
    for b in range(c["B"]):
        n, length = new[b], past[b] + new[b]
        if not n:
            continue
        i, j = np.arange(past[b], length)[:, None], np.arange(length)[None]
        if trees:
            see = np.ones((n, length), bool)
            see[:, past[b]:] = _ancestors(trees[b])
        else:
            see = (j <= i) & ((j < c["sinks"]) | (i - j < c["window"]))
        used = np.flatnonzero(see.any(0))
        hide = torch.from_numpy(~see[:, used]).cuda()
        used = torch.from_numpy(used).cuda()
        page, slot = s["table"][b].long()[used // P], used % P
        k = s["k"][page, :, slot].view(F8).double() * s["ks"][page].double()[..., None]
        v = s["v"][page, :, :, slot].view(F8).double() * s["vs"][page].double()[..., None]
        q = s["q"][at:at + n].double().view(n, kvh, G, hd)
        o = torch.zeros(n, kvh, G, hd, dtype=torch.float64, device="cuda")
        for h in range(kvh):
            kh, vh = k[:, h, :hd].t().contiguous(), v[:, h, :hd].contiguous()
            for r in range(G):
                a = torch.mm(q[:, h, r].contiguous(), kh) / math.sqrt(hd)
                o[:, h, r] = torch.mm(torch.softmax(a.masked_fill(hide, -math.inf), 1), vh)
        out.append(o.view(n, -1))
        at += n
    return torch.cat(out)


def _e4m3(x):
    """The nearest E4M3 value, ties to the even one, as float64."""
    m, e = np.frexp(np.abs(x))
    step = np.ldexp(1.0, np.maximum(e - 1, -6) - 3)
    return np.copysign(np.minimum(np.round(np.abs(x) / step) * step, FP8_MAX), x)


def _values(cache):
    return cache.view(F8).float().cpu().numpy().astype(np.float64)


def _exact_append(s):
    c = s["case"]
    heads, kvh, hd, P = c["heads"], c["kvh"], c["hd"], c["page"]
    x = s["qkv"].double().cpu().numpy()
    N, h = x.shape[0], hd // 2
    cs, sn = s["cos"].double().cpu().numpy(), s["sin"].double().cpu().numpy()
    table, past, new = s["table"].cpu().numpy(), *_lengths(c)
    K, V = _values(s["k"]), _values(s["v"]).swapaxes(2, 3)
    KS, VS = s["ks"].double().cpu().numpy(), s["vs"].double().cpu().numpy()
    qs, at = np.zeros((N, heads, hd)), 0
    for b, parents in enumerate(_trees(c)):
        if not new[b]:
            continue
        pos = past[b] + np.array(_depths(parents))
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
    return {"q": qs.reshape(N, heads * hd), "k": K, "v": np.ascontiguousarray(V.swapaxes(2, 3)), "k_scale": KS, "v_scale": VS}


def _exact_keep(s):
    c = s["case"]
    P = c["page"]
    table, keep, counts, past, new = s["table"].cpu().numpy(), s["keep"].cpu().numpy(), s["counts"].cpu().numpy(), *_lengths(c)
    K, V = _values(s["k"]), np.ascontiguousarray(_values(s["v"]).swapaxes(2, 3))
    KS, VS = s["ks"].double().cpu().numpy(), s["vs"].double().cpu().numpy()
    at = np.cumsum([0] + new)
    for X, S in ((K, KS), (V, VS)):
        for b in range(c["B"]):
            path = past[b] + keep[at[b]:at[b] + counts[b]]
            come = [(X[table[b, p // P], :, p % P].copy(), S[table[b, p // P]].copy()) for p in path]
            to = [table[b, (past[b] + i) // P] for i in range(len(come))]
            for page in set(to):
                more = np.max([S[page]] + [sc for p, (_, sc) in zip(to, come) if p == page], 0)
                X[page] = _e4m3(X[page] * (S[page] / more)[:, None, None])
                S[page] = more
            for i, (page, (x, sc)) in enumerate(zip(to, come)):
                X[page, :, (past[b] + i) % P] = _e4m3(x * (sc / S[page])[:, None])
    return {"k": K, "v": np.ascontiguousarray(V.swapaxes(2, 3)), "k_scale": KS, "v_scale": VS}


def _exact_adjust(s):
    h = {k: None if s[k] is None else s[k].cpu().numpy() for k in
         ("tokens", "token_lens", "prompt_lens", "bias_ids", "bias", "bias_lens", "allowed", "allowed_row")}
    out = s["z"].double().cpu().numpy()
    B, V = out.shape
    for b in range(B):
        z = out[b]
        if h["tokens"] is not None:
            r, f, p = (float(s[k][b]) for k in ("repetition", "frequency", "presence"))
            t = h["tokens"][b, :h["token_lens"][b]]
            used = np.unique(t)
            z[used] = np.where(z[used] > 0, z[used] / r, z[used] * r)
            ids, times = np.unique(t[h["prompt_lens"][b]:], return_counts=True)
            z[ids] -= f * times + p
        if h["bias"] is not None:
            n = h["bias_lens"][b]
            last = dict(zip(h["bias_ids"][b, :n].tolist(), h["bias"][b, :n].astype(np.float64).tolist()))
            for i, x in last.items():
                z[i] += x
        if h["allowed"] is not None and h["allowed_row"][b] >= 0:
            bits = np.unpackbits(h["allowed"][h["allowed_row"][b]].view(np.uint8), bitorder="little")[:V]
            z[bits == 0] = -np.inf
    return out
