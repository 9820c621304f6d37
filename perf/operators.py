"""The attention block of a quantized decoder, operator by operator, as cases
that can be timed and checked.

A case is a dict of plain values.  Five kinds, by the "kind" key:

  linear   an int8 W8A8 linear: activations quantized per token, weights held
           as int8 with a scale per output channel
  rope     rotary positions on the queries and keys of T tokens
  append   the same, with the keys and values stored in the pages of a cache
  attend   attention of one new token per sequence over a paged cache
  fork     finished sequences freed, then prompts forked into samples
  compact  the used pages of a cache moved to its low end

listed() holds the fixed cases, draw() makes more of the same ranges,
prepare() what a program holds before the call, run() is the call (the plain
form, or this library's operators where `own` is true), exact() the result in
64 bits.
"""
import math

import numpy as np
import torch

own = False

DTYPE = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16,
         "e4m3": torch.float8_e4m3fn}
SIZE = {"f32": 4, "f16": 2, "bf16": 2, "e4m3": 1}


def listed():
    return [
        # qkv projection of an 8B decoder for eight sequences: a stream of the
        # weight, where launches and host cost count too.
        dict(name="linear_decode_8", kind="linear", M=8, K=4096, N=6144, t="bf16", bias=False),
        # A short prompt through a matrix whose sizes fit no tile.
        dict(name="linear_ragged_201", kind="linear", M=201, K=3520, N=9001, t="f16", bias=True),
        # Prefill of a long prompt through the gate projection.
        dict(name="linear_prefill_4096", kind="linear", M=4096, K=4096, N=14336, t="bf16",
             bias=False),
        # One decode step of 32 sequences far into a stretched context:
        # rotation fused with the store into the cache.
        dict(name="append_decode_32", kind="append", T=32, Hq=32, Hkv=8, D=128, rot=128,
             inter=False, scaling="yarn", far=1 << 20, S=16, pages=2048, cache="bf16", t="bf16"),
        # A prompt of odd length stored as 8-bit pages; part of the head turns.
        dict(name="append_prompt_2047", kind="append", T=2047, Hq=16, Hkv=4, D=128, rot=96,
             inter=True, scaling="linear", far=2047, S=64, pages=64, cache="e4m3", t="f16"),
        # The gradient of the rotation over a training batch.
        dict(name="rope_inverse_8192", kind="rope", T=8192, Hq=32, Hkv=8, D=128, rot=128,
             inter=False, scaling="bands", far=32768, inverse=True, t="bf16"),
        # A single conversation: latency.
        dict(name="attend_1_short", kind="attend", B=1, Hq=32, Hkv=8, D=128, S=16, longest=700,
             even=True, t="bf16", cache="bf16", cap=0.0, window=0, slopes=False, lse=False),
        # A serving batch of sequences of every length, some of them empty.
        dict(name="attend_64_ragged", kind="attend", B=64, Hq=32, Hkv=8, D=128, S=16,
             longest=4096, even=False, t="bf16", cache="bf16", cap=0.0, window=0, slopes=False,
             lse=False),
        # A few very long contexts.
        dict(name="attend_4_long", kind="attend", B=4, Hq=32, Hkv=8, D=128, S=64, longest=100003,
             even=True, t="bf16", cache="bf16", cap=0.0, window=0, slopes=False, lse=True),
        # 8-bit pages, one kv head per query head, capped scores, a window and
        # a bias that grows with distance, on pages that are no power of two.
        dict(name="attend_24_e4m3", kind="attend", B=24, Hq=16, Hkv=16, D=80, S=24, longest=6000,
             even=False, t="f16", cache="e4m3", cap=30.0, window=2048, slopes=True, lse=True),
        # Parallel sampling: 8 finished groups leave, 8 prompts become 8
        # samples each, over all the layers of the cache.
        dict(name="fork_64", kind="fork", L=16, pages=1024, H=8, S=16, D=128, rows=128, src=8,
             n=64, width=64, t="bf16"),
        # A fragmented pool before a part of it is given back.
        dict(name="compact_2048", kind="compact", L=8, pages=2048, H=8, S=16, D=128, rows=96,
             width=64, used=0.55, t="bf16"),
    ]


def _log(rng, lo, hi):
    """A whole number from lo to hi, uniform in its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["linear", "linear", "rope", "append", "attend", "attend", "attend", "fork",
                       "compact"])
    if kind == "linear":
        K, N = _log(rng, 128, 14336), _log(rng, 128, 28672)
        M = min(_log(rng, 1, 4096), max(1, int(4.8e11 / (2 * K * N))))
        return dict(kind=kind, M=M, K=K, N=N, t=rng.choice(["bf16", "f16", "f32"]),
                    bias=rng.random() < 0.5)
    if kind in ("rope", "append"):
        Hkv, D = rng.choice([1, 2, 4, 8, 16]), rng.choice([40, 64, 80, 96, 128, 192, 256])
        Hq = Hkv * rng.choice([1, 2, 3, 4, 7, 8])
        T = min(_log(rng, 1, 8192), max(1, 8192 * 40 * 128 // ((Hq + 2 * Hkv) * D)))
        c = dict(kind=kind, T=T, Hq=Hq, Hkv=Hkv, D=D, rot=2 * rng.randint(1, D // 2),
                 inter=rng.random() < 0.5, scaling=rng.choice(["none", "linear", "ntk", "yarn", "bands"]),
                 far=_log(rng, 2048, 1 << 20), t=rng.choice(["bf16", "f16", "f32"]))
        if kind == "rope":
            return dict(c, inverse=rng.random() < 0.5)
        S = rng.choice([1, 8, 16, 24, 64, 256])
        t = rng.choice(["bf16", "f16"])
        return dict(c, t=t, S=S, pages=(T + S - 1) // S + rng.randint(1, 64),
                    cache=rng.choice([t, "e4m3"]))
    if kind == "attend":
        Hkv, D = rng.choice([1, 2, 4, 8, 16]), rng.choice([40, 64, 80, 96, 128, 192, 256])
        Hq = Hkv * rng.choice([1, 2, 3, 4, 7, 8, 16, 20])
        B, longest = _log(rng, 1, 256), _log(rng, 1, 100000)
        # no more than the largest listed case reads, nor than it has scores
        longest = max(1, min(longest, 4 * 8 * 128 * 100003 // (B * Hkv * D),
                             4 * 32 * 100003 // (B * Hq)))
        t = rng.choice(["bf16", "f16"])
        return dict(kind=kind, B=B, Hq=Hq, Hkv=Hkv, D=D, S=rng.choice([1, 8, 16, 24, 64, 256]),
                    longest=longest, even=rng.random() < 0.3, t=t, cache=rng.choice([t, "e4m3"]),
                    cap=rng.choice([0.0, 0.0, 30.0]), window=rng.choice([0, 0, _log(rng, 1, 8192)]),
                    slopes=rng.random() < 0.25, lse=rng.random() < 0.5)
    L, H, S, D = rng.choice([1, 4, 16]), rng.choice([1, 4, 8]), rng.choice([8, 16, 24, 64]), rng.choice([64, 80, 128])
    t = rng.choice(["bf16", "f16", "e4m3"])
    pages = min(_log(rng, 64, 65536), (1 << 30) // (2 * L * H * S * D * SIZE[t]))
    pages = max(64, pages)
    if kind == "fork":
        src = rng.randint(1, 8)
        n = src * rng.randint(1, 8)
        # the pool holds the prompts, the finished rows and a new page a sample
        width = max(1, min(64, (pages - n) // (src + n) - 1))
        return dict(kind=kind, L=L, pages=pages, H=H, S=S, D=D, rows=src + n + rng.randint(0, 8),
                    src=src, n=n, width=width, t=t)
    rows = rng.randint(1, 128)
    return dict(kind=kind, L=L, pages=pages, H=H, S=S, D=D, rows=rows,
                width=max(1, min(1024, pages // rows)), used=rng.uniform(0.05, 0.95), t=t)


# ------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _randn(g, *shape):
    return torch.randn(*shape, device="cuda", generator=g)


def _pages(g, *shape, t):
    """Cache values of size one."""
    out = torch.randn(*shape, device="cuda", generator=g,
                      dtype=torch.float16 if t == "f16" else torch.bfloat16)
    return out.to(DTYPE[t])


def _scaling(kind):
    """What a configuration says of a stretched context."""
    return {"none": None,
            "linear": dict(kind="linear", factor=4.0),
            "ntk": dict(kind="ntk", factor=4.0),
            "yarn": dict(kind="yarn", factor=32.0, original=32768),
            "bands": dict(kind="bands", factor=8.0, low=1.0, high=4.0, original=8192)}[kind]


BASE = 500000.0


def prepare(c, seed):
    g = _gen(seed)
    s = {"case": c}
    kind = c["kind"]
    if kind == "linear":
        M, K, N, T = c["M"], c["K"], c["N"], DTYPE[c["t"]]
        # activations whose channels differ in size, as hidden states do
        s["x"] = (_randn(g, M, K) * torch.exp(0.5 * _randn(g, K))).to(T)
        s["w"] = torch.clamp(torch.round(_randn(g, N, K) * 32), -127, 127).to(torch.int8)
        s["ws"] = torch.rand(N, device="cuda", generator=g) * 2e-3 + 1e-4
        s["bias"] = _randn(g, N) if c["bias"] else None
        if own:
            from ubridge_amd import int8
            s["linear"] = int8.Linear(s["w"], s["ws"], s["bias"])
        return s
    if kind in ("rope", "append"):
        T, Hq, Hkv, D = c["T"], c["Hq"], c["Hkv"], c["D"]
        # the heads of one fused projection: q, k and v are views of it
        qkv = _randn(g, T, (Hq + 2 * Hkv) * D).to(DTYPE[c["t"]])
        s["q"], s["k"], s["v"] = (x.unflatten(1, (-1, D)) for x in
                                  qkv.split([Hq * D, Hkv * D, Hkv * D], 1))
        s["positions"] = torch.randint(0, c["far"], (T,), device="cuda", generator=g)
        if own:
            from ubridge_amd import kvcache, rope
            s["rope"] = rope.Rope(c["rot"], base=BASE, interleaved=c["inter"],
                                  scaling=_scaling(c["scaling"]), device="cuda")
        if kind == "append":
            P, S = c["pages"], c["S"]
            s["kv"] = _pages(g, 1, 2, P, Hkv, S, D, t=c["cache"])
            s["slots"] = torch.randperm(P * S, device="cuda", generator=g)[:T]
            s["ks"] = s["vs"] = None
            if c["cache"] == "e4m3":
                s["ks"], s["vs"] = (torch.rand(Hkv, device="cuda", generator=g) * 0.02 + 0.01
                                    for _ in "kv")
            if own:
                s["cache"] = kvcache.PagedCache(s["kv"], rows=1, width=1, k_scale=s["ks"],
                                                v_scale=s["vs"])
        return s
    if kind == "attend":
        B, Hq, Hkv, D, S = c["B"], c["Hq"], c["Hkv"], c["D"], c["S"]
        lens = _lens(c, seed)
        width = max(1, -(-c["longest"] // S))
        need = [-(-n // S) for n in lens]
        P = sum(need) + 1
        order = torch.randperm(P - 1, device="cuda", generator=g).to(torch.int32) + 1
        at = torch.tensor([sum(need[:b]) for b in range(B)], device="cuda")[:, None]
        i = torch.arange(width, device="cuda")[None]
        live = i < torch.tensor(need, device="cuda")[:, None]
        s["tables"] = torch.where(live, order[(at + i).clamp(max=max(P - 2, 0))] if P > 1 else -1,
                                  -1).to(torch.int32)
        s["lens"] = torch.tensor(lens, device="cuda", dtype=torch.int32)
        s["kv"] = _pages(g, 1, 2, P, Hkv, S, D, t=c["cache"])
        s["q"] = _randn(g, B, Hq, D).to(DTYPE[c["t"]])
        s["ks"] = s["vs"] = s["slopes"] = None
        if c["cache"] == "e4m3":
            s["ks"], s["vs"] = (torch.rand(Hkv, device="cuda", generator=g) + 0.5 for _ in "kv")
        if c["slopes"]:
            s["slopes"] = torch.exp2(-8 * torch.arange(1, Hq + 1, device="cuda") / Hq)
        return s
    # fork, compact: a pool whose state is one int32 buffer [refs | lens | tables]
    L, P, H, S, D, rows, width = (c[k] for k in ("L", "pages", "H", "S", "D", "rows", "width"))
    s["kv"] = _pages(g, L, 2, P, H, S, D, t=c["t"])
    refs, lens, tables = _pool(c, seed)
    s["meta0"] = torch.from_numpy(np.concatenate([refs, lens, tables.ravel()])).cuda()
    s["meta"] = s["meta0"].clone()
    if kind == "fork":
        src, n = c["src"], c["n"]
        s["src"] = torch.arange(n, device="cuda", dtype=torch.int32) % src
        s["dst"] = torch.arange(n, device="cuda", dtype=torch.int32) + src
    if own:
        from ubridge_amd import kvcache
        s["cache"] = kvcache.PagedCache(s["kv"], rows=rows, width=width, meta=s["meta"])
    return s


def _lens(c, seed):
    """Cached tokens of each sequence: all the longest, or uniform in the
    logarithm with every sixteenth sequence empty."""
    if c["even"]:
        return [c["longest"]] * c["B"]
    r = np.random.RandomState(seed % (1 << 31))
    n = np.exp(r.uniform(0, np.log(c["longest"] + 1), c["B"])).astype(int)
    n[15::16] = 0
    return [int(x) for x in np.minimum(n, c["longest"])]


def _pool(c, seed):
    """refs [pages], lens [rows] and tables [rows, width] of a pool in use.
    fork: `src` prompts, then `n` finished samples of them that still share
    their pages.  compact: rows of odd lengths over pages in no order."""
    r = np.random.RandomState(seed % (1 << 31))
    P, S, rows, width = c["pages"], c["S"], c["rows"], c["width"]
    refs = np.zeros(P, np.int32)
    lens = np.zeros(rows, np.int32)
    tables = np.full((rows, width), -1, np.int32)
    order = r.permutation(P).astype(np.int32)
    at = 0

    def fill(row, tokens, shared=()):
        nonlocal at
        k = -(-tokens // S)
        pages = list(shared[:k])
        fresh = order[at:at + k - len(pages)]
        at += len(fresh)
        tables[row, :k] = pages + list(fresh)
        refs[tables[row, :k]] += 1
        lens[row] = tokens

    if c["kind"] == "fork":
        for b in range(c["src"]):
            fill(b, int(r.randint(1, width * S + 1)))
        for j in range(c["n"]):
            b = j % c["src"]
            full = tables[b, :lens[b] // S]
            fill(c["src"] + j, min(width * S, int(lens[b]) + int(r.randint(0, S))), list(full))
    else:
        for b in range(rows):
            left = int(P * c["used"]) - at
            if left <= 0:
                break
            fill(b, int(r.randint(1, min(left, width) * S + 1)))
    return refs, lens, tables


# ------------------------------------------------------------- plain forms
def _linear(s):
    x = s["x"].float()
    amax = x.abs().amax(1, keepdim=True)
    sx = torch.where(amax > 0, amax / 127.0, torch.ones_like(amax))
    q = torch.round(x / sx)
    y = (q @ s["w"].float().t()) * sx * s["ws"]
    if s["bias"] is not None:
        y = y + s["bias"]
    return y.to(s["x"].dtype)


def _freqs(rot, scaling, xp=torch):
    """Angle per position of each pair in 64 bits, and the factor on the
    rotated values."""
    kw = dict(device="cuda") if xp is torch else {}
    i = xp.arange(0, rot // 2, dtype=xp.float64, **kw)
    sc = _scaling(scaling)
    base, factor = BASE, 1.0
    if sc and sc["kind"] == "ntk":
        base = BASE * sc["factor"] ** (rot / (rot - 2.0)) if rot > 2 else BASE
    f = base ** (-2.0 * i / rot)
    if sc and sc["kind"] == "linear":
        f = f / sc["factor"]
    elif sc and sc["kind"] == "yarn":
        def turn(n):  # the pair that makes n turns over the original length
            return rot * math.log(sc["original"] / (n * 2 * math.pi)) / (2 * math.log(base))
        low, high = max(math.floor(turn(32)), 0), min(math.ceil(turn(1)), rot - 1)
        ramp = xp.clip((i - low) / max(high - low, 0.001), 0, 1)
        f = f / sc["factor"] * ramp + f * (1 - ramp)
        factor = 0.1 * math.log(sc["factor"]) + 1.0
    elif sc and sc["kind"] == "bands":
        turns = sc["original"] * f / (2 * math.pi)  # over the original length
        mix = xp.clip((turns - sc["low"]) / (sc["high"] - sc["low"]), 0, 1)
        f = f * (mix + (1 - mix) / sc["factor"])
    return f, factor


def _rotate(x, cos, sin, rot, inter):
    x = x.float()
    if inter:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        y = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        y = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([y, x[..., rot:]], -1)


def _rope(s):
    c = s["case"]
    f, factor = _freqs(c["rot"], c["scaling"])
    a = s["positions"].double()[:, None, None] * f
    cos, sin = (torch.cos(a) * factor).float(), (torch.sin(a) * factor).float()
    if c.get("inverse"):
        sin = -sin
    return [_rotate(s[n], cos, sin, c["rot"], c["inter"]) for n in "qk"]


def _append(s):
    c = s["case"]
    q, k = _rope(s)
    v, kv, slots, S = s["v"].float(), s["kv"], s["slots"], c["S"]
    if s["ks"] is not None:
        k = (k / s["ks"][:, None]).clamp(-448, 448)
        v = (v / s["vs"][:, None]).clamp(-448, 448)
    page, at = slots // S, slots % S
    raw = kv.view(torch.uint8) if c["cache"] == "e4m3" else kv
    for i, x in ((0, k), (1, v)):
        raw[0, i][page, :, at] = x.to(kv.dtype).view(raw.dtype)
    return [q.to(s["q"].dtype), kv]


def _attend(s):
    c = s["case"]
    B, Hq, Hkv, D, S = c["B"], c["Hq"], c["Hkv"], c["D"], c["S"]
    tables, lens, kv = s["tables"].long().clamp(min=0), s["lens"].long(), s["kv"]
    if c["cache"] == "e4m3":
        kv = kv.view(torch.uint8)
    n = tables.shape[1] * S
    k, v = (kv[0, i][tables].view(s["kv"].dtype).transpose(1, 2).reshape(B * Hkv, n, D).float()
            for i in (0, 1))
    q = s["q"].float().reshape(B * Hkv, Hq // Hkv, D) * D ** -0.5
    x = torch.bmm(q, k.transpose(1, 2).contiguous()).reshape(B, Hkv, Hq // Hkv, n)
    del k
    if s["ks"] is not None:
        x = x * s["ks"][None, :, None, None]
    if c["cap"]:
        x = c["cap"] * torch.tanh(x / c["cap"])
    t = torch.arange(n, device="cuda")
    last = lens[:, None] - 1
    if c["slopes"]:
        x = x + s["slopes"].reshape(1, Hkv, -1, 1) * (t - last).float()[:, None, None]
    seen = (t <= last) & ((t > last - c["window"]) if c["window"] else True)
    x = x.masked_fill(~seen[:, None, None], -math.inf)
    m = x.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, torch.zeros_like(m), m)
    p = torch.exp(x - m)
    l = p.sum(-1, keepdim=True)
    # what lies behind a masked place counts for nothing, whatever it holds
    v = v.masked_fill(~seen[:, None].expand(B, Hkv, n).reshape(B * Hkv, n, 1), 0.0)
    o = torch.bmm(p.reshape(B * Hkv, -1, n), v).reshape(B, Hkv, -1, D)
    o = o / torch.where(l > 0, l, torch.ones_like(l))
    if s["vs"] is not None:
        o = o * s["vs"][None, :, None, None]
    o = o.reshape(B, Hq, D).to(s["q"].dtype)
    return [o, (m + torch.log(l)).reshape(B, Hq)] if c["lse"] else o


def _fields(s):
    c = s["case"]
    P, rows = c["pages"], c["rows"]
    m = s["meta"]
    return m[:P], m[P:P + rows], m[P + rows:].view(rows, c["width"])


def _count(pages, P):
    """How often each page number appears (-1: none)."""
    z = torch.zeros(P + 1, device="cuda", dtype=torch.int32)
    p = pages.reshape(-1).long()
    return z.index_add(0, torch.where(p >= 0, p, P), torch.ones_like(p, dtype=torch.int32))[:P]


def _raw(kv):
    return kv.view(torch.uint8) if kv.dtype == torch.float8_e4m3fn else kv


def _fork(s):
    c = s["case"]
    refs, lens, tables = _fields(s)
    src, dst, S, P = s["src"].long(), s["dst"].long(), c["S"], c["pages"]
    # the finished rows leave
    refs -= _count(tables[dst], P)
    tables[dst] = -1
    lens[dst] = 0
    # the samples share their prompt's whole pages and copy a part-filled last one
    part = lens[src] % S != 0
    at = ((lens[src] - 1).clamp(min=0) // S).long()
    t = tables[src]
    old = t.gather(1, at[:, None])[:, 0]
    free = torch.argsort((refs != 0).int(), stable=True)
    new = torch.where(part, free[(torch.cumsum(part, 0) - 1).clamp(min=0)].int(), old)
    t = t.scatter(1, at[:, None], new[:, None])
    tables[dst] = t
    lens[dst] = lens[src]
    refs += _count(t, P)
    raw = _raw(s["kv"])
    raw[:, :, new.long()] = raw[:, :, old.long()]
    return [s["kv"], s["meta"], torch.where(part, new, -1)]


def _compact(s):
    c = s["case"]
    refs, lens, tables = _fields(s)
    P = c["pages"]
    used = refs != 0
    n = used.sum()
    i = torch.arange(P, device="cuda")
    # the k-th used page beyond the first n goes to the k-th free one below n
    out, hole = used & (i >= n), ~used & (i < n)
    holes = torch.argsort((~hole).int(), stable=True)
    to = torch.where(out, holes[(torch.cumsum(out, 0) - 1).clamp(min=0)], i)
    raw = _raw(s["kv"])
    src = torch.argsort((~out).int(), stable=True)[:P // 2]
    dst = to[src]
    keep = out[src]
    # (the last page is never a destination: with moves to make, n < P)
    src, dst = torch.where(keep, src, P - 1), torch.where(keep, dst, P - 1)
    raw[:, :, dst] = raw[:, :, src]
    tables.copy_(torch.where(tables >= 0, to[tables.clamp(min=0).long()].int(), -1))
    new = torch.zeros_like(refs)
    new.index_add_(0, torch.where(used, to, 0), torch.where(used, refs, 0))
    refs.copy_(new)
    return [s["kv"], s["meta"], n.int()]


PLAIN = {"linear": _linear, "append": _append, "attend": _attend, "fork": _fork,
         "compact": _compact,
         "rope": lambda s: [x.to(s["q"].dtype) for x in _rope(s)]}


def _own(s):
    from ubridge_amd import attention
    c = s["case"]
    kind = c["kind"]
    if kind == "linear":
        return s["linear"](s["x"])
    if kind == "rope":
        turn = s["rope"].backward if c["inverse"] else s["rope"]
        return turn(s["q"], s["k"], s["positions"])
    if kind == "append":
        q = s["cache"].append(0, s["q"], s["k"], s["v"], s["slots"], positions=s["positions"],
                              rope=s["rope"])
        return [q, s["kv"]]
    if kind == "attend":
        kv = s["kv"]
        return attention.paged_decode(s["q"], kv[0, 0], kv[0, 1], s["tables"], s["lens"],
                                      softcap=c["cap"], window=c["window"], slopes=s["slopes"],
                                      k_scale=s["ks"], v_scale=s["vs"], return_lse=c["lse"])
    if kind == "fork":
        s["cache"].free(s["dst"])
        new = s["cache"].fork(s["src"], s["dst"])
        return [s["kv"], s["meta"], new]
    return [s["kv"], s["meta"], s["cache"].compact()]


def run(s):
    if "meta0" in s:  # the pool as it was, so that a pass can be repeated
        s["meta"].copy_(s["meta0"])
    return _own(s) if own else PLAIN[s["case"]["kind"]](s)


# -------------------------------------------------------------------- work
def work(c):
    kind = c["kind"]
    if kind == "linear":
        M, K, N, e = c["M"], c["K"], c["N"], SIZE[c["t"]]
        return dict(bytes=M * K * e + N * K + 4 * N * (2 if c["bias"] else 1) + M * N * e,
                    flops=2 * M * N * K)
    if kind in ("rope", "append"):
        T, Hq, Hkv, D, e = c["T"], c["Hq"], c["Hkv"], c["D"], SIZE[c["t"]]
        if kind == "rope":
            return dict(bytes=2 * T * (Hq + Hkv) * D * e + 8 * T, flops=3 * T * (Hq + Hkv) * c["rot"])
        return dict(bytes=T * D * (2 * Hq * e + 2 * Hkv * (e + SIZE[c["cache"]])) + 16 * T,
                    flops=3 * T * (Hq + Hkv) * c["rot"])
    if kind == "attend":
        B, Hq, Hkv, D, e = c["B"], c["Hq"], c["Hkv"], c["D"], SIZE[c["cache"]]
        n = sum(min(x, c["window"] or x) for x in _lens(c, 0))
        return dict(bytes=2 * n * Hkv * D * e + 2 * B * Hq * D * SIZE[c["t"]] + 4 * n // c["S"],
                    flops=4 * n * Hq * D)
    page = 2 * c["L"] * c["H"] * c["S"] * c["D"] * SIZE[c["t"]]
    refs, lens, tables = _pool(c, 0)
    if kind == "fork":
        moved = int((lens[np.arange(c["n"]) % c["src"]] % c["S"] != 0).sum())
        small = 4 * (c["pages"] + 4 * c["n"] * c["width"])
    else:
        used = refs != 0
        moved = int(used[int(used.sum()):].sum())
        small = 8 * (c["pages"] + c["rows"] * c["width"])
    return dict(bytes=2 * moved * page + small, flops=0)


# ------------------------------------------------------------------- exact
def _e4m3(x):
    """64-bit values to the nearest e4m3 (ties to even), saturating."""
    x = np.clip(x, -448.0, 448.0)
    e = np.maximum(np.floor(np.log2(np.maximum(np.abs(x), 1e-30))), -6)
    step = 2.0 ** (e - 3)
    return np.rint(x / step) * step


def _turn64(x, pos, f, factor, rot, inter, sign):
    a = np.asarray(pos, np.float64)[:, None, None] * f
    w = factor * np.exp(1j * sign * a)
    y = x.copy()
    lo, hi = (slice(0, rot, 2), slice(1, rot, 2)) if inter else (slice(0, rot // 2), slice(rot // 2, rot))
    z = (x[..., lo] + 1j * x[..., hi]) * w
    y[..., lo], y[..., hi] = z.real, z.imag
    return y


def exact(c, seed):
    kind = c["kind"]
    if kind in ("fork", "compact"):
        return None
    s = prepare(c, seed)
    if kind == "linear":
        x = s["x"].double()
        top = x.abs().amax(1)
        # codes and scales are the format's: the scale is an f32 number
        sx = torch.where(top > 0, (top.float() / 127.0).double(), 1.0)
        q = torch.round((x.float() / sx.float()[:, None])).double()
        y = torch.cat([(q @ w.double().t()) for w in s["w"].split(4096)], 1)
        y = y * sx[:, None] * s["ws"].double()
        return y + s["bias"].double() if c["bias"] else y
    if kind in ("rope", "append"):
        f, factor = _freqs(c["rot"], c["scaling"], np)
        sign = -1.0 if c.get("inverse") else 1.0
        pos = s["positions"].cpu().numpy()
        q, k = (_turn64(s[n].double().cpu().numpy(), pos, f, factor, c["rot"], c["inter"], sign)
                for n in "qk")
        if kind == "rope":
            return [torch.from_numpy(q), torch.from_numpy(k)]
        kv = s["kv"].to(torch.float64).cpu().numpy()
        v = s["v"].double().cpu().numpy()
        if s["ks"] is not None:
            k = _e4m3(k / s["ks"].double().cpu().numpy()[:, None])
            v = _e4m3(v / s["vs"].double().cpu().numpy()[:, None])
        slots = s["slots"].cpu().numpy()
        kv[0, 0][slots // c["S"], :, slots % c["S"]] = k
        kv[0, 1][slots // c["S"], :, slots % c["S"]] = v
        return [torch.from_numpy(q), torch.from_numpy(kv)]
    Hq, Hkv, D, S = c["Hq"], c["Hkv"], c["D"], c["S"]
    out = torch.zeros(c["B"], Hq, D, dtype=torch.float64, device="cuda")
    lse = torch.full((c["B"], Hq), -math.inf, dtype=torch.float64, device="cuda")
    for b, n in enumerate(_lens(c, seed)):
        first = max(0, n - c["window"]) if c["window"] else 0
        if n <= first:
            continue
        pages = s["tables"][b, :-(-n // S)].long()
        for h in range(Hkv):
            heads = slice(h * Hq // Hkv, (h + 1) * Hq // Hkv)
            k, v = (_raw(s["kv"])[0, i][pages, h].view(s["kv"].dtype).double().reshape(-1, D)[first:n]
                    for i in (0, 1))
            x = s["q"][b, heads].double() @ k.t().contiguous() / math.sqrt(D)
            if s["ks"] is not None:
                x, v = x * s["ks"][h].double(), v * s["vs"][h].double()
            if c["cap"]:
                x = c["cap"] * torch.tanh(x / c["cap"])
            if c["slopes"]:
                back = torch.arange(first - n + 1, 1, device="cuda", dtype=torch.float64)
                x = x + s["slopes"][heads].double()[:, None] * back
            lse[b, heads] = torch.logsumexp(x, -1)
            out[b, heads] = torch.softmax(x, -1) @ v
    return [out, lse] if c["lse"] else out
