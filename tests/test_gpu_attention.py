"""Paged decode attention against the definition in 64 bits.

Tolerances.  A score is a sum of D products in f32: off by at most ex = (D + 8)
2^-24 scale sum |q k| (plus a few ulp of the cap where there is one and of the
bias where there is one), so each weight of the softmax is off by a factor of
at most 1 + 2 ex + 2^-15 (the weights carry at least 16 bits into the second
product; exp and the sums a few ulp), the output by that times sum p |v|, and
it rounds once.  lse is off by ex and a few ulp.
"""
import math

import pytest
import torch

from ubridge_amd import attention, kvcache, moe

pytestmark = pytest.mark.gpu

DT = {"f16": torch.float16, "bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn}


def make(dev, lens, Hq, Hkv, D, S, t="bf16", cache=None, seed=0, width=None, spare=3):
    """q, kv [2, P, Hkv, S, D], tables, lens: pages in no order, places that
    hold no token filled with NaN, unused table entries with a page that is not there."""
    g = torch.Generator().manual_seed(seed + sum(lens) + D)
    need = [-(-n // S) for n in lens]
    P = sum(need) + spare
    width = max(need + [1]) if width is None else width
    order = torch.randperm(P, generator=g).int()
    tables = torch.full((len(lens), width), 1 << 30, dtype=torch.int32)
    kv = torch.randn(2, P, Hkv, S, D, generator=g).to(DT[cache or t])
    raw = kv.view(torch.uint8) if cache == "e4m3" else kv
    at = 0
    held = torch.zeros(P, S, dtype=torch.bool)
    for b, n in enumerate(lens):
        tables[b, :need[b]] = order[at:at + need[b]]
        at += need[b]
        for i in range(need[b]):
            held[tables[b, i], :min(S, n - i * S)] = True
    free = ~held[None, :, None, :, None].expand(kv.shape)
    raw[free] = 0x7F if cache == "e4m3" else float("nan")
    q = torch.randn(len(lens), Hq, D, generator=g).to(DT[t])
    return q.to(dev), kv.to(dev), tables.to(dev), torch.tensor(lens, dtype=torch.int32).to(dev)


def check(got, q, kv, tables, lens, lse=None, scale=None, softcap=0.0, window=0, slopes=None,
          k_scale=None, v_scale=None, rows=None):
    B, Hq, D = q.shape
    S, Hkv = kv.shape[3], kv.shape[2]
    scale = D ** -0.5 if scale is None else scale
    half = torch.finfo(q.dtype).eps / 2
    G = Hq // Hkv
    for b in range(B) if rows is None else rows:
        n = int(lens[b])
        first = max(0, n - window) if window else 0
        if n <= first:
            assert not bool(got[b].any())
            assert lse is None or bool((lse[b] == -math.inf).all())
            continue
        pages = tables[b, :-(-n // S)].long()
        k, v = (kv[i].view(torch.uint8)[pages].view(kv.dtype) if kv.dtype == DT["e4m3"] else kv[i][pages]
                for i in (0, 1))
        k, v = (x.double().transpose(1, 2).reshape(-1, Hkv, D)[first:n].permute(1, 2, 0).contiguous()
                for x in (k, v))  # [Hkv, D, n]
        qq = q[b].double().view(Hkv, G, D) * scale
        x, size = torch.bmm(qq, k), torch.bmm(qq.abs(), k.abs())
        if k_scale is not None:
            x, size = x * k_scale.double()[:, None, None], size * k_scale.double()[:, None, None]
        ex = (D + 8) * 2.0**-24 * size.amax(-1)
        if softcap:
            x = softcap * torch.tanh(x / softcap)
            ex = ex + 8 * 2.0**-24 * softcap
        if slopes is not None:
            back = torch.arange(first - n + 1, 1, device=x.device, dtype=torch.float64)
            x = x + slopes.double().view(Hkv, G, 1) * back
            ex = ex + 4 * 2.0**-24 * (slopes.abs().double().view(Hkv, G) * (n - first))
        # exp(x - m) in f32: the difference rounds at 2^-24 of scores this large
        ex = ex + 2.0**-22 * x.abs().amax(-1)
        p = torch.softmax(x, -1)
        vt = v.transpose(1, 2).contiguous()
        if v_scale is not None:
            vt = vt * v_scale.double()[:, None, None]
        want, mag = torch.bmm(p, vt), torch.bmm(p, vt.abs())
        tol = half * want.abs() + (2 * ex + 2.0**-15)[..., None] * mag + torch.finfo(q.dtype).smallest_normal * half
        err = (got[b].double().view(Hkv, G, D) - want).abs()
        assert bool((err <= tol).all()), (b, n, float((err / tol).max()))
        if lse is not None:
            w = torch.logsumexp(x, -1)
            e = (lse[b].double().view(Hkv, G) - w).abs()
            assert bool((e <= ex + 2.0**-20 * (1 + w.abs())).all()), (b, n, float(e.max()))


@pytest.mark.parametrize("t,cache", [("bf16", "bf16"), ("f16", "f16"), ("bf16", "e4m3"), ("f16", "e4m3")])
@pytest.mark.parametrize("Hq,Hkv,D,S", [(4, 1, 128, 16), (3, 3, 40, 1), (16, 2, 64, 8), (14, 2, 80, 24),
                                        (20, 1, 96, 64), (8, 8, 192, 16), (32, 1, 256, 16), (40, 2, 128, 12)])
def test_lengths(dev, t, cache, Hq, Hkv, D, S):
    lens = [0, 1, 2, 7, 8, 9, 15, 16, 17, 31, 32, 33, 63, 64, 65, 100, 255, 256, 257, 700]
    q, kv, tables, n = make(dev, lens, Hq, Hkv, D, S, t, cache)
    out, lse = attention.paged_decode(q, kv[0], kv[1], tables, n, return_lse=True)
    check(out, q, kv, tables, n, lse)
    assert torch.equal(out, attention.paged_decode(q, kv[0], kv[1], tables, n))
    moe.device_error()


@pytest.mark.parametrize("t,cache", [("bf16", "bf16"), ("f16", "f16"), ("bf16", "e4m3"), ("f16", "e4m3")])
@pytest.mark.parametrize("Hq,Hkv,D,S", [(4, 1, 128, 16), (3, 3, 40, 1), (17, 1, 64, 8), (14, 2, 80, 24), (70, 1, 96, 64),
                                        (8, 8, 192, 16), (33, 1, 256, 5), (40, 2, 128, 12), (2, 1, 8, 3)])
def test_short(dev, t, cache, Hq, Hkv, D, S):
    # few rows and few steps: a workgroup a row, its wavefronts with and without steps
    for lens in ([0, 1, 31, 32, 33, 100, 200], [120], [0]):
        q, kv, tables, n = make(dev, lens, Hq, Hkv, D, S, t, cache)
        out, lse = attention.paged_decode(q, kv[0], kv[1], tables, n, return_lse=True)
        check(out, q, kv, tables, n, lse)
        out, lse = attention.paged_decode(q, kv[0], kv[1], tables, n, window=33, softcap=4.0, return_lse=True)
        check(out, q, kv, tables, n, lse, window=33, softcap=4.0)
    moe.device_error()


@pytest.mark.parametrize("Hq,Hkv,D", [(70, 1, 64), (130, 2, 128), (33, 1, 256)])
def test_many_heads(dev, Hq, Hkv, D):
    # more query heads to a kv head than one pass takes
    q, kv, tables, n = make(dev, [3000, 5, 0, 777], Hq, Hkv, D, 16, "bf16")
    out, lse = attention.paged_decode(q, kv[0], kv[1], tables, n, return_lse=True)
    check(out, q, kv, tables, n, lse)


@pytest.mark.parametrize("lens,Hq,Hkv,D,S", [([5000], 8, 2, 128, 16), ([20011, 3], 4, 4, 64, 64),
                                             ([1, 0, 9000, 4097], 16, 1, 128, 24), ([3001] * 5, 24, 3, 256, 8)])
@pytest.mark.parametrize("t,cache", [("bf16", "bf16"), ("f16", "e4m3")])
def test_long(dev, t, cache, lens, Hq, Hkv, D, S):
    # sequences that are split, beside short ones
    q, kv, tables, n = make(dev, lens, Hq, Hkv, D, S, t, cache)
    out, lse = attention.paged_decode(q, kv[0], kv[1], tables, n, return_lse=True)
    check(out, q, kv, tables, n, lse)
    for _ in range(3):  # the same bits again
        assert torch.equal(out, attention.paged_decode(q, kv[0], kv[1], tables, n))


@pytest.mark.parametrize("B", [97, 300])
def test_many_short(dev, B):
    g = torch.Generator().manual_seed(B)
    lens = [int(x) for x in torch.randint(0, 90, (B,), generator=g)]
    q, kv, tables, n = make(dev, lens, 8, 4, 64, 16, "f16")
    out, lse = attention.paged_decode(q, kv[0], kv[1], tables, n, return_lse=True)
    check(out, q, kv, tables, n, lse)


@pytest.mark.parametrize("cap,window,slopes,scaled", [
    (30.0, 0, False, False), (0.0, 1, False, True), (0.0, 100, True, False), (5.0, 33, True, True),
    (0.0, 5000, False, False), (2.0, 0, True, True)])
@pytest.mark.parametrize("D,S,cache", [(80, 24, "e4m3"), (128, 16, None), (64, 1, None)])
def test_masks_and_biases(dev, cap, window, slopes, scaled, D, S, cache):
    lens = [0, 1, 5, 32, 33, 34, 99, 100, 101, 640, 2300]
    q, kv, tables, n = make(dev, lens, 8, 4, D, S, "f16", cache)
    g = torch.Generator().manual_seed(1)
    sl = torch.exp2(-8 * torch.arange(1, 9) / 8).to(dev) if slopes else None
    ks, vs = (torch.rand(4, generator=g).to(dev) + 0.5 for _ in "kv") if scaled else (None, None)
    out, lse = attention.paged_decode(q, kv[0], kv[1], tables, n, softcap=cap, window=window, slopes=sl,
                                      k_scale=ks, v_scale=vs, scale=0.3, return_lse=True)
    check(out, q, kv, tables, n, lse, scale=0.3, softcap=cap, window=window, slopes=sl, k_scale=ks, v_scale=vs)


@pytest.mark.parametrize("t", ["bf16", "f16"])
def test_lse_of_few_tokens(dev, t):
    # one token: lse is its score, exact where the products are; equal tokens: the
    # logarithm of their number beside it, to an ulp or two of the sum
    q, kv, tables, n = make(dev, [1, 4, 64, 1000], 4, 2, 64, 16, t)
    q = torch.randint(-4, 5, q.shape, generator=torch.Generator().manual_seed(1)).to(q.dtype).to(dev)
    kv[0] = 0.5
    x = q.float().sum(-1) * 0.5 * 0.125
    lse = attention.paged_decode(q, kv[0], kv[1], tables, n, scale=0.125, return_lse=True)[1]
    assert torch.equal(lse[0], x[0])
    want = x.double() + torch.log(n.double())[:, None]
    assert bool(((lse.double() - want).abs() <= 2.0**-23 * (want.abs() + 8)).all())
    # capped: c tanh(x / c), to some ulp of the value
    x = x * 3
    lse = attention.paged_decode(q, kv[0], kv[1], tables, n, scale=0.375, softcap=5.0, return_lse=True)[1]
    want = 5 * torch.tanh(x[0].double() / 5)
    assert bool(((lse[0].double() - want).abs() <= 2.0**-21 * want.abs()).all())


def test_large_scores(dev):
    # scores far beyond exp's range, growing and falling along the sequence
    lens = [300, 2000]
    q, kv, tables, n = make(dev, lens, 4, 2, 64, 16, "bf16")
    out, lse = attention.paged_decode(q, kv[0], kv[1], tables, n, scale=40.0, return_lse=True)
    check(out, q, kv, tables, n, lse, scale=40.0)
    sl = torch.tensor([100.0, -100.0, 1e-3, -0.5], device=dev)
    out, lse = attention.paged_decode(q, kv[0], kv[1], tables, n, slopes=sl, return_lse=True)
    check(out, q, kv, tables, n, lse, slopes=sl)


def test_infinities(dev):
    # a value that is infinite, or a key that makes a score infinite or NaN,
    # counts where it is seen and only there
    q, kv, tables, n = make(dev, [70, 70, 70, 70], 2, 1, 64, 16, "bf16")
    q = q.abs() + 0.1
    for row, (i, t, val) in enumerate([(1, 40, math.inf), (0, 33, -math.inf), (0, 69, math.nan)]):
        kv[i, tables[row, t // 16].long(), 0, t % 16] = val
    out, lse = attention.paged_decode(q, kv[0], kv[1], tables, n, return_lse=True)
    assert bool((out[0] == math.inf).all())
    keep = torch.ones(70, dtype=torch.bool, device=dev)
    keep[33] = False  # (a score of -inf: as if it were not there)
    pages = tables[1, :5].long()
    k, v = (kv[i, pages, 0].double().reshape(-1, 64)[:70] for i in (0, 1))
    p = torch.softmax((q[1].double() @ k[keep].t().contiguous()) / 8, -1)
    want = p @ v[keep]
    assert bool(((out[1].double() - want).abs() <= 2.0**-8 * want.abs() + 2.0**-12 * (p @ v[keep].abs())).all())
    assert bool(out[2].isnan().all() and lse[2].isnan().all())
    check(out, q, kv, tables, n, lse, rows=[3])
    # outside the window none of them shows
    out = attention.paged_decode(q, kv[0], kv[1], tables, n - 1, window=28)
    check(out, q, kv, tables, n - 1, window=28)


def test_strides(dev):
    # q out of a fused projection; keys and values interleaved, slots before heads
    lens = [40, 0, 333]
    q, kv, tables, n = make(dev, lens, 8, 2, 64, 16, "f16")
    want = attention.paged_decode(q, kv[0], kv[1], tables, n)
    fused = torch.zeros(3, 8 * 64 + 24, device=dev, dtype=torch.float16)
    fused[:, 5:5 + 512] = q.view(3, -1)
    q2 = fused[:, 5:5 + 512].unflatten(1, (8, 64))
    kv2 = kv.permute(1, 3, 0, 2, 4).contiguous().permute(2, 0, 3, 1, 4)  # [P, S, 2, H, D] in memory
    t2 = torch.zeros(3, tables.shape[1] + 3, device=dev, dtype=torch.int32)
    t2[:, 2:-1] = tables
    got = attention.paged_decode(q2, kv2[0], kv2[1], t2[:, 2:-1], n)
    assert torch.equal(got, want)
    # keys that start at any element
    odd = torch.zeros(kv.numel() + 1, device=dev, dtype=torch.float16)[1:].view(kv.shape)
    odd.copy_(kv)
    assert torch.equal(attention.paged_decode(q, odd[0], odd[1], tables, n), want)


def test_bad_pages_and_lengths(dev):
    lens = [100, 100, 100, 100]
    q, kv, tables, n = make(dev, lens, 4, 2, 64, 16, "bf16")
    want = attention.paged_decode(q, kv[0], kv[1], tables, n)
    moe.device_error()
    bad = tables.clone()
    bad[0, 2], bad[1, 6], bad[2, 0] = -1, 1 << 29, kv.shape[1]
    got = attention.paged_decode(q, kv[0], kv[1], bad, n)
    with pytest.raises(Exception, match="out of range"):
        moe.device_error()
    assert bool(got[:3].isnan().all()) and torch.equal(got[3], want[3])
    # a length past the table is cut and reported, a negative one is an empty row
    n2 = torch.tensor([100, 7 * 16 + 1, -3, 100], dtype=torch.int32, device=dev)
    full = torch.where(torch.isnan(kv), torch.zeros_like(kv), kv)
    got = attention.paged_decode(q, full[0], full[1], tables, n2)
    with pytest.raises(Exception, match="out of range"):
        moe.device_error()
    n3 = n2.clamp(0, 7 * 16)
    check(got, q, full, tables, n3)
    moe.device_error()
    # no pages at all
    z = torch.zeros(1, dtype=torch.int32, device=dev)
    out = attention.paged_decode(q[:1], kv[0, :0], kv[1, :0], tables[:1], z)
    assert not bool(out.any())
    out = attention.paged_decode(q[:1], kv[0], kv[1], tables[:1, :0], z)
    assert not bool(out.any())


def test_far_offsets(dev):
    # pages beyond 2^31 and 2^32 elements of the cache
    P, S, D = 70000, 64, 256
    kv = torch.zeros(2, P, 2, S, D, device=dev, dtype=torch.bfloat16)  # 9.2 GB, 2.3e9 elements a half
    q, small, tables, n = make(dev, [200, 130], 4, 2, D, S, "bf16")
    far = torch.arange(P - small.shape[1], P, device=dev)
    kv[:, far] = small
    want = attention.paged_decode(q, small[0], small[1], tables, n)
    tables = torch.where(tables < small.shape[1], tables + (P - small.shape[1]), tables)
    assert torch.equal(attention.paged_decode(q, kv[0], kv[1], tables.int(), n), want)
    # keys and values of one page side by side: strides past 2^32 elements too
    both = kv.view(2 * P, 2, S, D)
    assert torch.equal(attention.paged_decode(q, both[:P], both[P:], tables.int(), n), want)


def test_streams_and_graph(dev):
    lens = [900, 0, 33, 6000]
    q, kv, tables, n = make(dev, lens, 8, 2, 128, 16, "bf16")
    c = kvcache.PagedCache(kv.unsqueeze(0).contiguous(), rows=4, width=tables.shape[1])
    want = attention.paged_decode(q, kv[0], kv[1], tables, n)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    got = c.attend(0, q, tables, n, stream=side)
    side.synchronize()
    assert torch.equal(got, want)
    out = torch.empty_like(want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        attention.paged_decode(q, kv[0], kv[1], tables, n, out=out)
    for i in range(4):
        q.copy_(torch.randn(q.shape, generator=torch.Generator().manual_seed(i)))
        n[2] = 40 if i % 2 else 20  # (within the pages the row has)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out[[0, 1, 3]], attention.paged_decode(q, kv[0], kv[1], tables, n)[[0, 1, 3]])
        assert bool(torch.isfinite(out[2]).all()) == (i % 2 == 0)


def test_refusals(dev):
    q, kv, tables, n = make(dev, [40, 33], 4, 2, 64, 16, "bf16")
    ok = dict(q=q, k_pages=kv[0], v_pages=kv[1], tables=tables, lens=n)
    attention.paged_decode(**ok)
    f = torch.zeros(3, device=dev)
    for bad in (dict(q=q.float()), dict(q=q.half()), dict(q=q[:, :3]), dict(q=q[0]), dict(q=q.cpu()),
                dict(q=q[..., :32]), dict(k_pages=kv[0].half()), dict(v_pages=kv[1, :1]),
                dict(tables=tables.long()), dict(tables=tables[:1]), dict(lens=n.long()), dict(lens=n[:1]),
                dict(window=-1), dict(softcap=-1.0), dict(softcap=math.nan), dict(slopes=f), dict(k_scale=f),
                dict(v_scale=f[:2].half()), dict(out=torch.empty_like(q).float()), dict(out=q[:1]),
                dict(q=q.transpose(1, 2)[..., :2].transpose(1, 2)[..., ::2]), dict(q=q[..., ::2])):
        with pytest.raises(ValueError):
            attention.paged_decode(**dict(ok, **bad))
    e = attention.paged_decode(q[:0], kv[0], kv[1], tables[:0], n[:0], return_lse=True)
    assert e[0].shape == (0, 4, 64) and e[1].shape == (0, 4)


def test_result_over_an_input_is_refused(dev):
    q, kv, tables, n = make(dev, [40, 33], 4, 2, 64, 16, "bf16")
    pool = torch.zeros(2 * q.numel(), dtype=q.dtype, device=dev)
    a, b = pool[:q.numel()].view_as(q), pool[q.numel():].view_as(q)
    a.copy_(q)
    for out in (a, pool[8:8 + q.numel()].view_as(q), kv.view(-1)[:q.numel()].view_as(q)):
        with pytest.raises(ValueError, match="overlaps"):
            attention.paged_decode(a, kv[0], kv[1], tables, n, out=out)
    want = attention.paged_decode(q, kv[0], kv[1], tables, n)
    assert attention.paged_decode(a, kv[0], kv[1], tables, n, out=b) is not None
    assert torch.equal(b, want)  # the neighbour in the same storage is fine


@pytest.mark.parametrize("lens,Hq,Hkv,D,S", [
    ([4100], 4, 1, 128, 16), ([3000, 0, 77, 2500], 40, 1, 128, 16), ([2000, 1500], 72, 2, 64, 8),
    ([1700, 0, 0, 900], 13, 1, 256, 16), ([900, 33], 48, 2, 256, 5), ([2600], 128, 1, 8, 16),
    ([700] * 3 + [0] + [40] * 60, 32, 8, 64, 16), ([300] * 63 + [0, 1], 16, 8, 40, 16)])
def test_rows_in_parts(dev, lens, Hq, Hkv, D, S):
    # one row to 520, each in many shares or few, their heads joined by one workgroup or several
    q, kv, tables, n = make(dev, lens, Hq, Hkv, D, S)
    out, lse = attention.paged_decode(q, kv[0], kv[1], tables, n, return_lse=True)
    check(out, q, kv, tables, n, lse)
    assert torch.equal(out, attention.paged_decode(q, kv[0], kv[1], tables, n))
    moe.device_error()


@pytest.mark.parametrize("t", ["bf16", "f16"])
@pytest.mark.parametrize("lens", [[1, 2, 33, 70, 200], [1, 2, 40, 3000, 5000]], ids=["rows", "shares"])
@pytest.mark.parametrize("place", ["greatest", "least", "last"])
def test_infinite_values(dev, t, lens, place):
    # an infinite value gives its infinity under any weight (their two parts of
    # either size, the greatest's second one zero, a single token's too), two of
    # opposite signs NaN, and the other dims keep their bits
    q, kv, tables, n = make(dev, lens, 32, 2, 64, 16, t)
    clean, lse = attention.paged_decode(q, kv[0], kv[1], tables, n, return_lse=True)
    check(clean, q, kv, tables, n, lse)
    bad = kv.clone()
    want = clean.clone()
    for b, m in enumerate(lens):
        for h in range(2):
            pages = tables[b, :-(-m // 16)].long()
            x = kv[0, pages, h].double().reshape(-1, 64)[:m] @ q[b, 16 * h].double()
            at = {"greatest": int(x.argmax()), "least": int(x.argmin()), "last": m - 1}[place]
            heads = slice(16 * h, 16 * h + 16)

            def plant(at, dims, val):
                bad[1, tables[b, at // 16].long(), h, at % 16, dims] = val
            plant(at, slice(0, 16), math.inf)
            plant(at, slice(16, 32), -math.inf)
            want[b, heads, :16], want[b, heads, 16:32] = math.inf, -math.inf
            if m > 1:
                plant(at, slice(32, 40), math.inf)
                plant((at + m // 2) % m, slice(32, 40), -math.inf)
                want[b, heads, 32:40] = math.nan
    got, lse2 = attention.paged_decode(q, bad[0], bad[1], tables, n, return_lse=True)
    assert torch.equal(lse, lse2)
    assert torch.equal(got.nan_to_num(7.0, 8.0, 9.0), want.nan_to_num(7.0, 8.0, 9.0))
    assert torch.equal(got.isnan(), want.isnan())


@pytest.mark.parametrize("t", ["bf16", "f16"])
@pytest.mark.parametrize("n", [30, 70, 6000])
@pytest.mark.parametrize("newest", [False, True])
def test_infinite_value_of_small_weight(dev, t, n, newest):
    # e^-60 of the greatest weight, in one step or over many: far below f16's
    # range, above f32's least
    q, kv, tables, lens = make(dev, [n], 4, 1, 64, 16, t)
    kv[0] *= 0.125
    at = n - 1 if newest else 0
    kv[1, tables[0, at // 16].long(), 0, at % 16, :8] = math.inf
    kv[1, tables[0, at // 16].long(), 0, at % 16, 8:16] = -math.inf
    slopes = torch.full((4,), (-60.0 if newest else 60.0) / (n - 1), device=dev)
    out = attention.paged_decode(q, kv[0], kv[1], tables, lens, slopes=slopes)
    assert bool((out[..., :8] == math.inf).all() and (out[..., 8:16] == -math.inf).all())
    assert bool(torch.isfinite(out[..., 16:]).all())


def test_caps_at_the_ends_of_the_range(dev):
    q, kv, tables, n = make(dev, [40, 33], 4, 2, 64, 16, "bf16")
    run = lambda cap: attention.paged_decode(q, kv[0], kv[1], tables, n, softcap=cap, return_lse=True)
    for cap in (math.inf, 1e300, 1e-39, 1e-60):
        with pytest.raises(ValueError, match="softcap"):
            run(cap)
    for cap in (1e-30, 1e-3, 1e6, 1e30):
        out, lse = run(cap)
        check(out, q, kv, tables, n, lse, softcap=cap if cap < 1e6 else 0.0)
