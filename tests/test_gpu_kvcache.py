"""Freeing, forking and compacting a paged cache against the same steps on
lists.  All of it is copies and counts: equality throughout."""
import copy
import pickle

import numpy as np
import pytest
import torch

from ubridge_amd import attention, int8, kvcache, moe, rope

pytestmark = pytest.mark.gpu


class Lists:
    """The pool in plain Python."""

    def __init__(self, P, S, rows, width):
        self.P, self.S, self.width = P, S, width
        self.refs = [0] * P
        self.lens = [0] * rows
        self.rows = [[] for _ in range(rows)]

    def load(self, meta):
        m = [int(x) for x in meta.cpu()]
        R = len(self.lens)
        self.refs, self.lens = m[:self.P], m[self.P:self.P + R]
        t = m[self.P + R:]
        self.rows = [[p for p in t[r * self.width:(r + 1) * self.width] if p >= 0] for r in range(R)]

    def meta(self):
        t = [p for r in self.rows for p in r + [-1] * (self.width - len(r))]
        return torch.tensor(self.refs + self.lens + t, dtype=torch.int32)

    def free(self, rows):
        for r in rows:
            for p in self.rows[r]:
                self.refs[p] -= 1
            self.rows[r], self.lens[r] = [], 0

    def fork(self, src, dst, kv):
        new, frozen = [], kv.clone()
        free = iter([p for p in range(self.P) if self.refs[p] == 0])
        state = [(list(self.rows[s]), self.lens[s]) for s in src]
        for (pages, n), d in zip(state, dst):
            pages, fresh = pages[:-(-n // self.S)], -1
            if n % self.S:
                fresh = next(free)
                kv[:, :, fresh] = frozen[:, :, pages[-1]]
                pages = pages[:-1] + [fresh]
            for p in pages:
                self.refs[p] += 1
            self.rows[d], self.lens[d] = pages, n
            new.append(fresh)
        return new

    def compact(self, kv):
        used = [p for p in range(self.P) if self.refs[p]]
        n = len(used)
        out, holes = [p for p in used if p >= n], [p for p in range(n) if not self.refs[p]]
        move = dict(zip(out, holes))
        for f, t in move.items():
            kv[:, :, t] = kv[:, :, f].clone()
            self.refs[t], self.refs[f] = self.refs[f], 0
        self.rows = [[move.get(p, p) for p in r] for r in self.rows]
        return n


def pool(dev, L, P, H, S, D, rows, width, dtype, seed, used=0.6, share=True):
    r = np.random.RandomState(seed)
    g = torch.Generator().manual_seed(seed)
    n = L * 2 * P * H * S * D
    kv = torch.randint(0, 120, (n * torch.empty(0, dtype=dtype).element_size(),), generator=g,
                       dtype=torch.uint8).view(dtype).view(L, 2, P, H, S, D)
    m = Lists(P, S, rows, width)
    order = list(r.permutation(P))
    for b in range(rows - rows // 3):
        left = int(P * used) - (P - len(order))
        if left <= 0:
            break
        k = r.randint(1, min(left, width) + 1)
        pages = [int(order.pop()) for _ in range(k)]
        if share and b and m.rows[b - 1] and r.rand() < 0.5:  # whole pages of the row before
            whole = m.rows[b - 1][:m.lens[b - 1] // S][:k]
            for i, p in enumerate(whole):
                order.insert(0, pages[i])
                pages[i] = p
        m.rows[b], m.lens[b] = pages, (k - 1) * S + r.randint(1, S + 1)
        for p in pages:
            m.refs[p] += 1
    c = kvcache.PagedCache(kv.to(dev), rows, width, meta=m.meta().to(dev))
    return c, m, kv


def raw(x):
    return x.cpu().view(torch.uint8) if x.dtype == torch.float8_e4m3fn else x.cpu().view(torch.int16)


def same(c, m, kv):
    assert torch.equal(c.meta.cpu(), m.meta())
    assert torch.equal(raw(c.kv), raw(kv))


SHAPES = [(1, 5, 1, 1, 1, 4, 3), (2, 40, 2, 8, 64, 12, 6), (3, 64, 1, 24, 80, 30, 3), (1, 33, 3, 5, 7, 9, 4),
          (2, 1500, 1, 8, 16, 200, 20), (1, 9000, 1, 2, 8, 3000, 4), (2, 70, 4, 64, 128, 10, 9)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float8_e4m3fn])
@pytest.mark.parametrize("shape", SHAPES)
def test_free_fork_compact(dev, shape, dtype):
    L, P, H, S, D, rows, width = shape
    for seed in range(3):
        c, m, kv = pool(dev, L, P, H, S, D, rows, width, dtype, seed)
        r = np.random.RandomState(seed + 100)
        live = [b for b in range(rows) if m.lens[b]]
        gone = [int(x) for x in r.permutation(live)[:len(live) // 3]]
        c.free(torch.tensor(gone, dtype=torch.int32, device=dev))
        m.free(gone)
        same(c, m, kv)
        empty = [b for b in range(rows) if not m.lens[b]]
        live = [b for b in range(rows) if m.lens[b]]
        free = sum(x == 0 for x in m.refs)
        dst = empty[:min(len(empty), free)]
        src = [int(r.choice(live)) for _ in dst] if live else []
        dst = dst[:len(src)]
        ti = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)
        new = c.fork(ti(src), ti(dst))
        assert new.tolist() == m.fork(src, dst, kv)
        same(c, m, kv)
        assert int(c.compact()) == m.compact(kv)
        same(c, m, kv)
        assert int(c.compact()) == m.compact(kv)  # nothing left to move
        same(c, m, kv)
        moe.device_error()


def test_more_samples_than_a_workgroup(dev):
    # 2500 samples of 3 prompts; pages far up the pool, behind 20000 in use
    P, S, rows, width = 24000, 4, 2600, 2
    m = Lists(P, S, rows, width)
    for p in range(20000):
        m.refs[p] = 1
    m.rows[0], m.lens[0], m.rows[1], m.lens[1], m.rows[2], m.lens[2] = [7, 19999], 6, [3], 4, [11], 1
    kv = torch.randint(0, 1000, (1, 2, P, 1, S, 4), dtype=torch.int16).view(torch.float16)
    c = kvcache.PagedCache(kv.to(dev), rows, width, meta=m.meta().to(dev))
    src, dst = [j % 3 for j in range(2500)], [2599 - j for j in range(2500)]
    ti = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)
    assert c.fork(ti(src), ti(dst)).tolist() == m.fork(src, dst, kv)
    same(c, m, kv)


def test_empty_and_full_pools(dev):
    for used in (0, 1):
        m = Lists(16, 4, 4, 16)
        if used:
            m.rows[1], m.lens[1], m.refs = list(range(15, -1, -1)), 64, [1] * 16
        kv = torch.randn(1, 2, 16, 1, 4, 8).half()
        c = kvcache.PagedCache(kv.to(dev), 4, 16, meta=m.meta().to(dev))
        assert int(c.compact()) == m.compact(kv) == 16 * used
        same(c, m, kv)
    # a prompt of whole pages needs no free page
    t = lambda *x: torch.tensor(x, dtype=torch.int32, device=dev)
    assert c.fork(t(1, 1, 0), t(0, 2, 3)).tolist() == m.fork([1, 1, 0], [0, 2, 3], kv) == [-1] * 3
    same(c, m, kv)
    fresh = kvcache.PagedCache(torch.zeros(1, 2, 3, 1, 4, 8, device=dev).half(), 2, 5)
    assert fresh.refs.tolist() == [0] * 3 and fresh.lens.tolist() == [0, 0]
    assert fresh.tables.tolist() == [[-1] * 5] * 2
    fresh.free(t())
    assert fresh.fork(t(), t()).shape == (0,)


def flagged():
    with pytest.raises(Exception, match="out of range"):
        moe.device_error()
    moe.device_error()


def test_errors_are_reported(dev):
    t = lambda *x: torch.tensor(x, dtype=torch.int32, device=dev)
    m = Lists(8, 4, 6, 4)
    m.rows[0], m.lens[0] = [2, 5], 6
    m.rows[1], m.lens[1] = [1], 4
    for p in (2, 5, 1):
        m.refs[p] = 1
    kv = torch.randn(1, 2, 8, 1, 4, 8).half()
    c = kvcache.PagedCache(kv.to(dev), 6, 4, meta=m.meta().to(dev))
    moe.device_error()
    # rows that are not there, a sample in a row that is in use: the others go on
    assert c.fork(t(0, -1, 0, 9, 0), t(2, 3, 1, 4, 6)).tolist() == m.fork([0], [2], kv) + [-1] * 4
    same(c, m, kv)
    flagged()
    c.free(t(6, 2, -1))
    m.free([2])
    same(c, m, kv)
    flagged()
    # a row named twice is freed once
    c.free(t(0, 0))
    m.free([0])
    same(c, m, kv)
    moe.device_error()
    # no page left: the samples that found one are whole, the rest stay empty
    m.rows[0], m.lens[0] = [2, 5], 6
    m.refs = [0, 1, 1, 1, 1, 1, 1, 1]
    c.meta.copy_(m.meta())
    got = c.fork(t(0, 0, 1), t(2, 3, 4)).tolist()
    assert got == [0, -1, -1]
    m.fork([0, 1], [2, 4], kv)
    same(c, m, kv)
    flagged()
    # a table that names a page that is not there
    c.tables[1, 0] = 8
    c.free(t(1))
    assert c.lens[1] == 0 and c.refs.tolist() == m.refs
    flagged()
    c.free(t(0, 2, 4))
    c.tables[0, 0], c.lens[0] = 99, 3
    assert c.fork(t(0), t(5)).tolist() == [-1] and c.lens[5] == 0
    flagged()


def test_graph(dev):
    c, m, kv = pool(dev, 2, 200, 2, 8, 32, 40, 8, torch.bfloat16, 5)
    meta0, kv0 = c.meta.clone(), c.kv.clone()
    live = [b for b in range(40) if m.lens[b]]
    t = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)
    gone, src, dst = t(live[:3]), t(live[4:7]), t(live[:3])
    def step():
        c.free(gone)
        return c.fork(src, dst), c.compact()
    graph = torch.cuda.CUDAGraph()
    step()
    want = c.meta.clone(), c.kv.clone()
    with torch.cuda.graph(graph):
        step()
    for _ in range(3):
        c.meta.copy_(meta0)
        c.kv.copy_(kv0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(c.meta, want[0]) and torch.equal(raw(c.kv), raw(want[1]))


def test_refusals(dev):
    kv = torch.zeros(1, 2, 4, 1, 4, 8, device=dev).half()
    t = torch.zeros(2, dtype=torch.int32, device=dev)
    s = torch.ones(1, device=dev)
    for args, kw in (((kv.float(), 2, 2), {}), ((kv[0], 2, 2), {}), ((kv.cpu(), 2, 2), {}), ((kv, -1, 2), {}),
                     ((kv.transpose(4, 5), 2, 2), {}), ((kv, 2, 2), dict(meta=t)), ((kv, 2, 2), dict(k_scale=s)),
                     ((kv[:, :1], 2, 2), {}), ((kv.to(torch.float8_e4m3fn), 2, 2), dict(v_scale=t.float()))):
        with pytest.raises(ValueError):
            kvcache.PagedCache(*args, **kw)
    c = kvcache.PagedCache(kv, 2, 2)
    for call in (lambda: c.free(t.long()), lambda: c.free(t.cpu()), lambda: c.fork(t, t[:1]),
                 lambda: c.fork(t.view(1, 2), t), lambda: c.free(torch.zeros(4, dtype=torch.int32, device=dev)[::2])):
        with pytest.raises(ValueError):
            call()


def test_state_is_written_in_place(dev):
    kv = torch.zeros(1, 2, 4, 2, 4, 8, device=dev, dtype=torch.bfloat16)
    c = kvcache.PagedCache(kv, 2, 2)
    for name in ("kv", "meta", "refs", "lens", "tables"):
        with pytest.raises(AttributeError):
            setattr(c, name, getattr(c, name).clone())
    c.lens += 1
    assert c.lens.tolist() == [1, 1] and c.meta[4:6].tolist() == [1, 1]
    x = torch.ones(1, 2, 8, device=dev, dtype=torch.bfloat16)
    slots = torch.zeros(1, dtype=torch.int64, device=dev)
    c.k_scale = torch.ones(1, device=dev)  # of two heads
    with pytest.raises(ValueError):
        c.append(0, None, x, x, slots)
    c.k_scale = None
    r = rope.Rope(8, device=dev)
    for turns in (r.turns[:3], r.turns.float()):
        bad = rope.Rope(8, device=dev)
        bad.turns = turns
        with pytest.raises(ValueError):
            c.append(0, x, x, x, slots, slots, bad)
        with pytest.raises(ValueError):
            bad(x, x, slots)


@pytest.mark.parametrize("how", [copy.deepcopy, lambda c: pickle.loads(pickle.dumps(c))], ids=["deepcopy", "pickle"])
def test_copies_are_caches_of_their_own(dev, how):
    c, m, kv = pool(dev, 2, 200, 2, 8, 32, 40, 8, torch.bfloat16, 5)
    live = [b for b in range(40) if m.lens[b]]
    meta0, kv0 = c.meta.clone(), c.kv.clone()
    other = how(c)
    t = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)
    other.free(t(live[:3]))
    m.free(live[:3])
    assert other.fork(t(live[4:7]), t(live[:3])).tolist() == m.fork(live[4:7], live[:3], kv)
    assert int(other.compact()) == m.compact(kv)
    same(other, m, kv)
    assert torch.equal(other.tables.flatten(), other.meta[240:])
    assert torch.equal(c.meta, meta0) and torch.equal(raw(c.kv), raw(kv0))


@pytest.mark.parametrize("rows,width", [(20, 4), (20, 5000)])
def test_fork_of_a_prompt_with_a_bad_page(dev, rows, width):
    # a page that is not there, the last or a whole one before it: the sample is
    # refused, its row and the counts stay, the next sample gets the lowest free page
    P, S = 40, 4
    m = Lists(P, S, rows, width)
    for b, n in enumerate((9, 9, 9, 8, 9)):
        m.rows[b], m.lens[b] = [6 * b + 1 + i for i in range(-(-n // S))], n
        for p in m.rows[b]:
            m.refs[p] = 1
    kv = torch.randint(0, 1000, (2, 2, P, 1, S, 8), dtype=torch.int16).view(torch.float16)
    c = kvcache.PagedCache(kv.to(dev), rows, width, meta=m.meta().to(dev))
    t = lambda *x: torch.tensor(x, dtype=torch.int32, device=dev)
    bad = {(0, 0): -1, (1, 1): P, (2, 3): 1 << 29, (3, 1): -7, (4, 2): 1 << 30}  # (row 2's lies past its pages)
    for at, page in bad.items():
        c.tables[at] = page
    moe.device_error()
    got = c.fork(t(0, 2, 1, 2, 3, 4, 2), t(9, 10, 11, 12, 13, 14, 15)).tolist()
    new = m.fork([2, 2, 2], [10, 12, 15], kv)
    assert got == [-1, new[0], -1, new[1], -1, -1, new[2]]
    flagged()
    want = kvcache.PagedCache(kv.to(dev), rows, width, meta=m.meta().to(dev))
    for at, page in bad.items():
        want.tables[at] = page
    assert torch.equal(c.meta, want.meta) and torch.equal(raw(c.kv), raw(kv))


def test_fork_of_long_tables(dev):
    # some 300 samples of rows of up to 64 pages, one of no tokens among their prompts
    r = np.random.RandomState(3)
    P, S, rows, width = 5000, 4, 300, 64
    m = Lists(P, S, rows, width)
    order = [int(p) for p in r.permutation(P)]
    for b in range(8):
        n = int(r.randint(1, width * S + 1))
        m.rows[b], m.lens[b] = [order.pop() for _ in range(-(-n // S))], n
        for p in m.rows[b]:
            m.refs[p] = 1
    kv = torch.randint(0, 1000, (1, 2, P, 1, S, 8), dtype=torch.int16).view(torch.float16)
    c = kvcache.PagedCache(kv.to(dev), rows, width, meta=m.meta().to(dev))
    src, dst = [j % 9 for j in range(291)], [8 + j for j in range(291)]
    src = [8 + 291 if s == 8 else s for s in src]  # (an empty prompt)
    t = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)
    assert c.fork(t(src), t(dst)).tolist() == m.fork(src, dst, kv)
    same(c, m, kv)
    moe.device_error()


def test_fork_into_a_row_that_holds_a_page(dev):
    # a row without tokens that was given its pages ahead is not empty: it keeps
    # them, and no page is lost to the pool
    P, S, rows, width = 12, 4, 6, 70
    m = Lists(P, S, rows, width)
    m.rows[0], m.lens[0] = [2, 5], 6
    m.rows[1], m.rows[2] = [7], [8, 9]  # (no tokens)
    for p in (2, 5, 7, 8, 9):
        m.refs[p] = 1
    kv = torch.randn(1, 2, P, 1, S, 8).half()
    c = kvcache.PagedCache(kv.to(dev), rows, width, meta=m.meta().to(dev))
    c.tables[2, :2] = torch.tensor([-1, 8], device=dev)  # one page, not the first
    m.refs[9], m.rows[2] = 0, []
    c.refs[9] = 0
    moe.device_error()
    t = lambda *x: torch.tensor(x, dtype=torch.int32, device=dev)

    def state():
        meta = m.meta()
        meta[P + rows + 2 * width + 1] = 8 if m.refs[8] else -1
        return meta
    assert c.fork(t(0, 0, 0), t(1, 2, 3)).tolist() == [-1, -1] + m.fork([0], [3], kv)
    assert torch.equal(c.meta.cpu(), state()) and torch.equal(raw(c.kv), raw(kv))
    flagged()
    # a prompt of no tokens leaves such a row as it is
    assert c.fork(t(4), t(1)).tolist() == [-1]
    assert torch.equal(c.meta.cpu(), state())
    moe.device_error()
    # freed, it is empty
    c.free(t(1, 2))
    m.free([1])
    m.refs[8] = 0
    assert c.fork(t(0, 3), t(2, 1)).tolist() == m.fork([0, 3], [2, 1], kv)
    same(c, m, kv)
    moe.device_error()
