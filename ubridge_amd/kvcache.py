"""A paged key-value cache whose state stays on the device: storing new tokens
(with their rotation), freeing, forking and compacting without a host copy of
page tables, so that the calls can be enqueued, or captured, ahead."""
import operator

import torch

from .attention import paged_decode
from .native import _native, call
from .ops import _need_cuda


_TYPES = (torch.float16, torch.bfloat16, torch.float8_e4m3fn)


def _in_place(name):
    """A tensor of a cache, one of several views of the same memory: it may be
    written (x += 1 assigns the same tensor again), not replaced."""
    def replace(self, t):
        if t is not getattr(self, "_" + name):
            raise AttributeError(f"PagedCache.{name} is written in place, not replaced")
    return property(operator.attrgetter("_" + name), replace)


class PagedCache:
    """kv [L, 2, P, H, S, D]: keys and values of L layers in P pages of S tokens
    (f16, bf16 or e4m3; k_scale, v_scale f32 [H] are what a stored e4m3 value
    stands for).  `rows` sequences of at most `width` pages each.

    The state is one int32 buffer `meta` [P + rows + rows * width]: refs [P],
    how many rows hold a page; lens [rows], tokens; tables [rows, width], pages
    in order, -1 for none.  The three are views a program may read and write
    in place (it gives a growing row its pages); without `meta` the pool starts empty.
    """

    def __init__(self, kv, rows, width, k_scale=None, v_scale=None, meta=None):
        _need_cuda(kv, k_scale, v_scale, meta)
        if kv.dim() != 6 or kv.shape[1] != 2 or not kv.is_contiguous() or kv.dtype not in _TYPES:
            raise ValueError("PagedCache takes a contiguous f16, bf16 or e4m3 [L, 2, P, H, S, D]")
        L, _, P, H, S, D = kv.shape
        if 0 in (L, H, S, D) or rows < 0 or width < 0:
            raise ValueError(f"PagedCache: kv {list(kv.shape)}, rows={rows}, width={width}")
        for name, t in (("k_scale", k_scale), ("v_scale", v_scale)):
            if t is not None and (t.shape != (H,) or t.dtype != torch.float32 or not t.is_contiguous()):
                raise ValueError(f"PagedCache: {name} must be contiguous float32 [{H}]")
            if t is not None and kv.dtype != torch.float8_e4m3fn:
                raise ValueError(f"PagedCache: {name} goes with e4m3 pages")
        n = P + rows + rows * width
        if meta is None:
            meta = torch.zeros(n, dtype=torch.int32, device=kv.device)
            meta[P + rows:] = -1
        elif meta.shape != (n,) or meta.dtype != torch.int32 or not meta.is_contiguous():
            raise ValueError(f"PagedCache: meta must be contiguous int32 [{n}]")
        self._kv, self._meta, self.k_scale, self.v_scale = kv, meta, k_scale, v_scale
        self.L, self.P, self.H, self.S, self.D, self.rows, self.width = L, P, H, S, D, rows, width
        self._views()

    def _views(self):
        P, rows, meta = self.P, self.rows, self._meta
        self._refs, self._lens = meta[:P], meta[P:P + rows]
        self._tables = meta[P + rows:].view(rows, self.width)

    # a copy (deepcopy, pickle) is a cache of its own: its views are of its own state
    def __getstate__(self):
        return {k: v for k, v in vars(self).items() if k not in ("_refs", "_lens", "_tables")}

    def __setstate__(self, state):
        vars(self).update(state)
        self._views()

    kv, meta, refs, lens, tables = map(_in_place, ("kv", "meta", "refs", "lens", "tables"))

    def layer(self, i):
        """(k_pages, v_pages) of a layer, [P, H, S, D] each."""
        return self.kv[i, 0], self.kv[i, 1]

    def append(self, layer, q, k, v, slots, positions=None, rope=None, stream=None):
        """Store k, v [T, H, D] of one layer at slots int64 [T] (page * S + place;
        negative: nowhere; no slot twice) and return q.  With a Rope and
        positions q and k are turned, in one launch with the store.  e4m3 pages
        take x / scale, saturating.  A slot past the cache raises the flag that
        moe.device_error() reads.  It has no gradient: what is stored, and a turned
        q, is cut from the graph of k, v and q (rope.Rope by itself is
        differentiable)."""
        turns, rot, inter, factor = (None, 0, False, 1.0) if rope is None else (
            rope.turns, rope.rot, rope.interleaved, rope.factor)
        return call(_native.append, stream, self.kv, layer, self.k_scale, self.v_scale, q, k, v, slots,
                    positions, turns, rot, inter, factor)

    def attend(self, layer, q, tables=None, lens=None, **kw):
        """attention.paged_decode of q [B, Hq, D] over a layer, for all rows or
        for the rows whose tables and lens are given.  It has no gradient."""
        k, v = self.layer(layer)
        return paged_decode(q, k, v, self.tables if tables is None else tables,
                            self.lens if lens is None else lens, k_scale=self.k_scale,
                            v_scale=self.v_scale, **kw)

    def free(self, rows, stream=None):
        """The rows named (int32 [n]) lose their pages and become empty."""
        call(_native.free, stream, self.kv, self.meta, self.rows, self.width, rows)

    def fork(self, src, dst, stream=None):
        """Empty rows dst (int32 [n], all different, without tokens or pages)
        become samples of rows src: whole pages are shared, a part-filled last page is copied to the lowest
        free page.  Returns int32 [n], the new page or -1.  A row that is not
        empty or not there, for which no page is left, or whose prompt has a
        page that is not there, keeps its state, gives -1 and raises the flag
        that moe.device_error() reads."""
        return call(_native.fork, stream, self.kv, self.meta, self.rows, self.width, src, dst)

    def compact(self, stream=None):
        """Move the used pages to the low end of the pool; tables and refs follow.
        Returns their number, an int32 tensor."""
        return call(_native.compact, stream, self.kv, self.meta, self.rows, self.width)
