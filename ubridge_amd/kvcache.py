"""A paged key-value cache whose state stays on the device: storing new tokens
(with their rotation), freeing, forking and compacting without a host copy of
page tables, so that the calls can be enqueued, or captured, ahead."""
import ctypes
import struct

import torch

from ._lib import check, lib, register
from .attention import _CODE, paged_decode
from .ops import _DT_CODE, _empty, _need_cuda, stream_ptr
from .rope import _ARGS as _ROPE_ARGS
from .rope import _heads, _positions

_vp, _i = ctypes.c_void_p, ctypes.c_int
register("ubridge_rope_append", _i, [_vp, _vp])
register("ubridge_kv_free", _i, [_vp, _vp, _i, _vp])
register("ubridge_kv_fork", _i, [_vp, _vp, _vp, _i, _vp, _vp])
register("ubridge_kv_compact", _i, [_vp, _vp, _vp])


class PagedCache:
    """kv [L, 2, P, H, S, D]: keys and values of L layers in P pages of S tokens
    (f16, bf16 or e4m3; k_scale, v_scale f32 [H] are what a stored e4m3 value
    stands for).  `rows` sequences of at most `width` pages each.

    The state is one int32 buffer `meta` [P + rows + rows * width]: refs [P],
    how many rows hold a page; lens [rows], tokens; tables [rows, width], pages
    in order, -1 for none.  The three are views a program may read and write
    (it gives a growing row its pages); without `meta` the pool starts empty.
    """

    def __init__(self, kv, rows, width, k_scale=None, v_scale=None, meta=None):
        _need_cuda(kv, k_scale, v_scale, meta)
        if kv.dim() != 6 or kv.shape[1] != 2 or not kv.is_contiguous() or kv.dtype not in _CODE:
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
        self.kv, self.meta, self.k_scale, self.v_scale = kv, meta, k_scale, v_scale
        self.L, self.P, self.H, self.S, self.D, self.rows, self.width = L, P, H, S, D, rows, width
        self.refs, self.lens = meta[:P], meta[P:P + rows]
        self.tables = meta[P + rows:].view(rows, width)
        page = H * S * D * kv.element_size()
        p = meta.data_ptr()
        self._pool = struct.pack("@4Pq6i", kv.data_ptr(), p, p + 4 * P, p + 4 * (P + rows), page, L,
                                 P, S, rows, width, 0)

    def layer(self, i):
        """(k_pages, v_pages) of a layer, [P, H, S, D] each."""
        return self.kv[i, 0], self.kv[i, 1]

    def append(self, layer, q, k, v, slots, positions=None, rope=None, stream=None):
        """Store k, v [T, H, D] of one layer at slots int64 [T] (page * S + place;
        negative: nowhere; no slot twice) and return q.  With a Rope and
        positions q and k are turned, in one launch with the store.  e4m3 pages
        take x / scale, saturating.  A slot past the cache raises the flag that
        moe.device_error() reads."""
        _need_cuda(q, k, v, slots, positions)
        dt, ct = _DT_CODE.get(k.dtype), _CODE[self.kv.dtype]
        if dt is None or v.dtype != k.dtype or ct not in (dt, 3):
            raise ValueError(f"PagedCache.append: {k.dtype} and {v.dtype} into {self.kv.dtype} pages")
        if not 0 <= layer < self.L:
            raise ValueError(f"PagedCache.append: layer {layer} of {self.L}")
        if (rope is None) != (positions is None):
            raise ValueError("PagedCache.append: rope and positions go together")
        T, H, D = k.shape if k.dim() == 3 else (0, -1, -1)
        if H != self.H or D != self.D or v.shape != k.shape:
            raise ValueError(f"PagedCache.append: k and v must be [T, {self.H}, {self.D}]")
        if slots.shape != (T,) or slots.dtype != torch.int64 or not slots.is_contiguous():
            raise ValueError(f"PagedCache.append: slots must be contiguous int64 [{T}]")
        kp, kt, kh = _heads("k", k, T, D)
        vp, vt, vh = _heads("v", v, T, D)
        qp = qt = qh = Hq = rot = pp = p64 = inter = turns = 0
        factor, qo = 1.0, q
        if rope is not None:
            if q.dtype != k.dtype:
                raise ValueError("PagedCache.append: q and k of one type")
            if rope.rot > D:
                raise ValueError(f"PagedCache.append: rot={rope.rot} of heads of {D}")
            _need_cuda(rope.turns)
            qp, qt, qh = _heads("q", q, T, D)
            Hq = q.shape[1]
            qo = _empty((T, Hq, D), q.dtype, q.device, stream)
            pp, p64 = _positions(positions, T)
            rot, inter, factor, turns = rope.rot, rope.interleaved, rope.factor, rope.turns.data_ptr()
        page = H * self.S * D
        base = self.kv.data_ptr() + 2 * layer * self.P * page * self.kv.element_size()
        args = _ROPE_ARGS.pack(qp, kp, vp, qo.data_ptr() if Hq else 0, 0, pp, turns, base,
                               base + self.P * page * self.kv.element_size(), slots.data_ptr(),
                               0 if self.k_scale is None else self.k_scale.data_ptr(),
                               0 if self.v_scale is None else self.v_scale.data_ptr(), qt, qh, kt,
                               kh, vt, vh, page, T, Hq, H, D, rot, inter, 0, p64, dt, ct, self.P,
                               self.S, factor, 0)
        rc = lib.ubridge_rope_append(args, stream_ptr(stream))
        if rc:
            check(rc)
        return qo

    def attend(self, layer, q, tables=None, lens=None, **kw):
        """attention.paged_decode of q [B, Hq, D] over a layer, for all rows or
        for the rows whose tables and lens are given."""
        k, v = self.layer(layer)
        return paged_decode(q, k, v, self.tables if tables is None else tables,
                            self.lens if lens is None else lens, k_scale=self.k_scale,
                            v_scale=self.v_scale, **kw)

    def _rows(self, name, t):
        _need_cuda(t)
        if t.dim() != 1 or t.dtype != torch.int32 or not t.is_contiguous():
            raise ValueError(f"PagedCache: {name} must be contiguous int32 [n]")
        return t.data_ptr(), t.shape[0]

    def free(self, rows, stream=None):
        """The rows named (int32 [n]) lose their pages and become empty."""
        p, n = self._rows("rows", rows)
        rc = lib.ubridge_kv_free(self._pool, p, n, stream_ptr(stream))
        if rc:
            check(rc)

    def fork(self, src, dst, stream=None):
        """Empty rows dst (int32 [n], all different) become samples of rows src:
        whole pages are shared, a part-filled last page is copied to the lowest
        free page.  Returns int32 [n], the new page or -1.  A row that is not
        empty or not there, or for which no page is left, keeps its state, gives
        -1 and raises the flag that moe.device_error() reads."""
        sp, n = self._rows("src", src)
        dp, m = self._rows("dst", dst)
        if m != n or n > 65535:
            raise ValueError(f"PagedCache.fork: {n} prompts, {m} samples (as many, at most 65535)")
        new = _empty((n,), torch.int32, self.kv.device, stream)
        rc = lib.ubridge_kv_fork(self._pool, sp, dp, n, new.data_ptr(), stream_ptr(stream))
        if rc:
            check(rc)
        return new

    def compact(self, stream=None):
        """Move the used pages to the low end of the pool; tables and refs follow.
        Returns their number, an int32 tensor."""
        n = _empty((), torch.int32, self.kv.device, stream)
        rc = lib.ubridge_kv_compact(self._pool, n.data_ptr(), stream_ptr(stream))
        if rc:
            check(rc)
        return n
