"""Attention over a paged key-value cache for decoding: one new token per
sequence, grouped heads, optional score cap, sliding window, bias by distance
and 8-bit pages."""
import ctypes
import struct

import torch

from ._lib import check, lib, register
from .ops import _empty, _need_cuda, stream_ptr

register("ubridge_paged_decode", ctypes.c_int, [ctypes.c_void_p, ctypes.c_void_p])

_CODE = {torch.float16: 1, torch.bfloat16: 2, torch.float8_e4m3fn: 3}
# UbridgePagedDecodeArgs: 10 pointers, 9 strides, 10 ints, scale, softcap
_ARGS = struct.Struct("@10P9q10i2f")


def _vector(name, t, n):
    if t is None:
        return 0
    if t.shape != (n,) or t.dtype != torch.float32 or not t.is_contiguous():
        raise ValueError(f"paged_decode: {name} must be contiguous float32 [{n}]")
    return t.data_ptr()


def paged_decode(q, k_pages, v_pages, tables, lens, scale=None, softcap=0.0, window=0, slopes=None,
                 k_scale=None, v_scale=None, out=None, return_lse=False, stream=None):
    """softmax(scale q K^T + ...) V for the newest token of every sequence.

    q [B, Hq, D] f16 or bf16; k_pages, v_pages [P, Hkv, S, D] of q's type or
    e4m3 (views of a cache are fine; the last dim is contiguous); tables int32
    [B, width] the pages of a sequence in order, lens int32 [B] its cached
    tokens, the new one among them.  Entries past a sequence's pages are not
    read.  Query head i reads kv head i // (Hq // Hkv).

    scale (default D ** -0.5) multiplies q . k; softcap c > 0 turns a score x
    into c tanh(x / c); slopes f32 [Hq] then add slope * (t - newest); window >
    0 keeps the newest `window` tokens; k_scale, v_scale f32 [Hkv] are what a
    stored value stands for.  Returns [B, Hq, D] of q's type, zeros for an
    empty sequence; with return_lse also the logarithm of the softmax's sum,
    f32 [B, Hq], -inf for an empty sequence.  It has no gradient.
    """
    _need_cuda(q, k_pages, v_pages, tables, lens, slopes, k_scale, v_scale)
    dt, ct = _CODE.get(q.dtype), _CODE.get(k_pages.dtype)
    if dt not in (1, 2) or ct not in (dt, 3) or v_pages.dtype != k_pages.dtype:
        raise ValueError("paged_decode takes f16 or bf16 queries and pages of that type or e4m3")
    if q.dim() != 3 or k_pages.dim() != 4 or v_pages.shape != k_pages.shape:
        raise ValueError("paged_decode: q [B, Hq, D], k_pages and v_pages [P, Hkv, S, D]")
    B, Hq, D = q.shape
    P, Hkv, S, Dk = k_pages.shape
    if Dk != D or D % 8 or not 0 < D <= 256:
        raise ValueError(f"paged_decode: heads of {D} and {Dk} (one multiple of 8, at most 256)")
    if Hkv == 0 or Hq % Hkv or S == 0:
        raise ValueError(f"paged_decode: {Hq} query heads over {Hkv} kv heads, {S} slots a page")
    if tables.dtype != torch.int32 or tables.dim() != 2 or tables.shape[0] != B:
        raise ValueError(f"paged_decode: tables must be int32 [{B}, width]")
    if lens.dtype != torch.int32 or lens.shape != (B,) or not lens.is_contiguous():
        raise ValueError(f"paged_decode: lens must be contiguous int32 [{B}]")
    qb, qh, qd = q.stride()
    kp, kh, ks, kd = k_pages.stride()
    vp, vh, vs, vd = v_pages.stride()
    tb, tw = tables.stride()
    width = tables.shape[1]
    if qd != 1 or kd != 1 or vd != 1 or (tw != 1 and width > 1):
        raise ValueError("paged_decode: the last dim of q, pages and tables must be contiguous")
    if window < 0 or not softcap >= 0:
        raise ValueError(f"paged_decode: window={window} softcap={softcap}")
    if out is None:
        out = _empty((B, Hq, D), q.dtype, q.device, stream)
    elif not out.is_cuda or out.shape != q.shape or out.dtype != q.dtype or not out.is_contiguous():
        raise ValueError(f"paged_decode: out must be a contiguous {q.dtype} {list(q.shape)}")
    lse = _empty((B, Hq), torch.float32, q.device, stream) if return_lse else None
    args = _ARGS.pack(q.data_ptr(), out.data_ptr(), lse.data_ptr() if return_lse else 0,
                      k_pages.data_ptr(), v_pages.data_ptr(), tables.data_ptr(), lens.data_ptr(),
                      _vector("slopes", slopes, Hq), _vector("k_scale", k_scale, Hkv),
                      _vector("v_scale", v_scale, Hkv), qb, qh, kp, kh, ks, vp, vh, vs, tb, B, Hq,
                      Hkv, D, S, P, width, min(int(window), 0x7fffffff), dt, ct,
                      D ** -0.5 if scale is None else scale, softcap)
    rc = lib.ubridge_paged_decode(args, stream_ptr(stream))
    if rc:
        check(rc)
    return [out, lse] if return_lse else out
