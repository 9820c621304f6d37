"""Attention over a paged key-value cache for decoding: one new token per
sequence, grouped heads, optional score cap, sliding window, bias by distance
and 8-bit pages."""
from .native import _native, call


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
    stored value stands for.  Returns [B, Hq, D] of q's type (in `out`, which
    overlaps no input, if it is given), zeros for an empty sequence; with return_lse also the logarithm of the softmax's sum,
    f32 [B, Hq], -inf for an empty sequence.  It has no gradient.
    """
    return call(_native.paged_decode, stream, q, k_pages, v_pages, tables, lens, scale, softcap, window,
                slopes, k_scale, v_scale, out, return_lse)
