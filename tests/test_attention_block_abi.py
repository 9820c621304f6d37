"""CPU checks of the attention block's C entries: each refuses what it cannot
take before it touches a device, and the argument blocks have the layout that
the header gives them."""
import copy
import math
import pickle
import struct

import pytest
import torch

from ubridge_amd import _lib, attention, int8, kvcache, rope

lib = _lib.lib
# UbridgeRopeArgs: 12 pointers, 7 strides, 12 ints, factor, padding;
# UbridgePagedDecodeArgs: 10 pointers, 9 strides, 10 ints, scale, softcap
ROPE_ARGS, DECODE_ARGS = struct.Struct("@12P7q12ifi"), struct.Struct("@10P9q10i2f")
P = 256  # a pointer that is never followed


def refused(rc, code, text):
    assert rc == code and text in lib.ubridge_last_error_string(), lib.ubridge_last_error_string()
    assert lib.ubridge_last_error() == code


def test_int8_linear():
    def call(x=P, dt=2, w=P, sw=P, b=0, y=P, M=1, K=100, N=8, ld=128):
        return lib.ubridge_int8_linear(x, dt, w, sw, b, y, M, K, N, ld, None)
    refused(call(dt=3), 1, b"dtype 3")
    refused(call(M=-1), 1, b"M=-1")
    refused(call(K=0), 1, b"K=0")
    refused(call(K=132105, ld=132224), 1, b"K=132105")
    refused(call(ld=100), 1, b"ld=100")
    refused(call(K=200), 1, b"ld=128")
    for a in ("x", "w", "sw", "y"):
        refused(call(**{a: 0}), 1, b"null pointer")
    refused(call(w=P + 1), 1, b"not 16-byte aligned")
    assert call(M=0) == 0 and call(N=0) == 0


ROPE = dict(q=P, k=P, v=P, qo=P, ko=P, pos=P, turns=P, kp=P, vp=P, slots=P, ks=0, vs=0, s0=0, s1=0, s2=0, s3=0,
            s4=0, s5=0, ps=0, T=1, Hq=1, Hkv=1, D=64, rot=64, inter=0, inv=0, p64=1, dt=2, ct=2, pages=1, S=1,
            factor=1.0, pad=0)


@pytest.mark.parametrize("name", ["ubridge_rope", "ubridge_rope_append"])
def test_rope(name):
    fn = getattr(lib, name)
    call = lambda **kw: fn(ROPE_ARGS.pack(*dict(ROPE, **kw).values()), None)
    refused(fn(None, None), 1, b"null argument block")
    refused(call(dt=5), 1, b"dtype 5")
    refused(call(T=-1), 1, b"T=-1")
    refused(call(D=0), 1, b"D=0")
    refused(call(D=5000), 1, b"D=5000")
    refused(call(rot=63), 1, b"rot=63")
    refused(call(rot=66), 1, b"rot=66")
    refused(call(pos=0), 1, b"null positions")
    refused(call(turns=0), 1, b"null positions")
    refused(call(q=0), 1, b"null q or k")
    refused(call(qo=0), 1, b"null q or k")
    refused(call(k=0), 1, b"null q or k")
    assert call(T=0) == 0
    if name == "ubridge_rope":
        refused(call(ko=0), 1, b"null k_out")
    else:
        refused(call(ct=1), 1, b"cache type 1")
        refused(call(S=0), 1, b"S=0")
        refused(call(slots=0), 1, b"S=1")
        refused(call(v=0), 1, b"null v or pages")
        refused(call(kp=0), 1, b"null v or pages")


DECODE = dict(q=P, out=P, lse=0, kp=P, vp=P, tables=P, lens=P, slopes=0, ks=0, vs=0, s0=0, s1=0, s2=0, s3=0, s4=0,
              s5=0, s6=0, s7=0, ts=0, B=1, Hq=8, Hkv=2, D=64, S=16, P=4, width=4, window=0, dt=2, ct=2, scale=1.0,
              cap=0.0)


def test_paged_decode():
    call = lambda **kw: lib.ubridge_paged_decode(DECODE_ARGS.pack(*dict(DECODE, **kw).values()), None)
    refused(lib.ubridge_paged_decode(None, None), 1, b"null argument block")
    refused(call(dt=0), 1, b"dtype 0")
    refused(call(ct=1), 1, b"cache type 1")
    refused(call(Hq=7), 1, b"Hq=7")
    refused(call(Hkv=0), 1, b"Hkv=0")
    refused(call(D=68), 1, b"D=68")
    refused(call(D=264), 1, b"D=264")
    refused(call(S=0), 1, b"S=0")
    refused(call(width=1 << 28), 1, b"width=268435456")
    refused(call(window=-1), 1, b"window=-1")
    refused(call(cap=-1.0), 1, b"softcap=-1")
    refused(call(cap=float("nan")), 1, b"softcap")
    refused(call(B=1 << 21), 1, b"B=2097152")
    for a in ("q", "out", "lens", "tables"):
        refused(call(**{a: 0}), 1, b"null pointer")
    refused(call(kp=0), 1, b"null pages")
    assert call(B=0) == 0 and call(Hq=0) == 0


def test_kv_pool():
    base = dict(kv=P, refs=P, lens=P, tables=P, page=64, L=1, P=4, S=4, rows=2, width=2, pad=0)
    pack = lambda **kw: struct.pack("@4Pq6i", *dict(base, **kw).values())
    free = lambda p, r=P, n=1: lib.ubridge_kv_free(p, r, n, None)
    fork = lambda p, s=P, d=P, n=1, o=P: lib.ubridge_kv_fork(p, s, d, n, o, None)
    compact = lambda p, o=P: lib.ubridge_kv_compact(p, o, None)
    for fn in (free, fork, compact):
        refused(fn(None), 1, b"null pool")
        for bad in (dict(L=0), dict(P=-1), dict(S=0), dict(rows=-1), dict(width=-1), dict(page=0)):
            refused(fn(pack(**bad)), 1, b"page_bytes=")
        refused(fn(pack(kv=0)), 1, b"null pages")
        refused(fn(pack(refs=0)), 1, b"null pages")
        refused(fn(pack(lens=0)), 1, b"null lengths")
        refused(fn(pack(tables=0)), 1, b"null lengths")
    refused(free(pack(), n=-1), 1, b"n=-1")
    refused(free(pack(), r=0), 1, b"null rows")
    refused(fork(pack(), n=65536), 1, b"n=65536")
    refused(fork(pack(), d=0), 1, b"null rows")
    refused(fork(pack(), o=0), 1, b"null rows")
    refused(compact(pack(), o=0), 1, b"null count")
    assert free(pack(), n=0) == 0 and fork(pack(), n=0) == 0


def test_host_tensors_are_refused():
    x = torch.zeros(2, 1, 8)
    with pytest.raises(ValueError):
        int8.Linear(torch.zeros(2, 8, dtype=torch.int8), torch.ones(2))
    with pytest.raises(ValueError):
        rope.Rope(8, device="cpu")(x, x, torch.arange(2))
    with pytest.raises(ValueError):
        attention.paged_decode(x.half(), x.half()[None], x.half()[None], torch.zeros(2, 1).int(), torch.zeros(2).int())
    with pytest.raises(ValueError):
        kvcache.PagedCache(torch.zeros(1, 2, 2, 1, 4, 8).half(), 1, 1)


def test_frequencies():
    # closed forms at the ends of each scaling
    f, a = rope.frequencies(128, 10000.0)
    assert f[0] == 1.0 and abs(f[-1] - 10000.0 ** (-126 / 128)) < 1e-18 and a == 1.0
    f, _ = rope.frequencies(128, 10000.0, dict(kind="linear", factor=4.0))
    assert f[0] == 0.25
    f, _ = rope.frequencies(128, 10000.0, dict(kind="ntk", factor=4.0))
    assert f[0] == 1.0 and abs(f[-1] * 10000.0 ** (126 / 128) - 0.25) < 1e-12  # the slowest pair by factor
    f, a = rope.frequencies(128, 10000.0, dict(kind="yarn", factor=8.0, original=4096))
    assert f[0] == 1.0 and abs(f[-1] * 10000.0 ** (126 / 128) - 1 / 8) < 1e-12
    assert a == 0.1 * math.log(8.0) + 1.0
    f, _ = rope.frequencies(128, 10000.0, dict(kind="bands", factor=8.0, low=1.0, high=4.0, original=4096))
    assert f[0] == 1.0 and abs(f[-1] * 10000.0 ** (126 / 128) - 1 / 8) < 1e-12
    for bad in (dict(kind="other"), dict(kind="linear"), dict(kind="linear", factor=0.0),
                dict(kind="yarn", factor=2.0), dict(kind="ntk", factor=2.0, original=5)):
        with pytest.raises(ValueError):
            rope.frequencies(64, 10000.0, bad)


@pytest.mark.parametrize("how", ["deepcopy", "pickle"])
def test_a_copied_cache_works_on_its_own_memory(monkeypatch, how):
    # what its page operations hand over: the copy's tensors, no address of the original's
    monkeypatch.setattr(kvcache, "_need_cuda", lambda *t: None)
    handed = []
    monkeypatch.setattr(kvcache, "call", lambda fn, stream, *args: handed.extend(args))
    c = kvcache.PagedCache(torch.zeros(1, 2, 4, 1, 4, 8).half(), 3, 2)
    other = copy.deepcopy(c) if how == "deepcopy" else pickle.loads(pickle.dumps(c))
    theirs = {c.kv.data_ptr(), c.meta.data_ptr(), c.lens.data_ptr(), c.tables.data_ptr()}
    rows = torch.zeros(1, dtype=torch.int32)
    for run in (lambda: other.free(rows), lambda: other.fork(rows, rows), other.compact):
        del handed[:]
        run()
        at = {t.data_ptr() for t in handed if isinstance(t, torch.Tensor)}
        for b in handed:
            if isinstance(b, bytes):
                at.update(struct.unpack(f"@{len(b) // 8}P", b[:len(b) // 8 * 8]))
        assert not at & theirs and {other.kv.data_ptr(), other.meta.data_ptr()} <= at
    other.refs[1], other.lens[2], other.tables[2, 1] = 5, 6, 7
    assert other.meta.tolist() == [0, 5, 0, 0, 0, 0, 6] + [-1] * 5 + [7]
    assert c.meta.tolist() == [0] * 7 + [-1] * 6
    assert (c.P, c.rows, c.width) == (other.P, other.rows, other.width)


def test_operators_without_a_gradient_say_so():
    for what in (attention.paged_decode, kvcache.PagedCache.append, kvcache.PagedCache.attend, int8):
        assert "no gradient" in " ".join(what.__doc__.split()), what


def test_paged_decode_refuses_an_infinite_cap():
    # c tanh(x / c) has no value there (it came out as NaN everywhere); 0 is no cap
    call = lambda **kw: lib.ubridge_paged_decode(DECODE_ARGS.pack(*dict(DECODE, **kw).values()), None)
    refused(call(cap=float("inf")), 1, b"softcap")
    refused(call(cap=1e-39), 1, b"softcap")
