"""CPU checks of the norm's and the feed-forward half's C entries: each refuses what
it cannot take before it touches a device, and the argument blocks have the layout
that the header gives them."""
import os
import struct
import subprocess
import sys

import pytest

import ubridge_amd
from conftest import ROOT
from test_launch_limits import STAND_IN
from ubridge_amd import int8, mx, norm  # noqa: F401  (they register the entries)

lib = ubridge_amd._lib.lib
P = 256  # a pointer that is never followed
# UbridgeRmsNormArgs: 6 pointers, eps, 6 ints; ...GradArgs: 6 pointers, eps, 4 ints;
# UbridgeMxLinearArgs: 7 pointers, 6 ints; UbridgeMoeDecodeArgs: 7 pointers, 8 ints
NORM, GRAD, MX, MOE = struct.Struct("@6Pd6i"), struct.Struct("@6Pd4i"), struct.Struct("@7P6i"), struct.Struct("@7P8i")


def refused(rc, code, text):
    assert rc == code and text in lib.ubridge_last_error_string(), lib.ubridge_last_error_string()
    assert lib.ubridge_last_error() == code


def caller(name, block, defaults):
    return lambda **kw: getattr(lib, name)(block.pack(*dict(defaults, **kw).values()), None)


def test_rms_norm():
    call = caller("ubridge_rms_norm", NORM, dict(x=P, res=0, w=P, h=0, y=P, scale=0, eps=1e-6, R=1, C=64, dt=2, wt=2,
                                                 out=0, pad=0))
    refused(lib.ubridge_rms_norm(None, None), 1, b"null argument block")
    refused(call(dt=3, wt=3), 1, b"dtype 3")
    refused(call(wt=1), 1, b"gain of type 1")
    refused(call(out=5), 1, b"out 5")
    refused(call(out=-1), 1, b"out -1")
    refused(call(R=-1), 1, b"R=-1")
    refused(call(R=1 << 22), 1, b"R=4194304")
    refused(call(C=0), 1, b"C=0")
    refused(call(C=32769), 1, b"C=32769")
    refused(call(C=16385, dt=0, wt=0), 1, b"C=16385")
    refused(call(eps=-1.0), 1, b"eps")
    refused(call(eps=float("nan")), 1, b"eps")
    for a in ("x", "w", "y"):
        refused(call(**{a: 0}), 1, b"null pointer")
    refused(call(res=P), 1, b"null pointer")  # and no place for the sum
    refused(call(out=1), 1, b"null pointer")  # and no place for the scales
    refused(call(out=3, scale=P, y=P + 8), 1, b"not 16-byte aligned")
    assert call(R=0) == 0


def test_rms_norm_grad():
    call = caller("ubridge_rms_norm_grad", GRAD, dict(h=P, w=P, dy=P, dh=0, dx=P, dw=0, eps=1e-6, R=1, C=64, dt=2, wt=0))
    refused(lib.ubridge_rms_norm_grad(None, None), 1, b"null argument block")
    refused(call(dt=5), 1, b"dtype 5")
    refused(call(wt=1), 1, b"gain of type 1")
    refused(call(C=0), 1, b"C=0")
    refused(call(C=40000), 1, b"C=40000")
    refused(call(eps=-1.0), 1, b"eps")
    for a in ("h", "w", "dy", "dx"):
        refused(call(**{a: 0}), 1, b"null pointer")
    assert call(R=0, h=0, dy=0) == 0


@pytest.mark.parametrize("name", ["ubridge_mx_quantize", "ubridge_mx_dequantize"])
def test_blocks(name):
    def call(x=P, dt=2, q=P, s=P, R=1, C=64, f=4):
        fn = getattr(lib, name)
        return fn(x, dt, q, s, R, C, f, None) if name == "ubridge_mx_quantize" else fn(q, s, x, dt, R, C, f, None)
    refused(call(dt=3), 1, b"dtype 3")
    refused(call(f=6), 1, b"format 6")
    refused(call(R=-1), 1, b"R=-1")
    refused(call(C=0), 1, b"C=0")
    refused(call(R=1 << 20, C=1 << 20), 1, b"R=1048576")
    for a in ("x", "q", "s"):
        refused(call(**{a: 0}), 1, b"null pointer")
    refused(call(q=P + 4), 1, b"not 16-byte aligned")
    assert call(R=0) == 0


def test_mx_pack():
    call = lambda q=P, s=P, w=P, ws=P, N=8, K=64: lib.ubridge_mx_pack(q, s, w, ws, N, K, None)
    refused(call(N=-1), 1, b"N=-1")
    refused(call(K=0), 1, b"K=0")
    refused(call(K=131073), 1, b"K=131073")
    refused(call(N=1 << 30, K=131072), 1, b"N=1073741824")
    for a in ("q", "s", "w", "ws"):
        refused(call(**{a: 0}), 1, b"null pointer")
    refused(call(w=P + 8), 1, b"not 16-byte aligned")
    assert call(N=0) == 0


def test_mx_linear():
    call = caller("ubridge_mx_linear", MX, dict(x=P, q=0, s=0, w=P, ws=P, bias=0, y=P, M=1, K=64, N=8, dt=2, f=4, pad=0))
    refused(lib.ubridge_mx_linear(None, None), 1, b"null argument block")
    refused(call(dt=3), 1, b"dtype 3")
    refused(call(f=5), 1, b"format 5")
    refused(call(M=-1), 1, b"M=-1")
    refused(call(K=0), 1, b"K=0")
    refused(call(K=131073), 1, b"K=131073")
    for a in ("x", "w", "ws", "y"):
        refused(call(**{a: 0}), 1, b"null pointer")
    refused(call(x=0, q=P), 1, b"null pointer")
    refused(call(x=0, q=P + 8, s=P), 1, b"codes not 16-byte")
    refused(call(x=0, q=P, s=P + 2), 1, b"scales not 4-byte")
    refused(call(w=P + 8), 1, b"weight not 16-byte aligned")
    refused(call(M=1 << 22), 1, b"M=4194304")
    refused(call(M=1 << 21, N=1 << 20), 1, b"N=1048576")
    refused(call(M=1 << 20, K=131072), 1, b"K=131072")
    assert call(M=0) == 0 and call(N=0) == 0


def test_int8_linear_codes():
    def call(a=P, sa=P, w=P, sw=P, b=0, y=P, dt=2, M=1, K=100, N=8, ld=128):
        return lib.ubridge_int8_linear_codes(a, sa, w, sw, b, y, dt, M, K, N, ld, None)
    refused(call(dt=3), 1, b"dtype 3")
    refused(call(K=0), 1, b"K=0")
    refused(call(K=200), 1, b"ld=128")
    refused(call(ld=100), 1, b"ld=100")
    for a in ("a", "sa", "w", "sw", "y"):
        refused(call(**{a: 0}), 1, b"null pointer")
    refused(call(a=P + 8), 1, b"not 16-byte aligned")
    refused(call(w=P + 8), 1, b"not 16-byte aligned")
    refused(call(M=1 << 22), 1, b"M=4194304")
    assert call(M=0) == 0 and call(N=0) == 0


def test_moe_decode():
    call = caller("ubridge_moe_decode", MOE, dict(x=P, lg=P, w13=P, s13=0, w2=P, s2=0, y=P, T=1, E=8, k=2, H=64, I=32, dt=2,
                                                  lt=0, norm=1))
    refused(lib.ubridge_moe_decode(None, None), 1, b"null argument block")
    refused(call(dt=0), 1, b"dtype 0")
    refused(call(lt=3), 1, b"logits of type 3")
    refused(call(T=17), 1, b"T=17")
    refused(call(T=-1), 1, b"T=-1")
    refused(call(E=1025), 1, b"E=1025")
    refused(call(k=0), 1, b"k=0")
    refused(call(k=9), 1, b"k=9")
    refused(call(E=64, k=17), 1, b"k=17")
    refused(call(H=48), 1, b"H=48")
    refused(call(I=0), 1, b"I=0")
    refused(call(I=40), 1, b"I=40")
    for a in ("x", "lg", "w13", "w2", "y"):
        refused(call(**{a: 0}), 1, b"null pointer")
    refused(call(s13=P), 1, b"one of two scales")
    refused(call(w2=P + 8), 1, b"not 16-byte aligned")
    assert call(T=0) == 0


LIMITS = r"""
import ctypes, struct, sys
shim = ctypes.CDLL(sys.argv[1], ctypes.RTLD_GLOBAL)
lib = ctypes.CDLL(sys.argv[2])
mx = struct.Struct("@7P6i")
for device in (0, 1, 0):
    shim.stand_in_device(device)
    for f in (4, 8):
        for dt in range(3):
            for M, K, N, pre in ((1, 14336, 4096, 0), (16, 8192, 512, 0), (16, 8192, 512, 1), (16, 14336, 64, 0),
                                 (40, 4096, 4096, 0), (64, 16384, 450, 1), (201, 3520, 9001, 0), (1024, 2048, 2048, 0),
                                 (4096, 4096, 14336, 0)):
                a = mx.pack(0 if pre else 4096, *[4096] * 4, 0, 4096, M, K, N, dt, f, 0)
                rc = lib.ubridge_mx_linear(a, None)
                assert rc == 0, (f, dt, M, K, N, rc)
"""


def test_lds_limits_of_two_devices(tmp_path):
    # (the HIP runtime's calls answered by a stand-in: nothing is run)
    src, shim = tmp_path / "stand_in.cpp", tmp_path / "stand_in.so"
    src.write_text(STAND_IN)
    subprocess.run(["g++", "-O1", "-shared", "-fPIC", "-std=c++17", "-o", str(shim), str(src)], check=True)
    lib = os.path.join(ROOT, "ubridge_amd", "lib", "libubridge_hip.so")
    r = subprocess.run([sys.executable, "-c", LIMITS, str(shim), lib], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stderr
    lines = [[int(x) for x in line.split()[1::2]] for line in r.stdout.splitlines()]
    for device, kernel, lds, limit in lines:
        assert lds <= limit <= 160 * 1024, (device, kernel, lds, limit)
    big = [{k for d, k, lds, _ in lines if d == device and lds > 65536} for device in (0, 1)]
    assert big[0] == big[1] and len(big[0]) >= 2 * 3 * 2  # few tokens, and the largest tiles, of each type
