"""Kernels that ask for more than 64 KiB of dynamic LDS have their limit raised on
every device that they are launched on: the attention block's launches, with the
HIP runtime's calls that they make answered by a stand-in for two devices (nothing
is run, no pointer is followed)."""
import os
import struct
import subprocess
import sys

import pytest

from conftest import ROOT

STAND_IN = r"""
#include <cstddef>
#include <cstdio>
#include <map>
#include <utility>
struct dim3 { unsigned x, y, z; };
static int device;
static std::map<std::pair<int, const void*>, int> limit;
static std::map<const void*, int> number;
static struct { dim3 g, b; size_t lds; void* s; } cfg;
static char memory[64];
extern "C" {
void stand_in_device(int d) { device = d; }
int hipGetDevice(int* d) { *d = device; return 0; }
int hipFuncSetAttribute(const void* f, int, int bytes) { limit[{device, f}] = bytes; return 0; }
int hipGetSymbolAddress(void** p, const void*) { *p = memory; return 0; }
int hipMalloc(void** p, size_t) { *p = memory; return 0; }
int hipStreamIsCapturing(void*, int* st) { *st = 0; return 0; }
int hipThreadExchangeStreamCaptureMode(int*) { return 0; }
int hipGetLastError() { return 0; }
int __hipPushCallConfiguration(dim3 g, dim3 b, size_t lds, void* s) { cfg = {g, b, lds, s}; return 0; }
int __hipPopCallConfiguration(dim3* g, dim3* b, size_t* lds, void** s) {
  *g = cfg.g, *b = cfg.b, *lds = cfg.lds, *s = cfg.s;
  return 0;
}
int hipLaunchKernel(const void* f, dim3, dim3, void**, size_t lds, void*) {
  const int n = number.emplace(f, (int)number.size()).first->second;
  const auto at = limit.find({device, f});
  printf("device %d kernel %d lds %zu limit %d\n", device, n, lds, at == limit.end() ? 65536 : at->second);
  fflush(stdout);
  return 0;
}
}
"""

RUN = r"""
import ctypes, struct, sys
shim = ctypes.CDLL(sys.argv[1], ctypes.RTLD_GLOBAL)
lib = ctypes.CDLL(sys.argv[2])
P = ctypes.c_void_p(4096)
decode = struct.Struct("@10P9q10i2f")
for device in (0, 1, 0):
    shim.stand_in_device(device)
    for dt in range(3):
        for M, K, N in ((16, 4096, 4096), (8, 8192, 512), (64, 4096, 512), (201, 3520, 9001), (512, 2048, 1024),
                        (1024, 2048, 2048), (4096, 4096, 14336), (40, 16384, 450)):
            ld = (K + 127) // 128 * 128
            rc = lib.ubridge_int8_linear(P, dt, P, P, None, P, M, K, N, ld, None)
            assert rc == 0, (M, K, N, rc)
    for dt in (1, 2):
        for G, D in ((32, 64), (16, 128), (32, 128), (16, 256), (32, 256)):
            a = decode.pack(*[4096] * 2, 0, *[4096] * 4, 0, 0, 0, *[0] * 9, 1, G, 1, D, 16, 4, 4, 0, dt, dt, 1.0, 0.0)
            assert lib.ubridge_paged_decode(a, None) == 0
"""


def test_lds_limits_of_two_devices(tmp_path):
    src, shim = tmp_path / "stand_in.cpp", tmp_path / "stand_in.so"
    src.write_text(STAND_IN)
    subprocess.run(["g++", "-O1", "-shared", "-fPIC", "-std=c++17", "-o", str(shim), str(src)], check=True)
    lib = os.path.join(ROOT, "ubridge_amd", "lib", "libubridge_hip.so")
    r = subprocess.run([sys.executable, "-c", RUN, str(shim), lib], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stderr
    lines = [[int(x) for x in line.split()[1::2]] for line in r.stdout.splitlines()]
    for device, kernel, lds, limit in lines:
        assert lds <= limit <= 160 * 1024, (device, kernel, lds, limit)
    big = [{k for d, k, lds, _ in lines if d == device and lds > 65536} for device in (0, 1)]
    # two forms for few tokens and two tiles of three types, five forms of attention of two
    assert big[0] == big[1] and len(big[0]) == 3 * 4 + 2 * 5
