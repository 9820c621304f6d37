"""The library's scratch.  Calls of two threads on one stream: the launches of a call that
takes scratch lie together, so that no other call's use of the stream's buffer, and no
growth of it, falls between them.  A call's several pieces.  Buffers of captured
graphs.  The HIP runtime's calls are answered by a stand-in: nothing is run."""
import itertools
import os
import subprocess
import sys

import pytest

from conftest import ROOT

STAND_IN = r"""
#include <cstddef>
#include <cstdio>
#include <cstdlib>
#include <unistd.h>
#include <sys/syscall.h>
struct dim3 { unsigned x, y, z; };
static thread_local struct { dim3 g, b; size_t lds; void* s; } cfg;
static void say(const char* what, const void* p) {
  char line[96];
  const int n = snprintf(line, sizeof line, "%ld %s %p\n", (long)syscall(SYS_gettid), what, p);
  if (write(1, line, n) != n) abort();
}
extern "C" {
int hipGetDevice(int* d) { *d = 0; return 0; }
int hipFuncSetAttribute(const void*, int, int) { return 0; }
int hipMalloc(void** p, size_t n) { *p = malloc(64); say("alloc", *p); return 0; }
int hipFree(void* p) { say("free", p); return 0; }
int hipEventCreateWithFlags(void** e, unsigned) { *e = (void*)1; return 0; }
int hipEventRecord(void*, void*) { return 0; }
int hipEventQuery(void*) { return 0; }
int hipEventDestroy(void*) { return 0; }
int hipStreamSynchronize(void*) { say("synchronize", 0); usleep(500); return 0; }
static int status;
static unsigned long long capture;
static int graphs[64];                                    // a graph is the address of one
static struct { void (*end)(void*); void* p; } kept[64];  // by graph
static void* object[2];
void stand_in_capture(int on) { status = on; capture += on; }
void stand_in_destroy(int graph) { if (kept[graph].end) kept[graph].end(kept[graph].p); }
int hipStreamIsCapturing(void*, int* st) { *st = status; return 0; }
int hipStreamGetCaptureInfo(void*, int* st, unsigned long long* id) { *st = status, *id = capture; return 0; }
int hipStreamGetCaptureInfo_v2(void*, int* st, unsigned long long* id, void** graph, const void** deps, size_t* n) {
  *st = status, *id = capture, *deps = 0, *n = 0;
  *graph = &graphs[capture];
  return 0;
}
int hipUserObjectCreate(void** o, void* p, void (*end)(void*), unsigned, unsigned) {
  object[0] = (void*)end, object[1] = p;
  *o = object;
  return 0;
}
int hipGraphRetainUserObject(void* g, void*, unsigned, unsigned) {
  kept[(int*)g - graphs] = {(void (*)(void*))object[0], object[1]};
  return 0;
}
int hipUserObjectRelease(void*, unsigned) { return 0; }
int hipThreadExchangeStreamCaptureMode(int*) { return 0; }
int hipGetLastError() { return 0; }
int hipblasLtCreate(void**) { return 1; }  // (no library products)
int __hipPushCallConfiguration(dim3 g, dim3 b, size_t lds, void* s) { cfg = {g, b, lds, s}; return 0; }
int __hipPopCallConfiguration(dim3* g, dim3* b, size_t* lds, void** s) {
  *g = cfg.g, *b = cfg.b, *lds = cfg.lds, *s = cfg.s;
  return 0;
}
int hipLaunchKernel(const void* f, dim3, dim3, void**, size_t, void*) {
  say("launch", 0);
  usleep(300);  // the other thread's turn, if it may
  return 0;
}
}
"""

RUN = r"""
import ctypes, struct, sys, threading
shim = ctypes.CDLL(sys.argv[1], ctypes.RTLD_GLOBAL)
lib = ctypes.CDLL(sys.argv[2])
mx, moe, grad = struct.Struct("@7P6i"), struct.Struct("@7P8i"), struct.Struct("@6Pd4i")
P, V = 4096, ctypes.c_void_p(4096)

def linear(M, K, N):
    return lambda: lib.ubridge_mx_linear(mx.pack(P, 0, 0, P, P, 0, P, M, K, N, 2, 4, 0), None)
def decode():
    return lib.ubridge_moe_decode(moe.pack(P, P, P, 0, P, 0, P, 16, 64, 8, 2048, 768, 2, 0, 1), None)
def norm_grad(C):
    return lambda: lib.ubridge_rms_norm_grad(grad.pack(P, P, P, 0, P, P, 1e-6, 4096, C, 2, 2), None)
def int8(M, K, N):
    return lambda: lib.ubridge_int8_linear(V, 2, V, V, None, V, M, K, N, K, None)
def release():
    return lib.ubridge_release_workspace(None)

calls = {"mx": linear(40, 4096, 512), "mx larger": linear(2000, 8192, 512), "mx parts": linear(40, 13952, 512),
         "decode": decode, "norm": norm_grad(4096), "norm larger": norm_grad(16384), "int8": int8(64, 4096, 512),
         "release": release}
mine = [calls[n] for n in sys.argv[3].split(",")], [calls[n] for n in sys.argv[4].split(",")]
def run(fs, n):
    for _ in range(n):
        for f in fs:
            assert f() == 0
for fs in mine:  # alone: what each call does
    for f in fs:
        print("call", flush=True)
        assert f() == 0
print("call", flush=True)
print("both", flush=True)
ts = [threading.Thread(target=run, args=(fs, 6)) for fs in mine]
for t in ts: t.start()
for t in ts: t.join()
"""


@pytest.fixture(scope="module")
def shim(tmp_path_factory):
    d = tmp_path_factory.mktemp("stand_in")
    src, so = d / "stand_in.cpp", d / "stand_in.so"
    src.write_text(STAND_IN)
    subprocess.run(["g++", "-O1", "-shared", "-fPIC", "-std=c++17", "-o", str(so), str(src)], check=True)
    return str(so)


@pytest.mark.parametrize("one,other", [("mx", "mx"), ("mx", "mx larger"), ("mx,mx larger", "mx parts"), ("decode", "norm"),
                                       ("norm", "norm larger"), ("decode,mx", "int8"), ("mx", "release"), ("norm,decode", "release")])
def test_a_call_s_launches_lie_together(shim, one, other):
    lib = os.path.join(ROOT, "ubridge_amd", "lib", "libubridge_hip.so")
    r = subprocess.run([sys.executable, "-c", RUN, shim, lib, one, other], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stderr
    alone, both = r.stdout.split("both\n")
    # launches of each thread's calls in turn
    names = one.split(",") + other.split(",")
    counts = [part.count("launch") for part in alone.split("call\n")[1:-1]]
    assert len(counts) == len(names) and all(c >= 2 for n, c in zip(names, counts) if n != "release")
    per = [counts[:len(one.split(","))], counts[len(one.split(",")):]]
    lines = [line.split() for line in both.splitlines()]
    threads = list(dict.fromkeys(t for t, *_ in lines))
    assert len(threads) == 2
    # which thread is which: by the number of its launches, or either way round if equal
    total = {t: sum(1 for a, what, _ in lines if a == t and what == "launch") for t in threads}

    def fits(order):
        if [total[t] for t in order] != [6 * sum(p) for p in per]:
            return False
        left = {t: itertools.cycle([c for c in p if c]) if any(p) else None for t, p in zip(order, per)}
        inside, n = None, 0  # the call going on, and its launches still to come
        for t, what, _ in lines:
            if inside is not None and t != inside:
                return False  # another thread's launch, allocation or release between two launches
            if what != "launch":
                continue
            if inside is None:
                inside, n = t, next(left[t])
            n -= 1
            if n == 0:
                inside = None
        return True
    assert fits(threads) or fits(threads[::-1]), both


LEVELS = r"""
import ctypes, sys
shim = ctypes.CDLL(sys.argv[1], ctypes.RTLD_GLOBAL)
lib = ctypes.CDLL(sys.argv[2])
V, odd = ctypes.c_void_p(4096), ctypes.c_void_p(4098)
for a in (V, odd):  # 72 x 4096 x 1544: parts of K
    print("call", flush=True)
    assert lib.ubridge_tune_set(b"w4a16_path", 3) == 0  # (not through the library product)
    assert lib.ubridge_w4a16_gemm(a, V, V, V, V, 72, 4096, 1544, 128, 2, None) == 0
"""


def test_two_pieces_of_one_call(shim):
    # an aligned call takes one buffer; the misaligned one a second, beside it
    lib = os.path.join(ROOT, "ubridge_amd", "lib", "libubridge_hip.so")
    r = subprocess.run([sys.executable, "-c", LEVELS, shim, lib], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stderr
    aligned, odd = [[line.split()[1] for line in part.splitlines()] for part in r.stdout.split("call\n")[1:]]
    assert aligned.count("alloc") == 1 and odd.count("alloc") == 1, r.stdout
    assert "free" not in aligned + odd and odd.count("launch") == aligned.count("launch") + 1, r.stdout


GRAPHS = r"""
import ctypes, struct, sys
shim = ctypes.CDLL(sys.argv[1], ctypes.RTLD_GLOBAL)
lib = ctypes.CDLL(sys.argv[2])
mx = struct.Struct("@7P6i")
P = 4096
def linear(M, K, N):
    assert lib.ubridge_mx_linear(mx.pack(P, 0, 0, P, P, 0, P, M, K, N, 2, 4, 0), None) == 0
def live():
    n, b, c = ctypes.c_size_t(), ctypes.c_size_t(), ctypes.c_long()
    assert lib.ubridge_workspace_stats(ctypes.byref(n), ctypes.byref(b), ctypes.byref(c)) == 0
    return n.value
def capture(M):
    shim.stand_in_capture(1)
    linear(M, 4096, 512)
    linear(M, 2048, 512)
    shim.stand_in_capture(0)
linear(40, 4096, 512)
assert live() == 1
for graph in range(1, 11):  # captured and destroyed in turn: one buffer serves all
    capture(200 if graph % 2 else 40)
    assert live() == 2, (graph, live())
    shim.stand_in_destroy(graph)
capture(40)  # graph 11 lives on
capture(40)  # 12 has its own beside it
assert live() == 3
shim.stand_in_destroy(12)
linear(40, 4096, 512)  # an eager call gives the ended one's back, and no other
assert live() == 2
capture(4000)  # 13: larger than what there is
assert live() == 3
assert lib.ubridge_release_workspace(None) == 0 and live() == 0
shim.stand_in_destroy(11)  # (graphs that end after the release)
shim.stand_in_destroy(13)
linear(40, 4096, 512)
assert live() == 1
"""


def test_buffers_of_ended_graphs_serve_others(shim):
    lib = os.path.join(ROOT, "ubridge_amd", "lib", "libubridge_hip.so")
    r = subprocess.run([sys.executable, "-c", GRAPHS, shim, lib], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stderr
