// runtime.cpp -- sticky error state and library identity for libubridge_hip.
#include <hip/hip_runtime.h>
#include <stdarg.h>
#include <stdio.h>
#include <stdlib.h>
#include <string.h>

#include <atomic>

#include "common.h"

namespace {
thread_local int g_err = UB_OK;
thread_local char g_msg[512] = {0};
}  // namespace

int ub_set_error(int code, const char* fmt, ...) {
  g_err = code;
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(g_msg, sizeof(g_msg), fmt, ap);
  va_end(ap);
  return code;
}

int ub_check_launch(const char* what) {
  hipError_t e = hipGetLastError();
  if (e != hipSuccess)
    return ub_set_error(UB_ERR_LAUNCH, "%s: launch failed: %s", what, hipGetErrorString(e));
  return UB_OK;
}

UB_API int ubridge_last_error(void) {
  int e = g_err;
  g_err = UB_OK;
  return e;
}

UB_API const char* ubridge_last_error_string(void) { return g_msg; }

UB_API const char* ubridge_version(void) { return "ubridge_amd 0.1 gfx950"; }

// ------------------------------------------------------- launch-shape knobs
// The reference picks GEMM tilings on the host from the problem shape
// (gemm_tuner.rs:326-600, GEMM_OP_PARAS :222-258, cached per shape).  Here
// each launcher applies its own shape rule; these knobs override a rule
// process-wide (0 = automatic), for tuning sweeps and for callers that
// know better.  Initial values come from the environment.
namespace {
struct Knob {
  const char* name;
  const char* env;
};
constexpr Knob kKnobs[UB_TUNE_COUNT] = {
    {"gemv_lds_rows", "UBRIDGE_GEMV_LDS"}, {"gemv_lds_waves", "UBRIDGE_GEMV_W"},
    {"gemv_rows", "UBRIDGE_GEMV_R"},       {"gemv_iters", "UBRIDGE_GEMV_U"},
    {"gemm_tile", "UBRIDGE_GEMM_TILE"},    {"gemv_mfma_m", "UBRIDGE_GEMV_MFMA_M"},
    {"w4a16_path", "UBRIDGE_W4A16_PATH"},    {"moe_gemm_path", "UBRIDGE_MOE_GEMM_PATH"},
    {"gemv_mm", "UBRIDGE_GEMV_MM"},        {"gemv_persist", "UBRIDGE_GEMV_PERSIST"},
    {"gemv_q80_lds", "UBRIDGE_GEMV_Q80_LDS"}, {"gemv_fuse_m", "UBRIDGE_GEMV_FUSE_M"},
};
std::atomic<int> g_knob[UB_TUNE_COUNT];
std::atomic<bool> g_knob_init[UB_TUNE_COUNT];

int knob_index(const char* name) {
  if (!name) return -1;
  for (int i = 0; i < UB_TUNE_COUNT; i++)
    if (strcmp(name, kKnobs[i].name) == 0) return i;
  return -1;
}
}  // namespace

int ub_tune(int k) {
  if (!g_knob_init[k].load(std::memory_order_acquire)) {
    const char* v = getenv(kKnobs[k].env);
    int expected = 0;
    g_knob[k].compare_exchange_strong(expected, v ? atoi(v) : 0);
    g_knob_init[k].store(true, std::memory_order_release);
  }
  return g_knob[k].load(std::memory_order_relaxed);
}

// Set a knob by name ("gemv_lds_rows", "gemv_lds_waves", "gemv_rows",
// "gemv_iters", "gemm_tile", "gemv_mfma_m", "w4a16_path", "moe_gemm_path",
// "gemv_mm", "gemv_persist", "gemv_q80_lds", "gemv_fuse_m"); 0
// restores the
// automatic rule.
UB_API int ubridge_tune_set(const char* name, int value) {
  const int k = knob_index(name);
  if (k < 0) return ub_set_error(UB_ERR_INVALID_ARG, "ubridge_tune_set: unknown knob '%s'",
                                 name ? name : "(null)");
  g_knob[k].store(value, std::memory_order_relaxed);
  g_knob_init[k].store(true, std::memory_order_release);
  return UB_OK;
}

// Current value of a knob (0 = automatic); unknown names set error 1 and
// return 0.
UB_API int ubridge_tune_get(const char* name) {
  const int k = knob_index(name);
  if (k < 0) {
    ub_set_error(UB_ERR_INVALID_ARG, "ubridge_tune_get: unknown knob '%s'", name ? name : "(null)");
    return 0;
  }
  return ub_tune(k);
}

// ------------------------------------------------------ device scratch
// Scratch for kernels that split work across workgroups and combine partial
// results in a second launch, and for the dequantized weight slabs of the
// prefill routes.  The reference's entry points take no workspace argument;
// its only device allocations (the topsaten MoE workspaces) go through a
// stream-ordered allocator the host registers
// (kernels/topsaten_moe_wrapper.cpp:18-48).  Here likewise:
//  * with an allocator registered (ubridge_set_workspace_allocator), every
//    call that needs scratch takes it from that allocator on its stream and
//    hands it back on the same stream once its kernels are enqueued; the
//    library then holds no device memory of its own;
//  * otherwise a per-(device, stream) pool buffer (one for each that a call holds at
//    once), grown on demand, of one call at a time: another thread's call on the
//    stream waits until the first has enqueued its kernels.  A buffer
//    it outgrows is retired: freed once an event recorded after its last use
//    has completed, unless it was handed out while the stream captured a
//    graph (graphs keep its address: it then lives until
//    ubridge_release_workspace).  Calls that ask for it draw, while they are
//    captured, on buffers of that capture alone, which are free again, for another
//    capture or at the next eager call, once its graph and the executables of it
//    are destroyed.  ubridge_release_workspace(stream)
//    synchronizes the stream and frees all of that stream's buffers.
// Growth during a graph capture allocates with the capture mode relaxed, so
// calls take the same route (and give the same bits) captured or eager.
#include <map>
#include <mutex>
#include <utility>
#include <vector>
namespace {
// What a buffer and the graph that names it share: the graph retains it as a user
// object, whose end is the end of the graph, of the executables made from it and of
// their launches.  That call may come on any thread, after the pool is gone too.
struct WsTie {
  std::atomic<bool> ended{false};
  std::atomic<int> refs{2};
  void drop() {
    if (refs.fetch_sub(1) == 1) delete this;
  }
  static void end(void* p) {
    ((WsTie*)p)->ended = true;
    ((WsTie*)p)->drop();
  }
};
struct WsBuf {
  void* p = nullptr;
  size_t bytes = 0;
  bool graph = false;  // handed out during a capture
  unsigned long long capture = 0;  // the one capture that it belongs to (0: any)
  size_t level = 0;                // there: scratch that its call held already
  WsTie* tie = nullptr;            // and its graph (null: not known, it lives until released)
};
struct WsRetired {
  WsBuf b;
  hipEvent_t ev = nullptr;  // completes after the buffer's last eager use
};
struct WsPool {
  // Held by a call from its first scratch to its last launch: its kernels lie together
  // on the stream, with no other call's on the same buffer in between and no buffer
  // outgrown (and freed) under it.  (recursive: a call may take several.)
  std::recursive_mutex call;
  // By how many the call holds already: a call that takes a second scratch while it
  // holds the first (a copy of misaligned activations, then parts of K) gets another.
  std::vector<WsBuf> cur;
  size_t held = 0;
  std::vector<WsRetired> retired;  // ev null: not yet ordered (see sweep)
};
std::mutex g_ws_mu;
std::map<std::pair<int, hipStream_t>, WsPool> g_ws;  // (never erased from: calls wait on them)
size_t g_ws_live_n = 0, g_ws_live_bytes = 0;  // pool buffers allocated, not freed
long g_ws_caller_out = 0;                     // caller-allocator blocks not yet handed back
ubridge_ws_alloc_fn g_ws_alloc = nullptr;
ubridge_ws_free_fn g_ws_free = nullptr;
void* g_ws_ctx = nullptr;

bool capturing(hipStream_t s) {
  hipStreamCaptureStatus st = hipStreamCaptureStatusNone;
  if (hipStreamIsCapturing(s, &st) != hipSuccess) {
    (void)hipGetLastError();
    return false;
  }
  return st != hipStreamCaptureStatusNone;
}

// The capture's own number and graph, or 0 (not known: the stream's shared buffer serves).
unsigned long long capture_id(hipStream_t s, hipGraph_t* graph) {
  hipStreamCaptureStatus st = hipStreamCaptureStatusNone;
  unsigned long long id = 0;
  const hipGraphNode_t* deps = nullptr;
  size_t n = 0;
  *graph = nullptr;
  if (hipStreamGetCaptureInfo_v2(s, &st, &id, graph, &deps, &n) != hipSuccess) {
    (void)hipGetLastError();
    return 0;
  }
  return st == hipStreamCaptureStatusActive ? id : 0;
}

// Ties a buffer to the graph being captured; null: it could not be.
WsTie* ws_tie(hipGraph_t graph) {
  if (!graph) return nullptr;
  WsTie* t = new WsTie;
  UbRelaxCapture relax;
  hipUserObject_t o = nullptr;
  if (hipUserObjectCreate(&o, t, WsTie::end, 1, hipUserObjectNoDestructorSync) != hipSuccess) {
    (void)hipGetLastError();
    delete t;
    return nullptr;
  }
  if (hipGraphRetainUserObject(graph, o, 1, hipGraphUserObjectMove) != hipSuccess) {
    (void)hipGetLastError();
    (void)hipUserObjectRelease(o, 1);  // (drops the graph's reference)
    t->drop();
    return nullptr;
  }
  return t;
}

void ws_untie(WsBuf& b) {
  if (b.tie) b.tie->drop();
  b.tie = nullptr;
}

void ws_free(WsBuf& b) {
  ws_untie(b);
  if (!b.p) return;
  (void)hipFree(b.p);
  (void)hipGetLastError();
  g_ws_live_n--;
  g_ws_live_bytes -= b.bytes;
}

// Retired buffers of a pool (s not capturing, caller holds g_ws_mu): order
// the unordered ones behind an event recorded now (everything that used them
// is already on s), free those whose event has completed.  Graph-held
// buffers stay until their graph has ended, or until released.
void ws_sweep(WsPool& pool, hipStream_t s) {
  for (size_t i = 0; i < pool.retired.size();) {
    WsRetired& r = pool.retired[i];
    if (r.b.tie && r.b.tie->ended) {
      ws_untie(r.b);
      r.b.graph = false;
    }
    if (r.b.graph) {
      i++;
      continue;
    }
    if (!r.ev) {
      if (hipEventCreateWithFlags(&r.ev, hipEventDisableTiming) != hipSuccess ||
          hipEventRecord(r.ev, s) != hipSuccess) {
        (void)hipGetLastError();
        if (r.ev) (void)hipEventDestroy(r.ev);
        r.ev = nullptr;
        i++;
        continue;
      }
    }
    if (hipEventQuery(r.ev) == hipSuccess) {
      (void)hipEventDestroy(r.ev);
      ws_free(r.b);
      pool.retired.erase(pool.retired.begin() + i);
    } else {
      (void)hipGetLastError();  // hipErrorNotReady
      i++;
    }
  }
}

// A new buffer (caller holds g_ws_mu); p null: none to be had.
WsBuf ws_new(size_t bytes) {
  WsBuf b;
  const size_t sz = bytes < ((size_t)1 << 20) ? ((size_t)1 << 20) : bytes;
  hipError_t e;
  {
    UbRelaxCapture relax;
    e = hipMalloc(&b.p, sz);
  }
  if (e != hipSuccess) {
    (void)hipGetLastError();
    b.p = nullptr;
    return b;
  }
  g_ws_live_n++;
  g_ws_live_bytes += sz;
  b.bytes = sz;
  return b;
}

WsPool* ws_pool(hipStream_t s) {
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess) return nullptr;
  std::lock_guard<std::mutex> lk(g_ws_mu);
  return &g_ws[{dev, s}];
}

// (the caller holds pool.call)
void* ws_pool_get(WsPool& pool, hipStream_t s, size_t bytes, bool per_graph) {
  const bool cap = capturing(s);
  std::lock_guard<std::mutex> lk(g_ws_mu);
  if (!cap && !pool.retired.empty()) ws_sweep(pool, s);
  const size_t level = pool.held - 1;
  hipGraph_t graph = nullptr;
  if (const unsigned long long id = cap && per_graph ? capture_id(s, &graph) : 0) {
    for (const WsRetired& r : pool.retired)
      if (r.b.capture == id && r.b.level == level && r.b.bytes >= bytes) return r.b.p;
    // one whose graph has ended, the smallest that suffices, or a new one
    size_t at = pool.retired.size();
    for (size_t i = 0; i < pool.retired.size(); i++) {
      const WsBuf& b = pool.retired[i].b;
      if (b.tie && b.tie->ended && b.bytes >= bytes && (at == pool.retired.size() || b.bytes < pool.retired[at].b.bytes)) at = i;
    }
    if (at == pool.retired.size()) {
      WsBuf b = ws_new(bytes);
      if (!b.p) return nullptr;
      pool.retired.push_back(WsRetired{b, nullptr});
    }
    WsBuf& b = pool.retired[at].b;
    ws_untie(b);
    b.graph = true, b.capture = id, b.level = level, b.tie = ws_tie(graph);
    return b.p;
  }
  if (pool.cur.size() <= level) pool.cur.resize(level + 1);
  WsBuf& cur = pool.cur[level];
  if (cur.bytes >= bytes) {
    cur.graph |= cap;
    return cur.p;
  }
  WsBuf b = ws_new(bytes);
  if (!b.p) return nullptr;
  if (cur.p) {
    pool.retired.push_back(WsRetired{cur, nullptr});
    if (!cap) ws_sweep(pool, s);  // orders it behind the work already on s
  }
  b.graph = cap;
  cur = b;
  return b.p;
}
}  // namespace

UbScratch::UbScratch(hipStream_t s, size_t bytes, bool per_graph) : s_(s) {
  if (bytes == 0) return;
  ubridge_ws_alloc_fn fa;
  void* ctx;
  {
    std::lock_guard<std::mutex> lk(g_ws_mu);
    fa = g_ws_alloc;
    ctx = g_ws_ctx;
  }
  if (fa) {
    void* p = nullptr;
    if (fa(&p, bytes, (void*)s, ctx) == 0 && p) {
      p_ = p;
      caller_ = true;
      std::lock_guard<std::mutex> lk(g_ws_mu);
      g_ws_caller_out++;
    }
    return;
  }
  try {
    WsPool* pool = ws_pool(s);
    if (!pool) return;
    pool->call.lock();
    pool_ = pool;
    pool->held++;
    p_ = ws_pool_get(*pool, s, bytes, per_graph);
  } catch (...) {  // (out of host memory: as without device memory)
    p_ = nullptr;
  }
}

UbScratch::~UbScratch() {
  if (WsPool* pool = (WsPool*)pool_) {
    pool->held--;
    pool->call.unlock();
  }
  if (!caller_) return;
  ubridge_ws_free_fn ff;
  void* ctx;
  {
    std::lock_guard<std::mutex> lk(g_ws_mu);
    ff = g_ws_free;
    ctx = g_ws_ctx;
    g_ws_caller_out--;
  }
  if (ff) ff(p_, (void*)s_, ctx);
}

UB_API int ubridge_set_workspace_allocator(ubridge_ws_alloc_fn alloc, ubridge_ws_free_fn free_fn,
                                           void* ctx) {
  if ((alloc == nullptr) != (free_fn == nullptr))
    return ub_set_error(UB_ERR_INVALID_ARG,
                        "ubridge_set_workspace_allocator: give both functions or neither");
  std::lock_guard<std::mutex> lk(g_ws_mu);
  g_ws_alloc = alloc;
  g_ws_free = free_fn;
  g_ws_ctx = ctx;
  return UB_OK;
}

UB_API int ubridge_release_workspace(void* stream) {
  hipStream_t s = ub_stream(stream);
  {
    std::lock_guard<std::mutex> lk(g_ws_mu);
    if (g_ws.empty()) return UB_OK;  // nothing to free (touches no device)
  }
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess) return ub_set_error(UB_ERR_LAUNCH, "no device");
  if (capturing(s))
    return ub_set_error(UB_ERR_INVALID_ARG,
                        "ubridge_release_workspace: the stream is capturing a graph");
  WsPool* pool = ws_pool(s);
  if (!pool) return ub_set_error(UB_ERR_LAUNCH, "no device");
  std::lock_guard<std::recursive_mutex> call(pool->call);  // (another thread's call ends first)
  if (hipStreamSynchronize(s) != hipSuccess) {
    const hipError_t e = hipGetLastError();
    return ub_set_error(UB_ERR_LAUNCH, "ubridge_release_workspace: %s", hipGetErrorString(e));
  }
  std::lock_guard<std::mutex> lk(g_ws_mu);
  for (WsRetired& r : pool->retired) {
    if (r.ev) (void)hipEventDestroy(r.ev);
    ws_free(r.b);
  }
  pool->retired.clear();
  for (WsBuf& b : pool->cur) ws_free(b);
  pool->cur.clear();
  return UB_OK;
}

UB_API int ubridge_workspace_stats(size_t* live_buffers, size_t* live_bytes,
                                   long* caller_blocks_out) {
  std::lock_guard<std::mutex> lk(g_ws_mu);
  if (live_buffers) *live_buffers = g_ws_live_n;
  if (live_bytes) *live_bytes = g_ws_live_bytes;
  if (caller_blocks_out) *caller_blocks_out = g_ws_caller_out;
  return UB_OK;
}
