// kvcache.hip -- page operations of a paged key-value cache, on the device
// throughout: no page number, length or count visits the host.
//
// The cache is [L, 2, P, H, S, D] (layers, keys / values, pages, heads, slots).
// Its state is one int32 buffer [refs P | lens rows | tables rows x width]:
// how many rows hold a page, the tokens of a row, its pages in order (-1:
// none).
//
// free     the rows' pages lose a reference each, the rows become empty
// fork     each sample shares its prompt's whole pages and gets a copy of a
//          part-filled last one; new pages are the lowest free ones, in the
//          order of the samples
// compact  with n pages in use, the k-th used page from n on moves to the k-th
//          free page below n; tables and counts follow
//
// free and the planning of fork and compact touch a few hundred KiB and are
// bound by latency (us: free 3.1, fork's check 3.4 and plan 4.7, compact's plan 4.9);
// the page copies are bound by HBM, with eight 16-byte loads in flight a thread: 507
// pages of 512 KiB (530 MB in and out) 109 us, 4.9 TB/s (four in flight 119).  Non-temporal
// access was 4% faster there and 40% slower on fork, whose pages stay in the
// last-level cache for the attention that reads them next.
#include "common.h"

namespace {

constexpr int PT = 1024, kNear = 4096;  // threads of a planning workgroup; pages it lists in LDS

// exclusive prefix sum over the workgroup; total in `sum`
__device__ __forceinline__ int block_scan(int v, int* lds, int& sum) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int x = v;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int y = __shfl_up(x, o, 64);
    if (lane >= o) x += y;
  }
  if (lane == 63) lds[wave] = x;
  __syncthreads();
  if (wave == 0) {
    int w = lane < PT / 64 ? lds[lane] : 0;
#pragma unroll
    for (int o = 1; o < PT / 64; o <<= 1) {
      const int y = __shfl_up(w, o, 64);
      if (lane >= o) w += y;
    }
    if (lane < PT / 64) lds[lane] = w;
  }
  __syncthreads();
  const int before = wave ? lds[wave - 1] : 0;
  sum = lds[PT / 64 - 1];
  __syncthreads();
  return before + x - v;
}

// One workgroup a row.  The exchange makes a row that is named twice harmless.
__global__ void __launch_bounds__(256) k_free(int* __restrict__ refs, int* __restrict__ lens,
                                              int* __restrict__ tables, const int* __restrict__ rows,
                                              int P, int nrows, int width, int* err) {
  const int r = rows[blockIdx.x];
  if (r < 0 || r >= nrows) {
    if (threadIdx.x == 0) *err = UB_ERR_INDEX;
    return;
  }
  for (int i = threadIdx.x; i < width; i += 256) {
    const int p = atomicExch(&tables[(size_t)r * width + i], -1);
    if (p < 0) continue;
    if (p >= P) {
      *err = UB_ERR_INDEX;
    } else if (atomicSub(&refs[p], 1) <= 0) {  // was not held: the count stays
      atomicAdd(&refs[p], 1);
      *err = UB_ERR_INDEX;
    }
  }
  if (threadIdx.x == 0) lens[r] = 0;
}

// Workgroup j: len[j], tokens of sample j, and old[j], the page to copy for it (-1:
// none).  A sample of a row that is not there, of a table with a page in use that is
// not there, or in a row that holds a page is refused: -1 tokens.  (A launch of its
// own, 2 us more of a graph: the planning workgroup took as long for 4096 entries
// and 8 us for 16384.)
__global__ void __launch_bounds__(256) k_fork_check(const int* __restrict__ lens,
                                                    const int* __restrict__ tables,
                                                    const int* __restrict__ src,
                                                    const int* __restrict__ dst, int* len, int* old,
                                                    int P, int S, int nrows, int width, int* err) {
  const int j = blockIdx.x, s = src[j], d = dst[j];
  const int m = s >= 0 && s < nrows && d >= 0 && d < nrows ? lens[s] : -1;
  int bad = m < 0 || m > (long)width * S;
  if (!bad)
    for (int i = threadIdx.x; i < width; i += 256) {
      const int p = tables[(size_t)s * width + i], own = tables[(size_t)d * width + i];
      if (m > 0) bad |= own >= 0 || (i <= (m - 1) / S && (p < 0 || p >= P));
    }
  bad = __syncthreads_or(bad);
  if (threadIdx.x != 0) return;
  len[j] = bad ? -1 : m;
  old[j] = bad || m % S == 0 ? -1 : tables[(size_t)s * width + m / S];
  if (bad) *err = UB_ERR_INDEX;
}

// One workgroup: who gets which new page.  plan: [n] tokens of the sample (-1:
// refused), [n] page to copy, [n] free pages found.  newp [n]: the sample's
// own page, -1 where it has none.
__global__ void __launch_bounds__(PT) k_fork_plan(const int* __restrict__ refs, int* lens,
                                                  const int* __restrict__ dst, int n, int* newp,
                                                  int* plan, int P, int* err) {
  __shared__ int lds[PT / 64];
  __shared__ int near[kNear];  // the first free pages, which is mostly all of them
  const int tid = threadIdx.x;
  int* len = plan;
  int* old = plan + n;
  int* found = plan + 2 * n;
  // asked for ahead of the rows: the counts of the first pages
  int f[16];
  auto counts = [&](int p) {
    if (p + 16 <= P) {
      __builtin_memcpy(f, refs + p, sizeof(f));
    } else {
#pragma unroll
      for (int i = 0; i < 16; i++) f[i] = p + i < P ? refs[p + i] : 1;
    }
  };
  counts(16 * tid);
  int need = 0;
  for (int j0 = 0; j0 < n; j0 += PT) {
    const int j = j0 + tid;
    int part = 0;
    if (j < n && len[j] >= 0) {
      const int m = len[j], d = dst[j];
      // the row must have no tokens; the claim gives it to one sample
      if (m == 0 ? lens[d] != 0 : atomicCAS(&lens[d], 0, m) != 0) {
        len[j] = -1;
        *err = UB_ERR_INDEX;
      } else {
        part = old[j] >= 0;
      }
    }
    int sum;
    const int k = block_scan(part, lds, sum);
    if (j < n) newp[j] = part ? need + k : -1;  // the rank, until the pages are known
    need += sum;
  }
  int have = 0;
  for (int p0 = 0; p0 < P && have < need; p0 += PT * 16) {
    const int p = p0 + 16 * tid;
    if (p0) counts(p);
    int c = 0;
#pragma unroll
    for (int i = 0; i < 16; i++) c += f[i] == 0;
    int sum;
    int k = have + block_scan(c, lds, sum);
#pragma unroll
    for (int i = 0; i < 16; i++)
      if (f[i] == 0) {
        if (k < need) {
          if (k < kNear) near[k] = p + i;
          else found[k] = p + i;
        }
        k++;
      }
    have += sum;
  }
  __syncthreads();
  for (int j = tid; j < n; j += PT) {
    const int k = newp[j];
    if (k < 0) continue;
    if (k < have) {
      newp[j] = k < kNear ? near[k] : found[k];
    } else {  // no page left: the sample stays empty
      lens[dst[j]] = 0;
      len[j] = newp[j] = -1;
      *err = UB_ERR_INDEX;
    }
  }
}

template <int B> struct Bytes;
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));
template <> struct Bytes<16> { typedef u32x4 T; };
template <> struct Bytes<8> { typedef u32x2 T; };
template <> struct Bytes<4> { typedef uint32_t T; };
template <> struct Bytes<2> { typedef uint16_t T; };
template <> struct Bytes<1> { typedef uint8_t T; };

// units of B bytes, by one workgroup of 256
template <int B>
__device__ __forceinline__ void copy_units(uint8_t* d, const uint8_t* s, long n) {
  typedef typename Bytes<B>::T T;
  constexpr int Q = 8;  // in flight a thread
  T* dp = (T*)d;
  const T* sp = (const T*)s;
  long i = threadIdx.x;
  for (; i + 256 * (Q - 1) < n; i += 256 * Q) {
    T v[Q];
#pragma unroll
    for (int q = 0; q < Q; q++) v[q] = sp[i + 256 * q];
#pragma unroll
    for (int q = 0; q < Q; q++) dp[i + 256 * q] = v[q];
  }
  for (; i < n; i += 256) dp[i] = sp[i];
}

// Workgroup (x, j): slice x of sample j's new page; x = 0 also writes its row.
template <int B>
__global__ void __launch_bounds__(256) k_fork(uint8_t* kv, int* refs, int* tables,
                                              const int* __restrict__ src,
                                              const int* __restrict__ dst,
                                              const int* __restrict__ newp,
                                              const int* __restrict__ plan, int n, int P, int S,
                                              int width, long page_bytes, int slices) {
  const int j = blockIdx.y, m = plan[j];
  if (m <= 0) return;
  const int np = newp[j];
  if (blockIdx.x == 0) {
    const int pages = (m + S - 1) / S;
    const int* from = tables + (size_t)src[j] * width;
    int* to = tables + (size_t)dst[j] * width;
    for (int i = threadIdx.x; i < pages; i += 256) {
      const int p = np >= 0 && i == pages - 1 ? np : from[i];
      to[i] = p;
      atomicAdd(&refs[p], 1);
    }
  }
  if (np < 0) return;
  const int lk = blockIdx.x / slices, sl = blockIdx.x - lk * slices;
  const long per = (page_bytes / B + slices - 1) / slices;
  const long u0 = sl * per, u1 = min(page_bytes / B, u0 + per);
  if (u0 >= u1) return;
  const long base = (long)lk * P;
  copy_units<B>(kv + (base + np) * page_bytes + u0 * B,
                kv + (base + plan[n + j]) * page_bytes + u0 * B, u1 - u0);
}

// One workgroup: the moves.  plan: [1] their number, [P / 2] from, [P / 2] to;
// map [P]: where a page of the old numbering lies now, or -2 - k for move k.
// Q: pages of a thread, in a tile of PT Q.
template <int Q>
__global__ void __launch_bounds__(PT) k_compact_plan(const int* refs, int P, int* plan, int* map,
                                                     int* n_out) {
  __shared__ int lds[PT / 64];
  __shared__ int below_n;
  const int tid = threadIdx.x;
  int f[Q];
  auto counts = [&](int p) {
    if (p + Q <= P) {
      __builtin_memcpy(f, refs + p, sizeof(f));
    } else {
#pragma unroll
      for (int i = 0; i < Q; i++) f[i] = p + i < P ? refs[p + i] : 0;
    }
    int c = 0;
#pragma unroll
    for (int i = 0; i < Q; i++) c += f[i] != 0;
    return c;
  };
  int n = 0, sum = 0, u = 0;
  for (int p0 = 0; p0 < P; p0 += PT * Q) {
    u = block_scan(counts(p0 + Q * tid), lds, sum);
    n += sum;
  }
  int* from = plan + 1;
  int* to = from + P / 2;
  int below = n;  // used pages below page n (all of them, if none lies from n on)
  for (int p0 = 0, before = 0; p0 < P; p0 += PT * Q, before += sum) {
    const int p = p0 + Q * tid;
    if (P > PT * Q) u = before + block_scan(counts(p), lds, sum);  // (else as it is)
    if (n >= p && n < p + Q && n < P) {
      int b = u;
#pragma unroll
      for (int i = 0; i < Q; i++)
        if (p + i < n) b += f[i] != 0;
      below_n = b;
    }
    __syncthreads();
    if (n >= p0 && n < p0 + PT * Q && n < P) below = below_n;
    int mv[Q];
#pragma unroll
    for (int i = 0; i < Q; i++) {
      mv[i] = p + i;
      if (p + i >= P) continue;
      const bool used = f[i] != 0;
      if (used && p + i >= n) mv[i] = below - u - 2;
      if (used && p + i >= n) from[u - below] = p + i;
      if (!used && p + i < n) to[p + i - u] = p + i;
      u += used;
    }
    if (p + Q <= P) {
      __builtin_memcpy(map + p, mv, sizeof(mv));
    } else {
#pragma unroll
      for (int i = 0; i < Q; i++)
        if (p + i < P) map[p + i] = mv[i];
    }
  }
  if (tid == 0) {
    plan[0] = n - below;
    *n_out = n;
  }
}

// A grid that walks the tables and counts, then the (move, layer, key / value,
// slice) units.  Sources are pages from n on, destinations pages below n.
template <int B>
__global__ void __launch_bounds__(256) k_compact(uint8_t* kv, int* refs, int* tables,
                                                 const int* __restrict__ plan,
                                                 const int* __restrict__ map, int L2, int P,
                                                 long entries, long page_bytes, int slices,
                                                 int* err) {
  const int moves = plan[0];
  const int* from = plan + 1;
  const int* to = from + P / 2;
  const long first = blockIdx.x * 256l + threadIdx.x, step = gridDim.x * 256l;
  for (long i = first; i < entries; i += step) {
    const int p = tables[i];
    if (p < 0) continue;
    if (p < P) {
      const int m = map[p];
      tables[i] = m >= 0 ? m : to[-2 - m];
    } else {
      *err = UB_ERR_INDEX;
    }
  }
  for (long k = first; k < moves; k += step) {
    refs[to[k]] = refs[from[k]];
    refs[from[k]] = 0;
  }
  const long units = page_bytes / B, per = (units + slices - 1) / slices;
  const long total = (long)moves * L2 * slices;
  for (long w = blockIdx.x; w < total; w += gridDim.x) {
    const long k = w / ((long)L2 * slices);
    const int r = (int)(w - k * L2 * slices), lk = r / slices, sl = r - lk * slices;
    const long u0 = sl * per, u1 = min(units, u0 + per);
    const long base = (long)lk * P;
    if (u0 < u1)
      copy_units<B>(kv + (base + to[k]) * page_bytes + u0 * B,
                    kv + (base + from[k]) * page_bytes + u0 * B, u1 - u0);
  }
}

int unit_bytes(const void* kv, long page_bytes) {
  int b = 16;
  while (b > 1 && (page_bytes % b != 0 || (uintptr_t)kv % b != 0)) b >>= 1;
  return b;
}

int check_pool(const char* nm, const UbridgeKvPool* p) {
  UB_REQUIRE(p, "%s: null pool", nm);
  UB_REQUIRE(p->L > 0 && p->P >= 0 && p->S > 0 && p->rows >= 0 && p->width >= 0 && p->page_bytes > 0,
             "%s: L=%d P=%d S=%d rows=%d width=%d page_bytes=%ld", nm, p->L, p->P, p->S, p->rows,
             p->width, (long)p->page_bytes);
  UB_REQUIRE(p->P == 0 || (p->kv && p->refs), "%s: null pages or counts", nm);
  UB_REQUIRE(p->rows == 0 || (p->lens && (p->tables || p->width == 0)), "%s: null lengths or tables", nm);
  return UB_OK;
}

}  // namespace

UB_API int ubridge_kv_free(const UbridgeKvPool* p, const int32_t* rows, int n, void* stream) {
  const char* nm = "ubridge_kv_free";
  if (int e = check_pool(nm, p)) return e;
  UB_REQUIRE(n >= 0 && n < 1 << 24, "%s: n=%d", nm, n);
  if (n == 0) return UB_OK;
  UB_REQUIRE(rows, "%s: null rows", nm);
  int* err = ub_error_flag();
  UB_REQUIRE(err, "%s: no device flag", nm);
  k_free<<<n, 256, 0, ub_stream(stream)>>>(p->refs, p->lens, p->tables, rows, p->P, p->rows,
                                           p->width, err);
  return ub_check_launch(nm);
}

UB_API int ubridge_kv_fork(const UbridgeKvPool* p, const int32_t* src, const int32_t* dst, int n,
                           int32_t* new_pages, void* stream) {
  const char* nm = "ubridge_kv_fork";
  if (int e = check_pool(nm, p)) return e;
  UB_REQUIRE(n >= 0 && n < 65536, "%s: n=%d (at most 65535)", nm, n);
  if (n == 0) return UB_OK;
  UB_REQUIRE(src && dst && new_pages, "%s: null rows", nm);
  int* err = ub_error_flag();
  UB_REQUIRE(err, "%s: no device flag", nm);
  hipStream_t s = ub_stream(stream);
  UbScratch ws(s, sizeof(int) * 3 * (size_t)n);
  int* plan = (int*)ws.get();
  if (!plan) return ub_set_error(UB_ERR_LAUNCH, "%s: no workspace", nm);
  k_fork_check<<<n, 256, 0, s>>>(p->lens, p->tables, src, dst, plan, plan + n, p->P, p->S, p->rows, p->width, err);
  k_fork_plan<<<1, PT, 0, s>>>(p->refs, p->lens, dst, n, new_pages, plan, p->P, err);
  const int b = unit_bytes(p->kv, p->page_bytes);
  const int slices = (int)(p->page_bytes / 32768 > 0 ? p->page_bytes / 32768 : 1);
  const dim3 grid(2 * p->L * slices, n);
#define UB_GO(B)                                                                                 \
  k_fork<B><<<grid, 256, 0, s>>>((uint8_t*)p->kv, p->refs, p->tables, src, dst, new_pages, plan, \
                                 n, p->P, p->S, p->width, p->page_bytes, slices)
  if (b == 16) UB_GO(16);
  else if (b == 8) UB_GO(8);
  else if (b == 4) UB_GO(4);
  else if (b == 2) UB_GO(2);
  else UB_GO(1);
#undef UB_GO
  return ub_check_launch(nm);
}

UB_API int ubridge_kv_compact(const UbridgeKvPool* p, int32_t* n_used, void* stream) {
  const char* nm = "ubridge_kv_compact";
  if (int e = check_pool(nm, p)) return e;
  UB_REQUIRE(n_used, "%s: null count", nm);
  int* err = ub_error_flag();
  UB_REQUIRE(err, "%s: no device flag", nm);
  hipStream_t s = ub_stream(stream);
  UbScratch ws(s, sizeof(int) * (2 * (size_t)p->P + 2));
  int* plan = (int*)ws.get();
  if (!plan) return ub_set_error(UB_ERR_LAUNCH, "%s: no workspace", nm);
  int* map = plan + 2 * (p->P / 2) + 1;
  // four pages a thread up to 4096: 2048 pages take 4.9 us (the least of 30 4.0), 5.0
  // (4.9) with sixteen
  if (p->P <= 4 * PT) k_compact_plan<4><<<1, PT, 0, s>>>(p->refs, p->P, plan, map, n_used);
  else k_compact_plan<16><<<1, PT, 0, s>>>(p->refs, p->P, plan, map, n_used);
  const int b = unit_bytes(p->kv, p->page_bytes);
  const int slices = (int)(p->page_bytes / 32768 > 0 ? p->page_bytes / 32768 : 1);
#define UB_GO(B)                                                                             \
  k_compact<B><<<2048, 256, 0, s>>>((uint8_t*)p->kv, p->refs, p->tables, plan, map, 2 * p->L, p->P,   \
                                    (long)p->rows * p->width, p->page_bytes, slices, err)
  if (b == 16) UB_GO(16);
  else if (b == 8) UB_GO(8);
  else if (b == 4) UB_GO(4);
  else if (b == 2) UB_GO(2);
  else UB_GO(1);
#undef UB_GO
  return ub_check_launch(nm);
}
