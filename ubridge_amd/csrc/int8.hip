// int8.hip -- int8 W8A8 linear on gfx950:
//
//   y[m, n] = T( (sum_k a[m, k] w[n, k]) sw[n] sa[m] + bias[n] )
//
// a[m, k] = round(x[m, k] / sa[m]) (ties to even), sa[m] = max_k |x[m, k]| /
// 127, or 1 for a row of zeros; sw one f32 scale an output channel.  The dot is
// exact in int32 (|a w| <= 127 * 128, so K <= 132104), the epilogue f32, and
// the sum rounds once, to x's type T.  The weight's scale is multiplied in first:
// sa reaches both ends of f32, and with it first rows near the top overflowed.  A
// row that holds an infinity or a NaN has no scale and gives a row of NaN.
//
// Rows of a and w are padded with zeros to ld bytes, a multiple of 128.
//
// Up to 16 tokens (of 64 KiB in all) the product is a stream of the weight and one
// kernel does it all (k_i8_dec); beyond, k_quant makes the codes and k_i8_gemm (or k_i8_ring, by
// plan_for) multiplies them.  us: 8 x 4096 x 6144 (M x K x N) 10.7, of which the
// weight's 25 MB are 4 and the rest is the launch, the activations' codes ahead of
// the first product and the sum over the wavefronts; 8 x 4096 x 28672 26 (4.5 TB/s);
// 201 x 3520 x 9001 4 + 19, bound by a tile's K-steps (0.55 us each, of which 0.2
// are products); 4096 x 4096 x 14336 10 + 243 (2.0 POP/s, 2.3 on 4096 x 8192 x 8192,
// where the library's own int8 product reaches 2.5); power is a part of it: with
// operands of zeros the call takes 0.7 of the time.
#include "common.h"
#include "lds_dma.h"

#include <type_traits>

namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));

template <int DT> struct Elem { typedef uint16_t T; static constexpr int E = 8; };  // 16-byte units
template <> struct Elem<UB_F32> { typedef float T; static constexpr int E = 4; };
constexpr int kSum = 100;  // "type" of the int32 sums over a part of K
template <> struct Elem<kSum> { typedef int T; static constexpr int E = 4; };

// element e of a unit
template <int DT>
__device__ __forceinline__ float get(const uint4& w, int e) {
  const uint32_t p[4] = {w.x, w.y, w.z, w.w};
  if constexpr (DT == UB_F32) return __uint_as_float(p[e]);
  else if constexpr (DT == UB_F16) return ub_f16_to_f32((uint16_t)(p[e >> 1] >> (16 * (e & 1))));
  else return __uint_as_float((e & 1) ? p[e >> 1] & 0xffff0000u : p[e >> 1] << 16);
}

// Unit i of a row at p that has V whole ones; zeros from there on.  The row
// may start at any element: gfx950 loads 16 bytes from there.  The K mod E
// elements behind the whole units are one lane's each (loads of their own in
// every unit made the kernels several times as long).
template <int DT>
__device__ __forceinline__ uint4 unit(const typename Elem<DT>::T* p, int i, int V) {
  uint4 v = make_uint4(0, 0, 0, 0);
  if (i < V) __builtin_memcpy(&v, p + i * Elem<DT>::E, 16);
  return v;
}

// A row's maximum is taken over bit patterns without sign, which order like
// the values and put infinities and NaN on top.
template <int DT>
__device__ __forceinline__ uint32_t top_of(const uint4& u, uint32_t t) {
#pragma unroll
  for (int e = 0; e < Elem<DT>::E; e++) t = max(t, __float_as_uint(get<DT>(u, e)) & 0x7fffffffu);
  return t;
}
__device__ __forceinline__ float scale_of(uint32_t top) {
  return top >= 0x7f800000u ? __builtin_nanf("") : top == 0 ? 1.0f : __fdiv_rn(__uint_as_float(top), 127.0f);
}

// The code of v under scale s, in the low byte.  The quotient is v r (r = 1 / s)
// corrected twice by its exact residual v - q s (Markstein's division: the
// second correction gives the correctly rounded v / s), 5 operations where the
// IEEE divide takes 11.  Adding 1.5 2^23 rounds to an integer, ties to even, in
// the low bits.  PLAIN, for s outside [2^-60, 2^60], where residuals underflow:
// the divide; and a clamp, since |v / s| <= 127 but for a denormal s, whose own
// rounding is as large as s.  A NaN or zero s has codes 0.
template <bool PLAIN>
__device__ __forceinline__ uint32_t code(float v, float s, float r) {
  float q;
  if constexpr (PLAIN) {
    q = __fdiv_rn(v, s);
    q = q == q ? fminf(fmaxf(q, -127.f), 127.f) : 0.f;
  } else {
    q = v * r;
    q = __builtin_fmaf(__builtin_fmaf(-q, s, v), r, q);
    q = __builtin_fmaf(__builtin_fmaf(-q, s, v), r, q);
  }
  return __float_as_uint(q + 12582912.f);
}
// of a unit
template <int DT, bool PLAIN>
__device__ __forceinline__ void codes(const uint4& u, float s, float r, uint32_t (&o)[Elem<DT>::E / 4]) {
  constexpr int E = Elem<DT>::E;
  uint32_t c[E];
#pragma unroll
  for (int e = 0; e < E; e++) c[e] = code<PLAIN>(get<DT>(u, e), s, r);
#pragma unroll
  for (int h = 0; h < E / 4; h++)
    o[h] = __builtin_amdgcn_perm(__builtin_amdgcn_perm(c[4 * h + 3], c[4 * h + 2], 0x0c0c0400u),
                                 __builtin_amdgcn_perm(c[4 * h + 1], c[4 * h], 0x0c0c0400u), 0x05040100u);
}
// (the same in every lane, as s is)
__device__ __forceinline__ bool plain_scale(float s) {
  return __builtin_amdgcn_readfirstlane(!(s >= 0x1p-60f && s <= 0x1p60f));
}

// One workgroup of NT threads a row; a thread keeps NV units of it in registers,
// so the row is read once.  NV = 0: rows of any length, read twice.
template <int DT, int NT, int NV>
__global__ void __launch_bounds__(NT) k_quant(const void* __restrict__ x, int8_t* __restrict__ q,
                                              float* __restrict__ scale, int K, int ld) {
  constexpr int E = Elem<DT>::E, N = NV ? NV : 1;
  __shared__ uint32_t wm[NT / 64];
  const int tid = threadIdx.x;
  const size_t row = blockIdx.x;
  const typename Elem<DT>::T* p = (const typename Elem<DT>::T*)x + row * K;
  const int V = K / E;
  uint4 u[N];
  uint32_t top = 0;
  typename Elem<DT>::T behind[1] = {0};  // element V E + tid
  if (tid < K - V * E) behind[0] = p[V * E + tid];
  if constexpr (NV > 0) {
#pragma unroll
    for (int j = 0; j < NV; j++) u[j] = unit<DT>(p, tid + j * NT, V);
#pragma unroll
    for (int j = 0; j < NV; j++) top = top_of<DT>(u[j], top);
  } else {
    for (int i = tid; i < V; i += NT) top = top_of<DT>(unit<DT>(p, i, V), top);
  }
  top = max(top, __float_as_uint(ub_load<DT>(behind, 0)) & 0x7fffffffu);
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, o, 64));
  if ((tid & 63) == 0) wm[tid >> 6] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < NT / 64; w++) top = max(top, wm[w]);
  const float s = scale_of(top);
  if (tid == 0) scale[row] = s;
  const bool plain = plain_scale(s);
  const float r = plain ? 0.f : __fdiv_rn(1.0f, s);
  int8_t* const qr = q + row * ld;
  auto store = [&](auto P, const uint4& v, int i) {
    constexpr bool PLAIN = decltype(P)::value;
    if (i == V) return;  // (below)
    uint32_t o[E / 4];
    codes<DT, PLAIN>(v, s, r, o);
    if constexpr (E == 4) ((uint32_t*)qr)[i] = o[0];
    else ((uint2*)qr)[i] = make_uint2(o[0], o[1]);
  };
  auto last = [&](auto P) {
    if (tid < E && V * E < ld) qr[V * E + tid] = (int8_t)code<decltype(P)::value>(ub_load<DT>(behind, 0), s, r);
  };
  if (NV == 0 || plain) {
    auto all = [&](auto P) {
      for (int i = tid; i * E < ld; i += NT) store(P, unit<DT>(p, i, V), i);
      last(P);
    };
    if (plain) all(std::true_type{});
    else all(std::false_type{});
  } else {
#pragma unroll
    for (int j = 0; j < N; j++)
      if ((tid + j * NT) * E < ld) store(std::false_type{}, u[j], tid + j * NT);
    last(std::false_type{});
  }
}

template <int DT>
__device__ __forceinline__ void put(void* y, size_t i, int acc, float sa, float sw, float b) {
  if constexpr (DT == kSum) ((int*)y)[i] = acc;
  else ub_store<DT>(y, i, (float)acc * sw * sa + b);
}

// ------------------------------------------------------------------ tiles
// A wavefront's 32 TM x 32 TN outputs, through its part of LDS (kStage bytes a
// wavefront, free by now) in rows, so that a store instruction writes whole runs
// of a row.  The weights are the products' left operand: lane (c, kh) holds row m
// = c and columns 8 q + 4 kh .. + 3 of a 32 x 32 tile, four to an LDS write.
template <int DT, int TM, int TN>
struct Epilogue {
  typedef typename Elem<DT>::T T;
  static constexpr int kPitch = 32 * TN * sizeof(T) + 16, kStage = 32 * kPitch;
  static __device__ __forceinline__ void run(const i32x16 (&acc)[TM][TN], uint8_t* st, const float* sa, const float* sw,
                                             const float* bias, void* y, int M, int N, int pitch, int m0, int n0) {
    constexpr int E = Elem<DT>::E, LR = 32 * TN / E, RI = 64 / LR;  // lanes a row, rows an instruction
    const int lane = threadIdx.x & 63, c = lane & 31, kh = lane >> 5;
    float s[TN][16], b[TN][16];
#pragma unroll
    for (int j = 0; j < TN; j++)
#pragma unroll
      for (int r = 0; r < 16; r++) {
        const int n = min(n0 + 32 * j + 8 * (r >> 2) + 4 * kh + (r & 3), N - 1);
        s[j][r] = DT == kSum ? 0.f : sw[n];
        b[j][r] = DT != kSum && bias ? bias[n] : 0.f;
      }
#pragma unroll
    for (int i = 0; i < TM; i++) {
      const float a = DT == kSum ? 0.f : sa[min(m0 + 32 * i + c, M - 1)];
#pragma unroll
      for (int j = 0; j < TN; j++)
#pragma unroll
        for (int q = 0; q < 4; q++) {
          T v[4];
#pragma unroll
          for (int e = 0; e < 4; e++) put<DT>(v, e, acc[i][j][4 * q + e], a, s[j][4 * q + e], b[j][4 * q + e]);
          __builtin_memcpy(st + c * kPitch + (32 * j + 8 * q + 4 * kh) * sizeof(T), v, sizeof(v));
        }
#pragma unroll
      for (int k = 0; k < 32; k += RI) {
        const int row = k + lane / LR, col = (lane % LR) * E;
        const uint4 v = *(const uint4*)(st + row * kPitch + col * sizeof(T));
        const int m = m0 + 32 * i + row, n = n0 + col;
        if (m < M && row < 32) {
          T* p = (T*)y + (size_t)m * pitch + n;
          if (n + E <= N) {
            __builtin_memcpy(p, &v, 16);
          } else {
            T w[E];
            __builtin_memcpy(w, &v, 16);
#pragma unroll
            for (int e = 0; e < E; e++)
              if (n + e < N) p[e] = w[e];
          }
        }
      }
    }
  }
};

// Workgroup i runs on XCD i % 8: its place in an order of `total` of which every
// XCD, each with its own L2, takes one contiguous run.
__device__ __forceinline__ int xcd_run(int i, int total) {
  const int x = i % 8;
  return x * (total / 8) + min(x, total % 8) + i / 8;
}

// WM x WN wavefronts of 32 TM x 32 TN outputs each, v_mfma_i32_32x32x32_i8.  The
// operands reach LDS by direct loads in a ring of NS 64-byte K-steps, each row of
// 64 bytes swizzled in 16-byte units (unit u of row r at u ^ ((r >> 2) & 3)) so
// that the 16 rows of a fragment read lie in distinct banks.  Fragments live in
// registers, two sets: step k multiplies those read during step k - 1 while
// step k + 1's are read, and sends for step k + NS into the slot whose reading
// ended with the barrier; NS - 1 steps are in flight.
template <int DT, int WM, int WN, int TM, int TN, int NS>
__device__ __forceinline__ void i8_tile(const int8_t* A, const float* sa, const int8_t* B, const float* sw, const float* bias,
                                        void* y, int M, int N, int ld, int m0, int n0, uint8_t* lds) {
  constexpr int BM = 32 * WM * TM, BN = 32 * WN * TN, NW = WM * WN;
  constexpr int NA = BM / 16 / NW, NB = BN / 16 / NW;  // load instructions of a wavefront and step
  constexpr int AB = BM * 64, ST = (BM + BN) * 64;     // bytes
  typedef Epilogue<DT, TM, TN> Out;
  static_assert(NA * NW * 16 == BM && NB * NW * 16 == BN, "whole load instructions");
  static_assert(NW * Out::kStage <= NS * ST, "epilogue fits");
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / WN, wn = wave % WN;
  // rows past the end lie past the buffers: zeros
  const ub_u32x4 ra = ub_desc(A + (size_t)m0 * ld, (uint64_t)min(BM, M - m0) * ld);
  const ub_u32x4 rb = ub_desc(B + (size_t)n0 * ld, (uint64_t)min(BN, N - n0) * ld);
  const uint32_t base = ub_lds_addr(lds);
  uint32_t va[NA], vb[NB];
#pragma unroll
  for (int i = 0; i < NA; i++) {
    const int u = (i * NW + wave) * 64 + lane, row = u >> 2;
    va[i] = (uint32_t)row * (uint32_t)ld + 16 * ((u & 3) ^ ((row >> 2) & 3));
  }
#pragma unroll
  for (int i = 0; i < NB; i++) {
    const int u = (i * NW + wave) * 64 + lane, row = u >> 2;
    vb[i] = (uint32_t)row * (uint32_t)ld + 16 * ((u & 3) ^ ((row >> 2) & 3));
  }
  const int nk = ld / 64;
  auto issue = [&](int k, uint32_t off) {  // (steps past K: the last again, not used)
    const uint32_t k0 = (uint32_t)(min(k, nk - 1) * 64), sb = base + off + wave * 1024;
#pragma unroll
    for (int i = 0; i < NA; i++) ub_lds_load16_at(ra, sb + i * NW * 1024, va[i], k0);
#pragma unroll
    for (int i = 0; i < NB; i++) ub_lds_load16_at(rb, sb + AB + i * NW * 1024, vb[i], k0);
  };
  i32x16 acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; i++)
#pragma unroll
    for (int j = 0; j < TN; j++)
#pragma unroll
      for (int r = 0; r < 16; r++) acc[i][j][r] = 0;
  const int l32 = lane & 31, kh = lane >> 5;
  // units 2 kh and 2 kh + 1 of a row: a lane's part of two products; the swizzle
  // depends on the lane alone, tiles being 32 rows
  const uint32_t u0 = l32 * 64 + (((2 * kh) ^ ((l32 >> 2) & 3)) * 16);
  const uint32_t u1 = l32 * 64 + (((2 * kh + 1) ^ ((l32 >> 2) & 3)) * 16);
  const uint32_t fa = wm * 32 * TM * 64, fb = AB + wn * 32 * TN * 64;
  i32x4 af[2][TM][2], bf[2][TN][2];
  auto read_frags = [&](uint32_t off, int b) {
    const uint8_t* p0 = lds + off + u0;
    const uint8_t* p1 = lds + off + u1;
#pragma unroll
    for (int j = 0; j < TN; j++) {
      bf[b][j][0] = *(const i32x4*)(p0 + fb + j * 2048);
      bf[b][j][1] = *(const i32x4*)(p1 + fb + j * 2048);
    }
#pragma unroll
    for (int i = 0; i < TM; i++) {
      af[b][i][0] = *(const i32x4*)(p0 + fa + i * 2048);
      af[b][i][1] = *(const i32x4*)(p1 + fa + i * 2048);
    }
  };
  uint32_t off = 0;  // of step k's slot
  auto step = [&](auto Bc, int k) {
    constexpr int Bf = decltype(Bc)::value;
    __builtin_amdgcn_s_waitcnt(0xC07F);     // lgkmcnt(0): this step's fragments are read
    ub_wait_vmcnt<(NS - 2) * (NA + NB)>();  // the next step has landed
    ub_barrier();
    issue(k + NS, off);
    off = off == (NS - 1) * ST ? 0 : off + ST;
    read_frags(off, Bf ^ 1);  // (after the last step: not used)
#pragma unroll
    for (int q = 0; q < 2; q++)
#pragma unroll
      for (int j = 0; j < TN; j++)
#pragma unroll
        for (int i = 0; i < TM; i++)
          acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(bf[Bf][j][q], af[Bf][i][q], acc[i][j], 0, 0, 0);
#pragma unroll
    for (int q = 0; q < 2 * TM * TN; q++) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);  // 1 MFMA
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);  // 1 DS read
    }
  };
#pragma unroll
  for (int k = 0; k < NS; k++) issue(k, k * ST);
  ub_wait_vmcnt<(NS - 1) * (NA + NB)>();
  ub_barrier();
  read_frags(0, 0);
  for (int k = 0; k < nk; k += 2) {  // (nk is even)
    step(std::integral_constant<int, 0>{}, k);
    step(std::integral_constant<int, 1>{}, k + 1);
  }
  __builtin_amdgcn_s_waitcnt(0xC07F);
  ub_wait_vmcnt<0>();
  ub_barrier();
  Out::run(acc, lds + wave * Out::kStage, sa, sw, bias, y, M, N, N, m0 + wm * 32 * TM, n0 + wn * 32 * TN);
}

// The tiles in ub_tile_at's order, dealt to the XCDs in runs; from tile `full` on (a multiple of the CUs) a tile is
// two workgroups, its upper and its lower half: the last round, where at most
// half the CUs had a tile, then takes about half as long.  full = all tiles
// otherwise, as for tiles of one product's height (TM = 1).
template <int DT, int WM, int WN, int TM, int TN, int NS>
__global__ void __launch_bounds__(64 * WM * WN) __attribute__((amdgpu_waves_per_eu(2, 2)))
k_i8_gemm(const int8_t* __restrict__ A, const float* __restrict__ sa, const int8_t* __restrict__ B,
          const float* __restrict__ sw, const float* __restrict__ bias, void* __restrict__ y, int M,
          int N, int ld, int full) {
  constexpr int BM = 32 * WM * TM, BN = 32 * WN * TN;
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  const int tm = (M + BM - 1) / BM, tn = (N + BN - 1) / BN;
  const int b = (int)blockIdx.x;
  int tile_m, tile_n;
  if (TM == 1 || b < full) {
    ub_tile_at(xcd_run(b, full), 0, tm, tn, 8, tile_m, tile_n);
    i8_tile<DT, WM, WN, TM, TN, NS>(A, sa, B, sw, bias, y, M, N, ld, tile_m * BM, tile_n * BN, lds);
  } else if constexpr (TM > 1) {
    ub_tile_at(full + ((b - full) >> 1), 0, tm, tn, 8, tile_m, tile_n);
    const int m0 = tile_m * BM + ((b - full) & 1) * (BM / 2);
    if (m0 < M) i8_tile<DT, WM, WN, TM / 2, TN, NS>(A, sa, B, sw, bias, y, M, N, ld, m0, tile_n * BN, lds);
  }
}

// The same product for grids that leave a workgroup or less to a CU, where the
// latency of a K-step's loads is what costs: a ring of NS 128-byte steps in LDS,
// NS - 1 of them in flight, one barrier a step.  Rows of 128 bytes, unit u of row
// r at u ^ ((r >> 1) & 7).  Long rows over few tiles are cut in parts of K, whose int32
// sums (DT = kSum, exact in any order) k_i8_sum adds.
template <int DT, int WM, int WN, int TM, int TN, int NS>
__global__ void __launch_bounds__(64 * WM * WN) __attribute__((amdgpu_waves_per_eu(2, 2)))
k_i8_ring(const int8_t* __restrict__ A, const float* __restrict__ sa, const int8_t* __restrict__ B,
          const float* __restrict__ sw, const float* __restrict__ bias, void* __restrict__ y, int M,
          int N, int ld, int part) {
  constexpr int BM = 32 * WM * TM, BN = 32 * WN * TN, NW = WM * WN;
  constexpr int NL = (BM + BN) / 8 / NW;  // load instructions of a wavefront and step: 8 rows each
  constexpr int ST = (BM + BN) * 128;
  static_assert(NL * NW * 8 == BM + BN && (BM / 8) % NW == 0, "whole load instructions");
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / WN, wn = wave % WN;
  int tile_m, tile_n;
  const int tm = (M + BM - 1) / BM, tn = (N + BN - 1) / BN;
  const int id = xcd_run((int)blockIdx.x, (int)gridDim.x), kp = id / (tm * tn);  // part kp of K
  ub_tile_at(id - kp * tm * tn, 0, tm, tn, 8, tile_m, tile_n);
  // rows and columns even over the tiles: what a tile does not need, it does not
  // load (rows past the end lie past the buffers: zeros)
  const int rows = (M + tm - 1) / tm, cols = min(BN, ((N + tn - 1) / tn + 15) & ~15);
  const int n0 = tile_n * cols, m0 = tile_m * rows, n1 = min(N, n0 + cols), m1 = min(M, m0 + rows);
  if (m0 >= m1 || n0 >= n1) return;  // (the same in every thread)
  const ub_u32x4 ra = ub_desc(A + (size_t)m0 * ld, (uint64_t)(m1 - m0) * ld);
  const ub_u32x4 rb = ub_desc(B + (size_t)n0 * ld, (uint64_t)(n1 - n0) * ld);
  const uint32_t base = ub_lds_addr(lds);
  uint32_t v[NL];
#pragma unroll
  for (int i = 0; i < NL; i++) {
    const int row = (i * NW + wave) * 8 + (lane >> 3);  // of A, then of B
    v[i] = (uint32_t)(row < BM ? row : row - BM) * (uint32_t)ld + 16 * ((lane & 7) ^ ((row >> 1) & 7));
  }
  auto issue = [&](int k, int slot) {
#pragma unroll
    for (int i = 0; i < NL; i++)
      ub_lds_load16_at(i * NW * 8 < BM ? ra : rb, base + slot * ST + (i * NW + wave) * 1024, v[i], (uint32_t)k * 128);
  };
  i32x16 acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; i++)
#pragma unroll
    for (int j = 0; j < TN; j++)
#pragma unroll
      for (int r = 0; r < 16; r++) acc[i][j][r] = 0;
  const int l32 = lane & 31, kh = lane >> 5;
  const int k0 = kp * part, nk = min(part, ld / 128 - k0);
  if constexpr (DT == kSum) y = (int*)y + (size_t)kp * M * N;
#pragma unroll
  for (int k = 0; k < NS - 1; k++) issue(k0 + min(k, nk - 1), k);  // (past K: loaded again, not used)
  int slot = 0;
  for (int k = 0; k < nk; k++) {
    ub_wait_vmcnt<(NS - 2) * NL>();  // step k has landed
    ub_barrier();                    // for everyone, and step k - 1 is read
    issue(k0 + min(k + NS - 1, nk - 1), slot == 0 ? NS - 1 : slot - 1);
    const uint8_t* st = lds + slot * ST;
    i32x4 af[TM][4], bf[TN][4];
#pragma unroll
    for (int q = 0; q < 4; q++) {
#pragma unroll
      for (int i = 0; i < TM; i++) {
        const int row = wm * 32 * TM + 32 * i + l32;
        af[i][q] = *(const i32x4*)(st + row * 128 + 16 * ((2 * q + kh) ^ ((row >> 1) & 7)));
      }
#pragma unroll
      for (int j = 0; j < TN; j++) {
        const int row = BM + wn * 32 * TN + 32 * j + l32;
        bf[j][q] = *(const i32x4*)(st + row * 128 + 16 * ((2 * q + kh) ^ ((row >> 1) & 7)));
      }
    }
#pragma unroll
    for (int q = 0; q < 4; q++)
#pragma unroll
      for (int j = 0; j < TN; j++)
#pragma unroll
        for (int i = 0; i < TM; i++)
          acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(bf[j][q], af[i][q], acc[i][j], 0, 0, 0);
    __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0): this step is read
    slot = slot == NS - 1 ? 0 : slot + 1;
  }
  ub_wait_vmcnt<0>();
  ub_barrier();
  typedef Epilogue<DT, TM, TN> Out;
  static_assert(NW * Out::kStage <= NS * ST, "epilogue fits");
  Out::run(acc, lds + wave * Out::kStage, sa, sw, bias, y, m1, n1, N, m0 + wm * 32 * TM, n0 + wn * 32 * TN);
}

template <int DT>
__global__ void __launch_bounds__(256) k_i8_sum(const int* __restrict__ part, const float* __restrict__ sa,
                                                const float* __restrict__ sw, const float* __restrict__ bias,
                                                void* __restrict__ y, int M, int N, int parts) {
  const unsigned i = blockIdx.x * 256u + threadIdx.x, all = (unsigned)M * (unsigned)N;
  if (i >= all) return;
  const unsigned m = i / (unsigned)N, n = i - m * (unsigned)N;
  const float a = sa[m], s = sw[n], b = bias ? bias[n] : 0.f;
  int v = 0;
#pragma unroll 8
  for (int p = 0; p < parts; p++) v += part[(size_t)p * all + i];
  put<DT>(y, i, v, a, s, b);
}

// ----------------------------------------------------------- few tokens
// Up to 16 tokens: HBM-bound, so shaped for bytes in flight.  A persistent grid
// of one 16-wavefront workgroup a CU walks tiles of 16 weight rows; the
// wavefronts split K in 64-byte steps (wavefront w the steps w, w + 16, ...),
// SP of which they load at once straight into registers, and the next SP are
// in flight while these are multiplied: v_mfma_i32_16x16x64_i8, tokens as A
// rows.  The codes of the activations lie in LDS for the whole launch, rows 16
// bytes further apart than they are long, so that the 16 rows of a fragment
// read spread over the banks.  Each workgroup makes them itself, while its first
// weight loads are on their way: a launch less, and quantizing M K values hides
// behind the stream.  The wavefronts' sums meet
// in LDS.
constexpr int DW = 16, kDecTiles = 64;  // wavefronts; tiles of a workgroup, at most

__device__ __forceinline__ __amdgpu_buffer_rsrc_t rsrc(const void* base, uint64_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, (int)bytes, 0x00020000);
}

template <int DT, int SP>
__global__ void __launch_bounds__(64 * DW) k_i8_dec(const void* __restrict__ x, const int8_t* __restrict__ W,
                                                    const float* __restrict__ sw, const float* __restrict__ bias,
                                                    void* __restrict__ y, int M, int K, int N, int ld) {
  constexpr int E = Elem<DT>::E, XU = 8;
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  int* red = (int*)lds;                       // [16 wavefronts][M][17]
  float* ssa = (float*)(red + DW * M * 17);   // [16]
  float* ssw = ssa + 16;                      // [1024]: the columns of all its tiles, and their bias
  float* sb = ssw + 16 * kDecTiles;
  uint8_t* a = (uint8_t*)(sb + 16 * kDecTiles);  // [M][ld + 16]
  const int tid = threadIdx.x, lane = tid & 63, r = lane & 15, h = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int steps = ld / 64, nc = (steps + DW * SP - 1) / (DW * SP), nt = (N + 15) / 16;
  const int pitch = ld + 16;
  const uint32_t row = (uint32_t)r * (uint32_t)ld + 16u * h;
  i32x4 b0[SP], b1[SP];
  // piece c of tile t; past the last tile or K: zeros
  auto load = [&](i32x4 (&b)[SP], int t, int c) {
    const int rows = t < nt ? min(16, N - 16 * t) : 0;
    const __amdgpu_buffer_rsrc_t rw = rsrc(W + (size_t)16 * min(t, nt - 1) * ld, (uint64_t)rows * ld);
#pragma unroll
    for (int i = 0; i < SP; i++) {
      const int s = (c * SP + i) * DW + wave;
      b[i] = __builtin_bit_cast(i32x4, __builtin_amdgcn_raw_buffer_load_b128(rw, (int)(s < steps ? row + 64u * s : 0x80000000u), 0, 0));
    }
  };
  // ---- codes: 16 / P wavefronts a row, P the power of two from M on.  A lane's
  // first XU units are asked for ahead of the weights (loads return in order)
  // and stay in registers; longer rows are read again.
  const int lg = M > 8 ? 0 : M > 4 ? 1 : M > 2 ? 2 : M > 1 ? 3 : 4;  // log2 of the wavefronts
  const int m = wave >> lg, u0 = ((wave & ((1 << lg) - 1)) << 6) + lane, us = 64 << lg;
  const typename Elem<DT>::T* p = (const typename Elem<DT>::T*)x + (size_t)min(m, M - 1) * K;
  const int V = K / E;
  uint4 xu[XU];
#pragma unroll
  for (int j = 0; j < XU; j++) xu[j] = unit<DT>(p, u0 + j * us, V);
  // the scales wait in LDS: asked for at the end of a tile, they would cost it
  // their latency and, loads returning in order, that of the weights in flight
  const int cn0 = 16 * ((int)blockIdx.x + (tid >> 4) * (int)gridDim.x) + (tid & 15);
  const float my_sw = cn0 < N ? sw[cn0] : 0.f, my_b = bias && cn0 < N ? bias[cn0] : 0.f;
  typename Elem<DT>::T behind[1] = {0};  // element V E + u0
  if (u0 < K - V * E) behind[0] = p[V * E + u0];
  int t = blockIdx.x, c = 0;  // the piece being multiplied
  auto next = [&](int& t, int& c) {
    if (++c == nc) {
      c = 0;
      t += gridDim.x;
    }
  };
  int tn = t, cn = c;
  load(b0, tn, cn);
  next(tn, cn);
  if constexpr (SP <= 4) {  // (no registers for the second set beside the activations' otherwise)
    load(b1, tn, cn);
    next(tn, cn);
  }
  {
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < XU; j++) top = top_of<DT>(xu[j], top);
    for (int i = u0 + XU * us; i < V; i += us) top = top_of<DT>(unit<DT>(p, i, V), top);
    top = max(top, __float_as_uint(ub_load<DT>(behind, 0)) & 0x7fffffffu);
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, o, 64));
    if (lane == 0) red[wave] = (int)top;
    ssw[tid] = my_sw;
    sb[tid] = my_b;
    __syncthreads();
    for (int w = 0; w < 1 << lg; w++) top = max(top, (uint32_t)red[(m << lg) + w]);
    __syncthreads();
    const float s = scale_of(top);
    const bool plain = plain_scale(s);
    const float rs = plain ? 0.f : __fdiv_rn(1.0f, s);
    if (lane == 0 && m < M) ssa[m] = s;
    auto store = [&](auto P, const uint4& v, int i) {
      if (i * E >= ld || i == V) return;  // (unit V: last)
      uint32_t o[E / 4];
      codes<DT, decltype(P)::value>(v, s, rs, o);
      if constexpr (E == 4) *(uint32_t*)(a + m * pitch + 4 * i) = o[0];
      else *(uint2*)(a + m * pitch + 8 * i) = make_uint2(o[0], o[1]);
    };
    auto rest = [&](auto P, int from) {
      for (int i = from; i * E < ld; i += us) store(P, unit<DT>(p, i, V), i);
      if (u0 < E && V * E < ld)
        a[m * pitch + V * E + u0] = (uint8_t)code<decltype(P)::value>(ub_load<DT>(behind, 0), s, rs);
    };
    if (m >= M) {
    } else if (plain) {
      rest(std::true_type{}, u0);
    } else {
#pragma unroll
      for (int j = 0; j < XU; j++) store(std::false_type{}, xu[j], u0 + j * us);
      rest(std::false_type{}, u0 + XU * us);
    }
  }
  if constexpr (SP > 4) {
    load(b1, tn, cn);
    next(tn, cn);
  }
  __syncthreads();
  i32x4 acc = {0, 0, 0, 0};
  int mine = 0;  // which of the workgroup's tiles
  const uint8_t* ar = a + min(r, M - 1) * pitch + 16 * h;  // (tokens past M: not used)
  auto work = [&](i32x4 (&b)[SP]) {
#pragma unroll
    for (int i = 0; i < SP; i++) {
      const int s = min((c * SP + i) * DW + wave, steps - 1);  // (past K: times zeros)
      acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(*(const i32x4*)(ar + 64 * s), b[i], acc, 0, 0, 0);
    }
    load(b, tn, cn);
    next(tn, cn);
    if (c == nc - 1) {
#pragma unroll
      for (int i = 0; i < 4; i++)
        if (4 * h + i < M) red[(wave * M + 4 * h + i) * 17 + r] = acc[i];
      acc = (i32x4){0, 0, 0, 0};
      __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0); the weight loads stay in flight
      ub_barrier();
      const int m = tid >> 4, n = 16 * t + (tid & 15);
      if (m < M) {
        int v = 0;
#pragma unroll
        for (int w = 0; w < DW; w++) v += red[(w * M + m) * 17 + (tid & 15)];
        if (n < N) put<DT>(y, (size_t)m * N + n, v, ssa[m], ssw[16 * mine + (tid & 15)], sb[16 * mine + (tid & 15)]);
      }
      __builtin_amdgcn_s_waitcnt(0xC07F);
      ub_barrier();
    }
    if (c == nc - 1) mine++;
    next(t, c);
  };
  while (t < nt) {
    work(b0);
    if (t >= nt) break;
    work(b1);
  }
}

// Every workgroup makes all the codes: past 64 KiB of them that costs more than the
// launch it saves.  us (M x K x N), k_i8_dec / the tiles: 16 x 4096 x 4096 10.4 / 11.4,
// 8 x 8192 x 8192 18.4 / 20.2, 4 x 14336 x 4096 17.2 / 18.4, then 12 x 8192 x 8192 23.9 /
// 20.4, 6 x 14336 x 4096 21.8 / 18.5, 4 x 28672 x 8192 54.8 / 49.1
constexpr int kDecCodes = 64 * 1024;
constexpr int kLds = 160 * 1024;  // of a CU
size_t dec_lds(int M, int ld) { return sizeof(int) * (DW * M * 17 + 16 + 32 * kDecTiles) + (size_t)M * (ld + 16); }

template <int DT, int SP>
void dec(const void* x, const int8_t* w, const float* sw, const float* bias, void* y, int M, int K, int N, int ld,
         hipStream_t s) {
  static UbLdsLimit limit;
  limit.raise((const void*)k_i8_dec<DT, SP>, kLds);
  const int nt = ub_cdiv(N, 16);
  k_i8_dec<DT, SP><<<nt < 256 ? nt : 256, 64 * DW, dec_lds(M, ld), s>>>(x, w, sw, bias, y, M, K, N, ld);
}
// SP: a wavefront's steps, evened out over as few pieces of at most eight
template <int DT>
void dec(const void* x, const int8_t* w, const float* sw, const float* bias, void* y, int M, int K, int N, int ld,
         hipStream_t s) {
  const int per = ub_cdiv(ld / 64, DW), sp = ub_cdiv(per, ub_cdiv(per, 8));
  if (sp <= 1) dec<DT, 1>(x, w, sw, bias, y, M, K, N, ld, s);
  else if (sp <= 2) dec<DT, 2>(x, w, sw, bias, y, M, K, N, ld, s);
  else if (sp <= 4) dec<DT, 4>(x, w, sw, bias, y, M, K, N, ld, s);
  else if (sp <= 6) dec<DT, 6>(x, w, sw, bias, y, M, K, N, ld, s);
  else dec<DT, 8>(x, w, sw, bias, y, M, K, N, ld, s);
}

template <int DT, int NT>
bool quant(const void* x, int8_t* q, float* sa, int M, int K, int ld, hipStream_t s) {
  const int nv = ub_cdiv(ld / Elem<DT>::E, NT);
  if (nv <= 1) k_quant<DT, NT, 1><<<M, NT, 0, s>>>(x, q, sa, K, ld);
  else if (nv <= 2) k_quant<DT, NT, 2><<<M, NT, 0, s>>>(x, q, sa, K, ld);
  else if (nv <= 4) k_quant<DT, NT, 4><<<M, NT, 0, s>>>(x, q, sa, K, ld);
  else if (nv <= 8) k_quant<DT, NT, 8><<<M, NT, 0, s>>>(x, q, sa, K, ld);
  else return false;
  return true;
}

// The tile and the number of K parts that take least, by the tile's measured
// time for 128 bytes of K (0.01 us) on a CU that has one workgroup of it, and for
// each of several (larger grids leave that many to a CU, side by side or in
// turn); parts cost a launch and their sums' way to memory and back.  us in a
// graph, with the quantizing launch, M x K x N on 256 x 256 / 128 x 128 / 64 x 128
// / 64 x 64 / 64 x 32: 64 x 4096 x 6144 32 / 23 / 19 / 15 / 13.7, 201 x 3520 x 9001
// 40 / 23 / 33 / 27 / 34, 512 x 4096 x 4096 36 / 26 / 22.3 / 22.3 / 30, 1024 x 2048 x
// 2048 25 / 18 / 16 / 15.5 / 21, 1024 x 4096 x 14336 74 / 97 / 97 / - / -; in parts,
// 40 x 13970 x 450 31 -> 13, 490 x 9272 x 361 32 -> 19.
struct Plan { int tile, parts; };
Plan plan_for(int M, int N, int nk) {
  static const struct { int m, n, one, each; bool parts; } t[5] = {
      {256, 256, 205, 205, false}, {128, 128, 64, 60, true}, {64, 128, 57, 50, false}, {64, 64, 32, 27, true},
      {64, 32, 30, 22, false}};
  Plan best = {0, 1};
  double least = 0;
  for (int i = 0; i < 5; i++) {
    const int64_t tiles = (int64_t)ub_cdiv(M, t[i].m) * ub_cdiv(N, t[i].n);
    for (int p = 1; p <= 32 && p <= nk; p *= 2) {
      if (p > 1 && (!t[i].parts || tiles * p > 1024 || (int64_t)M * N >= 1 << 26)) break;
      const int64_t per = (tiles * p + 255) / 256;
      double cost = per == 1 ? t[i].one : (double)per * t[i].each;
      if (i == 0 && per > 1 && tiles % 256 && tiles % 256 <= 128) cost -= 0.45 * t[i].each;  // (halves)
      cost *= ub_cdiv(nk, p);
      if (p > 1) cost += 400 + (double)M * N * 8 * p / 52e3;
      if ((i == 0 && p == 1) || cost < least) best = {i, p}, least = cost;
    }
  }
  return best;
}

template <int DT>
void gemm(Plan plan, const int8_t* q, const float* sa, const int8_t* w, const float* sw, const float* bias, void* y, int M,
          int N, int ld, hipStream_t s) {
  const int part = ub_cdiv(ld / 128, plan.parts);
#define UB_TILE(WM, WN, TM, TN, NS)                                                                      \
  {                                                                                                      \
    constexpr int lds = NS * 64 * 32 * (WM * TM + WN * TN);                                              \
    static UbLdsLimit limit;                                                                             \
    limit.raise((const void*)k_i8_gemm<DT, WM, WN, TM, TN, NS>, lds);                                    \
    const int tiles = ub_cdiv(M, 32 * WM * TM) * ub_cdiv(N, 32 * WN * TN), rest = tiles % 256;           \
    const int full = TM > 1 && tiles > 256 && rest <= 128 ? tiles - rest : tiles;                        \
    k_i8_gemm<DT, WM, WN, TM, TN, NS><<<2 * tiles - full, 64 * WM * WN, lds, s>>>(q, sa, w, sw, bias, y, M, N, ld, full); \
    return;                                                                                              \
  }
#define UB_RING(WM, WN, TM, TN, NS)                                                                      \
  {                                                                                                      \
    constexpr int lds = NS * 128 * 32 * (WM * TM + WN * TN);                                             \
    static UbLdsLimit limit;                                                                             \
    limit.raise((const void*)k_i8_ring<DT, WM, WN, TM, TN, NS>, lds);                                    \
    k_i8_ring<DT, WM, WN, TM, TN, NS><<<ub_cdiv(M, 32 * WM * TM) * ub_cdiv(N, 32 * WN * TN) * ub_cdiv(ld / 128, part), \
                                        64 * WM * WN, lds, s>>>(q, sa, w, sw, bias, y, M, N, ld, part);  \
    return;                                                                                              \
  }
  if (plan.tile == 1) UB_RING(2, 4, 2, 1, 4)
  if (plan.tile == 3) UB_RING(2, 2, 1, 1, 4)
  if constexpr (DT != kSum) {
    if (plan.tile == 0) UB_TILE(2, 4, 4, 2, 4)
    if (plan.tile == 2) UB_TILE(2, 2, 1, 2, 6)
    UB_TILE(2, 1, 1, 1, 8)
  }
#undef UB_TILE
#undef UB_RING
}

template <int DT>
int linear(const char* nm, const void* x, const int8_t* w, const float* sw, const float* bias, void* y, int M, int K,
           int N, int ld, hipStream_t s) {
  if (M <= 16 && M * ld <= kDecCodes && N <= 256 * 16 * kDecTiles) {
    dec<DT>(x, w, sw, bias, y, M, K, N, ld, s);
    return UB_OK;
  }
  const Plan plan = plan_for(M, N, ld / 128);
  const int parts = ub_cdiv(ld / 128, ub_cdiv(ld / 128, plan.parts));  // (none empty)
  const size_t sums = parts > 1 ? sizeof(int) * parts * (size_t)M * N : 0;
  UbScratch ws(s, (size_t)M * ld + sizeof(float) * (size_t)M + sums);
  int8_t* q = (int8_t*)ws.get();
  if (!q) return ub_set_error(UB_ERR_LAUNCH, "%s: no workspace", nm);
  float* sa = (float*)(q + (size_t)M * ld);
  if (!((M >= 512 || ld <= 2048) && quant<DT, 256>(x, q, sa, M, K, ld, s)) && !quant<DT, 1024>(x, q, sa, M, K, ld, s))
    k_quant<DT, 1024, 0><<<M, 1024, 0, s>>>(x, q, sa, K, ld);
  if (parts > 1) {
    int* part = (int*)(sa + M);
    gemm<kSum>(plan, q, sa, w, sw, bias, part, M, N, ld, s);
    k_i8_sum<DT><<<ub_cdiv((long)M * N, 256), 256, 0, s>>>(part, sa, sw, bias, y, M, N, parts);
  } else {
    gemm<DT>(plan, q, sa, w, sw, bias, y, M, N, ld, s);
  }
  return UB_OK;
}

}  // namespace

UB_API int ubridge_int8_linear(const void* x, int dtype, const int8_t* w, const float* sw,
                               const float* bias, void* y, int M, int K, int N, int ld,
                               void* stream) {
  const char* nm = "ubridge_int8_linear";
  UB_REQUIRE(dtype == UB_F32 || dtype == UB_F16 || dtype == UB_BF16, "%s: dtype %d", nm, dtype);
  UB_REQUIRE(M >= 0 && N >= 0 && K > 0 && K <= 132104, "%s: M=%d K=%d (1..132104) N=%d", nm, M, K, N);
  UB_REQUIRE(ld >= K && ld % 128 == 0 && ld <= 132224, "%s: ld=%d (a multiple of 128, at least K=%d)", nm, ld, K);
  if ((size_t)M * N == 0) return UB_OK;
  UB_REQUIRE(x && w && sw && y, "%s: null pointer", nm);
  UB_REQUIRE(((uintptr_t)w & 15) == 0, "%s: weight not 16-byte aligned", nm);
  UB_REQUIRE(M < 1 << 22 && (int64_t)M * N < 1ll << 38, "%s: M=%d N=%d", nm, M, N);  // (2^32 threads a launch)
  hipStream_t s = ub_stream(stream);
  const int e = dtype == UB_F32   ? linear<UB_F32>(nm, x, w, sw, bias, y, M, K, N, ld, s)
                : dtype == UB_F16 ? linear<UB_F16>(nm, x, w, sw, bias, y, M, K, N, ld, s)
                                  : linear<UB_BF16>(nm, x, w, sw, bias, y, M, K, N, ld, s);
  return e ? e : ub_check_launch(nm);
}
