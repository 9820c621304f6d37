// mx.hip -- microscaled blocks (mx_dev.h) and their linear on gfx950:
//
//   y[m, n] = T( sum_b 2^(ea[m, b] + ew[n, b]) sum_{k in b} a[m, k] w[n, k] + bias[n] )
//
// over blocks b of 32 along K; w e2m1, a e2m1 or e4m3, x rounded to blocks by the
// call.  The products are exact, the sums f32 in the matrix instructions
// (v_mfma_scale_f32_{32x32x64,16x16x128}_f8f6f4, which take the two powers of two a
// block with the operands), and y is rounded once.
//
// Of e4m3 the matrix unit aligns the products of neighbouring elements to the largest
// exponent among them and drops what lies more than 13 bits below it (measured: 2^-9
// is kept beside 2^4 and lost beside 2^5; e2m1's own products span less): up to 2^-10 of
// the sum of magnitudes, where large values cancel more than a result's rounding, 6e-6
// of it on values like hidden states.  So a is cut in two by magnitude, at 2, and
// multiplied twice (X, kSide, kTurn, kCut below): either part's products lie within 14
// bits, and nothing is dropped.  A caller may take one product instead (one_product) for
// 16-bit results of more than 16 tokens, where the second costs most: 4096 x 4096 x 14336
// (M K N) 300 us against 195, 201 x 3520 x 9001 19 against 16.
//
// Rows are padded with zero codes to a step of 128 elements.  Outside, codes and
// scales lie in rows; a weight is laid out once, activations by the kernel that
// rounds them, as [16 rows][step][row][bytes of the step], so that a load
// instruction of 64 lanes reads 1 KiB of consecutive memory, and the scales' four
// bytes a step as one word, [16 rows][step][row].
#include "lds_dma.h"
#include "mx_dev.h"

#include <type_traits>

namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int kSum = 100;  // "type" of the f32 sums over a part of K

// bytes of a row's step of 128 elements
template <int F> constexpr int kRowStep = 128 * F / 8;

// Places of block b of a row, in rows or laid out for the products (TWO: in two parts, the
// lower kLower bytes behind the higher, in every 16 rows of a step).
constexpr int kLower = 16 * kRowStep<MX_FP8>;
template <int F, bool PACKED, bool TWO = false>
__device__ __forceinline__ size_t code_at(size_t row, int b, int nk) {
  if constexpr (PACKED) return (((row >> 4) * nk + (b >> 2)) * (TWO ? 32 : 16) + (row & 15)) * kRowStep<F> + (b & 3) * (kRowStep<F> / 4);
  else return row * (size_t)nk * kRowStep<F> + (size_t)b * (kRowStep<F> / 4);
}
template <bool PACKED>
__device__ __forceinline__ size_t scale_at(size_t row, int b, int nk) {
  if constexpr (PACKED) return (((row >> 4) * nk + (b >> 2)) * 16 + (row & 15)) * 4 + (b & 3);
  else return row * (size_t)nk * 4 + b;
}

// e4m3 codes of magnitude 2 and more in `hi`, those below in `lo` (bit 6 of a code
// tells), zeros elsewhere.  v_perm fills bytes with the sign of bytes 1 and 3 of either
// operand: of v << 9 (codes 0 and 2) and of v << 1 (1 and 3).
__device__ __forceinline__ uint32_t cut(uint32_t v, uint32_t& lo) {
  const uint32_t m = __builtin_amdgcn_perm(v << 1, v << 9, 0x0b090a08u);
  lo = v & ~m;
  return v & m;
}
__device__ __forceinline__ void cut(const i32x8& v, i32x8& lo, i32x8& hi) {
#pragma unroll
  for (int i = 0; i < 8; i++) {
    uint32_t l;
    hi[i] = (int)cut((uint32_t)v[i], l);
    lo[i] = (int)l;
  }
}

// ------------------------------------------------------- blocks and back
// A thread takes two units of 16 bytes of x, 256 apart, both loaded before the first is
// rounded; the 4 (f32: 8) lanes of a block find its largest by DPP.  us, bf16 to e2m1 laid
// out, 1 / 2 / 4 units a thread: 201 x 3520 3.6 / 3.6 / 3.7, 4096 x 4096 9.4 / 9.7 / 9.9,
// and in rows 14336 x 4096 27.9 / 26.2 / 26.5 (5.7 TB/s).
// TWO: codes of e4m3 in their two parts (`cut`).
template <int DT, int F, bool PACKED, bool TWO>
__global__ void __launch_bounds__(256) k_mx_quant(const void* __restrict__ x, uint8_t* __restrict__ q,
                                                  uint8_t* __restrict__ sc, uint32_t units, int C, int nk) {
  typedef typename MxElem<DT>::T T;
  constexpr int E = MxElem<DT>::E, BL = 32 / E, U = 2;
  const uint32_t per = (uint32_t)nk * (128 / E);  // units a row
  uint4 v[U];
  const uint32_t i0 = blockIdx.x * (256u * U) + threadIdx.x;
#pragma unroll
  for (int j = 0; j < U; j++) {
    const uint32_t i = i0 + j * 256;
    v[j] = make_uint4(0, 0, 0, 0);
    if (i < units) {
      const uint32_t row = i / per;
      v[j] = mx_unit_at<DT>((const T*)x + (size_t)row * C, (int)(i - row * per), C);
    }
  }
#pragma unroll
  for (int j = 0; j < U; j++) {
    const uint32_t i = i0 + j * 256;
    uint32_t o[2];
    const uint32_t b = mx_round<DT, F>(v[j], o);
    if (i >= units) continue;  // (whole blocks: units is a multiple of theirs)
    const uint32_t row = i / per;
    const int u = (int)(i - row * per), blk = u / BL;
    uint8_t* p = q + code_at<F, PACKED, TWO>(row, blk, nk) + (u % BL) * (E * F / 8);
    if constexpr (TWO) {
      uint32_t lo[2];
      o[0] = cut(o[0], lo[0]), o[1] = cut(o[1], lo[1]);
      mx_store<DT, F>(p + kLower, lo);
    }
    mx_store<DT, F>(p, o);
    if (u % BL == 0) sc[scale_at<PACKED>(row, blk, nk)] = (uint8_t)b;
  }
}

// A thread takes 8 elements.
template <int DT, int F>
__global__ void __launch_bounds__(256) k_mx_back(const uint8_t* __restrict__ q, const uint8_t* __restrict__ sc,
                                                 void* __restrict__ y, uint32_t units, int C, int nk) {
  typedef typename MxElem<DT>::T T;
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  constexpr int E = MxElem<DT>::E;
  const uint32_t per = (uint32_t)(C + 7) / 8, i = blockIdx.x * 256u + threadIdx.x;
  if (i >= units) return;
  const uint32_t row = i / per;
  const int u = (int)(i - row * per);
  const uint8_t* p = q + code_at<F, false>(row, u / 4, nk) + (u & 3) * F;
  const uint32_t b = sc[scale_at<false>(row, u / 4, nk)];
  float f[8];
  if constexpr (F == MX_FP4) {
    const uint32_t w = *(const uint32_t*)p;
#pragma unroll
    for (int e = 0; e < 4; e++) {
      f32x2 v;
      if (e == 0) v = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.f, 0);
      else if (e == 1) v = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.f, 1);
      else if (e == 2) v = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.f, 2);
      else v = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.f, 3);
      f[2 * e] = v[0], f[2 * e + 1] = v[1];
    }
  } else {
    const uint2 w = *(const uint2*)p;
#pragma unroll
    for (int e = 0; e < 4; e++) {
      const int d = (int)(e < 2 ? w.x : w.y);
      const f32x2 v = e & 1 ? __builtin_amdgcn_cvt_pk_f32_fp8(d, true) : __builtin_amdgcn_cvt_pk_f32_fp8(d, false);
      f[2 * e] = v[0], f[2 * e + 1] = v[1];
    }
  }
  const float s = b == 255 ? __builtin_nanf("") : mx_unit(b);
#pragma unroll
  for (int e = 0; e < 8; e++) f[e] *= s;
#pragma unroll
  for (int h = 0; h < 8 / E; h++) mx_put<DT>((T*)y + (size_t)row * C, u * (8 / E) + h, C, mx_pack<DT>(f + h * E));
}

// From rows to the products' layout; rows past R up to a multiple of 16 are zero.
template <int F, bool TWO = false>
__global__ void __launch_bounds__(256) k_mx_pack(const uint8_t* __restrict__ q, const uint8_t* __restrict__ sc,
                                                 uint8_t* __restrict__ pq, uint32_t* __restrict__ ps, uint32_t units, int R,
                                                 int nk) {
  constexpr int UR = kRowStep<F> / 16;  // 16-byte units of a row's step
  const uint32_t i = blockIdx.x * 256u + threadIdx.x;  // of the result
  if (i >= units) return;
  const uint32_t rs = i / UR;  // (16 rows, step, row)
  const int u = (int)(i % UR), r = (int)(rs & 15);
  const uint32_t gs = rs >> 4, g = gs / (uint32_t)nk, s = gs - g * nk;
  const size_t row = (size_t)g * 16 + r;
  uint4 v = make_uint4(0, 0, 0, 0);
  uint32_t w = 0;
  if (row < (size_t)R) {
    __builtin_memcpy(&v, q + (row * nk + s) * kRowStep<F> + 16 * u, 16);
    if (u == 0) __builtin_memcpy(&w, sc + (row * nk + s) * 4, 4);
  }
  uint4* p = (uint4*)pq + (TWO ? i + (i / (16 * UR)) * (16 * UR) : i);
  if constexpr (TWO) {
    uint4 lo;
    v = make_uint4(cut(v.x, lo.x), cut(v.y, lo.y), cut(v.z, lo.z), cut(v.w, lo.w));
    p[kLower / 16] = lo;
  }
  *p = v;
  if (u == 0) ps[rs] = w;
}

// ------------------------------------------------------------------ tiles
struct MxArgs {
  const uint8_t *a, *w;    // laid out for the products
  const uint32_t *sa, *sw;
  const float* bias;
  void* y;
  int M, N, nk, part;      // steps of K in all, and of a part
};

// e4m3 activations on the tiles: one product; two parts, cut by each wavefront; or two
// parts in memory, on tiles of 32 rows, which four wavefronts would cut again each, 7 of
// 23 us of 201 x 3520 x 9001: cut / in memory 23.1 / 19.5, 64 x 4096 x 6144 18.5 / 14.7 (64
// x 64 tiles 18.8 / 20.3, 128 x 128 30.3 / 29.1).
enum { kOne, kCuts, kParts };

__device__ __forceinline__ i32x8 wide(const i32x4& v) { return __builtin_shufflevector(v, v, 0, 1, 2, 3, -1, -1, -1, -1); }
// Outputs of a wavefront, 32 TM x 32 TN, through its part of LDS in rows, so that
// a store instruction writes whole runs of a row.  The weights are the products'
// left operand: lane (c, kh) holds row m = c and columns 8 q + 4 kh .. + 3 of a 32 x
// 32 tile, four to an LDS write.
template <int DT, int TM, int TN>
struct MxOut {
  typedef std::conditional_t<DT == kSum || DT == UB_F32, float, uint16_t> T;
  static constexpr int E = 16 / sizeof(T), kPitch = 32 * TN * sizeof(T) + 16, kStage = 32 * kPitch;
  static __device__ __forceinline__ void run(const f32x16 (&acc)[TM][TN], uint8_t* st, const float* bias, void* y, int M,
                                             int N, int pitch, int m0, int n0) {
    constexpr int LR = 32 * TN / E, RI = 64 / LR;  // lanes a row, rows an instruction
    const int lane = threadIdx.x & 63, c = lane & 31, kh = lane >> 5;
    float b[TN][16];
#pragma unroll
    for (int j = 0; j < TN; j++)
#pragma unroll
      for (int r = 0; r < 16; r++) {
        const int n = min(n0 + 32 * j + 8 * (r >> 2) + 4 * kh + (r & 3), N - 1);
        b[j][r] = DT != kSum && bias ? bias[n] : 0.f;
      }
#pragma unroll
    for (int i = 0; i < TM; i++) {
#pragma unroll
      for (int j = 0; j < TN; j++)
#pragma unroll
        for (int q = 0; q < 4; q++) {
          float f[4];
          T v[4];
#pragma unroll
          for (int e = 0; e < 4; e++) f[e] = acc[i][j][4 * q + e] + b[j][4 * q + e];
#pragma unroll
          for (int e = 0; e < 4; e++) {
            if constexpr (sizeof(T) == 4) v[e] = f[e];
            else ub_store<DT>(v, e, f[e]);
          }
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

// WM x WN wavefronts of 32 TM x 32 TN outputs, 128 elements of K a step.  Codes and
// scale words reach LDS by direct loads into a ring of NS steps, NS - 1 in flight.
// A row's step is 4 (e4m3: 8) units of 16 bytes, unit u of row r at u ^ ((r >> 2) &
// 3) (u ^ ((r >> 1) & 7)), so that the rows of a fragment read lie in distinct
// banks.  A step is two products deep: lane (c, kh) takes blocks 2 kh + j of its
// rows in product j (of e4m3, whose operand holds 16 bytes of either lane half's
// block, bytes 16 kh .. of blocks j and 2 + j), and its scale is byte j of the row's
// word shifted by 16 kh.  Fragments are in registers, two sets: those of one
// product are read while the other's multiply.
// Measured, e2m1 x e2m1, 4096 x 4096 x 14336 (M K N): 141 us at best, 3.4 PFLOP/s (3.9 at 8192^3),
// among other work up to 171; with e4m3 activations 187, in two parts 290.  From registers the unit reaches 7.7: the clock falls to 1.9 GHz, the
// fill of LDS alone takes two thirds of the time (17 TB/s out of L2), its reads and the
// products as long each.  Small tiles are bound by that fill: 201 x 3520 x 9001 with e4m3
// 14.6 us, 176 MB.
template <int F, int DT, int X, int WM, int WN, int TM, int TN, int NS, int OCC>
__global__ void __launch_bounds__(64 * WM * WN) __attribute__((amdgpu_waves_per_eu(OCC, OCC))) k_mx_gemm(MxArgs a) {
  constexpr int BM = 32 * WM * TM, BN = 32 * WN * TN, NW = WM * WN, RB = kRowStep<F>;
  constexpr int PA = X == kParts ? 2 : 1, CA = PA * BM * RB / 1024, CB = BN * 64 / 1024;  // parts of a; chunks of 1 KiB
  constexpr int NL = (CA + CB + NW - 1) / NW;                                           // load instructions
  constexpr int SAR = BM < 64 ? 64 : BM, SL = ((SAR + BN) / 64 + NW - 1) / NW;           // and of scales
  constexpr int SO = NL * NW * 1024, ST = SO + SL * NW * 256;  // offset of the scales; bytes of a step
  typedef MxOut<DT, TM, TN> Out;
  static_assert(BN % 64 == 0 && NW * Out::kStage <= NS * ST, "epilogue fits");
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / WN, wn = wave % WN, nk = a.nk;
  int tile_m, tile_n;
  const int tm = (a.M + BM - 1) / BM, tn = (a.N + BN - 1) / BN;
  const int id = ub_xcd_run((int)blockIdx.x, (int)gridDim.x), kp = id / (tm * tn);  // part kp of K
  ub_tile_at(id - kp * tm * tn, 0, tm, tn, 8, tile_m, tile_n);
  const int m0 = tile_m * BM, n0 = tile_n * BN;
  // groups of 16 rows past the end lie past the buffers: zeros
  const int gm = min(BM, a.M - m0 + 15) / 16, gn = min(BN, a.N - n0 + 15) / 16;
  const ub_u32x4 ra = ub_desc(a.a + (size_t)(m0 / 16) * nk * 16 * RB * PA, (uint64_t)gm * nk * 16 * RB * PA);
  const ub_u32x4 rb = ub_desc(a.w + (size_t)(n0 / 16) * nk * 1024, (uint64_t)gn * nk * 1024);
  const ub_u32x4 rsa = ub_desc(a.sa + (size_t)(m0 / 16) * nk * 16, (uint64_t)gm * nk * 64);
  const ub_u32x4 rsb = ub_desc(a.sw + (size_t)(n0 / 16) * nk * 16, (uint64_t)gn * nk * 64);
  const uint32_t base = ub_lds_addr(lds);
  uint32_t v[NL], vs[SL];
#pragma unroll
  for (int i = 0; i < NL; i++) {
    const int c = i * NW + wave;  // chunk of 1 KiB: A's, then the weight's, then none
    const int r4 = lane >> 2, u4 = (lane & 3) ^ ((r4 >> 2) & 3);
    if (c < CA && F == MX_FP8) {  // (in LDS all rows' higher parts, then the lower)
      const int p = c * PA / CA, cr = c - p * (CA / PA);
      const int r = 8 * (cr & 1) + (lane >> 3), u = (lane & 7) ^ ((r >> 1) & 7);
      v[i] = (uint32_t)(cr >> 1) * nk * 2048 * PA + p * kLower + r * 128 + u * 16;
    } else {
      v[i] = c < CA + CB ? (uint32_t)(c < CA ? c : c - CA) * nk * 1024 + r4 * 64 + u4 * 16 : kDmaOOB;
    }
  }
#pragma unroll
  for (int i = 0; i < SL; i++) {
    const int row = (i * NW + wave) * 64 + lane, rr = row < SAR ? row : row - SAR;
    vs[i] = row < SAR + BN ? (uint32_t)(rr >> 4) * nk * 64 + (rr & 15) * 4 : kDmaOOB;
  }
  auto issue = [&](int k, uint32_t off) {
#pragma unroll
    for (int i = 0; i < NL; i++) {
      const int c = i * NW + wave;
      ub_lds_load16_at(c < CA ? ra : rb, base + off + c * 1024, v[i], (uint32_t)k * (c < CA ? 16 * RB * PA : 1024));
    }
#pragma unroll
    for (int i = 0; i < SL; i++) {
      const int c = i * NW + wave;
      ub_lds_load4_at(c * 64 < SAR ? rsa : rsb, base + off + SO + c * 256, vs[i], (uint32_t)k * 64);
    }
  };
  f32x16 acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; i++)
#pragma unroll
    for (int j = 0; j < TN; j++)
#pragma unroll
      for (int r = 0; r < 16; r++) acc[i][j][r] = 0.f;
  const int l32 = lane & 31, kh = lane >> 5;
  i32x4 wf[2][TN], af[2][TM], ag[2][TM];  // (ag: the second half of e4m3)
  i32x4 lf[X == kParts ? 2 : 1][TM], lg[X == kParts ? 2 : 1][TM];  // (of the lower parts)
  uint32_t sw[TN], sa[TM], sw2[TN], sa2[TM];
  auto read_frags = [&](uint32_t off, auto J) {
    constexpr int j = decltype(J)::value;
    const uint8_t* pw = lds + off + CA * 1024 + (wn * 32 * TN + l32) * 64 + (((2 * kh + j) ^ ((l32 >> 2) & 3)) * 16);
#pragma unroll
    for (int n = 0; n < TN; n++) wf[j][n] = *(const i32x4*)(pw + n * 32 * 64);
    if constexpr (F == MX_FP4) {
      const uint8_t* pa = lds + off + (wm * 32 * TM + l32) * 64 + (((2 * kh + j) ^ ((l32 >> 2) & 3)) * 16);
#pragma unroll
      for (int m = 0; m < TM; m++) af[j][m] = *(const i32x4*)(pa + m * 32 * 64);
    } else {
      const uint8_t* pa = lds + off + (wm * 32 * TM + l32) * 128;
      const int u0 = ((2 * j + kh) ^ ((l32 >> 1) & 7)) * 16, u1 = ((4 + 2 * j + kh) ^ ((l32 >> 1) & 7)) * 16;
#pragma unroll
      for (int m = 0; m < TM; m++) {
        af[j][m] = *(const i32x4*)(pa + m * 32 * 128 + u0);
        ag[j][m] = *(const i32x4*)(pa + m * 32 * 128 + u1);
        if constexpr (X == kParts) {
          lf[j][m] = *(const i32x4*)(pa + CA * 512 + m * 32 * 128 + u0);
          lg[j][m] = *(const i32x4*)(pa + CA * 512 + m * 32 * 128 + u1);
        }
      }
    }
  };
  auto read_scales = [&](uint32_t off) {
    const uint8_t* p = lds + off + SO;
#pragma unroll
    for (int n = 0; n < TN; n++) sw2[n] = *(const uint32_t*)(p + (SAR + wn * 32 * TN + n * 32 + l32) * 4);
#pragma unroll
    for (int m = 0; m < TM; m++) sa2[m] = *(const uint32_t*)(p + (wm * 32 * TM + m * 32 + l32) * 4);
  };
  auto take_scales = [&]() {
#pragma unroll
    for (int n = 0; n < TN; n++) sw[n] = sw2[n] >> (16 * kh);
#pragma unroll
    for (int m = 0; m < TM; m++) sa[m] = sa2[m] >> (16 * kh);
  };
  auto mul = [&](auto J) {
    constexpr int j = decltype(J)::value;
    auto add = [&](int m, int n, const i32x8& v) {
      acc[m][n] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(wide(wf[j][n]), v, acc[m][n], 4, F == MX_FP4 ? 4 : 0, j,
                                                                  (int)sw[n], j, (int)sa[m]);
    };
    auto act = [&](int m) {
      if constexpr (F == MX_FP4) return wide(af[j][m]);
      else return __builtin_shufflevector(af[j][m], ag[j][m], 0, 1, 2, 3, 4, 5, 6, 7);
    };
    if constexpr (X != kOne) {
#pragma unroll
      for (int m = 0; m < TM; m++) {  // (cut once for all columns)
        i32x8 lo, hi;
        if constexpr (X == kCuts) cut(act(m), lo, hi);
        else lo = __builtin_shufflevector(lf[j][m], lg[j][m], 0, 1, 2, 3, 4, 5, 6, 7), hi = act(m);
#pragma unroll
        for (int n = 0; n < TN; n++) add(m, n, lo);
#pragma unroll
        for (int n = 0; n < TN; n++) add(m, n, hi);
      }
    } else {
#pragma unroll
      for (int n = 0; n < TN; n++)
#pragma unroll
        for (int m = 0; m < TM; m++) add(m, n, act(m));
    }
  };
  constexpr int PW = NL + SL;  // loads of a step in a wavefront
  const int k0 = kp * a.part, n = min(a.part, nk - k0);
  void* y = a.y;
  if constexpr (DT == kSum) y = (float*)y + (size_t)kp * a.M * a.N;
  auto step_of = [&](int k) { return k0 + min(k, n - 1); };  // (past the part: loaded again, not used)
#pragma unroll
  for (int k = 0; k < NS; k++) issue(step_of(k), k * ST);
  ub_wait_vmcnt<(NS - 1) * PW>();
  ub_barrier();
  read_frags(0, std::integral_constant<int, 0>{});
  read_scales(0);
  uint32_t off = 0;
  // LDS reads early among the products, so that they are back when those are done
  auto spread = [&]() {
    __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);  // 2 DS reads
#pragma unroll
    for (int q = 0; q < TM * TN; q++) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);  // 1 MFMA
      __builtin_amdgcn_sched_group_barrier(0x100, 3, 0);
    }
    __builtin_amdgcn_sched_barrier(0);
  };
  for (int k = 0; k < n; k++) {
    __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0): the first product's fragments
    take_scales();
    read_frags(off, std::integral_constant<int, 1>{});
    mul(std::integral_constant<int, 0>{});
    spread();
    __builtin_amdgcn_s_waitcnt(0xC07F);  // the second product's: this step is read
    ub_wait_vmcnt<(NS - 2) * PW>();      // the next step has landed
    ub_barrier();
    issue(step_of(k + NS), off);
    off = off == (NS - 1) * ST ? 0 : off + ST;
    read_frags(off, std::integral_constant<int, 0>{});  // (after the last step: not used)
    read_scales(off);
    mul(std::integral_constant<int, 1>{});
    spread();
  }
  __builtin_amdgcn_s_waitcnt(0xC07F);
  ub_wait_vmcnt<0>();
  ub_barrier();
  Out::run(acc, lds + wave * Out::kStage, a.bias, y, a.M, a.N, a.N, m0 + wm * 32 * TM, n0 + wn * 32 * TN);
}

template <int DT>
__global__ void __launch_bounds__(256) k_mx_sum(const float* __restrict__ part, const float* __restrict__ bias,
                                                void* __restrict__ y, int64_t all, int N, int parts) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= all) return;
  float v = 0.f;
#pragma unroll 8
  for (int p = 0; p < parts; p++) v += part[p * all + i];
  ub_store<DT>(y, i, v + (bias ? bias[i % N] : 0.f));
}

// ----------------------------------------------------------- few tokens
// Up to 16 tokens: a stream of the weight.  A workgroup of 16 wavefronts takes
// `tiles` tiles of 16 weight rows at once, ks wavefronts to a tile, each a run of
// its steps: the tile's codes are consecutive in memory, and so are a wavefront's.
// Weights go straight to the registers of v_mfma_scale_f32_16x16x128 as its left
// operand, 2 P steps in flight; lane (r, h) holds block h of row r, and ends with
// columns 4 h .. + 3 of token r.  The activations' codes (of e4m3 both parts, where they
// fit) lie in LDS for the whole launch (rows 16 bytes further apart than they are long,
// for the banks); each workgroup makes them itself while its first weights are on their
// way, up to kRound values; beyond, a launch of its own makes them once.  The wavefronts'
// sums meet in LDS in their order.
// HBM bounds it where the weight is large, launch and first latency else.  us of a call
// among others with codes that are there, e2m1 / e4m3 (M x K x N): 1 x 14336 x 4096 7.5 / 8.2 (31 MB, 4 TB/s), 8 x 4096 x 28672
// 11.0 / 11.5 (64 MB, 5.8 TB/s), 16 x 4096 x 28672 11.4 / 13.6 (one product alone 11.8).
constexpr int DW = 16, RP = 20;  // wavefronts; floats of a token's row of sums

struct MxDecArgs {
  const void* x;             // T [M, K], or null: codes and scales in rows
  const uint8_t *q, *qs, *w;
  const uint32_t* sw;
  const float* bias;
  void* y;
  int M, K, N, nk, tiles, ks, per;  // per: steps of a wavefront
};

// Where the two parts of e4m3 activations (`cut`) are: of e2m1 none; cut in registers by
// every wavefront; or both in LDS, and multiplied as columns 0-7 and 8-15 of one product
// (up to 8 tokens), or in turn.  us, 16 x 4096 x 28672, in turn / in registers: 13.6 / 16.9.
enum { kWhole, kCut, kSide, kTurn };

template <int F, int DT, bool PRE, int PARTS>
__global__ void __launch_bounds__(64 * DW) k_mx_dec(MxDecArgs a) {
  typedef typename MxElem<DT>::T T;
  constexpr int E = MxElem<DT>::E, BL = 32 / E, XU = 8, P = 4, RB = kRowStep<F>;
  constexpr bool TWO = PARTS == kSide || PARTS == kTurn;
  static_assert((PARTS == kWhole) == (F == MX_FP4), "the parts of e4m3");
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  const int tid = threadIdx.x, lane = tid & 63, r = lane & 15, h = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int nk = a.nk, M = a.M, pitch = nk * RB + 16, spitch = nk * 4 + 4;
  float* red = (float*)lds;                       // [16 wavefronts][16 tokens][RP]
  uint8_t* ac = lds + sizeof(float) * DW * 16 * RP;  // codes [M][pitch], TWO: the lower parts behind them
  uint8_t* as = ac + (TWO ? 2 : 1) * M * pitch;  // scale bytes [M][spitch]
  const int nt = (a.N + 15) / 16, tl = wave / a.ks, kp = wave - tl * a.ks;
  const int s0 = kp * a.per, s1 = min(nk, s0 + a.per);
  const int pieces = (a.per + P - 1) / P;
  const bool idle = tl >= a.tiles;
  // ---- the activations' first units, ahead of the weights (loads return in order)
  const uint32_t per = (uint32_t)nk * (128 / E);
  const uint32_t units = PRE ? (uint32_t)M * nk * (RB / 16) : M * per;
  uint4 xu[XU];
#pragma unroll
  for (int j = 0; j < XU; j++) {
    const uint32_t i = tid + j * 64 * DW;
    xu[j] = make_uint4(0, 0, 0, 0);
    if (i < units) {
      if constexpr (PRE) {
        xu[j] = ((const uint4*)a.q)[i];
      } else {
        const uint32_t row = i / per;
        xu[j] = mx_unit_at<DT>((const T*)a.x + (size_t)row * a.K, i - row * per, a.K);
      }
    }
  }
  typedef i32x4 Set[P];
  typedef uint32_t Scales[P];
  // piece c of the wavefront's run in the workgroup's round at `group`; past it: zeros
  auto load = [&](Set& b, Scales& sc, int group, int c) {
    const int t = group * a.tiles + tl;
    const bool any = !idle && t < nt;
    const uint8_t* w = a.w + (size_t)(any ? t : 0) * nk * 1024;
    const uint8_t* sw = (const uint8_t*)(a.sw + (size_t)(any ? t : 0) * nk * 16);
#pragma unroll
    for (int i = 0; i < P; i++) {
      const int s = s0 + c * P + i;
      b[i] = (i32x4){0, 0, 0, 0};
      sc[i] = 0;
      if (any && s < s1) {  // (the same in every lane)
        b[i] = __builtin_nontemporal_load((const i32x4*)(w + (size_t)s * 1024 + r * 64 + h * 16));
        sc[i] = sw[s * 64 + r * 4 + h];
      }
    }
  };
  const int rounds = (nt + a.tiles - 1) / a.tiles;  // groups of tiles in all
  int g = blockIdx.x, c = 0, gn = g, cn = 0;
  auto next = [&](int& g, int& c) {
    if (++c == pieces) {
      c = 0;
      g += gridDim.x;
    }
  };
  Set b0, b1;
  Scales c0, c1;
  load(b0, c0, gn, cn);
  next(gn, cn);
  load(b1, c1, gn, cn);
  next(gn, cn);
  if constexpr (PRE) {
    constexpr int UR = RB / 16;
    const uint32_t rowu = (uint32_t)nk * UR;
    auto put = [&](const uint4& v, uint32_t i) {
      const uint32_t row = i / rowu;
      uint8_t* p = ac + row * pitch + (i - row * rowu) * 16;
      if constexpr (TWO) {
        uint4 lo;
        *(uint4*)p = make_uint4(cut(v.x, lo.x), cut(v.y, lo.y), cut(v.z, lo.z), cut(v.w, lo.w));
        *(uint4*)(p + M * pitch) = lo;
      } else {
        *(uint4*)p = v;
      }
    };
#pragma unroll
    for (int j = 0; j < XU; j++)
      if (tid + j * 64 * DW < units) put(xu[j], tid + j * 64 * DW);
    for (uint32_t i = tid + XU * 64 * DW; i < units; i += 64 * DW) put(((const uint4*)a.q)[i], i);
    for (uint32_t i = tid; i < (uint32_t)M * nk; i += 64 * DW)
      *(uint32_t*)(as + i / nk * spitch + i % nk * 4) = ((const uint32_t*)a.qs)[i];
  } else {
    auto put = [&](const uint4& v, uint32_t i) {  // (called by whole blocks' lanes)
      const uint32_t row = i / per, u = i - row * per;
      uint32_t o[2];
      const uint32_t b = mx_round<DT, F>(v, o);
      uint8_t* p = ac + row * pitch + u * (E * F / 8);
      if constexpr (TWO) {
        uint32_t lo[2];
        o[0] = cut(o[0], lo[0]), o[1] = cut(o[1], lo[1]);
        mx_store<DT, F>(p + M * pitch, lo);
      }
      mx_store<DT, F>(p, o);
      if (u % BL == 0) as[row * spitch + u / BL] = (uint8_t)b;
    };
#pragma unroll
    for (int j = 0; j < XU; j++)
      if (tid + j * 64 * DW < units) put(xu[j], tid + j * 64 * DW);
    for (uint32_t i = tid + XU * 64 * DW; i < units; i += 64 * DW) {
      const uint32_t row = i / per;
      put(mx_unit_at<DT>((const T*)a.x + (size_t)row * a.K, i - row * per, a.K), i);
    }
  }
  __syncthreads();
  const int tok = min(PARTS == kSide ? r & 7 : r, M - 1);  // (tokens past M: not used)
  const uint8_t* ar = ac + (PARTS == kSide && r >= 8 ? M + tok : tok) * pitch + 16 * h;
  const uint8_t* sr = as + tok * spitch + h;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  auto work = [&](Set& b, Scales& sc) {
    auto steps = [&](const uint8_t* ar) {
#pragma unroll
      for (int i = 0; i < P; i++) {
        const int s = min(s0 + c * P + i, nk - 1);  // (past the run: times zeros)
        const uint32_t sa = s0 + c * P + i < s1 ? sr[4 * s] : 0;  // (and no NaN of another's block)
        i32x8 act;
        if constexpr (F == MX_FP4) act = wide(*(const i32x4*)(ar + s * RB));
        else act = __builtin_shufflevector(*(const i32x4*)(ar + s * RB), *(const i32x4*)(ar + s * RB + 64), 0, 1, 2, 3, 4, 5, 6, 7);
        auto add = [&](const i32x8& v) {
          acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wide(b[i]), v, acc, 4, F == MX_FP4 ? 4 : 0, 0, (int)sc[i], 0,
                                                                 (int)sa);
        };
        if constexpr (PARTS == kCut) {
          i32x8 lo, hi;
          cut(act, lo, hi);
          add(lo), add(hi);
        } else {
          add(act);
        }
      }
    };
    if constexpr (PARTS == kTurn) {
#pragma unroll 1  // (of both parts at once the operands spill)
      for (int p = 1; p >= 0; p--) steps(ar + p * M * pitch);
    } else {
      steps(ar);
    }
    load(b, sc, gn, cn);
    next(gn, cn);
    if (c == pieces - 1) {
      *(f32x4*)&red[(wave * 16 + r) * RP + 4 * h] = acc;
      acc = (f32x4){0.f, 0.f, 0.f, 0.f};
      __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0); the weight loads stay in flight
      ub_barrier();
      for (int i = tid; i < a.tiles * M * 16; i += 64 * DW) {
        const int j = i & 15, mt = i >> 4, t = mt / M, m = mt - t * M, n = (g * a.tiles + t) * 16 + j;
        float v = 0.f;
        for (int p = 0; p < a.ks; p++) {
          v += red[((t * a.ks + p) * 16 + m) * RP + j];
          if constexpr (PARTS == kSide) v += red[((t * a.ks + p) * 16 + m + 8) * RP + j];
        }
        if (n < a.N) ub_store<DT>(a.y, (size_t)m * a.N + n, v + (a.bias ? a.bias[n] : 0.f));
      }
      __builtin_amdgcn_s_waitcnt(0xC07F);
      ub_barrier();
    }
    next(g, c);
  };
  while (g < rounds) {
    work(b0, c0);
    if (g >= rounds) break;
    work(b1, c1);
  }
}

// us, rounding in every workgroup / in a launch ahead / the tiles (M x K x N): 4 x 4096 x
// 4096 6.0 / 7.4 / 9.0, 4 x 14336 x 4096 10.5 / 10.8 / 11.7, 16 x 4096 x 4096 9.1 / 7.8 / 9.3, 16
// x 4096 x 28672 15.4 / 15.1 / 16.2, 16 x 8192 x 8192 15.7 / 11.9 / 13.8, 16 x 14336 x 4096 21.7 /
// 12.2 / 12.2; of codes that are there 5.2, 8.5, 5.4, 12.7, 9.3, 9.6.  1 x 28672 x 8192 22 (5.6
// TB/s).
constexpr int kRound = 60 * 1024;
constexpr int kCUs = 256, kLds = 160 * 1024;
size_t dec_lds(int F, int M, int nk, bool two) {
  return sizeof(float) * DW * 16 * RP + (size_t)M * ((two ? 2 : 1) * (nk * 128 * F / 8 + 16) + nk * 4 + 4) + 16;
}

template <int F, int DT, bool PRE, int PARTS>
void dec_as(MxDecArgs a, hipStream_t s) {
  static UbLdsLimit limit;
  limit.raise((const void*)k_mx_dec<F, DT, PRE, PARTS>, kLds);
  const int nt = ub_cdiv(a.N, 16);
  // a group of tiles for every CU, as many wavefronts to a tile as that leaves
  a.tiles = nt <= kCUs ? 1 : nt <= kCUs * DW ? ub_cdiv(nt, kCUs) : DW;
  a.ks = DW / a.tiles;
  a.per = ub_cdiv(a.nk, a.ks);
  const int groups = ub_cdiv(nt, a.tiles);
  k_mx_dec<F, DT, PRE, PARTS><<<groups < kCUs ? groups : kCUs, 64 * DW, dec_lds(F, a.M, a.nk, PARTS >= kSide), s>>>(a);
}

template <int F, int DT, bool PRE>
void dec(const MxDecArgs& a, hipStream_t s) {
  if constexpr (F == MX_FP4) dec_as<F, DT, PRE, kWhole>(a, s);
  else if (dec_lds(F, a.M, a.nk, true) > kLds) dec_as<F, DT, PRE, kCut>(a, s);
  else if (a.M <= 8) dec_as<F, DT, PRE, kSide>(a, s);
  else dec_as<F, DT, PRE, kTurn>(a, s);
}

// ------------------------------------------------------------- the choice
// (two: the codes in parts, packed)
template <int F, int DT>
void quantize(const void* x, uint8_t* q, uint8_t* sc, int R, int C, int nk, bool packed, bool two, hipStream_t s) {
  const uint32_t units = (uint32_t)((int64_t)R * nk * (128 / MxElem<DT>::E));
  const unsigned g = (units + 511) / 512;
  if constexpr (F == MX_FP8)
    if (two) return k_mx_quant<DT, F, true, true><<<g, 256, 0, s>>>(x, q, sc, units, C, nk);
  if (packed) k_mx_quant<DT, F, true, false><<<g, 256, 0, s>>>(x, q, sc, units, C, nk);
  else k_mx_quant<DT, F, false, false><<<g, 256, 0, s>>>(x, q, sc, units, C, nk);
}

// The tile and the number of K parts that take least, by measured times (0.01 us): a
// step of K on a CU that has one workgroup of the tile, the same for each of several
// (side by side or in turn), and what a tile takes beside its steps; parts cost a
// launch and their sums' way to memory and back.  us, M x K x N, e2m1 (e4m3) activations
// laid out, on 128 x 256 / 128 x 128 / 64 x 64 / 32 x 128: 64 x 4096 x 6144 23.5 / 12.7 / 9.1 /
// 9.9 (31 / 17 / 10.5 / 10.5), 201 x 3520 x 9001 24.5 / 13.1 / 13.1 / 12.5 (31 / 16.4 / 16.8 /
// 14.0), 512 x 4096 x 4096 23.5 / 13.9 / 12.1 / 13.6 (31 / 17 / 14.8 / 15.7), 1646 x 5413 x 4856
// 35 / 27 / 41 / -, 1024 x 4096 x 14336 42 / 46 / 58 / 80 (55 / 75 / 78 / 91); 160 x 10304 x 436
// in 8 parts 8.6 on the last two.  e4m3 in two parts, the call with codes that are there,
// on the same tiles: 64 x 4096 x 6144 - / 30 / 19 / 15, 201 x 3520 x 9001 52 / 31 / 29 / 19.5, 512 x
// 4096 x 4096 55 / 33 / 28 / 23, 1646 x 5413 x 4856 80 / 86 / 102 / -, 1024 x 4096 x 14336 89 / 120 /
// 127 / -.
struct Plan { int tile, parts; };
Plan plan_for(int F, bool X, int M, int N, int nk) {
  static const struct { int m, n, tile, one[3], each[3]; } t[4] = {{128, 256, 390, {63, 75, 124}, {50, 70, 122}},
                                                                   {128, 128, 150, {25, 38, 63}, {28, 51, 78}},
                                                                   {64, 64, 60, {17, 22, 37}, {12, 16, 26}},
                                                                   {32, 128, 60, {20, 22, 28}, {15, 18, 22}}};
  const int f = F == MX_FP4 ? 0 : X ? 2 : 1;
  Plan best = {-1, 1};
  double least = 0;
  for (int i = 0; i < 4; i++) {
    const int64_t tiles = (int64_t)ub_cdiv(M, t[i].m) * ub_cdiv(N, t[i].n);
    for (int p = 1; p <= 32 && p <= nk; p *= 2) {
      if (p > 1 && (tiles * p > 1024 || (int64_t)M * N >= 1 << 26)) break;
      const int64_t per = (tiles * p + kCUs - 1) / kCUs;
      double cost = (double)per * (t[i].tile + (per == 1 ? t[i].one[f] : t[i].each[f]) * ub_cdiv(nk, p));
      if (p > 1) cost += 300 + (double)M * N * 8 * p / 52e3;
      if (best.tile < 0 || cost < least) best = {i, p}, least = cost;
    }
  }
  return best;
}

template <int F, int DT, int X>
void gemm(int tile, const MxArgs& a, int parts, hipStream_t s) {
#define UB_MX(WM, WN, TM, TN, NS, OCC)                                                                   \
  {                                                                                                      \
    constexpr int BM = 32 * WM * TM, BN = 32 * WN * TN, NW = WM * WN;                                    \
    constexpr int nl = (BM * kRowStep<F> / 1024 * (X == kParts ? 2 : 1) + BN / 16 + NW - 1) / NW, sl = (((BM < 64 ? 64 : BM) + BN) / 64 + NW - 1) / NW; \
    constexpr int lds = NS * NW * (nl * 1024 + sl * 256);                                                \
    static UbLdsLimit limit;                                                                             \
    limit.raise((const void*)k_mx_gemm<F, DT, X, WM, WN, TM, TN, NS, OCC>, lds);                            \
    k_mx_gemm<F, DT, X, WM, WN, TM, TN, NS, OCC>                                                            \
        <<<ub_cdiv(a.M, BM) * ub_cdiv(a.N, BN) * parts, 64 * NW, lds, s>>>(a);                           \
    return;                                                                                              \
  }
  // rings as deep as leaves two workgroups of the large tiles to a CU, four of the small
  if constexpr (X == kParts) {
    UB_MX(1, 4, 1, 1, 3, 3)
  } else {
    if (tile == 0) UB_MX(2, 2, 2, 4, (F == MX_FP4 ? 3 : 2), 2)
    if constexpr (X == kCuts) {
      if (tile == 1) UB_MX(4, 2, 1, 2, 3, 2)
    } else {
      if (tile == 1) UB_MX(2, 4, 2, 1, 3, (F == MX_FP4 ? 4 : 2))
    }
    if (tile == 2) UB_MX(2, 2, 1, 1, (F == MX_FP4 ? 4 : 3), 4)
    if constexpr (X == kOne) UB_MX(1, 4, 1, 1, (F == MX_FP4 ? 6 : 5), 4)
  }
#undef UB_MX
}

template <int F, int DT>
int linear(const char* nm, const UbridgeMxLinearArgs& p, hipStream_t s) {
  const int nk = ub_cdiv(p.K, 128), M = p.M, N = p.N;
  const uint8_t* w = (const uint8_t*)p.w;
  const uint32_t* sw = (const uint32_t*)p.w_scales;
  if (M <= 16 && dec_lds(F, M, nk, false) <= kLds) {
    MxDecArgs d = {p.x, (const uint8_t*)p.codes, (const uint8_t*)p.scales, w, sw, p.bias, p.y, M, p.K, N, nk, 0, 0, 0};
    if (p.x && (int64_t)M * p.K <= kRound) {
      dec<F, DT, false>(d, s);
      return UB_OK;
    }
    const size_t codes = p.x ? (size_t)M * nk * kRowStep<F> : 0;
    UbScratch ws(s, codes + (p.x ? (size_t)M * nk * 4 : 0), true);
    if (p.x) {
      uint8_t* q = (uint8_t*)ws.get();
      if (!q) return ub_set_error(UB_ERR_LAUNCH, "%s: no workspace", nm);
      quantize<F, DT>(p.x, q, q + codes, M, p.K, nk, false, false, s);
      d.x = nullptr, d.q = q, d.qs = q + codes;
    }
    dec<F, DT, true>(d, s);
    return UB_OK;
  }
  // (of f32 results always: the rounding of 16 bits does not cover what one product drops)
  constexpr bool X = F == MX_FP8;
  const bool exact = X && (DT == UB_F32 || M <= 16 || !p.one_product);
  const Plan plan = plan_for(F, exact, M, N, nk);
  const int part = ub_cdiv(nk, plan.parts), parts = ub_cdiv(nk, part);  // (none empty)
  const bool two = exact && plan.tile == 3;
  const size_t rows = (size_t)ub_cdiv(M, 16) * 16, codes = rows * nk * kRowStep<F> * (two ? 2 : 1), words = rows * nk * 4;
  const size_t sums = parts > 1 ? sizeof(float) * parts * (size_t)M * N : 0;
  UbScratch ws(s, codes + words + sums, true);
  uint8_t* q = (uint8_t*)ws.get();
  if (!q) return ub_set_error(UB_ERR_LAUNCH, "%s: no workspace", nm);
  uint8_t* qs = q + codes;
  if (p.x) {
    quantize<F, DT>(p.x, q, qs, M, p.K, nk, true, two, s);
  } else {
    const uint32_t units = (uint32_t)(rows * nk * (kRowStep<F> / 16)), g = (units + 255) / 256;
    const uint8_t *c = (const uint8_t*)p.codes, *cs = (const uint8_t*)p.scales;
    if (two) k_mx_pack<F, F == MX_FP8><<<g, 256, 0, s>>>(c, cs, q, (uint32_t*)qs, units, M, nk);
    else k_mx_pack<F><<<g, 256, 0, s>>>(c, cs, q, (uint32_t*)qs, units, M, nk);
  }
  MxArgs a = {q, w, (const uint32_t*)qs, sw, p.bias, p.y, M, N, nk, part};
  auto product = [&](auto dt, int np) {
    constexpr int D = decltype(dt)::value;
    if constexpr (X) {
      if (two) return gemm<F, D, kParts>(plan.tile, a, np, s);
      if (exact) return gemm<F, D, kCuts>(plan.tile, a, np, s);
    }
    if constexpr (!X || DT != UB_F32) gemm<F, D, kOne>(plan.tile, a, np, s);
  };
  if (parts > 1) {
    a.y = qs + words;
    product(std::integral_constant<int, kSum>{}, parts);
    const int64_t all = (int64_t)M * N;
    k_mx_sum<DT><<<(unsigned)((all + 255) / 256), 256, 0, s>>>((const float*)a.y, p.bias, p.y, all, N, parts);
  } else {
    product(std::integral_constant<int, DT>{}, 1);
  }
  return UB_OK;
}

constexpr int kMaxK = 1 << 17;
bool dtype_ok(int dt) { return dt == UB_F32 || dt == UB_F16 || dt == UB_BF16; }

template <int F>
int linear(const char* nm, const UbridgeMxLinearArgs& p, hipStream_t s) {
  return p.dtype == UB_F32 ? linear<F, UB_F32>(nm, p, s) : p.dtype == UB_F16 ? linear<F, UB_F16>(nm, p, s) : linear<F, UB_BF16>(nm, p, s);
}

}  // namespace

UB_API int ubridge_mx_quantize(const void* x, int dtype, void* codes, void* scales, int R, int C, int format, void* stream) {
  const char* nm = "ubridge_mx_quantize";
  UB_REQUIRE(dtype_ok(dtype), "%s: dtype %d", nm, dtype);
  UB_REQUIRE(format == MX_FP4 || format == MX_FP8, "%s: format %d (4 or 8)", nm, format);
  UB_REQUIRE(R >= 0 && C > 0 && C <= 1 << 30 && (int64_t)R * (C + 127) <= 1ll << 33, "%s: R=%d C=%d", nm, R, C);  // (32-bit units)
  if (R == 0) return UB_OK;
  UB_REQUIRE(x && codes && scales, "%s: null pointer", nm);
  UB_REQUIRE(((uintptr_t)codes & 15) == 0, "%s: codes not 16-byte aligned", nm);
  const int nk = ub_cdiv(C, 128);
  hipStream_t s = ub_stream(stream);
  uint8_t *q = (uint8_t*)codes, *sc = (uint8_t*)scales;
  auto go = [&](auto f) {
    constexpr int F = decltype(f)::value;
    if (dtype == UB_F32) quantize<F, UB_F32>(x, q, sc, R, C, nk, false, false, s);
    else if (dtype == UB_F16) quantize<F, UB_F16>(x, q, sc, R, C, nk, false, false, s);
    else quantize<F, UB_BF16>(x, q, sc, R, C, nk, false, false, s);
  };
  if (format == MX_FP4) go(std::integral_constant<int, MX_FP4>{});
  else go(std::integral_constant<int, MX_FP8>{});
  return ub_check_launch(nm);
}

UB_API int ubridge_mx_dequantize(const void* codes, const void* scales, void* y, int dtype, int R, int C, int format,
                                 void* stream) {
  const char* nm = "ubridge_mx_dequantize";
  UB_REQUIRE(dtype_ok(dtype), "%s: dtype %d", nm, dtype);
  UB_REQUIRE(format == MX_FP4 || format == MX_FP8, "%s: format %d (4 or 8)", nm, format);
  UB_REQUIRE(R >= 0 && C > 0 && C <= 1 << 30 && (int64_t)R * (C + 127) <= 1ll << 33, "%s: R=%d C=%d", nm, R, C);  // (32-bit units)
  if (R == 0) return UB_OK;
  UB_REQUIRE(y && codes && scales, "%s: null pointer", nm);
  UB_REQUIRE(((uintptr_t)codes & 15) == 0, "%s: codes not 16-byte aligned", nm);
  const int nk = ub_cdiv(C, 128);
  const uint32_t units = (uint32_t)((int64_t)R * ub_cdiv(C, 8));
  const unsigned g = (units + 255) / 256;
  hipStream_t s = ub_stream(stream);
  auto go = [&](auto f) {
    constexpr int F = decltype(f)::value;
    const uint8_t *q = (const uint8_t*)codes, *sc = (const uint8_t*)scales;
    if (dtype == UB_F32) k_mx_back<UB_F32, F><<<g, 256, 0, s>>>(q, sc, y, units, C, nk);
    else if (dtype == UB_F16) k_mx_back<UB_F16, F><<<g, 256, 0, s>>>(q, sc, y, units, C, nk);
    else k_mx_back<UB_BF16, F><<<g, 256, 0, s>>>(q, sc, y, units, C, nk);
  };
  if (format == MX_FP4) go(std::integral_constant<int, MX_FP4>{});
  else go(std::integral_constant<int, MX_FP8>{});
  return ub_check_launch(nm);
}

UB_API int ubridge_mx_pack(const void* codes, const void* scales, void* w, void* w_scales, int N, int K, void* stream) {
  const char* nm = "ubridge_mx_pack";
  UB_REQUIRE(N >= 0 && K > 0 && K <= kMaxK, "%s: N=%d K=%d (1..%d)", nm, N, K, kMaxK);
  UB_REQUIRE((int64_t)N * ub_cdiv(K, 128) <= 1ll << 28, "%s: N=%d K=%d", nm, N, K);  // (32-bit units)
  if (N == 0) return UB_OK;
  UB_REQUIRE(codes && scales && w && w_scales, "%s: null pointer", nm);
  UB_REQUIRE((((uintptr_t)w | (uintptr_t)w_scales) & 15) == 0, "%s: result not 16-byte aligned", nm);
  const int nk = ub_cdiv(K, 128);
  const uint32_t units = (uint32_t)ub_cdiv(N, 16) * 16 * nk * 4;
  k_mx_pack<MX_FP4><<<(units + 255) / 256, 256, 0, ub_stream(stream)>>>(
      (const uint8_t*)codes, (const uint8_t*)scales, (uint8_t*)w, (uint32_t*)w_scales, units, N, nk);
  return ub_check_launch(nm);
}

UB_API int ubridge_mx_linear(const UbridgeMxLinearArgs* p, void* stream) {
  const char* nm = "ubridge_mx_linear";
  UB_REQUIRE(p, "%s: null argument block", nm);
  UB_REQUIRE(dtype_ok(p->dtype), "%s: dtype %d", nm, p->dtype);
  UB_REQUIRE(p->format == MX_FP4 || p->format == MX_FP8, "%s: format %d (4 or 8)", nm, p->format);
  UB_REQUIRE(p->M >= 0 && p->N >= 0 && p->K > 0 && p->K <= kMaxK, "%s: M=%d K=%d (1..%d) N=%d", nm, p->M, p->K, kMaxK, p->N);
  if ((size_t)p->M * p->N == 0) return UB_OK;
  UB_REQUIRE((p->x || (p->codes && p->scales)) && p->w && p->w_scales && p->y, "%s: null pointer", nm);
  UB_REQUIRE((((uintptr_t)p->w | (uintptr_t)p->w_scales) & 15) == 0, "%s: weight not 16-byte aligned", nm);
  UB_REQUIRE(p->x || (((uintptr_t)p->codes & 15) == 0 && ((uintptr_t)p->scales & 3) == 0), "%s: codes not 16-byte, scales not 4-byte aligned", nm);
  // (2^32 threads a launch, 32-bit units)
  UB_REQUIRE(p->M < 1 << 22 && (int64_t)p->M * p->N < 1ll << 38 && ((int64_t)p->M + 15) * (p->K + 127) <= 1ll << 33, "%s: M=%d N=%d K=%d", nm, p->M, p->N, p->K);
  hipStream_t s = ub_stream(stream);
  const int e = p->format == MX_FP4 ? linear<MX_FP4>(nm, *p, s) : linear<MX_FP8>(nm, *p, s);
  return e ? e : ub_check_launch(nm);
}
