// norm.hip -- root-mean-square norm on gfx950, with the residual's addition ahead
// of it and the rounding for the next product behind it, and its gradient:
//
//   h = T(x + residual)              (h = x without one)
//   y = h r w,   r = 1 / sqrt(mean(h^2) + eps)
//
// y goes out in T, as int8 or e4m3 codes with one f32 scale a row (amax / 127,
// amax / 448; 1 for a row of zeros; NaN, codes 0, where a value is not finite), or in
// blocks of 32 (mx_dev.h).  The norm is
// taken of h as it is stored, so that every later reader of the residual stream
// sees the values that were normed.  The sum of squares and r are formed in 64
// bits, which hold the square of every f32 (the additions hide behind the loads);
// y is f32 and rounded once, to what goes out.
//
// Gradient, with g = dy w:   dx = T(r (g - h r^2 mean(g h)) + dh),   dw = sum_rows
// dy h r;   r is formed again from h, which has to be read anyway.
//
// Bound by HBM for many rows, by one launch's latency for few.  A row stays in the
// registers of the workgroup (or, short, of the wavefront) that owns it: x and
// residual are read once, h and y written once.  us: 8 x 4096 with residual to e4m3 4.4;
// 8192 x 4096 bf16 with residual 51 (5.2 TB/s), its gradient 51 + 4 (5.2 TB/s); 2047 x
// 5003 f16 from odd places, f32 gain, 12.4.
#include "mx_dev.h"
#include "quotient.h"
#include "wave.h"

#include <type_traits>

namespace {

enum { OUT_T = 0, OUT_I8 = 1, OUT_E4M3 = 2, OUT_FP4 = 3, OUT_FP8 = 4 };

struct NormArgs {
  const void *x, *res, *w;
  void *h, *y, *scale;
  int R, C, ld, wf32, out;
  double eps;
};

// Unit i of the gain (T or f32) as floats
template <int DT>
__device__ __forceinline__ void gain(const void* w, int wf32, int i, int C, float (&o)[MxElem<DT>::E]) {
  constexpr int E = MxElem<DT>::E;
  if (DT == UB_F32 || wf32) {
#pragma unroll
    for (int q = 0; q < E / 4; q++) {
      const uint4 v = mx_unit_at<UB_F32>((const float*)w, i * (E / 4) + q, C);
#pragma unroll
      for (int e = 0; e < 4; e++) o[4 * q + e] = mx_get<UB_F32>(v, e);
    }
  } else {
    const uint4 v = mx_unit_at<DT>((const typename MxElem<DT>::T*)w, i, C);
#pragma unroll
    for (int e = 0; e < E; e++) o[e] = mx_get<DT>(v, e);
  }
}

// Sum (or maximum of bit patterns) over the NT threads of a row.  `part` is one
// of the workgroup's LDS arrays; each call takes its own, so that one barrier a
// call suffices.
template <int NT>
__device__ __forceinline__ double row_sum(double v, double* part) {
  v = ub_wave_all_sum(v);
  if constexpr (NT > 64) {
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0.0;
#pragma unroll
    for (int i = 0; i < NT / 64; i++) v += part[i];
  }
  return v;
}
template <int NT>
__device__ __forceinline__ uint32_t row_max(uint32_t v, uint32_t* part) {
  v = ub_wave_all_max(v);
  if constexpr (NT > 64) {
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NT / 64; i++) v = max(v, part[i]);
  }
  return v;
}

__device__ __forceinline__ uint32_t magnitude(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// Row scale from the bits of its largest magnitude (infinities and NaN are on top
// of that order): NaN then.  A scale below the smallest f32 is that.
__device__ __forceinline__ float scale_of(uint32_t top, float most) {
  if (top >= 0x7f800000u) return __builtin_nanf("");
  if (top == 0) return 1.f;
  return fmaxf(__fdiv_rn(__uint_as_float(top), most), 0x1p-149f);
}
// Codes of four values, int8 or e4m3 (whose zeros keep their sign, as in blocks and in
// ubridge_fp8_quantize_rows).  PLAIN: s is out of ub_quotient's range (bf16 with residual,
// 2048 x 4096 to e4m3: 15.4 us, with the divide for every row 16.5).
template <bool PLAIN, bool I8>
__device__ __forceinline__ uint32_t codes4(const float* v, float s, float r) {
  float q[4];
#pragma unroll
  for (int e = 0; e < 4; e++) {
    q[e] = PLAIN ? __fdiv_rn(v[e], s) : ub_quotient(v[e], s, r);
    q[e] = __builtin_amdgcn_fmed3f(q[e], I8 ? -127.f : -448.f, I8 ? 127.f : 448.f);
    if constexpr (!I8 && !PLAIN) q[e] = copysignf(q[e], v[e]);
  }
  if constexpr (I8) {
    uint32_t o = 0;
#pragma unroll
    for (int e = 0; e < 4; e++)  // 1.5 2^23 added: an integer, ties to even, in the low bits
      o |= (__float_as_uint(q[e] + 12582912.f) & 0xff) << (8 * e);
    return o;
  } else {
    const int o = __builtin_amdgcn_cvt_pk_fp8_f32(q[0], q[1], 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(q[2], q[3], o, true);
  }
}

// NT threads a row, NV units of it a thread.  NT = 64: four rows a workgroup of
// 256, no barrier.
template <int DT, int NT, int NV>
__global__ void __launch_bounds__(NT < 256 ? 256 : NT) k_norm(NormArgs a) {
  typedef typename MxElem<DT>::T T;
  constexpr int E = MxElem<DT>::E, RP = NT < 256 ? 256 / NT : 1;
  __shared__ double sums[NT / 64];
  __shared__ uint32_t tops[NT / 64];
  const int tid = threadIdx.x % NT, C = a.C;
  const size_t row = (size_t)blockIdx.x * RP + threadIdx.x / NT;
  if (row >= (size_t)a.R) return;  // (whole wavefronts, and no barrier where rows share a workgroup)
  const T* x = (const T*)a.x + row * C;
  const T* res = a.res ? (const T*)a.res + row * C : nullptr;
  uint4 u[NV];
  float w[NV][E];
#pragma unroll
  for (int j = 0; j < NV; j++) u[j] = mx_unit_at<DT>(x, tid + j * NT, C);
  if (res) {
    uint4 v[NV];
#pragma unroll
    for (int j = 0; j < NV; j++) v[j] = mx_unit_at<DT>(res, tid + j * NT, C);
#pragma unroll
    for (int j = 0; j < NV; j++) gain<DT>(a.w, a.wf32, tid + j * NT, C, w[j]);
#pragma unroll
    for (int j = 0; j < NV; j++) {
      float s[E];
#pragma unroll
      for (int e = 0; e < E; e++) s[e] = mx_get<DT>(u[j], e) + mx_get<DT>(v[j], e);
      u[j] = mx_pack<DT>(s);
      mx_put<DT>((T*)a.h + row * C, tid + j * NT, C, u[j]);
    }
  } else {
#pragma unroll
    for (int j = 0; j < NV; j++) gain<DT>(a.w, a.wf32, tid + j * NT, C, w[j]);
  }
  double ss = 0.0;
#pragma unroll
  for (int j = 0; j < NV; j++)
#pragma unroll
    for (int e = 0; e < E; e++) {
      const double f = mx_get<DT>(u[j], e);
      ss = __builtin_fma(f, f, ss);
    }
  ss = row_sum<NT>(ss, sums);
  const float r = (float)(1.0 / __builtin_sqrt(ss / C + a.eps));
  float y[NV][E];
  uint32_t top = 0;
#pragma unroll
  for (int j = 0; j < NV; j++)
#pragma unroll
    for (int e = 0; e < E; e++) {
      y[j][e] = mx_get<DT>(u[j], e) * r * w[j][e];  // (0 past the row: w is)
      // (past the row: no part in a maximum, though 0 times an infinite r is NaN)
      if (NT * E * NV > C && (tid + j * NT) * E + e >= C) y[j][e] = 0.f;
      top = max(top, magnitude(y[j][e]));
    }
  if (a.out == OUT_T) {
#pragma unroll
    for (int j = 0; j < NV; j++) mx_put<DT>((T*)a.y + row * C, tid + j * NT, C, mx_pack<DT>(y[j]));
  } else if (a.out == OUT_I8 || a.out == OUT_E4M3) {
    const bool i8 = a.out == OUT_I8;
    top = row_max<NT>(top, tops);
    const float s = scale_of(top, i8 ? 127.f : 448.f);
    if (tid == 0) ((float*)a.scale)[row] = s;
    uint8_t* q = (uint8_t*)a.y + row * C;
    // (the same in a wavefront, whose lanes have one row)
    const bool none = __builtin_amdgcn_readfirstlane(s != s), plain = __builtin_amdgcn_readfirstlane(!ub_exact_scale(s));
    const float rs = plain ? 0.f : __fdiv_rn(1.f, s);
    auto all = [&](auto pl, auto i) {
#pragma unroll
      for (int j = 0; j < NV; j++) {
        const int at = (tid + j * NT) * E;
        uint32_t o[E / 4];
#pragma unroll
        for (int p = 0; p < E / 4; p++) o[p] = none ? 0u : codes4<decltype(pl)::value, decltype(i)::value>(&y[j][4 * p], s, rs);
        if (at + E <= C) {
          __builtin_memcpy(q + at, o, E);
        } else {
#pragma unroll
          for (int e = 0; e < E; e++)
            if (at + e < C) q[at + e] = (uint8_t)(o[e >> 2] >> (8 * (e & 3)));
        }
      }
    };
    if (i8 && !plain) all(std::false_type{}, std::true_type{});
    else if (i8) all(std::true_type{}, std::true_type{});
    else if (!plain) all(std::false_type{}, std::false_type{});
    else all(std::true_type{}, std::false_type{});
  } else {
    auto blocks = [&](auto f) {
      constexpr int F = decltype(f)::value, BL = 32 / E;  // lanes a block
#pragma unroll
      for (int j = 0; j < NV; j++) {
        const int i = tid + j * NT;
        uint32_t t = 0;
#pragma unroll
        for (int e = 0; e < E; e++) t = max(t, magnitude(y[j][e]));
        const uint32_t b = mx_byte<F>(mx_top<BL>(t));
        if (i * E >= a.ld) continue;  // (whole blocks)
        uint32_t o[E / 4];
#pragma unroll
        for (int p = 0; p < E / 4; p++) o[p] = mx_codes4<F>(y[j][4 * p], y[j][4 * p + 1], y[j][4 * p + 2], y[j][4 * p + 3], b);
        uint8_t* q = (uint8_t*)a.y + row * (size_t)(a.ld * F / 8);
        if constexpr (F == MX_FP8) {
          __builtin_memcpy(q + i * E, o, E);
        } else if constexpr (E == 8) {
          ((uint32_t*)q)[i] = o[0] | o[1] << 16;
        } else {
          ((uint16_t*)q)[i] = (uint16_t)o[0];
        }
        if (i % BL == 0) ((uint8_t*)a.scale)[row * (size_t)(a.ld / 32) + i / BL] = (uint8_t)b;
      }
    };
    if (a.out == OUT_FP4) blocks(std::integral_constant<int, MX_FP4>{});
    else blocks(std::integral_constant<int, MX_FP8>{});
  }
}

// ---------------------------------------------------------------- gradient
struct NormGradArgs {
  const void *h, *w, *dy, *dh;
  void *dx, *dw;  // dw f32 partial sums [workgroups][C]
  int R, C, wf32;
  double eps;
};

// A workgroup takes rows b, b + grid, ...; a thread owns the same columns of all
// of them and keeps their part of dw, in registers up to 4 units a thread, else in LDS
// (4096 x 32768 bf16 270 us; in registers, which do not suffice, 602).
template <int DT, int NT, int NV>
__global__ void __launch_bounds__(NT) k_norm_grad(NormGradArgs a) {
  typedef typename MxElem<DT>::T T;
  constexpr int E = MxElem<DT>::E;
  __shared__ double s0[2][NT / 64], s1[2][NT / 64];
  const int tid = threadIdx.x, C = a.C;
  constexpr bool HELD = NV <= 4;
  __shared__ float held[HELD ? 1 : NV * E][HELD ? 1 : NT];
  float w[NV][E], dwr[HELD ? NV : 1][E];
  auto dw = [&](int j, int e) -> float& {
    if constexpr (HELD) return dwr[j][e];
    else return held[j * E + e][tid];
  };
#pragma unroll
  for (int j = 0; j < NV; j++) {
    gain<DT>(a.w, a.wf32, tid + j * NT, C, w[j]);
#pragma unroll
    for (int e = 0; e < E; e++) dw(j, e) = 0.f;
  }
  uint4 h[NV], d[NV], z[NV];
  auto load = [&](size_t row) {
#pragma unroll
    for (int j = 0; j < NV; j++) h[j] = mx_unit_at<DT>((const T*)a.h + row * C, tid + j * NT, C);
#pragma unroll
    for (int j = 0; j < NV; j++) d[j] = mx_unit_at<DT>((const T*)a.dy + row * C, tid + j * NT, C);
#pragma unroll
    for (int j = 0; j < NV; j++)
      z[j] = a.dh ? mx_unit_at<DT>((const T*)a.dh + row * C, tid + j * NT, C) : make_uint4(0, 0, 0, 0);
  };
  int turn = 0;  // two sets of partial sums by turns: one barrier a row suffices
  for (size_t row = blockIdx.x; row < (size_t)a.R; row += gridDim.x, turn ^= 1) {
    load(row);
    double ss = 0.0, gh = 0.0;
#pragma unroll
    for (int j = 0; j < NV; j++) {
#pragma unroll
      for (int e = 0; e < E; e++) {
        const double f = mx_get<DT>(h[j], e);
        ss = __builtin_fma(f, f, ss);
        gh = __builtin_fma((double)(mx_get<DT>(d[j], e) * w[j][e]), f, gh);
      }
    }
    if constexpr (!HELD) {  // unpacked once more below: not kept as f32 in between
#pragma unroll
      for (int j = 0; j < NV; j++)
        asm volatile("" : "+v"(h[j].x), "+v"(h[j].y), "+v"(h[j].z), "+v"(h[j].w), "+v"(d[j].x), "+v"(d[j].y), "+v"(d[j].z), "+v"(d[j].w));
    }
    ss = ub_wave_all_sum(ss);
    gh = ub_wave_all_sum(gh);
    if ((tid & 63) == 0) s0[turn][tid >> 6] = ss, s1[turn][tid >> 6] = gh;
    __syncthreads();
    ss = gh = 0.0;
#pragma unroll
    for (int i = 0; i < NT / 64; i++) ss += s0[turn][i], gh += s1[turn][i];
    const double var = ss / C + a.eps;
    const float r = (float)(1.0 / __builtin_sqrt(var)), m = (float)(gh / C / var);  // m = r^2 mean(g h)
#pragma unroll
    for (int j = 0; j < NV; j++) {
      float o[E];
#pragma unroll
      for (int e = 0; e < E; e++) {
        const float f = mx_get<DT>(h[j], e), y = mx_get<DT>(d[j], e);
        o[e] = r * (y * w[j][e] - f * m) + mx_get<DT>(z[j], e);
        dw(j, e) += y * (f * r);
      }
      if (a.dx) mx_put<DT>((T*)a.dx + row * C, tid + j * NT, C, mx_pack<DT>(o));
    }
  }
  if (a.dw) {
    float* p = (float*)a.dw + (size_t)blockIdx.x * C;
#pragma unroll
    for (int j = 0; j < NV; j++)
#pragma unroll
      for (int q = 0; q < E / 4; q++)
        mx_put<UB_F32>(p, (tid + j * NT) * (E / 4) + q, C,
                       make_uint4(__float_as_uint(dw(j, 4 * q)), __float_as_uint(dw(j, 4 * q + 1)),
                                  __float_as_uint(dw(j, 4 * q + 2)), __float_as_uint(dw(j, 4 * q + 3))));
  }
}

// dw [C] of type DT from G partial rows, in an order that depends on G alone: a
// workgroup owns 64 columns, wavefront i the rows i, i + 16, ...
template <int DT>
__global__ void __launch_bounds__(1024) k_norm_dw(const float* __restrict__ part, void* __restrict__ dw, int G, int C) {
  __shared__ float s[16][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = blockIdx.x * 64 + lane;
  float v = 0.f;
  if (c < C) {
#pragma unroll 8
    for (int g = wave; g < G; g += 16) v += part[(size_t)g * C + c];
  }
  s[wave][lane] = v;
  __syncthreads();
  if (wave == 0 && c < C) {
    v = 0.f;
#pragma unroll
    for (int i = 0; i < 16; i++) v += s[i][lane];
    ub_store<DT>(dw, c, v);
  }
}

// Threads a row and units a thread: a wavefront, four rows to a workgroup, for short
// rows of which there are many (a workgroup each, most of it would idle); else 256
// threads up to 4 units, more for longer rows.  us, bf16 with residual, wavefront / 256
// threads: 65536 x 128 26 / 87, 8192 x 512 8.5 / 14, 8192 x 1024 12.5 / 16, 1024 x 512 3.6 / 3.7;
// 256 / 512 / 1024 threads: 8 x 4096 3.6 / 3.7 / 3.7, 2048 x 4096 12.7 / 14.3 / 15.7, 8192 x 4096
// 48 / 46 / 58 (5.6 TB/s), 2048 x 5120 15.8 / 17.6 / 17.4, 64 x 8192 4.3 / 3.8 / 3.8, 512 x 8192
// 8.5 / 8.5 / 8.9.
template <int DT, class F>
void with_shape(int R, int ld, F f) {
  const int units = ld / MxElem<DT>::E;
#define UB_NORM(NT_, NV_) return f(std::integral_constant<int, NT_>{}, std::integral_constant<int, NV_>{})
  if (R >= 1024 && units <= 64) UB_NORM(64, 1);
  if (R >= 1024 && units <= 128) UB_NORM(64, 2);
  if (units <= 256) UB_NORM(256, 1);
  if (units <= 512) UB_NORM(256, 2);
  if (units <= 768) UB_NORM(256, 3);
  if (R >= 512 && units <= 1024) UB_NORM(256, 4);
  if (units <= 1024) UB_NORM(512, 2);
  if (units <= 2048) UB_NORM(1024, 2);
  UB_NORM(1024, 4);
#undef UB_NORM
}

template <int DT>
void norm(const NormArgs& a, hipStream_t s) {
  with_shape<DT>(a.R, a.ld, [&](auto nt, auto nv) {
    constexpr int NT = decltype(nt)::value, NV = decltype(nv)::value, RP = NT < 256 ? 256 / NT : 1;
    k_norm<DT, NT, NV><<<ub_cdiv(a.R, RP), NT * RP, 0, s>>>(a);
  });
}

constexpr int kGradGroups = 512;  // workgroups, at most: dw's partial sums stay small beside the rows

// Threads a row: 256 up to 4 units each.  us of the call with dx and dw, bf16 with dh, on 64 / 128 /
// 256 / 512 / 1024 threads: 65536 x 128 192 / 221 / 224 / 280 / 549, 8192 x 512 21 / 26 / 26 / 38 / 75, 1024
// 29 / 28 / 28 / 38 / 75, 2048 40 / 36 / 31 / 39 / 74, 4096 - / 59 / 51 / 52 / 78, 8192 - / - / 107 / 111
// / 111; 4096 x 16384 - / - / - / 119 / 116; 64 x 8192 - / - / 9.4 / 8.7 / 9.1; f32 8192 x 4096 - / - / 102 /
// 105 / 108.  (Rows under 1024 values would take 15-20% less on a wavefront each, and are far
// from HBM's time either way.)
template <int DT>
void norm_grad(const NormGradArgs& a, int groups, hipStream_t s) {
  const int units = ub_cdiv(a.C, MxElem<DT>::E);
  if (units <= 256) k_norm_grad<DT, 256, 1><<<groups, 256, 0, s>>>(a);
  else if (units <= 512) k_norm_grad<DT, 256, 2><<<groups, 256, 0, s>>>(a);
  else if (units <= 1024) k_norm_grad<DT, 256, 4><<<groups, 256, 0, s>>>(a);
  else if (units <= 2048) k_norm_grad<DT, 512, 4><<<groups, 512, 0, s>>>(a);
  else k_norm_grad<DT, 512, 8><<<groups, 512, 0, s>>>(a);
}

constexpr int kRow = 65536;  // bytes of a row, at most

// (2^32 threads a launch)
bool sizes_ok(int R, int C, int dt) {
  return R >= 0 && R < 1 << 22 && C > 0 && (int64_t)C * (dt == UB_F32 ? 4 : 2) <= kRow;
}

}  // namespace

UB_API int ubridge_rms_norm(const UbridgeRmsNormArgs* p, void* stream) {
  const char* nm = "ubridge_rms_norm";
  UB_REQUIRE(p, "%s: null argument block", nm);
  UB_REQUIRE(p->dtype >= UB_F32 && p->dtype <= UB_BF16, "%s: dtype %d", nm, p->dtype);
  UB_REQUIRE(p->w_dtype == p->dtype || p->w_dtype == UB_F32, "%s: gain of type %d", nm, p->w_dtype);
  UB_REQUIRE(p->out >= OUT_T && p->out <= OUT_FP8, "%s: out %d", nm, p->out);
  UB_REQUIRE(sizes_ok(p->R, p->C, p->dtype), "%s: R=%d C=%d (rows of up to 64 KiB)", nm, p->R, p->C);
  UB_REQUIRE(p->eps >= 0 && p->eps <= 3.4e38, "%s: eps", nm);
  if (p->R == 0) return UB_OK;
  UB_REQUIRE(p->x && p->w && p->y && (p->h || !p->residual) && (p->scale || p->out == OUT_T), "%s: null pointer", nm);
  const int ld = ub_cdiv(p->C, 128) * 128;
  UB_REQUIRE(p->out < OUT_FP4 || ((uintptr_t)p->y & 15) == 0, "%s: codes not 16-byte aligned", nm);
  const NormArgs a = {p->x, p->residual, p->w, p->h, p->y, p->scale, p->R, p->C, ld, p->w_dtype == UB_F32, p->out, p->eps};
  hipStream_t s = ub_stream(stream);
  if (p->dtype == UB_F32) norm<UB_F32>(a, s);
  else if (p->dtype == UB_F16) norm<UB_F16>(a, s);
  else norm<UB_BF16>(a, s);
  return ub_check_launch(nm);
}

UB_API int ubridge_rms_norm_grad(const UbridgeRmsNormGradArgs* p, void* stream) {
  const char* nm = "ubridge_rms_norm_grad";
  UB_REQUIRE(p, "%s: null argument block", nm);
  UB_REQUIRE(p->dtype >= UB_F32 && p->dtype <= UB_BF16, "%s: dtype %d", nm, p->dtype);
  UB_REQUIRE(p->w_dtype == p->dtype || p->w_dtype == UB_F32, "%s: gain of type %d", nm, p->w_dtype);
  UB_REQUIRE(sizes_ok(p->R, p->C, p->dtype), "%s: R=%d C=%d (rows of up to 64 KiB)", nm, p->R, p->C);
  UB_REQUIRE(p->eps >= 0 && p->eps <= 3.4e38, "%s: eps", nm);
  UB_REQUIRE((p->R == 0 || (p->h && p->dy)) && p->w && (p->dx || p->dw), "%s: null pointer", nm);
  if (p->R == 0 && !p->dw) return UB_OK;
  hipStream_t s = ub_stream(stream);
  const int groups = p->R < kGradGroups ? p->R : kGradGroups;
  UbScratch ws(s, p->dw ? sizeof(float) * (size_t)groups * p->C : 0, true);
  UB_REQUIRE(!p->dw || groups == 0 || ws.get(), "%s: no workspace", nm);
  const NormGradArgs a = {p->h, p->w, p->dy, p->dh, p->dx, p->dw ? ws.get() : nullptr, p->R, p->C, p->w_dtype == UB_F32, p->eps};
  if (groups) {
    if (p->dtype == UB_F32) norm_grad<UB_F32>(a, groups, s);
    else if (p->dtype == UB_F16) norm_grad<UB_F16>(a, groups, s);
    else norm_grad<UB_BF16>(a, groups, s);
  }
  if (p->dw) {  // (no rows: zeros)
    const int g = ub_cdiv(p->C, 64);
    const float* part = (const float*)ws.get();
    if (p->w_dtype == UB_F32) k_norm_dw<UB_F32><<<g, 1024, 0, s>>>(part, p->dw, groups, p->C);
    else if (p->w_dtype == UB_F16) k_norm_dw<UB_F16><<<g, 1024, 0, s>>>(part, p->dw, groups, p->C);
    else k_norm_dw<UB_BF16><<<g, 1024, 0, s>>>(part, p->dw, groups, p->C);
  }
  return ub_check_launch(nm);
}
