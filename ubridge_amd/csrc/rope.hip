// rope.hip -- rotary positions for gfx950, alone or fused with the store of
// the keys and values into the pages of a cache.
//
// Pair i of a head at position p turns by the angle 2 pi p t[i] (t: turns per
// position, f64, [rot / 2]; the context scaling is in t):
//
//   (a, b) -> f (a cos - b sin, b cos + a sin)        inverse: sin -> -sin
//
// The pairs are (x[i], x[i + rot / 2]) or, interleaved, (x[2 i], x[2 i + 1]);
// elements from rot on pass through.  The inverse turn is the gradient.
//
// Numerics.  p t is formed in f64 and reduced there to the nearest quarter
// turn: an f32 product would lose every fractional bit of a far position (p
// t = 2^17 turns at p = 2^20 leaves 2^-7 of a turn).  The remainder, at most an
// eighth of a turn, is rounded to f32 (angle error < 5e-8) and its sine and
// cosine are Taylor polynomials whose first dropped terms are below 2e-9 and
// 2e-9.  The rotation is f32 and rounds once, to the output's type.
//
// One workgroup turns the heads of one token (or a part of them, where the
// tokens alone leave CUs idle).  Its threads load their first 16 bytes of q, k
// and v, then each makes the sine and cosine of one pair into LDS, so that a
// pair costs one evaluation a token and not one a head, and the loads are in
// flight meanwhile.
#include "common.h"

namespace {

constexpr int NT = 256;

struct RopeDev {
  UbridgeRopeArgs a;
  int heads;    // q, k and (append) v heads of a token
  int parts;    // workgroups a token
  int lg;       // log2 of the lanes of a head
  int* err;
};

template <int DT> struct Elem;  // element type and elements of a 16-byte unit
template <> struct Elem<UB_F32> { typedef float T; static constexpr int E = 4; };
template <> struct Elem<UB_F16> { typedef uint16_t T; static constexpr int E = 8; };
template <> struct Elem<UB_BF16> { typedef uint16_t T; static constexpr int E = 8; };

// n <= E elements from p (element-aligned: gfx950 loads 16 bytes from there)
template <int DT>
__device__ __forceinline__ void ld(float (&v)[Elem<DT>::E], const typename Elem<DT>::T* p, int n) {
  constexpr int E = Elem<DT>::E;
  typename Elem<DT>::T r[E];
  if (n >= E) {
    __builtin_memcpy(r, p, 16);
  } else {
#pragma unroll
    for (int j = 0; j < E; j++) r[j] = j < n ? p[j] : (typename Elem<DT>::T)0;
  }
#pragma unroll
  for (int j = 0; j < E; j++) v[j] = ub_load<DT>(r, j);
}

template <int DT>
__device__ __forceinline__ void st(typename Elem<DT>::T* p, const float (&v)[Elem<DT>::E], int n) {
  constexpr int E = Elem<DT>::E;
  typename Elem<DT>::T r[E];
#pragma unroll
  for (int j = 0; j < E; j++) ub_store<DT>(r, j, v[j]);
  if (n >= E) {
    __builtin_memcpy(p, r, 16);
  } else {
#pragma unroll
    for (int j = 0; j < E; j++)
      if (j < n) p[j] = r[j];
  }
}

// x / s to e4m3, saturating, NaN kept
template <int E>
__device__ __forceinline__ void st8(uint8_t* p, const float (&v)[E], float s, int n) {
  float q[E];
#pragma unroll
  for (int j = 0; j < E; j++) {
    const float x = __fdiv_rn(v[j], s);
    q[j] = x != x ? x : fminf(fmaxf(x, -448.f), 448.f);
  }
  int w[E / 4];
#pragma unroll
  for (int h = 0; h < E / 4; h++) {
    w[h] = __builtin_amdgcn_cvt_pk_fp8_f32(q[4 * h], q[4 * h + 1], 0, false);
    w[h] = __builtin_amdgcn_cvt_pk_fp8_f32(q[4 * h + 2], q[4 * h + 3], w[h], true);
  }
  if (n >= E) {
    __builtin_memcpy(p, w, E);
  } else {
#pragma unroll
    for (int j = 0; j < E; j++)
      if (j < n) p[j] = (uint8_t)(w[j >> 2] >> (8 * (j & 3)));
  }
}

// cos and sin of p t turns, times f
__device__ __forceinline__ float2 turn(double pos, double t, float f, float sign) {
  const double x = pos * t;
  const double q = rint(4.0 * x);
  const float r = (float)(__builtin_fma(-0.25, q, x) * 6.283185307179586476925);  // |r| <= pi / 4
  const int k = (int)(q - 4.0 * floor(0.25 * q));                                 // quarter, 0..3
  const float z = r * r;
  const float s = r * (1.f + z * (-1.f / 6 + z * (1.f / 120 + z * (-1.f / 5040 + z * (1.f / 362880)))));
  const float c = 1.f + z * (-0.5f + z * (1.f / 24 + z * (-1.f / 720 + z * (1.f / 40320 - z * (1.f / 3628800)))));
  const float co = (k & 1) ? s : c, si = (k & 1) ? c : s;
  return make_float2(f * ((k == 1 || k == 2) ? -co : co), f * sign * (k >= 2 ? -si : si));
}

// CT: the cache's type (DT or UB_E4M3), -1 without a cache.
template <int DT, bool INTER, int CT>
__global__ void __launch_bounds__(NT) k_rope(const RopeDev d) {
  typedef typename Elem<DT>::T T;
  constexpr int E = Elem<DT>::E;
  constexpr bool APPEND = CT >= 0;
  extern __shared__ float2 cs[];
  const UbridgeRopeArgs& a = d.a;
  const int tid = threadIdx.x;
  const int t = blockIdx.x / d.parts, part = blockIdx.x - t * d.parts;
  const int half = a.rot / 2;
  const int lanes = 1 << d.lg, ul = tid & (lanes - 1);
  const int hstep = (NT >> d.lg) * d.parts;
  const int h0 = (tid >> d.lg) * d.parts + part;

  // where head h of the token lies, and its number of units
  const int PU = INTER ? 0 : (half + E - 1) / E;          // units of pairs
  const int nu_r = INTER ? (a.D + E - 1) / E : PU + (a.D - a.rot + E - 1) / E;
  const int nu_v = (a.D + E - 1) / E;
  auto head = [&](int h) -> const T* {
    if (h < a.Hq) return (const T*)a.q + t * a.q_st + h * a.q_sh;
    h -= a.Hq;
    if (h < a.Hkv) return (const T*)a.k + t * a.k_st + h * a.k_sh;
    return (const T*)a.v + t * a.v_st + (h - a.Hkv) * a.v_sh;
  };
  float x0[E], x1[E];
  // unit u of a rotated head: E pairs (x0, x1), or E elements (x0) that pass
  // through or (interleaved) hold E / 2 pairs
  auto load = [&](int h, int u) {
    const T* p = head(h);
    if (APPEND && h >= a.Hq + a.Hkv) {
      ld<DT>(x0, p + u * E, a.D - u * E);
    } else if (INTER) {
      ld<DT>(x0, p + u * E, a.D - u * E);
    } else if (u < PU) {
      ld<DT>(x0, p + u * E, half - u * E);
      ld<DT>(x1, p + half + u * E, half - u * E);
    } else {
      const int e = a.rot + (u - PU) * E;
      ld<DT>(x0, p + e, a.D - e);
    }
  };
  auto units = [&](int h) { return APPEND && h >= a.Hq + a.Hkv ? nu_v : nu_r; };
  int h = h0, u = ul;
  while (h < d.heads && u >= units(h)) h += hstep;  // (lanes past this head's units)
  const bool first = h < d.heads;
  if (first) load(h, u);

  const long pos = a.rot == 0 ? 0 : a.pos64 ? ((const long*)a.positions)[t] : (long)((const int*)a.positions)[t];
  for (int i = tid; i < half; i += NT)
    cs[i] = turn((double)pos, a.turns[i], a.factor, a.inverse ? -1.f : 1.f);
  long slot = 0;
  if constexpr (APPEND) {
    slot = a.slots[t];
    if (slot >= (long)a.P * a.S) {  // out of the cache: reported, not stored
      if (tid == 0 && part == 0) *d.err = UB_ERR_INDEX;
      slot = -1;
    }
  }
  __syncthreads();
  if (!first) return;
  const long page = APPEND && slot >= 0 ? slot / a.S : 0;
  const int at = APPEND && slot >= 0 ? (int)(slot - page * a.S) : 0;

  auto put = [&](int h, int e, const float (&v)[E], int n) {
    if (h < a.Hq) {
      st<DT>((T*)a.q_out + ((long)t * a.Hq + h) * a.D + e, v, n);
    } else if constexpr (!APPEND) {
      st<DT>((T*)a.k_out + ((long)t * a.Hkv + h - a.Hq) * a.D + e, v, n);
    } else {
      if (slot < 0) return;
      const bool key = h < a.Hq + a.Hkv;
      const int g = h - a.Hq - (key ? 0 : a.Hkv);
      const long o = page * a.page_stride + ((long)g * a.S + at) * a.D + e;
      void* base = key ? a.k_pages : a.v_pages;
      if constexpr (CT == UB_E4M3) {
        const float* sc = key ? a.k_scale : a.v_scale;
        st8<E>((uint8_t*)base + o, v, sc ? sc[g] : 1.f, n);
      } else {
        st<DT>((T*)base + o, v, n);
      }
    }
  };
  for (;;) {
    if (APPEND && h >= a.Hq + a.Hkv) {
      put(h, u * E, x0, a.D - u * E);
    } else if (INTER) {
      float y[E];
#pragma unroll
      for (int j = 0; j < E; j += 2) {
        const int p = (u * E + j) / 2;
        const float2 c = p < half ? cs[p] : make_float2(1.f, 0.f);
        y[j] = p < half ? x0[j] * c.x - x0[j + 1] * c.y : x0[j];
        y[j + 1] = p < half ? x0[j + 1] * c.x + x0[j] * c.y : x0[j + 1];
      }
      put(h, u * E, y, a.D - u * E);
    } else if (u < PU) {
      float y0[E], y1[E];
#pragma unroll
      for (int j = 0; j < E; j++) {
        const float2 c = cs[min(u * E + j, half - 1)];
        y0[j] = x0[j] * c.x - x1[j] * c.y;
        y1[j] = x1[j] * c.x + x0[j] * c.y;
      }
      put(h, u * E, y0, half - u * E);
      put(h, half + u * E, y1, half - u * E);
    } else {
      const int e = a.rot + (u - PU) * E;
      put(h, e, x0, a.D - e);
    }
    u += lanes;
    while (h < d.heads && u >= units(h)) h += hstep, u = ul;
    if (h >= d.heads) break;
    load(h, u);
  }
}

template <int DT, bool INTER>
void launch(const RopeDev& d, int ct, hipStream_t s) {
  const dim3 grid((unsigned)d.a.T * d.parts);
  const size_t lds = sizeof(float2) * (size_t)(d.a.rot / 2 > 0 ? d.a.rot / 2 : 1);
  if (ct < 0) k_rope<DT, INTER, -1><<<grid, NT, lds, s>>>(d);
  else if (ct == UB_E4M3) k_rope<DT, INTER, UB_E4M3><<<grid, NT, lds, s>>>(d);
  else k_rope<DT, INTER, DT><<<grid, NT, lds, s>>>(d);
}

int rope(const char* nm, const UbridgeRopeArgs* p, bool append, void* stream) {
  UB_REQUIRE(p, "%s: null argument block", nm);
  const UbridgeRopeArgs& a = *p;
  UB_REQUIRE(a.dtype == UB_F32 || a.dtype == UB_F16 || a.dtype == UB_BF16, "%s: dtype %d", nm, a.dtype);
  UB_REQUIRE(a.T >= 0 && a.Hq >= 0 && a.Hkv >= 0 && a.D > 0 && a.D <= 4096, "%s: T=%d Hq=%d Hkv=%d D=%d",
             nm, a.T, a.Hq, a.Hkv, a.D);
  UB_REQUIRE(a.rot >= 0 && a.rot % 2 == 0 && a.rot <= a.D, "%s: rot=%d of D=%d (even, at most D)", nm,
             a.rot, a.D);
  if (a.T == 0 || a.Hq + a.Hkv == 0) return UB_OK;
  UB_REQUIRE(a.rot == 0 || (a.positions && a.turns), "%s: null positions or turns", nm);
  UB_REQUIRE((a.Hq == 0 || (a.q && a.q_out)) && (a.Hkv == 0 || a.k), "%s: null q or k", nm);
  if (append) {
    UB_REQUIRE(a.cache_dtype == UB_E4M3 || a.cache_dtype == a.dtype, "%s: cache type %d for inputs of type %d",
               nm, a.cache_dtype, a.dtype);
    UB_REQUIRE(a.S > 0 && a.P >= 0 && a.slots, "%s: S=%d P=%d", nm, a.S, a.P);
    UB_REQUIRE(a.Hkv == 0 || (a.v && a.k_pages && a.v_pages), "%s: null v or pages", nm);
  } else {
    UB_REQUIRE(a.Hkv == 0 || a.k_out, "%s: null k_out", nm);
  }
  RopeDev d;
  d.a = a;
  d.heads = a.Hq + (append ? 2 : 1) * a.Hkv;
  d.err = append ? ub_error_flag() : nullptr;
  UB_REQUIRE(!append || d.err, "%s: no device flag", nm);
  const int E = a.dtype == UB_F32 ? 4 : 8;
  int nu = a.interleaved ? ub_cdiv(a.D, E) : ub_cdiv(a.rot / 2, E) + ub_cdiv(a.D - a.rot, E);
  if (append && nu < ub_cdiv(a.D, E)) nu = ub_cdiv(a.D, E);
  d.lg = 0;
  while ((1 << d.lg) < nu && d.lg < 8) d.lg++;
  // parts: workgroups of one token while that leaves CUs idle and a part still
  // fills its threads
  const int rounds = ub_cdiv(d.heads, NT >> d.lg);
  d.parts = 1;
  while (d.parts * 2 <= rounds && (long)a.T * d.parts < 512) d.parts *= 2;
  UB_REQUIRE((uint64_t)a.T * d.parts * NT < 1ull << 32, "%s: T=%d", nm, a.T);
  hipStream_t s = ub_stream(stream);
  const int ct = append ? a.cache_dtype : -1;
#define UB_GO(DT)                                   \
  {                                                 \
    if (a.interleaved) launch<DT, true>(d, ct, s);  \
    else launch<DT, false>(d, ct, s);               \
  }
  if (a.dtype == UB_F32) UB_GO(UB_F32)
  else if (a.dtype == UB_F16) UB_GO(UB_F16)
  else UB_GO(UB_BF16)
#undef UB_GO
  return ub_check_launch(nm);
}

}  // namespace

UB_API int ubridge_rope(const UbridgeRopeArgs* args, void* stream) {
  return rope("ubridge_rope", args, false, stream);
}
UB_API int ubridge_rope_append(const UbridgeRopeArgs* args, void* stream) {
  return rope("ubridge_rope_append", args, true, stream);
}
