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
// A wavefront turns the heads of one token, or a part of them where there are too
// few tokens to fill the CUs, and no wavefront waits for another.  Lanes stand
// for 16-byte units of a head, so a lane's pairs are the same in every head: one
// sine and cosine a pair and token, made by 64 lanes at once and dealt out
// through LDS, then in registers for all heads.  HBM-bound: the next head's loads
// are in flight while one is turned, in many wavefronts a SIMD.  8192 tokens of 40
// heads of 128 in bf16, 168 MB in and out: 31 us (5.4 TB/s, where copies reach 5.2
// to 5.5); 32 tokens stored into a cache 4.2 us, which is latency.
#include "common.h"

namespace {

constexpr int NW = 4;  // wavefronts of a workgroup

struct RopeDev {
  UbridgeRopeArgs a;
  int heads;    // q, k and (append) v heads of a token
  int parts;    // wavefronts a token
  int lg;       // log2 of the lanes of a head
  int* err;
};

template <int DT> struct Elem;  // element type and elements of a 16-byte unit
template <> struct Elem<UB_F32> { typedef float T; static constexpr int E = 4; };
template <> struct Elem<UB_F16> { typedef uint16_t T; static constexpr int E = 8; };
template <> struct Elem<UB_BF16> { typedef uint16_t T; static constexpr int E = 8; };

// Unit u of a run of `len` elements: its first element.  The last unit of a run
// that is not whole units ends with the run and overlaps the one before (the
// same values twice), unless the run is shorter than a unit.
template <int E, bool WHOLE>
__device__ __forceinline__ int place(int u, int len) { return WHOLE ? u * E : max(0, min(u * E, len - E)); }

// n elements from p, at most a unit (element-aligned: gfx950 loads 16 bytes
// from there)
template <int DT, bool WHOLE>
__device__ __forceinline__ uint4 ld(const typename Elem<DT>::T* p, int n) {
  constexpr int E = Elem<DT>::E;
  uint4 v = make_uint4(0, 0, 0, 0);
  if (WHOLE || n >= E) {
    __builtin_memcpy(&v, p, 16);
  } else {
    typename Elem<DT>::T x[E];  // (all in flight at once)
#pragma unroll
    for (int e = 0; e < E; e++) x[e] = p[min(e, n - 1)];
    uint64_t lo = 0, hi = 0;
    constexpr int B = 8 * sizeof(typename Elem<DT>::T);
#pragma unroll
    for (int e = 0; e < E; e++) {
      uint64_t b;
      if constexpr (DT == UB_F32) b = __float_as_uint(x[e]);
      else b = x[e];
      if (e >= n) b = 0;
      if (e < E / 2) lo |= b << (B * e);
      else hi |= b << (B * (e - E / 2));
    }
    v = make_uint4((uint32_t)lo, (uint32_t)(lo >> 32), (uint32_t)hi, (uint32_t)(hi >> 32));
  }
  return v;
}
template <int DT>
__device__ __forceinline__ float get(const uint4& w, int e) {
  const uint32_t p[4] = {w.x, w.y, w.z, w.w};
  if constexpr (DT == UB_F32) return __uint_as_float(p[e]);
  else if constexpr (DT == UB_F16) return ub_f16_to_f32((uint16_t)(p[e >> 1] >> (16 * (e & 1))));
  else return __uint_as_float((e & 1) ? p[e >> 1] & 0xffff0000u : p[e >> 1] << 16);
}

template <int DT>
__device__ __forceinline__ uint4 pack(const float (&v)[Elem<DT>::E]) {
  if constexpr (DT == UB_F32) {
    return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
  } else {
    uint32_t w[4];
    typedef float f32x2 __attribute__((ext_vector_type(2)));
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const f32x2 x = {v[2 * i], v[2 * i + 1]};
      if constexpr (DT == UB_BF16) {
        typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
        w[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector(x, bf16x2));
      } else {
        typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
        w[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector(x, f16x2));
      }
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
}
template <int DT, bool WHOLE>
__device__ __forceinline__ void st(typename Elem<DT>::T* p, const uint4& v, int n) {
  constexpr int E = Elem<DT>::E;
  if (WHOLE || n >= E) {
    __builtin_memcpy(p, &v, 16);
  } else {
    uint64_t lo = (uint64_t)v.y << 32 | v.x, hi = (uint64_t)v.w << 32 | v.z;
    constexpr int B = 8 * sizeof(typename Elem<DT>::T);
#pragma nounroll
    for (int e = 0; e < n; e++) {
      if (e == E / 2) lo = hi;
      if constexpr (DT == UB_F32) p[e] = __uint_as_float((uint32_t)lo);
      else p[e] = (uint16_t)lo;
      lo >>= B;
    }
  }
}

// x / s to e4m3, saturating, NaN kept
template <int E, bool WHOLE>
__device__ __forceinline__ void st8(uint8_t* p, const float (&v)[E], float s, int n) {
  uint32_t w[E / 4];
#pragma unroll
  for (int h = 0; h < E / 4; h++) {
    float q[4];
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const float x = __fdiv_rn(v[4 * h + j], s);
      q[j] = x != x ? x : fminf(fmaxf(x, -448.f), 448.f);
    }
    w[h] = __builtin_amdgcn_cvt_pk_fp8_f32(q[0], q[1], 0, false);
    w[h] = __builtin_amdgcn_cvt_pk_fp8_f32(q[2], q[3], w[h], true);
  }
  if (WHOLE || n >= E) {
    __builtin_memcpy(p, w, E);
  } else {
    uint64_t x = w[0];
    if constexpr (E == 8) x |= (uint64_t)w[1] << 32;
#pragma nounroll
    for (int j = 0; j < n; j++, x >>= 8) p[j] = (uint8_t)x;
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

struct Two { uint4 a, b; };

// CT: the cache's type (DT or UB_E4M3), -1 without a cache.  WHOLE: every run is
// whole units (without the code for other runs the kernel needs 20 registers
// less: 8192 tokens of 40 heads of 128 36.9 us a call, in the general form 39.7).
template <int DT, bool INTER, int CT, bool WHOLE>
__global__ void __launch_bounds__(64 * NW) k_rope(const RopeDev d) {
  typedef typename Elem<DT>::T T;
  constexpr int E = Elem<DT>::E, NP = INTER ? E / 2 : E;  // pairs of a unit
  constexpr bool APPEND = CT >= 0;
  extern __shared__ float2 lds[];
  const UbridgeRopeArgs& a = d.a;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const unsigned id = blockIdx.x * NW + wave;
  const int t = (int)(id / (unsigned)d.parts), part = (int)(id - (unsigned)t * d.parts);
  if (t >= a.T) return;
  const int half = a.rot / 2;
  float2* cs = lds + wave * (half > 0 ? half : 1);
  const int lanes = 1 << d.lg, ul = lane & (lanes - 1);
  const int step = (64 >> d.lg) * d.parts;

  const int PU = INTER ? 0 : (half + E - 1) / E;  // units of pairs, ahead of those that pass through
  const int nu_r = INTER ? (a.D + E - 1) / E : PU + (a.D - a.rot + E - 1) / E;
  const int nu_v = (a.D + E - 1) / E;
  const int hr = a.Hq + a.Hkv;  // heads that turn
  const T* const qt = (const T*)a.q + t * a.q_st;
  const T* const kt = (const T*)a.k + t * a.k_st;
  const T* const vt = (const T*)a.v + t * a.v_st;
  const long pos = a.rot == 0 ? 0 : a.pos64 ? ((const long*)a.positions)[t] : (long)((const int*)a.positions)[t];
  long slot = APPEND ? a.slots[t] : 0;

  // unit u of head h: E pairs (a, b), or E elements (a) that pass through or
  // (interleaved) hold E / 2 pairs
  struct Where { int e, n; bool pairs; };
  auto where = [&](int h, int u) {
    Where w;
    w.pairs = !INTER && h < hr && u < PU;
    if (w.pairs) {
      w.e = place<E, WHOLE>(u, half);
      w.n = half - w.e;
    } else if (INTER && !WHOLE && (a.D & 1) && h < hr) {  // (whole pairs a unit)
      w.e = u * E;
      w.n = a.D - w.e;
    } else {
      const int from = INTER || h >= hr ? 0 : a.rot;
      w.e = from + place<E, WHOLE>(from ? u - PU : u, a.D - from);
      w.n = a.D - w.e;
    }
    return w;
  };
  Where at_q;  // of the unit at hand: the same in every head that turns
  auto load = [&](int h, int u) {
    const T* p = h < a.Hq ? qt + h * a.q_sh : h < hr ? kt + (h - a.Hq) * a.k_sh : vt + (h - hr) * a.v_sh;
    const Where w = !APPEND || h < hr ? at_q : where(h, u);
    Two r;
    r.a = ld<DT, WHOLE>(p + w.e, w.n);
    r.b = make_uint4(0, 0, 0, 0);
    if (!INTER && w.pairs) r.b = ld<DT, WHOLE>(p + half + w.e, w.n);
    return r;
  };
  long page = 0;
  int at = 0;
  auto put = [&](int h, int e, const float (&v)[E], int n) {
    if (h < a.Hq) {
      st<DT, WHOLE>((T*)a.q_out + ((long)t * a.Hq + h) * a.D + e, pack<DT>(v), n);
    } else if constexpr (!APPEND) {
      st<DT, WHOLE>((T*)a.k_out + ((long)t * a.Hkv + h - a.Hq) * a.D + e, pack<DT>(v), n);
    } else {
      if (slot < 0) return;
      const bool key = h < hr;
      const int g = h - (key ? a.Hq : hr);
      const long o = page * a.page_stride + ((long)g * a.S + at) * a.D + e;
      void* base = key ? a.k_pages : a.v_pages;
      if constexpr (CT == UB_E4M3) {
        const float* sc = key ? a.k_scale : a.v_scale;
        st8<E, WHOLE>((uint8_t*)base + o, v, sc ? sc[g] : 1.f, n);
      } else {
        st<DT, WHOLE>((T*)base + o, pack<DT>(v), n);
      }
    }
  };

  // this lane's heads of unit u: from h on, below end
  int h = 0, end = 0;
  auto range = [&](int u) {
    h = (lane >> d.lg) * d.parts + part;
    end = u < nu_r ? (APPEND && u < nu_v ? d.heads : hr) : u < nu_v ? d.heads : 0;
    if (u >= nu_r && h < hr) h += (hr - h + step - 1) / step * step;  // (only v has this unit)
    at_q = where(0, u);
  };
  Two x = {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
  int u = ul;
  range(u);
  if (h < end) x = load(h, u);
  for (int i = lane; i < half; i += 64)
    cs[i] = turn((double)pos, a.turns[i], a.factor, a.inverse ? -1.f : 1.f);
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();  // (a wavefront's LDS accesses are in order)
  if constexpr (APPEND) {
    if (slot >= (long)a.P * a.S) {  // out of the cache: reported, not stored
      if (lane == 0 && part == 0) *d.err = UB_ERR_INDEX;
      slot = -1;
    }
    page = slot >= 0 ? slot / a.S : 0;
    at = slot >= 0 ? (int)(slot - page * a.S) : 0;
  }
  const int nu = APPEND && nu_v > nu_r ? nu_v : nu_r;
  while (u < nu) {
    float2 w[NP];  // of this unit's pairs
#pragma unroll
    for (int j = 0; j < NP; j++) {
      const int i = (INTER ? at_q.e / 2 : at_q.e) + j;
      w[j] = i < half ? cs[i] : make_float2(1.f, 0.f);
    }
    while (h < end) {
      const uint4 c0 = x.a, c1 = x.b;
      const int hi = h;
      h += step;
      if (h < end) x = load(h, u);
      float y[E];
      const Where v = !APPEND || hi < hr ? at_q : where(hi, u);
      if (INTER && hi < hr) {
#pragma unroll
        for (int j = 0; j < E; j += 2) {  // (pairs past rot turn by nothing)
          const float x = get<DT>(c0, j), z = get<DT>(c0, j + 1);
          const bool in = v.e + j < a.rot;
          y[j] = in ? x * w[j / 2].x - z * w[j / 2].y : x;
          y[j + 1] = in ? z * w[j / 2].x + x * w[j / 2].y : z;
        }
      } else if (!INTER && v.pairs) {
#pragma unroll
        for (int j = 0; j < E; j++) y[j] = get<DT>(c1, j) * w[j % NP].x + get<DT>(c0, j) * w[j % NP].y;
        put(hi, half + v.e, y, v.n);
#pragma unroll
        for (int j = 0; j < E; j++) y[j] = get<DT>(c0, j) * w[j % NP].x - get<DT>(c1, j) * w[j % NP].y;
      } else {
#pragma unroll
        for (int j = 0; j < E; j++) y[j] = get<DT>(c0, j);
      }
      put(hi, v.e, y, v.n);
    }
    u += lanes;
    range(u);
    if (h < end) x = load(h, u);
  }
}

template <int DT, bool INTER, bool WHOLE>
void launch(const RopeDev& d, int ct, hipStream_t s) {
  const dim3 grid(ub_cdiv((long)d.a.T * d.parts, NW));
  const size_t lds = sizeof(float2) * NW * (size_t)(d.a.rot / 2 > 0 ? d.a.rot / 2 : 1);
  if (ct < 0) k_rope<DT, INTER, -1, WHOLE><<<grid, 64 * NW, lds, s>>>(d);
  else if (ct == UB_E4M3) k_rope<DT, INTER, UB_E4M3, WHOLE><<<grid, 64 * NW, lds, s>>>(d);
  else k_rope<DT, INTER, DT, WHOLE><<<grid, 64 * NW, lds, s>>>(d);
}
template <int DT>
void launch(const RopeDev& d, int ct, hipStream_t s) {
  constexpr int E = Elem<DT>::E;
  const bool whole = d.a.D % E == 0 && (d.a.interleaved || (d.a.rot / 2 % E == 0 && (d.a.D - d.a.rot) % E == 0));
  if (d.a.interleaved && whole) launch<DT, true, true>(d, ct, s);
  else if (d.a.interleaved) launch<DT, true, false>(d, ct, s);
  else if (whole) launch<DT, false, true>(d, ct, s);
  else launch<DT, false, false>(d, ct, s);
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
  while ((1 << d.lg) < nu && d.lg < 6) d.lg++;
  // parts: as many wavefronts a token as have a head each, while the CUs are not
  // full (8192 tokens of 40 heads of 128: one, 32 tokens of 48: six)
  const int rounds = ub_cdiv(d.heads, 64 >> d.lg);
  d.parts = 1;
  while (d.parts < rounds && (long)a.T * d.parts < 4096) d.parts++;
  UB_REQUIRE((uint64_t)a.T * d.parts * 64 < 1ull << 32, "%s: T=%d", nm, a.T);
  hipStream_t s = ub_stream(stream);
  const int ct = append ? a.cache_dtype : -1;
  if (a.dtype == UB_F32) launch<UB_F32>(d, ct, s);
  else if (a.dtype == UB_F16) launch<UB_F16>(d, ct, s);
  else launch<UB_BF16>(d, ct, s);
  return ub_check_launch(nm);
}

}  // namespace

UB_API int ubridge_rope(const UbridgeRopeArgs* args, void* stream) {
  return rope("ubridge_rope", args, false, stream);
}
UB_API int ubridge_rope_append(const UbridgeRopeArgs* args, void* stream) {
  return rope("ubridge_rope_append", args, true, stream);
}
