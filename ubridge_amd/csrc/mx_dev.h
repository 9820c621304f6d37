// mx_dev.h -- microscaled blocks: 32 values under one power of two (e8m0 byte),
// elements e2m1 (two a byte, the even one low) or e4m3.  Shared by mx.hip and
// norm.hip.
//
// The power of two is 2^(floor(log2 amax) - emax), emax the exponent of the
// format's largest binade (2 or 8), held to bytes 0 .. 254 (2^-127 .. 2^127); an
// element is x / 2^e to the nearest, ties to even, values past the largest to the
// largest.  A block with an infinity or a NaN has the byte 255, which makes every
// value NaN, and codes 0.  All of it is exact: there is no rounding ahead of the
// one to the element.
#pragma once
#include "common.h"

namespace {

enum { MX_FP4 = 4, MX_FP8 = 8 };  // element bits

// The byte of a block from the bits (without sign) of its largest magnitude in f32:
// the biased exponent less emax.  Denormals lie below every byte.
template <int F>
__device__ __forceinline__ uint32_t mx_byte(uint32_t top) {
  constexpr uint32_t emax = F == MX_FP4 ? 2 : 8;
  const uint32_t e = top >> 23;
  return e == 255 ? 255u : e > emax ? e - emax : 0u;
}
// 2^(byte - 127)
__device__ __forceinline__ float mx_unit(uint32_t byte) {
  return __uint_as_float(byte ? byte << 23 : 0x00400000u);
}

// Codes of four values (four e2m1 in 16 bits, four e4m3 in 32).  The instructions
// divide by the unit and round to even; e2m1 saturates by itself, e4m3 gives NaN
// past 464, so values are held to the largest first (a block reaches 512 units).
template <int F>
__device__ __forceinline__ uint32_t mx_codes4(float a, float b, float c, float d, uint32_t byte) {
  if (byte == 255) return 0;
  const float u = mx_unit(byte);
  if constexpr (F == MX_FP4) {
    uint32_t o = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, a, b, u, 0);
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(o, c, d, u, 1) & 0xffffu;
  } else {
    typedef short i16x2 __attribute__((ext_vector_type(2)));
    const float m = 448.f * u;
    auto hold = [&](float v) { return fminf(fmaxf(v, -m), m); };
    i16x2 o = {0, 0};
    o = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(o, hold(a), hold(b), u, false);
    o = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(o, hold(c), hold(d), u, true);
    return __builtin_bit_cast(uint32_t, o);
  }
}

// Largest of the 4 or 8 neighbouring lanes that hold a block.
template <int LANES>
__device__ __forceinline__ uint32_t mx_top(uint32_t v) {
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xf, 0xf, false));  // quad_perm [1,0,3,2]
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xf, 0xf, false));  // quad_perm [2,3,0,1]
  if constexpr (LANES == 8)
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x141, 0xf, 0xf, false));  // row_half_mirror
  return v;
}

// A row as 16-byte units of E elements: unit i of the row at p, `C` elements long;
// zeros from C on.  The row may start at any element (gfx950 loads 16 bytes from
// there).  The last, partial unit is the row's last E elements shifted down.
template <int DT> struct MxElem { typedef uint16_t T; static constexpr int E = 8; };
template <> struct MxElem<UB_F32> { typedef float T; static constexpr int E = 4; };

template <int DT>
__device__ __forceinline__ uint4 mx_unit_at(const typename MxElem<DT>::T* p, int i, int C) {
  typedef typename MxElem<DT>::T T;
  constexpr int E = MxElem<DT>::E;
  const int at = i * E;
  uint4 v = make_uint4(0, 0, 0, 0);
  if (at + E <= C) {
    __builtin_memcpy(&v, p + at, 16);
  } else if (at < C) {
    if (C >= E) {
      unsigned __int128 w;
      __builtin_memcpy(&w, p + C - E, 16);
      w >>= 8 * sizeof(T) * (at + E - C);
      __builtin_memcpy(&v, &w, 16);
    } else {
      T w[E] = {};
      for (int e = 0; e < E; e++)
        if (e < C) w[e] = p[e];
      __builtin_memcpy(&v, w, 16);
    }
  }
  return v;
}
template <int DT>
__device__ __forceinline__ float mx_get(const uint4& w, int e) {
  const uint32_t p[4] = {w.x, w.y, w.z, w.w};
  if constexpr (DT == UB_F32) return __uint_as_float(p[e]);
  else if constexpr (DT == UB_F16) return ub_f16_to_f32((uint16_t)(p[e >> 1] >> (16 * (e & 1))));
  else return __uint_as_float((e & 1) ? p[e >> 1] & 0xffff0000u : p[e >> 1] << 16);
}
// E values to a unit of type DT, each rounded once
template <int DT>
__device__ __forceinline__ uint4 mx_pack(const float* f) {
  if constexpr (DT == UB_F32) {
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
  } else {
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
    uint32_t o[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const f32x2 v = {f[2 * i], f[2 * i + 1]};
      if constexpr (DT == UB_BF16) o[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector(v, bf16x2));
      else o[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector(v, f16x2));
    }
    return make_uint4(o[0], o[1], o[2], o[3]);
  }
}
// Stores unit i of the row at p; of the last, partial one only what lies in the row.
template <int DT>
__device__ __forceinline__ void mx_put(typename MxElem<DT>::T* p, int i, int C, const uint4& v) {
  typedef typename MxElem<DT>::T T;
  constexpr int E = MxElem<DT>::E;
  const int at = i * E;
  if (at + E <= C) {
    __builtin_memcpy(p + at, &v, 16);
  } else if (at < C) {
    T w[E];
    __builtin_memcpy(w, &v, 16);
#pragma unroll
    for (int e = 0; e < E; e++)
      if (at + e < C) p[at + e] = w[e];
  }
}

// Rounds the E values of a unit, one of the 4 or 8 neighbouring lanes' that make a
// block (all of them here): codes in o (e2m1 in o[0]), returns the block's byte.  16-bit
// values stay packed: the largest magnitude by integer maxima, the elements by the
// instructions that take pairs, half the operations of going through f32.
template <int DT, int F>
__device__ __forceinline__ uint32_t mx_round(const uint4& v, uint32_t (&o)[2]) {
  typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
  typedef short i16x2 __attribute__((ext_vector_type(2)));
  typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
  typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
  o[0] = o[1] = 0;
  if constexpr (DT == UB_F32) {
    float f[4];
    uint32_t t = 0;
#pragma unroll
    for (int e = 0; e < 4; e++) {
      f[e] = mx_get<DT>(v, e);
      t = max(t, __float_as_uint(f[e]) & 0x7fffffffu);
    }
    const uint32_t b = mx_byte<F>(mx_top<8>(t));
    o[0] = mx_codes4<F>(f[0], f[1], f[2], f[3], b);
    return b;
  } else {
    uint32_t w[4] = {v.x, v.y, v.z, v.w};
    u16x2 m = {0, 0};
#pragma unroll
    for (int i = 0; i < 4; i++) m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, w[i] & 0x7fff7fffu));
    const uint32_t top = mx_top<4>(max((uint32_t)m[0], (uint32_t)m[1]));
    const uint32_t b = mx_byte<F>(DT == UB_BF16 ? top << 16 : __float_as_uint(ub_f16_to_f32((uint16_t)top)));
    if (b == 255) return b;
    const float u = mx_unit(b);
    if constexpr (F == MX_FP8) {  // held to 448 units (f16: to what it has below that)
      uint32_t lim;
      if constexpr (DT == UB_BF16) lim = ((b + 8) << 7 | 0x60) * 0x10001u;
      else lim = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(448.f * u, 448.f * u));
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const u16x2 a = __builtin_elementwise_min(__builtin_bit_cast(u16x2, w[i] & 0x7fff7fffu), __builtin_bit_cast(u16x2, lim));
        w[i] = __builtin_bit_cast(uint32_t, a) | (w[i] & 0x80008000u);
      }
    }
    auto pair = [&](int i) {
      if constexpr (DT == UB_BF16) return __builtin_bit_cast(bf16x2, w[i]);
      else return __builtin_bit_cast(f16x2, w[i]);
    };
    if constexpr (F == MX_FP4 && DT == UB_BF16) {
      o[0] = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(0u, pair(0), u, 0);
      o[0] = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(o[0], pair(1), u, 1);
      o[0] = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(o[0], pair(2), u, 2);
      o[0] = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(o[0], pair(3), u, 3);
    } else if constexpr (F == MX_FP4) {
      o[0] = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(0u, pair(0), u, 0);
      o[0] = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(o[0], pair(1), u, 1);
      o[0] = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(o[0], pair(2), u, 2);
      o[0] = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(o[0], pair(3), u, 3);
    } else {
#pragma unroll
      for (int h = 0; h < 2; h++) {
        i16x2 c = {0, 0};
        if constexpr (DT == UB_BF16) {
          c = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(c, pair(2 * h), u, false);
          c = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(c, pair(2 * h + 1), u, true);
        } else {
          c = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(c, pair(2 * h), u, false);
          c = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(c, pair(2 * h + 1), u, true);
        }
        o[h] = __builtin_bit_cast(uint32_t, c);
      }
    }
    return b;
  }
}
template <int DT, int F>
__device__ __forceinline__ void mx_store(uint8_t* p, const uint32_t (&o)[2]) {
  if constexpr (DT == UB_F32 && F == MX_FP4) *(uint16_t*)p = (uint16_t)o[0];
  else if constexpr (DT == UB_F32 || F == MX_FP4) *(uint32_t*)p = o[0];
  else *(uint2*)p = make_uint2(o[0], o[1]);
}

}  // namespace
