// moe_decode.hip -- a mixture-of-experts layer for up to 16 tokens in two launches
// (gfx950):
//
//   p = softmax(logits[t]),  the k largest (ties to the lowest expert), / their sum
//   a[t, j] = silu(g) u,     g, u = (w13[e] x[t]) rows [0, I), [I, 2 I)
//   y[t] = T(sum_j p_j (w2[e_j] a[t, j]))
//
// int8 weights are exact in T; their scales, the routed weights and all sums are f32.
// Only y is rounded to T.  a, an operand of the next product, is the sum of two bf16, its
// rounding and what that leaves: 2^-17 of it, over the range of f32 (one f16 would be
// infinite from 65520 on, where y need not be).  So the second product is of bf16: int8
// weights are exact there too, an f16 weight is the sum of two.
//
// A stream of the weights of the experts in use, read once each: bound by HBM where
// they are many, by the chain of latencies (logits, weights, sums; twice) for a token
// or two.  16 tokens are one operand of v_mfma_f32_16x16x32, so no rows are gathered
// and no list of blocks is built: a product is of 16 weight rows with every token, and
// an expert's result is kept for the tokens that chose it.
//  * k_up: every workgroup finds the top-k itself (a wavefront a token; 2.6 us of the
//    call, against a launch).  An item is 8 columns of an expert: 8 gate rows and their 8
//    up rows are the 16 rows of one product.  Groups of 8 or 16 wavefronts take the items
//    in turn and split K, each one run of its rows, two items in flight.
//  * k_down: a workgroup owns 8 or 16 output columns and adds all experts' parts, so no
//    sums cross workgroups.  16 rows of an expert are the rows of a product, both parts of
//    up to 8 tokens' a its columns (an expert with more is listed again).  Or, while there
//    are too few columns to give every CU 16, 8 rows of each of two experts, and up to 4
//    tokens of either: the two quarters where rows and tokens belong together are kept.
//  * Scales are asked for ahead of the weights that they go with: loads return in order,
//    and one asked for at the end of an item would wait for all weights in flight.
// Measured (medians), k_up + k_down: 16 tokens, 8 of 128 int8 experts of 2048 x 768 57 + 37 us
// (4.5 and 3.5 TB/s), 5 tokens, 6 of 64 f16 ones of 2048 x 1408 55 + 34 (5.2, 4.2), one token
// of the former 12 + 7.
#include "lds_dma.h"
#include "moe_dev.h"
#include "wave.h"

#include <algorithm>
#include <type_traits>

namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int kTok = 16, kK = 16, kE = 1024, kUsed = kTok * kK;  // most tokens, top-k, experts; experts in use
constexpr int kEnt = kUsed;  // entries of the list below: at most one a token and expert

// The routing, in scratch memory from k_up to k_down: experts in use, each with up to 4 or
// 8 (`per`) of its tokens (more: another entry): rows of the activations (t k + j; -1:
// none), tokens and weights, `per` to an entry.
struct Route {
  int n, pad[3];
  int expert[kEnt];
  int16_t row[kEnt * 8];
  int8_t tok[kEnt * 8];
  float w[kEnt * 8];
};

struct DecodeArgs {
  const void *x, *logits, *w13, *s13, *w2, *s2;
  void *y, *act;  // act: bf16 [T k][I / 8][2][8], a rounded and the rest
  Route* route;
  int T, E, k, H, I, ldt, norm, per;
};

template <int DT>
__device__ __forceinline__ f32x4 mfma(const uint4& a, const uint4& b, const f32x4& c) {
  if constexpr (DT == UB_BF16)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
// 16 bytes of a weight row by the activations that meet them: 16 int8 (two products)
// or 8 T
template <int DT, bool Q8>
__device__ __forceinline__ f32x4 product(const uint4& w, const uint4 (&x)[Q8 ? 2 : 1], f32x4 c) {
  if constexpr (Q8) {
    c = mfma<DT>(i8x8_to_t<DT>(w.x, w.y), x[0], c);
    return mfma<DT>(i8x8_to_t<DT>(w.z, w.w), x[1], c);
  } else {
    return mfma<DT>(w, x[0], c);
  }
}
// The same for the second product, of bf16: 16 int8, 8 bf16, or 8 f16 as the first 8 of
// their 11 bits and the rest
template <int DT, bool Q8>
__device__ __forceinline__ f32x4 product_bf16(const uint4& w, const uint4 (&x)[Q8 ? 2 : 1], f32x4 c) {
  if constexpr (Q8 || DT == UB_BF16) return product<UB_BF16, Q8>(w, x, c);
  else {
    const uint32_t p[4] = {w.x, w.y, w.z, w.w};
    uint32_t hi[4], lo[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const float a = ub_f16_to_f32((uint16_t)p[i]), b = ub_f16_to_f32((uint16_t)(p[i] >> 16));
      const uint32_t ha = __float_as_uint(a) & 0xffff0000u, hb = __float_as_uint(b) & 0xffff0000u;
      hi[i] = ha >> 16 | hb;
      lo[i] = __float_as_uint(a - __uint_as_float(ha)) >> 16 | (__float_as_uint(b - __uint_as_float(hb)) & 0xffff0000u);
    }
    c = mfma<UB_BF16>(make_uint4(lo[0], lo[1], lo[2], lo[3]), x[0], c);
    return mfma<UB_BF16>(make_uint4(hi[0], hi[1], hi[2], hi[3]), x[0], c);
  }
}
// 16 bytes of a weight row, as one vector (of a struct's four parts the conversions to T
// make loads byte by byte)
__device__ __forceinline__ uint4 ld16(const void* p) {
  typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
  return __builtin_bit_cast(uint4, *(const u32x4*)p);
}

// Token t's experts, by one wavefront holding its logits (expert lane + 64 j): f(round,
// expert, weight) in lane `round`.  A round is a maximum over the wavefront and, for
// the lowest expert that has it, a ballot for each j: every workgroup finds the top-k of
// all tokens, so what counts is the number of instructions.
template <int NPL, class F>
__device__ __forceinline__ void top_k(float (&v)[NPL], int k, int norm, F f) {
  const int lane = threadIdx.x & 63;
  float m = -INFINITY, all = 0.f, picked = -INFINITY;
  int which = 0, got = 0;
  for (int i = 0; i < k; i++) {
    float best = v[0];
#pragma unroll
    for (int j = 1; j < NPL; j++) best = fmaxf(best, v[j]);
    const float wb = ub_wave_all_max(best);
    if (wb == -INFINITY) break;
    if (i == 0) {
      m = wb;
      if (!norm) {
#pragma unroll
        for (int j = 0; j < NPL; j++) all += expf(v[j] - m);
        all = ub_wave_all_sum(all);
      }
    }
    bool found = false;
#pragma unroll
    for (int j = 0; j < NPL; j++) {
      const uint64_t has = __ballot(v[j] == wb);
      if (!found && has) {  // (the same in every lane)
        found = true;
        const int l = __builtin_ctzll(has);
        if (lane == l) v[j] = -INFINITY;
        if (lane == i) picked = wb, which = l + 64 * j;
      }
    }
    got++;
  }
  if (got == 0) return;
  const float p = lane < got ? expf(picked - m) : 0.f;
  if (norm) all = ub_wave_all_sum(p);
  if (lane < got) f(lane, which, p / all);
}

// SP: 64-byte steps of a row that a wavefront takes at once.  MULTI: K in several such
// pieces, the activations loaded with each; else they stay in registers.  NG groups of
// W1 wavefronts, 16 in all, have an item each: the routing is found once a CU.  NI: items
// side by side, taken together.
template <int DT, bool Q8, int NPL, int SP, bool MULTI, int NG, int NI>
__global__ void __launch_bounds__(1024) k_up(DecodeArgs a) {
  constexpr int NT = 1024, W1 = 16 / NG, NB = NI == 1 ? 2 : 1, CI = 8 * NI;  // CI: columns of an item and its neighbours
  constexpr int WB = Q8 ? 1 : 2, EL = 64 / WB, XN = Q8 ? 2 : 1;  // bytes of a weight; elements of a step; operands
  __shared__ __attribute__((aligned(16))) int8_t slot[kE][kTok];
  __shared__ uint16_t used[kUsed], tokens[kUsed], entry[kUsed];  // experts in use, their tokens (bits), first entries
  __shared__ int nused, nent;
  __shared__ __attribute__((aligned(16))) float red[NB][NG][NI][W1][16][20];
  const int tid = threadIdx.x, lane = tid & 63, r = lane & 15, h = lane >> 4;
  const int wv = __builtin_amdgcn_readfirstlane(tid >> 6), wave = wv % W1, grp = wv / W1;
  const int T = a.T, E = a.E, H = a.H, I = a.I;
  // ---- routing
  float lg[NPL];  // of token wv
#pragma unroll
  for (int j = 0; j < NPL; j++) {
    const int e = lane + 64 * j;
    float v = -INFINITY;
    if (wv < T && e < E) {
      const size_t at = (size_t)wv * E + e;
      v = a.ldt == UB_F32 ? ((const float*)a.logits)[at] : a.ldt == UB_F16 ? ub_load<UB_F16>(a.logits, at) : ub_load<UB_BF16>(a.logits, at);
      if (v != v) v = -INFINITY;
    }
    lg[j] = v;
  }
  // ---- activations of the wavefront's steps: lane (token r, h) takes what meets the
  // 16 bytes at 64 s + 16 h of a weight row
  uint4 xf[MULTI ? 1 : SP][XN];
  const int rowb = H * WB;
  auto acts = [&](uint4 (&o)[XN], int s) {
    const int at = s * 64 + 16 * h;  // byte of the row
#pragma unroll
    for (int u = 0; u < XN; u++) {
      o[u] = make_uint4(0, 0, 0, 0);
      if (r < T && at < rowb) o[u] = *(const uint4*)((const uint16_t*)a.x + (size_t)r * H + at / WB + 8 * u);
    }
  };
  if constexpr (!MULTI) {
#pragma unroll
    for (int i = 0; i < SP; i++) acts(xf[i], wave * SP + i);
  }
  for (int i = tid; i < E * kTok / 4; i += NT) ((int*)slot)[i] = -1;
  __syncthreads();
  const bool first = blockIdx.x == 0;
  __shared__ float wts[kTok][kK];
  if (wv < T)
    top_k<NPL>(lg, a.k, a.norm, [&](int j, int e, float w) {
      slot[e][wv] = (int8_t)j;
      wts[wv][j] = w;
    });
  __syncthreads();
  if (wv == 0) {
    int n = 0, m = 0;
    for (int e0 = 0; e0 < E; e0 += 64) {
      const int e = e0 + lane;
      uint32_t bits = 0;
      if (e < E) {
        const int4 v = *(const int4*)slot[e];
        const int w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int q = 0; q < 4; q++) {  // the sign bits of four bytes, together
          const uint32_t s = ~(uint32_t)w[q] & 0x80808080u;
          bits |= ((s >> 7 | s >> 14 | s >> 21 | s >> 28) & 15u) << (4 * q);
        }
      }
      const uint64_t one = __ballot(bits != 0), below = (1ull << lane) - 1;
      int ahead = 0, all = 0;  // entries of the lanes below, and of all
      for (int q = 0; q < kTok; q += a.per) {
        const uint64_t more = __ballot(__popc(bits) > q);
        ahead += __popcll(more & below);
        all += __popcll(more);
      }
      if (bits) {
        const int at = n + __popcll(one & below);
        used[at] = (uint16_t)e;
        tokens[at] = (uint16_t)bits;
        entry[at] = (uint16_t)(m + ahead);
      }
      n += __popcll(one);
      m += all;
    }
    if (lane == 0) nused = n, nent = m;
  }
  __syncthreads();
  const int nu = __builtin_amdgcn_readfirstlane(nused);
  if (first) {
    if (tid == 0) a.route->n = nent;
    for (int l = tid; l < nu * 16; l += NT) {
      const int u = l >> 4, p = l & 15, e = used[u], bits = tokens[u], n = __popc(bits), at = entry[u] + p / a.per;
      if (p >= (n + a.per - 1) / a.per * a.per) continue;
      int b = bits;  // the p-th token of the expert
      for (int q = 0; q < p; q++) b &= b - 1;
      const int t = b ? __builtin_ctz(b) : -1, j = t >= 0 ? slot[e][t] : 0;
      const int i = at * a.per + p % a.per;
      a.route->expert[at] = e;
      a.route->row[i] = (int16_t)(t >= 0 ? t * a.k + j : -1);
      a.route->tok[i] = (int8_t)t;
      a.route->w[i] = t >= 0 ? wts[t][j] : 0.f;
    }
  }
  // ---- items
  // (expert in use, 8 columns); all groups walk along one front, which memory likes better
  // than runs of their own
  const int nc = I / CI, G = gridDim.x * NG, run = blockIdx.x + grp * gridDim.x;
  const int items = nu * nc, longest = (items + G - 1) / G;  // the groups meet at one barrier an item
  const int pieces = MULTI ? ((rowb + 63) / 64 + W1 * SP - 1) / (W1 * SP) : 1;
  struct Set {
    uint4 w[SP][NI];
    uint4 x[MULTI ? SP : 1][XN];
    float sg, su;  // scales of the thread's output
  };
  const int gt = tid - grp * 64 * W1, ot = gt / CI, oc = gt % CI;  // its token and column
  auto load = [&](Set& b, int it, int p) {
    const int at0 = min(it, items - 1), u = at0 / nc, c = at0 - u * nc, e = used[u];
    if (Q8 && gt < CI * T && p == pieces - 1) {
      const size_t at = (size_t)e * 2 * I + CI * c + oc;
      b.sg = ub_load<DT>(a.s13, at);
      b.su = ub_load<DT>(a.s13, at + I);
    }
    const uint8_t* row = (const uint8_t*)a.w13 + ((size_t)e * 2 * I + (r < 8 ? CI * c + r : I + CI * c + r - 8)) * rowb;
#pragma unroll
    for (int i = 0; i < SP; i++) {
      const int s = p * W1 * SP + wave * SP + i, at = s * 64 + 16 * h;
#pragma unroll
      for (int n = 0; n < NI; n++) b.w[i][n] = make_uint4(0, 0, 0, 0);
      if (it < items && at < rowb) {
#pragma unroll
        for (int n = 0; n < NI; n++) b.w[i][n] = ld16(row + (size_t)n * 8 * rowb + at);
      }
      if constexpr (MULTI) acts(b.x[i], s);
    }
  };
  const int total = longest * pieces;
  auto item = [&](int q) { return (MULTI ? q / pieces : q) * G + run; };
  auto piece = [&](int q) { return MULTI ? q % pieces : 0; };
  f32x4 acc[NI];
#pragma unroll
  for (int n = 0; n < NI; n++) acc[n] = (f32x4){0.f, 0.f, 0.f, 0.f};
  // piece q, in b; then piece q + 2's loads
  auto mul = [&](Set& b, int q, int buf) {
    const int it = item(q);
#pragma unroll
    for (int i = 0; i < SP; i++)
#pragma unroll
      for (int n = 0; n < NI; n++) {
        if constexpr (MULTI) acc[n] = product<DT, Q8>(b.w[i][n], b.x[i], acc[n]);
        else acc[n] = product<DT, Q8>(b.w[i][n], xf[i], acc[n]);
      }
    const bool last = piece(q) == pieces - 1;
    const float sg = b.sg, su = b.su;
    load(b, item(q + 2), piece(q + 2));
    if (!last) return;
    // lane (token r, h) holds rows 4 h .. + 3: gate rows for h < 2, up rows above
    if (NB == 1) buf = 0;
#pragma unroll
    for (int n = 0; n < NI; n++) {
      *(f32x4*)&red[buf][grp][n][wave][r][4 * h] = acc[n];
      acc[n] = (f32x4){0.f, 0.f, 0.f, 0.f};
    }
    __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0); weight loads stay in flight
    ub_barrier();
    if (gt < CI * T && it < items) {
      const int u = it / nc, col = (it - u * nc) * CI + oc, j = slot[used[u]][ot];
      if (j >= 0) {
        float g = 0.f, up = 0.f;
#pragma unroll
        for (int w = 0; w < W1; w++) g += red[buf][grp][oc >> 3][w][ot][oc & 7], up += red[buf][grp][oc >> 3][w][ot][8 + (oc & 7)];
        if constexpr (Q8) g *= sg, up *= su;
        const float v = g / (1.f + expf(-g)) * up;
        const uint16_t hi = ub_f32_to_bf16(v);
        const float f = ub_bf16_to_f32(hi);
        uint16_t* at = (uint16_t*)a.act + (((size_t)ot * a.k + j) * I + (col & ~7)) * 2 + (col & 7);
        at[0] = hi;
        at[8] = ub_f32_to_bf16(__builtin_isinf(f) ? 0.f : v - f);
      }
    }
    if constexpr (NB == 1) {  // (two of them by turns need no second barrier)
      __builtin_amdgcn_s_waitcnt(0xC07F);
      ub_barrier();
    }
  };
  if (items == 0) return;
  Set b0, b1;
  load(b0, item(0), piece(0));
  load(b1, item(1), piece(1));
  int done = 0;  // items summed: their buffers alternate
  for (int q = 0; q < total; q += 2) {
    mul(b0, q, done & 1);
    if (piece(q) == pieces - 1) done++;
    if (q + 1 >= total) break;
    mul(b1, q + 1, done & 1);
    if (piece(q + 1) == pieces - 1) done++;
  }
}

// NC output columns a workgroup: 16 of one expert, or 8 of each of two (above).
constexpr int W2 = 8;  // wavefronts
template <int DT, bool Q8, int NC>
__global__ void __launch_bounds__(64 * W2) __attribute__((amdgpu_waves_per_eu(4, 4))) k_down(DecodeArgs a, int most) {
  constexpr int WB = Q8 ? 1 : 2, XN = Q8 ? 2 : 1, P = 4;  // P: steps of a unit
  constexpr int PER = NC / 2, SIDES = 16 / NC;            // tokens of an entry, entries of a unit
  __shared__ int expert[kEnt];
  __shared__ int16_t row[kEnt * PER];
  __shared__ int8_t tok[kEnt * PER];
  __shared__ float wts[kEnt * PER], sc[kEnt * NC];
  __shared__ float ys[W2][kTok][NC];  // a wavefront's sums
  const int tid = threadIdx.x, lane = tid & 63, r = lane & 15, h = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int T = a.T, H = a.H, I = a.I, n0 = blockIdx.x * NC;
  const int n = a.route->n;
  // units: P 64-byte steps of the rows of an entry, or a pair, dealt out in turn, so that
  // all workgroups walk through the experts together
  const int rowb = I * WB, per = ((rowb + 63) / 64 + P - 1) / P, units = (n + SIDES - 1) / SIDES * per;
  // the first half of a side's columns are the first parts of its tokens, the other half
  // the second, backwards (so that the two are mirror images in a row of lanes, or half one)
  const int side = r / NC, c = r % NC, rest = c / PER, ct = rest ? NC - 1 - c : c;
  struct Set {
    uint4 w[P], x[P][XN];
  };
  // Unit q's weights and activations.  FIRST: where they lie is read from scratch memory
  // itself, not from LDS, which is being filled meanwhile.
  auto load = [&](Set& b, int q, auto first) {
    constexpr bool FIRST = decltype(first)::value;
    const int p = q / per, u = SIDES * p + side, at0 = (q - p * per) * (64 * P) + 16 * h;
    const bool any = q < units && u < n;
    int ar = -1, e = 0;
    if (any) ar = FIRST ? a.route->row[u * PER + ct] : row[u * PER + ct], e = FIRST ? a.route->expert[u] : expert[u];
    const uint8_t* pw = (const uint8_t*)a.w2 + ((size_t)e * H + n0 + c) * rowb + at0;
    // (bytes: at most 256 rows of 2^20 values)
    const uint32_t px = (uint32_t)max(ar, 0) * I * 4 + at0 / WB * 4 + 16 * rest;
#pragma unroll
    for (int i = 0; i < P; i++) {
      b.w[i] = make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int v = 0; v < XN; v++) b.x[i][v] = make_uint4(0, 0, 0, 0);
      if (any && at0 + 64 * i < rowb) {
        b.w[i] = ld16(pw + 64 * i);
        if (ar >= 0) {
#pragma unroll
          for (int v = 0; v < XN; v++) b.x[i][v] = *(const uint4*)((const uint8_t*)a.act + px + (64 * i / WB + 8 * v) * 4);
        }
      }
    }
  };
  // Unit q's products, to the sums.  Lane (column r, h): rows 4 h .. + 3, of two entries
  // r's own if both are of the same half.  The two may share a token: one after the other.
  auto mul = [&](Set& b, int q) {
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < P; i++) acc = product_bf16<DT, Q8>(b.w[i], b.x[i], acc);
    load(b, q + 2 * W2, std::false_type{});
    const int u = SIDES * (q / per) + side, at = u * PER + ct, out = (4 * h) % NC;
    const bool mine = u < n && (SIDES == 1 || (h >> 1) == side) && !rest && row[at] >= 0;
#pragma unroll
    for (int i = 0; i < 4; i++) {  // the other part of the token's (row_mirror, row_half_mirror)
      const float v = acc[i];
      acc[i] = v + __uint_as_float(__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(v), NC == 16 ? 0x140 : 0x141, 0xf, 0xf, false));
    }
#pragma unroll
    for (int s = 0; s < SIDES; s++) {
      if (mine && side == s) {
        float* y = &ys[wave][tok[at]][out];
#pragma unroll
        for (int i = 0; i < 4; i++) y[i] += acc[i] * (Q8 ? wts[at] * sc[u * NC + out + i] : wts[at]);
      }
      __builtin_amdgcn_wave_barrier();
      asm volatile("" ::: "memory");
    }
  };
  Set b0, b1;
  // (entries past n, up to what there can be, are read with the others and not used)
  for (int i = tid; i < most * PER; i += 64 * W2) {
    row[i] = a.route->row[i];
    tok[i] = a.route->tok[i];
    wts[i] = a.route->w[i];
    if (i % PER == 0) expert[i / PER] = a.route->expert[i / PER];
  }
  load(b0, wave, std::true_type{});
  load(b1, wave + W2, std::true_type{});
  if constexpr (Q8)
    for (int i = tid; i < n * NC; i += 64 * W2)
      sc[i] = ub_load<DT>(a.s2, (size_t)a.route->expert[i / NC] * H + n0 + i % NC);
  for (int i = tid; i < W2 * kTok * NC; i += 64 * W2) (&ys[0][0][0])[i] = 0.f;
  __syncthreads();
  for (int q = wave; q < units; q += 2 * W2) {
    mul(b0, q);
    if (q + W2 < units) mul(b1, q + W2);
  }
  __syncthreads();
  if (tid < NC * T) {
    const int t = tid / NC, o = tid % NC;
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < W2; w++) v += ys[w][t][o];
    ub_store<DT>(a.y, (size_t)t * H + n0 + o, v);
  }
}

template <int DT, bool Q8, int NPL>
void up(const DecodeArgs& a, hipStream_t s) {
  const int steps = ub_cdiv(a.H * (Q8 ? 1 : 2), 64);
  const long items = (long)std::min(a.T * a.k, a.E) * (a.I / 8);
  auto go = [&](auto sp, auto multi, auto ng, auto ni) {
    constexpr int SP = decltype(sp)::value, NG = decltype(ng)::value, NI = decltype(ni)::value;
    const unsigned g = (unsigned)std::min<long>((items / NI + NG - 1) / NG, 256);  // a workgroup a CU
    k_up<DT, Q8, NPL, SP, decltype(multi)::value, NG, NI><<<g, 1024, 0, s>>>(a);
  };
  // As few steps a wavefront as hold the row, with two items to a workgroup up to 4 (more
  // bytes in flight; 8 of int8 are too many registers for 16 wavefronts).  Longer rows in
  // pieces: four items side by side, so that activations are loaded a quarter as often,
  // where there are enough items and those loads weigh something: int8, whose are twice the
  // weights' bytes, or half of the tokens at least.  us of the layer, E 64, k 8, one by one /
  // four, bf16 7168 x 512: T 4 137 / 140, 8 220 / 209, 16 318 / 277; int8: T 2 60 / 54, 16
  // 230 / 172.
  std::integral_constant<int, 1> one;
  std::integral_constant<int, 2> two;
  std::integral_constant<int, 4> four;
  std::integral_constant<int, 8> eight;
  std::false_type once;
  if (steps <= 8) return go(one, once, two, one);
  if (steps <= 16) return go(two, once, two, one);
  if (steps <= 32) return go(four, once, two, one);
  if constexpr (Q8) {
    if (steps <= 64) return go(four, once, one, one);
  } else {
    if (steps <= 64) return go(eight, once, two, one);
    if (steps <= 128) return go(eight, once, one, one);
  }
  std::true_type multi;
  if (items / 4 >= 256 && (Q8 || a.T >= 8)) return go(one, multi, one, four);
  go(four, multi, two, one);
}
template <int DT, bool Q8>
void decode(DecodeArgs a, hipStream_t s) {
  // 16 columns a workgroup, unless that gives some CU more than 8 would.  us of the layer, 8 /
  // 16 columns, E 64, k 8, I 512, one token bf16 (16 int8): 2048 16.8 / 18.8 (47 / 56), 2560 20.8 /
  // 20.8 (68 / 64), 4096 - (88 / 81), 5120 30.2 / 30.6, 6144 32.8 / 32.8 (146 / 148), 7168 37.7 /
  // 35.3 (173 / 161); 16 tokens, 2 of 8 experts, 4096 x 1024 bf16 47.9 / 41.4, 4096 x 4096 int8 111 /
  // 94.  8 wavefronts: 4 or 16 are up to 10% slower where workgroups and CUs are as many, 4
  // up to 6% faster for one token where workgroups are many.
  const int narrow = ub_cdiv(a.H / 8, 256), wides = 2 * ub_cdiv(a.H / 16, 256);
  const bool wide = wides <= narrow;
  a.per = wide ? 8 : 4;
  if (a.E <= 128) up<DT, Q8, 2>(a, s);
  else if (a.E <= 256) up<DT, Q8, 4>(a, s);
  else up<DT, Q8, kE / 64>(a, s);
  // entries, at most: one an expert in use, another for each `per` tokens past the first
  const int slots = a.T * a.k, used = std::min(slots, a.E), most = used + (slots - used) / a.per;
  if (wide) k_down<DT, Q8, 16><<<a.H / 16, 64 * W2, 0, s>>>(a, most);
  else k_down<DT, Q8, 8><<<a.H / 8, 64 * W2, 0, s>>>(a, most);
}

}  // namespace

UB_API int ubridge_moe_decode(const UbridgeMoeDecodeArgs* p, void* stream) {
  const char* nm = "ubridge_moe_decode";
  UB_REQUIRE(p, "%s: null argument block", nm);
  UB_REQUIRE(p->dtype == UB_F16 || p->dtype == UB_BF16, "%s: dtype %d", nm, p->dtype);
  UB_REQUIRE(p->logits_dtype >= UB_F32 && p->logits_dtype <= UB_BF16, "%s: logits of type %d", nm, p->logits_dtype);
  UB_REQUIRE(p->T >= 0 && p->T <= kTok, "%s: T=%d (at most %d tokens)", nm, p->T, kTok);
  UB_REQUIRE(p->E > 0 && p->E <= kE && p->k > 0 && p->k <= kK && p->k <= p->E, "%s: E=%d k=%d (E <= %d, 0 < k <= min(E, %d))", nm, p->E,
             p->k, kE, kK);
  UB_REQUIRE(p->H > 0 && p->H % 32 == 0 && p->I > 0 && p->I % 32 == 0 && p->H <= 1 << 20 && p->I <= 1 << 20,
             "%s: H=%d I=%d (multiples of 32)", nm, p->H, p->I);
  if (p->T == 0) return UB_OK;
  UB_REQUIRE(p->x && p->logits && p->w13 && p->w2 && p->y, "%s: null pointer", nm);
  UB_REQUIRE(!p->s13 == !p->s2, "%s: one of two scales", nm);
  UB_REQUIRE((((uintptr_t)p->x | (uintptr_t)p->w13 | (uintptr_t)p->w2) & 15) == 0, "%s: x or weights not 16-byte aligned", nm);
  hipStream_t s = ub_stream(stream);
  const size_t act = ((size_t)p->T * p->k * p->I * 4 + 255) / 256 * 256;
  UbScratch ws(s, act + sizeof(Route), true);
  UB_REQUIRE(ws.get(), "%s: no workspace", nm);
  const DecodeArgs a = {p->x, p->logits, p->w13, p->s13, p->w2, p->s2, p->y, ws.get(), (Route*)((char*)ws.get() + act),
                        p->T, p->E, p->k, p->H, p->I, p->logits_dtype, p->renormalize};
  if (p->s13) p->dtype == UB_F16 ? decode<UB_F16, true>(a, s) : decode<UB_BF16, true>(a, s);
  else p->dtype == UB_F16 ? decode<UB_F16, false>(a, s) : decode<UB_BF16, false>(a, s);
  return ub_check_launch(nm);
}
