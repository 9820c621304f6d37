// attn.hip -- attention of one new token per sequence over a paged cache.
//
//   x[t] = scale k_scale[h] (q . k[t]);  capped: x = c tanh(x / c)
//   x[t] += slope (t - (n - 1));  seen: n - 1 - window < t <= n - 1 (window 0: all)
//   o = v_scale[h] sum_t softmax(x)[t] v[t],  lse = log sum_t exp(x[t])
//
// for each query head, h its key / value head, n the tokens of its sequence.
// A sequence that sees nothing gives zeros and lse = -inf.
//
// The work is a stream of the cache (2 D values a token and kv head against 4 D
// G flops, G query heads to a kv head), so the kernel is shaped for bytes in
// flight and for an even share of them per CU:
//
//  * All query heads of a kv head are taken together, as the 16 columns of MFMA
//    tiles, so the cache is read once.  Keys and values go from memory
//    straight into the registers that the MFMAs read: no LDS, no barrier in
//    the loop, every wavefront walks its own tokens.
//  * A step is 32 tokens.  Scores are S^T = K Q^T in two 16 x 16 x 32 products
//    whose rows are dealt so that lane (c, g) ends with head c and the eight
//    tokens 8 g .. 8 g + 7 -- which is the layout of the second product's right
//    operand, O^T = V^T P^T over 32 tokens, so the weights never leave their
//    lane.  A lane reads its eight values rows of V 16 bytes each (8 dims) and
//    swaps tokens against dims with one byte permute a dword.
//  * The steps of all (sequence, kv head) rows, whose number only the device
//    knows, are laid end to end and cut into equal shares, one a wavefront (a
//    row counts two steps more than it has, for the latency of its first loads,
//    so that short rows are not heaped on one share).  A row inside one share
//    is finished there; a row that is cut leaves f32 partial sums, which k_join
//    adds in the order of the shares.  Where a workgroup a row is enough, there
//    are no shares and one launch (ROW).
//
// us of the kernels: 4 sequences of 100003 tokens, 8 kv heads of 128 in bf16 (1.64
// GB) 283 + 8 (5.8 TB/s); 64 sequences of up to 4096 (118 MB) 26 + 5.8, where a row's
// first loads wait for the last one's sums; 24 of up to 6000 under a window of 2048,
// 16 e4m3 heads of 80 (43 MB) 14 + 5.3, where half the time is latency and the
// softmax of one head in sixteen columns; one of 700 tokens 6.9 + 4.8, all latency:
// the search for the share, the page, the row, then the join's own reads.
//
// Numerics.  Scores, the running maximum and sum, and the output's sum are f32.
// The weights exp(x - m) enter the second product as the sum of two 16-bit
// numbers (off by at most 2^-16 of the weight for bf16, 2^-22 for f16; f16 weights
// are scaled by 2^14 so that those far below the maximum keep them): one number
// would cost as much as the output's own rounding, and the products are not what
// bounds the kernel.  The first is cut toward zero, and neither part of a weight
// above zero is zero: an infinite value then gives infinities of one sign, where
// parts of two signs, or a zero one, made it NaN (rounding the first to nearest
// would be worth one more bit).  e4m3 values are exact in both types.
#include "common.h"

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

constexpr float kInf = __builtin_inff();
constexpr float kLog2e = 1.4426950408889634f;
constexpr int W = 4;         // wavefronts of a workgroup
constexpr int kRowCost = 2;  // steps that the first loads of a row are worth
// Workgroups of k_join up to which the heads of a row are dealt out to several
// (its ROWS).  us of the whole call, one workgroup a row / dealt: 1 x 4096 tokens, 8 kv
// heads of 128 20.0 / 16.5, 1 x 131072 118 / 108, 32 x 4096 with 32 query heads on one
// kv head 56 / 43; up to 1024 workgroups 256 rows took 2 us longer, at 512 as long
constexpr int kJoins = 512;
constexpr int kShares = 2048;  // two wavefronts a SIMD (three: 64 ragged sequences 30 -> 47 us, by spills)

template <int DT>
__device__ __forceinline__ f32x4 mfma(uint4 a, uint4 b, f32x4 c) {
  if constexpr (DT == UB_BF16)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a),
                                                   __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a),
                                                  __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

template <int DT>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  const f32x2 v = {lo, hi};
  if constexpr (DT == UB_BF16) {
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, bf16x2));
  } else {
    typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, f16x2));
  }
}
// the same, toward zero
template <int DT>
__device__ __forceinline__ uint32_t cut2(float lo, float hi) {
  if constexpr (DT == UB_BF16) return __builtin_amdgcn_perm(__float_as_uint(hi), __float_as_uint(lo), 0x07060302u);
  else return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(lo, hi));
}
template <int DT>
__device__ __forceinline__ float half_of(uint32_t w, int hi) {
  if constexpr (DT == UB_BF16) return __uint_as_float(hi ? w & 0xffff0000u : w << 16);
  else return ub_f16_to_f32((uint16_t)(hi ? w >> 16 : w));
}

// two e4m3 bytes (the low or the high two of w) as two T
template <int DT, bool HI>
__device__ __forceinline__ uint32_t from_e4m3(uint32_t w) {
  if constexpr (DT == UB_BF16)
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)w, 1.0f, HI));
  else
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)w, 1.0f, HI));
}

// 8 stored values (element-aligned: gfx950 loads 16 bytes from there)
template <int CT> struct Raw { typedef uint4 T; static constexpr int B = 2; };
template <> struct Raw<UB_E4M3> { typedef uint2 T; static constexpr int B = 1; };
template <int CT>
__device__ __forceinline__ typename Raw<CT>::T ld8(const uint8_t* p) {
  typename Raw<CT>::T v;
  __builtin_memcpy(&v, p, sizeof(v));
  return v;
}
template <int DT, int CT>
__device__ __forceinline__ uint4 widen(const typename Raw<CT>::T& v) {
  if constexpr (CT == UB_E4M3)
    return make_uint4(from_e4m3<DT, false>(v.x), from_e4m3<DT, true>(v.x),
                      from_e4m3<DT, false>(v.y), from_e4m3<DT, true>(v.y));
  else
    return v;
}

struct Dev {
  UbridgePagedDecodeArgs a;
  int G, HG;       // query heads of a kv head; head groups of it (rows of one sequence: Hkv HG)
  int shares;      // wavefronts of k_decode
  uint64_t s_mul;  // t / S = t s_mul >> s_shift for 0 <= t < 2^31
  int s_shift;
  float* po;       // [2 shares][heads of a group][D] partial sums, relative to the maximum
  float* pml;      // [2 shares][heads of a group][2] maximum and sum
  int2* cut;       // [shares] the row that starts in a share and ends past it (-1: none), and its shares
  int* err;
};

// tokens [first, n) of sequence b, its steps; lengths past the table are cut
struct Span { int first, n, steps; };
__device__ __forceinline__ Span span(const Dev& d, int b) {
  const UbridgePagedDecodeArgs& a = d.a;
  Span s;
  s.n = max(a.lens[b], 0);
  const int top = a.P == 0 ? 0 : a.width * a.S;
  if (s.n > top) {
    *d.err = UB_ERR_INDEX;
    s.n = top;
  }
  s.first = a.window > 0 && s.n > a.window ? s.n - a.window : 0;
  s.steps = s.n > s.first ? (s.n + 31) / 32 - s.first / 32 : 0;
  return s;
}
// what a row costs, in steps: its own and the latency of its first loads
__device__ __forceinline__ int cost(const Span& s) { return s.steps ? s.steps + kRowCost : 0; }

// e^x 2^off: of differences to a maximum, which f32 holds exactly where they are
// small (scores kept in powers of two would carry the error of their own factor)
__device__ __forceinline__ float exp_of(float x, float off = 0.f) {
  return __builtin_amdgcn_exp2f(__builtin_fmaf(x, kLog2e, off));
}
// tanh z = (1 - t) / (1 + t), t = e^(-2 |z|); below a quarter, where 1 - t would
// keep t's rounding, the series, whose next term is below 1e-8 of it
__device__ __forceinline__ float tanh_of(float z) {
  const float t = exp_of(-2.f * fabsf(z)), u = z * z;
  const float far = copysignf((1.f - t) * __builtin_amdgcn_rcpf(1.f + t), z);
  const float near = z * (1.f + u * (-1.f / 3 + u * (2.f / 15 + u * (-17.f / 315 + u * (62.f / 2835)))));
  return fabsf(z) < 0.25f ? near : far;
}
// maximum and sum of a row -> log of the sum
template <int DT>
__device__ __forceinline__ float lse_of(float m, float l) {
  return m == -kInf ? m + l : m + logf(DT == UB_F16 ? l * 0x1p-14f : l);
}

// inclusive sum over the lanes, by DPP: no LDS round trip a step
__device__ __forceinline__ int lane_scan(int x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);  // row_shr 1, 2, 4, 8
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);  // lane 15 to rows 1 and 3
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);  // lane 31 to rows 2 and 3
  return x;
}

// DK: 32-dim pieces of a head; PG8: S is a multiple of 8, so eight tokens 8 i
// .. 8 i + 7 share a page; HT: tiles of 16 query heads.
// ROW: a workgroup per row, whose wavefronts take its steps in turn and meet in
// LDS; otherwise a share per wavefront.
template <int DK, int HT> constexpr int kRowWaves = DK * HT > 4 ? 4 : 8;  // (by their registers)
template <int DT, int CT, int DK, bool PG8, int HT, bool ROW>
__global__ void __launch_bounds__(64 * (ROW ? kRowWaves<DK, HT> : W)) __attribute__((amdgpu_waves_per_eu(DK * HT > 4 ? 1 : 2)))
k_decode(const Dev d) {
  constexpr int NW = ROW ? kRowWaves<DK, HT> : W, SS = ROW ? NW : 1;  // steps from one of a wavefront's to the next
  constexpr int NB = (DK + 3) / 4;      // 128-dim blocks of a head
  constexpr int NP = PG8 ? 1 : 2, NV = PG8 ? 1 : 8;  // pages a lane looks up for K and V
  constexpr int EB = Raw<CT>::B;
  constexpr int kLeastD = DK == 2 ? 8 : DK == 3 ? 72 : DK == 4 ? 104 : DK == 6 ? 136 : 200;  // that takes this DK
  constexpr float kOff = DT == UB_F16 ? 14.f : 0.f;
  constexpr float kLeast = DT == UB_F16 ? 0x1p-24f : 0x1p-126f;  // of a weight's parts
  typedef typename Raw<CT>::T R;
  const UbridgePagedDecodeArgs& a = d.a;
  const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int Hh = a.Hkv * d.HG;

  // ---- this wavefront's share [cur, end) of the costs of all rows: the sum
  // over the sequences (lane: four neighbours of every 256), then the place
  int cur = 0, end = 1, b = 0, hh = 0, at_row = 0, chunk = 1, share = 0;
  Span sp;
  int2 cut = make_int2(-1, 0);
  if constexpr (ROW) {
    b = (int)blockIdx.x / Hh, hh = (int)blockIdx.x - b * Hh;
    sp = span(d, b);
  } else {
    int four[4], tot = 0;
    auto costs = [&](int b0) {
      int s = 0;
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const int b = b0 + 4 * lane + i;
        four[i] = b < a.B ? cost(span(d, b)) : 0;
        s += four[i];
      }
      return s;
    };
    for (int b0 = (a.B - 1) & ~255; b0 >= 0; b0 -= 256) tot += costs(b0);
    int mine = four[0] + four[1] + four[2] + four[3], b0 = 0;  // (four holds the first 256)
    int x = lane_scan(mine);
    tot = (a.B <= 256 ? __builtin_amdgcn_readlane(x, 63) : __builtin_amdgcn_readlane(lane_scan(tot), 63)) * Hh;
    chunk = max(1, (int)(((unsigned)tot + d.shares - 1) / (unsigned)d.shares));
    share = blockIdx.x * W + wave;
    for (int i = share; i < a.B; i += d.shares)  // rows without tokens are nobody's share
      if (span(d, i).steps == 0) {
        const uint4 z = make_uint4(0, 0, 0, 0);
        uint16_t* p = (uint16_t*)a.out + (size_t)i * a.Hq * a.D;
        for (int e = 8 * lane; e < a.Hq * a.D; e += 512) __builtin_memcpy(p + e, &z, 16);
        if (a.lse)
          for (int e = lane; e < a.Hq; e += 64) a.lse[(size_t)i * a.Hq + e] = -kInf;
      }
    if ((int64_t)share * chunk >= tot) {
      if (lane == 0) d.cut[share] = cut;
      return;
    }
    cur = share * chunk;
    end = (int)min((int64_t)tot, (int64_t)cur + chunk);
    mine *= Hh, x *= Hh;
    for (int before; cur >= (before = __builtin_amdgcn_readlane(x, 63));) {
      b0 += 256;
      mine = costs(b0) * Hh;
      x = before + lane_scan(mine);
    }
    const int owner = __builtin_ctzll(__ballot(cur < x));  // the lane whose sequences hold cur
    at_row = cur - __builtin_amdgcn_readlane(x - mine, owner);
    b = b0 + 4 * owner;
#pragma unroll
    for (int i = 0; i < 3; i++) {
      const int s = __builtin_amdgcn_readlane(four[i], owner) * Hh;
      if (b == b0 + 4 * owner + i && at_row >= s) {
        at_row -= s;
        b++;
      }
    }
    sp = span(d, b);
    hh = (int)((unsigned)at_row / (unsigned)cost(sp));
    at_row -= hh * cost(sp);  // the share starts this far into the row
  }

  const float cap = a.softcap;
  const uint8_t* const kbase = (const uint8_t*)a.k_pages;
  const uint8_t* const vbase = (const uint8_t*)a.v_pages;
  // dims of this lane's pieces; a piece past D reads the head's first dims
  // instead (in bounds) and counts for nothing
  bool kin[DK];
#pragma unroll
  for (int j = 0; j < DK; j++) kin[j] = 32 * j + 8 * g < a.D;
  int vdim[NB];
#pragma unroll
  for (int nb = 0; nb < NB; nb++) vdim[nb] = 128 * nb + 8 * c < a.D ? 128 * nb + 8 * c : 0;

  while (cur < end) {
    // ---- one row, or the part of it that lies in the share
    const int len = ROW ? 1 : min(end - cur, cost(sp) - at_row);
    const int st = ROW ? wave : max(at_row - kRowCost, 0), s1 = ROW ? sp.steps : at_row + len - kRowCost;
    cur += len;
    const int h = hh / d.HG, hg = hh - h * d.HG;
    const int row_of_b = hh, bb = b;
    const Span sq = sp;
    at_row = 0;
    if (cur < end && ++hh == Hh) {
      hh = 0;
      do sp = span(d, ++b);
      while (sp.steps == 0);
    }
    if (!ROW && s1 <= st) continue;  // (only the row's head)
    const int q0 = hg * 16 * HT, nq = min(d.G - q0, 16 * HT);  // its query heads
    const size_t row0 = (size_t)bb * a.Hq + h * d.G + q0;
    if (ROW && sq.steps == 0) {
      for (int e = (int)threadIdx.x; e < nq * a.D; e += 64 * NW) ((uint16_t*)a.out)[row0 * a.D + e] = 0;
      if (a.lse && (int)threadIdx.x < nq) a.lse[row0 + threadIdx.x] = -kInf;
      return;
    }
    const int base = sq.first / 32;
    const int* tb = a.tables + bb * a.table_stride;

    uint4 qf[HT][DK];
    float slope[HT];
#pragma unroll
    for (int t = 0; t < HT; t++) {
      const bool live = 16 * t + c < nq;
      const int hq = h * d.G + q0 + 16 * t + c;
      const uint16_t* p = (const uint16_t*)a.q + bb * a.q_sb + (live ? hq : 0) * a.q_sh;
#pragma unroll
      for (int j = 0; j < DK; j++) {
        qf[t][j] = make_uint4(0, 0, 0, 0);
        if (live && kin[j]) __builtin_memcpy(&qf[t][j], p + 32 * j + 8 * g, 16);
      }
      slope[t] = live && a.slopes ? a.slopes[hq] : 0.f;
    }
    const float ks = a.scale * (a.k_scale ? a.k_scale[h] : 1.f);
    const float kx = cap > 0.f ? ks / cap : ks;  // on q . k

    f32x4 o[HT][NB][8];
    float m[HT], l[HT];
#pragma unroll
    for (int t = 0; t < HT; t++) {
      m[t] = -kInf;
      l[t] = 0.f;
#pragma unroll
      for (int nb = 0; nb < NB; nb++)
#pragma unroll
        for (int j = 0; j < 8; j++) o[t][nb][j] = (f32x4){0.f, 0.f, 0.f, 0.f};
    }

    R kf[2][DK], vf[NB][8];
    int pk[NP], pv[NV];
    // tokens that a lane reads keys of (tau = 0, 1) and values of (e = 0..7),
    // kept inside [first, n); with PG8 the page of a group of eight, whose
    // unseen tokens lie in the page too
    auto tok = [&](int s, int i) {
      const int t = 32 * (base + s) + i;
      return PG8 ? min(max(t, sq.first & ~7), (sq.n - 1) & ~7) : min(max(t, sq.first), sq.n - 1);
    };
    auto quo = [&](int t) { return (int)((uint64_t)t * d.s_mul >> d.s_shift); };  // t / S
    auto lookup = [&](int s) {
      if constexpr (PG8) {
        pk[0] = tb[quo(tok(s, 8 * (c >> 2)))];
        pv[0] = tb[quo(tok(s, 8 * g))];
      } else {
#pragma unroll
        for (int i = 0; i < 2; i++) pk[i] = tb[quo(tok(s, 8 * (c >> 2) + 4 * i + (c & 3)))];
#pragma unroll
        for (int e = 0; e < 8; e++) pv[e] = tb[quo(tok(s, 8 * g + e))];
      }
    };
    auto page = [&](int p) { return (unsigned)p < (unsigned)a.P ? p : 0; };
    auto load_k = [&](int s) {
#pragma unroll
      for (int i = 0; i < 2; i++) {
        const int t = tok(s, 8 * (c >> 2) + (PG8 ? 0 : 4 * i + (c & 3)));
        const int at = t - quo(t) * a.S + (PG8 ? 4 * i + (c & 3) : 0);
        const uint8_t* p = kbase + EB * (page(pk[PG8 ? 0 : i]) * a.k_sp + h * a.k_sh + at * a.k_ss);
#pragma unroll
        for (int j = 0; j < DK; j++) kf[i][j] = ld8<CT>(p + EB * (kin[j] ? 32 * j + 8 * g : 0));
      }
    };
    unsigned bad = 0;  // of the values being multiplied: tokens whose page is not there
    unsigned bad_next = 0;
    auto load_v = [&](int s) {
      bad_next = 0;
#pragma unroll
      for (int e = 0; e < 8; e++) {
        const int t = tok(s, 8 * g + (PG8 ? 0 : e));
        const int at = t - quo(t) * a.S + (PG8 ? e : 0);
        const int pg = pv[PG8 ? 0 : e];
        if ((unsigned)pg >= (unsigned)a.P) bad_next |= 1u << e;
        const uint8_t* p = vbase + EB * (page(pg) * a.v_sp + h * a.v_sh + at * a.v_ss);
#pragma unroll
        for (int nb = 0; nb < NB; nb++) vf[nb][e] = ld8<CT>(p + EB * vdim[nb]);
      }
    };

    int s = st;
    if (s < s1) {
      lookup(s);
      load_k(s);
      load_v(s);
      bad = bad_next;
      if (s + SS < s1) lookup(s + SS);
    }
    for (; s < s1; s += SS) {
      const int t0 = 32 * (base + s) + 8 * g;  // this lane's first token
      const bool edge = 32 * (base + s) < sq.first || 32 * (base + s) + 32 > sq.n;
      // scores: x[t][tau * 4 + i] of head c, token t0 + 4 tau + i
      f32x4 acc[HT][2];
#pragma unroll
      for (int i = 0; i < 2; i++) {
#pragma unroll
        for (int t = 0; t < HT; t++) acc[t][i] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < DK; j++) {
          uint4 k = widen<DT, CT>(kf[i][j]);
          if (32 * (j + 1) > kLeastD && !kin[j]) k = make_uint4(0, 0, 0, 0);
#pragma unroll
          for (int t = 0; t < HT; t++) acc[t][i] = mfma<DT>(k, qf[t][j], acc[t][i]);
        }
      }
      const int sn = s + SS;
      if (sn < s1) {
        load_k(sn);
      }
      if (bad) *d.err = UB_ERR_INDEX;
      uint4 ph[HT], pl[HT];
#pragma unroll
      for (int t = 0; t < HT; t++) {
        float x[8], mx = -kInf;
#pragma unroll
        for (int e = 0; e < 8; e++) {
          float v = acc[t][e >> 2][e & 3] * kx;
          if (cap > 0.f) v = cap * tanh_of(v);
          v += slope[t] * (float)(t0 + e - (sq.n - 1));
          if (bad >> e & 1) v = __builtin_nanf("");
          if (edge && (t0 + e < sq.first || t0 + e >= sq.n)) v = -kInf;
          x[e] = v;
          mx = fmaxf(mx, v);
        }
        mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
        mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
        const float mn = fmaxf(m[t], mx), ms = mn == -kInf ? 0.f : mn;  // (a NaN score: its weight is NaN)
        const float al = exp_of(m[t] - ms);
        m[t] = mn;
        float p[8], sum = 0.f;
#pragma unroll
        for (int e = 0; e < 8; e++) {
          p[e] = exp_of(x[e] - ms, kOff);
          sum += p[e];
          p[e] = p[e] > 0.f ? fmaxf(p[e], kLeast) : 0.f;  // (a NaN is in the sum)
        }
        l[t] = l[t] * al + sum;
        uint32_t* hi = (uint32_t*)&ph[t];
        uint32_t* lo = (uint32_t*)&pl[t];
#pragma unroll
        for (int q = 0; q < 4; q++) {
          const float a = p[2 * q], b = p[2 * q + 1];
          hi[q] = cut2<DT>(a, b);
          lo[q] = pack2<DT>(fmaxf(a - half_of<DT>(hi[q], 0), fminf(a, kLeast)),
                            fmaxf(b - half_of<DT>(hi[q], 1), fminf(b, kLeast)));
        }
        if (__any(al != 1.f)) {
#pragma unroll
          for (int nb = 0; nb < NB; nb++)
#pragma unroll
            for (int j = 0; j < 8; j++) o[t][nb][j] *= al;
        }
      }
      if (edge) {  // what lies behind a masked place may be anything
#pragma unroll
        for (int e = 0; e < 8; e++)
          if (t0 + e < sq.first || t0 + e >= sq.n)
#pragma unroll
            for (int nb = 0; nb < NB; nb++) vf[nb][e] = R{};
      }
#pragma unroll
      for (int nb = 0; nb < NB; nb++)
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
          uint32_t v0[4], v1[4];  // dims j and j + 1, two tokens a dword
#pragma unroll
          for (int q = 0; q < 4; q++) {
            if constexpr (CT == UB_E4M3) {
              const uint32_t x0 = j < 4 ? vf[nb][2 * q].x : vf[nb][2 * q].y;
              const uint32_t x1 = j < 4 ? vf[nb][2 * q + 1].x : vf[nb][2 * q + 1].y;
              const uint32_t w = __builtin_amdgcn_perm(x1, x0, j & 2 ? 0x07030602u : 0x05010400u);
              v0[q] = from_e4m3<DT, false>(w);
              v1[q] = from_e4m3<DT, true>(w);
            } else {
              const uint32_t x0 = ((const uint32_t*)&vf[nb][2 * q])[j / 2];
              const uint32_t x1 = ((const uint32_t*)&vf[nb][2 * q + 1])[j / 2];
              v0[q] = __builtin_amdgcn_perm(x1, x0, 0x05040100u);
              v1[q] = __builtin_amdgcn_perm(x1, x0, 0x07060302u);
            }
          }
          const uint4 w0 = make_uint4(v0[0], v0[1], v0[2], v0[3]), w1 = make_uint4(v1[0], v1[1], v1[2], v1[3]);
#pragma unroll
          for (int t = 0; t < HT; t++) {
            o[t][nb][j] = mfma<DT>(w0, ph[t], o[t][nb][j]);
            o[t][nb][j + 1] = mfma<DT>(w1, ph[t], o[t][nb][j + 1]);
            o[t][nb][j] = mfma<DT>(w0, pl[t], o[t][nb][j]);
            o[t][nb][j + 1] = mfma<DT>(w1, pl[t], o[t][nb][j + 1]);
          }
        }
      if (sn < s1) {
        load_v(sn);
        bad = bad_next;
        if (sn + SS < s1) lookup(sn + SS);
      }
    }

    if constexpr (ROW) {
      // ---- the wavefronts' sums meet in LDS, in their order
      extern __shared__ __attribute__((aligned(16))) float so[];  // [NW][nq][D + 4]
      __shared__ float2 sml[NW][16 * HT];
      const int pitch = a.D + 4;
#pragma unroll
      for (int t = 0; t < HT; t++) {
        l[t] += __shfl_xor(l[t], 16, 64);
        l[t] += __shfl_xor(l[t], 32, 64);
        const int q = 16 * t + c;
        if (q >= nq) continue;
        if (g == 0) sml[wave][q] = make_float2(m[t], l[t]);
        float* p = so + (wave * nq + q) * pitch;
#pragma unroll
        for (int nb = 0; nb < NB; nb++)
#pragma unroll
          for (int i = 0; i < 4; i++) {
            const int dim = 128 * nb + 32 * g + 8 * i;
            if (dim >= a.D) continue;
#pragma unroll
            for (int j = 0; j < 8; j += 4)
              *(float4*)(p + dim + j) = make_float4(o[t][nb][j][i], o[t][nb][j + 1][i], o[t][nb][j + 2][i], o[t][nb][j + 3][i]);
          }
      }
      __syncthreads();
      const int V = a.D / 4;
      for (int e = (int)threadIdx.x; e < nq * V; e += 64 * NW) {
        const int q = e / V, v = e - q * V;
        float M = -kInf, L = 0.f;
#pragma unroll
        for (int w = 0; w < NW; w++) M = fmaxf(M, sml[w][q].x);
        const float Ms = M == -kInf ? 0.f : M;
        float4 O = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < NW; w++) {
          const float2 ml = sml[w][q];
          const float4 x = *(const float4*)(so + (w * nq + q) * pitch + 4 * v);
          const float f = exp_of(ml.x - Ms);
          O.x += f * x.x, O.y += f * x.y, O.z += f * x.z, O.w += f * x.w;
          L += f * ml.y;
        }
        const float f = L == 0.f ? 0.f : (a.v_scale ? a.v_scale[h] : 1.f) / L;
        const uint32_t w[2] = {pack2<DT>(O.x * f, O.y * f), pack2<DT>(O.z * f, O.w * f)};
        __builtin_memcpy((uint16_t*)a.out + (row0 + q) * a.D + 4 * v, w, 8);
        if (v == 0 && a.lse) a.lse[row0 + q] = lse_of<DT>(M, L);
      }
      return;
    }
    // ---- a whole row is finished here; a part leaves its sums
    const bool whole = st == 0 && s1 == sq.steps;
    const int slot = 2 * share + (st == 0);
    const float vs = a.v_scale ? a.v_scale[h] : 1.f;
#pragma unroll
    for (int t = 0; t < HT; t++) {
      l[t] += __shfl_xor(l[t], 16, 64);
      l[t] += __shfl_xor(l[t], 32, 64);
      const int q = 16 * t + c;
      if (q >= nq) continue;
      if (whole) {
        const float f = l[t] == 0.f ? 0.f : vs / l[t];
#pragma unroll
        for (int nb = 0; nb < NB; nb++)
#pragma unroll
          for (int i = 0; i < 4; i++) {
            const int dim = 128 * nb + 32 * g + 8 * i;
            if (dim >= a.D) continue;
            uint32_t w[4];
#pragma unroll
            for (int j = 0; j < 4; j++) w[j] = pack2<DT>(o[t][nb][2 * j][i] * f, o[t][nb][2 * j + 1][i] * f);
            __builtin_memcpy((uint16_t*)a.out + (row0 + q) * a.D + dim, w, 16);
          }
        if (g == 0 && a.lse) a.lse[row0 + q] = lse_of<DT>(m[t], l[t]);
      } else {
        float* po = d.po + ((size_t)slot * 16 * HT + q) * a.D;
#pragma unroll
        for (int nb = 0; nb < NB; nb++)
#pragma unroll
          for (int i = 0; i < 4; i++) {
            const int dim = 128 * nb + 32 * g + 8 * i;
            if (dim >= a.D) continue;
#pragma unroll
            for (int j = 0; j < 8; j += 4)
              *(float4*)(po + dim + j) = make_float4(o[t][nb][j][i], o[t][nb][j + 1][i], o[t][nb][j + 2][i], o[t][nb][j + 3][i]);
          }
        if (g == 0) *(float2*)(d.pml + ((size_t)slot * 16 * HT + q) * 2) = make_float2(m[t], l[t]);
      }
    }
    if (st == 0 && !whole)
      cut = make_int2(bb * Hh + row_of_b, 1 + (int)(((unsigned)(sq.steps - s1) + chunk - 1) / (unsigned)chunk));
  }
  if (lane == 0) d.cut[share] = cut;
}

// Workgroup (i, j): `part` heads of row i (ROWS, at most 512: where it lies follows
// from the costs), else of the row that starts in share i; nothing if that row
// is not cut.  Thread (u, column) adds four dims of one head over every U-th of the row's
// shares, four of them in flight, under a running maximum; the U sums meet in
// LDS, in order.
template <int DT, bool ROWS>
__global__ void __launch_bounds__(512) k_join(const Dev d, int heads, int part) {
  __shared__ float4 so[512];
  __shared__ float2 sml[512];
  const UbridgePagedDecodeArgs& a = d.a;
  const int Hh = a.Hkv * d.HG;
  int row, first, parts;  // its first share and their number
  if constexpr (ROWS) {
    __shared__ int2 sums[8];  // of a wavefront's costs: all, those of sequences ahead of the row's
    row = blockIdx.x;
    const int b = row / Hh, own = cost(span(d, b)), i = threadIdx.x;
    const int c = i < a.B ? cost(span(d, i)) : 0;
    const int x = lane_scan(c), y = lane_scan(i < b ? c : 0);
    if ((i & 63) == 63) sums[i >> 6] = make_int2(x, y);
    __syncthreads();
    int tot = 0, at = 0;
#pragma unroll
    for (int w = 0; w < 8; w++) tot += sums[w].x, at += sums[w].y;
    const int chunk = max(1, (int)(((unsigned)(tot * Hh) + d.shares - 1) / (unsigned)d.shares));
    at = at * Hh + (row - b * Hh) * own;
    first = (unsigned)(at + kRowCost) / (unsigned)chunk;  // of its first step
    parts = own ? (int)((unsigned)(at + own - 1) / (unsigned)chunk) - first + 1 : 0;
    if (parts <= 1) return;
  } else {
    const int2 cut = d.cut[blockIdx.x];
    if (cut.x < 0) return;
    row = cut.x, first = blockIdx.x, parts = cut.y;
  }
  const int b = row / Hh, hh = row - b * Hh;
  const int h = hh / d.HG, q0 = (hh - h * d.HG) * heads;
  const int qa = (int)blockIdx.y * part, V = a.D / 4, cols = min(min(d.G - q0, heads) - qa, part) * V;
  if (cols <= 0) return;
  const int U = cols < 512 ? 512 / cols : 1;
  const float vs = a.v_scale ? a.v_scale[h] : 1.f;
  for (int c0 = 0; c0 < cols; c0 += 512) {
    const int u = (int)threadIdx.x / cols, col = c0 + (int)threadIdx.x - u * cols;
    const int q = qa + col / V, v = col % V;
    const bool live = u < U && col < cols;
    float4 O = make_float4(0.f, 0.f, 0.f, 0.f);
    float M = -kInf, L = 0.f;
    if (live)
      for (int p0 = u; p0 < parts; p0 += 4 * U) {
        float2 ml[4];
        float4 x[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const int p = min(p0 + i * U, parts - 1);
          const size_t slot = (size_t)(2 * (first + p) + (p == 0)) * heads + q;
          ml[i] = *(const float2*)(d.pml + 2 * slot);
          x[i] = *(const float4*)(d.po + slot * a.D + 4 * v);
        }
        float mn = M;
#pragma unroll
        for (int i = 0; i < 4; i++) mn = fmaxf(mn, ml[i].x);
        const float ms = mn == -kInf ? 0.f : mn, al = exp_of(M - ms);
        M = mn;
        O.x *= al, O.y *= al, O.z *= al, O.w *= al, L *= al;
#pragma unroll
        for (int i = 0; i < 4; i++) {
          if (p0 + i * U >= parts) continue;
          const float w = exp_of(ml[i].x - ms);
          O.x += w * x[i].x, O.y += w * x[i].y, O.z += w * x[i].z, O.w += w * x[i].w;
          L += w * ml[i].y;
        }
      }
    if (U > 1) {
      so[threadIdx.x] = O;
      sml[threadIdx.x] = make_float2(M, L);
      __syncthreads();
      if (u == 0) {
        float mn = M;
        for (int i = 1; i < U; i++) mn = fmaxf(mn, sml[threadIdx.x + i * cols].x);
        const float ms = mn == -kInf ? 0.f : mn, al = exp_of(M - ms);
        M = mn;
        O.x *= al, O.y *= al, O.z *= al, O.w *= al, L *= al;
        for (int i = 1; i < U; i++) {
          const float2 ml = sml[threadIdx.x + i * cols];
          const float4 x = so[threadIdx.x + i * cols];
          const float w = exp_of(ml.x - ms);
          O.x += w * x.x, O.y += w * x.y, O.z += w * x.z, O.w += w * x.w;
          L += w * ml.y;
        }
      }
    }
    if (live && u == 0) {
      const size_t to = (size_t)b * a.Hq + h * d.G + q0 + q;
      const float f = L == 0.f ? 0.f : vs / L;
      const uint32_t w[2] = {pack2<DT>(O.x * f, O.y * f), pack2<DT>(O.z * f, O.w * f)};
      __builtin_memcpy((uint16_t*)a.out + to * a.D + 4 * v, w, 8);
      if (v == 0 && a.lse) a.lse[to] = lse_of<DT>(M, L);
    }
  }
}

template <int DT, int CT, int DK, bool PG8, int HT>
void decode(const Dev& d, hipStream_t s) {
  if (d.shares) {
    k_decode<DT, CT, DK, PG8, HT, false><<<d.shares / W, 64 * W, 0, s>>>(d);
    return;
  }
  constexpr int NW = kRowWaves<DK, HT>;
  static UbLdsLimit limit;
  limit.raise((const void*)k_decode<DT, CT, DK, PG8, HT, true>, NW * 16 * HT * (32 * DK + 4) * (int)sizeof(float));
  const size_t lds = sizeof(float) * NW * (d.G < 16 * HT ? d.G : 16 * HT) * (d.a.D + 4);
  k_decode<DT, CT, DK, PG8, HT, true><<<d.a.B * d.a.Hkv * d.HG, 64 * NW, lds, s>>>(d);
}
template <int DT, int CT, int DK, bool PG8>
void decode(const Dev& d, int HT, hipStream_t s) {
  if (HT == 1) decode<DT, CT, DK, PG8, 1>(d, s);
  else decode<DT, CT, DK, PG8, 2>(d, s);
}
template <int DT, int CT, int DK>
void decode(const Dev& d, int HT, hipStream_t s) {
  if (d.a.S % 8 == 0) decode<DT, CT, DK, true>(d, HT, s);
  else decode<DT, CT, DK, false>(d, HT, s);
}
template <int DT, int CT>
void decode(const Dev& d, int HT, hipStream_t s) {
  if (d.a.D <= 64) decode<DT, CT, 2>(d, HT, s);
  else if (d.a.D <= 96) decode<DT, CT, 3>(d, HT, s);
  else if (d.a.D <= 128) decode<DT, CT, 4>(d, HT, s);
  else if (d.a.D <= 192) decode<DT, CT, 6>(d, HT, s);
  else decode<DT, CT, 8>(d, HT, s);
  if (!d.shares) return;
  const int rows = d.a.B * d.a.Hkv * d.HG, heads = d.G < 16 * HT ? d.G : 16 * HT;
  if (rows > kJoins) {
    k_join<DT, false><<<d.shares, 512, 0, s>>>(d, 16 * HT, heads);
    return;
  }
  int part = 1;
  while (rows * ub_cdiv(heads, part) > kJoins && part < heads) part *= 2;
  k_join<DT, true><<<dim3(rows, ub_cdiv(heads, part)), 512, 0, s>>>(d, 16 * HT, part);
}

void go(const Dev& d, int HT, hipStream_t s) {
  const int dt = d.a.dtype, ct = d.a.cache_dtype;
  if (dt == UB_BF16 && ct == UB_BF16) decode<UB_BF16, UB_BF16>(d, HT, s);
  else if (dt == UB_BF16) decode<UB_BF16, UB_E4M3>(d, HT, s);
  else if (ct == UB_F16) decode<UB_F16, UB_F16>(d, HT, s);
  else decode<UB_F16, UB_E4M3>(d, HT, s);
}

}  // namespace

UB_API int ubridge_paged_decode(const UbridgePagedDecodeArgs* p, void* stream) {
  const char* nm = "ubridge_paged_decode";
  UB_REQUIRE(p, "%s: null argument block", nm);
  const UbridgePagedDecodeArgs& a = *p;
  UB_REQUIRE(a.dtype == UB_F16 || a.dtype == UB_BF16, "%s: dtype %d", nm, a.dtype);
  UB_REQUIRE(a.cache_dtype == a.dtype || a.cache_dtype == UB_E4M3, "%s: cache type %d for queries of type %d",
             nm, a.cache_dtype, a.dtype);
  UB_REQUIRE(a.B >= 0 && a.Hq >= 0 && a.Hkv > 0 && a.Hq % a.Hkv == 0,
             "%s: B=%d Hq=%d (a multiple of Hkv=%d)", nm, a.B, a.Hq, a.Hkv);
  UB_REQUIRE(a.D > 0 && a.D % 8 == 0 && a.D <= 256, "%s: D=%d (a multiple of 8, at most 256)", nm, a.D);
  UB_REQUIRE(a.S > 0 && a.P >= 0 && a.width >= 0 && (int64_t)a.width * a.S <= 0x7fffffc0,
             "%s: S=%d P=%d width=%d", nm, a.S, a.P, a.width);
  UB_REQUIRE(a.window >= 0 && (a.softcap == 0.f || (a.softcap >= 0x1p-126f && a.softcap < kInf)),
             "%s: window=%d softcap=%g (0, or normal and finite)", nm, a.window, a.softcap);
  if (a.B == 0 || a.Hq == 0) return UB_OK;
  UB_REQUIRE(a.q && a.out && a.lens && (a.tables || a.width == 0), "%s: null pointer", nm);
  UB_REQUIRE(a.P == 0 || (a.k_pages && a.v_pages), "%s: null pages", nm);
  UB_REQUIRE((int64_t)a.B * a.Hq < 1 << 23, "%s: B=%d Hq=%d", nm, a.B, a.Hq);
  Dev d;
  d.a = a;
  d.G = a.Hq / a.Hkv;
  d.err = ub_error_flag();
  UB_REQUIRE(d.err, "%s: no device flag", nm);
  const int HT = d.G > 16 ? 2 : 1, heads = 16 * HT;
  d.HG = ub_cdiv(d.G, heads);
  const int64_t rows = (int64_t)a.B * a.Hkv * d.HG;
  int64_t steps = (int64_t)a.width * a.S / 32 + 1;  // of a row, at most
  if (a.window > 0 && steps > a.window / 32 + 2) steps = a.window / 32 + 2;
  const int64_t most = rows * (steps + kRowCost);  // the costs of all rows
  UB_REQUIRE(most < 0x7fffffff, "%s: %ld rows of %ld tokens", nm, (long)rows, (long)a.width * a.S);
  d.s_shift = 31;
  while ((1ll << (d.s_shift - 31)) < a.S) d.s_shift++;
  d.s_mul = (1ull << d.s_shift) / a.S + 1;
  hipStream_t s = ub_stream(stream);
  // A workgroup a row where the CUs have one each at most and a wavefront two
  // steps: one launch.  us of the kernels, shares + join / rows: 8 rows of 64 tokens
  // 6.4 + 3.5 / 5.4, of 500 6.9 + 4.5 / 7.0, of 700 (three steps) 6.9 + 4.5 / 12.0;
  // 256 rows of 64 tokens 9.6 + 3.7 / 5.6
  const int nw = ub_cdiv(a.D, 32) * HT > 4 ? 4 : 8;
  if (rows <= 256 && steps <= 2 * nw) {
    d.shares = 0;
    d.po = d.pml = nullptr;
    d.cut = nullptr;
    go(d, HT, s);
    return ub_check_launch(nm);
  }
  // one wavefront a SIMD where the registers allow no more: half the partial sums.  us
  // with 2048 / 1024 shares: 32 x 4096 tokens, 32 query heads on one kv head of 128
  // 43 / 30, 8 x 4 heads of 256 201 / 196, in e4m3 120 / 110
  const int shares = nw == 4 ? kShares / 2 : kShares;
  d.shares = most >= shares ? shares : ub_cdiv(most, W) * W;
  const size_t nml = sizeof(float) * 4 * heads * d.shares, no = nml / 2 * a.D;
  UbScratch ws(s, no + nml + sizeof(int2) * d.shares);
  if (!ws.get()) return ub_set_error(UB_ERR_LAUNCH, "%s: no workspace", nm);
  d.po = (float*)ws.get();
  d.pml = d.po + no / sizeof(float);
  d.cut = (int2*)((char*)ws.get() + no + nml);
  go(d, HT, s);
  return ub_check_launch(nm);
}
