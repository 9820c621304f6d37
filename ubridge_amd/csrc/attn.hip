// attn.hip -- attention of one new token per sequence over a paged cache.
//
//   x[t] = scale k_scale[h] (q . k[t]);  capped: x = c tanh(x / c)
//   x[t] += slope (t - (n - 1));  seen: n - 1 - window < t <= n - 1 (window 0: all)
//   o = v_scale[h] sum_t softmax(x)[t] v[t],  lse = log sum_t exp(x[t])
//
// for each query head, h its key / value head, n the tokens of its sequence.
// A sequence that sees nothing gives zeros and lse = -inf.  Scores, the
// running maximum and sum, and the output's sum are f32.
#include "common.h"

namespace {

template <int CT>
__device__ __forceinline__ float ldc(const void* p, long i) {
  if constexpr (CT == UB_E4M3) return __builtin_amdgcn_cvt_f32_fp8(((const uint8_t*)p)[i], 0);
  else return ub_load<CT>(p, i);
}

// One workgroup per (sequence, query head): four wavefronts, each a quarter of
// the tokens, a lane the dims lane, lane + 64, ...
template <int DT, int CT>
__global__ void __launch_bounds__(256) k_decode(const UbridgePagedDecodeArgs a, int* err) {
  __shared__ float sm[4], sl[4], so[4][256];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int b = blockIdx.x / a.Hq, hq = blockIdx.x - b * a.Hq, h = hq / (a.Hq / a.Hkv);
  int n = a.lens[b];
  if (n > (long)a.width * a.S || (n > 0 && a.P == 0)) {
    if (tid == 0) *err = UB_ERR_INDEX;
    n = a.P == 0 ? 0 : a.width * a.S;
  }
  const int first = a.window > 0 && n > a.window ? n - a.window : 0;
  const float slope = a.slopes ? a.slopes[hq] : 0.f;
  const float ks = a.scale * (a.k_scale ? a.k_scale[h] : 1.f);
  float q[4], o[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int j = 0; j < 4; j++)
    q[j] = lane + 64 * j < a.D ? ub_load<DT>(a.q, b * a.q_sb + hq * a.q_sh + lane + 64 * j) : 0.f;
  float m = -__builtin_inff(), l = 0.f;
  for (int t = first + wave; t < n; t += 4) {
    int page = a.tables[b * a.table_stride + t / a.S];
    const bool bad = page < 0 || page >= a.P;
    if (bad) {
      page = 0;
      *err = UB_ERR_INDEX;
    }
    const long ko = page * a.k_sp + h * a.k_sh + (t % a.S) * a.k_ss;
    const long vo = page * a.v_sp + h * a.v_sh + (t % a.S) * a.v_ss;
    float x = 0.f;
#pragma unroll
    for (int j = 0; j < 4; j++)
      if (lane + 64 * j < a.D) x += q[j] * ldc<CT>(a.k_pages, ko + lane + 64 * j);
    x = ub_wave_sum(x) * ks;
    if (a.softcap > 0.f) x = a.softcap * tanhf(x / a.softcap);
    x += slope * (float)(t - (n - 1));
    if (bad) x = __builtin_nanf("");
    const float mn = fmaxf(m, x), ms = mn == -__builtin_inff() ? 0.f : mn;  // (a NaN score: p is NaN)
    const float al = expf(m - ms), p = expf(x - ms);
    l = l * al + p;
    m = mn;
#pragma unroll
    for (int j = 0; j < 4; j++)
      if (lane + 64 * j < a.D) o[j] = o[j] * al + p * ldc<CT>(a.v_pages, vo + lane + 64 * j);
  }
  if (lane == 0) sm[wave] = m, sl[wave] = l;
#pragma unroll
  for (int j = 0; j < 4; j++) so[wave][lane + 64 * j] = o[j];
  __syncthreads();
  const float M = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3]));
  float L = 0.f, O = 0.f;
  for (int w = 0; w < 4; w++) {
    const float f = expf(sm[w] - (M == -__builtin_inff() ? 0.f : M));
    L += f * sl[w];
    O += f * so[w][tid];
  }
  const size_t row = (size_t)b * a.Hq + hq;
  if (tid < a.D)
    ub_store<DT>(a.out, row * a.D + tid, L == 0.f ? 0.f : O / L * (a.v_scale ? a.v_scale[h] : 1.f));
  if (tid == 0 && a.lse) a.lse[row] = M + logf(L);
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
  UB_REQUIRE(a.S > 0 && a.P >= 0 && a.width >= 0 && (int64_t)a.width * a.S <= 0x7fffffff,
             "%s: S=%d P=%d width=%d", nm, a.S, a.P, a.width);
  UB_REQUIRE(a.window >= 0 && a.softcap >= 0.f, "%s: window=%d softcap=%g", nm, a.window, a.softcap);
  if (a.B == 0 || a.Hq == 0) return UB_OK;
  UB_REQUIRE(a.q && a.out && a.lens && (a.tables || a.width == 0), "%s: null pointer", nm);
  UB_REQUIRE(a.P == 0 || (a.k_pages && a.v_pages), "%s: null pages", nm);
  UB_REQUIRE((int64_t)a.B * a.Hq < 1 << 23, "%s: B=%d Hq=%d", nm, a.B, a.Hq);
  int* err = ub_error_flag();
  UB_REQUIRE(err, "%s: no device flag", nm);
  hipStream_t s = ub_stream(stream);
  const int grid = a.B * a.Hq;
  if (a.dtype == UB_BF16 && a.cache_dtype == UB_BF16) k_decode<UB_BF16, UB_BF16><<<grid, 256, 0, s>>>(a, err);
  else if (a.dtype == UB_BF16) k_decode<UB_BF16, UB_E4M3><<<grid, 256, 0, s>>>(a, err);
  else if (a.cache_dtype == UB_F16) k_decode<UB_F16, UB_F16><<<grid, 256, 0, s>>>(a, err);
  else k_decode<UB_F16, UB_E4M3><<<grid, 256, 0, s>>>(a, err);
  return ub_check_launch(nm);
}
