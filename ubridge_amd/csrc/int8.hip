// int8.hip -- int8 W8A8 linear on gfx950:
//
//   y[m, n] = T( (sum_k a[m, k] w[n, k]) sa[m] sw[n] + bias[n] )
//
// a[m, k] = round(x[m, k] / sa[m]) (ties to even), sa[m] = max_k |x[m, k]| /
// 127, or 1 for a row of zeros; sw one f32 scale an output channel.  The dot is
// exact in int32 (|a w| <= 127 * 128, so K <= 132104), the epilogue f32, and
// the sum rounds once, to x's type T.  The weight's scale is multiplied in first:
// sa reaches both ends of f32, and with it first rows near the top overflowed.  A row that holds an infinity or a NaN
// has no scale and gives a row of NaN.
//
// Rows of a and w are padded with zeros to ld bytes, a multiple of 128.
#include "common.h"

namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));

template <int DT>
__device__ __forceinline__ float row_scale(float amax) {
  // (an infinite or NaN maximum: no scale)
  return !(amax < __builtin_inff()) ? __builtin_nanf("") : amax > 0.f ? __fdiv_rn(amax, 127.0f) : 1.0f;
}

// code of x under scale s: |x / s| <= 127 up to the rounding of s, which for
// a denormal s is as large as s (hence the clamp); 0 where s is NaN or 0
__device__ __forceinline__ int code(float x, float s) {
  const float q = rintf(__fdiv_rn(x, s));
  return q == q ? (int)fminf(fmaxf(q, -127.f), 127.f) : 0;
}

// One workgroup a row.
template <int DT>
__global__ void __launch_bounds__(256) k_quant(const void* __restrict__ x, int8_t* __restrict__ q,
                                               float* __restrict__ scale, int K, int ld) {
  __shared__ float wm[4];
  const int tid = threadIdx.x;
  const size_t r = blockIdx.x;
  float amax = 0.f;
  bool bad = false;
  for (int c = tid; c < K; c += 256) {
    const float v = fabsf(ub_load<DT>(x, r * K + c));
    bad |= !(v < __builtin_inff());
    amax = fmaxf(amax, v);
  }
  if (bad) amax = __builtin_inff();
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) amax = fmaxf(amax, __shfl_xor(amax, o, 64));
  if ((tid & 63) == 0) wm[tid >> 6] = amax;
  __syncthreads();
  amax = fmaxf(fmaxf(wm[0], wm[1]), fmaxf(wm[2], wm[3]));
  const float s = row_scale<DT>(amax);
  for (int c = tid; c < ld; c += 256)
    q[r * ld + c] = c < K ? (int8_t)code(ub_load<DT>(x, r * K + c), s) : (int8_t)0;
  if (tid == 0) scale[r] = s;
}

// One wavefront per 16 x 16 outputs: v_mfma_i32_16x16x64_i8 on fragments
// straight from memory.
template <int DT>
__global__ void __launch_bounds__(64) k_i8_gemm(const int8_t* __restrict__ a,
                                                const float* __restrict__ sa,
                                                const int8_t* __restrict__ w,
                                                const float* __restrict__ sw,
                                                const float* __restrict__ bias,
                                                void* __restrict__ y, int M, int N, int ld) {
  const int lane = threadIdx.x, r = lane & 15, h = lane >> 4;
  const int m0 = blockIdx.y * 16, n0 = blockIdx.x * 16;
  const int8_t* pa = a + (size_t)min(m0 + r, M - 1) * ld + 16 * h;
  const int8_t* pw = w + (size_t)min(n0 + r, N - 1) * ld + 16 * h;
  i32x4 acc = {0, 0, 0, 0};
  for (int k = 0; k < ld; k += 64)
    acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(*(const i32x4*)(pa + k), *(const i32x4*)(pw + k), acc,
                                                0, 0, 0);
  const int n = n0 + r;
  if (n >= N) return;
  const float s = sw[n], b = bias ? bias[n] : 0.f;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const int m = m0 + 4 * h + i;
    if (m < M) ub_store<DT>(y, (size_t)m * N + n, (float)acc[i] * s * sa[m] + b);
  }
}

template <int DT>
void linear(const void* x, const int8_t* w, const float* sw, const float* bias, void* y, int8_t* q,
            float* sa, int M, int K, int N, int ld, hipStream_t s) {
  k_quant<DT><<<M, 256, 0, s>>>(x, q, sa, K, ld);
  k_i8_gemm<DT><<<dim3(ub_cdiv(N, 16), ub_cdiv(M, 16)), 64, 0, s>>>(q, sa, w, sw, bias, y, M, N, ld);
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
  hipStream_t s = ub_stream(stream);
  UbScratch ws(s, (size_t)M * ld + sizeof(float) * (size_t)M);
  int8_t* q = (int8_t*)ws.get();
  if (!q) return ub_set_error(UB_ERR_LAUNCH, "%s: no workspace", nm);
  float* sa = (float*)(q + (size_t)M * ld);
  if (dtype == UB_F32) linear<UB_F32>(x, w, sw, bias, y, q, sa, M, K, N, ld, s);
  else if (dtype == UB_F16) linear<UB_F16>(x, w, sw, bias, y, q, sa, M, K, N, ld, s);
  else linear<UB_BF16>(x, w, sw, bias, y, q, sa, M, K, N, ld, s);
  return ub_check_launch(nm);
}
