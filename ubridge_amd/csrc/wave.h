// wave.h -- reductions over a wavefront by DPP: within rows of 16 lanes by shifts, from
// each row into the next and from the lower half into the upper, the last lane's result
// read back into every lane.  Six steps of one instruction (two or three of 64 bits); a
// butterfly over LDS takes about 120 cycles a step.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>
#include <type_traits>

namespace {

// f(own value, another lane's) step by step; where there is no such lane 0 stands in
// (`zero`), or the own value.
template <class T, class F>
__device__ __forceinline__ T ub_wave_steps(T v, bool zero, F f) {
  static_assert(sizeof(T) == 4 || sizeof(T) == 8, "one or two registers");
  struct Parts { int w[sizeof(T) / 4]; };
  auto step = [&](auto c) {
    constexpr int C = decltype(c)::value, rows = C == 0x142 ? 0xa : C == 0x143 ? 0xc : 0xf;
    Parts p = __builtin_bit_cast(Parts, v), o;
#pragma unroll
    for (unsigned i = 0; i < sizeof(T) / 4; i++) o.w[i] = __builtin_amdgcn_update_dpp(zero ? 0 : p.w[i], p.w[i], C, rows, 0xf, false);
    v = f(v, __builtin_bit_cast(T, o));
  };
  step(std::integral_constant<int, 0x111>{});  // row_shr:1
  step(std::integral_constant<int, 0x112>{});
  step(std::integral_constant<int, 0x114>{});
  step(std::integral_constant<int, 0x118>{});
  step(std::integral_constant<int, 0x142>{});  // row_bcast:15
  step(std::integral_constant<int, 0x143>{});  // row_bcast:31
  Parts p = __builtin_bit_cast(Parts, v);
#pragma unroll
  for (unsigned i = 0; i < sizeof(T) / 4; i++) p.w[i] = __builtin_amdgcn_readlane(p.w[i], 63);
  return __builtin_bit_cast(T, p);
}
template <class T>
__device__ __forceinline__ T ub_wave_all_sum(T v) {
  return ub_wave_steps(v, true, [](T a, T b) { return a + b; });
}
__device__ __forceinline__ float ub_wave_all_max(float v) {
  return ub_wave_steps(v, false, [](float a, float b) { return fmaxf(a, b); });
}
__device__ __forceinline__ uint32_t ub_wave_all_max(uint32_t v) {
  return ub_wave_steps(v, false, [](uint32_t a, uint32_t b) { return max(a, b); });
}

}  // namespace
