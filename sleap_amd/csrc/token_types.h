// What the token operators (rotary.hip, attention.hip, attention_bwd.hip, adamw.hip) share: element types chosen by an argument of
// the call (not by the library build), and divisions by numbers that are known at the launch.
#pragma once
#include <hip/hip_runtime.h>

#include <cstdint>

namespace sa {

// element <-> float; rounding to 16 bits is to nearest even (v_cvt_pk_bf16_f32 / v_cvt_f16_f32)
template <typename T>
__device__ __forceinline__ float to_f32(T v) {
  return static_cast<float>(v);
}
template <typename T>
__device__ __forceinline__ T from_f32(float v) {
  return static_cast<T>(v);
}

// n / d for n < 2^31 by one multiplication: m = ceil(2^32 (2^s - d) / d), s = ceil(log2 d) (Granlund, Montgomery 1994)
struct FastDiv {
  uint32_t d, m, s;
};
inline FastDiv fast_div(uint32_t d) {
  uint32_t s = 0;
  while ((1ull << s) < d) ++s;
  return {d, (uint32_t)((((1ull << s) - d) << 32) / d + 1), s};
}
__device__ __forceinline__ uint32_t div_by(uint32_t n, const FastDiv& f) { return (__umulhi(n, f.m) + n) >> f.s; }

// A grid dimension has less than 2^32 threads; a launch of more runs some of them and reports no error. Workgroups (256 threads at most) are
// counted along rows of 2^23; a kernel returns, or stores nothing, where its workgroup's number is not below the launch's.
constexpr uint32_t GRID_ROW = 1u << 23;
inline dim3 grid_of(uint64_t blocks) {
  return blocks <= GRID_ROW ? dim3((uint32_t)blocks) : dim3(GRID_ROW, (uint32_t)((blocks + GRID_ROW - 1) / GRID_ROW));
}
__device__ __forceinline__ uint32_t workgroup() { return blockIdx.y * GRID_ROW + blockIdx.x; }

}  // namespace sa
