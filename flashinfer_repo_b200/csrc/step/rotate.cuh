// rotate.cuh -- element types and rotation angles shared by the rotary kernels.
#pragma once
#include <cuda_fp16.h>

#include "../common.cuh"

namespace dsa {

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// 16 bytes of a tensor, loaded and stored at once.
template <typename T>
struct __align__(16) Vec {
  static constexpr int kN = 16 / sizeof(T);
  T v[kN];
};

// cos and sin of position * inv_freq.  The angle is taken in turns in 64 bits
// and reduced to half a turn before it is rounded to 32 (a 32-bit product is
// 0.01 rad off at position 1e5): the error is then 2^-25 turns plus 2^-53 of
// the turns made, and sincospif needs no further reduction.
__device__ __forceinline__ void rotation(int64_t position, double inv_freq, float scale, float* c, float* s) {
  constexpr double kInvTwoPi = 0.15915494309189533577;
  const double turns = (double)position * (inv_freq * kInvTwoPi);
  const float half_turns = (float)(2.0 * (turns - rint(turns)));
  sincospif(half_turns, s, c);
  *c *= scale;
  *s *= scale;
}

__device__ __forceinline__ int64_t load_position(const void* positions, int is64, int64_t i) {
  return is64 ? static_cast<const int64_t*>(positions)[i] : static_cast<const int32_t*>(positions)[i];
}

}  // namespace dsa
