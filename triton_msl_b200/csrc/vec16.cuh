// 16-bit values two to a register: widening and narrowing by whole registers, where
// converting value by value costs an extraction or a merge each.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cstdint>

namespace b2 {

template <typename T> __device__ __forceinline__ void widen2(uint32_t w, float& lo, float& hi);
template <> __device__ __forceinline__ void widen2<__nv_bfloat16>(uint32_t w, float& lo, float& hi) {
  lo = __uint_as_float(w << 16);
  hi = __uint_as_float(w & 0xffff0000u);
}
template <> __device__ __forceinline__ void widen2<__half>(uint32_t w, float& lo, float& hi) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
  lo = f.x;
  hi = f.y;
}
template <typename T> __device__ __forceinline__ uint32_t narrow2(float lo, float hi);
template <> __device__ __forceinline__ uint32_t narrow2<__nv_bfloat16>(float lo, float hi) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <> __device__ __forceinline__ uint32_t narrow2<__half>(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

}  // namespace b2
