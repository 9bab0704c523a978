// f32 values to elements of an array of yahkv_dtype, rounded to nearest even: one, or four consecutive ones (element index a
// multiple of 4).
#ifndef YAHKV_STORE_HPP_
#define YAHKV_STORE_HPP_

#include "common.hpp"

namespace yahkv {

__device__ __forceinline__ void Store1(void* dst, size_t i, int dtype, float v) {
  if (dtype == YAHKV_F32) static_cast<float*>(dst)[i] = v;
  else if (dtype == YAHKV_F16) static_cast<_Float16*>(dst)[i] = static_cast<_Float16>(v);
  else static_cast<__bf16*>(dst)[i] = static_cast<__bf16>(v);
}

__device__ __forceinline__ void Store4(void* dst, size_t i, int dtype, float4 v) {
  if (dtype == YAHKV_F32) {
    *reinterpret_cast<float4*>(static_cast<float*>(dst) + i) = v;
    return;
  }
  uint32_t lo, hi;
  if (dtype == YAHKV_F16) {
    typedef _Float16 h2v __attribute__((ext_vector_type(2)));
    lo = __builtin_bit_cast(uint32_t, h2v{static_cast<_Float16>(v.x), static_cast<_Float16>(v.y)});
    hi = __builtin_bit_cast(uint32_t, h2v{static_cast<_Float16>(v.z), static_cast<_Float16>(v.w)});
  } else {
    typedef __bf16 b2v __attribute__((ext_vector_type(2)));
    lo = __builtin_bit_cast(uint32_t, b2v{static_cast<__bf16>(v.x), static_cast<__bf16>(v.y)});
    hi = __builtin_bit_cast(uint32_t, b2v{static_cast<__bf16>(v.z), static_cast<__bf16>(v.w)});
  }
  *reinterpret_cast<uint2*>(static_cast<uint16_t*>(dst) + i) = uint2{lo, hi};
}

}  // namespace yahkv

#endif  // YAHKV_STORE_HPP_
