// Codes of the block formats as f16, exact.
#ifndef YAHKV_CODES_HPP_
#define YAHKV_CODES_HPP_

#include "decode_cut.hpp"

namespace yahkv {

// Eight int8 codes (two dwords) as eight f16, exact. 0x6400 | u is the f16 1024 + u; u = code + 128.
__device__ __forceinline__ h8v Codes8(uint32_t w0, uint32_t w1) {
  const h2v off = {static_cast<_Float16>(-1152.0f), static_cast<_Float16>(-1152.0f)};
  const uint32_t x0 = w0 ^ 0x80808080u, x1 = w1 ^ 0x80808080u;
  const h2v a = __builtin_bit_cast(h2v, __builtin_amdgcn_perm(0x64646464u, x0, 0x04010400u)) + off;
  const h2v b = __builtin_bit_cast(h2v, __builtin_amdgcn_perm(0x64646464u, x0, 0x04030402u)) + off;
  const h2v c = __builtin_bit_cast(h2v, __builtin_amdgcn_perm(0x64646464u, x1, 0x04010400u)) + off;
  const h2v d = __builtin_bit_cast(h2v, __builtin_amdgcn_perm(0x64646464u, x1, 0x04030402u)) + off;
  return h8v{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// Eight nibbles of two dwords as eight f16 holding (nibble - 8), exact. Low nibbles: 0x6400 | n is 1024 + n. High
// nibbles stay in place: 0x6400 | (n << 4) is 1024 + 16 n, and one fused multiply-add takes it to n - 8.
__device__ __forceinline__ h8v NibblesLo8(uint32_t w0, uint32_t w1) {
  const h2v off = {static_cast<_Float16>(-1032.0f), static_cast<_Float16>(-1032.0f)};
  const uint32_t x0 = w0 & 0x0F0F0F0Fu, x1 = w1 & 0x0F0F0F0Fu;
  const h2v a = __builtin_bit_cast(h2v, __builtin_amdgcn_perm(0x64646464u, x0, 0x04010400u)) + off;
  const h2v b = __builtin_bit_cast(h2v, __builtin_amdgcn_perm(0x64646464u, x0, 0x04030402u)) + off;
  const h2v c = __builtin_bit_cast(h2v, __builtin_amdgcn_perm(0x64646464u, x1, 0x04010400u)) + off;
  const h2v d = __builtin_bit_cast(h2v, __builtin_amdgcn_perm(0x64646464u, x1, 0x04030402u)) + off;
  return h8v{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}
__device__ __forceinline__ h8v NibblesHi8(uint32_t w0, uint32_t w1) {
  const h2v mul = {static_cast<_Float16>(0.0625f), static_cast<_Float16>(0.0625f)};
  const h2v off = {static_cast<_Float16>(-72.0f), static_cast<_Float16>(-72.0f)};
  const uint32_t x0 = w0 & 0xF0F0F0F0u, x1 = w1 & 0xF0F0F0F0u;
  const h2v a = __builtin_elementwise_fma(__builtin_bit_cast(h2v, __builtin_amdgcn_perm(0x64646464u, x0, 0x04010400u)), mul, off);
  const h2v b = __builtin_elementwise_fma(__builtin_bit_cast(h2v, __builtin_amdgcn_perm(0x64646464u, x0, 0x04030402u)), mul, off);
  const h2v c = __builtin_elementwise_fma(__builtin_bit_cast(h2v, __builtin_amdgcn_perm(0x64646464u, x1, 0x04010400u)), mul, off);
  const h2v d = __builtin_elementwise_fma(__builtin_bit_cast(h2v, __builtin_amdgcn_perm(0x64646464u, x1, 0x04030402u)), mul, off);
  return h8v{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

}  // namespace yahkv

#endif  // YAHKV_CODES_HPP_
