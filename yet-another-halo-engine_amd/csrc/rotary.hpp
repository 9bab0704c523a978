// Rotary positions: the angle of a pair, the launch view of yahkv_rotary / yahkv_rows, and their checks. Shared by the
// fused append (append.hip) and the rows kernel (rotary.hip).
#ifndef YAHKV_ROTARY_HPP_
#define YAHKV_ROTARY_HPP_

#include "common.hpp"

namespace yahkv {

struct RotaryArgs {
  const uint64_t* turns;
  int32_t rot, first, layout, normalise;
  float magnitude, eps;
  const float* q_weight;
  const float* k_weight;
};
struct RowsArgs {
  void* data;
  int32_t dtype, n_heads;
  int64_t seq, token, head;  // strides in elements
};

// cos and sin of the angle pos * f, f in turns as a 0.64 binary fraction: the product modulo 2^64 is the angle's exact
// fraction of a turn (f itself is rounded to 2^-65 turns: at position 2^31 that is 2^-34 turns). Its top 32 bits split
// into a quarter turn and a remainder of at most an eighth of a turn either way, which f32 holds to 2^-24 relative.
__device__ __forceinline__ void TurnCosSin(int pos, uint64_t turns, float* c, float* s) {
  const uint64_t angle = static_cast<uint64_t>(static_cast<int64_t>(pos)) * turns;
  const uint32_t top = static_cast<uint32_t>(angle >> 32);
  const uint32_t quarter = (top + 0x20000000u) >> 30;
  const int32_t rest = static_cast<int32_t>(top - (quarter << 30));
  float sv, cv;
  sincospif(static_cast<float>(rest) * 0x1p-31f, &sv, &cv);  // half turns
  const float a = quarter & 1 ? sv : cv, b = quarter & 1 ? cv : sv;
  *c = quarter == 1 || quarter == 2 ? -a : a;
  *s = quarter >= 2 ? -b : b;
}

inline bool KnownDtype(int32_t t) { return t == YAHKV_F32 || t == YAHKV_F16 || t == YAHKV_BF16; }
inline bool Aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

inline int CheckRotary(const yahkv_rotary* r, int32_t head_dim, RotaryArgs* a) {
  if (r == nullptr || r->turns == nullptr || (reinterpret_cast<uintptr_t>(r->turns) & 7)) return YAHKV_ERR_ARG;
  if (r->rotary_dim < 8 || r->rotary_dim % 8 != 0 || r->first_dim < 0 || r->first_dim % 4 != 0) return YAHKV_ERR_ARG;
  if (r->rotary_dim > head_dim || r->first_dim > head_dim - r->rotary_dim) return YAHKV_ERR_ARG;
  if (r->layout != YAHKV_ROTARY_HALF && r->layout != YAHKV_ROTARY_INTERLEAVED) return YAHKV_ERR_ARG;
  if (r->normalise != 0 && !(r->eps >= 0.0f)) return YAHKV_ERR_ARG;
  if (!Aligned16(r->q_weight) || !Aligned16(r->k_weight)) return YAHKV_ERR_ARG;
  *a = RotaryArgs{r->turns, r->rotary_dim, r->first_dim, r->layout, r->normalise != 0, r->magnitude, r->eps, r->q_weight, r->k_weight};
  return YAHKV_OK;
}
inline int CheckRows(const yahkv_rows* r, RowsArgs* a) {
  if (r == nullptr || r->data == nullptr || !Aligned16(r->data) || !KnownDtype(r->dtype) || r->n_heads <= 0) return YAHKV_ERR_ARG;
  const int64_t unit = r->dtype == YAHKV_F32 ? 4 : 8;  // elements in 16 bytes
  if (r->seq_stride % unit != 0 || r->token_stride % unit != 0 || r->head_stride % unit != 0) return YAHKV_ERR_ARG;
  *a = RowsArgs{r->data, r->dtype, r->n_heads, r->seq_stride, r->token_stride, r->head_stride};
  return YAHKV_OK;
}

}  // namespace yahkv

#endif  // YAHKV_ROTARY_HPP_
