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
// fraction of a turn (yahkv_rotary_table's f is within 2^-63 turns: at position 2^31 that is 2^-32 turns). Its top 32 bits split
// into a quarter turn and a remainder x of at most an eighth of a turn either way, which f32 holds to 2^-24 relative; on
// |x| <= pi / 4 the Taylor sums up to x^9 and x^8 are short of sine and cosine by x^11 / 11! < 2^-28 and x^10 / 10! < 2^-25.
__device__ __forceinline__ void TurnCosSin(int pos, uint64_t turns, float* c, float* s) {
  const uint32_t p = static_cast<uint32_t>(pos), lo = static_cast<uint32_t>(turns), hi = static_cast<uint32_t>(turns >> 32);
  // the high word of the product's low 64 bits, pos as a signed number
  const uint32_t top = __umulhi(p, lo) + p * hi - (pos < 0 ? lo : 0u);
  const uint32_t quarter = (top + 0x20000000u) >> 30;
  const float x = static_cast<float>(static_cast<int32_t>(top - (quarter << 30))) * 0x1.921fb6p-30f;  // 2 pi / 2^32
  const float x2 = x * x;
  float sv = __builtin_fmaf(x2, 1.0f / 362880.0f, -1.0f / 5040.0f);
  sv = __builtin_fmaf(x2, sv, 1.0f / 120.0f), sv = __builtin_fmaf(x2, sv, -1.0f / 6.0f);
  sv = __builtin_fmaf(x2 * x, sv, x);
  float cv = __builtin_fmaf(x2, 1.0f / 40320.0f, -1.0f / 720.0f);
  cv = __builtin_fmaf(x2, cv, 1.0f / 24.0f), cv = __builtin_fmaf(x2, cv, -0.5f);
  cv = __builtin_fmaf(x2, cv, 1.0f);
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

// Destination rows: two tokens or heads at one address would be written in any order.
inline int CheckRowsOut(const yahkv_rows* r, int32_t n_seqs, int32_t n_new, RowsArgs* a) {
  if (const int st = CheckRows(r, a)) return st;
  if ((n_seqs > 1 && a->seq == 0) || (n_new > 1 && a->token == 0) || (a->n_heads > 1 && a->head == 0)) return YAHKV_ERR_ARG;
  return YAHKV_OK;
}

// The rows kernel (rotary.hip): q and / or k rows (n_heads 0: none) of n_seqs x n_new tokens, turned by positions[s][t] or,
// where that is null, by start_pos[s] + t; rows at or past n_valid[s] (null: n_new) are left alone. Arguments are checked.
int LaunchRotaryRows(const RotaryArgs& r, int32_t head_dim, const int32_t* positions, const int32_t* start_pos,
                     const int32_t* n_valid, int32_t n_seqs, int32_t n_new, const RowsArgs& q_src, const RowsArgs& q_dst,
                     const RowsArgs& k_src, const RowsArgs& k_dst, hipStream_t st);

}  // namespace yahkv

#endif  // YAHKV_ROTARY_HPP_
