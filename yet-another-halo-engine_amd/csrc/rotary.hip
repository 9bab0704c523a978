// Rotary positions of query and key rows, and the frequency table they are turned by.
//
// A pair (x, y) of a row becomes (x c - y s, y c + x s), c and s the cosine and sine of pos * f_p times a magnitude; before
// that a row may be normalised by its root mean square. The rows are read and written once, so memory is the bound; what
// keeps a kernel from it here is the number of loads in flight and the sines. A workgroup takes a token: its pairs'
// cosines and sines (they depend on the position and the pair, not on the head) are worked out once into LDS, one pair
// a thread, and its rows are dealt to groups of lanes, a lane holding two pieces of four dims. In the half layout the
// pieces are four first and their four second members, in the interleaved layout they are neighbours: either way a lane
// holds whole pairs, and no value crosses lanes but the sum of squares. 8 x 2048 tokens of 24 + 4 heads of 256 dims, bf16: 87
// us for 470 MB, 5.4 TB/s; a step of 64 tokens 4.3 us, most of it the way from positions to sines to rows.
#include <cmath>

#include "common.hpp"
#include "quant.hpp"
#include "rotary.hpp"
#include "store.hpp"

namespace yahkv {
namespace {

struct ApplyArgs {
  RotaryArgs r;
  const int32_t* positions;
  const int32_t* start_pos;
  const int32_t* n_valid;
  int32_t n_new, hd, lanes;  // lanes: lanes of a row, a power of two, at least hd / 8
  int32_t n_rows, rows_per_group;  // rows of a token (query heads, then key heads), and of one workgroup of it
  RowsArgs qs, qd, ks, kd;   // qs.n_heads may be 0
};

constexpr int kRowThreads = 256;

// AT_ONCE: rows that a lane has on their way. Two for long calls (8 x 2048 tokens of 28 rows of 256 dims 87 us, with one 90, with
// four 89; 5 x 1037 tokens of 32 rows of 128: 22.7, 23.3, 25.1), one for short ones, which wait for their code (64 tokens:
// 4.3 us, with two 5.4, with four 7.5).
template <int SRC, int AT_ONCE>
__global__ __launch_bounds__(kRowThreads) void RotaryRows(const ApplyArgs a) {
  const int token = blockIdx.x, s = token / a.n_new, t = token % a.n_new;
  const int lanes = a.lanes, lane = threadIdx.x & (lanes - 1), slot = threadIdx.x / lanes, slots = kRowThreads / lanes;
  if (a.n_valid != nullptr && t >= a.n_valid[s]) return;  // padding row of a short chunk
  const int row_end = min(a.n_rows, static_cast<int>(blockIdx.y + 1) * a.rows_per_group);
  // this lane's two pieces: whole pairs, or dims that pass through
  const int rot = a.r.rot, half = rot / 2, first = a.r.first;
  const bool has = lane < a.hd / 8, turned = lane < rot / 8;
  int e0 = 0, e1 = 4;
  if (turned) {
    e0 = a.r.layout == YAHKV_ROTARY_HALF ? first + 4 * lane : first + 8 * lane;
    e1 = a.r.layout == YAHKV_ROTARY_HALF ? e0 + half : e0 + 4;
  } else if (has) {
    const int p0 = 8 * (lane - rot / 8), p1 = p0 + 4;  // places among the dims that are not rotated
    e0 = p0 < first ? p0 : p0 + rot, e1 = p1 < first ? p1 : p1 + rot;
  }
  auto place = [&](int row, bool src, const RowsArgs** rows) -> int64_t {
    const bool is_q = row < a.qs.n_heads;
    const RowsArgs& r = src ? (is_q ? a.qs : a.ks) : (is_q ? a.qd : a.kd);
    *rows = &r;
    return s * r.seq + t * r.token + (is_q ? row : row - a.qs.n_heads) * r.head;
  };
  uint4 raw[AT_ONCE][2];
  auto request = [&](int row0) {
#pragma unroll
    for (int j = 0; j < AT_ONCE; ++j) {
      const RowsArgs* r;
      const int64_t at = place(min(row0 + slots * j, row_end - 1), true, &r);
      raw[j][0] = LoadRaw4(r->data, at + e0, SRC), raw[j][1] = LoadRaw4(r->data, at + e1, SRC);
    }
  };
  const int row_first = blockIdx.y * a.rows_per_group + slot;
  request(row_first);  // (asked for before the sines are worked out)

  __shared__ __align__(16) float cs[256], sn[256];
  const int pos = a.positions != nullptr ? a.positions[static_cast<int64_t>(s) * a.n_new + t] : a.start_pos[s] + t;
  for (int p = threadIdx.x; p < half; p += kRowThreads) {
    float c, v;
    TurnCosSin(pos, a.r.turns[p], &c, &v);
    cs[p] = c * a.r.magnitude, sn[p] = v * a.r.magnitude;
  }
  __syncthreads();
  float4 c4 = {1.0f, 1.0f, 1.0f, 1.0f}, s4 = {0.0f, 0.0f, 0.0f, 0.0f};
  if (turned) c4 = *reinterpret_cast<const float4*>(&cs[4 * lane]), s4 = *reinterpret_cast<const float4*>(&sn[4 * lane]);
  const bool halves = !turned || a.r.layout == YAHKV_ROTARY_HALF;

  for (int row0 = row_first; row0 < row_end; row0 += slots * AT_ONCE) {
    float4 x[AT_ONCE], y[AT_ONCE];
#pragma unroll
    for (int j = 0; j < AT_ONCE; ++j) x[j] = Widen4(raw[j][0], SRC), y[j] = Widen4(raw[j][1], SRC);
    if (row0 + slots * AT_ONCE < row_end) request(row0 + slots * AT_ONCE);
#pragma unroll
    for (int j = 0; j < AT_ONCE; ++j) {
      const int row = row0 + slots * j;
      if (row >= row_end) break;
      float4 u = x[j], v = y[j];
      if (a.r.normalise) {
        float ss = u.x * u.x + u.y * u.y + u.z * u.z + u.w * u.w + v.x * v.x + v.y * v.y + v.z * v.z + v.w * v.w;
        if (!has) ss = 0.0f;
        for (int o = lanes / 2; o > 0; o >>= 1) ss += __shfl_xor(ss, o, 64);
        const float inv = 1.0f / sqrtf(ss / static_cast<float>(a.hd) + a.r.eps);
        const float* w = row < a.qs.n_heads ? a.r.q_weight : a.r.k_weight;
        float4 w0 = {1.0f, 1.0f, 1.0f, 1.0f}, w1 = w0;
        if (w != nullptr) w0 = *reinterpret_cast<const float4*>(w + e0), w1 = *reinterpret_cast<const float4*>(w + e1);
        u = float4{u.x * inv * w0.x, u.y * inv * w0.y, u.z * inv * w0.z, u.w * inv * w0.w};
        v = float4{v.x * inv * w1.x, v.y * inv * w1.y, v.z * inv * w1.z, v.w * inv * w1.w};
      }
      float4 p, q;
      if (halves) {
        p = float4{u.x * c4.x - v.x * s4.x, u.y * c4.y - v.y * s4.y, u.z * c4.z - v.z * s4.z, u.w * c4.w - v.w * s4.w};
        q = float4{v.x * c4.x + u.x * s4.x, v.y * c4.y + u.y * s4.y, v.z * c4.z + u.z * s4.z, v.w * c4.w + u.w * s4.w};
      } else {
        p = float4{u.x * c4.x - u.y * s4.x, u.y * c4.x + u.x * s4.x, u.z * c4.y - u.w * s4.y, u.w * c4.y + u.z * s4.y};
        q = float4{v.x * c4.z - v.y * s4.z, v.y * c4.z + v.x * s4.z, v.z * c4.w - v.w * s4.w, v.w * c4.w + v.z * s4.w};
      }
      if (!turned) p = u, q = v;  // (NaN and infinities of the other dims must not meet a zero sine)
      if (has) {
        const RowsArgs* r;
        const int64_t at = place(row, false, &r);
        Store4(r->data, at + e0, r->dtype, p), Store4(r->data, at + e1, r->dtype, q);
      }
    }
  }
}

template <int AT_ONCE>
void LaunchRows(int32_t src, dim3 grid, hipStream_t st, const ApplyArgs& a) {
  if (src == YAHKV_F32) hipLaunchKernelGGL((RotaryRows<YAHKV_F32, AT_ONCE>), grid, dim3(kRowThreads), 0, st, a);
  else if (src == YAHKV_F16) hipLaunchKernelGGL((RotaryRows<YAHKV_F16, AT_ONCE>), grid, dim3(kRowThreads), 0, st, a);
  else hipLaunchKernelGGL((RotaryRows<YAHKV_BF16, AT_ONCE>), grid, dim3(kRowThreads), 0, st, a);
}

}  // namespace

int LaunchRotaryRows(const RotaryArgs& r, int32_t head_dim, const int32_t* positions, const int32_t* start_pos,
                     const int32_t* n_valid, int32_t n_seqs, int32_t n_new, const RowsArgs& q_src, const RowsArgs& q_dst,
                     const RowsArgs& k_src, const RowsArgs& k_dst, hipStream_t st) {
  const int64_t tokens = int64_t(n_seqs) * n_new;
  ApplyArgs a{};
  a.r = r, a.positions = positions, a.start_pos = start_pos, a.n_valid = n_valid, a.n_new = n_new, a.hd = head_dim;
  a.qs = q_src, a.qd = q_dst, a.ks = k_src, a.kd = k_dst, a.n_rows = q_src.n_heads + k_src.n_heads;
  a.lanes = 1;
  while (a.lanes < head_dim / 8) a.lanes *= 2;
  // Few tokens: a token's rows go to several workgroups, each with one round of loads; many: all rows of a token share
  // one workgroup's sines.
  const bool few = tokens < 1024;
  a.rows_per_group = few ? kRowThreads / a.lanes : a.n_rows;
  const unsigned groups = static_cast<unsigned>((a.n_rows + a.rows_per_group - 1) / a.rows_per_group);
  const dim3 grid(static_cast<unsigned>(tokens), groups);
  const int32_t src = q_src.n_heads != 0 ? q_src.dtype : k_src.dtype;
  if (few) LaunchRows<1>(src, grid, st, a);
  else LaunchRows<2>(src, grid, st, a);
  return LaunchStatus();
}

}  // namespace yahkv

using namespace yahkv;

extern "C" int yahkv_rotary_table(const yahkv_rotary_spec* spec, uint64_t* turns, float* magnitude) {
  if (spec == nullptr || turns == nullptr || magnitude == nullptr) return YAHKV_ERR_ARG;
  const int r = spec->rotary_dim, half = r / 2;
  if (r < 8 || r % 8 != 0 || !(spec->theta > 1.0) || !std::isfinite(spec->theta)) return YAHKV_ERR_ARG;
  if (spec->scaling < YAHKV_ROTARY_PLAIN || spec->scaling > YAHKV_ROTARY_BANDS) return YAHKV_ERR_ARG;
  const bool bands = spec->scaling == YAHKV_ROTARY_YARN || spec->scaling == YAHKV_ROTARY_BANDS;
  const double f = spec->scaling == YAHKV_ROTARY_PLAIN ? 1.0 : spec->factor;
  if (!(f >= 1.0) || !std::isfinite(f)) return YAHKV_ERR_ARG;
  if (bands && (!(spec->original_len > 0.0) || !std::isfinite(spec->original_len) || !(spec->low > 0.0) ||
                !(spec->high > spec->low) || !std::isfinite(spec->high)))
    return YAHKV_ERR_ARG;
  // In 64 bits of significand: an entry's unit is 2^-64 of a turn, and a double's last bit of the fast pairs is 2^8 of them,
  // 3e-7 radians at position 2^31. The entries are within 2^-63 turns.
  typedef long double real;  // (x86-64's)
  const real pi2 = 6.283185307179586476925286766559005768L, factor = f, length = spec->original_len, low = spec->low, high = spec->high;
  real theta = spec->theta;
  if (spec->scaling == YAHKV_ROTARY_NTK) theta *= std::pow(factor, real(r) / (r - 2));
  // YaRN: the pairs that make `high` and `low` turns within the original context bound the ramp, in whole pairs
  real ramp0 = 0, ramp1 = 1;
  if (spec->scaling == YAHKV_ROTARY_YARN) {
    auto pair_of = [&](real n) { return r * std::log(length / (n * pi2)) / (2 * std::log(theta)); };
    ramp0 = std::fmax(std::floor(pair_of(high)), real(0)), ramp1 = std::fmin(std::ceil(pair_of(low)), real(r - 1));
  }
  for (int p = 0; p < half; ++p) {
    const real inv = std::pow(theta, -2 * real(p) / r);
    real w = inv;
    if (spec->scaling == YAHKV_ROTARY_LINEAR) w = inv / factor;
    if (spec->scaling == YAHKV_ROTARY_YARN) {
      const real x = std::fmin(std::fmax((p - ramp0) / std::fmax(ramp1 - ramp0, real(0.001)), real(0)), real(1));
      w = inv / factor * x + inv * (1 - x);
    }
    if (spec->scaling == YAHKV_ROTARY_BANDS) {
      const real n = length * inv / pi2;  // turns within the original context
      const real x = std::fmin(std::fmax((n - low) / (high - low), real(0)), real(1));
      w = inv / factor * (1 - x) + inv * x;
    }
    turns[p] = static_cast<uint64_t>(std::rint(std::ldexp(w / pi2, 64)));  // w <= 1: below 2^62
  }
  *magnitude = spec->scaling == YAHKV_ROTARY_YARN ? static_cast<float>(0.1 * std::log(f) + 1.0) : 1.0f;
  return YAHKV_OK;
}

extern "C" int yahkv_rotary_apply(const yahkv_rotary* rotary, int32_t head_dim, const int32_t* positions, int32_t n_seqs,
                                  int32_t n_new, const yahkv_rows* q_src, const yahkv_rows* q_dst, const yahkv_rows* k_src,
                                  const yahkv_rows* k_dst, void* stream) {
  if (head_dim < 8 || head_dim > 512 || head_dim % 8 != 0) return YAHKV_ERR_SHAPE;
  ApplyArgs a{};
  if (const int st = CheckRotary(rotary, head_dim, &a.r)) return st;
  if (positions == nullptr || n_seqs <= 0 || n_new <= 0) return YAHKV_ERR_ARG;
  if ((q_src == nullptr) != (q_dst == nullptr) || (k_src == nullptr) != (k_dst == nullptr)) return YAHKV_ERR_ARG;
  if (q_src == nullptr && k_src == nullptr) return YAHKV_ERR_ARG;
  if (q_src != nullptr) {
    if (const int st = CheckRows(q_src, &a.qs)) return st;
    if (const int st = CheckRowsOut(q_dst, n_seqs, n_new, &a.qd)) return st;
    if (a.qs.n_heads != a.qd.n_heads) return YAHKV_ERR_ARG;
  }
  if (k_src != nullptr) {
    if (const int st = CheckRows(k_src, &a.ks)) return st;
    if (const int st = CheckRowsOut(k_dst, n_seqs, n_new, &a.kd)) return st;
    if (a.ks.n_heads != a.kd.n_heads || (q_src != nullptr && a.ks.dtype != a.qs.dtype)) return YAHKV_ERR_ARG;
  }
  const int64_t tokens = int64_t(n_seqs) * n_new, rows = int64_t(a.qs.n_heads) + a.ks.n_heads;
  if (tokens > 0x7FFFFFFF || rows > 65536) return YAHKV_ERR_SHAPE;
  return LaunchRotaryRows(a.r, head_dim, positions, nullptr, nullptr, n_seqs, n_new, a.qs, a.qd, a.ks, a.kd, static_cast<hipStream_t>(stream));
}
