// Decode attention of a batch whose sequences share prefixes: each prefix's keys are read and decoded once for all the
// query rows that see them.
//
// Attention splits over any partition of the keys: with m a reference point, l = sum 2^(s_t - m) and o = sum 2^(s_t - m)
// V_t of each part, the whole is (sum 2^(m_p - M) o_p) / (sum 2^(m_p - M) l_p). The prefix's part of a group's rows is a
// matrix product with many rows (sequences x query heads of a kv head), where the tails, one sequence's query heads each,
// stay with the split-K kernel of yahkv_decode_part. So: `SharedPart` leaves partials of the prefixes, the decode kernel
// partials of the tails (from lengths and table rows that begin behind the prefix, which SharedPart writes), `SharedMerge`
// puts them together.
//
// SharedPart is the transposed scheme of the prefill kernels (keys along MFMA rows, query rows along lanes):
//   S^T[key][row] = sum_dim K[key][dim] Q[row][dim]     A = K tile from LDS (16 keys x 32 dims), B = Q^T (registers)
//   O^T[dim][row] += sum_key V^T[dim][key] P^T[key][row]  A = V^T tile from LDS (16 dims x 32 keys), B = P^T (registers)
// A workgroup owns RB * WR * 16 query rows of one (group, kv head) and one stretch of the prefix; its 4 waves are WR along
// the rows and 4 / WR along the keys of a tile. A tile's codes are decoded once per workgroup, into f16 in LDS, by packed
// f16 arithmetic: perm, add, multiply for two values, the product d * code rounded once.
#include "codes.hpp"
#include "common.hpp"
#include "decode_cut.hpp"
#include "store.hpp"

namespace yahkv {
namespace {

constexpr int kSharedWaves = 4;
constexpr float kNone = -1.0e30f;  // reference point of a row before its first tile
// Numerators are 2^(score - m) with m a whole number kBias below the largest score seen: f16 holds them up to 2^kBias and
// down to 2^-14 - kBias with full precision.
constexpr float kBias = 10.0f;

struct SharedArgs {
  Geom g;
  Pools pools;
  const int32_t* table;
  const int32_t* seq_len;
  const int32_t* group_first;
  const int32_t* shared_len;
  int32_t stride, n_seqs, n_groups, max_shared, max_tail;
  const void* q;
  int32_t q_dtype;
  float scale;
  int32_t max_blocks, n_split;  // row blocks of all groups at most; pieces a prefix is cut into
  // workspace
  int32_t* tail_len;    // [n_seqs]
  int32_t* tail_table;  // [n_seqs][tail_stride]
  int32_t tail_stride;
  float* ml;   // [n_seqs][n_q][slots][2]: reference point (base 2) and sum
  float* acc;  // [n_seqs][n_q][slots][D]
  int32_t slots;  // n_split * waves along the keys
};

__device__ __forceinline__ int GroupFirst(const SharedArgs& a, int j) { return min(max(a.group_first[j], 0), a.n_seqs); }
__device__ __forceinline__ int GroupShared(const SharedArgs& a, int j) {  // whole 64-key tiles of its prefix
  return min(min(max(a.shared_len[j], 0), a.max_shared), a.stride * a.g.pt) / kTile * kTile;
}
// The group of sequence s, or -1: the last one that begins at or before it.
__device__ __forceinline__ int GroupOf(const SharedArgs& a, int s) {
  int lo = 0, hi = a.n_groups;  // the first group that begins behind s lies in [lo, hi]
  while (lo < hi) {
    const int mid = (lo + hi) / 2;
    if (GroupFirst(a, mid) <= s) lo = mid + 1;
    else hi = mid;
  }
  return lo > 0 && s < GroupFirst(a, lo) ? lo - 1 : -1;
}
// The keys that a sequence of `len` tokens takes from the prefix of group j: all its whole tiles, or, if it is shorter than
// they are, none: it is then all tail. So every row of SharedPart sees every key, nothing is masked there, and whatever a
// prefix holds that a shorter sequence must not see (an infinity would pass through a zero numerator as NaN) stays
// out of that sequence's sums.
__device__ __forceinline__ int PrefixOf(const SharedArgs& a, int j, int len) {
  const int shared = j < 0 ? 0 : GroupShared(a, j);
  return len < shared ? 0 : shared;
}
// A prefix's pieces: tiles per piece, and how many pieces hold any.
__device__ __forceinline__ int TilesPerPiece(int tiles, int n_split) { return (tiles + n_split - 1) / n_split; }

// Sixteen q8_0 codes times one scale / sixteen scales, or the low or high nibbles of sixteen bytes, as sixteen f16.
template <int FMT>
__device__ __forceinline__ void Halves(const uint4 c, int high, h8v* lo, h8v* hi) {
  if constexpr (FMT == 8) {
    *lo = Codes8(c.x, c.y), *hi = Codes8(c.z, c.w);
  } else if (high) {
    *lo = NibblesHi8(c.x, c.y), *hi = NibblesHi8(c.z, c.w);
  } else {
    *lo = NibblesLo8(c.x, c.y), *hi = NibblesLo8(c.z, c.w);
  }
}
// Products beyond the f16 range saturate (they would be infinite, and an infinite score a NaN): only a scale above
// 65504 / 128 can make one, so the test is one per scale and the slow form is rare.
constexpr float kLargeScale = 511.0f;
__device__ __forceinline__ h8v TimesSaturated(h8v codes, h8v scale) {
  h8v r;
#pragma unroll
  for (int e = 0; e < 8; ++e) r[e] = SaturateToF16(static_cast<float>(codes[e]) * static_cast<float>(scale[e]));
  return r;
}

template <int FMT, int D, int PT, int RB, int WR>
__global__ __launch_bounds__(64 * kSharedWaves) void SharedPart(const SharedArgs a) {
  constexpr int NB = D / 32, NDT = D / 16, KS = D / 32;
  constexpr int WK = kSharedWaves / WR, KT = 4 / WK, S2 = 2 / WK;  // 16-key tiles and 32-key steps of a wave
  static_assert(WK == 1 || WK == 2, "a wave takes whole 32-key steps");
  constexpr int ROWS = 16 * RB * WR;
  constexpr int KSTR = D + 8, VSTR = kTile + 8;  // LDS row strides (f16), padded against bank conflicts
  constexpr int NCH = kTile * D / 16 / 256;      // 16-code chunks of a tile per thread
  const Geom g = a.g;
  const int G = g.group(), H = g.n_kv;
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid / 64), lane = tid % 64;
  const int wr = wave % WR, wk = wave / WR;
  const int qn = lane % 16, jg = lane / 16;

  // ---- where the tails begin, for the decode kernel behind this one
  for (int64_t i = int64_t(blockIdx.x) * 256 + tid; i < int64_t(a.n_seqs) * a.tail_stride; i += int64_t(gridDim.x) * 256) {
    const int s = int(i / a.tail_stride), p = int(i % a.tail_stride), j = GroupOf(a, s);
    const int len = min(max(a.seq_len[s], 0), a.stride * PT), from = PrefixOf(a, j, len);
    a.tail_table[i] = a.table[int64_t(s) * a.stride + min(from / PT + p, a.stride - 1)];
    if (p == 0) a.tail_len[s] = min(len - from, a.max_tail);
  }

  // ---- this workgroup's rows and keys. Workgroups that read the same keys (the row blocks of a piece of a prefix) run on
  // one XCD, side by side.
  const int xcd = blockIdx.x % 8, local = blockIdx.x / 8;
  const int pair = xcd + 8 * (local / a.max_blocks), block = local % a.max_blocks;
  if (pair >= H * a.n_split) return;
  const int h = pair % H, piece = pair / H;
  int group = -1, row0 = 0;
  for (int j0 = 0, before = 0; j0 < a.n_groups; j0 += 64) {  // lane = group: which one row block `block` lies in
    const int j = j0 + lane;
    const int n = j < a.n_groups ? (max(GroupFirst(a, j + 1) - GroupFirst(a, j), 0) * G + ROWS - 1) / ROWS : 0;
    int incl = n;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int v = __shfl_up(incl, o, 64);
      if (lane >= o) incl += v;
    }
    const unsigned long long mine = __ballot(before + incl > block && before + incl - n <= block);
    if (mine != 0) {
      const int l = __builtin_ctzll(mine);
      group = j0 + l, row0 = (block - before - __shfl(incl - n, l, 64)) * ROWS;
      break;
    }
    before += __shfl(incl, 63, 64);
  }
  group = __builtin_amdgcn_readfirstlane(group), row0 = __builtin_amdgcn_readfirstlane(row0);
  if (group < 0) return;
  const int first = GroupFirst(a, group), n_rows = (GroupFirst(a, group + 1) - first) * G;
  const int shared = GroupShared(a, group), tiles = shared / kTile;
  const int per = TilesPerPiece(tiles, a.n_split);
  const int tile0 = piece * per, tile1 = min(tile0 + per, tiles);
  if (tile0 >= tile1) return;

  __shared__ __align__(16) _Float16 lk[kTile][KSTR];  // K tile, [key][dim]
  __shared__ __align__(16) _Float16 lv[D][VSTR];      // V^T tile, [dim][key]
  __shared__ __align__(16) _Float16 lvs[NB][kTile];   // V scales of the tile, [block][key]
  __shared__ int large_v;                             // some of them are above kLargeScale

  h8v qb[RB][KS];
  size_t prow[RB];  // (sequence, query head) of this lane's row in block i
  bool live[RB];    // it exists and its sequence is as long as the prefix
#pragma unroll
  for (int i = 0; i < RB; ++i) {
    const int r = row0 + (wr * RB + i) * 16 + qn, rr = min(r, n_rows - 1);
    const int s = first + rr / G;
    live[i] = r < n_rows && min(a.seq_len[s], a.stride * PT) >= shared;
    prow[i] = size_t(s) * g.n_q + size_t(h) * G + rr % G;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) qb[i][ks] = LoadQ8(a.q, prow[i] * D + 32 * ks + 8 * jg, a.q_dtype);
  }
  f4v o[RB][NDT], lacc[RB];
  float m[RB];
#pragma unroll
  for (int i = 0; i < RB; ++i) {
    m[i] = kNone, lacc[i] = f4v{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt) o[i][dt] = f4v{0.0f, 0.0f, 0.0f, 0.0f};
  }
  const float sscale = a.scale * 1.4426950408889634f;
  const int32_t* row = a.table + int64_t(first) * a.stride;
  auto page_head = [&](int key) -> size_t { return size_t(ClampPage(row[key / PT], g.n_pages)) * H + h; };

  uint4 kraw[NCH], vraw[NCH], vsr;
  uint16_t ksr[NCH];
  auto fetch_k = [&](int tile) {  // chunk c: block c / 128, key (c % 128) / 2, half c % 2
#pragma unroll
    for (int j = 0; j < NCH; ++j) {
      const int c = tid + 256 * j, b = c / 128, key = (c % 128) / 2, hf = c % 2, kk = tile * kTile + key;
      const size_t ph = page_head(kk);
      kraw[j] = FMT == 8 ? *reinterpret_cast<const uint4*>(a.pools.kq + ((ph * NB + b) * PT + kk % PT) * 32 + 16 * hf)
                         : *reinterpret_cast<const uint4*>(a.pools.kq + ((ph * NB + b) * PT + kk % PT) * 16);
      ksr[j] = a.pools.ks[(ph * PT + kk % PT) * NB + b];
    }
  };
  auto stage_k = [&](int j) {
    const int c = tid + 256 * j, b = c / 128, key = (c % 128) / 2, hf = c % 2;
    const _Float16 d = __builtin_bit_cast(_Float16, ksr[j]);
    const h8v d8 = {d, d, d, d, d, d, d, d};
    h8v lo, hi;
    Halves<FMT>(kraw[j], hf, &lo, &hi);
    if (__builtin_expect(__ballot(!(fabsf(static_cast<float>(d)) <= kLargeScale)) != 0, 0))
      lo = TimesSaturated(lo, d8), hi = TimesSaturated(hi, d8);
    else
      lo *= d8, hi *= d8;
    h8v* dst = reinterpret_cast<h8v*>(&lk[key][32 * b + 16 * hf]);
    dst[0] = lo, dst[1] = hi;
  };
  auto fetch_v = [&](int tile) {  // chunk c: dim c / 4, keys 16 (c % 4) .. + 15
#pragma unroll
    for (int j = 0; j < NCH; ++j) {
      const int c = tid + 256 * j, d = c / 4, kk = tile * kTile + 16 * (c % 4);
      const size_t ph = page_head(kk);
      vraw[j] = FMT == 8 ? *reinterpret_cast<const uint4*>(a.pools.vq + (ph * D + d) * PT + kk % PT)
                         : *reinterpret_cast<const uint4*>(a.pools.vq + ((ph * NB + d / 32) * 16 + d % 16) * PT + kk % PT);
    }
  };
  auto fetch_vs = [&](int tile) {  // thread = (block, 8 keys)
    if (tid < NB * 8) {
      const int b = tid / 8, kk = tile * kTile + 8 * (tid % 8);
      vsr = *reinterpret_cast<const uint4*>(a.pools.vs + (page_head(kk) * NB + b) * PT + kk % PT);
    }
  };
  auto stage_vs = [&]() {
    if (tid < 64) {  // (NB * 8 threads: one wave, or half of one)
      bool large = false;
      if (tid < NB * 8) {
        const h8v sc = __builtin_bit_cast(h8v, vsr);
#pragma unroll
        for (int e = 0; e < 8; ++e) large |= !(fabsf(static_cast<float>(sc[e])) <= kLargeScale);
        *reinterpret_cast<uint4*>(&lvs[tid / 8][8 * (tid % 8)]) = vsr;
      }
      const bool any = __ballot(large) != 0;
      if (tid == 0) large_v = any;
    }
  };
  auto stage_v = [&](int j) {
    const int c = tid + 256 * j, d = c / 4, k0 = 16 * (c % 4);
    const h8v s0 = *reinterpret_cast<const h8v*>(&lvs[d / 32][k0]), s1 = *reinterpret_cast<const h8v*>(&lvs[d / 32][k0 + 8]);
    h8v lo, hi;
    Halves<FMT>(vraw[j], d % 32 / 16, &lo, &hi);
    if (__builtin_expect(large_v != 0, 0)) lo = TimesSaturated(lo, s0), hi = TimesSaturated(hi, s1);
    else lo *= s0, hi *= s1;
    h8v* dst = reinterpret_cast<h8v*>(&lv[d][k0]);
    dst[0] = lo, dst[1] = hi;
  };

  // Pipeline: while the matrix cores run a tile's K Q^T out of lk, the vector units decode its V into lv; while they run
  // V^T P^T out of lv, the next tile's K is decoded into lk. Codes are fetched a tile before they are decoded.
  fetch_k(tile0);
  fetch_vs(tile0);
  fetch_v(tile0);
#pragma unroll
  for (int j = 0; j < NCH; ++j) stage_k(j);
  stage_vs();
  if (tile0 + 1 < tile1) fetch_k(tile0 + 1), fetch_vs(tile0 + 1);
  __syncthreads();
  for (int tile = tile0; tile < tile1; ++tile) {
    f4v st[RB][KT];
#pragma unroll
    for (int i = 0; i < RB; ++i)
#pragma unroll
      for (int kt = 0; kt < KT; ++kt) st[i][kt] = f4v{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      h8v ka[KT];
#pragma unroll
      for (int kt = 0; kt < KT; ++kt) ka[kt] = *reinterpret_cast<const h8v*>(&lk[16 * (wk * KT + kt) + qn][32 * ks + 8 * jg]);
#pragma unroll
      for (int kt = 0; kt < KT; ++kt)
#pragma unroll
        for (int i = 0; i < RB; ++i) st[i][kt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka[kt], qb[i][ks], st[i][kt], 0, 0, 0);
      if (ks % (KS / NCH) == KS / NCH - 1) stage_v(ks / (KS / NCH));
    }
    if (tile + 1 < tile1) fetch_v(tile + 1);
    h8v pv[RB][S2];
#pragma unroll
    for (int i = 0; i < RB; ++i) {
      float mx = kNegMax;
#pragma unroll
      for (int kt = 0; kt < KT; ++kt)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float v = st[i][kt][r] * sscale;
          st[i][kt][r] = v;
          mx = fmaxf(mx, v);
        }
      mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
      mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
      const float mn = fmaxf(m[i], __builtin_ceilf(mx) - kBias);  // whole numbers: rescaling is exact
      const float alpha = __builtin_amdgcn_exp2f(m[i] - mn);
      m[i] = mn;
      uint32_t w[S2][4];
#pragma unroll
      for (int kt = 0; kt < KT; ++kt) {
        _Float16 p[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) p[r] = static_cast<_Float16>(__builtin_amdgcn_exp2f(st[i][kt][r] - mn));
        // 32-key step kt / 2 takes keys 4 jg + r of its even 16-key tile, then of its odd one
        w[kt / 2][2 * (kt % 2)] = __builtin_bit_cast(uint32_t, h2v{p[0], p[1]});
        w[kt / 2][2 * (kt % 2) + 1] = __builtin_bit_cast(uint32_t, h2v{p[2], p[3]});
      }
#pragma unroll
      for (int s2 = 0; s2 < S2; ++s2) pv[i][s2] = __builtin_bit_cast(h8v, uint4{w[s2][0], w[s2][1], w[s2][2], w[s2][3]});
      if (__ballot(alpha != 1.0f) != 0) {
#pragma unroll
        for (int r = 0; r < 4; ++r) lacc[i][r] *= alpha;
#pragma unroll
        for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
          for (int r = 0; r < 4; ++r) o[i][dt][r] *= alpha;
      }
    }
    __syncthreads();  // every wave is done with lk, and the tile's V is complete in lv
    const h8v ones = __builtin_bit_cast(h8v, uint4{0x3C003C00u, 0x3C003C00u, 0x3C003C00u, 0x3C003C00u});
#pragma unroll
    for (int s2 = 0; s2 < S2; ++s2)
#pragma unroll
      for (int i = 0; i < RB; ++i) lacc[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ones, pv[i][s2], lacc[i], 0, 0, 0);
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt) {
#pragma unroll
      for (int s2 = 0; s2 < S2; ++s2) {
        const uint2 v0 = *reinterpret_cast<const uint2*>(&lv[16 * dt + qn][32 * (wk * S2 + s2) + 4 * jg]);
        const uint2 v1 = *reinterpret_cast<const uint2*>(&lv[16 * dt + qn][32 * (wk * S2 + s2) + 16 + 4 * jg]);
        const h8v va = __builtin_bit_cast(h8v, uint4{v0.x, v0.y, v1.x, v1.y});
#pragma unroll
        for (int i = 0; i < RB; ++i) o[i][dt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va, pv[i][s2], o[i][dt], 0, 0, 0);
      }
      if (tile + 1 < tile1 && dt % (NDT / NCH) == NDT / NCH - 1) stage_k(dt / (NDT / NCH));
    }
    stage_vs();  // (of the next tile, or once more the last one's)
    if (tile + 2 < tile1) fetch_k(tile + 2), fetch_vs(tile + 2);
    __syncthreads();  // every wave is done with lv; the next tile's K and V scales are in place
  }
#pragma unroll
  for (int i = 0; i < RB; ++i) {
    if (!live[i]) continue;
    const size_t at = prow[i] * a.slots + piece * WK + wk;
    if (jg == 0) *reinterpret_cast<float2*>(&a.ml[at * 2]) = float2{m[i], lacc[i][0]};
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt)
      *reinterpret_cast<float4*>(&a.acc[at * D + 16 * dt + 4 * jg]) = float4{o[i][dt][0], o[i][dt][1], o[i][dt][2], o[i][dt][3]};
  }
}

// One workgroup per (query head, sequence): the prefix's partials and the tail's, weighed by 2^(m - M) and 1 / l. A group of
// D / 4 lanes takes every n-th partial, four dims a lane; the groups' sums meet in LDS.
struct MergeArgs {
  SharedArgs s;
  DecodeArgs tail;
  int32_t waves_along_keys;
  const float* gate;
  void* out;
  int32_t out_dtype;
};
constexpr int kMergeThreads = 256;
__global__ __launch_bounds__(kMergeThreads) void SharedMerge(const MergeArgs a) {
  constexpr float kLog2e = 1.4426950408889634f;
  const Geom g = a.s.g;
  const int D = g.hd, G = g.group(), H = g.n_kv, hq = blockIdx.x, s = blockIdx.y, t = threadIdx.x, h = hq / G, gi = hq % G;
  const size_t row = size_t(s) * g.n_q + hq;
  // the prefix's pieces
  const int j = GroupOf(a.s, s);
  const int tiles = PrefixOf(a.s, j, min(max(a.s.seq_len[s], 0), a.s.stride * g.pt)) / kTile;
  const int per = max(TilesPerPiece(tiles, a.s.n_split), 1);
  const int n_pre = (tiles + per - 1) / per * a.waves_along_keys;
  // the places of the tail's partials (decode_cut.hpp)
  const DecodeArgs& d = a.tail;
  const int ts = TilesOf(d, s);
  size_t p0 = 0, p1 = 0;
  if (ts > 0) {
    const int Hc = CutHeads(d);
    const long long A = ChunkUnits(d, static_cast<long long>(d.tprefix[d.n_seqs]) * Hc);
    const long long first = static_cast<long long>(d.tprefix[s]) * Hc +
                            static_cast<long long>(Hc == 1 ? 0 : h) * UnitsOf(d, ts) + d.pair_cost;
    const int k0 = ChunkOf(d, A, first), k1 = ChunkOf(d, A, first + ts - 1);
    p0 = size_t(k0 + s * H + h) * d.wpc, p1 = size_t(k1 + s * H + h + 1) * d.wpc;
    if (Hc == 1 && H > 1) {
      const size_t r = size_t(h) * (d.n_chunks + d.n_seqs) + s;
      p0 = (r + k0) * d.wpc, p1 = (r + k1 + 1) * d.wpc;
    }
  }
  const int n = n_pre + static_cast<int>(p1 - p0);
  // partial i: reference point in base 2 and sum (0: nothing there, and its accumulator was not written)
  auto ml_of = [&](int i) -> float2 {
    if (i < n_pre) return *reinterpret_cast<const float2*>(&a.s.ml[(row * a.s.slots + i) * 2]);
    const float2 v = *reinterpret_cast<const float2*>(&d.ml[((p0 + (i - n_pre)) * G + gi) * 2]);
    return float2{v.x * kLog2e, v.y};
  };
  auto acc_of = [&](int i) -> const float* {
    return i < n_pre ? &a.s.acc[(row * a.s.slots + i) * D] : &d.acc[((p0 + (i - n_pre)) * G + gi) * D];
  };
  __shared__ float red[kMergeThreads / 64];
  __shared__ __align__(16) float sums[kMergeThreads * 4];
  __shared__ float lsum[kMergeThreads / 32];
  float M = kNegMax;
  for (int i = t; i < n; i += kMergeThreads) {
    const float2 v = ml_of(i);
    if (v.y > 0.0f) M = fmaxf(M, v.x);
  }
  M = WaveMax(M);
  if (t % 64 == 0) red[t / 64] = M;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kMergeThreads / 64; ++w) M = fmaxf(M, red[w]);
  const int lanes = D / 4, grp = t / lanes, dl = t % lanes, groups = kMergeThreads / lanes;
  float4 A = {0.0f, 0.0f, 0.0f, 0.0f};
  float L = 0.0f;
  for (int i = grp; i < n; i += groups) {
    const float2 v = ml_of(i);
    if (!(v.y > 0.0f)) {
      if (v.y != v.y) L = v.y;  // NaN queries or pools: the row is NaN, as in the decode attention
      continue;
    }
    const float w = __builtin_amdgcn_exp2f(v.x - M);
    const float4 x = *reinterpret_cast<const float4*>(acc_of(i) + 4 * dl);
    A.x = __builtin_fmaf(w, x.x, A.x), A.y = __builtin_fmaf(w, x.y, A.y);
    A.z = __builtin_fmaf(w, x.z, A.z), A.w = __builtin_fmaf(w, x.w, A.w);
    L = __builtin_fmaf(w, v.y, L);
  }
  *reinterpret_cast<float4*>(&sums[grp * D + 4 * dl]) = A;
  if (dl == 0) lsum[grp] = L;
  __syncthreads();
  for (int e = t; e < D; e += kMergeThreads) {
    float v = 0.0f, l = 0.0f;
    for (int q = 0; q < groups; ++q) v += sums[q * D + e], l += lsum[q];
    v = l == 0.0f ? 0.0f : v / l;  // (a sequence without keys)
    if (a.gate != nullptr) v *= 1.0f / (1.0f + __expf(-a.gate[row * D + e]));
    Store1(a.out, row * D + e, a.out_dtype, v);
  }
}

struct SharedPlan {
  int rows, waves_along_keys;  // query rows of a workgroup
  int32_t max_blocks, n_split, slots, tail_stride;
  size_t off_len, off_table, off_ml, off_acc, off_part, part_bytes, bytes;
};
SharedPlan MakeSharedPlan(const Geom& m, int32_t n_seqs, int32_t n_groups, int32_t max_shared, int32_t max_tail) {
  SharedPlan p;
  const int64_t rows = int64_t(n_seqs) * m.group();
  // A workgroup's rows follow the rows of an average group: fewer, and the tile's decode is paid more often; more, and
  // matrix rows go unused.
  const int64_t per_group = (rows + n_groups - 1) / n_groups;
  p.rows = per_group <= 32 ? 32 : per_group <= 64 ? 64 : 128;
  p.waves_along_keys = p.rows == 128 ? 1 : 2;
  p.max_blocks = static_cast<int32_t>(rows / p.rows + n_groups);
  const int64_t max_tiles = max_shared / kTile;
  const int64_t want = (2 * int64_t(ComputeUnits()) + int64_t(p.max_blocks) * m.n_kv - 1) / (int64_t(p.max_blocks) * m.n_kv);
  p.n_split = static_cast<int32_t>(std::max<int64_t>(1, std::min<int64_t>(want, (max_tiles + 3) / 4)));
  p.slots = max_tiles > 0 ? p.n_split * p.waves_along_keys : 0;
  p.tail_stride = (max_tail + m.pt - 1) / m.pt;
  const size_t parts = size_t(n_seqs) * m.n_q * p.slots;
  p.off_len = 0;
  p.off_table = Align(sizeof(int32_t) * size_t(n_seqs));
  p.off_ml = Align(p.off_table + sizeof(int32_t) * size_t(n_seqs) * p.tail_stride);
  p.off_acc = Align(p.off_ml + sizeof(float) * 2 * parts);
  p.off_part = Align(p.off_acc + sizeof(float) * parts * m.hd);
  p.part_bytes = MakePlan(m, n_seqs, max_tail, MakeTuning(nullptr)).bytes;
  p.bytes = p.off_part + p.part_bytes;
  return p;
}

template <int FMT, int D, int PT>
void LaunchShared(const SharedArgs& a, int rows, dim3 grid, hipStream_t st) {
  const dim3 block(64 * kSharedWaves);
  if (rows == 128) hipLaunchKernelGGL((SharedPart<FMT, D, PT, 2, 4>), grid, block, 0, st, a);
  else if (rows == 64) hipLaunchKernelGGL((SharedPart<FMT, D, PT, 2, 2>), grid, block, 0, st, a);
  else hipLaunchKernelGGL((SharedPart<FMT, D, PT, 1, 2>), grid, block, 0, st, a);
}
template <int FMT>
void LaunchSharedFormat(const SharedArgs& a, int rows, dim3 grid, hipStream_t st) {
  const Geom& m = a.g;
  if (m.hd == 256 && m.pt == 64) LaunchShared<FMT, 256, 64>(a, rows, grid, st);
  else if (m.hd == 256 && m.pt == 32) LaunchShared<FMT, 256, 32>(a, rows, grid, st);
  else if (m.hd == 256) LaunchShared<FMT, 256, 16>(a, rows, grid, st);
  else if (m.pt == 64) LaunchShared<FMT, 128, 64>(a, rows, grid, st);
  else if (m.pt == 32) LaunchShared<FMT, 128, 32>(a, rows, grid, st);
  else LaunchShared<FMT, 128, 16>(a, rows, grid, st);
}

int CheckSharedShape(const yahkv_geometry* g, int32_t n_seqs, int32_t n_groups, int32_t max_shared_len, int32_t max_tail_len) {
  if (const int st = CheckGeometry(g)) return st;
  if (n_seqs <= 0 || n_groups <= 0 || n_groups > n_seqs || max_shared_len < 0 || max_tail_len <= 0) return YAHKV_ERR_ARG;
  if (n_seqs > kMaxSeqs) return YAHKV_ERR_SHAPE;
  return YAHKV_OK;
}

}  // namespace
}  // namespace yahkv

using namespace yahkv;

extern "C" size_t yahkv_decode_shared_workspace_bytes(const yahkv_geometry* g, int32_t n_seqs, int32_t n_groups,
                                                      int32_t max_shared_len, int32_t max_tail_len) {
  if (CheckSharedShape(g, n_seqs, n_groups, max_shared_len, max_tail_len)) return 0;
  return MakeSharedPlan(MakeGeom(*g), n_seqs, n_groups, max_shared_len, max_tail_len).bytes;
}

extern "C" int yahkv_decode_attend_shared(const yahkv_geometry* g, const yahkv_pools* pools, const int32_t* page_table,
                                          int32_t page_table_stride, const int32_t* seq_len, int32_t n_seqs,
                                          const int32_t* group_first, const int32_t* shared_len, int32_t n_groups,
                                          int32_t max_shared_len, int32_t max_tail_len, const void* q, int32_t q_dtype,
                                          float softmax_scale, const float* gate, void* out, int32_t out_dtype,
                                          void* workspace, size_t workspace_bytes, void* stream) {
  if (const int st = CheckSharedShape(g, n_seqs, n_groups, max_shared_len, max_tail_len)) return st;
  if (const int st = CheckPools(g, pools)) return st;
  if (page_table == nullptr || seq_len == nullptr || group_first == nullptr || shared_len == nullptr || q == nullptr ||
      out == nullptr || workspace == nullptr || page_table_stride <= 0 || !(softmax_scale > 0.0f))
    return YAHKV_ERR_ARG;
  auto known = [](int32_t t) { return t == YAHKV_F32 || t == YAHKV_F16 || t == YAHKV_BF16; };
  if (!known(q_dtype) || !known(out_dtype)) return YAHKV_ERR_ARG;
  if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(workspace)) & 15)
    return YAHKV_ERR_ARG;
  const Geom m = MakeGeom(*g);
  if (int64_t(page_table_stride) * m.pt > 0x7FFFFFFF) return YAHKV_ERR_SHAPE;
  const SharedPlan p = MakeSharedPlan(m, n_seqs, n_groups, max_shared_len, max_tail_len);
  if (workspace_bytes < p.bytes) return YAHKV_ERR_WORKSPACE;
  const int64_t blocks = (int64_t(m.n_kv) * p.n_split + 7) / 8 * 8 * p.max_blocks;
  if (blocks > 0x7FFFFFFF) return YAHKV_ERR_SHAPE;
  char* ws = static_cast<char*>(workspace);
  SharedArgs a{};
  a.g = m, a.pools = MakePools(*pools), a.table = page_table, a.seq_len = seq_len, a.group_first = group_first;
  a.shared_len = shared_len, a.stride = page_table_stride, a.n_seqs = n_seqs, a.n_groups = n_groups;
  a.max_shared = max_shared_len, a.max_tail = max_tail_len, a.q = q, a.q_dtype = q_dtype, a.scale = softmax_scale;
  a.max_blocks = p.max_blocks, a.n_split = p.n_split, a.slots = p.slots, a.tail_stride = p.tail_stride;
  a.tail_len = reinterpret_cast<int32_t*>(ws + p.off_len), a.tail_table = reinterpret_cast<int32_t*>(ws + p.off_table);
  a.ml = reinterpret_cast<float*>(ws + p.off_ml), a.acc = reinterpret_cast<float*>(ws + p.off_acc);
  hipStream_t st = static_cast<hipStream_t>(stream);
  MergeArgs ma{};
  if (const int rc = Prepare(m, p.tail_stride, a.tail_len, n_seqs, max_tail_len, ws + p.off_part, p.part_bytes, nullptr, &ma.tail)) return rc;
  const dim3 grid(static_cast<unsigned>(blocks));
  if (m.format == YAHKV_Q8_0) LaunchSharedFormat<8>(a, p.rows, grid, st);
  else LaunchSharedFormat<4>(a, p.rows, grid, st);
  if (const int rc = LaunchStatus()) return rc;
  if (const int rc = yahkv_decode_part(g, pools, a.tail_table, p.tail_stride, a.tail_len, n_seqs, max_tail_len, q, q_dtype,
                                       softmax_scale, ws + p.off_part, p.part_bytes, nullptr, stream))
    return rc;
  ma.s = a, ma.waves_along_keys = p.waves_along_keys, ma.gate = gate, ma.out = out, ma.out_dtype = out_dtype;
  hipLaunchKernelGGL(SharedMerge, dim3(static_cast<unsigned>(m.n_q), static_cast<unsigned>(n_seqs)), dim3(kMergeThreads), 0, st, ma);
  return LaunchStatus();
}
