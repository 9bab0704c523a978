// Decode attention of a batch whose sequences share prefixes: each prefix's keys are read and decoded once for all the
// query rows that see them.
//
// Attention splits over any partition of the keys: with m a reference point, l = sum 2^(s_t - m) and o = sum 2^(s_t - m)
// V_t of each part, the whole is (sum 2^(m_p - M) o_p) / (sum 2^(m_p - M) l_p). The prefix's part of a group's rows is a
// matrix product with many rows (sequences x query heads of a kv head); the tails have one sequence's query heads each.
// `SharedPart` leaves partials of both, in one launch or (tails that fill the chip by themselves) two, `SharedMerge` puts
// them together.
//
// SharedPart: a wave takes 16 RB query rows and 64-key tiles, everything transposed (keys along MFMA rows, query rows along
// lanes), and works alone: codes go from memory to its registers, are decoded there and feed the products directly.
//   S^T[key][row] = sum_dim K[key][dim] Q[row][dim]       A = 16 keys x 32 dims, B = Q^T (registers)
//   O^T[dim][row] += sum_key V^T[dim][key] P^T[key][row]  A = 16 dims x 32 keys, B = P^T (registers)
// The order of the contraction index is free as long as both operands agree, and so is which key a row of S^T is, so
// every operand is what a 16-byte load brings: a lane's K load is half a block of one key (q4_0: a block), its V load 16
// keys of one dim (q4_0: of two). Row i of key tile kt is key 16 (i / 4) + 4 kt + i % 4: then the scores that lane group jg
// holds after the four key tiles are those of keys 16 jg .. 16 jg + 15, the ones its V load has. P never leaves its lane.
// A register is asked for again (for the wave's next tile) as soon as its codes are decoded, so a load has about a tile's
// time to arrive, without a barrier anywhere in the loop. (Not with 16-token pages: a tile's four page numbers, picked by
// lane, lie in scratch memory there, and the waits for them are waits for every load that is out, two or three times a
// tile.) Decoding is packed f16 arithmetic, perm, add, multiply for two
// values, the product d * code rounded once; beyond the f16 range V's saturates (Saturates), K's takes a power of two
// (ShrinkLargeKeys).
// Roundings to f16 (11 bits): queries given as f32, K, V and the numerators, each once; products and sums are f32. With scores
// of a standard deviation of two K's costs 3.5e-4 of the output's norm, the numerators' 2.0e-4, V's 1.6e-4 (an f16 output's own
// is 2.1e-4). Exact K codes with their scales on the sums, as yahkv_decode_attend has them, were built: the error of an f32
// output falls from 4.9e-4 to 2.8e-4 (yahkv_decode_attend: 2.2e-4) and 64 sequences on 32K take 146 us instead of 122, 32 on 8K 44
// instead of 39, 45 in 3 groups 31.5 instead of 28.5: four multiply-adds a row block for every four multiplications saved, on
// sums that the matrix unit leaves in the other half of the register file.
//
// What bounds it: with few rows the reads and a workgroup's beginning and end (12 query rows on 32K keys of 4 x 256 dims: 23
// us, 71 MB); with three row blocks of 256 dims the vector unit, which issues 1520 instructions of 4 cycles for a tile's 192
// matrix instructions of 16 and is busy with 900 of them decoding (384 rows x 32K keys: 98 us, 0.53 PFLOP/s, 4.5 us a tile of
// each wave, of which a matrix product at this card's rate would take 2.7). Three row blocks are what fits: accumulators 192
// registers, queries 96, codes 64, scores 48. Decoding once for four waves of other rows, through LDS, brings a tile to 3.2 us, but
// then no two waves share rows, and writing four times the partials and reading them again takes all of it back.
#include "codes.hpp"
#include "common.hpp"
#include "decode_cut.hpp"
#include "quant.hpp"
#include "store.hpp"

namespace yahkv {
namespace {

constexpr int kSharedWaves = 4;
constexpr float kNone = kNegMax;  // reference point of a row before its first tile
// Numerators are 2^(score - m). m is a whole number, so that moving it rescales exactly, kBias below the largest score when
// it was set, and is moved when a score exceeds it by kBias + kSlack: numerators stay within f16's range and those
// 2^-24 of the largest are still normal numbers.
constexpr float kBias = 10.0f, kSlack = 4.0f;
// Scores are rounded before m is subtracted (an unrounded product, as in a multiply-add, is half a unit of the last place off
// the largest score: 32 at 2^30, far past f16's range), and where they are beyond kFar m is the largest score itself (from 2^27
// on ten below it need not be a float).
constexpr float kFar = 0x1p20f;

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
  int32_t max_blocks;           // row blocks of all groups at most
  int32_t n_split, tail_split;  // pieces a prefix / a tail is cut into
  int32_t prefix_groups;        // workgroups of the prefixes; those of the tails follow
  // workspace, [n_seqs][n_q][n_split + tail_split]: reference point (base 2) and sum, accumulator [D]
  float* ml;
  float* acc;
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
// What a sequence takes from its group's prefix, all the whole tiles, and from its own row behind them. A sequence that is
// shorter than those tiles takes none: it is all tail. So every row of a prefix sees every key, nothing is masked there, and
// whatever a prefix holds that a shorter sequence must not see (an infinity would pass through a zero numerator as NaN)
// stays out of that sequence's sums.
struct Keys {
  int prefix, tail;
};
__device__ __forceinline__ Keys KeysOf(const SharedArgs& a, int s) {
  const int len = min(max(a.seq_len[s], 0), a.stride * a.g.pt), j = GroupOf(a, s);
  const int shared = j < 0 ? 0 : GroupShared(a, j), prefix = len < shared ? 0 : shared;
  return Keys{prefix, min(len - prefix, a.max_tail)};
}
// `tiles` cut into at most n pieces (0 where the host allows no prefix): tiles per piece
__device__ __forceinline__ int PerPiece(int tiles, int n) { return max((tiles + n - 1) / max(n, 1), 1); }

// Maximum and sum over the four lane groups of a wave (lanes n, n + 16, n + 32, n + 48), in every lane.
template <typename Op>
__device__ __forceinline__ float OverLaneGroups(float v, Op op) {
  const uint32_t u = __builtin_bit_cast(uint32_t, v);
  const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  const uint32_t r0 = r[0], r1 = r[1];
  const float w = op(__builtin_bit_cast(float, r0), __builtin_bit_cast(float, r1));
  const uint32_t x = __builtin_bit_cast(uint32_t, w);
  const auto q = __builtin_amdgcn_permlane32_swap(x, x, false, false);
  const uint32_t q0 = q[0], q1 = q[1];
  return op(__builtin_bit_cast(float, q0), __builtin_bit_cast(float, q1));
}

// Products d * code pass the f16 range where a scale is above 511.75 (128 x 511.75 is the largest f16).
constexpr uint32_t kLargeScale = 0x5FFF;
typedef uint16_t us2v __attribute__((ext_vector_type(2)));
// The larger magnitudes of two pairs of f16 values, as bits.
__device__ __forceinline__ us2v Magnitudes(uint32_t a, uint32_t b) {
  return __builtin_elementwise_max(__builtin_bit_cast(us2v, a & 0x7FFF7FFFu), __builtin_bit_cast(us2v, b & 0x7FFF7FFFu));
}
__device__ __forceinline__ uint32_t Larger(us2v x) { return x[0] > x[1] ? x[0] : x[1]; }

// V's saturate. MODE.FP16_OVFL (bit 23) does that in the multiply for nothing, but while it is set the matrix unit drops NaN
// operands: it is set for the second product alone (a NaN among the numerators is in their sum as well, a NaN score
// would be lost), and only for tiles that need it, those with a large scale and none that is not finite. v: the tile's
// scales, eight a lane. Returns whether it is such a tile.
__device__ __forceinline__ bool Saturates(const uint4 v) {
  const uint32_t most = Larger(__builtin_elementwise_max(Magnitudes(v.x, v.y), Magnitudes(v.z, v.w)));
  return __builtin_amdgcn_ballot_w64(most > kLargeScale) != 0 && __builtin_amdgcn_ballot_w64(most >= 0x7C00u) == 0;
}
__device__ __forceinline__ void SetSaturation(bool on) {
  __builtin_amdgcn_sched_barrier(0);
  if (on) __builtin_amdgcn_s_setreg((0 << 11) | (23 << 6) | 1, 1);
  else __builtin_amdgcn_s_setreg((0 << 11) | (23 << 6) | 1, 0);
  __builtin_amdgcn_sched_barrier(0);
}

// K's do not: a saturated product would be another score, and an infinite one a NaN. A tile with a large scale enters the
// product with all its scales times 2^-7, and its scores are multiplied by 2^7 behind it. That is exact but for scales below
// 2^-7, those of ordinary keys in such a tile, which become whole multiples of 2^-24: 2^-18 off at most, which is to keys of
// values about one what f16's rounding of them is. k: the tile's scales, eight a lane (0 for keys behind the end, so that what
// they hold has no say in it). Returns whether it is such a tile.
__device__ __forceinline__ bool ShrinkLargeKeys(uint4& k) {
  const uint32_t most = Larger(__builtin_elementwise_max(Magnitudes(k.x, k.y), Magnitudes(k.z, k.w)));
  if (__builtin_expect(__builtin_amdgcn_ballot_w64(most > kLargeScale) == 0, 1)) return false;
  const _Float16 s = static_cast<_Float16>(0x1p-7f);
  k = __builtin_bit_cast(uint4, __builtin_bit_cast(h8v, k) * h8v{s, s, s, s, s, s, s, s});
  return true;
}

// A barrier behind LDS accesses alone: __syncthreads() would wait for the loads on their way in as well.
__device__ __forceinline__ void LdsBarrier() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0)
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

template <int D>
struct WaveScales {  // a tile's scales in LDS, [key][block] and [block][key]
  _Float16 k[kTile * D / 32], v[D / 32 * kTile];
};

// A workgroup's query rows on their way to LDS, as f16: asked for first, converted when the first tile's loads are out too.
// (Converted by every wave for its own operands, in all three types of the source, they were half of the kernel's code; a
// workgroup runs most of its code once or a few times, and fetching it was what a small call waited for.)
template <int D, int RB>
struct QueryRows {
  static constexpr int ROWS = 16 * RB, STR = D + 8, PER = ROWS * (D / 8) / (64 * kSharedWaves);
  _Float16 (*lds)[STR];
  RawQ8 raw[PER];
  template <typename RowOf>
  __device__ __forceinline__ void Request(const void* q, int dtype, RowOf row_of) {
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      const int u = threadIdx.x + 64 * kSharedWaves * j;
      raw[j] = LoadRawQ8(q, row_of(u / (D / 8)) * D + u % (D / 8) * 8, dtype);
    }
  }
  __device__ __forceinline__ void Stage(int dtype) {
    auto put = [&](int j, h8v v) {
      const int u = threadIdx.x + 64 * kSharedWaves * j;
      *reinterpret_cast<h8v*>(&lds[u / (D / 8)][u % (D / 8) * 8]) = v;
    };
    if (dtype == YAHKV_F16) {
#pragma unroll
      for (int j = 0; j < PER; ++j) put(j, __builtin_bit_cast(h8v, raw[j].a));
    } else if (dtype == YAHKV_BF16) {
#pragma unroll
      for (int j = 0; j < PER; ++j) put(j, ConvertQ8(raw[j], YAHKV_BF16));
    } else {
#pragma unroll
      for (int j = 0; j < PER; ++j) put(j, ConvertQ8(raw[j], YAHKV_F32));
    }
    LdsBarrier();
  }
  __device__ __forceinline__ h8v At(int row, int d) const { return *reinterpret_cast<const h8v*>(&lds[row][d]); }
};

// Numerators of one row block's tile: this lane's 16 keys 16 jg + 4 kt + r of its row, scores st in, second operand pv out.
template <int D>
__device__ __forceinline__ void Numerators(const f4v (&st)[4], float sscale, float& m, float& l, f4v (&o)[D / 16], h8v (&pv)[2]) {
#pragma clang fp contract(off)
  constexpr int NDT = D / 16;
  float mx = fmaxf(st[0][0], st[0][1]);
  mx = fmaxf(fmaxf(mx, st[0][2]), st[0][3]);
#pragma unroll
  for (int kt = 1; kt < 4; ++kt) mx = fmaxf(fmaxf(mx, st[kt][0]), st[kt][1]), mx = fmaxf(fmaxf(mx, st[kt][2]), st[kt][3]);
  mx = OverLaneGroups(mx, [](float x, float y) { return fmaxf(x, y); }) * sscale;
  if (__builtin_expect(__builtin_amdgcn_ballot_w64(mx - m > kBias + kSlack) != 0, 0)) {
    const float mn = mx - m > kBias + kSlack ? __builtin_ceilf(mx) - (fabsf(mx) > kFar ? 0.0f : kBias) : m;
    const float alpha = __builtin_amdgcn_exp2f(m - mn);
    m = mn, l *= alpha;
    // (the rescaled accumulators go back through a matrix instruction with zero factors: that keeps them in the
    // accumulation registers on this path as on the common one)
    const h8v zero = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt) {
      f4v x = o[dt];
      asm volatile("" : "+a"(x));
#pragma unroll
      for (int r = 0; r < 4; ++r) x[r] *= alpha;
      o[dt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(zero, zero, x, 0, 0, 0);
    }
  }
  const h2v one = {static_cast<_Float16>(1.0f), static_cast<_Float16>(1.0f)};
  uint32_t w[2][4];
#pragma unroll
  for (int kt = 0; kt < 4; ++kt) {
    float p[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) p[r] = __builtin_amdgcn_exp2f(st[kt][r] * sscale - m);
    const h2v p0 = {static_cast<_Float16>(p[0]), static_cast<_Float16>(p[1])};
    const h2v p1 = {static_cast<_Float16>(p[2]), static_cast<_Float16>(p[3])};
    // (the sum is of the rounded numerators, as the second product's is)
    l = __builtin_amdgcn_fdot2(p0, one, l, false), l = __builtin_amdgcn_fdot2(p1, one, l, false);
    w[kt / 2][2 * (kt % 2)] = __builtin_bit_cast(uint32_t, p0), w[kt / 2][2 * (kt % 2) + 1] = __builtin_bit_cast(uint32_t, p1);
  }
#pragma unroll
  for (int s = 0; s < 2; ++s) pv[s] = __builtin_bit_cast(h8v, uint4{w[s][0], w[s][1], w[s][2], w[s][3]});
}

// Tiles tile0, tile0 + step, .. below tile1 of the sequence behind table row `row`, from key `origin` on, `n_keys` keys in
// all (those at or past it are masked), against RB row blocks: reference points, this lane's part of the sums, accumulators.
// All four waves of the workgroup call it together (the queries go through LDS behind one barrier); a wave without a tile
// loads one all the same.
template <int FMT, int D, int PT, int RB, bool TWO>
__device__ __forceinline__ void StreamKeys(const SharedArgs& a, const int32_t* row, int origin, int h, int tile0, int step,
                                           int tile1, int n_keys, QueryRows<D, RB>& queries, WaveScales<D>& lds, float (&m)[RB],
                                           float (&l)[RB], f4v (&o)[RB][D / 16]) {
  constexpr int NB = D / 32, NDT = D / 16, KS = D / 32, PPT = kTile / PT;
  constexpr bool Q8 = FMT == 8;
  constexpr int NP = Q8 ? KS / 2 : NB / 4;  // K loads per key tile
  constexpr int SP = KS / NP;               // steps of the first product per K load
  constexpr int NV = Q8 ? NDT : NB;         // V loads
  const Geom& g = a.g;
  const int H = g.n_kv, lane = threadIdx.x % 64, qn = lane % 16, jg = lane / 16;
  const float sscale = a.scale * 1.4426950408889634f;

  // pages of a tile, through the constant address space (scalar loads, which the vector memory counter does not see)
  typedef const int32_t __attribute__((address_space(4))) * ConstRow;
  const ConstRow crow = (ConstRow)(reinterpret_cast<uintptr_t>(row + origin / PT));
  const int last_page = a.stride - 1 - origin / PT;
  auto load_pages = [&](int tile, int (&pg)[PPT]) {
#pragma unroll
    for (int j = 0; j < PPT; ++j) pg[j] = ClampPage(crow[min(tile * PPT + j, last_page)], g.n_pages);
  };
  auto page_head = [&](const int (&pg)[PPT], int key) -> size_t {  // (page, kv head) of a key of the tile
    int p = pg[0];
#pragma unroll
    for (int j = 1; j < PPT; ++j) p = key / PT == j ? pg[j] : p;
    return size_t(p) * H + h;
  };
  // Codes on their way in: a tile's K loads, then its V loads, then the next tile's, `kDepth` of them at a time. As soon as
  // the codes of one are decoded its register is asked for the one kDepth later. (Eight where 256 registers have to do for
  // accumulators of 256 dims a row block: 32K keys x 12 rows 23 us with two workgroups a CU, 31 with one and 32 loads.)
  constexpr int NK = 4 * NP, NL = NK + NV, kMost = TWO && Q8 && RB * D == 256 ? 8 : 16, kDepth = NL < kMost ? NL : kMost;
  static_assert(NL % kDepth == 0, "the same registers in every tile");
  uint4 codes[kDepth], ksr, vsr;
  constexpr uint32_t KB = Q8 ? 32 : 16;
  // Where a tile is one page, through a buffer resource of the (page, kv head) region: scalar base and offsets, one lane
  // offset for all loads.
  auto read = [&](const uint8_t* base, uint32_t lane_off, uint32_t off) -> uint4 {
    if constexpr (PPT == 1) {
      const auto rs = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(base), 0, 0x7fffffff, 0x00020000);
      return __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(rs, lane_off, off, 0));
    } else {
      return *reinterpret_cast<const uint4*>(base + lane_off + off);
    }
  };
  const int key0 = 16 * (qn / 4) + qn % 4;  // this lane's key of key tile 0
  const uint32_t k_off = ((Q8 ? jg >> 1 : jg) * PT + key0 % PT) * KB + (Q8 ? 16 * (jg & 1) : 0);
  const uint32_t v_off = qn * PT + 16 * jg % PT;
  auto load_k = [&](const int (&pg)[PPT], int j) {  // load j = NP kt + p (the four key tiles of a lane lie in one page)
    codes[j % kDepth] = read(a.pools.kq + page_head(pg, key0) * (NB * PT * KB), k_off, (j % NP * (Q8 ? 2 : 4) * PT + 4 * (j / NP)) * KB);
  };
  auto load_v = [&](const int (&pg)[PPT], int j) {  // q8_0: dim 16 j + qn; q4_0: byte row qn of block j
    codes[(NK + j) % kDepth] = read(a.pools.vq + page_head(pg, 16 * jg) * (Q8 ? D * PT : NB * 16 * PT), v_off, 16 * j * PT);
  };
  auto load_scales = [&](const int (&pg)[PPT]) {  // lane: 8 K scales of the tile in [key][block] order, 8 V scales in [block][key]
    ksr = vsr = uint4{0u, 0u, 0u, 0u};
    if (lane < NB * 8) {
      const int key = lane * 8 / NB, chunk = lane % 8;
      ksr = *reinterpret_cast<const uint4*>(a.pools.ks + (page_head(pg, key) * PT + key % PT) * NB + lane * 8 % NB);
      vsr = *reinterpret_cast<const uint4*>(a.pools.vs + (page_head(pg, 8 * chunk) * NB + lane / 8) * PT + 8 * chunk % PT);
    }
  };

  int pgc[PPT], pgn[PPT];
  auto load = [&](int j) {  // load j of the tile of pgc, and on into that of pgn
    if (j < NK) load_k(pgc, j);
    else if (j < NL) load_v(pgc, j - NK);
    else if (j < NL + NK) load_k(pgn, j - NL);
    else load_v(pgn, j - NL - NK);
  };
  load_pages(tile0, pgn);
  load_scales(pgn);
#pragma unroll
  for (int j = 0; j < kDepth; ++j) load(NL + j);
  // the queries, which were asked for before all this: through LDS into the first product's operands
  queries.Stage(a.q_dtype);
  h8v qb[RB][KS];
#pragma unroll
  for (int i = 0; i < RB; ++i) {
    m[i] = kNone, l[i] = 0.0f;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {  // the dims of step (p, sub) that this lane group holds
      const int p = ks / SP, sub = ks % SP;
      qb[i][ks] = queries.At(16 * i + qn, Q8 ? 32 * (2 * p + (jg >> 1)) + 16 * (jg & 1) + 8 * sub
                                             : 32 * (4 * p + jg) + 8 * (sub & 1) + 16 * (sub >> 1));
    }
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt) o[i][dt] = f4v{0.0f, 0.0f, 0.0f, 0.0f};
  }
  for (int tile = tile0; tile < tile1; tile += step) {
    // (the last tile's successor is itself: every pass issues the same loads, which keeps the waits exact where a tile has at
    // most two pages)
#pragma unroll
    for (int j = 0; j < PPT; ++j) pgc[j] = pgn[j];
    load_pages(tile + step < tile1 ? tile + step : tile, pgn);
    const bool cut = (tile + 1) * kTile > n_keys;
    bool saturates;
    int up = 0;  // this tile's scores come times 2^-up
    {  // scales to LDS; those of masked keys become 0, which makes their V rows 0 whatever they hold
      uint32_t w[4] = {vsr.x, vsr.y, vsr.z, vsr.w};
      if (cut) {
        const int k0 = tile * kTile + 8 * (lane % 8);
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (k0 + e >= n_keys) w[e / 2] &= e % 2 ? 0x0000FFFFu : 0xFFFF0000u;
        const int key = tile * kTile + lane * 8 / NB;  // K's: a lane has all of a key, or of two
        if (key >= n_keys) ksr.x = ksr.y = 0u;
        if (key + (NB == 4 ? 1 : 0) >= n_keys) ksr.z = ksr.w = 0u;
      }
      if (ShrinkLargeKeys(ksr)) up = 7;
      if (lane < NB * 8) {
        *reinterpret_cast<uint4*>(&lds.k[lane * 8]) = ksr;
        *reinterpret_cast<uint4*>(&lds.v[lane * 8]) = uint4{w[0], w[1], w[2], w[3]};
      }
      saturates = Saturates(uint4{w[0], w[1], w[2], w[3]});
    }
    load_scales(pgn);
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    // ---- S^T
    f4v st[RB][4];
#pragma unroll
    for (int kt = 0; kt < 4; ++kt) {
      const int key = 16 * (qn / 4) + 4 * kt + qn % 4;
#pragma unroll
      for (int i = 0; i < RB; ++i) st[i][kt] = f4v{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int p = 0; p < NP; ++p) {
        const _Float16 d = lds.k[key * NB + (Q8 ? 2 * p + (jg >> 1) : 4 * p + jg)];
        const h8v d8 = {d, d, d, d, d, d, d, d};
        const uint4 c = codes[(NP * kt + p) % kDepth];
        h8v ka[SP];
        if constexpr (Q8) {
          ka[0] = Codes8(c.x, c.y), ka[1] = Codes8(c.z, c.w);
        } else {
          ka[0] = NibblesLo8(c.x, c.y), ka[1] = NibblesLo8(c.z, c.w), ka[2] = NibblesHi8(c.x, c.y), ka[3] = NibblesHi8(c.z, c.w);
        }
        load(NP * kt + p + kDepth);
#pragma unroll
        for (int sub = 0; sub < SP; ++sub) {
          ka[sub] *= d8;
#pragma unroll
          for (int i = 0; i < RB; ++i)
            st[i][kt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka[sub], qb[i][p * SP + sub], st[i][kt], 0, 0, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    asm volatile("" : "+s"(up));  // (a whole number in a scalar register till here: the scale itself would take a vector register)
    const float tscale = __builtin_ldexpf(sscale, up);
    h8v pv[RB][2];
#pragma unroll
    for (int i = 0; i < RB; ++i) {
      if (cut) {
#pragma unroll
        for (int kt = 0; kt < 4; ++kt)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (tile * kTile + 16 * jg + 4 * kt + r >= n_keys) st[i][kt][r] = -__builtin_inff();
      }
      Numerators<D>(st[i], tscale, m[i], l[i], o[i], pv[i]);
    }
    // ---- O^T
    if (__builtin_expect(saturates, 0)) SetSaturation(true);
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      const h8v s0 = *reinterpret_cast<const h8v*>(&lds.v[b * kTile + 16 * jg]);
      const h8v s1 = *reinterpret_cast<const h8v*>(&lds.v[b * kTile + 16 * jg + 8]);
#pragma unroll
      for (int e = 0; e < 2; ++e) {  // dims 32 b + 16 e + 0..15
        const int dt = 2 * b + e;
        const uint4 c = codes[(NK + (Q8 ? dt : b)) % kDepth];
        h8v v0, v1;
        if constexpr (Q8) v0 = Codes8(c.x, c.y), v1 = Codes8(c.z, c.w);
        else if (e == 0) v0 = NibblesLo8(c.x, c.y), v1 = NibblesLo8(c.z, c.w);
        else v0 = NibblesHi8(c.x, c.y), v1 = NibblesHi8(c.z, c.w);
        if (Q8 || e == 1) load(NK + (Q8 ? dt : b) + kDepth);
        v0 *= s0, v1 *= s1;
#pragma unroll
        for (int i = 0; i < RB; ++i) o[i][dt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v0, pv[i][0], o[i][dt], 0, 0, 0);
#pragma unroll
        for (int i = 0; i < RB; ++i) o[i][dt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v1, pv[i][1], o[i][dt], 0, 0, 0);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    if (__builtin_expect(saturates, 0)) SetSaturation(false);
    __builtin_amdgcn_wave_barrier();  // (the scales in LDS are rewritten for the next tile)
  }
}

constexpr int kRoundDims = 128;  // dims of a row that the waves' shares meet in LDS with at a time
template <int D, int RB>
struct SharedLds {
  static constexpr int ROWS = 16 * RB, STR = kRoundDims + 4;
  WaveScales<D> scales[kSharedWaves];
  float m[kSharedWaves][ROWS], l[kSharedWaves][ROWS];
  union {
    _Float16 q[ROWS][D + 8];  // until every wave has its operands
    float sums[kSharedWaves][ROWS][STR];  // (MergeWaves writes it behind a barrier)
  };
};

// The four waves' shares of the same rows become one partial in slot `slot` of every live row.
template <int D, int RB, typename RowOf>
__device__ __forceinline__ void MergeWaves(const SharedArgs& a, SharedLds<D, RB>& lds, const float (&m)[RB], float (&l)[RB],
                                           f4v (&o)[RB][D / 16], int n_rows, RowOf row_of, int slot) {
  constexpr int ROWS = 16 * RB;
  const int tid = threadIdx.x, wave = tid / 64, lane = tid % 64, qn = lane % 16, jg = lane / 16;
  const int slots = a.n_split + a.tail_split;
#pragma unroll
  for (int i = 0; i < RB; ++i) {
    l[i] = OverLaneGroups(l[i], [](float x, float y) { return x + y; });
    if (jg == 0) lds.m[wave][16 * i + qn] = m[i], lds.l[wave][16 * i + qn] = l[i];
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < RB; ++i) {
    float M = kNone;
#pragma unroll
    for (int w = 0; w < kSharedWaves; ++w) M = fmaxf(M, lds.m[w][16 * i + qn]);
    const float f = __builtin_amdgcn_exp2f(m[i] - M);
#pragma unroll
    for (int dt = 0; dt < D / 16; ++dt)
#pragma unroll
      for (int r = 0; r < 4; ++r) o[i][dt][r] *= f;
  }
  if (tid < ROWS && tid < n_rows) {
    float M = kNone, L = 0.0f;
#pragma unroll
    for (int w = 0; w < kSharedWaves; ++w) M = fmaxf(M, lds.m[w][tid]);
#pragma unroll
    for (int w = 0; w < kSharedWaves; ++w) L = __builtin_fmaf(lds.l[w][tid], __builtin_amdgcn_exp2f(lds.m[w][tid] - M), L);
    *reinterpret_cast<float2*>(&a.ml[(row_of(tid) * slots + slot) * 2]) = float2{M, L};
  }
#pragma unroll
  for (int c = 0; c < D / kRoundDims; ++c) {
    if (c > 0) __syncthreads();
#pragma unroll
    for (int i = 0; i < RB; ++i)
#pragma unroll
      for (int e = 0; e < kRoundDims / 16; ++e) {
        const f4v x = o[i][c * (kRoundDims / 16) + e];
        *reinterpret_cast<float4*>(&lds.sums[wave][16 * i + qn][16 * e + 4 * jg]) = float4{x[0], x[1], x[2], x[3]};
      }
    __syncthreads();
    for (int u = tid; u < min(ROWS, n_rows) * (kRoundDims / 4); u += 64 * kSharedWaves) {
      const int r = u / (kRoundDims / 4), d = u % (kRoundDims / 4) * 4;
      float4 v = *reinterpret_cast<const float4*>(&lds.sums[0][r][d]);
#pragma unroll
      for (int w = 1; w < kSharedWaves; ++w) {
        const float4 x = *reinterpret_cast<const float4*>(&lds.sums[w][r][d]);
        v.x += x.x, v.y += x.y, v.z += x.z, v.w += x.w;
      }
      *reinterpret_cast<float4*>(&a.acc[(row_of(r) * slots + slot) * D + c * kRoundDims + d]) = v;
    }
  }
}

// A piece of a prefix against a block of ROWS of its group's rows, by workgroup. Those that read the same keys (the row
// blocks of a piece) run on one XCD, side by side.
struct PrefixPiece {
  // group -1: nothing; n_rows: rows from row0 on. The pages are read through the row of sequence `reader`, the group's first
  // one that takes the prefix (KeysOf): the row of a shorter one, an idle slot's above all, need not name them.
  int group, h, piece, first, reader, row0, n_rows, tile0, tile1;
  __device__ __forceinline__ size_t Row(const SharedArgs& a, int r) const {  // row r of the block among all (sequence, query head) rows
    const int G = a.g.group(), rr = row0 + min(r, n_rows - 1);
    return (size_t(first) + rr / G) * a.g.n_q + size_t(h) * G + rr % G;
  }
};
template <int ROWS>
__device__ __forceinline__ PrefixPiece FindPiece(const SharedArgs& a) {
  const int G = a.g.group(), H = a.g.n_kv, lane = threadIdx.x % 64;
  const int xcd = blockIdx.x % 8, local = blockIdx.x / 8;
  const int pair = xcd + 8 * (local / a.max_blocks), block = local % a.max_blocks;
  PrefixPiece p{-1, pair % H, pair / H, 0, 0, 0, 0, 0, 0};
  if (pair >= H * a.n_split) return p;
  int tiles = 0, n_seqs = 0, first_len = 0;
  for (int j0 = 0, before = 0; j0 < a.n_groups; j0 += 64) {  // lane = group: which one row block `block` lies in
    const int j = min(j0 + lane, a.n_groups - 1);
    const int first = GroupFirst(a, j), rows = j0 + lane < a.n_groups ? max(GroupFirst(a, j + 1) - first, 0) * G : 0;
    const int shared = GroupShared(a, j), n = (rows + ROWS - 1) / ROWS, len = a.seq_len[min(first, a.n_seqs - 1)];
    int incl = n;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int v = __shfl_up(incl, o, 64);
      if (lane >= o) incl += v;
    }
    const unsigned long long mine = __ballot(before + incl > block && before + incl - n <= block);
    if (mine != 0) {
      const int at = __builtin_ctzll(mine);
      auto its = [&](int v) { return __builtin_amdgcn_readlane(v, at); };
      p.group = j0 + at, p.row0 = (block - before - its(incl - n)) * ROWS;
      p.first = its(first), n_seqs = its(rows) / G, p.n_rows = its(rows) - p.row0, tiles = its(shared) / kTile, first_len = its(len);
      break;
    }
    before += __builtin_amdgcn_readlane(incl, 63);
  }
  if (p.group < 0) return p;
  const int per = PerPiece(tiles, a.n_split);
  p.tile0 = p.piece * per, p.tile1 = min(p.tile0 + per, tiles);
  if (p.tile0 >= p.tile1) p.group = -1;
  if (p.group < 0) return p;
  p.reader = p.first;
  if (__builtin_expect(first_len < tiles * kTile, 0)) {
    const int group = p.group;
    p.group = -1;  // (if there is none, nobody reads the partials)
    for (int m0 = 0; m0 < n_seqs; m0 += 64) {
      const bool takes = m0 + lane < n_seqs && a.seq_len[p.first + min(m0 + lane, n_seqs - 1)] >= tiles * kTile;
      const unsigned long long who = __ballot(takes);
      if (who != 0) {
        p.group = group, p.reader = p.first + m0 + __builtin_ctzll(who);
        break;
      }
    }
  }
  return p;
}

template <int FMT, int D, int PT, int RB>
__global__ __launch_bounds__(64 * kSharedWaves, RB * D <= 256 ? 2 : 1) void SharedPart(const SharedArgs a) {
  constexpr int ROWS = 16 * RB;
  constexpr bool TWO = RB * D <= 256;  // workgroups a CU
  const Geom g = a.g;
  const int G = g.group(), H = g.n_kv;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  __shared__ __align__(16) SharedLds<D, RB> lds;

  if (static_cast<int>(blockIdx.x) >= a.prefix_groups) {  // ---- a piece of a tail: the query heads of one kv head of a sequence
    const int u = blockIdx.x - a.prefix_groups, h = u % H, piece = u / H % a.tail_split, s = u / H / a.tail_split;
    const Keys k = KeysOf(a, s);
    const int tiles = (k.tail + kTile - 1) / kTile, per = PerPiece(tiles, a.tail_split);
    const int tile0 = piece * per, tile1 = min(tile0 + per, tiles);
    if (tile0 >= tile1) return;
    const size_t row0 = size_t(s) * g.n_q + size_t(h) * G;
    auto& lds1 = reinterpret_cast<SharedLds<D, 1>&>(lds);
    QueryRows<D, 1> queries;
    queries.lds = lds1.q;
    queries.Request(a.q, a.q_dtype, [&](int r) { return row0 + min(r, G - 1); });
    float m[1], l[1];
    f4v o[1][D / 16];
    StreamKeys<FMT, D, PT, 1, TWO>(a, a.table + int64_t(s) * a.stride, k.prefix, h, tile0 + wave, kSharedWaves, tile1, k.tail, queries,
                              lds1.scales[wave], m, l, o);
    MergeWaves<D, 1>(a, lds1, m, l, o, G, [&](int r) { return row0 + r; }, a.n_split + piece);
    return;
  }
  const PrefixPiece pp = FindPiece<ROWS>(a);
  if (pp.group < 0) return;
  auto row_of = [&](int r) -> size_t { return pp.Row(a, r); };
  QueryRows<D, RB> queries;
  queries.lds = lds.q;
  queries.Request(a.q, a.q_dtype, row_of);
  float m[RB], l[RB];
  f4v o[RB][D / 16];
  StreamKeys<FMT, D, PT, RB, TWO>(a, a.table + int64_t(pp.reader) * a.stride, 0, pp.h, pp.tile0 + wave, kSharedWaves, pp.tile1,
                             pp.tile1 * kTile, queries, lds.scales[wave], m, l, o);
  // (rows of sequences shorter than the prefix leave partials that nobody reads)
  MergeWaves<D, RB>(a, lds, m, l, o, pp.n_rows, row_of, pp.piece);
}

// One workgroup per (query head, sequence): the prefix's partials and the tail's, weighed by 2^(m - M) and 1 / l. A group of
// D / 4 lanes takes every n-th partial, four dims a lane; the groups' sums meet in LDS. (64 x 24 rows of up to ten partials of 256
// dims: 6.0 us, a round trip behind a round trip; the partials are in the caches.)
struct MergeArgs {
  SharedArgs s;
  const float* gate;
  void* out;
  int32_t out_dtype;
};
constexpr int kMergeThreads = 256;
__global__ __launch_bounds__(kMergeThreads) void SharedMerge(const MergeArgs a) {
  const Geom g = a.s.g;
  const int D = g.hd, hq = blockIdx.x, s = blockIdx.y, t = threadIdx.x;
  const size_t row = size_t(s) * g.n_q + hq;
  const int slots = a.s.n_split + a.s.tail_split;
  const Keys k = KeysOf(a.s, s);
  const int pre_tiles = k.prefix / kTile, tail_tiles = (k.tail + kTile - 1) / kTile;
  const int pre_per = PerPiece(pre_tiles, a.s.n_split), tail_per = PerPiece(tail_tiles, a.s.tail_split);
  const int n_pre = (pre_tiles + pre_per - 1) / pre_per, n = n_pre + (tail_tiles + tail_per - 1) / tail_per;
  auto slot_of = [&](int i) -> size_t { return row * slots + (i < n_pre ? i : a.s.n_split + i - n_pre); };
  __shared__ float red[kMergeThreads / 64];
  __shared__ __align__(16) float sums[kMergeThreads * 4];
  __shared__ float lsum[kMergeThreads / 32];
  const int lanes = D / 4, grp = t / lanes, dl = t % lanes, groups = kMergeThreads / lanes;
  auto sum_of = [&](int i) { return *reinterpret_cast<const float2*>(&a.s.ml[slot_of(i) * 2]); };
  auto acc_of = [&](int i) { return *reinterpret_cast<const float4*>(&a.s.acc[slot_of(i) * D + 4 * dl]); };
  // (a lane's first partials are asked for before the maximum is known: one round trip less)
  constexpr int kEarly = 4;
  float2 v0[kEarly];
  float4 x0[kEarly];
#pragma unroll
  for (int e = 0; e < kEarly; ++e)
    if (grp + e * groups < n) v0[e] = sum_of(grp + e * groups), x0[e] = acc_of(grp + e * groups);
  float M = kNegMax;
  for (int i = t; i < n; i += kMergeThreads) M = fmaxf(M, a.s.ml[slot_of(i) * 2]);
  M = WaveMax(M);
  if (t % 64 == 0) red[t / 64] = M;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kMergeThreads / 64; ++w) M = fmaxf(M, red[w]);
  float4 A = {0.0f, 0.0f, 0.0f, 0.0f};
  float L = 0.0f;
  auto add = [&](const float2 v, const float4 x) {
    const float w = __builtin_amdgcn_exp2f(v.x - M);
    A.x = __builtin_fmaf(w, x.x, A.x), A.y = __builtin_fmaf(w, x.y, A.y);
    A.z = __builtin_fmaf(w, x.z, A.z), A.w = __builtin_fmaf(w, x.w, A.w);
    L = __builtin_fmaf(w, v.y, L);
  };
#pragma unroll
  for (int e = 0; e < kEarly; ++e)
    if (grp + e * groups < n) add(v0[e], x0[e]);
#pragma unroll 4
  for (int i = grp + kEarly * groups; i < n; i += groups) add(sum_of(i), acc_of(i));
  *reinterpret_cast<float4*>(&sums[grp * D + 4 * dl]) = A;
  if (dl == 0) lsum[grp] = L;
  __syncthreads();
  for (int e = t; e < D; e += kMergeThreads) {
    float v = 0.0f, sum = 0.0f;
    for (int q = 0; q < groups; ++q) v += sums[q * D + e], sum += lsum[q];
    v = n == 0 ? 0.0f : v / sum;  // (a sequence without keys)
    if (a.gate != nullptr) v *= 1.0f / (1.0f + __expf(-a.gate[row * D + e]));
    Store1(a.out, row * D + e, a.out_dtype, v);
  }
}

struct SharedPlan {
  int row_blocks;  // of 16 query rows, that a wave of a prefix takes
  int32_t max_blocks, n_split, tail_split, prefix_groups;
  int64_t groups;  // workgroups in all
  size_t off_ml, off_acc, bytes;
};
SharedPlan MakeSharedPlan(const Geom& m, int32_t n_seqs, int32_t n_groups, int32_t max_shared, int32_t max_tail) {
  SharedPlan p;
  const int64_t rows = int64_t(n_seqs) * m.group(), per_group = (rows + n_groups - 1) / n_groups;
  auto blocks = [&](int rb) { return (per_group + 16 * rb - 1) / (16 * rb); };
  const int64_t cus = ComputeUnits(), pre_tiles = max_shared / kTile, tail_tiles = (int64_t(max_tail) + kTile - 1) / kTile;
  // One row block a wave, or as many as registers allow (three of 128 dims would, but two leave a CU two workgroups:
  // 256 rows of an 8K prefix 41 us against 44). Four tiles cost a CU 1.1 us with one, 1.6 us with two, 1.25 us with three,
  // whose one workgroup a CU also takes 14 us more to begin and to end. (32K keys x 12 rows of 256 dims: 23 us with one, 37
  // with three; 32K x 384 rows: 223 and 107.)
  const int most = m.hd == 128 ? 2 : 3;
  const double work = double(n_groups) * m.n_kv * pre_tiles / cus;
  p.row_blocks = work * blocks(most) * (most == 2 ? 1.6 : 1.25) + (most == 2 ? 0.0 : 14.0) < work * blocks(1) * 1.1 ? most : 1;
  p.max_blocks = static_cast<int32_t>(n_groups == 1 ? blocks(p.row_blocks) : rows / (16 * p.row_blocks) + n_groups);
  // A prefix is cut so that the row blocks of an average group give every CU a workgroup, or two if its registers hold them
  // and each still has four tiles a wave (256 rows x 32K keys of 128 dims: 95 us, with one 117; 64 rows x 8K: 24 and 20). A
  // tail is cut into pieces of at most sixteen tiles, and finer while that leaves CUs idle; a piece has a tile for every wave.
  // Sixteen workgroups a CU are enough of them: what a bound far above the lengths costs is their places in the workspace.
  const int64_t per_piece = std::max<int64_t>(1, std::min<int64_t>(int64_t(n_groups) * blocks(p.row_blocks), p.max_blocks)) * m.n_kv;
  const bool two = p.row_blocks * m.hd <= 256 && 2 * cus / per_piece * 4 * 4 <= pre_tiles;
  p.n_split = static_cast<int32_t>(std::max<int64_t>(1, std::min((two ? 2 * cus : cus) / per_piece, (pre_tiles + 3) / 4)));
  if (pre_tiles == 0) p.n_split = 0;
  const int64_t tails = int64_t(n_seqs) * m.n_kv;
  const int64_t pieces = std::min(std::max((cus + tails - 1) / tails, (tail_tiles + 15) / 16), std::max<int64_t>(16 * cus / tails, 1));
  p.tail_split = static_cast<int32_t>(std::max<int64_t>(1, std::min(pieces, (tail_tiles + 3) / 4)));
  p.prefix_groups = static_cast<int32_t>((int64_t(m.n_kv) * p.n_split + 7) / 8 * 8 * p.max_blocks);
  p.groups = p.prefix_groups + tails * p.tail_split;
  const size_t parts = size_t(n_seqs) * m.n_q * (p.n_split + p.tail_split);
  p.off_ml = 0;
  p.off_acc = Align(sizeof(float) * 2 * parts);
  p.bytes = Align(p.off_acc + sizeof(float) * parts * m.hd);
  return p;
}

template <int FMT, int D, int PT>
void LaunchShared(const SharedArgs& all, int row_blocks, dim3 grid, hipStream_t st) {
  constexpr int MOST = D == 128 ? 2 : 3;
  const dim3 block(64 * kSharedWaves);
  SharedArgs a = all;
  // Tails that fill the chip twice have a launch of their own, where a CU takes two workgroups of them (64 of 1500 keys
  // beside 32K shared ones: 136 us, with the prefixes 146).
  if (row_blocks * D > 256 && grid.x - a.prefix_groups >= 2u * ComputeUnits()) {
    a.prefix_groups = 0;
    hipLaunchKernelGGL((SharedPart<FMT, D, PT, 1>), dim3(grid.x - all.prefix_groups), block, 0, st, a);
    grid.x = a.prefix_groups = all.prefix_groups;
  }
  if (row_blocks == 1) hipLaunchKernelGGL((SharedPart<FMT, D, PT, 1>), grid, block, 0, st, a);
  else hipLaunchKernelGGL((SharedPart<FMT, D, PT, MOST>), grid, block, 0, st, a);
}
template <int FMT>
void LaunchSharedFormat(const SharedArgs& a, int row_blocks, dim3 grid, hipStream_t st) {
  const Geom& m = a.g;
  if (m.hd == 256 && m.pt == 64) LaunchShared<FMT, 256, 64>(a, row_blocks, grid, st);
  else if (m.hd == 256 && m.pt == 32) LaunchShared<FMT, 256, 32>(a, row_blocks, grid, st);
  else if (m.hd == 256) LaunchShared<FMT, 256, 16>(a, row_blocks, grid, st);
  else if (m.pt == 64) LaunchShared<FMT, 128, 64>(a, row_blocks, grid, st);
  else if (m.pt == 32) LaunchShared<FMT, 128, 32>(a, row_blocks, grid, st);
  else LaunchShared<FMT, 128, 16>(a, row_blocks, grid, st);
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
  if (int64_t(page_table_stride) * m.pt > 0x7FFFFFFF - kTile * kSharedWaves) return YAHKV_ERR_SHAPE;
  const SharedPlan p = MakeSharedPlan(m, n_seqs, n_groups, max_shared_len, max_tail_len);
  if (workspace_bytes < p.bytes) return YAHKV_ERR_WORKSPACE;
  if (p.groups > 0x7FFFFFFF) return YAHKV_ERR_SHAPE;
  char* ws = static_cast<char*>(workspace);
  SharedArgs a{};
  a.g = m, a.pools = MakePools(*pools), a.table = page_table, a.seq_len = seq_len, a.group_first = group_first;
  a.shared_len = shared_len, a.stride = page_table_stride, a.n_seqs = n_seqs, a.n_groups = n_groups;
  a.max_shared = max_shared_len, a.max_tail = max_tail_len, a.q = q, a.q_dtype = q_dtype, a.scale = softmax_scale;
  a.max_blocks = p.max_blocks, a.n_split = p.n_split, a.tail_split = p.tail_split, a.prefix_groups = p.prefix_groups;
  a.ml = reinterpret_cast<float*>(ws + p.off_ml), a.acc = reinterpret_cast<float*>(ws + p.off_acc);
  hipStream_t st = static_cast<hipStream_t>(stream);
  const dim3 grid(static_cast<unsigned>(p.groups));
  if (m.format == YAHKV_Q8_0) LaunchSharedFormat<8>(a, p.row_blocks, grid, st);
  else LaunchSharedFormat<4>(a, p.row_blocks, grid, st);
  if (const int rc = LaunchStatus()) return rc;
  const MergeArgs ma{a, gate, out, out_dtype};
  hipLaunchKernelGGL(SharedMerge, dim3(static_cast<unsigned>(m.n_q), static_cast<unsigned>(n_seqs)), dim3(kMergeThreads), 0, st, ma);
  return LaunchStatus();
}
