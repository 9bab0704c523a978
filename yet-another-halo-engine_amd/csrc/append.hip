// Token append: block-quantize K and V rows and scatter them into their pages, optionally with the head RMSNorm and
// NeoX RoPE of K (and of the queries) fused in; and the inverse gather used by tests.
//
// Placement follows the reference's page mapping (engine/gpu/loom/tools/gen_kvq.py:48-71): token at position p goes
// to page table[p / PT] (clamped into the pool), slot p % PT; positions are clamped to the table
// (gen_decode_attn.py:59-63). The quantizers are in quant.hpp.
//
// The fused form follows the reference's decode kernel (engine/gpu/loom/yah_fused_qk_rope_f32.loom:1-10, Q branch
// :96-146, K branch :147-241) and its batched, paged rewrite for prefill chunks
// (engine/gpu/loom/tools/emit_prefill_pp.py:31-111): per head
//   inv_rms = rsqrt(sum_i x[i]^2 / head_dim + eps); normed[i] = (x[i] * inv_rms) * weight[i]
//   angle(p) = pos * (1 / theta^(2 p / rotary_dim)), p < half = rotary_dim / 2
//   out[p] = normed[p] cos - normed[p + half] sin; out[p + half] = normed[p] sin + normed[p + half] cos
// and dims at or past rotary_dim are only normalised (yahkv_rotary_append: rotary.hpp's angles, either layout, a part of
// the head, positions and row strides of their own, the norm optional). The angle uses the token's position as given; the page slot
// uses the position clamped to the table, as in the reference (:89-94). What the reference stores as f16 rows is
// stored here as q8_0 / q4_0 blocks: the rotated K never makes a round trip through memory as f32.
#include "common.hpp"
#include "quant.hpp"
#include "rotary.hpp"
#include "store.hpp"

namespace yahkv {
namespace {

struct RopeArgs {
  Geom g;
  Pools pools;
  const int32_t* table;
  int32_t stride;
  const int32_t* start_pos;
  const int32_t* n_valid;
  int32_t n_seqs, n_new;
  const void* k_src;
  const void* v_src;
  int32_t src_dtype;
  const float* k_weight;
  const float* q_weight;
  float theta, eps;
  int32_t rotary_dim;
  const void* q_src;  // [n_seqs][n_new][n_q][D] of src_dtype, or null
  void* q_out;        // same shape, of q_out_dtype
  int32_t q_out_dtype;
  float* k_out;       // [n_seqs][n_new][H][D] f32 or null: the rotated K rows, for callers that want them
  int32_t per_xcd;    // AppendRows: tokens per XCD and sequence (a multiple of the page), or 0: tokens in order
  int32_t skip_v;     // AppendRows: the V rows are left to another launch (AppendPages with skip_k)
  int32_t skip_k;     // AppendPages: V only
  // yahkv_rotary_append (kGeneral rows): the rotation, positions of its own (or null), and rows at strides of their own
  RotaryArgs rotary;
  const int32_t* positions;
  RowsArgs k_rows, v_rows, q_rows, q_out_rows;
};
// What AppendRows does to K and query rows before it stores them.
enum RowsMode { kAsTheyAre = 0, kNeox = 1, kGeneral = 2 };

// One workgroup of four wavefronts per token (or several: FLIGHT below). With ROPE, the token's angles (they depend on the position and the
// pair, not on the head) are computed once into LDS; without, K rows are quantized as they are (plain append) and
// there are no query rows. The token's rows of head_dim values (its H K heads, its H V heads, then its
// query heads) are dealt to the wavefronts in turn; a row lies across a wavefront, four consecutive dims per lane, so
// every load and store is 16 (or 8) bytes per lane, the sum of squares and the block maxima are DPP reductions, and
// the partner of a rotated pair comes through one lane shuffle: rows never go through LDS. A wavefront issues the
// loads of all its rows (up to eight at a time) before it works on the first; for that the loads must not sit behind
// branches, so the source rows' type SRC is known when compiling (as in AppendPages: with the type a run-time value
// each load waited for the one before) and a row or lane that has nothing to load asks for an address that exists.
// FLIGHT: rows whose loads a wavefront issues at a time. Eight fill the memory system in a long call; a short one waits for its
// code, and its rows go to several workgroups a token (grid y) with one at a time instead (yahkv_rotary_append, 64 tokens of 4
// + 4 + 24 rows of 256 dims: 5.8 us, with two 6.5, with four 7.4, with eight and one workgroup a token 10).
constexpr int kRopeWaves = 4, kRowsInFlight = 8;
template <int FMT, int MODE, int SRC, int FLIGHT>
__global__ __launch_bounds__(64 * kRopeWaves) void AppendRows(const RopeArgs a) {
#pragma clang fp contract(off)
  constexpr bool ROPE = MODE != kAsTheyAre;
  const Geom g = a.g;
  const int H = g.n_kv, PT = g.pt, D = g.hd, NQ = a.q_src != nullptr ? g.n_q : 0;
  // (with a.skip_v the token's rows are its K heads and its query heads: row numbers H .. 2 H - 1 are passed over)
  const int rows_per_token = (a.skip_v ? H : 2 * H) + NQ;
  auto row_of = [&](int r) -> int { return a.skip_v && r >= H ? r + H : r; };
  const int wave = threadIdx.x / 64, lane = threadIdx.x % 64;
  // Token i of sequence s. Workgroup b of a dispatch runs on XCD b % 8, and V's codes are single bytes of the
  // transposed page: with a long chunk's tokens dealt to the workgroups in order, every line of a page would be put
  // together from bytes in eight L2 caches, each of which writes its part back on its own. a.per_xcd > 0: workgroups
  // b, b + 8, ... take per_xcd consecutive tokens (whole pages), so a page's bytes meet in one L2.
  int i = int(blockIdx.x % a.n_new), s = int(blockIdx.x / a.n_new);
  if (a.per_xcd > 0) {
    const int span = 8 * a.per_xcd, r = int(blockIdx.x % span);
    s = int(blockIdx.x / span), i = (r % 8) * a.per_xcd + r / 8;
    if (i >= a.n_new) return;
  }
  const int nv = a.n_valid != nullptr ? min(a.n_valid[s], a.n_new) : a.n_new;
  if (i >= nv) return;  // padding row of a short chunk
  const int start = a.start_pos[s], pos_raw = start + i, last_pos = a.stride * PT - 1;
  const int pos = min(max(pos_raw, 0), last_pos);
  // Where several tokens of the call clamp to the table's first or last slot, the one a loop over the tokens would
  // leave there writes it (AppendPages' token_at); the others only produce their query rows and rotated K rows.
  const bool owns_slot = pos_raw >= last_pos ? i == nv - 1 : (pos_raw <= 0 ? i == min(nv - 1, -start) : true);
  const int page = ClampPage(a.table[int64_t(s) * a.stride + pos / PT], g.n_pages);
  const int t = pos % PT;

  __shared__ __align__(16) float cs[128], sn[128];  // rotary_dim / 2 <= 128
  const int rot = a.rotary_dim, half = rot / 2;
  const float posf = static_cast<float>(pos_raw);
  if constexpr (MODE == kNeox) {
    for (int p = threadIdx.x; p < half; p += 64 * kRopeWaves) {
      const float inv_freq = 1.0f / powf(a.theta, (2.0f * static_cast<float>(p)) / static_cast<float>(rot));
      float sv, cv;
      sincosf(posf * inv_freq, &sv, &cv);
      cs[p] = cv, sn[p] = sv;
    }
    __syncthreads();
  }
  if constexpr (MODE == kGeneral) {
    const int turn_pos = a.positions != nullptr ? a.positions[int64_t(s) * a.n_new + i] : pos_raw;
    for (int p = threadIdx.x; p < half; p += 64 * kRopeWaves) {
      float cv, sv;
      TurnCosSin(turn_pos, a.rotary.turns[p], &cv, &sv);
      cs[p] = cv * a.rotary.magnitude, sn[p] = sv * a.rotary.magnitude;
    }
    __syncthreads();
  }
  const int d0 = 4 * lane;  // this lane's four dims of every row
  const bool has = d0 < D;
  // This lane's part of the rotation, the same for every row: element e = d0 + j is the first of its pair
  // (e < half: out = x c - partner s, partner = e + half), the second (half <= e < rot: out = partner s + x c,
  // partner = e - half) or past the rotated dims. rotary_dim / 2 is a multiple of 4 (checked by the entry point), so
  // the four partners lie in one lane. (The general rotation counts from its first dim, a multiple of 4; in its
  // interleaved layout a lane holds two whole pairs.)
  float c4[4] = {1.0f, 1.0f, 1.0f, 1.0f}, s4[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  int partner_lane = lane;
  const int r0 = MODE == kGeneral ? d0 - a.rotary.first : d0;
  const bool pairs_inside = MODE == kGeneral && a.rotary.layout == YAHKV_ROTARY_INTERLEAVED;
  const bool turned = ROPE && has && r0 >= 0 && r0 < rot;
  if (turned) {
    const bool first = r0 < half;
    if (!pairs_inside) partner_lane = first ? lane + half / 4 : lane - half / 4;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int p = pairs_inside ? (r0 + j) / 2 : first ? r0 + j : r0 + j - half;
      c4[j] = cs[p];
      s4[j] = (pairs_inside ? j % 2 == 0 : first) ? -sn[p] : sn[p];
    }
  }
  float4 wk = {1.0f, 1.0f, 1.0f, 1.0f}, wq = wk;  // this lane's norm weights
  if (ROPE && a.k_weight != nullptr && has) wk = *reinterpret_cast<const float4*>(a.k_weight + d0);
  if (ROPE && a.q_weight != nullptr && has) wq = *reinterpret_cast<const float4*>(a.q_weight + d0);
  // source of row `row` of the token and its element offset
  auto source = [&](int row, const void** src, size_t* off) {
    if constexpr (MODE == kGeneral) {
      const RowsArgs& r = row < H ? a.k_rows : row < 2 * H ? a.v_rows : a.q_rows;
      *src = r.data;
      *off = static_cast<size_t>(s * r.seq + i * r.token + (row < H ? row : row < 2 * H ? row - H : row - 2 * H) * r.head);
      return;
    }
    const size_t tok = size_t(s) * a.n_new + i;
    if (row < H) *src = a.k_src, *off = (tok * H + row) * D;
    else if (row < 2 * H) *src = a.v_src, *off = (tok * H + (row - H)) * D;
    else *src = a.q_src, *off = (tok * g.n_q + (row - 2 * H)) * D;
  };
  for (int first_row = wave + kRopeWaves * FLIGHT * blockIdx.y; first_row < rows_per_token; first_row += kRopeWaves * FLIGHT * gridDim.y) {
    uint4 raw[FLIGHT];
#pragma unroll
    for (int j = 0; j < FLIGHT; ++j) {
      const void* src;
      size_t off;
      source(row_of(min(first_row + kRopeWaves * j, rows_per_token - 1)), &src, &off);
      raw[j] = LoadRaw4(src, off + (has ? d0 : 0), SRC);
    }
#pragma unroll
    for (int j = 0; j < FLIGHT; ++j) {
      if (first_row + kRopeWaves * j >= rows_per_token) break;
      const int row = row_of(first_row + kRopeWaves * j);
      const bool is_v = row >= H && row < 2 * H, is_q = row >= 2 * H;
      float4 v = Widen4(raw[j], SRC);
      if (!has) v = float4{0.0f, 0.0f, 0.0f, 0.0f};
      if (ROPE && !is_v) {
        if (MODE == kNeox || a.rotary.normalise) {
          const float ss = WaveSum(v.x * v.x + v.y * v.y + v.z * v.z + v.w * v.w);
          const float inv_rms = 1.0f / sqrtf(ss / static_cast<float>(D) + a.eps);
          const float4 w = is_q ? wq : wk;
          v = float4{(v.x * inv_rms) * w.x, (v.y * inv_rms) * w.y, (v.z * inv_rms) * w.z, (v.w * inv_rms) * w.w};
        }
        float px, py, pz, pw;
        if (pairs_inside) {
          px = v.y, py = v.x, pz = v.w, pw = v.z;
        } else {
          px = __shfl(v.x, partner_lane, 64), py = __shfl(v.y, partner_lane, 64);
          pz = __shfl(v.z, partner_lane, 64), pw = __shfl(v.w, partner_lane, 64);
        }
        // first of a pair: x c - partner s; second: partner s + x c (s4 carries the sign); past rot: c = 1, s = 0
        if (MODE == kNeox || turned)
          v = float4{v.x * c4[0] + px * s4[0], v.y * c4[1] + py * s4[1], v.z * c4[2] + pz * s4[2], v.w * c4[3] + pw * s4[3]};
      }
      const void* src;
      size_t off;
      source(row, &src, &off);
      if (is_q) {
        if constexpr (MODE == kGeneral) off = static_cast<size_t>(s * a.q_out_rows.seq + i * a.q_out_rows.token + (row - 2 * H) * a.q_out_rows.head);
        if (has) Store4(a.q_out, off + d0, a.q_out_dtype, v);
        continue;
      }
      if constexpr (MODE == kGeneral) off = ((size_t(s) * a.n_new + i) * H + row) * D;  // of k_out, for the K rows
      if (!is_v && a.k_out != nullptr && has) *reinterpret_cast<float4*>(a.k_out + off + d0) = v;
      // quantize: block b = lanes 8 b .. 8 b + 7
      const int h = is_v ? row - H : row, lb = lane % 8;
      uint16_t scale;
      const uint32_t codes = FMT == 8 ? QuantizeLanesQ8(v, &scale) : QuantizeLanesQ4(v, lb, &scale);
      if (!has || !owns_slot) continue;
      if (!is_v)
        StoreRowK<FMT>(a.pools, g, page, h, t, lane, codes, scale);
      else
        StoreRowV<FMT>(a.pools, g, page, h, t, lane, codes, scale);
    }
  }
}

// Chunks: one workgroup per (sequence, page touched by the chunk, kv head). A token at a time per wavefront, the rows
// are quantized exactly as above, but the codes and scales go to an LDS image of the page's (page, head) regions, and
// the image leaves for HBM in 16-byte pieces once the page's tokens are done. Token by token the V codes would be
// single bytes 64 bytes apart (V lies transposed, [dim][token], so that decode reads 16 tokens of a dim at once) and
// every K block a 32-byte piece; page by page they are whole lines.
// Positions clamp to the table as everywhere (gen_decode_attn.py:59-63); where several tokens of a chunk clamp to
// the same slot (the first or the last of the table), the last token wins, as in a loop over the tokens.
constexpr int kPageWaves = 4;
constexpr int kPageAppendMin = 8;  // tokens per sequence from which a call is treated as a chunk
// SRC: the source rows' type, known when compiling (as a run-time value it put a three-way branch around every
// row's conversion). D: the head dim (as a run-time value whether a wavefront's sets are one or two made every token's address the
// vector unit's: 8 x 2048 tokens of 4 heads of 256 dims 31.1 us, 29.9 as a constant).
// TURN: yahkv_rotary_append's chunks: the K rows of a wave's four tokens are normalised and turned before they are quantized.
// Their cosines and sines are worked out by the wave into LDS, again for every kv head's workgroup (a twentieth of the
// kernel's instructions; a table for all heads would need memory and a launch of its own).
template <int FMT, int SRC, bool TURN, int D>
__global__ __launch_bounds__(64 * kPageWaves) void AppendPages(const RopeArgs a) {
#pragma clang fp contract(off)
  const Geom g = a.g;
  const int H = g.n_kv, PT = g.pt;
  constexpr int NB = D / 32, KB = FMT == 8 ? 32 : 16;    // blocks, bytes of K codes per token and block
  constexpr int v_rows = FMT == 8 ? D : NB * 16;             // byte rows of the V image, PT bytes each
  const int wave = threadIdx.x / 64, lane = threadIdx.x % 64, h = blockIdx.y, s = blockIdx.z;
  const int nv = a.n_valid != nullptr ? min(max(a.n_valid[s], 0), a.n_new) : a.n_new;
  if (nv <= 0) return;
  const int start = a.start_pos[s], last_pos = a.stride * PT - 1;
  const int p_first = min(max(start, 0), last_pos), p_last = min(max(start + nv - 1, 0), last_pos);
  const int pi = p_first / PT + blockIdx.x;
  if (pi > p_last / PT) return;
  const int t_lo = max(p_first, pi * PT) - pi * PT, t_hi = min(p_last, pi * PT + PT - 1) - pi * PT + 1;
  const int page = ClampPage(a.table[int64_t(s) * a.stride + pi], g.n_pages);
  // the token of the chunk that ends up at position pos (the last one, where several clamp to it)
  auto token_at = [&](int pos) -> int {
    if (pos == last_pos && start + nv - 1 >= last_pos) return nv - 1;
    if (pos == 0 && start <= 0) return min(nv - 1, -start);
    return pos - start;
  };

  __shared__ __align__(16) uint8_t lk[8 * 64 * 32], lv[256 * (64 + 4)];  // images of the K and V code regions
  __shared__ __align__(16) uint16_t lks[64 * 8], lvs[8 * 64];      // and of the scale regions
  // A row lies across D / 4 lanes, so that at 128 dims a wavefront has two sets of four tokens side by side (5 x 1037 tokens of 8
  // heads, pages of 32: 14.4 us, turned 24.4; with half the lanes idle 18.9 and 31.6).
  constexpr int row_lanes = D / 4, sets = 64 / row_lanes;
  const int set = lane / row_lanes, rl = lane % row_lanes;
  const int d0 = 4 * rl, b = rl / 8, lb = rl % 8;
  // A set of lanes takes four consecutive tokens at a time (their rows in flight together): a lane then holds, for each
  // of its four dims, the codes of four neighbouring tokens, which is one dword of the V image instead of four bytes.
  // (The image's rows are padded by a dword: with rows of exactly PT bytes the 64 lanes of such a store would all
  // hit one LDS bank.)
  // The rows of the wave's next four tokens are requested before the current four are quantized.
  uint4 rk[4], rv[4];
  auto request = [&](int q) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int t = 4 * q + j;
      rk[j] = rv[j] = uint4{0u, 0u, 0u, 0u};  // reads as 0.0 in every source type
      if (t >= t_lo && t < t_hi) {
        const int tok = token_at(pi * PT + t);
        rv[j] = LoadRaw4(a.v_src, static_cast<size_t>(s * a.v_rows.seq + tok * a.v_rows.token + h * a.v_rows.head) + d0, SRC);
        if (!a.skip_k) {
          if constexpr (TURN) rk[j] = LoadRaw4(a.k_src, static_cast<size_t>(s * a.k_rows.seq + tok * a.k_rows.token + h * a.k_rows.head) + d0, SRC);
          else rk[j] = LoadRaw4(a.k_src, ((size_t(s) * a.n_new + tok) * H + h) * D + d0, SRC);
        }
      }
    }
  };
  __shared__ __align__(16) float lcs[TURN ? kPageWaves : 1][TURN ? 512 : 4], lsn[TURN ? kPageWaves : 1][TURN ? 512 : 4];
  auto angle = [&](int j, int p) -> int { return (4 * set + j) * (D / 2) + p; };  // place of pair p of the set's token j
  float4 wk = {1.0f, 1.0f, 1.0f, 1.0f};
  if constexpr (TURN)
    if (a.k_weight != nullptr) wk = *reinterpret_cast<const float4*>(a.k_weight + d0);
  // the K rows of the set's tokens 4 q .. 4 q + 3, normalised and turned (see AppendRows for a lane's part of the rotation)
  auto turn = [&](int q, float4 (&kx)[4]) {
    const int rot = a.rotary.rot, half = rot / 2, r0 = d0 - a.rotary.first;
    const bool turned = r0 >= 0 && r0 < rot, inside = a.rotary.layout == YAHKV_ROTARY_INTERLEAVED, first = r0 < half;
    const int partner = turned && !inside ? (first ? lane + half / 4 : lane - half / 4) : lane;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int t = min(max(4 * q + j, t_lo), t_hi - 1), tok = token_at(pi * PT + t);
      const int pos = a.positions != nullptr ? a.positions[static_cast<int64_t>(s) * a.n_new + tok] : start + tok;
      for (int p = rl; p < half; p += row_lanes) {
        float c, v;
        TurnCosSin(pos, a.rotary.turns[p], &c, &v);
        lcs[wave][angle(j, p)] = c * a.rotary.magnitude, lsn[wave][angle(j, p)] = v * a.rotary.magnitude;
      }
    }
    if (a.rotary.normalise) {
      float ss[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) ss[j] = RowSum(kx[j].x * kx[j].x + kx[j].y * kx[j].y + kx[j].z * kx[j].z + kx[j].w * kx[j].w, sets == 1);
      // (lane l works out the reciprocal of row l % 4 for everybody)
      const float mine = lane & 2 ? (lane & 1 ? ss[3] : ss[2]) : (lane & 1 ? ss[1] : ss[0]);
      const float inv = 1.0f / sqrtf(mine / static_cast<float>(D) + a.eps);
      const float i4[4] = {Dpp<0x00>(inv), Dpp<0x55>(inv), Dpp<0xAA>(inv), Dpp<0xFF>(inv)};
#pragma unroll
      for (int j = 0; j < 4; ++j)
        kx[j] = float4{(kx[j].x * i4[j]) * wk.x, (kx[j].y * i4[j]) * wk.y, (kx[j].z * i4[j]) * wk.z, (kx[j].w * i4[j]) * wk.w};
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float4 v = kx[j];
      float4 x;
      if (inside) {
        const int p = turned ? r0 / 2 : 0;
        const float2 c = *reinterpret_cast<const float2*>(&lcs[wave][angle(j, p)]), sv = *reinterpret_cast<const float2*>(&lsn[wave][angle(j, p)]);
        x = float4{v.x * c.x - v.y * sv.x, v.y * c.x + v.x * sv.x, v.z * c.y - v.w * sv.y, v.w * c.y + v.z * sv.y};
      } else {
        const int p = turned ? (first ? r0 : r0 - half) : 0;
        const float4 c = *reinterpret_cast<const float4*>(&lcs[wave][angle(j, p)]);
        float4 sv = *reinterpret_cast<const float4*>(&lsn[wave][angle(j, p)]);
        if (first) sv = float4{-sv.x, -sv.y, -sv.z, -sv.w};
        const float px = __shfl(v.x, partner, 64), py = __shfl(v.y, partner, 64);
        const float pz = __shfl(v.z, partner, 64), pw = __shfl(v.w, partner, 64);
        x = float4{v.x * c.x + px * sv.x, v.y * c.y + py * sv.y, v.z * c.z + pz * sv.z, v.w * c.w + pw * sv.w};
      }
      if (turned) kx[j] = x;
    }
    __builtin_amdgcn_wave_barrier();  // (the table is rewritten for the next four tokens)
  };
  const int span = 4 * sets;  // tokens of a wavefront at a time (pages are multiples of 16)
  int w0 = t_lo / span + wave;
  if (span * w0 < t_hi) request(sets * w0 + set);
  for (; span * w0 < t_hi; w0 += kPageWaves) {
    const int q = sets * w0 + set;
    float4 kx[4], vx[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) kx[j] = Widen4(rk[j], SRC), vx[j] = Widen4(rv[j], SRC);
    if (span * (w0 + kPageWaves) < t_hi) request(q + sets * kPageWaves);
    if constexpr (TURN) turn(q, kx);
    uint32_t vc[4];
    if constexpr (FMT == 8) {
      // Eight rows are in flight (K and V of four tokens) and a block has eight lanes: lane lb of a block takes row
      // lb's amax and does the two divisions for it (the same operations on the same values, so the same bits),
      // instead of every lane doing them for every row; the reciprocals go back through lane shuffles.
      float am[8];
#pragma unroll
      for (int j = 0; j < 4; ++j) am[j] = BlockAmaxQ8(kx[j]), am[4 + j] = BlockAmaxQ8(vx[j]);
      float mine = am[0];
#pragma unroll
      for (int r = 1; r < 8; ++r) mine = lb == r ? am[r] : mine;
      float inv;
      uint16_t sc;
      ScaleQ8(mine, &inv, &sc);
      {
        const int t = 4 * q + lb % 4;  // row lb is K (lb < 4) or V of this token
        if (t >= t_lo && t < t_hi) {
          if (lb < 4) lks[t * NB + b] = sc;
          else lvs[b * PT + t] = sc;
        }
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int t = 4 * q + j;
        const uint32_t kc = CodesLanesQ8(kx[j], __shfl(inv, (lane & ~7) | j, 64));
        vc[j] = CodesLanesQ8(vx[j], __shfl(inv, (lane & ~7) | (4 + j), 64));
        if (t < t_lo || t >= t_hi) continue;
        *reinterpret_cast<uint32_t*>(&lk[(b * PT + t) * KB + 4 * lb]) = kc;
      }
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int t = 4 * q + j;
        uint16_t ksc, vsc;
        const uint32_t kc = QuantizeLanesQ4(kx[j], lb, &ksc);
        vc[j] = QuantizeLanesQ4(vx[j], lb, &vsc);
        if (t < t_lo || t >= t_hi) continue;
        if (lb == 0) lks[t * NB + b] = ksc, lvs[b * PT + t] = vsc;
        if (lb < 4) *reinterpret_cast<uint32_t*>(&lk[(b * PT + t) * KB + 4 * lb]) = kc;
      }
    }
    if (FMT == 8 || lb < 4) {
      const int r0 = FMT == 8 ? d0 : b * 16 + 4 * lb;  // this lane's four byte rows of the V image
#pragma unroll
      for (int e = 0; e < 4; ++e)
        *reinterpret_cast<uint32_t*>(&lv[(r0 + e) * (PT + 4) + 4 * q]) =
            ((vc[0] >> (8 * e)) & 0xFF) | (((vc[1] >> (8 * e)) & 0xFF) << 8) | (((vc[2] >> (8 * e)) & 0xFF) << 16) |
            (((vc[3] >> (8 * e)) & 0xFF) << 24);
    }
  }
  __syncthreads();
  // ---- the images' written parts to the pools
  const size_t ph = size_t(page) * H + h;
  const int n_t = t_hi - t_lo, tid = threadIdx.x, NT = 64 * kPageWaves;
  const int lg_pt = __builtin_ctz(static_cast<unsigned>(PT));  // pages are 16, 32 or 64 tokens
  if (!a.skip_k) {  // K codes: per block the tokens' pieces are contiguous
    uint8_t* dst = a.pools.kq + ph * (size_t(NB) * PT * KB);
    if (n_t == PT) {  // a whole page (most of a chunk's): the region as it lies, no division by a run-time value
      for (int u = tid; u < (NB * KB / 16) << lg_pt; u += NT)
        *reinterpret_cast<uint4*>(dst + u * 16) = *reinterpret_cast<const uint4*>(&lk[u * 16]);
    } else {
      const int per_block = n_t * KB / 16;
      for (int u = tid; u < NB * per_block; u += NT) {
        const int off = ((u / per_block) * PT + t_lo) * KB + (u % per_block) * 16;
        *reinterpret_cast<uint4*>(dst + off) = *reinterpret_cast<const uint4*>(&lk[off]);
      }
    }
  }
  if (!a.skip_k) {  // K scales: [token][block], 8 bytes at a time
    uint8_t* dst = reinterpret_cast<uint8_t*>(a.pools.ks) + ph * (size_t(PT) * NB * 2);
    for (int u = tid; u < n_t * NB / 4; u += NT) {
      const int off = t_lo * NB * 2 + u * 8;
      *reinterpret_cast<uint2*>(dst + off) = *reinterpret_cast<const uint2*>(reinterpret_cast<const uint8_t*>(lks) + off);
    }
  }
  uint8_t* vdst = a.pools.vq + ph * (size_t(v_rows) * PT);
  uint16_t* sdst = a.pools.vs + ph * (size_t(NB) * PT);
  if (n_t == PT) {  // a whole page: both V regions are contiguous
    for (int u = tid; u < (v_rows << lg_pt) / 16; u += NT) {
      const uint32_t* src = reinterpret_cast<const uint32_t*>(&lv[((u * 16) >> lg_pt) * (PT + 4) + ((u * 16) & (PT - 1))]);
      *reinterpret_cast<uint4*>(vdst + u * 16) = uint4{src[0], src[1], src[2], src[3]};
    }
    for (int u = tid; u < NB * PT / 8; u += NT)
      *reinterpret_cast<uint4*>(sdst + u * 8) = *reinterpret_cast<const uint4*>(&lvs[u * 8]);
  } else {  // the chunk's first or last page: the tokens' bytes of every row
    for (int u = tid; u < v_rows * n_t; u += NT) {
      const int r = u / n_t, t = t_lo + u % n_t;
      vdst[r * PT + t] = lv[r * (PT + 4) + t];
    }
    for (int u = tid; u < NB * n_t; u += NT) {
      const int off = (u / n_t) * PT + t_lo + u % n_t;
      sdst[off] = lvs[off];
    }
  }
}

// One thread per (K|V, token, kv head, block): the block back in ggml order (scale, then codes).
template <int FMT>
__global__ __launch_bounds__(256) void GatherBlocks(Geom g, Pools pools, const int32_t* table_row, int n_tokens,
                                                     uint8_t* dst_k, uint8_t* dst_v) {
  const int NB = g.nb(), H = g.n_kv, PT = g.pt;
  constexpr int CB = FMT == 8 ? 32 : 16;
  const int64_t per_side = int64_t(n_tokens) * H * NB;
  const int64_t idx = int64_t(blockIdx.x) * blockDim.x + threadIdx.x;
  if (idx >= 2 * per_side) return;
  const bool is_v = idx >= per_side;
  int64_t r = is_v ? idx - per_side : idx;
  const int b = int(r % NB);
  r /= NB;
  const int h = int(r % H);
  const int p = int(r / H);
  const int page = ClampPage(table_row[p / PT], g.n_pages);
  const int t = p % PT;
  const size_t ph = size_t(page) * H + h;
  uint8_t* out = (is_v ? dst_v : dst_k) + ((size_t(p) * H + h) * NB + b) * (CB + 2);
  uint16_t hd;
  if (!is_v) {
    hd = pools.ks[(ph * PT + t) * NB + b];
    const uint8_t* src = pools.kq + ((ph * NB + b) * PT + t) * CB;
    for (int j = 0; j < CB; ++j) out[2 + j] = src[j];
  } else {
    hd = pools.vs[(ph * NB + b) * PT + t];
    const uint8_t* src = pools.vq + (ph * NB + b) * CB * PT + t;
    for (int j = 0; j < CB; ++j) out[2 + j] = src[size_t(j) * PT];
  }
  out[0] = static_cast<uint8_t>(hd & 0xFF);
  out[1] = static_cast<uint8_t>(hd >> 8);
}

}  // namespace
}  // namespace yahkv

using namespace yahkv;

namespace {
int CheckAppend(const yahkv_geometry* g, const yahkv_pools* pools, const int32_t* page_table,
                int32_t page_table_stride, const int32_t* start_pos, int32_t n_seqs, int32_t n_new, const void* k_src,
                const void* v_src, int32_t src_dtype) {
  if (const int st = CheckPools(g, pools)) return st;
  if (page_table == nullptr || start_pos == nullptr || k_src == nullptr || v_src == nullptr) return YAHKV_ERR_ARG;
  if (n_seqs <= 0 || n_new <= 0 || page_table_stride <= 0) return YAHKV_ERR_ARG;
  if (src_dtype != YAHKV_F32 && src_dtype != YAHKV_F16 && src_dtype != YAHKV_BF16) return YAHKV_ERR_ARG;
  if ((reinterpret_cast<uintptr_t>(k_src) | reinterpret_cast<uintptr_t>(v_src)) & 15) return YAHKV_ERR_ARG;
  if (int64_t(n_seqs) * n_new > 0x7FFFFFFF) return YAHKV_ERR_SHAPE;
  return YAHKV_OK;
}
}  // namespace

namespace {
// AppendRows for the pools' format and the source rows' type (the kernel is compiled for each pair)
// AppendPages likewise: one workgroup per (page the chunk touches, kv head, sequence)
template <bool TURN, int D>
void LaunchPagesOf(int32_t format, int32_t src_dtype, dim3 grid, hipStream_t st, const RopeArgs& a) {
  const dim3 block(64 * kPageWaves);
  if (format == YAHKV_Q8_0) {
    if (src_dtype == YAHKV_F32) hipLaunchKernelGGL((AppendPages<8, YAHKV_F32, TURN, D>), grid, block, 0, st, a);
    else if (src_dtype == YAHKV_F16) hipLaunchKernelGGL((AppendPages<8, YAHKV_F16, TURN, D>), grid, block, 0, st, a);
    else hipLaunchKernelGGL((AppendPages<8, YAHKV_BF16, TURN, D>), grid, block, 0, st, a);
  } else {
    if (src_dtype == YAHKV_F32) hipLaunchKernelGGL((AppendPages<4, YAHKV_F32, TURN, D>), grid, block, 0, st, a);
    else if (src_dtype == YAHKV_F16) hipLaunchKernelGGL((AppendPages<4, YAHKV_F16, TURN, D>), grid, block, 0, st, a);
    else hipLaunchKernelGGL((AppendPages<4, YAHKV_BF16, TURN, D>), grid, block, 0, st, a);
  }
}
template <bool TURN>
void LaunchPages(int32_t format, int32_t src_dtype, int32_t n_seqs, int32_t n_new, hipStream_t st, const RopeArgs& a) {
  const dim3 grid(static_cast<unsigned>((n_new + a.g.pt - 2) / a.g.pt + 1), static_cast<unsigned>(a.g.n_kv),
                  static_cast<unsigned>(n_seqs));
  if (a.g.hd == 256) LaunchPagesOf<TURN, 256>(format, src_dtype, grid, st, a);
  else LaunchPagesOf<TURN, 128>(format, src_dtype, grid, st, a);
}
template <int ROPE, int FLIGHT = kRowsInFlight>
void LaunchRows(int32_t format, int32_t src_dtype, dim3 grid, hipStream_t st, const RopeArgs& a) {
  const dim3 block(64 * kRopeWaves);
  if (format == YAHKV_Q8_0) {
    if (src_dtype == YAHKV_F32) hipLaunchKernelGGL((AppendRows<8, ROPE, YAHKV_F32, FLIGHT>), grid, block, 0, st, a);
    else if (src_dtype == YAHKV_F16) hipLaunchKernelGGL((AppendRows<8, ROPE, YAHKV_F16, FLIGHT>), grid, block, 0, st, a);
    else hipLaunchKernelGGL((AppendRows<8, ROPE, YAHKV_BF16, FLIGHT>), grid, block, 0, st, a);
  } else {
    if (src_dtype == YAHKV_F32) hipLaunchKernelGGL((AppendRows<4, ROPE, YAHKV_F32, FLIGHT>), grid, block, 0, st, a);
    else if (src_dtype == YAHKV_F16) hipLaunchKernelGGL((AppendRows<4, ROPE, YAHKV_F16, FLIGHT>), grid, block, 0, st, a);
    else hipLaunchKernelGGL((AppendRows<4, ROPE, YAHKV_BF16, FLIGHT>), grid, block, 0, st, a);
  }
}
// Rows [n_seqs][n_new][n_kv][D] without gaps.
RowsArgs DenseRows(const RopeArgs& a, const void* data) {
  const int64_t token = int64_t(a.g.n_kv) * a.g.hd;
  return RowsArgs{const_cast<void*>(data), a.src_dtype, a.g.n_kv, token * a.n_new, token, a.g.hd};
}
// The fused forms: K and query rows turned, V as it is.
template <int MODE>
int LaunchTurned(RopeArgs a, hipStream_t st) {
  const Geom& m = a.g;
  const int n_seqs = a.n_seqs, n_new = a.n_new, format = a.g.format, src_dtype = a.src_dtype;
  const int64_t tokens = int64_t(n_seqs) * n_new;
  if (tokens > 0x7FFFFFFF) return YAHKV_ERR_SHAPE;
  if (n_new >= kPageAppendMin && n_seqs <= 65535) {
    // A chunk: V page by page, as the plain append takes it (whole lines from an image of the page, where the
    // token's workgroup would store V's codes byte by byte into the transposed page), K and the query rows by token.
    // The general rotation has K page by page as well, unless the caller wants the rotated rows of every token (those that
    // clamp to a slot another token takes are not visited there), and the query rows by the rows kernel, which has eight
    // dims a lane and several rows a wave where AppendRows has four and one (5 x 1037 tokens of 32 + 8 heads of 128 dims:
    // 101 -> 47 us).
    const bool k_pages = MODE == kGeneral && a.k_out == nullptr;
    RopeArgs v = a;
    v.skip_k = !k_pages;
    if (k_pages) LaunchPages<true>(format, src_dtype, n_seqs, n_new, st, v);
    else LaunchPages<false>(format, src_dtype, n_seqs, n_new, st, v);
    if (const int rc = LaunchStatus()) return rc;
    a.skip_v = 1;
    if constexpr (MODE == kGeneral) {
      if (a.q_src != nullptr) {
        if (const int rc = LaunchRotaryRows(a.rotary, m.hd, a.positions, a.start_pos, a.n_valid, n_seqs, n_new, a.q_rows, a.q_out_rows,
                                            RowsArgs{}, RowsArgs{}, st))
          return rc;
        a.q_src = nullptr;
      }
      if (k_pages) return YAHKV_OK;
    }
  }
  int64_t blocks = tokens;
  if (n_new >= 8 * m.pt) {  // a long chunk: a page's tokens to one XCD (see AppendRows)
    a.per_xcd = ((n_new + 7) / 8 + m.pt - 1) / m.pt * m.pt;
    blocks = int64_t(n_seqs) * 8 * a.per_xcd;
    if (blocks > 0x7FFFFFFF) return YAHKV_ERR_SHAPE;
  }
  if constexpr (MODE == kGeneral) {
    if (blocks < 1024) {
      const int rows = (a.skip_v ? 1 : 2) * m.n_kv + (a.q_src != nullptr ? m.n_q : 0), parts = (rows + kRopeWaves - 1) / kRopeWaves;
      LaunchRows<MODE, 1>(format, src_dtype, dim3(static_cast<unsigned>(blocks), static_cast<unsigned>(parts)), st, a);
      return LaunchStatus();
    }
  }
  LaunchRows<MODE>(format, src_dtype, dim3(static_cast<unsigned>(blocks)), st, a);
  return LaunchStatus();
}
}  // namespace

extern "C" int yahkv_append(const yahkv_geometry* g, const yahkv_pools* pools, const int32_t* page_table,
                            int32_t page_table_stride, const int32_t* start_pos, const int32_t* n_valid,
                            int32_t n_seqs, int32_t n_new, const void* k_src, const void* v_src, int32_t src_dtype,
                            void* stream) {
  if (const int st = CheckAppend(g, pools, page_table, page_table_stride, start_pos, n_seqs, n_new, k_src, v_src,
                                 src_dtype))
    return st;
  RopeArgs a{};
  a.g = MakeGeom(*g), a.pools = MakePools(*pools), a.table = page_table, a.stride = page_table_stride;
  a.start_pos = start_pos, a.n_valid = n_valid, a.n_seqs = n_seqs, a.n_new = n_new, a.k_src = k_src, a.v_src = v_src;
  a.src_dtype = src_dtype, a.rotary_dim = 8, a.theta = 1.0f, a.v_rows = DenseRows(a, v_src);
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (n_new >= kPageAppendMin && n_seqs <= 65535) {  // a chunk: page by page (the grid's z extent is the batch)
    LaunchPages<false>(g->format, src_dtype, n_seqs, n_new, st, a);
    return LaunchStatus();
  }
  const dim3 grid(static_cast<unsigned>(n_seqs) * static_cast<unsigned>(n_new));
  LaunchRows<kAsTheyAre>(g->format, src_dtype, grid, st, a);
  return LaunchStatus();
}

extern "C" int yahkv_append_rope(const yahkv_geometry* g, const yahkv_pools* pools, const int32_t* page_table,
                                 int32_t page_table_stride, const int32_t* start_pos, const int32_t* n_valid,
                                 int32_t n_seqs, int32_t n_new, const void* k_src, const void* v_src,
                                 int32_t src_dtype, const yahkv_rope* rope, const void* q_src, void* q_out,
                                 int32_t q_out_dtype, float* k_out, void* stream) {
  if (const int st = CheckAppend(g, pools, page_table, page_table_stride, start_pos, n_seqs, n_new, k_src, v_src,
                                 src_dtype))
    return st;
  if (rope == nullptr) return YAHKV_ERR_ARG;
  if ((q_src == nullptr) != (q_out == nullptr)) return YAHKV_ERR_ARG;
  if (q_src != nullptr && q_out_dtype != YAHKV_F32 && q_out_dtype != YAHKV_F16 && q_out_dtype != YAHKV_BF16)
    return YAHKV_ERR_ARG;
  const Geom m = MakeGeom(*g);
  if (rope->rotary_dim < 8 || rope->rotary_dim > m.hd || rope->rotary_dim % 8 != 0) return YAHKV_ERR_ARG;
  if (!(rope->theta > 0.0f) || !(rope->eps >= 0.0f)) return YAHKV_ERR_ARG;
  RopeArgs a{};
  a.g = m, a.pools = MakePools(*pools), a.table = page_table, a.stride = page_table_stride, a.start_pos = start_pos;
  a.n_valid = n_valid, a.n_seqs = n_seqs, a.n_new = n_new, a.k_src = k_src, a.v_src = v_src, a.src_dtype = src_dtype;
  a.k_weight = rope->k_weight, a.q_weight = rope->q_weight, a.theta = rope->theta, a.eps = rope->eps;
  a.rotary_dim = rope->rotary_dim, a.q_src = q_src, a.q_out = q_out, a.q_out_dtype = q_out_dtype, a.k_out = k_out;
  a.v_rows = DenseRows(a, v_src);
  return LaunchTurned<kNeox>(a, static_cast<hipStream_t>(stream));
}

extern "C" int yahkv_rotary_append(const yahkv_geometry* g, const yahkv_pools* pools, const int32_t* page_table,
                                   int32_t page_table_stride, const int32_t* start_pos, const int32_t* n_valid,
                                   int32_t n_seqs, int32_t n_new, const yahkv_rotary* rotary, const int32_t* positions,
                                   const yahkv_rows* k, const yahkv_rows* v, const yahkv_rows* q_src,
                                   const yahkv_rows* q_dst, float* k_out, void* stream) {
  if (k == nullptr || v == nullptr) return YAHKV_ERR_ARG;
  if (const int st = CheckAppend(g, pools, page_table, page_table_stride, start_pos, n_seqs, n_new, k->data, v->data, k->dtype))
    return st;
  RopeArgs a{};
  a.g = MakeGeom(*g), a.pools = MakePools(*pools), a.table = page_table, a.stride = page_table_stride;
  if (const int st = CheckRotary(rotary, a.g.hd, &a.rotary)) return st;
  if (const int st = CheckRows(k, &a.k_rows)) return st;
  if (const int st = CheckRows(v, &a.v_rows)) return st;
  if (k->n_heads != g->n_kv_heads || v->n_heads != g->n_kv_heads || v->dtype != k->dtype) return YAHKV_ERR_ARG;
  if ((q_src == nullptr) != (q_dst == nullptr) || !Aligned16(k_out)) return YAHKV_ERR_ARG;
  if (q_src != nullptr) {
    if (const int st = CheckRows(q_src, &a.q_rows)) return st;
    if (const int st = CheckRowsOut(q_dst, n_seqs, n_new, &a.q_out_rows)) return st;
    if (q_src->n_heads != g->n_q_heads || q_dst->n_heads != g->n_q_heads || q_src->dtype != k->dtype) return YAHKV_ERR_ARG;
    a.q_src = q_src->data, a.q_out = q_dst->data, a.q_out_dtype = q_dst->dtype;
  }
  a.start_pos = start_pos, a.n_valid = n_valid, a.n_seqs = n_seqs, a.n_new = n_new, a.src_dtype = k->dtype;
  a.k_src = k->data, a.v_src = v->data, a.k_out = k_out, a.positions = positions;
  a.rotary_dim = a.rotary.rot, a.eps = a.rotary.eps, a.k_weight = a.rotary.k_weight, a.q_weight = a.rotary.q_weight;
  return LaunchTurned<kGeneral>(a, static_cast<hipStream_t>(stream));
}

extern "C" int yahkv_gather_blocks(const yahkv_geometry* g, const yahkv_pools* pools, const int32_t* table_row,
                                   int32_t n_tokens, void* dst_k, void* dst_v, void* stream) {
  if (const int st = CheckPools(g, pools)) return st;
  if (table_row == nullptr || dst_k == nullptr || dst_v == nullptr || n_tokens <= 0) return YAHKV_ERR_ARG;
  const Geom m = MakeGeom(*g);
  const int64_t items = int64_t(2) * n_tokens * m.n_kv * m.nb();
  const unsigned blocks = static_cast<unsigned>((items + 255) / 256);
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (g->format == YAHKV_Q8_0)
    hipLaunchKernelGGL(GatherBlocks<8>, dim3(blocks), dim3(256), 0, st, m, MakePools(*pools), table_row, n_tokens,
                       static_cast<uint8_t*>(dst_k), static_cast<uint8_t*>(dst_v));
  else
    hipLaunchKernelGGL(GatherBlocks<4>, dim3(blocks), dim3(256), 0, st, m, MakePools(*pools), table_row, n_tokens,
                       static_cast<uint8_t*>(dst_k), static_cast<uint8_t*>(dst_v));
  return LaunchStatus();
}
