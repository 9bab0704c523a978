// Eviction: the keys a sequence keeps when it is cut to a budget, and their move to fresh pages.
//
// The choice. Per (sequence, kv head) the kept keys are the first `sink`, the last `recent`, and of those between them the
// m = budget - sink - recent of largest weight, ties to the lowest position. Non-negative floats order as their bits do, so
// the m-th largest is found digit by digit (11, 11 and 9 bits from the top): a histogram of the digit over the keys that
// share the digits found so far, and a scan of its bins from above. What is left after the last digit is the threshold
// itself and how many keys equal to it are kept. The first digit, exponent and three bits, leaves a few percent of the keys,
// which go to a list in LDS for the rest. One workgroup does it all, with the row in its LDS; a thread owns consecutive
// keys, so that the kept positions come out in order from its own count and one scan over the threads. What bounds it is the
// instructions of the one CU that a row has: loops over lanes' own keys with a few instructions a key, not wave-wide votes.
// One 32K row a head, cut to 4K: 20.6 us (5 to load and count, 2.4 the list, 2.5 two digits, 5.3 the places and the way out;
// the rest launch and scans); 32 ragged rows of up to 16K for each of 4 heads: 15.6 us.
//
// The move. A workgroup fills one new page of one kv head. K blocks are contiguous pieces of 32 (or 16) bytes; V lies
// transposed, so that a key is a byte in each of its rows, and any key of a page costs that page's whole V region in lines
// from memory: kept keys spread over all pages mean that all of V is read, whatever the budget. 32 ragged sequences of up to 16K
// cut to 2K, 4 heads of 256 dims: 119 us for 442 MB of lines read and 163 MB written, 5.1 TB/s, a large copy's rate on this
// card (4.85); one of 32K cut to 4K: 15.3 us.
#include "common.hpp"
#include "quant.hpp"

namespace yahkv {
namespace {

struct SelectArgs {
  const int32_t* seq_len;
  const float* weights;
  int32_t max_len, stride, n_kv, budget, sink, recent;
  int32_t* kept;
  int32_t* n_kept;
};

constexpr int kSelectThreads = 1024, kSelectWaves = kSelectThreads / 64;
constexpr int kOwn = 32;                           // keys of a thread at most, consecutive ones, in LDS rows of 33 words
constexpr int kSegment = kOwn * kSelectThreads;    // (all banks in use); longer rows go through LDS segment by segment
constexpr int kBins = 2048, kListed = 4096, kStaged = 2 * kListed;

// Keys as the passes see them, without a question about positions: a weight's bits + 1 (1 .. 0x7F800001), all ones for a
// position that is kept whatever it weighs, 0 for none.
constexpr uint32_t kAlways = 0xFFFFFFFFu;
__device__ __forceinline__ uint32_t WeightKey(float w) { return w > 0.0f ? __builtin_bit_cast(uint32_t, w) + 1u : 1u; }
__device__ __forceinline__ bool Weighed(uint32_t key) { return static_cast<int32_t>(key) > 0; }

__global__ __launch_bounds__(kSelectThreads) void EvictSelect(const SelectArgs a) {
  const int h = blockIdx.x, s = blockIdx.y, tid = threadIdx.x, wave = tid / 64, lane = tid % 64;
  const int len = min(max(a.seq_len[s], 0), a.max_len);
  const size_t row = static_cast<size_t>(s) * a.n_kv + h;
  int32_t* const out = a.kept + row * a.budget;
  if (h == 0 && tid == 0) a.n_kept[s] = min(len, a.budget);
  if (len <= a.budget) {
    for (int i = tid; i < a.budget; i += kSelectThreads) out[i] = i < len ? i : -1;
    return;
  }
  const float* const w = a.weights + row * a.stride;
  const int lo = a.sink, hi = len - a.recent;  // the keys that are weighed: [lo, hi)

  __shared__ uint32_t keys[kSelectThreads * (kOwn + 1)];
  __shared__ uint32_t bins[kBins];
  __shared__ union {
    uint32_t list[kListed];    // the keys that share the threshold's first digit, in any order
    uint16_t staged[kStaged];  // kept positions on their way out, within the segment
  } shared;
  auto& list = shared.list;
  auto& staged = shared.staged;
  __shared__ uint32_t totals[kSelectWaves];
  __shared__ uint32_t found[3];       // the digit, how many of the keys that share it are kept, and how many there are
  __shared__ int list_n;
  const int n_segments = (len + kSegment - 1) / kSegment;
  int lg_own = 3;                     // a thread owns 2^lg_own consecutive keys of a segment
  while ((kSelectThreads << lg_own) < min(len, kSegment)) ++lg_own;
  const int own = 1 << lg_own;
  int loaded = -1;
  auto load_and = [&](int seg, auto also) {  // (a barrier on either side; nothing if it is there already); also(key) for each
    if (seg == loaded) return;
    __syncthreads();
    const int base = seg * kSegment, n = min(len - base, kSegment);
    const float* const from = w + base;
    auto put = [&](int e, float v) {
      const int t = base + e;
      const uint32_t key = t >= len ? 0u : t < lo || t >= hi ? kAlways : WeightKey(v);
      keys[(e >> lg_own) * (kOwn + 1) + (e & (own - 1))] = key;
      also(key);
    };
    const int n4 = (reinterpret_cast<uintptr_t>(from) & 15) == 0 ? n & ~3 : 0;
#pragma unroll 8
    for (int e = 4 * tid; e < n4; e += 4 * kSelectThreads) {
      const float4 v = *reinterpret_cast<const float4*>(from + e);
      put(e, v.x), put(e + 1, v.y), put(e + 2, v.z), put(e + 3, v.w);
    }
    for (int e = n4 + tid; e < own * kSelectThreads; e += kSelectThreads) put(e, from[min(e, n - 1)]);
    loaded = seg;
    __syncthreads();
  };
  auto load = [&](int seg) { load_and(seg, [](uint32_t) {}); };
  auto each = [&](auto f) {  // f(key, its place among this thread's keys of the segment), in order
    for (int j0 = 0; j0 < own; j0 += 8) {
      uint32_t k[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) k[j] = keys[tid * (kOwn + 1) + j0 + j];
#pragma unroll
      for (int j = 0; j < 8; ++j) f(k[j], j0 + j);
    }
  };
  // exclusive sum over the threads before this one, and the sum of all
  auto scan = [&](uint32_t v, uint32_t* all) -> uint32_t {
    uint32_t incl = v;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const uint32_t x = __shfl_up(incl, o, 64);
      if (lane >= o) incl += x;
    }
    __syncthreads();  // (the totals of the scan before have been read)
    if (lane == 63) totals[wave] = incl;
    __syncthreads();
    uint32_t before = incl - v, sum = 0;
#pragma unroll
    for (int i = 0; i < kSelectWaves; ++i) {
      before += i < wave ? totals[i] : 0u;
      sum += totals[i];
    }
    *all = sum;
    return before;
  };

  uint32_t prefix = 0, mask = 0;
  uint32_t take = static_cast<uint32_t>(a.budget - a.sink - a.recent);  // of the keys that agree with `prefix` so far
  const bool any = take > 0;
  auto clear_bins = [&]() {
    __syncthreads();
    for (int i = tid; i < kBins; i += kSelectThreads) bins[i] = 0u;
    __syncthreads();
  };
  auto find_digit = [&](int shift, uint32_t digits) {  // the bins from the top: thread i takes 2047 - 2 i and 2046 - 2 i
    __syncthreads();
    const uint32_t c0 = bins[kBins - 1 - 2 * tid], c1 = bins[kBins - 2 - 2 * tid];
    uint32_t all;
    const uint32_t above = scan(c0 + c1, &all);
    if (above < take && above + c0 + c1 >= take) {  // one thread: the digit is in its bins
      const bool first = above + c0 >= take;
      found[0] = static_cast<uint32_t>(kBins - (first ? 1 : 2) - 2 * tid);
      found[1] = first ? take - above : take - above - c0;
      found[2] = first ? c0 : c1;
    }
    __syncthreads();
    prefix |= found[0] << shift, mask |= digits << shift, take = found[1];
  };
  if (any) {  // (the sign bit is never set: eleven bits from bit 30 down)
    if (tid == 0) list_n = 0;
    clear_bins();
    for (int seg = 0; seg < n_segments; ++seg)  // (counted on their way in)
      load_and(seg, [&](uint32_t key) {
        if (Weighed(key)) atomicAdd(&bins[key >> 20], 1u);
      });
    find_digit(20, 2047u);
    const bool listed = found[2] <= static_cast<uint32_t>(kListed);
    const uint32_t top = prefix, top_mask = mask;
    if (listed) {
      for (int seg = 0; seg < n_segments; ++seg) {
        load(seg);
        each([&](uint32_t key, int) {
          if (Weighed(key) & ((key & top_mask) == top)) list[atomicAdd(&list_n, 1)] = key;
        });
      }
    }
    for (int pass = 1; pass < 3; ++pass) {
      const int shift = pass == 1 ? 9 : 0;
      const uint32_t digits = pass == 1 ? 2047u : 511u;
      clear_bins();
      auto count = [&](uint32_t key) {
        if ((key & mask) == prefix) atomicAdd(&bins[(key >> shift) & digits], 1u);
      };
      if (listed) {
        const int n = list_n;
        for (int i = tid; i < n; i += kSelectThreads) count(list[i]);
      } else {  // too many for the list (equal weights): over all keys again
        for (int seg = 0; seg < n_segments; ++seg) {
          load(seg);
          each([&](uint32_t key, int) {
            if (Weighed(key)) count(key);
          });
        }
      }
      find_digit(shift, digits);
    }
  }
  // Kept: keys above the threshold, and the first `take` of those equal to it (if nothing is to be taken, what is kept
  // whatever it weighs). Counts of both in one word: a segment has 32768 keys at most.
  if (!any) prefix = kAlways - 1;
  uint32_t sure_before = 0, equal_before = 0;
  for (int seg = 0; seg < n_segments; ++seg) {
    load(seg);
    uint32_t mine = 0;
    each([&](uint32_t key, int) { mine += (key > prefix ? 1u : 0u) + (key == prefix ? 0x10000u : 0u); });
    uint32_t all;
    const uint32_t before = scan(mine, &all);
    // to their places by way of LDS, 8192 at a time: a thread's own are a few, far apart in time and in memory
    const uint32_t sure0 = sure_before + (before & 0xFFFFu), equal0 = equal_before + (before >> 16);
    const uint32_t first = sure_before + min(equal_before, take);
    const uint32_t last = sure_before + (all & 0xFFFFu) + min(equal_before + (all >> 16), take);
    for (uint32_t from = first; from < last; from += kStaged) {
      uint32_t sure = sure0, equal = equal0;
      each([&](uint32_t key, int j) {
        const bool above = key > prefix, same = key == prefix;
        const uint32_t at = sure + min(equal, take) - from;
        if ((above | (same & (equal < take))) & (at < static_cast<uint32_t>(kStaged)))
          staged[at] = static_cast<uint16_t>((tid << lg_own) + j);
        sure += above, equal += same;
      });
      __syncthreads();
      for (uint32_t i = tid; i < min(last - from, static_cast<uint32_t>(kStaged)); i += kSelectThreads)
        out[from + i] = seg * kSegment + staged[i];
      __syncthreads();
    }
    sure_before += all & 0xFFFFu, equal_before += all >> 16;
  }
}

struct CompactArgs {
  Geom g;
  Pools pools;
  const int32_t* table;
  const int32_t* kept;
  const int32_t* n_kept;
  const int32_t* dst_table;
  const float* w_in;
  float* w_out;
  int32_t stride, budget, dst_stride, w_in_stride, w_out_stride;
};

// Bytes b0 .. b3 of four rows, one slot a lane (byte e of `v` is row e's), become four slots of one row: lane 4 m + k of the
// wave gets row k's slots 4 m .. 4 m + 3.
__device__ __forceinline__ uint32_t TransposeQuad(uint32_t v, int lane) {
  const uint32_t sel = 0x0c0c0c00u | static_cast<uint32_t>(lane & 3);  // byte k of a lane's word, zeros above
  uint32_t r = 0;
  r |= __builtin_amdgcn_perm(0u, static_cast<uint32_t>(DppI<0x00>(static_cast<int>(v))), sel);
  r |= __builtin_amdgcn_perm(0u, static_cast<uint32_t>(DppI<0x55>(static_cast<int>(v))), sel) << 8;
  r |= __builtin_amdgcn_perm(0u, static_cast<uint32_t>(DppI<0xAA>(static_cast<int>(v))), sel) << 16;
  r |= __builtin_amdgcn_perm(0u, static_cast<uint32_t>(DppI<0xFF>(static_cast<int>(v))), sel) << 24;
  return r;
}

constexpr int kCompactThreads = 256;
template <int FMT, int D, int PT>
__global__ __launch_bounds__(kCompactThreads) void EvictCompact(const CompactArgs a) {
  constexpr int NB = D / 32, KB = FMT == 8 ? 32 : 16, VR = FMT == 8 ? D : NB * 16;
  const Geom g = a.g;
  const int H = g.n_kv, h = blockIdx.y, s = blockIdx.z, tid = threadIdx.x, lane = tid % 64, wave = tid / 64;
  // New pages that follow each other draw on the same old ones at their seam: an XCD takes a stretch of them.
  const int per_xcd = gridDim.x / 8, page_i = static_cast<int>(blockIdx.x) < 8 * per_xcd
                                                 ? static_cast<int>(blockIdx.x % 8) * per_xcd + static_cast<int>(blockIdx.x / 8)
                                                 : static_cast<int>(blockIdx.x);
  const int n_t = min(min(max(a.n_kept[s], 0), a.budget) - page_i * PT, PT);  // live slots of this page
  if (n_t <= 0) return;
  const size_t row = static_cast<size_t>(s) * H + h;
  __shared__ int src_ph[PT], src_slot[PT];  // (page, kv head) and slot of each slot's key (of the last live one's behind it)
  if (tid < PT) {
    const int i = page_i * PT + min(tid, n_t - 1);
    const int t = min(max(a.kept[row * a.budget + i], 0), a.stride * PT - 1);
    src_ph[tid] = ClampPage(a.table[static_cast<int64_t>(s) * a.stride + t / PT], g.n_pages) * H + h;
    src_slot[tid] = t % PT;
    if (a.w_out != nullptr && tid < n_t) a.w_out[row * a.w_out_stride + i] = a.w_in[row * a.w_in_stride + min(t, a.w_in_stride - 1)];
  }
  __syncthreads();
  const int dst_page = ClampPage(a.dst_table[static_cast<int64_t>(s) * a.dst_stride + page_i], g.n_pages);
  const size_t dph = static_cast<size_t>(dst_page) * H + h;
  // K, asked for before V and stored after V's first loads are asked for: codes 16 bytes at a time, scales four blocks at a
  // time. (Where a thread has two pieces or more the compiler keeps them in scratch memory on the way, and reading them back
  // waits for V's first loads as well.)
  constexpr int KP = NB * PT * (KB / 16), KN = (KP + kCompactThreads - 1) / kCompactThreads;
  uint4 kc[KN];
  auto k_place = [&](int u, int* t) -> int {  // offset of piece u behind its token's place, pieces of a block by token
    *t = u / (KB / 16) % PT;
    return u / (KB / 16) / PT * (PT * KB) + u % (KB / 16) * 16;
  };
#pragma unroll
  for (int j = 0; j < KN; ++j) {
    int t;
    const int u = min(tid + kCompactThreads * j, KP - 1), off = k_place(u, &t);
    kc[j] = *reinterpret_cast<const uint4*>(a.pools.kq + static_cast<size_t>(src_ph[t]) * (NB * PT * KB) + (off + src_slot[t] * KB));
  }
  // V: a wave takes four groups of 64 / PT rows at a time, lane = (row, slot): a load is one byte of every slot's key, the
  // bytes of a row come from as few lines as its keys' pages are; four of them are put together to dwords of a row.
  constexpr int RPL = 64 / PT, STEP = 4 * RPL, VB = 4;  // rows of a load and of a store; stores' rows in flight
  const int slot = lane % PT, sub = lane / PT;
  const uint8_t* vsrc = a.pools.vq + static_cast<size_t>(src_ph[slot]) * (VR * PT) + src_slot[slot];
  uint8_t* vdst = a.pools.vq + dph * (VR * PT);
  constexpr int PER_WAVE = VR / (kCompactThreads / 64);
  static_assert(PER_WAVE % (STEP * VB) == 0 || STEP * VB > PER_WAVE, "a wave's rows");
  constexpr int BATCH = STEP * VB > PER_WAVE ? PER_WAVE / STEP : VB;
  bool k_stored = false;
  for (int r0 = wave * PER_WAVE; r0 < (wave + 1) * PER_WAVE; r0 += STEP * BATCH) {
    uint32_t b[BATCH][4];
#pragma unroll
    for (int j = 0; j < BATCH; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) b[j][e] = vsrc[(r0 + STEP * j + RPL * e + sub) * PT];
    if (!k_stored) {
      k_stored = true;
#pragma unroll
      for (int j = 0; j < KN; ++j) {
        int t;
        const int u = tid + kCompactThreads * j, off = k_place(u, &t);
        if (u < KP && t < n_t) *reinterpret_cast<uint4*>(a.pools.kq + dph * (NB * PT * KB) + (off + t * KB)) = kc[j];
      }
    }
#pragma unroll
    for (int j = 0; j < BATCH; ++j) {
      const uint32_t w = TransposeQuad(b[j][0] | b[j][1] << 8 | b[j][2] << 16 | b[j][3] << 24, lane);
      // this lane now has slots slot / 4 * 4 .. + 3 of row r0 + STEP j + RPL (lane % 4) + sub
      uint8_t* dst = vdst + (r0 + STEP * j + RPL * (lane & 3) + sub) * PT + (slot & ~3);
      const int n = n_t - (slot & ~3);
      if (n >= 4) *reinterpret_cast<uint32_t*>(dst) = w;
      else
        for (int e = 0; e < n; ++e) dst[e] = static_cast<uint8_t>(w >> (8 * e));
    }
  }
  for (int u = tid; u < PT * (NB / 4); u += kCompactThreads) {
    const int t = u / (NB / 4), blk = u % (NB / 4) * 4;
    if (t < n_t)
      *reinterpret_cast<uint2*>(a.pools.ks + (dph * PT + t) * NB + blk) =
          *reinterpret_cast<const uint2*>(a.pools.ks + (static_cast<size_t>(src_ph[t]) * PT + src_slot[t]) * NB + blk);
  }
  for (int u = tid; u < NB * PT; u += kCompactThreads) {  // V scales
    const int blk = u / PT, t = u % PT;
    if (t < n_t) a.pools.vs[(dph * NB + blk) * PT + t] = a.pools.vs[(static_cast<size_t>(src_ph[t]) * NB + blk) * PT + src_slot[t]];
  }
}

template <int FMT>
void LaunchCompact(const CompactArgs& a, dim3 grid, hipStream_t st) {
  const dim3 block(kCompactThreads);
  if (a.g.hd == 256 && a.g.pt == 64) hipLaunchKernelGGL((EvictCompact<FMT, 256, 64>), grid, block, 0, st, a);
  else if (a.g.hd == 256 && a.g.pt == 32) hipLaunchKernelGGL((EvictCompact<FMT, 256, 32>), grid, block, 0, st, a);
  else if (a.g.hd == 256) hipLaunchKernelGGL((EvictCompact<FMT, 256, 16>), grid, block, 0, st, a);
  else if (a.g.pt == 64) hipLaunchKernelGGL((EvictCompact<FMT, 128, 64>), grid, block, 0, st, a);
  else if (a.g.pt == 32) hipLaunchKernelGGL((EvictCompact<FMT, 128, 32>), grid, block, 0, st, a);
  else hipLaunchKernelGGL((EvictCompact<FMT, 128, 16>), grid, block, 0, st, a);
}

}  // namespace
}  // namespace yahkv

using namespace yahkv;

extern "C" int yahkv_evict_select(const yahkv_geometry* g, const int32_t* seq_len, int32_t n_seqs, int32_t max_seq_len,
                                  const float* weights, int32_t weights_stride, int32_t budget, int32_t sink,
                                  int32_t recent, int32_t* kept, int32_t* n_kept, void* stream) {
  if (const int st = CheckGeometry(g)) return st;
  if (seq_len == nullptr || weights == nullptr || kept == nullptr || n_kept == nullptr) return YAHKV_ERR_ARG;
  if (n_seqs <= 0 || max_seq_len <= 0 || weights_stride < max_seq_len || budget <= 0) return YAHKV_ERR_ARG;
  if (sink < 0 || recent < 0 || int64_t(sink) + recent > budget) return YAHKV_ERR_ARG;
  if (n_seqs > 65535 || max_seq_len > (1 << 30)) return YAHKV_ERR_SHAPE;
  const SelectArgs a{seq_len, weights, max_seq_len, weights_stride, g->n_kv_heads, budget, sink, recent, kept, n_kept};
  const dim3 grid(static_cast<unsigned>(g->n_kv_heads), static_cast<unsigned>(n_seqs));
  hipStream_t st = static_cast<hipStream_t>(stream);
  hipLaunchKernelGGL(EvictSelect, grid, dim3(kSelectThreads), 0, st, a);
  return LaunchStatus();
}

extern "C" int yahkv_evict_compact(const yahkv_geometry* g, const yahkv_pools* pools, const int32_t* page_table,
                                   int32_t page_table_stride, const int32_t* kept, const int32_t* n_kept, int32_t n_seqs,
                                   int32_t budget, const int32_t* dst_table, int32_t dst_table_stride,
                                   const float* weights_in, int32_t weights_in_stride, float* weights_out,
                                   int32_t weights_out_stride, void* stream) {
  if (const int st = CheckPools(g, pools)) return st;
  if (page_table == nullptr || kept == nullptr || n_kept == nullptr || dst_table == nullptr) return YAHKV_ERR_ARG;
  if (n_seqs <= 0 || budget <= 0 || page_table_stride <= 0) return YAHKV_ERR_ARG;
  const int pages = (budget - 1) / g->page_tokens + 1;
  if (dst_table_stride < pages || dst_table == page_table) return YAHKV_ERR_ARG;
  if ((weights_in == nullptr) != (weights_out == nullptr)) return YAHKV_ERR_ARG;
  if (weights_in != nullptr && (weights_in_stride <= 0 || weights_out_stride < budget || weights_in == weights_out)) return YAHKV_ERR_ARG;
  if (n_seqs > 65535 || g->n_kv_heads > 65535 || int64_t(page_table_stride) * g->page_tokens > 0x7FFFFFFF) return YAHKV_ERR_SHAPE;
  const CompactArgs a{MakeGeom(*g), MakePools(*pools), page_table, kept, n_kept, dst_table, weights_in, weights_out,
                      page_table_stride, budget, dst_table_stride, weights_in_stride, weights_out_stride};
  const dim3 grid(static_cast<unsigned>(pages), static_cast<unsigned>(g->n_kv_heads), static_cast<unsigned>(n_seqs));
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (g->format == YAHKV_Q8_0) LaunchCompact<8>(a, grid, st);
  else LaunchCompact<4>(a, grid, st);
  return LaunchStatus();
}
