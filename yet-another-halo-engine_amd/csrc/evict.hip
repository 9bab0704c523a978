// Eviction: the keys a sequence keeps when it is cut to a budget, and their move to fresh pages.
//
// The choice. Per (sequence, kv head) the kept keys are the first `sink`, the last `recent`, and of those between them the
// m = budget - sink - recent of largest weight, ties to the lowest position. Non-negative floats order as their bits do, so
// the m-th largest is found digit by digit (11, 11 and 10 bits from the top): a histogram of the digit over the keys that
// share the digits found so far, and a scan of its bins from above. What is left after the last digit is the threshold
// itself and how many keys equal to it are kept. One workgroup does it all; its sixteen waves own sixteen consecutive
// stretches of the row, so that the kept positions come out in order from ballots and one scan over the waves.
//
// The move. A workgroup fills one new page of one kv head. K blocks are contiguous pieces of 32 (or 16) bytes; V lies
// transposed, so that a key is a byte in each of its rows: four neighbouring slots' bytes are put together into a dword.
#include "common.hpp"

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
constexpr int kBins = 2048;
constexpr int kHeld = 32;  // keys a thread keeps in registers: rows up to 32768 keys are read once

__device__ __forceinline__ uint32_t WeightKey(float w) { return w > 0.0f ? __builtin_bit_cast(uint32_t, w) : 0u; }

template <bool HELD>
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
  // wave w owns positions [w * span, w * span + span), 64 at a time
  const int steps = (len + kSelectThreads - 1) / kSelectThreads, t0 = wave * steps * 64 + lane;
  uint32_t held[HELD ? kHeld : 1];
  if constexpr (HELD) {
#pragma unroll
    for (int j = 0; j < kHeld; ++j) {
      const int t = t0 + 64 * j;
      held[j] = j < steps && t < len ? WeightKey(w[t]) : 0u;
    }
  }
  auto each = [&](auto f) {  // f(position, its key, whether it is weighed), for this lane's positions in order
    if constexpr (HELD) {
#pragma unroll
      for (int j = 0; j < kHeld; ++j)
        if (j < steps) {
          const int t = t0 + 64 * j;
          f(t, held[j], t >= lo && t < hi);
        }
    } else {
      for (int j = 0; j < steps; ++j) {
        const int t = t0 + 64 * j;
        f(t, t < len ? WeightKey(w[t]) : 0u, t >= lo && t < hi);
      }
    }
  };

  __shared__ uint32_t bins[kBins];
  __shared__ int totals[kSelectWaves][2];
  __shared__ uint32_t found[2];  // the digit, and how many of the keys that share it are kept
  uint32_t prefix = 0, mask = 0;
  int take = a.budget - a.sink - a.recent;  // of the keys that agree with `prefix` so far
  if (take > 0) {
    for (int pass = 0; pass < 3; ++pass) {
      const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
      const uint32_t digits = pass == 2 ? 1023u : 2047u;
      for (int i = tid; i < kBins; i += kSelectThreads) bins[i] = 0u;
      __syncthreads();
      each([&](int, uint32_t key, bool weighed) {
        if (weighed && (key & mask) == prefix) atomicAdd(&bins[(key >> shift) & digits], 1u);
      });
      __syncthreads();
      // from the top: thread i takes bins 2047 - 2 i and 2046 - 2 i
      const int c0 = static_cast<int>(bins[kBins - 1 - 2 * tid]), c1 = static_cast<int>(bins[kBins - 2 - 2 * tid]);
      int incl = c0 + c1;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const int v = __shfl_up(incl, o, 64);
        if (lane >= o) incl += v;
      }
      if (lane == 63) totals[wave][0] = incl;
      __syncthreads();
      int above = incl - c0 - c1;
      for (int v = 0; v < wave; ++v) above += totals[v][0];
      if (above < take && above + c0 + c1 >= take) {  // one thread: the digit is in its bins
        const bool first = above + c0 >= take;
        found[0] = static_cast<uint32_t>(kBins - (first ? 1 : 2) - 2 * tid);
        found[1] = static_cast<uint32_t>(first ? take - above : take - above - c0);
      }
      __syncthreads();
      prefix |= found[0] << shift, mask |= digits << shift, take = static_cast<int>(found[1]);
      __syncthreads();
    }
  }
  // kept: what is not weighed, keys above the threshold, and the first `take` of those equal to it (none if nothing is
  // to be taken: then no key is above it either)
  const bool any = a.budget > a.sink + a.recent;
  auto above_it = [&](uint32_t key, bool weighed) { return weighed && any && key > prefix; };
  auto equal_it = [&](uint32_t key, bool weighed) { return weighed && any && key == prefix; };
  int sure = 0, equal = 0;
  each([&](int t, uint32_t key, bool weighed) {
    sure += __popcll(__ballot(t < len && (!weighed || above_it(key, weighed))));
    equal += __popcll(__ballot(equal_it(key, weighed)));
  });
  if (lane == 0) totals[wave][0] = sure, totals[wave][1] = equal;
  __syncthreads();
  int at = 0, eq_before = 0;
  for (int v = 0; v < wave; ++v) {
    at += totals[v][0] + min(max(take - eq_before, 0), totals[v][1]);
    eq_before += totals[v][1];
  }
  const unsigned long long below = (1ull << lane) - 1;
  each([&](int t, uint32_t key, bool weighed) {
    const unsigned long long eq = __ballot(equal_it(key, weighed));
    const bool keep = t < len && (!weighed || above_it(key, weighed) ||
                                  (equal_it(key, weighed) && eq_before + static_cast<int>(__popcll(eq & below)) < take));
    const unsigned long long keeps = __ballot(keep);
    if (keep) out[at + __popcll(keeps & below)] = t;
    at += __popcll(keeps), eq_before += __popcll(eq);
  });
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

template <int FMT>
__global__ __launch_bounds__(256) void EvictCompact(const CompactArgs a) {
  const Geom g = a.g;
  const int PT = g.pt, NB = g.nb(), H = g.n_kv, page_i = blockIdx.x, h = blockIdx.y, s = blockIdx.z, tid = threadIdx.x;
  constexpr int KB = FMT == 8 ? 32 : 16;
  const int n_t = min(min(max(a.n_kept[s], 0), a.budget) - page_i * PT, PT);  // live slots of this page
  if (n_t <= 0) return;
  const size_t row = static_cast<size_t>(s) * H + h;
  __shared__ int src_ph[64], src_slot[64];  // (page, kv head) and slot of each live slot's key
  if (tid < n_t) {
    const int t = min(max(a.kept[row * a.budget + page_i * PT + tid], 0), a.stride * PT - 1);
    src_ph[tid] = ClampPage(a.table[static_cast<int64_t>(s) * a.stride + t / PT], g.n_pages) * H + h;
    src_slot[tid] = t % PT;
    if (a.w_out != nullptr)
      a.w_out[row * a.w_out_stride + page_i * PT + tid] = a.w_in[row * a.w_in_stride + min(t, a.w_in_stride - 1)];
  }
  __syncthreads();
  const int dst_page = ClampPage(a.dst_table[static_cast<int64_t>(s) * a.dst_stride + page_i], g.n_pages);
  const size_t dph = static_cast<size_t>(dst_page) * H + h;
  for (int u = tid; u < NB * n_t * (KB / 16); u += 256) {  // K codes, 16 bytes at a time
    const int piece = u % (KB / 16), t = (u / (KB / 16)) % n_t, b = u / (KB / 16) / n_t;
    *reinterpret_cast<uint4*>(a.pools.kq + ((dph * NB + b) * PT + t) * KB + 16 * piece) = *reinterpret_cast<const uint4*>(
        a.pools.kq + ((static_cast<size_t>(src_ph[t]) * NB + b) * PT + src_slot[t]) * KB + 16 * piece);
  }
  for (int u = tid; u < n_t * NB / 4; u += 256) {  // K scales, four blocks at a time
    const int t = u / (NB / 4), b = u % (NB / 4) * 4;
    *reinterpret_cast<uint2*>(a.pools.ks + (dph * PT + t) * NB + b) = *reinterpret_cast<const uint2*>(
        a.pools.ks + (static_cast<size_t>(src_ph[t]) * PT + src_slot[t]) * NB + b);
  }
  const int v_rows = FMT == 8 ? g.hd : NB * 16;
  for (int u = tid; u < v_rows * (PT / 4); u += 256) {  // V codes: four slots of a row
    const int r = u / (PT / 4), t = u % (PT / 4) * 4, n = min(n_t - t, 4);
    if (n <= 0) continue;
    uint8_t* dst = a.pools.vq + (dph * v_rows + r) * PT + t;
    uint32_t v = 0;
    for (int j = 0; j < n; ++j)
      v |= static_cast<uint32_t>(a.pools.vq[(static_cast<size_t>(src_ph[t + j]) * v_rows + r) * PT + src_slot[t + j]]) << (8 * j);
    if (n == 4) *reinterpret_cast<uint32_t*>(dst) = v;
    else
      for (int j = 0; j < n; ++j) dst[j] = static_cast<uint8_t>(v >> (8 * j));
  }
  for (int u = tid; u < NB * n_t; u += 256) {  // V scales
    const int b = u / n_t, t = u % n_t;
    a.pools.vs[(dph * NB + b) * PT + t] = a.pools.vs[(static_cast<size_t>(src_ph[t]) * NB + b) * PT + src_slot[t]];
  }
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
  if (max_seq_len <= kHeld * kSelectThreads) hipLaunchKernelGGL(EvictSelect<true>, grid, dim3(kSelectThreads), 0, st, a);
  else hipLaunchKernelGGL(EvictSelect<false>, grid, dim3(kSelectThreads), 0, st, a);
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
  if (g->format == YAHKV_Q8_0) hipLaunchKernelGGL(EvictCompact<8>, grid, dim3(256), 0, st, a);
  else hipLaunchKernelGGL(EvictCompact<4>, grid, dim3(256), 0, st, a);
  return LaunchStatus();
}
