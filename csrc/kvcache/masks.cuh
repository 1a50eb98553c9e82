// Which keys a query of the cache attention sees, and which pages a tile of queries reads.
#pragma once
#include "../common/ptx.cuh"
#include "kvcache.h"

namespace ddb {

// A query at position `pos` sees keys [0, sinks) and [lo, hi); never one at or behind hi.
struct KvSpan {
  int lo, hi;
};

__device__ __forceinline__ KvSpan kv_span(const KvAttendArgs& a, int pos, int len, int first) {
  KvSpan s;
  const int frame = a.unit == 1 ? pos : pos / a.unit;
  s.hi = a.causal ? min(len, (frame + 1) * a.unit) : len;
  s.lo = a.window > 0 ? max(first, (frame - a.window + 1) * a.unit) : first;
  return s;
}

// The visible keys of the page at `key0`, a bit each.
__device__ __forceinline__ uint64_t kv_bits(const KvSpan& s, int sinks, int key0) {
  auto below = [](int n) -> uint64_t { return n <= 0 ? 0ull : n >= 64 ? ~0ull : (1ull << n) - 1; };
  return below(s.hi - key0) & (~below(s.lo - key0) | below(sinks - key0));
}
// bytes of a word for four of those bits
__device__ __forceinline__ uint32_t kv_bytes(uint32_t bits) { return ((bits & 15u) * 0x00204081u & 0x01010101u) * 255u; }

// The pages that some query of a tile sees: the first `n_sink`, then from `page0` on. `lo`
// and `hi` are the tile's smallest and largest (both grow with the position).
struct KvPages {
  int n_sink, page0, n;
  int skip = 0;  // sink pages left out
  __device__ __forceinline__ int at(int i) const { return i < n_sink ? skip + i : page0 + i - n_sink; }
};
__device__ __forceinline__ KvPages kv_pages(int lo, int hi, int sinks, int width) {
  KvPages p;
  const int end = min((hi + kKvPage - 1) / kKvPage, width);
  const int near = lo / kKvPage;
  p.n_sink = lo > 0 ? min((min(sinks, hi) + kKvPage - 1) / kKvPage, min(near, end)) : 0;
  p.page0 = near;
  p.n = p.n_sink + max(0, end - near);
  return p;
}

// Of those the ones from page `from` on, or before it.
__device__ __forceinline__ KvPages kv_pages_from(KvPages p, int from) {
  const int near = p.page0 + p.n - p.n_sink;  // behind the last
  p.skip = min(from, p.n_sink);
  p.n_sink -= p.skip;
  p.page0 = max(p.page0, from);
  p.n = p.n_sink + max(0, near - p.page0);
  return p;
}
__device__ __forceinline__ KvPages kv_pages_before(KvPages p, int to) {
  const int near = min(p.page0 + p.n - p.n_sink, to);
  p.n_sink = min(p.n_sink, to);
  p.n = p.n_sink + max(0, near - p.page0);
  return p;
}

constexpr int kNoKey = 0x7fffffff;  // `lo` of a row that sees nothing

// One row of a block of a group's rows: (sequence, token, head of the group of heads)
struct KvGroupRow {
  int i, t, g;    // sequence of the group
  KvSpan span;
  int sinks;
};
// A block of `R` of a group's rows from r0 on: the pages that some row of it sees, those that the
// group shares first, then its sequences' own in turn.
struct KvGroup {
  const KvAttendArgs& a;
  int grp, G, TG, rows, P;  // P: pages that the group shares
  const int* shared;        // the group's row of the step's table
  __device__ __forceinline__ KvGroup(const KvAttendArgs& args, int group) : a(args), grp(group) {
    G = a.H / a.pool.heads;
    TG = a.T * G;
    rows = a.step.branches * TG;
    shared = a.step.rows + static_cast<long>(a.step.B + grp) * a.step.ld;
    P = group >= 0 ? min(max(shared[0], 0), a.step.width) : 0;  // (-1: no group)
  }
  // What a launch reads first, ahead of what says which of it: the ids of the shared pages, and rows of q
  __device__ __forceinline__ void prefetch_ids() const {
    for (int i = threadIdx.x * 32; i < a.step.ld; i += blockDim.x * 32) prefetch_l2(shared + i);
  }
  __device__ __forceinline__ void prefetch_q(int r, int kh) const {
    const int i = r / TG, t = (r - i * TG) / G;
    if (r < rows)
      prefetch_l2(reinterpret_cast<const __nv_bfloat16*>(a.q) + seq(i) * a.q_sb + t * a.q_st + (kh * G + r - i * TG - t * G) * a.q_sh);
  }
  __device__ __forceinline__ int seq(int i) const { return grp * a.step.branches + i; }
  __device__ __forceinline__ const int* seq_row(int i) const { return a.step.rows + static_cast<long>(seq(i)) * a.step.ld; }
  // rows behind the last, and tokens behind a sequence's own, see nothing
  __device__ __forceinline__ KvGroupRow row(int r) const {
    KvGroupRow x{0, 0, 0, {kNoKey, 0}, 0};
    if (r >= rows) return x;
    x.i = r / TG;
    x.t = (r - x.i * TG) / G;
    x.g = r - x.i * TG - x.t * G;
    const int* s = seq_row(x.i);
    if (x.t >= min(s[1], a.T)) return x;
    x.span = kv_span(a, s[0] - s[1] + x.t, s[0], s[2]);
    x.sinks = s[3] >= 0 ? s[3] : a.sinks;
    return x;
  }
};
// What a block's rows of one sequence see, and where its own pages begin in the block's list
struct __align__(16) KvBranch {
  int lo, hi, sinks, start;
};
// The block's list: `n_shared` pages that it sees of the shared ones, `n` in all
struct KvGroupPages {
  KvPages shared;
  int n, first, count;  // sequences of the group in the block
  int lo_min, lo_max, sinks_min, sinks_max;  // of the block's rows
  // The page at k: its index in the sequence, its sequence in the block (-1: shared), its id
  __device__ __forceinline__ void at(const KvGroup& g, const KvBranch* table, int k, int& page, int& branch, int& id) const {
    if (k < shared.n) {
      page = shared.at(k);
      branch = -1;
      id = g.shared[kKvInfo + page];
      return;
    }
    int b = 0;  // the last that begins at k or before
    for (int step = 128; step; step >>= 1)
      if (b + step < count && table[b + step].start <= k) b += step;
    const KvBranch t = table[b];
    page = kv_pages_from(kv_pages(t.lo, t.hi, t.sinks, g.a.step.width), g.P).at(k - t.start);
    branch = b;
    id = g.seq_row(first + b)[kKvInfo + page];
  }
};
// The list of the block of R <= 256 rows from r0 on. All threads of the CTA, which meet in it; one from
// kv_row_thread<R>(0) on for each row, with that row in `mine` (the others: a row that sees nothing),
// beside those that see to the sequences. `table` and `low` (4 words a warp) are shared memory.
template <int R>
__device__ __forceinline__ int kv_row_thread(int row) { return (R + 31) / 32 * 32 + row; }
template <int R>
__device__ __forceinline__ KvGroupPages kv_group_pages(const KvGroup& g, int r0, const KvGroupRow& mine, KvBranch* table, int* low) {
  KvGroupPages p;
  const int last = min(g.rows, r0 + R) - 1;
  p.first = r0 / g.TG;
  p.count = last < r0 ? 0 : last / g.TG - p.first + 1;
  const int b = threadIdx.x, lane = threadIdx.x & 31;
  if (b < p.count) {
    KvBranch x{kNoKey, 0, 0, 0};
    const int i = p.first + b, base = i * g.TG;
    const int* s = g.seq_row(i);
    const int len = s[0], own = s[1], first = s[2], sinks = s[3] >= 0 ? s[3] : g.a.sinks;
    const int t0 = (max(r0, base) - base) / g.G, t1 = min((min(last, base + g.TG - 1) - base) / g.G, min(own, g.a.T) - 1);
    if (t0 <= t1) {
      const int lo = kv_span(g.a, len - own + t0, len, first).lo, hi = kv_span(g.a, len - own + t1, len, first).hi;
      x = KvBranch{lo, hi, sinks, kv_pages_from(kv_pages(lo, hi, sinks, g.a.step.width), g.P).n};
    }
    table[b] = x;
  }
  constexpr int kUsed = (R + 31) / 32;  // warps with rows
  if (threadIdx.x >= kUsed * 32 && threadIdx.x < 2 * kUsed * 32) {
    const bool sees = mine.span.lo != kNoKey;
    const int v[4] = {__reduce_min_sync(0xffffffffu, mine.span.lo), __reduce_max_sync(0xffffffffu, sees ? mine.span.lo : 0),
                      __reduce_min_sync(0xffffffffu, sees ? mine.sinks : kNoKey), __reduce_max_sync(0xffffffffu, mine.sinks)};
    if (lane == 0)
      for (int k = 0; k < 4; ++k) low[((threadIdx.x >> 5) - kUsed) * 4 + k] = v[k];
  }
  __syncthreads();
  p.lo_min = low[0], p.lo_max = low[1], p.sinks_min = low[2], p.sinks_max = low[3];
  for (int w = 1; w < kUsed; ++w) {
    p.lo_min = min(p.lo_min, low[4 * w]);
    p.lo_max = max(p.lo_max, low[4 * w + 1]);
    p.sinks_min = min(p.sinks_min, low[4 * w + 2]);
    p.sinks_max = max(p.sinks_max, low[4 * w + 3]);
  }
  p.shared = KvPages{0, 0, 0};
  // every key of a shared page is before all of the block's queries
  if (p.lo_min != kNoKey) p.shared = kv_pages_before(kv_pages(p.lo_min, g.P * kKvPage, p.sinks_max, g.a.step.width), g.P);
  int start = p.shared.n, all = p.shared.n;
  for (int k = 0; k < p.count; ++k) {
    const int own = table[k].start;  // still its number of pages
    start += k < b ? own : 0;
    all += own;
  }
  p.n = all;
  __syncthreads();
  if (b < p.count) table[b].start = start;
  __syncthreads();
  return p;
}

}  // namespace ddb
