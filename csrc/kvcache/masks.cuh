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

}  // namespace ddb
