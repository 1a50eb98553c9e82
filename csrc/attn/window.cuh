// Windowed attention masks: which keys a query sees, which key tiles a query tile reads,
// which queries see a key. Positions are absolute (offsets q_pos_offset, kv_pos_offset),
// keys and queries local indexes.
#pragma once
#include <atomic>

#include "../common/ptx.cuh"
#include "../common/tma.h"
#include "attn.h"

namespace ddb {

// keys [0, sink) and [lo, hi) are visible, none at or behind hi; sink <= hi
struct WindowSpan {
  int lo, hi, sink;
  __host__ __device__ __forceinline__ bool sees(int key) const { return key < hi && (key >= lo || key < sink); }
  // every key of [key, key + n) is visible
  __host__ __device__ __forceinline__ bool whole(int key, int n) const {
    return key + n <= hi && (key >= lo || key + n <= sink);
  }
};

__host__ __device__ __forceinline__ int clamp_int(int x, int lo, int hi) { return x < lo ? lo : x > hi ? hi : x; }

__host__ __device__ __forceinline__ WindowSpan window_span(const AttnArgs& a, int q) {
  WindowSpan s{0, a.S, 0};
  const int f = (a.q_pos_offset + q) / a.tpf;
  if (a.causal != kCausalNone) {
    s.hi = clamp_int((f + 1) * a.tpf - a.kv_pos_offset, 0, a.S);
    if (a.window > 0) s.lo = clamp_int((f - a.window + 1) * a.tpf - a.kv_pos_offset, 0, a.S);
  }
  s.sink = clamp_int(a.sink_tokens - a.kv_pos_offset, 0, s.hi);
  return s;
}

// The 128-key tiles that some query of [q0, q1] sees (lo and hi grow with the query).
struct WindowTiles {
  WindowSpan span;          // of all the queries together
  int n_sink, first, n;     // tiles [0, n_sink), then from `first` on; n in all
  __host__ __device__ __forceinline__ int at(int i) const { return i < n_sink ? i : first + i - n_sink; }
};
__host__ __device__ __forceinline__ WindowTiles window_tiles(const AttnArgs& a, int q0, int q1) {
  WindowTiles t;
  const WindowSpan s0 = window_span(a, q0), s1 = window_span(a, q1);
  t.span = WindowSpan{s0.lo, s1.hi, s1.sink};
  const int end = (s1.hi + 127) / 128;
  t.first = s0.lo / 128 < end ? s0.lo / 128 : end;
  t.n_sink = (s1.sink + 127) / 128 < t.first ? (s1.sink + 127) / 128 : t.first;
  t.n = t.n_sink + end - t.first;
  return t;
}

// The queries [lo, hi) that see key k.
struct WindowQueries {
  int lo, hi;
};
__host__ __device__ __forceinline__ WindowQueries window_queries(const AttnArgs& a, int k) {
  WindowQueries w{0, a.Tq};
  if (a.causal != kCausalNone) {
    const int f = (a.kv_pos_offset + k) / a.tpf;
    w.lo = clamp_int(f * a.tpf - a.q_pos_offset, 0, a.Tq);
    if (a.window > 0 && a.kv_pos_offset + k >= a.sink_tokens)
      w.hi = clamp_int((f + a.window) * a.tpf - a.q_pos_offset, 0, a.Tq);
  }
  return w;
}

// 4-D map of [B, rows, H, 64] bf16: boxes of 64 rows of one head, 128-byte swizzle
inline CUtensorMap window_tmap(const void* base, int B, int rows, int H, long sb, long st, long sh) {
  const uint64_t dims[4] = {64, static_cast<uint64_t>(H), static_cast<uint64_t>(rows), static_cast<uint64_t>(B)};
  const uint64_t strides[3] = {static_cast<uint64_t>(sh) * 2, static_cast<uint64_t>(st) * 2, static_cast<uint64_t>(sb) * 2};
  const uint32_t box[4] = {64, 1, 64, 1};
  return make_tmap_nd(base, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, 4, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

// Raises a kernel's dynamic shared memory limit once on each device.
template <auto Kernel>
inline void raise_smem_limit(int bytes, int dev) {
  static std::atomic<uint64_t> done{0};
  if (done.load() >> (dev & 63) & 1) return;
  check_cuda(cudaFuncSetAttribute(Kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes),
             "cudaFuncSetAttribute(windowed attention)");
  done.fetch_or(1ull << (dev & 63));
}

}  // namespace ddb
