// Shared by the cache attention's kernels.
#pragma once
#include "kvcache.h"

namespace ddb {

// e of the power of two 2^e that brings a query row's largest magnitude into [2^14, 2^15), in
// [-120, 113]; 0 for a row of zeros, or one that holds an infinity or a NaN (its output
// is not finite in any case)
__device__ __forceinline__ int row_exponent(float amax) {
  const int k = static_cast<int>(__float_as_uint(amax) >> 23) - 127;
  return amax > 0.f && k < 128 ? max(k - 14, -120) : 0;
}

// Pages that a query sees at most: all, or the sinks', the window's and the call's own.
inline int kv_seen_pages(const KvAttendArgs& a) {
  const long all = a.max_tokens;
  const long near = a.sinks + (a.window + 1L) * a.unit + a.T + 2 * kKvPage;
  return static_cast<int>(((a.window > 0 && near < all ? near : all) + kKvPage - 1) / kKvPage);
}

// attend_tiles.cu: blocks of 256 rows on the tensor cores' 128-row products
KvPlan kv_attend_tiles_plan(const KvAttendArgs& a, int dev);
void kv_attend_tiles_launch(KvAttendArgs a, const KvPlan& plan, int dev, cudaStream_t stream);

}  // namespace ddb
