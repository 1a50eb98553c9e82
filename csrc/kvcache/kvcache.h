// Paged key/value cache in 8 bits: writing tokens, attention over it, moving pages.
//
// A page holds 64 consecutive tokens of one sequence for every layer and head:
//   keys    [layer][page][head][64 tokens][64 channels]  e4m3 codes
//   values  [layer][page][head][64 channels][64 tokens]  e4m3 codes, channel-major
//   scales  [layer][page][head]  fp32, a power of two, keys and values apart
// and stands for code * scale. A scale is 2^e with the smallest e for which the block's
// largest finite magnitude is at most 448 * 2^e. A power of two costs no mantissa bit of a
// floating-point code, makes a re-coding to a larger scale exact (but for codes that
// become subnormal) and lets the attention kernels apply it without a rounding.
// Values lie channel-major so that the P V product reads tokens, its reduced index,
// contiguously (as both the register and the shared-memory operand formats want them).
//
// A call works on a step's table, int32 rows [sequence][4 + width]:
//   tokens in the cache with the call's own | the call's own tokens | first token kept
//   behind the sinks (0: all) | sinks of a trimmed sequence, or -1 | page ids of the
//   sequence, 64 tokens each (-1: none)
#pragma once
#include <cuda_runtime.h>
#include <cstdint>

namespace ddb {

constexpr int kKvPage = 64;  // tokens of a page
constexpr int kKvInfo = 4;   // words of a step row before its page ids

struct KvPool {  // one layer
  uint8_t* k = nullptr;
  uint8_t* v = nullptr;
  float* k_scale = nullptr;
  float* v_scale = nullptr;
  int pages = 0;
  int heads = 0;
};

struct KvStep {
  const int* rows = nullptr;
  int ld = 0;     // words between rows
  int width = 0;  // page ids of a row
  int B = 0;
};

struct KvWriteArgs {
  KvPool pool;
  KvStep step;
  const void* k = nullptr;  // bf16 [B, T, H, 64]: element strides, channels contiguous
  const void* v = nullptr;
  long k_sb = 0, k_st = 0, k_sh = 0;
  long v_sb = 0, v_st = 0, v_sh = 0;
  int T = 0;
};

// Writes each sequence's own tokens (the first n of its T rows) into its pages. The
// committed tokens of an unfinished page are kept, re-coded if its scale changes; its
// slots behind the last token become zero.
void kv_cache_write(const KvWriteArgs& a, cudaStream_t s);

struct KvAttendArgs {
  KvPool pool;
  KvStep step;
  const void* q = nullptr;  // bf16 [B, T, H, 64]: element strides, channels contiguous
  long q_sb = 0, q_st = 0, q_sh = 0;
  void* o = nullptr;     // bf16 [B, T, H, 64] contiguous
  float* lse = nullptr;  // [B, H, T], log2 domain, or null
  int T = 0;
  int H = 0;             // query heads; head h reads cached head h / (H / pool.heads)
  bool causal = true;    // keys of the query's frame and earlier ones (unit 1: token-causal)
  int unit = 1;          // tokens per frame
  int window = 0;        // frames visible behind (and with) the query's own; 0: all
  int sinks = 0;         // first tokens that stay visible beside the window
  float scale = 0.125f;
  int max_tokens = 0;    // no sequence is longer (sets the launch's shape only)
  int ranks = 1;         // CTAs that share a row tile (set by the launch)
  float* part = nullptr; // the plan's scratch, 16-byte aligned
};

// How a call is launched: the kernel, how many CTAs share a row tile's pages, and the scratch
// that they meet in (0: distributed shared memory); with an estimate of its time.
struct KvPlan {
  bool blocks = false;   // 256-row blocks (attend_tiles.cu), not few rows (attend_rows.cu)
  int ranks = 1;
  long scratch = 0;      // floats
  double us = 0.;
};
KvPlan kv_cache_attend_plan(const KvAttendArgs& a);

// Attention of each sequence's own tokens (its newest) over its cached ones. Rows with no
// visible key, and rows behind a sequence's own tokens, get zeros and lse = -inf.
void kv_cache_attend(const KvAttendArgs& a, const KvPlan& plan, cudaStream_t s);

// Copies pages src[i] -> dst[i] in every layer (codes and scales). The dst are distinct and
// none is a src.
void kv_cache_copy_pages(uint8_t* k, uint8_t* v, float* k_scale, float* v_scale, int layers,
                         int pages, int heads, const int* src, const int* dst, int n,
                         cudaStream_t s);

}  // namespace ddb
