// Attention over the 8-bit paged cache for many query rows (chunks of frames, prompts).
//
// One CTA = 256 rows (token, query head of the group) of one (sequence, cached head), as
// two tiles of 128, and a share of its pages; tiles of 128 keys are two pages. Both row
// tiles use each key tile, so a code is converted once for 256 rows. Roles (512 threads,
// one CTA per SM):
//   warp 0       bulk copies of the pages' codes (keys 4 KB, values 4 KB each), 3 stages
//   warp 1       TMEM owner and MMA issuer: S = Q K^T (M 128, N 128, K 64) and
//                O += P V (M 128, N 64, K 128; P from TMEM), per row tile
//   warps 4-7    e4m3 -> fp16 into the swizzled operand tiles (3 stages of 16 KB each),
//                exactly; tokens that no row sees become zeros
//   warps 8-15   softmax: one thread per row and tile, as in the bf16 kernel; it also
//                brings Q to fp16, scaled by a power of two per row
// Scales: a page's key scale multiplies its half of the scores, in fp32. Its value scale goes
// into its weights, whose reference is the largest product of weight and scale that the row
// itself has met: a page that a row does not see, or hardly weighs, takes nothing from the others.
// (Scales in the converted codes, relative to the CTA's largest, took 222 us at the shape below
// where this takes 227, but lost pages 2^25 below it. With a loop of its own for scales that lie
// too far apart for that: 226, and 436 where they do. The exponents' constants made only after
// the scores: 231.)
// P <= 2^8 (the running maximum may lag by that) is held as 2^7 P in fp16: rounded by at most
// 2^-11 of itself, finer than the bf16 kernel's P, or by 2^-32 where it is below 2^-21.
// The CTAs that share a row block form a cluster and meet through distributed shared memory,
// in one launch; or, where the clusters' sizes would leave SMs idle, meet in scratch memory
// that a second launch adds up (kv_attend_tiles_plan).
// Bound by a row's chain of softmax steps: of the 3300 clocks (1.75 us) that a step of 256 x 128
// takes, the exponentials (16 a clock and SM) are 2048, and the matrix products that run beside
// them 1072. While one row tile is in its exponentials the other loads scores, takes its
// maximum and stores weights (they take turns); where that takes longer than the exponentials
// their unit waits (busy 57 % of the time). 2048 rows over 20,480 visible tokens of 12 heads (129
// GFLOP): 227 us, 0.57 PFLOP/s (in one launch of clusters 248 us, with 222 for this one then).
// Tried against those 248, and slower: the next scores
// loaded under the exponentials (266-320 us), two threads a row (304), four streams by row tile
// and page with one MMA warp (306) or one each (300), waits that spin (258).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <algorithm>
#include <atomic>
#include <type_traits>

#include "../common/ptx.cuh"
#include "../common/tma.h"
#include "attend.h"
#include "masks.cuh"

namespace ddb {
namespace {

constexpr int kThreads = 512;
constexpr int kRows = 256;
constexpr int NR = 3;  // stages of codes
constexpr int NS = 3;  // stages of fp16 tiles
constexpr int TILE = 16384;
constexpr int OFF_Q = 0;
constexpr int OFF_K = OFF_Q + 2 * TILE;
constexpr int OFF_V = OFF_K + NS * TILE;
constexpr int OFF_RAW = OFF_V + NS * TILE;   // per stage: keys of both pages, values of both
constexpr int OFF_BAR = OFF_RAW + NR * TILE;
constexpr int NF = 8;  // stages of page factors: more than the softmax can lie behind (NR + NS)
constexpr int N_BARS = 1 + 2 * NR + 4 * NS + 10 + 1 + NF;
constexpr int OFF_FACTOR = OFF_BAR + (N_BARS + 1) / 2 * 16;
constexpr int OFF_META = OFF_FACTOR + NF * 16;
constexpr int OFF_MISC = OFF_META + (NR + 1) / 2 * 8;
static_assert(NF > NR + NS && (NF & (NF - 1)) == 0, "stages of page factors");
constexpr int SMEM_BYTES = OFF_MISC + 16;
static_assert(OFF_FACTOR % 16 == 0 && OFF_MISC % 8 == 0, "alignment");
static_assert(SMEM_BYTES <= 232448, "shared memory per CTA");
constexpr int OFF_RES = OFF_K;                    // results, once K and V are no longer read
constexpr int OFF_RES_ML = OFF_RES + kRows * 256; // (max, sum) per row
static_assert(OFF_RES_ML + kRows * 8 <= OFF_RAW, "results fit the operand tiles");
constexpr uint32_t C_S = 0, C_O = 256, C_P = 384;  // + 128 / 64 / 64 per row tile
constexpr float kRescaleLog2 = 8.f;
// Scores (log2) from which the rounding of a maximum, 2^-24 of it, moves the weights against it by
// more than 2^(1/2), all alike; from 2^24 on they would overflow.
constexpr float kFar = 8388608.f;
constexpr float kHeadroom = 7.f;  // log2 of what a weight of 1 is in fp16; with the lag 2^15 at most
constexpr long kPartFloats = kRows * 66;  // a CTA's result in scratch
constexpr int kHandOver = 3;  // quarters of a row's exponentials after which the other tile may begin

// kind::f16 with fp16 A and B, fp32 D, both K-major
__host__ __device__ constexpr uint32_t idesc_f16(int M, int N) {
  return (1u << 4) | (static_cast<uint32_t>(N >> 3) << 17) | (static_cast<uint32_t>(M >> 4) << 24);
}
constexpr uint32_t IDESC_S = idesc_f16(128, 128);
constexpr uint32_t IDESC_PV = idesc_f16(128, 64);

__device__ __forceinline__ uint32_t pack_half(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t half2_of(uint32_t two) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(two), __NV_E4M3);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float log2_of_power(float p) { return static_cast<float>((__float_as_int(p) >> 23) - 127); }
// every warp has its role's registers
__device__ __forceinline__ void registers_split() { asm volatile("bar.sync 1, %0;" ::"n"(kThreads) : "memory"); }

__global__ void __launch_bounds__(kThreads, 1)
    kv_attend_tiles(const KvAttendArgs a, int row_tiles, int* status) {
  extern __shared__ __align__(1024) uint8_t smem[];
  if ((smem_u32(smem) & 1023) != 0) {  // uniform over the grid
    if (threadIdx.x == 0 && status) atomicCAS(status, 0, kStatusBadArgument);
    return;
  }
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + OFF_BAR);
  uint64_t* q_full = bars;
  uint64_t* raw_full = bars + 1;
  uint64_t* raw_empty = raw_full + NR;
  uint64_t* k_full = raw_empty + NR;
  uint64_t* k_empty = k_full + NS;
  uint64_t* v_full = k_empty + NS;
  uint64_t* v_empty = v_full + NS;
  uint64_t* s_full = v_empty + NS;  // [2], and so on
  uint64_t* s_free = s_full + 2;
  uint64_t* p_full = s_full + 4;
  uint64_t* o_done = s_full + 6;
  uint64_t* turn = s_full + 8;
  uint64_t* drain = s_full + 10;
  uint64_t* f_full = drain + 1;  // [NF]
  int* meta = reinterpret_cast<int*>(smem + OFF_META);  // per stage: which of both pages are there
  // key scales and log2 of the value scales of a pair, for the softmax
  float4* factor = reinterpret_cast<float4*>(smem + OFF_FACTOR);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + OFF_MISC);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + OFF_MISC + 4);
  // largest key scale of the CTA's pages (positive floats order like their bits)
  int* k_most = reinterpret_cast<int*>(smem + OFF_MISC + 8);

  const int warp = warp_id(), lane = lane_id();
  const int ranks = a.ranks, rank = blockIdx.x % ranks;
  int item = blockIdx.x / ranks;
  const int tile = row_tiles - 1 - item % row_tiles;  // long (late) tiles first
  item /= row_tiles;
  const int kh = item % a.pool.heads, b = item / a.pool.heads;
  const int G = a.H / a.pool.heads;
  const int* row = a.step.rows + static_cast<long>(b) * a.step.ld;
  const int len = row[0], own = min(row[1], a.T), first = row[2], old = len - row[1];
  const int sinks = row[3] >= 0 ? row[3] : a.sinks;  // a trimmed sequence has its own
  const int r0 = tile * kRows, rows = own * G;       // rows behind `rows` are padding
  const int n_t = rows - r0 > 128 ? 2 : 1;

  // the block's pages, and this CTA's run of key tiles (page pairs)
  KvPages pages{0, 0, 0};
  KvSpan all{0, 0};
  if (r0 < rows) {
    const KvSpan s0 = kv_span(a, old + r0 / G, len, first);
    const KvSpan s1 = kv_span(a, old + (min(rows, r0 + kRows) - 1) / G, len, first);
    all = KvSpan{s0.lo, s1.hi};
    pages = kv_pages(s0.lo, s1.hi, sinks, a.step.width);
  }
  const int pairs = (pages.n + 1) / 2, per = (pairs + ranks - 1) / ranks;
  const int j0 = min(pairs, rank * per), n = min(pairs, j0 + per) - j0;

  if (threadIdx.x == 0) {
    mbar_init(q_full, 8);
    for (int s = 0; s < NR; ++s) {
      mbar_init(&raw_full[s], 1);
      mbar_init(&raw_empty[s], 4);
    }
    for (int s = 0; s < NS; ++s) {
      mbar_init(&k_full[s], 4);
      mbar_init(&k_empty[s], 1);
      mbar_init(&v_full[s], 4);
      mbar_init(&v_empty[s], 1);
    }
    for (int t = 0; t < 2; ++t) {
      mbar_init(&s_full[t], 1);
      mbar_init(&s_free[t], 4);
      mbar_init(&p_full[t], 4);
      mbar_init(&o_done[t], 1);
      mbar_init(&turn[t], 4);
    }
    mbar_init(drain, 1);
    for (int s = 0; s < NF; ++s) mbar_init(&f_full[s], 1);
    *abort_flag = 0;
    *k_most = 0;
    fence_barrier_init();
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  {
    int most = 0;
    for (int i = 2 * j0 + threadIdx.x; i < min(pages.n, 2 * (j0 + n)); i += kThreads) {
      const int id = row[kKvInfo + pages.at(i)];
      if (static_cast<unsigned>(id) < static_cast<unsigned>(a.pool.pages))
        most = max(most, __float_as_int(a.pool.k_scale[static_cast<long>(id) * a.pool.heads + kh]));
    }
    most = __reduce_max_sync(0xffffffffu, most);
    if (lane == 0 && most) atomicMax(k_most, most);
  }
  __syncthreads();

  // Registers by role: 56 + 72 + 2 * 192 = 512 = 4 * 128, the launch's own. All go back to 128
  // before the common end; none may before every role has its share (registers_split),
  // or a role with nothing to do would take back what the softmax warps still wait for.
  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
    registers_split();
    if (warp == 0) {
      // ---------------------------------------------------------- copies of the codes
      bool ok = true;
      int ids = -1, issued = 0;
      float ks = 0.f, vs = 0.f;
      for (int j = 0; j < n; ++j) {
        if ((j & 15) == 0) {  // the next 16 pairs, one page a lane
          const int i = 2 * (j0 + j) + lane;
          ids = i < min(pages.n, 2 * (j0 + n)) ? row[kKvInfo + pages.at(i)] : -2;
          if (ids != -2 && static_cast<unsigned>(ids) >= static_cast<unsigned>(a.pool.pages)) {
            record_bad_index(status, ids);  // recorded, read as zeros
            ids = -2;
          }
          ks = vs = 0.f;
          if (ids >= 0) {
            const long block = static_cast<long>(ids) * a.pool.heads + kh;
            ks = a.pool.k_scale[block];
            vs = a.pool.v_scale[block];
          }
        }
        const int l0 = 2 * (j & 15), s = j % NR;
        const int id0 = __shfl_sync(0xffffffffu, ids, l0), id1 = __shfl_sync(0xffffffffu, ids, l0 + 1);
        const float4 f = make_float4(__shfl_sync(0xffffffffu, ks, l0), __shfl_sync(0xffffffffu, ks, l0 + 1),
                                     __shfl_sync(0xffffffffu, vs, l0), __shfl_sync(0xffffffffu, vs, l0 + 1));
        ok = __all_sync(0xffffffffu, mbar_wait(&raw_empty[s], ((j / NR) & 1) ^ 1, abort_flag));
        if (!ok) break;
        if (lane == 0) {
          uint8_t* dst = smem + OFF_RAW + s * TILE;
          // The softmax has read the factors NF pairs back: codes 3 pairs back have been converted,
          // so the scores of the pair 6 back are made, and those before it read.
          factor[j % NF] = make_float4(f.x, f.y, log2_of_power(f.z), log2_of_power(f.w));
          mbar_arrive(&f_full[j % NF]);
          meta[s] = (id0 >= 0 ? 1 : 0) | (id1 >= 0 ? 2 : 0);
          mbar_arrive_expect_tx(&raw_full[s], (id0 >= 0 ? 8192 : 0) + (id1 >= 0 ? 8192 : 0));
          const int id[2] = {id0, id1};
#pragma unroll
          for (int p = 0; p < 2; ++p)
            if (id[p] >= 0) {
              const long at = (static_cast<long>(id[p]) * a.pool.heads + kh) * 4096;
              bulk_load(dst + p * 4096, a.pool.k + at, 4096, &raw_full[s]);
              bulk_load(dst + 8192 + p * 4096, a.pool.v + at, 4096, &raw_full[s]);
            }
        }
        ++issued;
        __syncwarp();
      }
      if (lane == 0) {
        if (!ok) {
          if (status) atomicCAS(status, 0, kStatusTimeoutProducer);
          *abort_flag = 1;
        }
        for (int j = max(0, issued - NR); j < issued; ++j) {  // copies in flight land
          const long long t0 = clock64();
          while (!mbar_try_wait(&raw_full[j % NR], (j / NR) & 1) && clock64() - t0 < kSpinLimitCycles / 8) {
          }
        }
      }
    } else if (warp == 1) {
      // ---------------------------------------------------------- MMA issuer
      // The whole warp walks the loop, so that addresses and descriptors stay in uniform
      // registers, where the instruction takes them; one elected lane issues.
      auto wait = [&](uint64_t* bar, uint32_t parity) -> bool {
        return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag));
      };
      bool ok = n == 0 || wait(q_full, 0);
      const uint64_t dq = make_sw128_desc(smem_u32(smem + OFF_Q), 16, 1024);
      const uint64_t dk = make_sw128_desc(smem_u32(smem + OFF_K), 16, 1024);
      const uint64_t dv = make_sw128_desc(smem_u32(smem + OFF_V), 16, 1024);
      auto issue_pv = [&](int i) -> bool {
        if (!wait(&v_full[i % NS], (i / NS) & 1)) return false;
        const uint64_t d = dv + (i % NS) * (TILE >> 4);
        for (int t = 0; t < n_t; ++t) {
          if (!wait(&p_full[t], i & 1)) return false;
          tc_fence_after();
          if (elect_one()) {
#pragma unroll
            for (int kk = 0; kk < 8; ++kk)  // 16 tokens a step: page kk / 4
              mma_bf16_ts(tmem + C_O + t * 64, tmem + C_P + t * 64 + kk * 8, d + (kk >> 2) * 512 + (kk & 3) * 2, IDESC_PV,
                          (i > 0 || kk > 0) ? 1u : 0u);
            mma_commit(&o_done[t]);
          }
          __syncwarp();
        }
        if (elect_one()) mma_commit(&v_empty[i % NS]);
        return true;
      };
      for (int j = 0; j < n && ok; ++j) {
        ok = wait(&k_full[j % NS], (j / NS) & 1);
        const uint64_t d = dk + (j % NS) * (TILE >> 4);
        for (int t = 0; t < n_t && ok; ++t) {
          if (j > 0) ok = wait(&s_free[t], (j - 1) & 1);
          if (!ok) break;
          tc_fence_after();
          if (elect_one()) {
#pragma unroll
            for (int kk = 0; kk < 4; ++kk)
              mma_bf16_ss(tmem + C_S + t * 128, dq + t * (TILE >> 4) + kk * 2, d + kk * 2, IDESC_S, kk > 0 ? 1u : 0u);
            mma_commit(&s_full[t]);
          }
          __syncwarp();
        }
        if (ok && elect_one()) mma_commit(&k_empty[j % NS]);
        __syncwarp();
        if (ok && j > 0) ok = issue_pv(j - 1);
      }
      if (ok && n > 0) ok = issue_pv(n - 1);
      if (lane == 0) {
        if (!ok) {
          if (status) atomicCAS(status, 0, kStatusTimeoutMma);
          *abort_flag = 1;
        }
      }
      __syncwarp();
      if (elect_one()) mma_commit(drain);
      __syncwarp();
      const long long t0 = clock64();
      while (!mbar_try_wait(drain, 0) && clock64() - t0 < kSpinLimitCycles / 8) {
      }
    }
    __syncwarp();
    asm volatile("setmaxnreg.inc.sync.aligned.u32 128;");
  } else if (warp < 8) {
    // ------------------------------------------------------------ conversion
    asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
    registers_split();
    const int t = threadIdx.x - 128;
    const int r = t >> 2, c = t & 3;  // row of 32, 16-byte piece of it; then rows r + 32 i
    bool ok = true;
    auto convert = [&](const uint8_t* raw, uint32_t dst, const uint32_t (&keep)[2][4]) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint4 w = *reinterpret_cast<const uint4*>(raw + t * 16 + i * 2048);
        const uint32_t ws[4] = {w.x & keep[i >> 1][0], w.y & keep[i >> 1][1], w.z & keep[i >> 1][2], w.w & keep[i >> 1][3]};
        uint32_t o[8];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          o[2 * k] = half2_of(ws[k] & 0xffff);
          o[2 * k + 1] = half2_of(ws[k] >> 16);
        }
        const int R = r + 32 * i;
        const uint32_t d = dst + R * 128;
        st_shared_v4(d + (((2 * c) ^ (R & 7)) << 4), o[0], o[1], o[2], o[3]);
        st_shared_v4(d + (((2 * c + 1) ^ (R & 7)) << 4), o[4], o[5], o[6], o[7]);
      }
    };
    for (int j = 0; j < n; ++j) {
      const int sr = j % NR, s = j % NS;
      ok = mbar_wait(&raw_full[sr], (j / NR) & 1, abort_flag) &&
           mbar_wait(&k_empty[s], ((j / NS) & 1) ^ 1, abort_flag);
      if (!__all_sync(0xffffffffu, ok)) {
        ok = false;
        break;
      }
      const int there = meta[sr];
      const uint8_t* raw = smem + OFF_RAW + sr * TILE;
      uint32_t keep[2][4];
#pragma unroll
      for (int p = 0; p < 2; ++p)  // an absent page holds whatever the stage held
#pragma unroll
        for (int k = 0; k < 4; ++k) keep[p][k] = there >> p & 1 ? ~0u : 0u;
      convert(raw, smem_u32(smem + OFF_K + s * TILE), keep);
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&k_full[s]);
      // tokens that no row of the block sees stay out of P V whatever they hold
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        const int i = 2 * (j0 + j) + p;
        const int key = pages.at(i) * kKvPage;
        if (keep[p][0] && !(key + kKvPage <= all.hi && (key >= all.lo || key + kKvPage <= sinks))) {
          const uint32_t see = static_cast<uint32_t>(kv_bits(all, sinks, key) >> (16 * c));
#pragma unroll
          for (int k = 0; k < 4; ++k) keep[p][k] = kv_bytes(see >> (4 * k));
        }
      }
      ok = mbar_wait(&v_empty[s], ((j / NS) & 1) ^ 1, abort_flag);
      if (!__all_sync(0xffffffffu, ok)) {
        ok = false;
        break;
      }
      convert(raw + 8192, smem_u32(smem + OFF_V + s * TILE), keep);
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&v_full[s]);
        mbar_arrive(&raw_empty[sr]);
      }
    }
    if (!ok) {
      if (lane == 0 && status) atomicCAS(status, 0, kStatusTimeoutProducer);
      *abort_flag = 1;
    }
    __syncwarp();
    asm volatile("setmaxnreg.inc.sync.aligned.u32 128;");
  } else {
    // ------------------------------------------------------------ softmax
    asm volatile("setmaxnreg.inc.sync.aligned.u32 192;");
    registers_split();
    const int t = (warp - 8) >> 2, quad = warp & 3;
    const int lr = quad * 32 + lane;
    const int r = r0 + t * 128 + lr;
    const bool active = t < n_t;  // of a second tile that is all padding nothing is computed
    const uint32_t trow = tmem + (static_cast<uint32_t>(quad * 32) << 16);
    // a padding row keeps zeros and the span of the last row: its result is not used
    const KvSpan span = kv_span(a, old + (min(max(rows, 1), r + 1) - 1) / G, len, first);
    float sl2, bound;
    {
      uint4 w[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i] = make_uint4(0, 0, 0, 0);
      if (r < rows) {
        const __nv_bfloat16* q = reinterpret_cast<const __nv_bfloat16*>(a.q) + b * a.q_sb + (r / G) * a.q_st +
                                 (kh * G + r % G) * a.q_sh;
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = ld_global_v4(q + i * 8);
      }
      float amax = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t ws[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float2 f = unpack_bf16(ws[k]);
          amax = fmaxf(amax, fmaxf(fabsf(f.x), fabsf(f.y)));
        }
      }
      const int e = row_exponent(amax);
      const float down = __int_as_float((127 - e) << 23);
      const uint32_t dst = smem_u32(smem + OFF_Q + t * TILE) + lr * 128;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t ws[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
        uint32_t h[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float2 f = unpack_bf16(ws[k]);
          h[k] = pack_half(f.x * down, f.y * down);
        }
        st_shared_v4(dst + ((i ^ (lr & 7)) << 4), h[0], h[1], h[2], h[3]);
      }
      sl2 = a.scale * 1.4426950408889634f * __int_as_float((127 + e) << 23);
      // |S| < 2^30, 64 products of numbers up to 2^15 and 448; zero for a row of zeros (padding)
      bound = amax > 0.f ? sl2 * 0x1p30f * __int_as_float(*k_most) : 0.f;
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(q_full);
    }
    // The weights of the sum are relative to 2^m; those of the product, times their page's value
    // scale, to 2^(m + d).
    float m = -INFINITY, d = 0.f, l = 0.f;
    auto steps = [&](auto far_scores) -> bool {
      constexpr bool kFarScores = decltype(far_scores)::value;
      for (int j = 0; j < n; ++j) {
        if (!mbar_wait(&f_full[j % NF], (j / NF) & 1, abort_flag)) return false;
        const float4 f = factor[j % NF];
        // of the scores; not zero: a masked score is -inf times it
        const float f0 = fmaxf(sl2 * f.x, 1e-37f), f1 = fmaxf(sl2 * f.y, 1e-37f);
        // The page's exponents hold its value scale; its sum is brought back. A scale far below the
        // reference counts as 2^-64 of it, so that no weight that counts in the sum underflows.
        float e0, e1, down0, down1;
        auto shifts = [&] {
          const float use = (m == -INFINITY ? 0.f : m) - kHeadroom;
          e0 = fmaxf(f.z - d, -64.f), e1 = fmaxf(f.w - d, -64.f);
          down0 = use - e0, down1 = use - e1;
        };
        shifts();
        if (!mbar_wait(&s_full[t], j & 1, abort_flag)) return false;
        tc_fence_after();
        float sf[128];
        {
          uint32_t x0[32], x1[32], x2[32], x3[32];
          tmem_ld32(trow + C_S + t * 128, x0);
          tmem_ld32(trow + C_S + t * 128 + 32, x1);
          tmem_ld32(trow + C_S + t * 128 + 64, x2);
          tmem_ld32(trow + C_S + t * 128 + 96, x3);
          tmem_wait_ld();
#pragma unroll
          for (int c = 0; c < 32; ++c) {
            sf[c] = __uint_as_float(x0[c]);
            sf[32 + c] = __uint_as_float(x1[c]);
            sf[64 + c] = __uint_as_float(x2[c]);
            sf[96 + c] = __uint_as_float(x3[c]);
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&s_free[t]);
#pragma unroll
        for (int p = 0; p < 2; ++p) {
          const int i = 2 * (j0 + j) + p;
          const int key = i < pages.n ? pages.at(i) * kKvPage : 0x40000000;  // no page: no key
          if (!(key + kKvPage <= span.hi && (key >= span.lo || key + kKvPage <= sinks))) {
            const uint64_t see = kv_bits(span, sinks, key);
            const uint32_t word[2] = {static_cast<uint32_t>(see), static_cast<uint32_t>(see >> 32)};
#pragma unroll
            for (int c = 0; c < 64; ++c)
              if (!(word[c >> 5] >> (c & 31) & 1)) sf[p * 64 + c] = -INFINITY;
          }
        }
        float mp[8];  // of the first page, of the second
#pragma unroll
        for (int i = 0; i < 8; ++i) mp[i] = sf[(i >> 2) * 64 + (i & 3)];
#pragma unroll
        for (int c = 4; c < 64; ++c) {
          mp[c & 3] = fmaxf(mp[c & 3], sf[c]);
          mp[4 + (c & 3)] = fmaxf(mp[4 + (c & 3)], sf[64 + c]);
        }
        const float m0 = __fmul_rn(f0, fmaxf(fmaxf(mp[0], mp[1]), fmaxf(mp[2], mp[3])));
        const float m1 = __fmul_rn(f1, fmaxf(fmaxf(mp[4], mp[5]), fmaxf(mp[6], mp[7])));
        // A reference moves only when something passes it by 2^8: P <= 256, few rescales of O,
        // and what the exponentials need is known before the scores are.
        float alpha = 1.f, alpha_o = 1.f;
        const float lag = kFarScores ? 0.f : kRescaleLog2;
        const bool moves = __any_sync(0xffffffffu, fmaxf(fmaxf(m0, m1), fmaxf(m0 + e0, m1 + e1)) > m + lag);
        if (moves) {
          const float mx2 = fmaxf(m0, m1);
          if (mx2 > m + lag) {
            alpha = exp2f(m - mx2);
            d += m - mx2;
            m = mx2;
          }
          if (m != -INFINITY) {
            const float top = fmaxf(m0 - m + f.z, m1 - m + f.w);
            if (top > d + kRescaleLog2) {
              alpha_o = exp2f(d - top);
              d = top;
            }
          }
          shifts();
        }
        if (kFarScores) {  // products rounded as the maximum's was: none passes it
          const float use = m == -INFINITY ? 0.f : m;
#pragma unroll
          for (int c = 0; c < 64; ++c) {
            sf[c] = __fadd_rn(__fmul_rn(sf[c], f0), -use);
            sf[64 + c] = __fadd_rn(__fmul_rn(sf[64 + c], f1), -use);
          }
          down0 = -e0 - kHeadroom, down1 = -e1 - kHeadroom;
        }
        // P V of the last key tile is done: O may be rescaled and P overwritten
        if (j > 0) {
          if (!mbar_wait(&o_done[t], (j - 1) & 1, abort_flag)) return false;
          tc_fence_after();
          if (moves && __any_sync(0xffffffffu, alpha_o != 1.f)) {
#pragma unroll
            for (int c = 0; c < 64; c += 16) {
              uint32_t ov[16];
              tmem_ld16(trow + C_O + t * 64 + c, ov);
              tmem_wait_ld();
#pragma unroll
              for (int i = 0; i < 16; ++i) ov[i] = __float_as_uint(__uint_as_float(ov[i]) * alpha_o);
              tmem_st16(trow + C_O + t * 64 + c, ov);
            }
          }
        }
        // The tiles take turns at their exponentials, which one tile alone issues near the
        // unit's full rate: in step, both would leave it idle during their loads and maxima.
        if (n_t == 2 && (t == 1 || j > 0) && !mbar_wait(&turn[1 - t], (j - 1 + t) & 1, abort_flag)) return false;
        float sp[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int ch = 0; ch < 4; ++ch) {  // stored 32 columns at a time, to hold few registers
          if (ch == kHandOver) {
            __syncwarp();
            if (lane == 0) mbar_arrive(&turn[t]);
          }
          const float by = kFarScores ? 1.f : ch < 2 ? f0 : f1, down = ch < 2 ? down0 : down1;
          uint32_t pk[16];
#pragma unroll
          for (int c = 0; c < 32; c += 2) {
            const float p0 = exp2f(sf[ch * 32 + c] * by - down);
            const float p1 = exp2f(sf[ch * 32 + c + 1] * by - down);
            sp[c & 7] += p0;
            sp[(c + 1) & 7] += p1;
            pk[c >> 1] = pack_half(p0, p1);
          }
          tmem_st16(trow + C_P + t * 64 + ch * 16, pk);
          if (ch & 1) {
            l = (ch == 1 ? l * alpha : l) +
                (((sp[0] + sp[1]) + (sp[2] + sp[3])) + ((sp[4] + sp[5]) + (sp[6] + sp[7]))) * exp2f(ch == 1 ? -e0 : -e1);
#pragma unroll
            for (int i = 0; i < 8; ++i) sp[i] = 0.f;
          }
        }
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[t]);
      }
      return true;
    };
    // Scores that may be far from zero go through a loop of their own, twice as slow (in the other
    // one the test and the code for them took 229-235 us where this takes 227).
    const bool far = __any_sync(0xffffffffu, bound >= kFar);
    const bool ok = !active || (far ? steps(std::true_type{}) : steps(std::false_type{}));
    if (!ok) {
      if (lane == 0 && status) atomicCAS(status, 0, kStatusTimeoutEpilogue);
      *abort_flag = 1;
    }
    // every MMA is done: O may be read, and the operand tiles overwritten
    float ov[64];
    l *= exp2f(-kHeadroom);
    const float up = exp2f(d - kHeadroom);
    const bool done = __all_sync(0xffffffffu, mbar_wait(drain, 0, abort_flag) && ok);
    if (done && active && n > 0) {
      tc_fence_after();
      uint32_t x0[32], x1[32];
      tmem_ld32(trow + C_O + t * 64, x0);
      tmem_ld32(trow + C_O + t * 64 + 32, x1);
      tmem_wait_ld();
#pragma unroll
      for (int c = 0; c < 32; ++c) {
        ov[c] = __uint_as_float(x0[c]) * up;
        ov[32 + c] = __uint_as_float(x1[c]) * up;
      }
    } else {
#pragma unroll
      for (int c = 0; c < 64; ++c) ov[c] = 0.f;
    }
    if (r >= rows) {
      l = 0.f;
#pragma unroll
      for (int c = 0; c < 64; ++c) ov[c] = 0.f;
    }
    if (m == -INFINITY && l != 0.f) m = 0.f;  // only NaN scores
    if (a.part) {
      // 256 rows of 64 channels, then their (maximum, sum), for kv_tiles_merge
      float* part = a.part + blockIdx.x * kPartFloats;
      if (r < a.T * G) {
        float* o = part + (t * 128 + lr) * 64;
#pragma unroll
        for (int c = 0; c < 16; ++c)
          *reinterpret_cast<float4*>(o + 4 * c) = make_float4(ov[4 * c], ov[4 * c + 1], ov[4 * c + 2], ov[4 * c + 3]);
        *reinterpret_cast<float2*>(part + kRows * 64 + (t * 128 + lr) * 2) = make_float2(r < rows ? m : -INFINITY, l);
      }
    } else if (ranks > 1) {
      if (done) {  // not while something may still read the operand tiles
        const uint32_t dst = smem_u32(smem + OFF_RES) + (t * 128 + lr) * 256;
#pragma unroll
        for (int c = 0; c < 16; ++c)
          st_shared_v4(dst + ((c ^ (lr & 15)) << 4), __float_as_uint(ov[4 * c]), __float_as_uint(ov[4 * c + 1]),
                       __float_as_uint(ov[4 * c + 2]), __float_as_uint(ov[4 * c + 3]));
        *reinterpret_cast<float2*>(smem + OFF_RES_ML + (t * 128 + lr) * 8) = make_float2(r < rows ? m : -INFINITY, l);
      }
    } else if (r < a.T * G) {
      const float inv = l == 0.f ? 0.f : 1.f / l;
      const int tok = r / G, h = kh * G + r % G;
      const long at = (static_cast<long>(b) * a.T + tok) * a.H + h;
      __nv_bfloat16* o = reinterpret_cast<__nv_bfloat16*>(a.o) + at * 64;
#pragma unroll
      for (int c = 0; c < 64; c += 8)
        st_global_v4(o + c, pack_bf16(ov[c] * inv, ov[c + 1] * inv), pack_bf16(ov[c + 2] * inv, ov[c + 3] * inv),
                     pack_bf16(ov[c + 4] * inv, ov[c + 5] * inv), pack_bf16(ov[c + 6] * inv, ov[c + 7] * inv));
      if (a.lse) a.lse[(static_cast<long>(b) * a.H + h) * a.T + tok] = l == 0.f ? -INFINITY : m + __log2f(l);
    }
    __syncwarp();
    asm volatile("setmaxnreg.dec.sync.aligned.u32 128;");
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
  if (ranks > 1 && !a.part) {
    // ---- each CTA of the cluster adds up its share of the rows, in rank order; 16 threads a
    // row, 4 channels each
    cluster_sync_all();
    const uint32_t res = smem_u32(smem + OFF_RES), ml = smem_u32(smem + OFF_RES_ML);
    for (int i = threadIdx.x + rank * kThreads; i < kRows * 16; i += ranks * kThreads) {
      const int lr = i >> 4, c = i & 15, r = r0 + lr;
      if (r >= a.T * G) break;
      float top = -INFINITY, sum = 0.f;
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int k = 0; k < ranks; ++k) top = fmaxf(top, ld_cluster_v2(mapa_shared(ml + lr * 8, k)).x);
      if (top != -INFINITY)
        for (int k = 0; k < ranks; ++k) {
          const float2 x = ld_cluster_v2(mapa_shared(ml + lr * 8, k));
          const float4 y = ld_cluster_v4(mapa_shared(res + lr * 256 + ((c ^ (lr & 15)) << 4), k));
          const float w = exp2f(x.x - top);
          sum += w * x.y;
          v.x += w * y.x;
          v.y += w * y.y;
          v.z += w * y.z;
          v.w += w * y.w;
        }
      const float inv = sum == 0.f ? 0.f : 1.f / sum;
      const int tok = r / G, h = kh * G + r % G;
      const long at = (static_cast<long>(b) * a.T + tok) * a.H + h;
      *reinterpret_cast<uint2*>(reinterpret_cast<__nv_bfloat16*>(a.o) + at * 64 + c * 4) =
          make_uint2(pack_bf16(v.x * inv, v.y * inv), pack_bf16(v.z * inv, v.w * inv));
      if (a.lse && c == 0)
        a.lse[(static_cast<long>(b) * a.H + h) * a.T + tok] = sum == 0.f ? -INFINITY : top + __log2f(sum);
    }
    cluster_sync_all();  // no CTA leaves while another reads its results
  }
}

// Adds up the CTAs' results of each row, in rank order; 16 threads a row, 4 channels each.
__global__ void __launch_bounds__(256) kv_tiles_merge(const KvAttendArgs a, int row_tiles) {
  const int G = a.H / a.pool.heads;
  const int lr = (blockIdx.x % (kRows / 16)) * 16 + (threadIdx.x >> 4), c = threadIdx.x & 15;
  int item = blockIdx.x / (kRows / 16);
  const float* part = a.part + static_cast<long>(item) * a.ranks * kPartFloats;
  const int r = (row_tiles - 1 - item % row_tiles) * kRows + lr;  // the other kernel's order
  item /= row_tiles;
  const int kh = item % a.pool.heads, b = item / a.pool.heads;
  if (r >= a.T * G) return;
  float top = -INFINITY, sum = 0.f;
  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int k = 0; k < a.ranks; ++k) top = fmaxf(top, part[k * kPartFloats + kRows * 64 + lr * 2]);
  if (top != -INFINITY)
    for (int k = 0; k < a.ranks; ++k) {
      const float2 x = *reinterpret_cast<const float2*>(part + k * kPartFloats + kRows * 64 + lr * 2);
      const float4 y = *reinterpret_cast<const float4*>(part + k * kPartFloats + lr * 64 + c * 4);
      const float w = exp2f(x.x - top);
      sum += w * x.y;
      v.x += w * y.x;
      v.y += w * y.y;
      v.z += w * y.z;
      v.w += w * y.w;
    }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  const int tok = r / G, h = kh * G + r % G;
  const long at = (static_cast<long>(b) * a.T + tok) * a.H + h;
  *reinterpret_cast<uint2*>(reinterpret_cast<__nv_bfloat16*>(a.o) + at * 64 + c * 4) =
      make_uint2(pack_bf16(v.x * inv, v.y * inv), pack_bf16(v.z * inv, v.w * inv));
  if (a.lse && c == 0)
    a.lse[(static_cast<long>(b) * a.H + h) * a.T + tok] = sum == 0.f ? -INFINITY : top + __log2f(sum);
}

}  // namespace

namespace {
void raise_limit(int dev) {
  static std::atomic<uint64_t> set{0};  // devices whose shared-memory limit is raised
  if (set.load() >> (dev & 63) & 1) return;
  check_cuda(cudaFuncSetAttribute(kv_attend_tiles, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_BYTES),
             "cudaFuncSetAttribute(kv_attend_tiles)");
  set.fetch_or(1ull << (dev & 63));
}
int row_blocks(const KvAttendArgs& a) { return static_cast<int>((a.T * static_cast<long>(a.H / a.pool.heads) + kRows - 1) / kRows); }
long row_items(const KvAttendArgs& a) { return static_cast<long>(a.step.B) * a.pool.heads * row_blocks(a); }
cudaLaunchConfig_t config(int ranks, cudaLaunchAttribute* attr) {
  attr->id = cudaLaunchAttributeClusterDimension;
  attr->val.clusterDim.x = ranks;
  attr->val.clusterDim.y = attr->val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ranks);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = SMEM_BYTES;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cfg;
}
}  // namespace

// The way with the smallest estimate. How many clusters of a size run at once is the device's to
// say: of 3 CTAs only 45 do on 148 SMs (the GPCs' SMs are no multiple), so 96 of them take
// three waves; apart, meeting in scratch, two. Measured, as clusters and apart: 96 blocks of
// 160 steps 248 and 222 us, 48 of 40 61 and 50, 49 of 33 54 and 42. A CTA's start and merge
// take about 15 us, a step (128 keys) 1.3 us with one row tile and 1.75 us with two (512 CTAs
// of 24 steps, 4 waves: 190 / 254 us; 96 of 20 steps, one wave: 40 / 51 us); the second
// launch 4 us and 0.015 us a CTA (288 CTAs: 7 us).
KvPlan kv_attend_tiles_plan(const KvAttendArgs& a, int dev) {
  raise_limit(dev);
  static std::atomic<int> fits[64][9];
  const int pairs = (kv_seen_pages(a) + 1) / 2;
  const double step = a.T * static_cast<long>(a.H / a.pool.heads) > 128 ? 1.75 : 1.3;
  const long items = row_items(a);
  KvPlan best;
  best.blocks = true;
  for (int s = 1; s <= 8 && (s == 1 || pairs >= 2 * s); ++s) {
    int slots = s == 1 ? num_sms(dev) : fits[dev & 63][s].load();
    if (slots == 0) {
      cudaLaunchAttribute attr[1];
      const cudaLaunchConfig_t cfg = config(s, attr);
      check_cuda(cudaOccupancyMaxActiveClusters(&slots, kv_attend_tiles, &cfg), "cudaOccupancyMaxActiveClusters");
      slots = std::max(slots, 1);
      fits[dev & 63][s].store(slots);
    }
    const double each = 15. + step * ((pairs + s - 1) / s);
    const double us = static_cast<double>((items + slots - 1) / slots) * each;
    if (s == 1 || us < best.us) best.ranks = s, best.scratch = 0, best.us = us;
    if (s == 1 || items * s > 4L * num_sms(dev)) continue;  // more waves even out by themselves
    const double apart = static_cast<double>((items * s + num_sms(dev) - 1) / num_sms(dev)) * each + 4. + items * s * 0.015;
    if (apart < best.us) best.ranks = s, best.scratch = items * s * kPartFloats, best.us = apart;
  }
  return best;
}

void kv_attend_tiles_launch(KvAttendArgs a, const KvPlan& plan, int dev, cudaStream_t stream) {
  raise_limit(dev);
  const long ctas = row_items(a) * plan.ranks;
  if (ctas > 0x7fffffffL / (kRows / 16)) throw std::runtime_error("kv_cache_attend: too many rows for one launch");
  if (plan.scratch && !a.part) throw std::runtime_error("kv_cache_attend: no scratch");
  a.ranks = plan.ranks;
  if (!plan.scratch) a.part = nullptr;
  cudaLaunchAttribute attr[1];
  cudaLaunchConfig_t cfg = config(plan.ranks, attr);
  cfg.gridDim = dim3(static_cast<unsigned>(ctas));
  cfg.stream = stream;
  cfg.numAttrs = plan.ranks > 1 && !a.part ? 1 : 0;
  check_cuda(cudaLaunchKernelEx(&cfg, kv_attend_tiles, a, row_blocks(a), device_status(dev)), "kv_attend_tiles launch");
  count_launch();
  if (a.part) {
    kv_tiles_merge<<<static_cast<unsigned>(row_items(a) * (kRows / 16)), 256, 0, stream>>>(a, row_blocks(a));
    check_cuda(cudaGetLastError(), "kv_tiles_merge launch");
    count_launch();
  }
}

}  // namespace ddb
