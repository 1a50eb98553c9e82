// Attention over the 8-bit paged cache for few query rows (generated tokens).
//
// Rows are (token, query head of the group): all query heads that share a cached head read
// its pages once. One CTA = 8 * NT rows of one (sequence, cached head) and a share of its
// pages, as 4 groups of NT warps: a group walks pages of its own, a ring of bulk copies
// (keys 4 KB, values 4 KB) ahead of it, and each of its warps keeps a running maximum,
// sum and output for 8 rows.
//   S^T = K Q^T and O^T = V^T P^T run on the warp-level 16x8x16 matrix instruction in fp16
//   with fp32 sums: these kernels wait for memory, not for matrix rate, and the register
//   operands take the codes without a pass through shared memory. The codes are the
//   16-row operand, the 8-column one holds 8 query rows, so one generated token wastes
//   little. e4m3 -> fp16 is exact, one instruction for two codes. Q is scaled by a power of
//   two per row (largest element near 2^14), exact but for elements 2^-28 of the row's
//   largest. P <= 1 is held as 2^15 P in fp16: rounded by at most 2^-11 of itself down to
//   2^-29, by at most 2^-40 below, so that a long tail of small weights is in the product as
//   it is in the sum. A page's key scale multiplies its scores, its value scale (and
//   2^-15) its P V product, both in fp32.
//   Reduced indexes are permuted so that a lane's operand bytes are contiguous: of a key
//   row, lane c of a quad holds channels 16c..16c+15 (a word of 4 codes is one k-step of
//   16), of a value channel tokens 16c..16c+15. Row r < 8 of key tile i is token
//   16 (r / 2) + 4 i + r % 2, row 8 + r the token 2 behind it; an 8x8 transpose of the packed
//   weights then gives the P operand of k-step i.
// The warps' results meet in shared memory; the CTAs that share a (sequence, cached head)
// form a cluster and meet through distributed shared memory. No scratch memory, no second
// launch, and a fixed order of sums.
// Measured: 64 streams of 16 heads and up to 16,384 cached tokens, one new token each,
// 255-285 us by GPU: 1.62 GB of codes at 0.97-0.87 of the rate of a plain copy, bound by memory. One token
// of one stream of 1,500 tokens, 12 heads: 6.5 us, a chain of latencies (launch, table, page,
// scores, merge). 5 tokens of 16 streams, 16 heads over 4 cached ones, window 2,048: 14.7 us a
// call, 2.6 us of bytes: the 3 warps of a group each convert the page's codes, for 8 rows each, and only
// 4 pages of a CTA are in work at once.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <algorithm>
#include <atomic>

#include "../common/ptx.cuh"
#include "../common/tma.h"
#include "attend.h"
#include "masks.cuh"

namespace ddb {
namespace {

constexpr int kGroups = 4;
constexpr int kMaxStages = 6;
constexpr int kPageBytes = 8192;  // keys, then values
constexpr float kHeadroom = 15.f;  // log2 of what a weight of 1 is in fp16 (largest: 2^16 less a step)
// Scores (log2) from which the rounding of a maximum, 2^-24 of it, moves the weights against it by
// more than 2^(1/2), all alike; from 2^24 on they would overflow.
constexpr float kFar = 8388608.f;
constexpr int kPitch = 68;        // floats between result rows (their writes then hit distinct banks)

// the CTA's result and its rows' (m, l) | barriers | page scales | flag | rings, later the
// groups' results
constexpr int out_floats(int NT) { return 8 * NT * kPitch; }
constexpr int off_ml(int NT) { return out_floats(NT) * 4; }
constexpr int off_bar(int NT) { return off_ml(NT) + 64 * NT; }
constexpr int off_scale(int NT) { return off_bar(NT) + kGroups * kMaxStages * 16; }
constexpr int off_flag(int NT) { return off_scale(NT) + kGroups * kMaxStages * 16; }
constexpr int off_ring(int NT) { return (off_flag(NT) + 16 + 127) / 128 * 128; }
constexpr int smem_bytes(int NT, int stages) { return off_ring(NT) + kGroups * stages * kPageBytes; }
static_assert(kGroups * (out_floats(4) * 4 + 64 * 4) <= kGroups * 2 * kPageBytes, "results fit the rings");
static_assert(smem_bytes(4, kMaxStages) <= 232448, "shared memory per CTA");

__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t half2_of(uint32_t two) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(two), __NV_E4M3);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack_half(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint4 lds128(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
  return v;
}
// transposes an 8x8 matrix of 16-bit values held two to a lane (row lane / 4)
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

template <int NT>
__global__ void __launch_bounds__(kGroups * NT * 32)
    kv_attend_rows(const KvAttendArgs a, int row_tiles, int stages, uint32_t group_inv, int* status) {
  extern __shared__ __align__(128) uint8_t smem[];
  constexpr int R = 8 * NT, kThreads = kGroups * NT * 32;
  const int warp = warp_id(), lane = lane_id();
  const int rg = warp % NT, pg = warp / NT;  // the warp's 8 rows, and its group
  const int g = lane >> 2, c = lane & 3;
  const int ranks = a.ranks, rank = blockIdx.x % ranks;
  int item = blockIdx.x / ranks;
  const int tile = item % row_tiles;
  item /= row_tiles;
  const int kh = item % a.pool.heads, b = item / a.pool.heads;
  const int G = a.H / a.pool.heads;
  const int* row = a.step.rows + static_cast<long>(b) * a.step.ld;
  const int len = row[0], own = min(row[1], a.T), first = row[2], old = len - row[1];
  const int sinks = row[3] >= 0 ? row[3] : a.sinks;  // a trimmed sequence has its own
  const int r0 = tile * R, rows = own * G;           // rows behind `rows` are padding
  // token of a row: at most 256 rows, so the product with 2^32 / G rounded up is exact
  auto token = [&](int r) -> int { return G == 1 ? r : __umulhi(r, group_inv); };

  uint64_t* full = reinterpret_cast<uint64_t*>(smem + off_bar(NT)) + pg * 2 * kMaxStages;
  uint64_t* empty = full + kMaxStages;
  float4* scales = reinterpret_cast<float4*>(smem + off_scale(NT)) + pg * kMaxStages;
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + off_flag(NT));
  uint8_t* ring = smem + off_ring(NT) + pg * stages * kPageBytes;
  if (rg == 0 && lane == 0) {
    for (int s = 0; s < stages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], NT);
    }
    if (pg == 0) *abort_flag = 0;
    fence_barrier_init();
  }
  __syncthreads();

  // the tile's pages; none when it holds padding only
  KvPages pages{0, 0, 0};
  int lo_max = 0, hi_min = 0, lo_min = 0, hi_max = 0;
  if (r0 < rows) {
    const KvSpan s0 = kv_span(a, old + token(r0), len, first);
    const KvSpan s1 = kv_span(a, old + token(min(rows, r0 + R) - 1), len, first);
    lo_min = s0.lo, hi_min = s0.hi, lo_max = s1.lo, hi_max = s1.hi;
    pages = kv_pages(lo_min, hi_max, sinks, a.step.width);
  }
  const int part = rank * kGroups + pg, parts = ranks * kGroups;
  const int mine = pages.n > part ? (pages.n - part + parts - 1) / parts : 0;

  // Q's loads go out first: row g of the warp's 8, channels 16c..16c+15
  uint4 qraw[2] = {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
  if (r0 + rg * 8 + g < rows) {
    const int r = r0 + rg * 8 + g, t = token(r);
    const __nv_bfloat16* q = reinterpret_cast<const __nv_bfloat16*>(a.q) + b * a.q_sb + t * a.q_st + (kh * G + r - t * G) * a.q_sh + 16 * c;
    qraw[0] = ld_global_v4(q);
    qraw[1] = ld_global_v4(q + 8);
  }

  // the group's next 32 pages, one a lane: block of codes (-1: not in the pool) and scales
  long block = -1;
  float ks = 0.f, vs = 0.f;
  int put = 0, put_stage = 0, put_phase = 1;
  auto issue = [&]() -> bool {  // the group's next page; its first warp, whole
    if ((put & 31) == 0) {
      const int n = part + (put + lane) * parts;
      block = -1;
      if (n < pages.n) {
        const int id = row[kKvInfo + pages.at(n)];
        if (static_cast<unsigned>(id) < static_cast<unsigned>(a.pool.pages)) {
          block = static_cast<long>(id) * a.pool.heads + kh;
          ks = a.pool.k_scale[block];
          vs = a.pool.v_scale[block];
        } else {  // no call's mask reaches a page that the table lacks: recorded, hidden
          record_bad_index(status, id);
        }
      }
    }
    if (NT > 1 && !__all_sync(0xffffffffu, mbar_wait(&empty[put_stage], put_phase, abort_flag))) return false;
    const long at = __shfl_sync(0xffffffffu, block, put & 31);
    if (lane == 0) {  // the copies first: the scales may still be on their way
      const long from = max(at, 0L) * 4096;
      uint64_t* bar = &full[put_stage];
      uint8_t* dst = ring + put_stage * kPageBytes;
      bulk_load(dst, a.pool.k + from, 4096, bar);
      bulk_load(dst + 4096, a.pool.v + from, 4096, bar);
    }
    const float kf = __shfl_sync(0xffffffffu, ks, put & 31), vf = __shfl_sync(0xffffffffu, vs, put & 31);
    if (lane == 0) {
      scales[put_stage] = make_float4(kf, vf, at >= 0 ? 1.f : 0.f, 0.f);
      mbar_arrive_expect_tx(&full[put_stage], kPageBytes);
    }
    ++put;
    if (++put_stage == stages) {
      put_stage = 0;
      put_phase ^= 1;
    }
    return true;
  };
  bool ok = true;
  if (rg == 0)
    for (int i = 0; i < min(mine, stages); ++i) issue();  // no wait: the stages are empty

  uint32_t qf[4][2];
  float sl2[2];   // score factors of rows 2c and 2c + 1, which this lane's scores belong to
  KvSpan span[2];
  {
    float x[16];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint32_t ws[4] = {qraw[i].x, qraw[i].y, qraw[i].z, qraw[i].w};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float2 f = unpack_bf16(ws[k]);
        x[i * 8 + 2 * k] = f.x;
        x[i * 8 + 2 * k + 1] = f.y;
      }
    }
    float amax = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) amax = fmaxf(amax, fabsf(x[i]));
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
    const int e = row_exponent(amax);
    const float down = __int_as_float((127 - e) << 23);
    const float up = a.scale * 1.4426950408889634f * __int_as_float((127 + e) << 23);
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      qf[s][0] = pack_half(x[4 * s] * down, x[4 * s + 1] * down);
      qf[s][1] = pack_half(x[4 * s + 2] * down, x[4 * s + 3] * down);
    }
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      sl2[u] = __shfl_sync(0xffffffffu, up, (2 * c + u) * 4);
      // a padding row keeps zeros and the span of the last row: its result is not used
      span[u] = kv_span(a, old + token(min(max(rows, 1), r0 + rg * 8 + 2 * c + u + 1) - 1), len, first);
    }
  }

  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
  float o[4][4];  // channels 16 i + g, + 8 of rows 2c, 2c + 1
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int k = 0; k < 4; ++k) o[i][k] = 0.f;

  const int krow = 16 * (g >> 1) + (g & 1);
  int st = 0, phase = 0;
  for (int i = 0; i < mine; ++i) {
    ok = __all_sync(0xffffffffu, mbar_wait(&full[st], phase, abort_flag));
    if (!ok) break;
    const uint32_t sk = smem_u32(ring + st * kPageBytes), sv = sk + 4096;
    const float4 f = scales[st];
    const bool there = f.z != 0.f;
    const int key0 = pages.at(part + i * parts) * kKvPage;

    float s[4][4];  // keys krow + 4 t (and 2 behind it) of rows 2c, 2c + 1
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const uint4 w0 = lds128(sk + (krow + 4 * t) * 64 + c * 16), w1 = lds128(sk + (krow + 4 * t + 2) * 64 + c * 16);
      const uint32_t x0[4] = {w0.x, w0.y, w0.z, w0.w}, x1[4] = {w1.x, w1.y, w1.z, w1.w};
#pragma unroll
      for (int k = 0; k < 4; ++k) s[t][k] = 0.f;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint32_t av[4] = {half2_of(x0[k] & 0xffff), half2_of(x1[k] & 0xffff), half2_of(x0[k] >> 16), half2_of(x1[k] >> 16)};
        mma_f16(s[t], av, qf[k][0], qf[k][1]);
      }
    }
    // a page that every row of the tile sees whole needs no mask
    const bool whole = there && key0 + kKvPage <= hi_min && (key0 >= lo_max || key0 + kKvPage <= sinks);
    float p[4][4], alpha[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const float fu = sl2[u] * f.x;
      if (!whole) {
        const uint32_t see = there ? static_cast<uint32_t>(kv_bits(span[u], sinks, key0) >> krow) : 0u;
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
          for (int k = 0; k < 2; ++k)
            if (!(see >> (4 * t + 2 * k) & 1)) s[t][2 * k + u] = -INFINITY;
      }
      float mx = fmaxf(fmaxf(s[0][u], s[0][2 + u]), fmaxf(s[1][u], s[1][2 + u]));
      mx = fmaxf(mx, fmaxf(fmaxf(s[2][u], s[2][2 + u]), fmaxf(s[3][u], s[3][2 + u])));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
      const float top = mx == -INFINITY ? m[u] : fmaxf(m[u], __fmul_rn(mx, fu));
      const float use = top == -INFINITY ? 0.f : top;
      alpha[u] = exp2f(m[u] - use);
      m[u] = top;
      float down = use - kHeadroom, by = fu;
      if (fabsf(use) >= kFar) {  // products rounded as the maximum's was: none passes it
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
          for (int k = 0; k < 2; ++k) s[t][2 * k + u] = __fadd_rn(__fmul_rn(s[t][2 * k + u], fu), -use);
        down = -kHeadroom;
        by = 1.f;
      }
      float sum = 0.f;
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const float x = s[t][2 * k + u];
          float w = exp2f(x * by - down);
          if (!whole && x == -INFINITY) w = 0.f;  // a masked score, whatever the factor is
          p[t][2 * k + u] = w;
          sum += w;
        }
      l[u] = l[u] * alpha[u] + sum;
    }
    uint32_t pf[4][2];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      pf[t][0] = transpose8x8(pack_half(p[t][0], p[t][1]));
      pf[t][1] = transpose8x8(pack_half(p[t][2], p[t][3]));
    }
    // tokens that no row of the tile sees are left out of P V whatever they hold
    uint32_t keep[4] = {~0u, ~0u, ~0u, ~0u};
    if (!(there && key0 + kKvPage <= hi_max && (key0 >= lo_min || key0 + kKvPage <= sinks))) {
      const uint32_t see = there ? static_cast<uint32_t>(kv_bits(KvSpan{lo_min, hi_max}, sinks, key0) >> (16 * c)) : 0u;
#pragma unroll
      for (int k = 0; k < 4; ++k) keep[k] = kv_bytes(see >> (4 * k));
    }
    const float vf = f.y * exp2f(-kHeadroom);
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const uint4 w0 = lds128(sv + (t * 16 + g) * 64 + c * 16), w1 = lds128(sv + (t * 16 + 8 + g) * 64 + c * 16);
      const uint32_t x0[4] = {w0.x & keep[0], w0.y & keep[1], w0.z & keep[2], w0.w & keep[3]};
      const uint32_t x1[4] = {w1.x & keep[0], w1.y & keep[1], w1.z & keep[2], w1.w & keep[3]};
      float d[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint32_t av[4] = {half2_of(x0[k] & 0xffff), half2_of(x1[k] & 0xffff), half2_of(x0[k] >> 16), half2_of(x1[k] >> 16)};
        mma_f16(d, av, pf[k][0], pf[k][1]);
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) o[t][k] = o[t][k] * alpha[k & 1] + d[k] * vf;
    }
    __syncwarp();  // every lane has read the stage
    if (NT > 1 && lane == 0) mbar_arrive(&empty[st]);
    // The next page goes into the stage that the group has just left; with several warps
    // into the one before, which the others have left too.
    if (rg == 0 && put < mine && (NT == 1 || i > 0)) ok = issue();
    if (!ok) break;
    if (++st == stages) {
      st = 0;
      phase ^= 1;
    }
  }
  if (!ok) {
    if (lane == 0) {
      if (status) atomicCAS(status, 0, kStatusTimeoutEpilogue);
      *abort_flag = 1;
      const long long t0 = clock64();  // copies in flight land before the ring is reused
      for (int s = 0; s < stages; ++s)
        for (int ph = 0; ph < 2; ++ph)
          while (!mbar_try_wait(&full[s], ph) && clock64() - t0 < kSpinLimitCycles / 8) {
          }
    }
    __syncwarp();
  }
  // ---- the groups' results: unnormalised O, m and l (whole sums), over the rings
#pragma unroll
  for (int u = 0; u < 2; ++u) {
#pragma unroll
    for (int x = 4; x < 32; x *= 2) l[u] += __shfl_xor_sync(0xffffffffu, l[u], x);
    l[u] *= exp2f(-kHeadroom);
    if (m[u] == -INFINITY && l[u] != 0.f) m[u] = 0.f;  // only NaN scores so far
  }
  __syncthreads();
  float* wo = reinterpret_cast<float*>(smem + off_ring(NT));  // [group][row][kPitch], then [group][row] (m, l)
  float2* wml = reinterpret_cast<float2*>(wo + kGroups * out_floats(NT));
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int r = rg * 8 + 2 * c + u;
    float* w = wo + pg * out_floats(NT) + r * kPitch + g;
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      w[t * 16] = o[t][u];
      w[t * 16 + 8] = o[t][2 + u];
    }
    if (g == 0) wml[pg * R + r] = make_float2(m[u], l[u]);
  }
  __syncthreads();
  float* co = reinterpret_cast<float*>(smem);  // the CTA's [row][kPitch], then [row] (m, l)
  float2* cml = reinterpret_cast<float2*>(smem + off_ml(NT));
  for (int i = threadIdx.x; i < R * 16; i += kThreads) {
    const int r = i >> 4, d = (i & 15) * 4;
    float top = -INFINITY, sum = 0.f;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kGroups; ++w) top = fmaxf(top, wml[w * R + r].x);
    if (top != -INFINITY) {
#pragma unroll
      for (int w = 0; w < kGroups; ++w) {
        const float2 ml = wml[w * R + r];
        const float k = exp2f(ml.x - top);
        const float4 x = *reinterpret_cast<const float4*>(wo + w * out_floats(NT) + r * kPitch + d);
        v.x += k * x.x;
        v.y += k * x.y;
        v.z += k * x.z;
        v.w += k * x.w;
        sum += k * ml.y;
      }
    }
    *reinterpret_cast<float4*>(co + r * kPitch + d) = v;
    if (d == 0) cml[r] = make_float2(top, sum);
  }
  if (ranks > 1) cluster_sync_all(); else __syncthreads();
  // ---- the cluster's CTAs share the rows; each adds the others' parts in rank order
  const uint32_t so = smem_u32(co), sml = smem_u32(cml);
  __nv_bfloat16* out = reinterpret_cast<__nv_bfloat16*>(a.o);
  for (int i = threadIdx.x + rank * kThreads; i < R * 16; i += ranks * kThreads) {
    const int r = i >> 4, d = (i & 15) * 4, row_id = r0 + r;
    if (row_id >= a.T * G) break;
    float top = -INFINITY, sum = 0.f;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int k = 0; k < ranks; ++k) top = fmaxf(top, ld_cluster_v2(ranks > 1 ? mapa_shared(sml + r * 8, k) : sml + r * 8).x);
    if (top != -INFINITY)
      for (int k = 0; k < ranks; ++k) {
        const uint32_t ml = ranks > 1 ? mapa_shared(sml + r * 8, k) : sml + r * 8;
        const uint32_t ov = ranks > 1 ? mapa_shared(so + (r * kPitch + d) * 4, k) : so + (r * kPitch + d) * 4;
        const float2 x = ld_cluster_v2(ml);
        const float4 y = ld_cluster_v4(ov);
        const float w = exp2f(x.x - top);
        sum += w * x.y;
        v.x += w * y.x;
        v.y += w * y.y;
        v.z += w * y.z;
        v.w += w * y.w;
      }
    const int t = token(row_id), h = kh * G + row_id - t * G;
    if (t >= own) {  // behind the sequence's own tokens
      sum = 0.f;
      v = make_float4(0.f, 0.f, 0.f, 0.f);
    }
    // a NaN among the scores makes the row NaN, as the formula has it
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    const long at = (static_cast<long>(b) * a.T + t) * a.H + h;
    *reinterpret_cast<uint2*>(out + at * 64 + d) = make_uint2(pack_bf16(v.x * inv, v.y * inv), pack_bf16(v.z * inv, v.w * inv));
    if (a.lse && d == 0)
      a.lse[(static_cast<long>(b) * a.H + h) * a.T + t] = sum == 0.f ? -INFINITY : top + __log2f(sum);
  }
  if (ranks > 1) cluster_sync_all();  // no CTA leaves while another reads its results
}

// Share the pages of an item over the CTAs of a cluster while SMs stand idle (with few rows,
// three CTAs fit one) and every group keeps a page or more. A CTA's start and merge
// measured 5 us, a group's page 2.1 us with 32 rows (512 CTAs of 12 pages a group,
// 4 waves: 118 us; 96 of 10, one wave: 28 us).
KvPlan rows_plan(const KvAttendArgs& a, int NT, int dev) {
  const long slots = static_cast<long>(num_sms(dev)) * (NT == 1 ? 3 : NT == 2 ? 2 : 1);
  const int tiles = (a.T * (a.H / a.pool.heads) + 8 * NT - 1) / (8 * NT);
  const long items = static_cast<long>(a.step.B) * a.pool.heads * tiles;
  const int pages = kv_seen_pages(a);
  KvPlan p;
  while (p.ranks < 8 && items * p.ranks * 2 <= slots && pages >= p.ranks * 2 * kGroups) p.ranks *= 2;
  const int each = (pages + p.ranks * kGroups - 1) / (p.ranks * kGroups);
  p.us = static_cast<double>((items * p.ranks + slots - 1) / slots) * (5. + 2.1 * each);
  return p;
}

template <int NT>
void launch(KvAttendArgs a, int ranks, int dev, cudaStream_t stream) {
  static std::atomic<uint64_t> set{0};  // devices whose shared-memory limit is raised
  if (!(set.load() >> (dev & 63) & 1)) {
    check_cuda(cudaFuncSetAttribute(kv_attend_rows<NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem_bytes(NT, kMaxStages)),
               "cudaFuncSetAttribute(kv_attend_rows)");
    set.fetch_or(1ull << (dev & 63));
  }
  const int G = a.H / a.pool.heads;
  const int tiles = (a.T * G + 8 * NT - 1) / (8 * NT);
  const long ctas = static_cast<long>(a.step.B) * a.pool.heads * tiles * ranks;
  if (ctas > 0x7fffffffL) throw std::runtime_error("kv_cache_attend: too many rows for one launch");
  a.ranks = ranks;
  // Stages: all that fit where an SM holds one CTA anyway (few rows of few sequences wait for
  // the copies' latency), fewer where more CTAs share it.
  const int stages = NT > 2 || ctas <= num_sms(dev) ? kMaxStages : NT == 2 ? 3 : 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(ctas));
  cfg.blockDim = dim3(kGroups * NT * 32);
  cfg.dynamicSmemBytes = smem_bytes(NT, stages);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ranks;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = ranks > 1 ? 1 : 0;
  check_cuda(cudaLaunchKernelEx(&cfg, kv_attend_rows<NT>, a, tiles, stages, 0xffffffffu / G + 1, device_status(dev)),
             "kv_attend_rows launch");
  count_launch();
}

// Rows beyond which only the 256-row blocks are tried: there each page is read by 8 row
// tiles of the other kernel. (Its rows' division by multiplication is exact far beyond.)
constexpr long kMaxRows = 256;
// 8-row warps of a row tile
int row_warps(long rows) { return rows <= 24 ? static_cast<int>(rows + 7) / 8 : 4; }

}  // namespace

// Up to 32 rows one row tile of kv_attend_rows takes them, the narrowest that does (32 rows:
// 28 us against the blocks' 42 at 12 heads of 20,000 tokens, 118 against 195 at 512 of
// 3,000). Beyond, its pages are read once for every 32 rows, and the smaller estimate
// decides: 64 rows take 15 us against 17 at 48 heads of 1,000 visible tokens, 205 against
// 196 at 512 of 3,000; 128 rows 28 against 18, 412 against 216; few and short sequences stay
// with it longer.
KvPlan kv_cache_attend_plan(const KvAttendArgs& a) {
  if (a.step.B <= 0 || a.T <= 0 || a.H <= 0) return KvPlan{};
  int dev = 0;
  check_cuda(cudaGetDevice(&dev), "cudaGetDevice");
  const long rows = a.T * static_cast<long>(a.H / a.pool.heads);
  const KvPlan few = rows <= kMaxRows ? rows_plan(a, row_warps(rows), dev) : KvPlan{};
  if (rows <= 32) return few;
  const KvPlan many = kv_attend_tiles_plan(a, dev);
  return rows > kMaxRows || many.us < few.us ? many : few;
}

void kv_cache_attend(const KvAttendArgs& a, const KvPlan& plan, cudaStream_t stream) {
  if (a.step.B <= 0 || a.T <= 0 || a.H <= 0) return;
  int dev = 0;
  check_cuda(cudaGetDevice(&dev), "cudaGetDevice");
  if (plan.blocks) {
    kv_attend_tiles_launch(a, plan, dev, stream);
    return;
  }
  switch (row_warps(a.T * static_cast<long>(a.H / a.pool.heads))) {
    case 1: launch<1>(a, plan.ranks, dev, stream); break;
    case 2: launch<2>(a, plan.ranks, dev, stream); break;
    case 3: launch<3>(a, plan.ranks, dev, stream); break;
    default: launch<4>(a, plan.ranks, dev, stream); break;
  }
}

}  // namespace ddb
