// Attention over the 8-bit paged cache for few query rows (generated tokens).
//
// Rows are (token, query head of the group): all query heads that share a cached head read
// its pages once. One CTA = 16 * MT rows of one (sequence, cached head) and a share of its
// pages; each of its 4 warps walks pages of its own, a ring of bulk copies (keys 4 KB,
// values 4 KB) ahead of it, and keeps a running maximum, sum and output.
//   S = Q K^T and O = P V run on the warp-level 16x8x16 matrix instruction in fp16 with fp32
//   sums: these kernels wait for memory, not for matrix rate, and the register operands
//   take the codes without a pass through shared memory. e4m3 -> fp16 is exact, one
//   instruction for two codes. Q is scaled by a power of two per row (largest element near
//   2^14), exact but for elements 2^-28 of the row's largest. P <= 1 in fp16 is rounded by
//   at most 2^-11 of itself. A page's key scale multiplies its scores, its value scale
//   its P V product, both in fp32.
//   Reduced indexes are permuted so that a lane's operand bytes are contiguous: of a key
//   row, lane c of a quad holds channels 16c..16c+15 (a word of 4 codes is one k-step of
//   16), of a value channel tokens 16c..16c+15; the score columns are the tokens in the
//   order that makes the score registers the P operand (column 2c+i of tile j is token
//   16c + 4(j/2) + 2(j%2) + i).
// The warps' results meet in shared memory; the CTAs that share a (sequence, cached head)
// form a cluster and meet through distributed shared memory. No scratch memory, no second
// launch, and a fixed order of sums.
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

constexpr int kWarps = 4;
constexpr int kStages = 3;
constexpr int kPageBytes = 8192;  // keys, then values

__host__ __device__ constexpr int out_floats(int MT) { return 16 * MT * 64; }
// ring | barriers | page scales | results: [warp] O, m, l, then the CTA's O, m, l
__host__ __device__ constexpr int off_bar() { return kWarps * kStages * kPageBytes; }
__host__ __device__ constexpr int off_scale() { return off_bar() + kWarps * kStages * 8; }
__host__ __device__ constexpr int off_flag() { return off_scale() + kWarps * kStages * 16; }
__host__ __device__ constexpr int off_cta(int) { return off_flag() + 32; }
__host__ __device__ constexpr int smem_bytes(int MT) { return off_cta(MT) + (out_floats(MT) + 32 * MT) * 4; }

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
__device__ __forceinline__ float ld_cluster(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}

template <int MT>
__global__ void __launch_bounds__(kWarps * 32) kv_attend_rows(const KvAttendArgs a, int row_tiles, int* status) {
  extern __shared__ __align__(128) uint8_t smem[];
  const int warp = warp_id(), lane = lane_id();
  const int g = lane >> 2, c = lane & 3;
  const int ranks = a.cluster, rank = blockIdx.x % ranks;
  int item = blockIdx.x / ranks;
  const int tile = item % row_tiles;
  item /= row_tiles;
  const int kh = item % a.pool.heads, b = item / a.pool.heads;
  const int G = a.H / a.pool.heads;
  const int* row = a.step.rows + static_cast<long>(b) * a.step.ld;
  const int len = row[0], own = min(row[1], a.T), first = row[2], old = len - row[1];
  const int sinks = row[3] >= 0 ? row[3] : a.sinks;  // a trimmed sequence has its own
  const int r0 = tile * 16 * MT, rows = own * G;  // rows behind `rows` are padding

  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + off_bar()) + warp * kStages;
  float* scales = reinterpret_cast<float*>(smem + off_scale()) + warp * kStages * 4;
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + off_flag());
  uint8_t* ring = smem + warp * kStages * kPageBytes;
  if (lane == 0) {
    for (int s = 0; s < kStages; ++s) mbar_init(&bars[s], 1);
    if (warp == 0) *abort_flag = 0;
    fence_barrier_init();
  }
  __syncthreads();

  // the tile's pages; none when it holds padding only
  KvPages pages{0, 0, 0};
  int lo_max = 0, hi_min = 0, lo_min = 0, hi_max = 0;
  if (r0 < rows) {
    const KvSpan s0 = kv_span(a, old + r0 / G, len, first);
    const KvSpan s1 = kv_span(a, old + (min(rows, r0 + 16 * MT) - 1) / G, len, first);
    lo_min = s0.lo, hi_min = s0.hi, lo_max = s1.lo, hi_max = s1.hi;
    pages = kv_pages(lo_min, hi_max, sinks, a.step.width);
  }
  const int part = rank * kWarps + warp, parts = ranks * kWarps;
  const int mine = pages.n > part ? (pages.n - part + parts - 1) / parts : 0;

  // page ids of the warp's next 32 pages, one a lane
  int ids = -1;
  auto issue = [&](int i) {  // i-th page of this warp; whole warp
    if ((i & 31) == 0) {
      const int n = part + (i + lane) * parts;
      ids = n < pages.n ? row[kKvInfo + pages.at(n)] : -1;
    }
    int id = __shfl_sync(0xffffffffu, ids, i & 31);
    if (lane == 0) {
      const int s = i % kStages;
      const bool there = static_cast<unsigned>(id) < static_cast<unsigned>(a.pool.pages);
      if (!there) {  // no call's mask reaches a page that the table lacks: recorded, hidden
        record_bad_index(status, id);
        id = 0;
      }
      const long block = static_cast<long>(id) * a.pool.heads + kh;
      mbar_arrive_expect_tx(&bars[s], kPageBytes);
      bulk_load(ring + s * kPageBytes, a.pool.k + block * 4096, 4096, &bars[s]);
      bulk_load(ring + s * kPageBytes + 4096, a.pool.v + block * 4096, 4096, &bars[s]);
      scales[s * 4] = a.pool.k_scale[block];
      scales[s * 4 + 1] = a.pool.v_scale[block];
      scales[s * 4 + 2] = there ? 1.f : 0.f;
    }
  };
  for (int i = 0; i < min(mine, kStages); ++i) issue(i);

  // Q: rows g and g + 8 of each 16, channels 16c..16c+15
  uint32_t qf[MT][4][4];
  float sl2[MT][2];
  KvSpan span[MT][2];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt)
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int r = r0 + mt * 16 + u * 8 + g;
      float x[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) x[i] = 0.f;
      // a padding row keeps zeros and the span of the last row: its result is not used
      span[mt][u] = kv_span(a, old + (min(max(rows, 1), r + 1) - 1) / G, len, first);
      if (r < rows) {
        const int t = r / G, h = kh * G + r % G;
        const __nv_bfloat16* q = reinterpret_cast<const __nv_bfloat16*>(a.q) + b * a.q_sb + t * a.q_st + h * a.q_sh + 16 * c;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint4 w = ld_global_v4(q + i * 8);
          const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const float2 f = unpack_bf16(ws[k]);
            x[i * 8 + 2 * k] = f.x;
            x[i * 8 + 2 * k + 1] = f.y;
          }
        }
      }
      float amax = 0.f;
#pragma unroll
      for (int i = 0; i < 16; ++i) amax = fmaxf(amax, fabsf(x[i]));
      amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
      amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
      const int e = row_exponent(amax);
      const float down = __int_as_float((127 - e) << 23);
      sl2[mt][u] = a.scale * 1.4426950408889634f * __int_as_float((127 + e) << 23);
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        qf[mt][s][u] = pack_half(x[4 * s] * down, x[4 * s + 1] * down);
        qf[mt][s][2 + u] = pack_half(x[4 * s + 2] * down, x[4 * s + 3] * down);
      }
    }

  float m[MT][2], l[MT][2], o[MT][8][4];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      m[mt][u] = -INFINITY;
      l[mt][u] = 0.f;
    }
#pragma unroll
    for (int n = 0; n < 8; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) o[mt][n][i] = 0.f;
  }

  bool ok = true;
  const int krow = 16 * (g >> 1) + (g & 1);
  for (int i = 0; i < mine; ++i) {
    const int st = i % kStages;
    ok = __all_sync(0xffffffffu, mbar_wait(&bars[st], (i / kStages) & 1, abort_flag));
    if (!ok) break;
    const uint32_t sk = smem_u32(ring + st * kPageBytes), sv = sk + 4096;
    const float ks = scales[st * 4], vs = scales[st * 4 + 1];
    const bool there = scales[st * 4 + 2] != 0.f;
    const int key0 = pages.at(part + i * parts) * kKvPage;

    float s[MT][8][4];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint4 w = lds128(sk + (krow + 4 * (j >> 1) + 2 * (j & 1)) * 64 + c * 16);
      const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int k = 0; k < 4; ++k) s[mt][j][k] = 0.f;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint32_t b0 = half2_of(ws[k] & 0xffff), b1 = half2_of(ws[k] >> 16);
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) mma_f16(s[mt][j], qf[mt][k], b0, b1);
      }
    }
    // a page that every row of the tile sees whole needs no mask
    const bool whole = there && key0 + kKvPage <= hi_min && (key0 >= lo_max || key0 + kKvPage <= sinks);
    uint32_t pf[MT][4][4];
    float alpha[MT][2];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const float f = sl2[mt][u] * ks;
        float mx = -INFINITY;
        if (!whole) {
#pragma unroll
          for (int j = 0; j < 8; ++j)
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              const int key = key0 + 16 * c + 4 * (j >> 1) + 2 * (j & 1) + k;
              if (!there || !kv_visible(span[mt][u], sinks, key)) s[mt][j][2 * u + k] = -INFINITY;
            }
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) mx = fmaxf(mx, fmaxf(s[mt][j][2 * u], s[mt][j][2 * u + 1]));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        const float top = mx == -INFINITY ? m[mt][u] : fmaxf(m[mt][u], mx * f);
        const float use = top == -INFINITY ? 0.f : top;
        alpha[mt][u] = exp2f(m[mt][u] - use);
        m[mt][u] = top;
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          float p0, p1;
          if (!whole) {  // a masked score stays -inf whatever the factor is
            p0 = s[mt][j][2 * u] == -INFINITY ? 0.f : exp2f(s[mt][j][2 * u] * f - use);
            p1 = s[mt][j][2 * u + 1] == -INFINITY ? 0.f : exp2f(s[mt][j][2 * u + 1] * f - use);
          } else {
            p0 = exp2f(s[mt][j][2 * u] * f - use);
            p1 = exp2f(s[mt][j][2 * u + 1] * f - use);
          }
          sum += p0 + p1;
          pf[mt][j >> 1][(j & 1) * 2 + u] = pack_half(p0, p1);
        }
        l[mt][u] = l[mt][u] * alpha[mt][u] + sum;
      }
    }
    // tokens that no row of the tile sees are left out of P V whatever they hold
    uint32_t keep[4] = {~0u, ~0u, ~0u, ~0u};
    if (!(there && key0 + kKvPage <= hi_max && (key0 >= lo_min || key0 + kKvPage <= sinks))) {
      const KvSpan all{lo_min, hi_max};
#pragma unroll
      for (int k = 0; k < 16; ++k)
        if (!there || !kv_visible(all, sinks, key0 + 16 * c + k)) keep[k >> 2] &= ~(0xffu << (8 * (k & 3)));
    }
#pragma unroll
    for (int n = 0; n < 8; ++n) {
      const uint4 w = lds128(sv + (n * 8 + g) * 64 + c * 16);
      const uint32_t ws[4] = {w.x & keep[0], w.y & keep[1], w.z & keep[2], w.w & keep[3]};
      float d[MT][4];
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int k = 0; k < 4; ++k) d[mt][k] = 0.f;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint32_t b0 = half2_of(ws[k] & 0xffff), b1 = half2_of(ws[k] >> 16);
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) mma_f16(d[mt], pf[mt][k], b0, b1);
      }
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int k = 0; k < 4; ++k) o[mt][n][k] = o[mt][n][k] * alpha[mt][k >> 1] + d[mt][k] * vs;
    }
    __syncwarp();  // every lane has read the stage
    if (i + kStages < mine) issue(i + kStages);
  }
  if (!ok) {
    if (lane == 0 && status) atomicCAS(status, 0, kStatusTimeoutEpilogue);
    *abort_flag = 1;
    if (lane == 0) {  // copies in flight land before the ring is reused or the CTA retires
      const long long t0 = clock64();
      for (int s = 0; s < kStages; ++s)
        for (int ph = 0; ph < 2; ++ph)
          while (!mbar_try_wait(&bars[s], ph) && clock64() - t0 < kSpinLimitCycles / 8) {
          }
    }
  }
  // ---- the warps' results: unnormalised O, m, l (quad sums), over the rings
#pragma unroll
  for (int mt = 0; mt < MT; ++mt)
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      l[mt][u] += __shfl_xor_sync(0xffffffffu, l[mt][u], 1);
      l[mt][u] += __shfl_xor_sync(0xffffffffu, l[mt][u], 2);
      if (m[mt][u] == -INFINITY && l[mt][u] != 0.f) m[mt][u] = 0.f;  // only NaN scores so far
    }
  __syncthreads();
  float* wo = reinterpret_cast<float*>(smem);                // [warp][row][64]
  float* wml = wo + kWarps * out_floats(MT);                 // [warp][row][2]
#pragma unroll
  for (int mt = 0; mt < MT; ++mt)
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int r = mt * 16 + u * 8 + g;
#pragma unroll
      for (int n = 0; n < 8; ++n)
        *reinterpret_cast<float2*>(wo + warp * out_floats(MT) + r * 64 + n * 8 + 2 * c) =
            make_float2(o[mt][n][2 * u], o[mt][n][2 * u + 1]);
      if (c == 0) {
        wml[(warp * 16 * MT + r) * 2] = m[mt][u];
        wml[(warp * 16 * MT + r) * 2 + 1] = l[mt][u];
      }
    }
  __syncthreads();
  float* co = reinterpret_cast<float*>(smem + off_cta(MT));  // the CTA's [row][64], then [row][2]
  float* cml = co + out_floats(MT);
  for (int i = threadIdx.x; i < out_floats(MT); i += kWarps * 32) {
    const int r = i >> 6;
    float top = -INFINITY, sum = 0.f, v = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) top = fmaxf(top, wml[(w * 16 * MT + r) * 2]);
    if (top != -INFINITY) {
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float k = exp2f(wml[(w * 16 * MT + r) * 2] - top);
        v += k * wo[w * out_floats(MT) + i];
        sum += k * wml[(w * 16 * MT + r) * 2 + 1];
      }
    }
    co[i] = v;
    if ((i & 63) == 0) {
      cml[r * 2] = top;
      cml[r * 2 + 1] = sum;
    }
  }
  if (ranks > 1) cluster_sync_all(); else __syncthreads();
  // ---- the cluster's CTAs share the rows; each adds the others' parts in rank order
  const uint32_t so = smem_u32(co), sml = smem_u32(cml);
  __nv_bfloat16* out = reinterpret_cast<__nv_bfloat16*>(a.o);
  for (int i = threadIdx.x + rank * kWarps * 32; i < out_floats(MT) / 2; i += ranks * kWarps * 32) {
    const int r = i >> 5, d = (i & 31) * 2, R = r0 + r;
    if (R >= a.T * G) break;
    float top = -INFINITY, sum = 0.f, v0 = 0.f, v1 = 0.f;
    for (int k = 0; k < ranks; ++k) top = fmaxf(top, ld_cluster(ranks > 1 ? mapa_shared(sml + r * 8, k) : sml + r * 8));
    if (top != -INFINITY) {
      for (int k = 0; k < ranks; ++k) {
        const uint32_t ml = ranks > 1 ? mapa_shared(sml + r * 8, k) : sml + r * 8;
        const uint32_t ov = ranks > 1 ? mapa_shared(so + (r * 64 + d) * 4, k) : so + (r * 64 + d) * 4;
        const float w = exp2f(ld_cluster(ml) - top);
        sum += w * ld_cluster(ml + 4);
        v0 += w * ld_cluster(ov);
        v1 += w * ld_cluster(ov + 4);
      }
    }
    const int t = R / G, h = kh * G + R % G;
    if (t >= own) sum = v0 = v1 = 0.f;  // behind the sequence's own tokens
    // a NaN among the scores makes the row NaN, as the formula has it
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    const long at = (static_cast<long>(b) * a.T + t) * a.H + h;
    *reinterpret_cast<uint32_t*>(out + at * 64 + d) = pack_bf16(v0 * inv, v1 * inv);
    if (a.lse && d == 0)
      a.lse[(static_cast<long>(b) * a.H + h) * a.T + t] = sum == 0.f ? -INFINITY : top + __log2f(sum);
  }
  if (ranks > 1) cluster_sync_all();  // no CTA leaves while another reads its results
}

template <int MT>
void launch(KvAttendArgs a, int dev, cudaStream_t stream) {
  static std::atomic<uint64_t> set{0};  // devices whose shared-memory limit is raised
  if (!(set.load() >> (dev & 63) & 1)) {
    check_cuda(cudaFuncSetAttribute(kv_attend_rows<MT>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem_bytes(MT)),
               "cudaFuncSetAttribute(kv_attend_rows)");
    set.fetch_or(1ull << (dev & 63));
  }
  const int G = a.H / a.pool.heads;
  const int tiles = (a.T * G + 16 * MT - 1) / (16 * MT);
  const long items = static_cast<long>(a.step.B) * a.pool.heads * tiles;
  // Share the pages of an item over more CTAs while the SMs' two slots are not filled and
  // every warp keeps two pages or more.
  const int pages = (a.max_tokens + kKvPage - 1) / kKvPage;
  int ranks = 1;
  while (ranks < 8 && items * ranks < 2L * num_sms(dev) && pages >= ranks * 2 * kWarps * 2) ranks *= 2;
  if (items * ranks > 0x7fffffffL) throw std::runtime_error("kv_cache_attend: too many rows for one launch");
  a.cluster = ranks;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(items * ranks));
  cfg.blockDim = dim3(kWarps * 32);
  cfg.dynamicSmemBytes = smem_bytes(MT);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ranks;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = ranks > 1 ? 1 : 0;
  check_cuda(cudaLaunchKernelEx(&cfg, kv_attend_rows<MT>, a, tiles, device_status(dev)), "kv_attend_rows launch");
  count_launch();
}

}  // namespace

void kv_cache_attend(const KvAttendArgs& a, cudaStream_t stream) {
  if (a.step.B <= 0 || a.T <= 0 || a.H <= 0) return;
  int dev = 0;
  check_cuda(cudaGetDevice(&dev), "cudaGetDevice");
  if (a.T * static_cast<long>(a.H / a.pool.heads) > 64)
    kv_attend_tiles_launch(a, dev, stream);
  else
    launch<1>(a, dev, stream);
}

}  // namespace ddb
