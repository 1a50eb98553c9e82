// Attention of branches over the pages that they share: the first of two launches, the second one
// (attend_rows.cu) reads each sequence's own pages and adds what this one found.
//
// Rows are (sequence of the group, token, query head of the group of heads): all that read one
// cached head of the shared past. One CTA = 8 * NJ rows and a share of the visible shared pages,
// as 8 warps with pages of their own, each with all the rows: a code is brought to fp16 once
// for NJ 8-row products, and no warp waits for another until the end. Formats, permutations
// and the softmax are those of attend_rows.cu (S^T = K Q^T, O^T = V^T P^T with the codes as the
// 16-row operand of the 16x8x16 instruction). Every key of a shared page is older than every
// query, so only the window, the sinks and what was trimmed mask it.
// The second launch starts beside this one and waits for it only where it adds the results up.
#include <algorithm>
#include <atomic>

#include "../common/tma.h"
#include "attend.h"
#include "masks.cuh"
#include "rows.cuh"

namespace ddb {
namespace {

constexpr int kWarps = 8;
constexpr int kThreads = kWarps * 32;
constexpr int kStages = 3;

// barriers | page scales | rows' first key behind the sinks and sinks | flag | rings, later results
constexpr int OFF_SCALE = kWarps * kStages * 8;
constexpr int OFF_ROWS = OFF_SCALE + kWarps * kStages * 16;
constexpr int OFF_FLAG = OFF_ROWS + 32 * 8;
constexpr int OFF_RING = (OFF_FLAG + 16 + 127) / 128 * 128;
constexpr int SMEM_BYTES = OFF_RING + kWarps * kStages * kPageBytes;
static_assert(kWarps * 32 * (kPitch * 4 + 8) <= kWarps * kStages * kPageBytes, "results fit the rings");
static_assert(SMEM_BYTES <= 232448, "shared memory per CTA");

template <int NJ>
__global__ void __launch_bounds__(kThreads, 1) kv_attend_past(const KvAttendArgs a, int row_tiles, int* status) {
  extern __shared__ __align__(128) uint8_t smem[];
  constexpr int R = 8 * NJ;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int warp = warp_id(), lane = lane_id();
  const int g = lane >> 2, c = lane & 3;
  const int ranks = a.past_ranks, rank = blockIdx.x % ranks;
  const int out_tile = blockIdx.x / ranks;
  int item = out_tile;
  const int r0 = item % row_tiles * R;
  item /= row_tiles;
  const int kh = item % a.pool.heads, grp = item / a.pool.heads;
  const int n = a.step.branches, G = a.H / a.pool.heads, TG = a.T * G, rows = n * TG;
  const int* shared = a.step.rows + static_cast<long>(a.step.B + grp) * a.step.ld;
  const int P = min(max(shared[0], 0), a.step.width);

  uint64_t* full = reinterpret_cast<uint64_t*>(smem) + warp * kStages;
  float4* scales = reinterpret_cast<float4*>(smem + OFF_SCALE) + warp * kStages;
  int2* spans = reinterpret_cast<int2*>(smem + OFF_ROWS);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + OFF_FLAG);
  uint8_t* ring = smem + OFF_RING + warp * kStages * kPageBytes;
  if (lane == 0) {
    for (int s = 0; s < kStages; ++s) mbar_init(&full[s], 1);
    if (warp == 0) *abort_flag = 0;
    fence_barrier_init();
  }

  // Which shared keys a row sees: [0, sinks) and from `lo` on; none if it is padding
  auto span_of = [&](int r, const int*& seq, int& t) -> int2 {
    const int i = r / TG;
    t = (r - i * TG) / G;
    seq = a.step.rows + static_cast<long>(grp * n + i) * a.step.ld;
    if (r >= rows || t >= min(seq[1], a.T)) return make_int2(0x7fffffff, 0);
    const KvSpan s = kv_span(a, seq[0] - seq[1] + t, seq[0], seq[2]);
    return make_int2(s.lo, seq[3] >= 0 ? seq[3] : a.sinks);
  };
  int lo_min, lo_max, sinks_min, sinks_max;
  {
    const int* seq;
    int t;
    const bool row = lane < R && r0 + lane < rows;
    const int2 s = row ? span_of(r0 + lane, seq, t) : make_int2(0x7fffffff, 0);
    const bool sees = s.x != 0x7fffffff;
    if (warp == 0 && lane < R) spans[lane] = s;
    lo_min = __reduce_min_sync(0xffffffffu, s.x);
    lo_max = __reduce_max_sync(0xffffffffu, sees ? s.x : 0);
    sinks_min = __reduce_min_sync(0xffffffffu, sees ? s.y : 0x7fffffff);
    sinks_max = __reduce_max_sync(0xffffffffu, s.y);
  }
  KvPages pages{0, 0, 0};
  if (lo_min != 0x7fffffff) pages = kv_pages_before(kv_pages(lo_min, P * kKvPage, sinks_max, a.step.width), P);
  const int part = rank * kWarps + warp, parts = ranks * kWarps;
  const int mine = pages.n > part ? (pages.n - part + parts - 1) / parts : 0;

  // Q: row g of each 8, channels 16c..16c+15
  uint4 qraw[NJ][2];
#pragma unroll
  for (int j = 0; j < NJ; ++j) {
    qraw[j][0] = qraw[j][1] = make_uint4(0, 0, 0, 0);
    const int r = r0 + j * 8 + g;
    if (r < rows) {
      const int i = r / TG, t = (r - i * TG) / G, h = r - i * TG - t * G;
      if (t < a.step.rows[static_cast<long>(grp * n + i) * a.step.ld + 1]) {
        const __nv_bfloat16* q = reinterpret_cast<const __nv_bfloat16*>(a.q) + (grp * n + i) * a.q_sb + t * a.q_st + (kh * G + h) * a.q_sh + 16 * c;
        qraw[j][0] = ld_global_v4(q);
        qraw[j][1] = ld_global_v4(q + 8);
      }
    }
  }
  __syncthreads();

  // the warp's next 32 pages, one a lane: block of codes (-1: not in the pool) and scales
  long block = -1;
  float ks = 0.f, vs = 0.f;
  int put = 0, put_stage = 0;
  auto issue = [&]() {  // the warp's next page
    if ((put & 31) == 0) {
      const int k = part + (put + lane) * parts;
      block = -1;
      if (k < pages.n) {
        const int id = shared[kKvInfo + pages.at(k)];
        if (static_cast<unsigned>(id) < static_cast<unsigned>(a.pool.pages)) {
          block = static_cast<long>(id) * a.pool.heads + kh;
          ks = a.pool.k_scale[block];
          vs = a.pool.v_scale[block];
        } else if (id != -1) {  // (that no sequence has any more: hidden by their spans)
          record_bad_index(status, id);
        }
      }
    }
    const long at = __shfl_sync(0xffffffffu, block, put & 31);
    const float kf = __shfl_sync(0xffffffffu, ks, put & 31), vf = __shfl_sync(0xffffffffu, vs, put & 31);
    if (lane == 0) {
      const long from = max(at, 0L) * 4096;
      uint64_t* bar = &full[put_stage];
      uint8_t* dst = ring + put_stage * kPageBytes;
      bulk_load(dst, a.pool.k + from, 4096, bar);
      bulk_load(dst + 4096, a.pool.v + from, 4096, bar);
      scales[put_stage] = make_float4(kf, vf, at >= 0 ? 1.f : 0.f, 0.f);
      mbar_arrive_expect_tx(bar, kPageBytes);
    }
    ++put;
    if (++put_stage == kStages) put_stage = 0;
  };
  for (int i = 0; i < min(mine, kStages); ++i) issue();

  uint32_t qf[NJ][4][2];
  float sl2[NJ][2];  // score factors of rows 8j + 2c and 8j + 2c + 1, which this lane's scores belong to
#pragma unroll
  for (int j = 0; j < NJ; ++j) {
    float x[16];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint32_t ws[4] = {qraw[j][i].x, qraw[j][i].y, qraw[j][i].z, qraw[j][i].w};
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
      qf[j][s][0] = pack_half(x[4 * s] * down, x[4 * s + 1] * down);
      qf[j][s][1] = pack_half(x[4 * s + 2] * down, x[4 * s + 3] * down);
    }
#pragma unroll
    for (int u = 0; u < 2; ++u) sl2[j][u] = __shfl_sync(0xffffffffu, up, (2 * c + u) * 4);
  }

  float m[NJ][2], l[NJ][2];
  float o[NJ][4][4];  // channels 16 i + g, + 8 of rows 8j + 2c, 2c + 1
#pragma unroll
  for (int j = 0; j < NJ; ++j) {
    m[j][0] = m[j][1] = -INFINITY;
    l[j][0] = l[j][1] = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int k = 0; k < 4; ++k) o[j][i][k] = 0.f;
  }

  const int krow = 16 * (g >> 1) + (g & 1);
  int st = 0, phase = 0;
  bool ok = true;
  for (int i = 0; i < mine; ++i) {
    ok = __all_sync(0xffffffffu, mbar_wait(&full[st], phase, abort_flag));
    if (!ok) break;
    const uint32_t sk = smem_u32(ring + st * kPageBytes), sv = sk + 4096;
    const float4 f = scales[st];
    const bool there = f.z != 0.f;
    const int key0 = pages.at(part + i * parts) * kKvPage;

    float s[NJ][4][4];  // keys krow + 4 t (and 2 behind it) of rows 8j + 2c, 2c + 1
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const uint4 w0 = lds128(sk + (krow + 4 * t) * 64 + c * 16), w1 = lds128(sk + (krow + 4 * t + 2) * 64 + c * 16);
      const uint32_t x0[4] = {w0.x, w0.y, w0.z, w0.w}, x1[4] = {w1.x, w1.y, w1.z, w1.w};
#pragma unroll
      for (int j = 0; j < NJ; ++j)
#pragma unroll
        for (int k = 0; k < 4; ++k) s[j][t][k] = 0.f;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint32_t av[4] = {half2_of(x0[k] & 0xffff), half2_of(x1[k] & 0xffff), half2_of(x0[k] >> 16), half2_of(x1[k] >> 16)};
#pragma unroll
        for (int j = 0; j < NJ; ++j) mma_f16(s[j][t], av, qf[j][k][0], qf[j][k][1]);
      }
    }
    // a page that every row of the tile sees whole needs no mask
    const bool whole = there && (key0 >= lo_max || key0 + kKvPage <= sinks_min);
    uint32_t pf[NJ][4][2];
    float alpha[NJ][2];
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      float p[4][4];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const float fu = sl2[j][u] * f.x;
        if (!whole) {
          const int2 span = spans[j * 8 + 2 * c + u];
          const uint32_t see = there ? static_cast<uint32_t>(kv_bits(KvSpan{span.x, 0x7fffffff}, span.y, key0) >> krow) : 0u;
#pragma unroll
          for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int k = 0; k < 2; ++k)
              if (!(see >> (4 * t + 2 * k) & 1)) s[j][t][2 * k + u] = -INFINITY;
        }
        float mx = fmaxf(fmaxf(s[j][0][u], s[j][0][2 + u]), fmaxf(s[j][1][u], s[j][1][2 + u]));
        mx = fmaxf(mx, fmaxf(fmaxf(s[j][2][u], s[j][2][2 + u]), fmaxf(s[j][3][u], s[j][3][2 + u])));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
        const float top = mx == -INFINITY ? m[j][u] : fmaxf(m[j][u], __fmul_rn(mx, fu));
        const float use = top == -INFINITY ? 0.f : top;
        alpha[j][u] = exp2f(m[j][u] - use);
        m[j][u] = top;
        float down = use - kHeadroom, by = fu;
        if (fabsf(use) >= kFar) {  // products rounded as the maximum's was: none passes it
#pragma unroll
          for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int k = 0; k < 2; ++k) s[j][t][2 * k + u] = __fadd_rn(__fmul_rn(s[j][t][2 * k + u], fu), -use);
          down = -kHeadroom;
          by = 1.f;
        }
        float sum = 0.f;
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const float x = s[j][t][2 * k + u];
            float w = exp2f(x * by - down);
            if (!whole && x == -INFINITY) w = 0.f;  // a masked score, whatever the factor is
            p[t][2 * k + u] = w;
            sum += w;
          }
        l[j][u] = l[j][u] * alpha[j][u] + sum;
      }
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        pf[j][t][0] = transpose8x8(pack_half(p[t][0], p[t][1]));
        pf[j][t][1] = transpose8x8(pack_half(p[t][2], p[t][3]));
      }
    }
    // tokens that no row of the tile sees are left out of P V whatever they hold
    uint32_t keep[4] = {~0u, ~0u, ~0u, ~0u};
    if (!(there && (key0 >= lo_min || key0 + kKvPage <= sinks_max))) {
      const uint32_t see = there ? static_cast<uint32_t>(kv_bits(KvSpan{lo_min, 0x7fffffff}, sinks_max, key0) >> (16 * c)) : 0u;
#pragma unroll
      for (int k = 0; k < 4; ++k) keep[k] = kv_bytes(see >> (4 * k));
    }
    const float vf = f.y * exp2f(-kHeadroom);
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const uint4 w0 = lds128(sv + (t * 16 + g) * 64 + c * 16), w1 = lds128(sv + (t * 16 + 8 + g) * 64 + c * 16);
      const uint32_t x0[4] = {w0.x & keep[0], w0.y & keep[1], w0.z & keep[2], w0.w & keep[3]};
      const uint32_t x1[4] = {w1.x & keep[0], w1.y & keep[1], w1.z & keep[2], w1.w & keep[3]};
      float d[NJ][4];
#pragma unroll
      for (int j = 0; j < NJ; ++j)
#pragma unroll
        for (int k = 0; k < 4; ++k) d[j][k] = 0.f;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint32_t av[4] = {half2_of(x0[k] & 0xffff), half2_of(x1[k] & 0xffff), half2_of(x0[k] >> 16), half2_of(x1[k] >> 16)};
#pragma unroll
        for (int j = 0; j < NJ; ++j) mma_f16(d[j], av, pf[j][k][0], pf[j][k][1]);
      }
#pragma unroll
      for (int j = 0; j < NJ; ++j)
#pragma unroll
        for (int k = 0; k < 4; ++k) o[j][t][k] = o[j][t][k] * alpha[j][k & 1] + d[j][k] * vf;
    }
    __syncwarp();  // every lane has read the stage
    if (put < mine) issue();
    if (++st == kStages) {
      st = 0;
      phase ^= 1;
    }
  }
  if (!ok) {
    if (lane == 0) {
      if (status) atomicCAS(status, 0, kStatusTimeoutEpilogue);
      *abort_flag = 1;
      const long long t0 = clock64();  // copies in flight land before the ring is reused
      for (int s = 0; s < kStages; ++s)
        for (int ph = 0; ph < 2; ++ph)
          while (!mbar_try_wait(&full[s], ph) && clock64() - t0 < kSpinLimitCycles / 8) {
          }
    }
    __syncwarp();
  }
  // ---- the warps' results: unnormalised O, m and l (whole sums), over the rings
#pragma unroll
  for (int j = 0; j < NJ; ++j)
#pragma unroll
    for (int u = 0; u < 2; ++u) {
#pragma unroll
      for (int x = 4; x < 32; x *= 2) l[j][u] += __shfl_xor_sync(0xffffffffu, l[j][u], x);
      l[j][u] *= exp2f(-kHeadroom);
      if (m[j][u] == -INFINITY && l[j][u] != 0.f) m[j][u] = 0.f;  // only NaN scores so far
    }
  __syncthreads();
  float* wo = reinterpret_cast<float*>(smem + OFF_RING);  // [warp][row][kPitch], then [warp][row] (m, l)
  float2* wml = reinterpret_cast<float2*>(wo + kWarps * R * kPitch);
#pragma unroll
  for (int j = 0; j < NJ; ++j)
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int r = j * 8 + 2 * c + u;
      float* w = wo + (warp * R + r) * kPitch + g;
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        w[t * 16] = o[j][t][u];
        w[t * 16 + 8] = o[j][t][2 + u];
      }
      if (g == 0) wml[warp * R + r] = make_float2(m[j][u], l[j][u]);
    }
  __syncthreads();
  float* out = a.part + (static_cast<long>(out_tile) * ranks + rank) * kv_past_floats(R);
  for (int i = threadIdx.x; i < R * 16; i += kThreads) {
    const int r = i >> 4, d = (i & 15) * 4;
    float top = -INFINITY, sum = 0.f;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) top = fmaxf(top, wml[w * R + r].x);
    if (top != -INFINITY) {
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float2 ml = wml[w * R + r];
        const float k = exp2f(ml.x - top);
        const float4 x = *reinterpret_cast<const float4*>(wo + (w * R + r) * kPitch + d);
        v.x += k * x.x;
        v.y += k * x.y;
        v.z += k * x.z;
        v.w += k * x.w;
        sum += k * ml.y;
      }
    }
    *reinterpret_cast<float4*>(out + r * 64 + d) = v;
    if (d == 0) *reinterpret_cast<float2*>(out + R * 64 + r * 2) = make_float2(top, sum);
  }
}

template <int NJ>
void launch(const KvAttendArgs& a, int dev, cudaStream_t stream) {
  static std::atomic<uint64_t> set{0};  // devices whose shared-memory limit is raised
  if (!(set.load() >> (dev & 63) & 1)) {
    check_cuda(cudaFuncSetAttribute(kv_attend_past<NJ>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_BYTES),
               "cudaFuncSetAttribute(kv_attend_past)");
    set.fetch_or(1ull << (dev & 63));
  }
  const long tiles = kv_past_tiles(a, 8 * NJ);
  const long ctas = a.step.B / a.step.branches * static_cast<long>(a.pool.heads) * tiles * a.past_ranks;
  if (ctas > 0x7fffffffL) throw std::runtime_error("kv_cache_attend: too many rows for one launch");
  kv_attend_past<NJ><<<static_cast<unsigned>(ctas), kThreads, SMEM_BYTES, stream>>>(a, static_cast<int>(tiles), device_status(dev));
  check_cuda(cudaGetLastError(), "kv_attend_past launch");
  count_launch();
}

}  // namespace

KvPlan kv_attend_past_plan(const KvAttendArgs& a, int dev) {
  KvPlan p;
  p.split = true;
  const long rows = kv_group_rows(a);
  p.past_rows = rows <= 8 ? 8 : rows <= 16 ? 16 : 32;
  const long items = a.step.B / a.step.branches * static_cast<long>(a.pool.heads) * kv_past_tiles(a, p.past_rows);
  const long seen = kv_seen_pages(a);  // visible ones, own pages among them
  const long pages = std::min<long>(a.shared_pages, seen);
  // as many CTAs as the device runs at once, none with less than a page a warp
  const long most = std::max(1L, (pages + kWarps - 1) / kWarps);
  p.past_ranks = static_cast<int>(std::clamp(num_sms(dev) / std::max(items, 1L), 1L, most));
  p.scratch = items * p.past_ranks * kv_past_floats(p.past_rows);
  return p;
}

void kv_attend_past_launch(const KvAttendArgs& a, int dev, cudaStream_t stream) {
  switch (a.past_rows) {
    case 8: launch<1>(a, dev, stream); break;
    case 16: launch<2>(a, dev, stream); break;
    default: launch<4>(a, dev, stream); break;
  }
}

}  // namespace ddb
