// Writing tokens into the 8-bit paged cache, and moving its pages.
#include <cuda_bf16.h>
#include <cuda_fp8.h>

#include <algorithm>

#include "../common/ptx.cuh"
#include "../common/tma.h"
#include "kvcache.h"

namespace ddb {
namespace {

// smallest e with amax <= 448 * 2^e (448 = 1.75 * 2^8), kept in [-100, 119]: below, codes
// reach zero at 2^-109 (under any bf16 a model holds); above, 448 * 2^e would overflow
__device__ __forceinline__ int scale_exponent(float amax) {
  const uint32_t u = __float_as_uint(amax);
  const int k = static_cast<int>(u >> 23) - 127;
  const int e = k - 8 + ((u & 0x7fffff) > 0x600000 ? 1 : 0);
  return amax > 0.f ? min(max(e, -100), 119) : -100;
}
__device__ __forceinline__ float two_to(int e) { return __int_as_float((e + 127) << 23); }

__device__ __forceinline__ float2 unpack_e4m3(uint32_t two) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(two), __NV_E4M3);
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}
__device__ __forceinline__ uint32_t pack_e4m3(float a, float b) {
  return __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
}

constexpr int kVPitch = 80;  // bytes between channel rows of the value tile in shared memory

// One CTA = one page of one (sequence, head): a block's scale needs its maximum before its
// first code. Threads 0-127 keys, 128-255 values; two threads a token, 32 channels each. The
// page's tokens (kept ones decoded, new ones read) stay in registers between the maximum and
// the coding, so each byte moves once. Bound by latency: the loads of the table, of the page
// and of the tokens depend on one another. One token of 64 streams of 12 heads takes
// 6.6 us (its bytes 1.5 us at the copy rate), 2048 tokens of 4 streams 9.7 us (38 MB, 3.9 TB/s).
__global__ void __launch_bounds__(256) kv_write_kernel(const KvWriteArgs a, int* status) {
  const int b = blockIdx.z, h = blockIdx.y;
  const int* row = a.step.rows + static_cast<long>(b) * a.step.ld;
  const int len = row[0], own = min(row[1], a.T);
  const int old = len - row[1];
  const int j = old / kKvPage + blockIdx.x;
  if (own <= 0 || old < 0 || j * kKvPage >= old + own || j >= a.step.width) return;
  const int page = row[kKvInfo + j];
  if (static_cast<unsigned>(page) >= static_cast<unsigned>(a.pool.pages)) {
    if (threadIdx.x == 0) record_bad_index(status, page);
    return;
  }
  __shared__ __align__(16) uint8_t tile[64 * kVPitch];
  __shared__ float red[8];
  const bool is_v = threadIdx.x >= 128;
  const int t = threadIdx.x & 127;
  const int r = t >> 1, c0 = (t & 1) * 32;
  const long block = static_cast<long>(page) * a.pool.heads + h;
  uint8_t* codes = (is_v ? a.pool.v : a.pool.k) + block * 4096;
  float* scale = (is_v ? a.pool.v_scale : a.pool.k_scale) + block;
  const int pos = j * kKvPage + r;

  if (j * kKvPage < old) {  // uniform in the CTA: the page keeps tokens
    if (is_v) {
      const int d = t >> 1, o = (t & 1) * 32;
      const uint4* src = reinterpret_cast<const uint4*>(codes + d * 64 + o);
      *reinterpret_cast<uint4*>(tile + d * kVPitch + o) = src[0];
      *reinterpret_cast<uint4*>(tile + d * kVPitch + o + 16) = src[1];
    }
    __syncthreads();
  }
  float x[32];
#pragma unroll
  for (int i = 0; i < 32; ++i) x[i] = 0.f;
  if (pos < old) {
    const float s = *scale;
    if (is_v) {
#pragma unroll
      for (int i = 0; i < 32; i += 2) {
        const float2 f = unpack_e4m3(tile[(c0 + i) * kVPitch + r] | tile[(c0 + i + 1) * kVPitch + r] << 8);
        x[i] = f.x * s;
        x[i + 1] = f.y * s;
      }
    } else {
      const uint4* src = reinterpret_cast<const uint4*>(codes + r * 64 + c0);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint4 w = src[i];
        const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const float2 lo = unpack_e4m3(ws[u] & 0xffff), hi = unpack_e4m3(ws[u] >> 16);
          x[i * 16 + u * 4 + 0] = lo.x * s;
          x[i * 16 + u * 4 + 1] = lo.y * s;
          x[i * 16 + u * 4 + 2] = hi.x * s;
          x[i * 16 + u * 4 + 3] = hi.y * s;
        }
      }
    }
  } else if (pos < old + own) {
    const __nv_bfloat16* src =
        is_v ? reinterpret_cast<const __nv_bfloat16*>(a.v) + b * a.v_sb + (pos - old) * a.v_st + h * a.v_sh
             : reinterpret_cast<const __nv_bfloat16*>(a.k) + b * a.k_sb + (pos - old) * a.k_st + h * a.k_sh;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint4 w = ld_global_v4(src + c0 + i * 8);
      const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const float2 f = unpack_bf16(ws[u]);
        x[i * 8 + u * 2] = f.x;
        x[i * 8 + u * 2 + 1] = f.y;
      }
    }
  }
  float amax = 0.f;  // of the finite values: an infinity saturates, a NaN keeps its code
#pragma unroll
  for (int i = 0; i < 32; ++i) {
    const float m = fabsf(x[i]);
    amax = m <= 3.4028234e38f ? fmaxf(amax, m) : amax;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = amax;
  __syncthreads();  // also: every kept value has left the tile
  const float* rd = red + (is_v ? 4 : 0);
  const int e = scale_exponent(fmaxf(fmaxf(rd[0], rd[1]), fmaxf(rd[2], rd[3])));
  const float inv = two_to(-e);
  uint32_t w[8];
#pragma unroll
  for (int i = 0; i < 8; ++i)
    w[i] = pack_e4m3(x[4 * i] * inv, x[4 * i + 1] * inv) | pack_e4m3(x[4 * i + 2] * inv, x[4 * i + 3] * inv) << 16;
  if (is_v) {
#pragma unroll
    for (int i = 0; i < 32; ++i)
      tile[(c0 + i) * kVPitch + r] = static_cast<uint8_t>(w[i >> 2] >> (8 * (i & 3)));
  } else {
    uint4* dst = reinterpret_cast<uint4*>(codes + r * 64 + c0);
    dst[0] = make_uint4(w[0], w[1], w[2], w[3]);
    dst[1] = make_uint4(w[4], w[5], w[6], w[7]);
  }
  if (t == 0) *scale = two_to(e);
  __syncthreads();
  if (is_v) {
    const int d = t >> 1, o = (t & 1) * 32;
    uint4* dst = reinterpret_cast<uint4*>(codes + d * 64 + o);
    dst[0] = *reinterpret_cast<const uint4*>(tile + d * kVPitch + o);
    dst[1] = *reinterpret_cast<const uint4*>(tile + d * kVPitch + o + 16);
  }
}

constexpr int kPairs = 256;
struct PagePairs {
  int src[kPairs];
  int dst[kPairs];
};

// blockIdx.x: the pair, y: the layer, z: keys or values. A page of one layer is heads * 4 KB
// in one piece. The pairs travel as launch arguments: no copy to the device comes first, and
// no call waits for an earlier one's upload. Four loads in flight a thread. Bound by memory:
// 256 pages of 12 heads and 12 layers (302 MB read, as much written) take 93 us, 6.5 TB/s.
__global__ void __launch_bounds__(256)
    kv_copy_kernel(uint8_t* k, uint8_t* v, float* k_scale, float* v_scale, int pages, int heads,
                   const __grid_constant__ PagePairs pairs) {
  uint8_t* base = blockIdx.z ? v : k;
  float* scales = blockIdx.z ? v_scale : k_scale;
  const long layer = static_cast<long>(blockIdx.y) * pages;
  const long from = (layer + pairs.src[blockIdx.x]) * heads, to = (layer + pairs.dst[blockIdx.x]) * heads;
  const uint4* s = reinterpret_cast<const uint4*>(base + from * 4096);
  uint4* d = reinterpret_cast<uint4*>(base + to * 4096);
  const int n = heads * 256;  // a multiple of the block
  int i = threadIdx.x;
  for (; i + 768 < n; i += 1024) {
    const uint4 w0 = s[i], w1 = s[i + 256], w2 = s[i + 512], w3 = s[i + 768];
    d[i] = w0;
    d[i + 256] = w1;
    d[i + 512] = w2;
    d[i + 768] = w3;
  }
  for (; i < n; i += 256) d[i] = s[i];
  for (int c = threadIdx.x; c < heads; c += 256) scales[to + c] = scales[from + c];
}

}  // namespace

void kv_cache_write(const KvWriteArgs& a, cudaStream_t stream) {
  if (a.step.B <= 0 || a.T <= 0 || a.pool.heads <= 0) return;
  int dev = 0;
  check_cuda(cudaGetDevice(&dev), "cudaGetDevice");
  // T tokens touch at most (T + 62) / 64 + 1 pages
  const dim3 grid(std::min((a.T + kKvPage - 2) / kKvPage + 1, a.step.width), a.pool.heads, a.step.B);
  if (grid.x == 0) return;
  kv_write_kernel<<<grid, 256, 0, stream>>>(a, device_status(dev));
  count_launch();
  check_cuda(cudaGetLastError(), "kv_write_kernel launch");
}

void kv_cache_copy_pages(uint8_t* k, uint8_t* v, float* k_scale, float* v_scale, int layers,
                         int pages, int heads, const int* src, const int* dst, int n,
                         cudaStream_t stream) {
  if (layers <= 0 || heads <= 0) return;
  for (int i = 0; i < n; i += kPairs) {
    const int m = std::min(kPairs, n - i);
    PagePairs p;
    std::copy(src + i, src + i + m, p.src);
    std::copy(dst + i, dst + i + m, p.dst);
    kv_copy_kernel<<<dim3(m, layers, 2), 256, 0, stream>>>(k, v, k_scale, v_scale, pages, heads, p);
    count_launch();
    check_cuda(cudaGetLastError(), "kv_copy_kernel launch");
  }
}

}  // namespace ddb
