// Rotary positions and per-head norms of queries and keys.
//
//   forward    h = x r w, r = (mean x^2 + eps)^-1/2 (without a norm h = x); each pair (a, b) of
//              h becomes (a c - b s, a s + b c), (c, s) from the table's row of its token
//   backward   g = the transposed rotation of dy; dw = sum g x r; u = g w; with h = x r
//              dx = r (u - h mean(u h))
// r is made again from x in the backward: nothing but x is kept between the two.
//
// Bound by memory: every value is read and written once. Wide heads (rot_wide): 16 channels
// to a lane, as two runs of 8 that hold 8 whole pairs in either layout, so that a pair never
// leaves its lane and both layouts take 16-byte accesses; D / 16 lanes make a head, its sum of
// squares is a shuffle over them. A lane's pairs are 8 l .. 8 l + 7 in every layout, so its
// 64 bytes of the table are contiguous; the heads of a token find them in L1. Heads whose
// sizes, strides or bases do not allow that (rot_any): 8 or 16 lanes a head, a channel pair at
// a time.
// Everything is fp32 inside, without contraction of a c - b s (the same bits as the PyTorch
// statement of the rotation), rounded once.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <stdexcept>

#include "../common/ptx.cuh"
#include "../common/tma.h"
#include "rotary.h"

namespace ddb {
namespace {

constexpr int kThreads = 256;

// n / d for n < 2^31 (round-up multiplication)
struct Div {
  uint32_t m = 0, s = 0;
  Div() = default;
  explicit Div(uint32_t n) {
    const uint32_t d = n ? n : 1;
    while ((1ull << s) < d) ++s;
    m = static_cast<uint32_t>(((1ull << 32) * ((1ull << s) - d)) / d + 1);
  }
  __device__ __forceinline__ uint32_t operator()(uint32_t n) const { return (__umulhi(n, m) + n) >> s; }
};

struct Launch {
  RotArgs a;
  Div by_T, by_H[2];
  int ctas0 = 0;       // CTAs of the first tensor
  int ctas1 = 0;
  int log_lanes = 0;   // lanes of a head
  int* status = nullptr;
};

template <typename T>
struct Io;
template <>
struct Io<__nv_bfloat16> {
  static __device__ __forceinline__ float get(const __nv_bfloat16* p) { return __bfloat162float(*p); }
  static __device__ __forceinline__ void put(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }
  static __device__ __forceinline__ void get8(const __nv_bfloat16* p, float* v) {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = __uint_as_float(w[i] << 16);
      v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
  static __device__ __forceinline__ void put8(__nv_bfloat16* p, const float* v) {
    *reinterpret_cast<uint4*>(p) = make_uint4(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7]));
  }
};
template <>
struct Io<__half> {
  static __device__ __forceinline__ float get(const __half* p) { return __half2float(*p); }
  static __device__ __forceinline__ void put(__half* p, float v) { *p = __float2half_rn(v); }
  static __device__ __forceinline__ void get8(const __half* p, float* v) {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      v[2 * i] = f.x;
      v[2 * i + 1] = f.y;
    }
  }
  static __device__ __forceinline__ void put8(__half* p, const float* v) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __half2 h = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  }
};
template <>
struct Io<float> {
  static __device__ __forceinline__ float get(const float* p) { return *p; }
  static __device__ __forceinline__ void put(float* p, float v) { *p = v; }
  static __device__ __forceinline__ void get8(const float* p, float* v) {
    const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
  }
  static __device__ __forceinline__ void put8(float* p, const float* v) {
    *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
    *reinterpret_cast<float4*>(p + 4) = make_float4(v[4], v[5], v[6], v[7]);
  }
};

// One (token, head): where its channels lie, and its row of the table (-1: no such row)
struct Item {
  long b, t, h;
  long row;
  bool there;
};

__device__ __forceinline__ Item item_of(const Launch& L, int which, uint32_t i, uint32_t n) {
  const RotArgs& a = L.a;
  Item it;
  it.there = i < n;
  const uint32_t token = L.by_H[which](it.there ? i : 0);
  it.h = (it.there ? i : 0) - token * a.t[which].H;
  const uint32_t b = L.by_T(token);
  it.b = b;
  it.t = token - b * a.T;
  it.row = 0;
  if (a.R > 0 && it.there) {
    if (a.pos) {
      const long at = it.b * a.pos_sb + it.t * a.pos_st;
      it.row = a.pos64 ? reinterpret_cast<const long long*>(a.pos)[at] : reinterpret_cast<const int*>(a.pos)[at];
      if (it.row < 0 || it.row >= a.places) {  // recorded; the token's rotated channels become NaN
        record_bad_index(L.status, it.row);
        it.row = -1;
      }
    } else {
      it.row = a.offset + it.t;
    }
  }
  return it;
}

__device__ __forceinline__ float2 turn(float x, float y, float c, float s) {
  return make_float2(__fsub_rn(__fmul_rn(x, c), __fmul_rn(y, s)), __fadd_rn(__fmul_rn(x, s), __fmul_rn(y, c)));
}

// (mean + eps)^-1/2 of a sum of squares. `down`: a power of two by which the squares' roots were
// brought down so that the sum stays finite.
__device__ __forceinline__ float rms_inv(float sum, float D, float eps, float down) {
  return __frcp_rn(__fsqrt_rn(__fdiv_rn(sum, D) + eps * down * down));
}
constexpr float kDown = 0x1p-70f;  // its square times a sum of 256 squares of the largest fp32 is finite

template <typename T, bool IN_H, bool OUT_H, bool NORM, bool BWD, int U>
__global__ void __launch_bounds__(kThreads, 2) rot_wide(const Launch L) {
  const RotArgs& a = L.a;
  const int which = blockIdx.x >= L.ctas0;
  const RotTensor& t = a.t[which];
  const int lg = L.log_lanes, l = threadIdx.x & ((1 << lg) - 1);
  const bool active = l < a.D >> 4, rot = l < a.R >> 4;
  const uint32_t n = static_cast<uint32_t>(a.B) * a.T * t.H;
  const uint32_t per = kThreads >> lg;
  const int in0 = rot && IN_H ? 8 * l : 16 * l, in1 = rot && IN_H ? a.R / 2 + 8 * l : 16 * l + 8;
  const int out0 = rot && OUT_H ? 8 * l : 16 * l, out1 = rot && OUT_H ? a.R / 2 + 8 * l : 16 * l + 8;
  float w[16], dw[16];
  if (NORM) {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      w[i] = t.w && active ? t.w[(i < 8 ? in0 : in1) + (i & 7)] : 1.f;
      dw[i] = 0.f;
    }
  }
  const uint32_t cta = blockIdx.x - (which ? L.ctas0 : 0), ctas = which ? L.ctas1 : L.ctas0;
  for (uint32_t i0 = cta * per * U; i0 < n; i0 += ctas * per * U) {  // one turn in the forward
    float v[U][16], g[U][16];
    Item it[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      it[u] = item_of(L, which, i0 + u * per + (threadIdx.x >> lg), n);
      if (it[u].there && active) {
        const T* x = reinterpret_cast<const T*>(t.x) + it[u].b * t.x_sb + it[u].t * t.x_st + it[u].h * t.x_sh;
        Io<T>::get8(x + in0, v[u]);
        Io<T>::get8(x + in1, v[u] + 8);
        if (BWD) {
          const T* y = reinterpret_cast<const T*>(t.g) + it[u].b * t.g_sb + it[u].t * t.g_st + it[u].h * t.g_sh;
          Io<T>::get8(y + out0, g[u]);
          Io<T>::get8(y + out1, g[u] + 8);
        }
      } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) v[u][i] = g[u][i] = 0.f;
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float r = 1.f;
      if (NORM) {
        float down = 1.f;
        auto sum = [&]() {
          float s = 0.f;
#pragma unroll
          for (int i = 0; i < 16; ++i) s = fmaf(v[u][i], v[u][i], s);
          for (int o = 1; o < 1 << lg; o *= 2) s += __shfl_xor_sync(0xffffffffu, s, o);
          return s;
        };
        float s = sum();
        if (__any_sync(0xffffffffu, !(s < 1e38f))) {  // squares too large for fp32, infinities, NaN
          if (!(s < 1e38f)) down = kDown;
#pragma unroll
          for (int i = 0; i < 16; ++i) v[u][i] *= down;
          s = sum();
        }
        r = rms_inv(s, static_cast<float>(a.D), a.eps, down);
        if (BWD) {
#pragma unroll
          for (int i = 0; i < 16; ++i) v[u][i] *= r;
          r *= down;
        } else {
#pragma unroll
          for (int i = 0; i < 16; ++i) v[u][i] = v[u][i] * r * w[i];
        }
      }
      float z[16];  // the rotated, or rotated back
      const float* from = BWD ? g[u] : v[u];
      if (a.R > 0) {
        float2 cs[8];
        if (rot && it[u].there && it[u].row >= 0) {
          const float4* tab = reinterpret_cast<const float4*>(a.table + it[u].row * (a.R / 2) + 8 * l);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float4 f = __ldg(tab + i);
            cs[2 * i] = make_float2(f.x, f.y);
            cs[2 * i + 1] = make_float2(f.z, f.w);
          }
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) cs[i] = make_float2(NAN, NAN);
        }
        const bool back = a.inverse;  // the backward of a rotation is its inverse
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          // forward: pairs as they are read, to where they are written; backward: the other way
          constexpr bool kFrom = BWD ? OUT_H : IN_H, kTo = BWD ? IN_H : OUT_H;
          const int f0 = kFrom ? j : 2 * j, f1 = kFrom ? j + 8 : 2 * j + 1;
          const int t0 = kTo ? j : 2 * j, t1 = kTo ? j + 8 : 2 * j + 1;
          const float2 q = turn(from[f0], from[f1], cs[j].x, back != BWD ? -cs[j].y : cs[j].y);
          z[t0] = q.x;
          z[t1] = q.y;
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) z[i] = rot ? z[i] : from[i];
      } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) z[i] = from[i];
      }
      if (BWD) {
        float m = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          if (it[u].there) dw[i] = fmaf(z[i], v[u][i], dw[i]);
          z[i] *= w[i];
          m = fmaf(z[i], v[u][i], m);
        }
        for (int o = 1; o < 1 << lg; o *= 2) m += __shfl_xor_sync(0xffffffffu, m, o);
        m = __fdiv_rn(m, static_cast<float>(a.D));
#pragma unroll
        for (int i = 0; i < 16; ++i) v[u][i] = r * (z[i] - v[u][i] * m);
      } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) v[u][i] = z[i];
      }
    }
    __syncwarp();  // every lane has read what another one may write (a result in the place of its input)
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (it[u].there && active) {
        T* y = reinterpret_cast<T*>(t.y) + it[u].b * t.y_sb + it[u].t * t.y_st + it[u].h * t.y_sh;
        Io<T>::put8(y + (BWD ? in0 : out0), v[u]);
        Io<T>::put8(y + (BWD ? in1 : out1), v[u] + 8);
      }
    if (!BWD) break;
  }
  if (BWD) {
    // the CTA's sums of each channel: lanes of a warp, then warps, in a fixed order
    __shared__ float red[kThreads / 32][256];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      for (int o = 1 << lg; o < 32; o *= 2) dw[i] += __shfl_xor_sync(0xffffffffu, dw[i], o);
      if ((threadIdx.x & 31) == l && active) red[threadIdx.x >> 5][(i < 8 ? in0 : in1) + (i & 7)] = dw[i];
    }
    __syncthreads();
    for (int c = threadIdx.x; c < a.D; c += kThreads) {
      float s = 0.f;
#pragma unroll
      for (int k = 0; k < kThreads / 32; ++k) s += red[k][c];
      a.part[static_cast<long>(blockIdx.x) * a.D + c] = s;
    }
  }
}

// Heads of any even size up to 256, any strides: 8 lanes (16 above 128 channels) a head, 8 pairs a lane.
template <typename T, bool NORM, bool BWD>
__global__ void __launch_bounds__(kThreads) rot_any(const Launch L) {
  const RotArgs& a = L.a;
  const int which = blockIdx.x >= L.ctas0;
  const RotTensor& t = a.t[which];
  const int lg = L.log_lanes, l = threadIdx.x & ((1 << lg) - 1);
  const uint32_t n = static_cast<uint32_t>(a.B) * a.T * t.H, per = kThreads >> lg;
  const int pairs = a.D / 2, turned = a.R / 2;
  // channels of a lane's pair i as one side has them
  auto chan = [&](int i, bool halves, int& c0, int& c1) {
    const int p = l + (i << lg);
    if (p < turned && halves) c0 = p, c1 = p + turned;
    else c0 = 2 * p, c1 = 2 * p + 1;
    return p < pairs;
  };
  float dw[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) dw[i] = 0.f;
  const uint32_t cta = blockIdx.x - (which ? L.ctas0 : 0), ctas = which ? L.ctas1 : L.ctas0;
  for (uint32_t i0 = cta * per; i0 < n; i0 += ctas * per) {
    const Item it = item_of(L, which, i0 + (threadIdx.x >> lg), n);
    const T* x = reinterpret_cast<const T*>(t.x) + it.b * t.x_sb + it.t * t.x_st + it.h * t.x_sh;
    const T* dy = reinterpret_cast<const T*>(t.g) + it.b * t.g_sb + it.t * t.g_st + it.h * t.g_sh;
    T* y = reinterpret_cast<T*>(t.y) + it.b * t.y_sb + it.t * t.y_st + it.h * t.y_sh;
    float v[16], g[16];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      int c0, c1;
      v[2 * i] = v[2 * i + 1] = g[2 * i] = g[2 * i + 1] = 0.f;
      if (chan(i, a.layout.in_halves, c0, c1) && it.there) v[2 * i] = Io<T>::get(x + c0), v[2 * i + 1] = Io<T>::get(x + c1);
      if (BWD && chan(i, a.layout.out_halves, c0, c1) && it.there) g[2 * i] = Io<T>::get(dy + c0), g[2 * i + 1] = Io<T>::get(dy + c1);
    }
    float r = 1.f;
    if (NORM) {
      float down = 1.f;
      auto sum = [&]() {
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) s = fmaf(v[i], v[i], s);
        for (int o = 1; o < 1 << lg; o *= 2) s += __shfl_xor_sync(0xffffffffu, s, o);
        return s;
      };
      float s = sum();
      if (__any_sync(0xffffffffu, !(s < 1e38f))) {
        if (!(s < 1e38f)) down = kDown;
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] *= down;
        s = sum();
      }
      r = rms_inv(s, static_cast<float>(a.D), a.eps, down);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        int c0, c1;
        v[2 * i] *= r, v[2 * i + 1] *= r;
        if (!BWD && chan(i, a.layout.in_halves, c0, c1) && t.w) v[2 * i] *= t.w[c0], v[2 * i + 1] *= t.w[c1];
      }
      r *= down;
    }
    float* z = BWD ? g : v;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int p = l + (i << lg);
      if (p < turned) {
        float2 cs = make_float2(NAN, NAN);
        if (it.there && it.row >= 0) cs = __ldg(a.table + it.row * turned + p);
        const float2 q = turn(z[2 * i], z[2 * i + 1], cs.x, a.inverse != BWD ? -cs.y : cs.y);
        z[2 * i] = q.x;
        z[2 * i + 1] = q.y;
      }
    }
    if (BWD) {
      float m = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        int c0, c1;
        const bool have = chan(i, a.layout.in_halves, c0, c1);
        if (have && it.there) dw[2 * i] = fmaf(g[2 * i], v[2 * i], dw[2 * i]), dw[2 * i + 1] = fmaf(g[2 * i + 1], v[2 * i + 1], dw[2 * i + 1]);
        if (have && t.w) g[2 * i] *= t.w[c0], g[2 * i + 1] *= t.w[c1];
        m = fmaf(g[2 * i], v[2 * i], m);
        m = fmaf(g[2 * i + 1], v[2 * i + 1], m);
      }
      for (int o = 1; o < 1 << lg; o *= 2) m += __shfl_xor_sync(0xffffffffu, m, o);
      m = __fdiv_rn(m, static_cast<float>(a.D));
#pragma unroll
      for (int i = 0; i < 16; ++i) v[i] = r * (g[i] - v[i] * m);
    }
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      int c0, c1;
      if (chan(i, BWD ? a.layout.in_halves : a.layout.out_halves, c0, c1) && it.there) Io<T>::put(y + c0, v[2 * i]), Io<T>::put(y + c1, v[2 * i + 1]);
    }
  }
  if (BWD) {
    __shared__ float red[kThreads / 32][256];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      int c0, c1;
      const bool have = chan(i, a.layout.in_halves, c0, c1);
      for (int o = 1 << lg; o < 32; o *= 2) {
        dw[2 * i] += __shfl_xor_sync(0xffffffffu, dw[2 * i], o);
        dw[2 * i + 1] += __shfl_xor_sync(0xffffffffu, dw[2 * i + 1], o);
      }
      if ((threadIdx.x & 31) == l && have) red[threadIdx.x >> 5][c0] = dw[2 * i], red[threadIdx.x >> 5][c1] = dw[2 * i + 1];
    }
    __syncthreads();
    for (int c = threadIdx.x; c < a.D; c += kThreads) {
      float s = 0.f;
#pragma unroll
      for (int k = 0; k < kThreads / 32; ++k) s += red[k][c];
      a.part[static_cast<long>(blockIdx.x) * a.D + c] = s;
    }
  }
}

// The weights' gradients from the CTAs' sums, in a fixed order: 32 channels a block, 32 threads each.
__global__ void __launch_bounds__(1024) rot_weight_grad(const Launch L) {
  const RotArgs& a = L.a;
  const int which = blockIdx.y, c = blockIdx.x * 32 + (threadIdx.x & 31), k = threadIdx.x >> 5;
  const int ctas = which ? L.ctas1 : L.ctas0;
  __shared__ double red[32][33];
  double s = 0.;
  if (c < a.D && a.t[which].dw) {
    const float* p = a.part + static_cast<long>(which ? L.ctas0 : 0) * a.D + c;
    for (int i = k; i < ctas; i += 32) s += p[static_cast<long>(i) * a.D];
  }
  red[k][threadIdx.x & 31] = s;
  __syncthreads();
  if (k == 0 && c < a.D && a.t[which].dw) {
    for (int i = 1; i < 32; ++i) s += red[i][threadIdx.x];
    float* dw = a.t[which].dw + c;
    *dw = a.t[which].dw_add ? static_cast<float>(*dw + s) : static_cast<float>(s);
  }
}

int size_of(RotType t) { return t == RotType::kF32 ? 4 : 2; }

// 16-byte accesses of runs of 8 channels: heads of whole 16s, rotated channels too
bool wide(const RotArgs& a, bool bwd) {
  const int size = size_of(a.type);
  if (a.D % 16 || a.R % 16 || reinterpret_cast<uintptr_t>(a.table) % 16) return false;
  auto ok = [&](const void* p, long sb, long st, long sh) {
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && sb * size % 16 == 0 && st * size % 16 == 0 && sh * size % 16 == 0;
  };
  for (int i = 0; i < a.n; ++i) {
    const RotTensor& t = a.t[i];
    if (!ok(t.x, t.x_sb, t.x_st, t.x_sh) || !ok(t.y, t.y_sb, t.y_st, t.y_sh)) return false;
    if (bwd && !ok(t.g, t.g_sb, t.g_st, t.g_sh)) return false;
  }
  return true;
}

constexpr int unroll(bool bwd) { return bwd ? 1 : 2; }  // heads of a lane at once

int log2_up(int n) {
  int lg = 0;
  while (1 << lg < n) ++lg;
  return lg;
}

Launch plan(const RotArgs& a, bool bwd, bool is_wide, int dev) {
  Launch L;
  L.a = a;
  L.log_lanes = is_wide ? log2_up(a.D / 16) : a.D <= 128 ? 3 : 4;
  L.by_T = Div(a.T);
  L.status = device_status(dev);
  const long per = (kThreads >> L.log_lanes) * (is_wide ? unroll(bwd) : 1);
  long need[2] = {0, 0};
  for (int i = 0; i < a.n; ++i) {
    L.by_H[i] = Div(a.t[i].H);
    need[i] = (static_cast<long>(a.B) * a.T * a.t[i].H + per - 1) / per;
  }
  if (bwd || !is_wide) {  // CTAs that stay: their sums of the weights' gradients are added up behind them
    const long room = static_cast<long>(num_sms(dev)) * (bwd ? 2 : 8);
    const long all = need[0] + need[1];
    if (all > room)
      for (int i = 0; i < a.n; ++i) need[i] = std::max(1L, need[i] * room / all);
  }
  L.ctas0 = static_cast<int>(need[0]);
  L.ctas1 = static_cast<int>(need[1]);
  return L;
}

template <typename T, bool NORM, bool BWD>
void launch(const Launch& L, bool is_wide, cudaStream_t s) {
  const int grid = L.ctas0 + L.ctas1;
  const bool ih = L.a.layout.in_halves, oh = L.a.layout.out_halves;
  if (!is_wide) rot_any<T, NORM, BWD><<<grid, kThreads, 0, s>>>(L);
  else if (!ih && !oh) rot_wide<T, false, false, NORM, BWD, unroll(BWD)><<<grid, kThreads, 0, s>>>(L);
  else if (ih && oh) rot_wide<T, true, true, NORM, BWD, unroll(BWD)><<<grid, kThreads, 0, s>>>(L);
  else if (oh) rot_wide<T, false, true, NORM, BWD, unroll(BWD)><<<grid, kThreads, 0, s>>>(L);
  else if constexpr (!NORM) rot_wide<T, true, false, NORM, BWD, unroll(BWD)><<<grid, kThreads, 0, s>>>(L);
  else throw std::runtime_error("rotary: a norm is not behind an inverse rotation");
  check_cuda(cudaGetLastError(), "rotary launch");
  count_launch();
}

template <bool NORM, bool BWD>
void launch(const Launch& L, bool is_wide, cudaStream_t s) {
  switch (L.a.type) {
    case RotType::kBf16: launch<__nv_bfloat16, NORM, BWD>(L, is_wide, s); break;
    case RotType::kF16: launch<__half, NORM, BWD>(L, is_wide, s); break;
    default: launch<float, NORM, BWD>(L, is_wide, s);
  }
}

void check(const RotArgs& a) {
  long items = 0;
  for (int i = 0; i < a.n; ++i) items = std::max(items, static_cast<long>(a.B) * a.T * a.t[i].H);
  if (a.n < 1 || a.n > 2 || a.D < 2 || a.D > 256 || a.D % 2 || a.R < 0 || a.R > a.D || a.R % 2 || items >= 1L << 30)
    throw std::runtime_error("rotary: sizes out of range");
}

int current_device() {
  int dev = 0;
  check_cuda(cudaGetDevice(&dev), "cudaGetDevice");
  return dev;
}

}  // namespace

void rot_forward(const RotArgs& a, cudaStream_t s) {
  check(a);
  const bool w = wide(a, false);
  const Launch L = plan(a, false, w, current_device());
  if (L.ctas0 + L.ctas1 == 0) return;
  if (a.norm) launch<true, false>(L, w, s);
  else launch<false, false>(L, w, s);
}

long rot_parts(const RotArgs& a) {
  const Launch L = plan(a, true, wide(a, true), current_device());
  return (static_cast<long>(L.ctas0) + L.ctas1) * a.D;
}

void rot_backward(const RotArgs& a, cudaStream_t s) {
  check(a);
  const bool w = wide(a, true);
  const Launch L = plan(a, true, w, current_device());
  if (L.ctas0 + L.ctas1 > 0) launch<true, true>(L, w, s);
  if (a.t[0].dw || (a.n > 1 && a.t[1].dw)) {
    rot_weight_grad<<<dim3((a.D + 31) / 32, a.n), 1024, 0, s>>>(L);
    check_cuda(cudaGetLastError(), "rotary weight gradient launch");
    count_launch();
  }
}

}  // namespace ddb
