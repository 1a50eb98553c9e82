// Rotary positions of heads in three pair layouts, and norms of queries and keys in the same
// pass, forward and backward.
#pragma once
#include <cuda_runtime.h>
#include <cstdint>

namespace ddb {

enum class RotType { kBf16, kF16, kF32 };

// Where the two channels of pair i < R / 2 lie: side by side (2i, 2i + 1), or in halves
// (i, i + R / 2). A layout is the pair of both, read and written; channels from R on pass.
struct RotLayout {
  bool in_halves = false, out_halves = false;
};

// Heads of one tensor [B, T, H, D]: element strides, channels contiguous.
struct RotTensor {
  const void* x = nullptr;
  void* y = nullptr;         // forward: the result; backward: the gradient of x. May be x (forward), g (backward)
  const void* g = nullptr;   // backward: the result's gradient
  long x_sb = 0, x_st = 0, x_sh = 0;
  long y_sb = 0, y_st = 0, y_sh = 0;
  long g_sb = 0, g_st = 0, g_sh = 0;
  int H = 0;
  const float* w = nullptr;  // weight of each channel, or null (ones)
  float* dw = nullptr;       // backward: its gradient [D], or null
  bool dw_add = false;       // added to what dw holds
};

struct RotArgs {
  RotTensor t[2];
  int n = 1;                 // tensors
  RotType type = RotType::kBf16;
  RotLayout layout;
  bool inverse = false;      // by the negative angle (its layout given as it reads and writes)
  bool norm = false;
  int B = 0, T = 0, D = 0, R = 0;
  const float2* table = nullptr;  // (cos, sin) [places][R / 2]
  long places = 0;
  const void* pos = nullptr;      // position of each token, int32 or int64, or null: offset + t
  bool pos64 = false;
  long pos_sb = 0, pos_st = 0;
  long offset = 0;
  float eps = 0.f;
  float* part = nullptr;          // backward of a norm: rot_parts(a) floats
};

// Rotation of a.t[0 .. n), behind a division by each head's root mean square if a.norm.
void rot_forward(const RotArgs& a, cudaStream_t s);
// Gradients of the normed and rotated tensors' inputs and weights. x is the forward's input.
void rot_backward(const RotArgs& a, cudaStream_t s);
long rot_parts(const RotArgs& a);

}  // namespace ddb
