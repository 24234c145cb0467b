// The exact linear layer: argument blocks shared by its kernels.
//
//   pre = x w^T + bias,  y = act(pre) + residual          x (R, D), w (M, D)
//   dpre = dy * act'(pre),  dx = dpre w,  dw = dpre^T x,  db = column sums of dpre
#pragma once

#include "act8.cuh"

namespace scmp {
namespace lin {

__device__ __forceinline__ float act_value(int act, float v) {
  switch (act) {
    case SCMP_ACT_RELU:
      return v < 0.f ? 0.f : v;
    case SCMP_ACT_GELU:
      return 0.5f * v * (1.f + erff(v * 0.70710678118654752f));
    case SCMP_ACT_GELU_TANH: {
      const float u = 0.79788456080286536f * fmaf(0.044715f * v * v, v, v);
      return 0.5f * v * (1.f + tanhf(u));
    }
    case SCMP_ACT_SILU:
      return v / (1.f + expf(-v));
    default:
      return v;
  }
}
__device__ __forceinline__ float act_grad(int act, float v) {
  switch (act) {
    case SCMP_ACT_RELU:
      return v > 0.f ? 1.f : 0.f;
    case SCMP_ACT_GELU:
      return fmaf(v * 0.39894228040143268f, expf(-0.5f * v * v), 0.5f * (1.f + erff(v * 0.70710678118654752f)));
    case SCMP_ACT_GELU_TANH: {
      const float u = 0.79788456080286536f * fmaf(0.044715f * v * v, v, v);
      const float t = tanhf(u);
      return fmaf(0.5f * v * (1.f - t * t), 0.79788456080286536f * fmaf(0.134145f * v, v, 1.f), 0.5f * (1.f + t));
    }
    case SCMP_ACT_SILU: {
      const float s = 1.f / (1.f + expf(-v));
      return s * fmaf(v, 1.f - s, 1.f);
    }
    default:
      return 1.f;
  }
}

// What happens to an output element after the product's sum.
struct Epilogue {
  const void* bias;      // (m) or null
  int bias_f32;          // bias is float32, not the tensors' type
  const void* residual;  // or null
  long long ldr;
  int act;
  void* out;
  long long ldo;
  void* pre;             // the pre-activation in the tensors' type (rows of m), or null
  int8_t* codes;         // its 8-bit checkpoint, or null
  uint8_t* exps;
};

// A float32 value as three bfloat16 (leading 8 bits, the next 8, the last 8)
// whose sum it is. Truncated, so that no part overflows; an infinity or a NaN is
// the first part alone.
__device__ __forceinline__ void split3(float v, uint32_t (&part)[3]) {
  uint32_t u = __float_as_uint(v);
  const bool finite = (u & 0x7F800000u) != 0x7F800000u;
  if ((u & 0x7FFFFFFFu) > 0x7F800000u) u |= 0x00400000u;  // a NaN keeps a set mantissa bit
  part[0] = u >> 16;
  v = finite ? v - __uint_as_float(u & 0xFFFF0000u) : 0.f;
  u = __float_as_uint(v);
  part[1] = u >> 16;
  v -= __uint_as_float(u & 0xFFFF0000u);
  part[2] = __float_as_uint(v) >> 16;
}

}  // namespace lin
}  // namespace scmp
