// The exact linear layer: argument blocks shared by its kernels.
//
//   pre = x w^T + bias,  y = act(pre) + residual          x (R, D), w (M, D)
//   dpre = dy * act'(pre),  dx = dpre w,  dw = dpre^T x,  db = column sums of dpre
#pragma once

#include "act8.cuh"

namespace scmp {
namespace lin {

// The activations are evaluated for every element of a large product, so they
// use the hardware's exp2 and reciprocal (a few 2^-23 relative each; results
// below 2^-126 are zero).
__device__ __forceinline__ float reciprocal(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float exp2_fast(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// Phi(-z) = erfc(z / sqrt 2) / 2 for z >= 0, and e = exp(-z^2 / 2):
// exp(z^2 / 2) Phi(-z) as a polynomial in t = 1 / (1 + 0.3 z), least relative
// error over z in [0, 14] (1.5e-7; below that exp(-98) the product is nothing).
// Relative error in float32 5e-7, so the tail of gelu keeps its digits.
__device__ __forceinline__ float normal_tail(float z, float& e) {
  const float t = reciprocal(fmaf(0.3f, z, 1.f));
  float p = 0.03567476570606232f;
  p = fmaf(p, t, -0.15720303356647491f);
  p = fmaf(p, t, 0.20635342597961426f);
  p = fmaf(p, t, -0.0536835603415966f);
  p = fmaf(p, t, 0.1285615712404251f);
  p = fmaf(p, t, 0.09991350769996643f);
  p = fmaf(p, t, 0.1207539513707161f);
  p = fmaf(p, t, 0.11962930113077164f);
  e = exp2_fast(-0.72134752044448170f * z * z);
  return p * t * e;
}
__device__ __forceinline__ float sigmoid(float v) { return reciprocal(1.f + exp2_fast(-1.4426950408889634f * v)); }
// exp(-v), finite: 1 - sigmoid(v) = exp(-v) sigmoid(v) keeps its digits where
// sigmoid(v) is near 1.
__device__ __forceinline__ float exp_minus(float v) { return exp2_fast(fminf(-1.4426950408889634f * v, 115.f)); }
// 0.5 (1 + tanh u) = sigmoid(2 u)
__device__ __forceinline__ float gelu_tanh_arg(float v) { return 1.5957691216057308f * fmaf(0.044715f * v * v, v, v); }

__device__ __forceinline__ float act_value(int act, float v) {
  switch (act) {
    case SCMP_ACT_RELU:
      return v < 0.f ? 0.f : v;
    case SCMP_ACT_GELU: {
      float e;
      const float q = normal_tail(fabsf(v), e);
      return v * (v >= 0.f ? 1.f - q : q);
    }
    case SCMP_ACT_GELU_TANH:
      return v * sigmoid(gelu_tanh_arg(v));
    case SCMP_ACT_SILU:
      return v * sigmoid(v);
    default:
      return v;
  }
}
__device__ __forceinline__ float act_grad(int act, float v) {
  switch (act) {
    case SCMP_ACT_RELU:
      return v > 0.f ? 1.f : 0.f;
    case SCMP_ACT_GELU: {
      float e;
      const float q = normal_tail(fabsf(v), e);
      return fmaf(v * 0.39894228040143268f, e, v >= 0.f ? 1.f - q : q);
    }
    case SCMP_ACT_GELU_TANH: {
      const float e = exp_minus(gelu_tanh_arg(v)), s = reciprocal(1.f + e);
      return fmaf(v * (e * s * s), 1.5957691216057308f * fmaf(0.134145f * v, v, 1.f), s);
    }
    case SCMP_ACT_SILU: {
      const float e = exp_minus(v), s = reciprocal(1.f + e);
      return s * fmaf(v, e * s, 1.f);
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
