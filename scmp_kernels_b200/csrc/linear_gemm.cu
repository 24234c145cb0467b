// Matrix product of the linear layer on the CUDA cores: 64 x 32 output tiles,
// a lane per column, eight rows per thread.
#include "linear.cuh"
#include "status.cuh"

namespace scmp {
namespace lin {

template <class T>
__global__ void __launch_bounds__(256) gemm_simt_kernel(Product p, Epilogue e) {
  __shared__ float sa[64][17], sb[32][17];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long i0 = (long long)blockIdx.x * 64;
  const int j0 = blockIdx.y * 32;
  float acc[8];
#pragma unroll
  for (int r = 0; r < 8; ++r) acc[r] = 0.f;
  for (int k0 = 0; k0 < p.k; k0 += 16) {
    for (int t = threadIdx.x; t < 64 * 16; t += 256) {
      // neighbouring threads along the axis that is contiguous in memory
      const int ii = p.ak == 1 ? t >> 4 : t & 63, kk = p.ak == 1 ? t & 15 : t >> 6;
      sa[ii][kk] = i0 + ii < p.m && k0 + kk < p.k
                       ? Elem<T>::to_f(((const T*)p.a)[(i0 + ii) * p.ai + (long long)(k0 + kk) * p.ak]) : 0.f;
    }
    for (int t = threadIdx.x; t < 32 * 16; t += 256) {
      const int jj = p.bk == 1 ? t >> 4 : t & 31, kk = p.bk == 1 ? t & 15 : t >> 5;
      sb[jj][kk] = j0 + jj < p.n && k0 + kk < p.k
                       ? Elem<T>::to_f(((const T*)p.b)[(long long)(j0 + jj) * p.bj + (long long)(k0 + kk) * p.bk]) : 0.f;
    }
    __syncthreads();
#pragma unroll
    for (int kk = 0; kk < 16; ++kk) {
      const float b = sb[lane][kk];
#pragma unroll
      for (int r = 0; r < 8; ++r) acc[r] = fmaf(sa[warp * 8 + r][kk], b, acc[r]);
    }
    __syncthreads();
  }
  const int j = j0 + lane;
  const bool jok = j < p.n;
  const float bias = e.bias && jok ? (e.bias_f32 ? ((const float*)e.bias)[j] : Elem<T>::to_f(((const T*)e.bias)[j])) : 0.f;
#pragma unroll
  for (int r = 0; r < 8; ++r) {
    const long long i = i0 + warp * 8 + r;
    if (i >= p.m) break;  // whole warps
    const float v = jok ? acc[r] + bias : 0.f;
    if (e.pre && jok) ((T*)e.pre)[i * p.n + j] = Elem<T>::from_f(v);
    if (e.codes) {
      const uint32_t byte = act8_exponent(__reduce_max_sync(0xffffffffu, __float_as_uint(v) & 0x7FFFFFFFu), act8_floor<T>());
      if (jok) e.codes[i * p.n + j] = (int8_t)act8_code(v, act8_inverse(byte), byte == kAct8Nan);
      if (lane == 0) e.exps[i * act8_blocks(p.n) + (j >> 5)] = (uint8_t)byte;
    }
    if (!jok) continue;
    float y = act_value(e.act, v);
    if (e.residual) y += Elem<T>::to_f(((const T*)e.residual)[i * e.ldr + j]);
    ((T*)e.out)[i * e.ldo + j] = Elem<T>::from_f(y);
  }
}

static cudaError_t launch_gemm(const Product& p, const Epilogue& e, int dtype, cudaStream_t st) {
  with_dtype(dtype, [&](auto* tag) {
    using T = std::remove_pointer_t<decltype(tag)>;
    gemm_simt_kernel<T><<<dim3(cdiv(p.m, 64), cdiv(p.n, 32)), 256, 0, st>>>(p, e);
  });
  count_launch();
  return cudaGetLastError();
}

}  // namespace lin
}  // namespace scmp
