// Packing and unpacking of 8-bit activation checkpoints.
#include "act8.cuh"
#include "status.cuh"

namespace scmp {

// Four threads hold a block of 32 values, eight each.
template <class T, bool VEC>
__global__ void __launch_bounds__(256) act8_pack_kernel(const T* __restrict__ x, long long rows, int cols, long long ld,
                                                        int8_t* __restrict__ codes, uint8_t* __restrict__ exps) {
  const int nb = act8_blocks(cols);
  const int quarter = threadIdx.x & 3;
  const long long stride = (long long)gridDim.x * (blockDim.x >> 2);
  const long long total = rows * nb;
  // whole warps stay in the loop for the shuffles
  for (long long blk0 = (long long)blockIdx.x * (blockDim.x >> 2) + ((threadIdx.x >> 5) << 3); blk0 < total; blk0 += stride) {
    const long long blk = blk0 + ((threadIdx.x & 31) >> 2);
    const bool live = blk < total;
    const long long row = live ? blk / nb : 0;
    const int b = (int)(live ? blk - row * nb : 0);
    const int c0 = b * kAct8Block + quarter * 8;
    const T* src = x + row * ld + c0;
    float v[8];
    if (VEC) {
      if (live && c0 < cols) {
        unpack8(ldg8(src), v);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = 0.f;
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = live && c0 + i < cols ? Elem<T>::to_f(src[i]) : 0.f;
    }
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(v[i]) & 0x7FFFFFFFu);
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
    const uint32_t byte = act8_exponent(top, act8_floor<T>());
    const float inv = act8_inverse(byte);
    const bool nan = byte == kAct8Nan;
    const uint32_t w[2] = {act8_codes4(v[0], v[1], v[2], v[3], inv, nan), act8_codes4(v[4], v[5], v[6], v[7], inv, nan)};
    if (!live) continue;
    int8_t* dst = codes + row * cols + c0;
    if (VEC) {
      if (c0 < cols) *reinterpret_cast<uint2*>(dst) = make_uint2(w[0], w[1]);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (c0 + i < cols) dst[i] = (int8_t)(w[i >> 2] >> (8 * (i & 3)));
    }
    if (quarter == 0) exps[blk] = (uint8_t)byte;
  }
}

template <class T, bool VEC>
__global__ void __launch_bounds__(256) act8_unpack_kernel(const int8_t* __restrict__ codes, const uint8_t* __restrict__ exps,
                                                          long long rows, int cols, long long ldo,
                                                          T* __restrict__ out) {
  const int nb = act8_blocks(cols);
  const long long total = rows * nb * 4;
  const long long stride = (long long)gridDim.x * blockDim.x;
  for (long long t = (long long)blockIdx.x * blockDim.x + threadIdx.x; t < total; t += stride) {
    const long long blk = t >> 2, row = blk / nb;
    const int b = (int)(blk - row * nb), c0 = b * kAct8Block + (int)(t & 3) * 8;
    if (c0 >= cols) continue;
    const float s = act8_scale(__ldg(exps + blk));
    const int8_t* src = codes + row * cols + c0;
    T* dst = out + row * ldo + c0;
    if (VEC) {
      const uint2 q = __ldg(reinterpret_cast<const uint2*>(src));
      float v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = act8_value(i < 4 ? q.x : q.y, i & 3, s);
      stg8(dst, v);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (c0 + i < cols) dst[i] = Elem<T>::from_f(fmul((float)src[i], s));
    }
  }
}

static int elementwise_grid(long long items, int per_block) {
  const long long want = (items + per_block - 1) / per_block;
  return (int)(want < 148 * 8 ? (want > 0 ? want : 1) : 148 * 8);
}

cudaError_t launch_act8_unpack(const int8_t* codes, const uint8_t* exps, long long rows, int cols, void* out,
                               long long ldo, int dtype, cudaStream_t st) {
  const bool vec = cols % 8 == 0 && (reinterpret_cast<uintptr_t>(codes) & 7) == 0 && rows_aligned16(out, ldo, dtype_size(dtype));
  const int grid = elementwise_grid(rows * act8_blocks(cols) * 4, 256);
  with_dtype(dtype, [&](auto* tag) {
    using T = std::remove_pointer_t<decltype(tag)>;
    if (vec)
      act8_unpack_kernel<T, true><<<grid, 256, 0, st>>>(codes, exps, rows, cols, ldo, (T*)out);
    else
      act8_unpack_kernel<T, false><<<grid, 256, 0, st>>>(codes, exps, rows, cols, ldo, (T*)out);
  });
  count_launch();
  return cudaGetLastError();
}

}  // namespace scmp

using namespace scmp;

extern "C" {

int scmp_act8_pack(const void* x, int dtype, long long rows, int cols, long long ld, int8_t* codes, uint8_t* exps,
                   void* stream) {
  if (!dtype_ok(dtype)) return fail(SCMP_ERR_INVALID_ARG, "act8_pack: unknown dtype");
  if (rows < 0 || cols < 1 || ld < cols) return fail(SCMP_ERR_INVALID_ARG, "act8_pack: bad shape (rows >= 0, cols >= 1, ld >= cols)");
  if (rows == 0) return SCMP_OK;
  if (!x || !codes || !exps) return fail(SCMP_ERR_INVALID_ARG, "act8_pack: null pointer");
  const cudaStream_t st = (cudaStream_t)stream;
  const bool vec = cols % 8 == 0 && rows_aligned16(x, ld, dtype_size(dtype)) && (reinterpret_cast<uintptr_t>(codes) & 7) == 0;
  const int grid = elementwise_grid(rows * act8_blocks(cols) * 4, 256);
  with_dtype(dtype, [&](auto* tag) {
    using T = std::remove_pointer_t<decltype(tag)>;
    if (vec)
      act8_pack_kernel<T, true><<<grid, 256, 0, st>>>((const T*)x, rows, cols, ld, codes, exps);
    else
      act8_pack_kernel<T, false><<<grid, 256, 0, st>>>((const T*)x, rows, cols, ld, codes, exps);
  });
  count_launch();
  SCMP_CUDA(cudaGetLastError(), "act8_pack");
  return SCMP_OK;
}

int scmp_act8_unpack(const int8_t* codes, const uint8_t* exps, long long rows, int cols, void* out, int dtype,
                     void* stream) {
  if (!dtype_ok(dtype)) return fail(SCMP_ERR_INVALID_ARG, "act8_unpack: unknown dtype");
  if (rows < 0 || cols < 1) return fail(SCMP_ERR_INVALID_ARG, "act8_unpack: bad shape (rows >= 0, cols >= 1)");
  if (rows == 0) return SCMP_OK;
  if (!codes || !exps || !out) return fail(SCMP_ERR_INVALID_ARG, "act8_unpack: null pointer");
  SCMP_CUDA(launch_act8_unpack(codes, exps, rows, cols, out, cols, dtype, (cudaStream_t)stream), "act8_unpack");
  return SCMP_OK;
}

}  // extern "C"
