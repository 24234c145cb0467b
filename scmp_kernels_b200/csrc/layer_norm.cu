// Layer norm over the last axis, forward and backward.
//
//   mean = sum x / D, rstd = 1 / sqrt(sum (x - mean)^2 / D + eps),
//   xh = (x - mean) * rstd,  y = xh * w + b
//   g = dy * w,  dx = rstd * (g - mean(g) - xh * mean(g * xh)),
//   dw = sum over rows of dy * xh,  db = sum over rows of dy
//
// Statistics and sums are float32 whatever the tensors' type. Both passes are
// bound by memory: a row is read once into registers (TPR threads hold NB
// times eight values each) and the variance is the second moment about the
// mean, which costs nothing from registers and does not cancel. The backward
// pass accumulates dw and db in registers, a thread owning its columns over
// all rows of its block, and leaves one partial row per block that a second
// kernel adds in a fixed order: no atomics, the same bits every time. Rows too
// long for registers take the three-pass kernels at the end.
#include "act8.cuh"
#include "status.cuh"

namespace scmp {
namespace ln {

constexpr int kMaxFused = 16384;  // columns held in registers (512 threads x 4 x 8)

struct Args {
  long long rows, ldx, ldy, ldo;  // row pitches of x, dy and the result (y or dx), in elements
  int cols;
  float eps;
  const void* x;
  const int8_t* codes;
  const uint8_t* exps;
  const void* dy;
  const void* weight;  // may be null (ones)
  const void* bias;    // may be null (zeros)
  int w_f32;           // weight and bias are float32, not x's type
  int w_vec;           // weight and bias are 16-byte aligned
  void* out;
  float* mean;
  float* rstd;
  int8_t* codes_out;   // forward: 8-bit checkpoint of x, or null
  uint8_t* exps_out;
  float* part;         // backward: (blocks, 2, cols) partial sums of dw and db
};

// Columns of chunk i, element j of a thread: eight neighbours per thread where
// rows can be read 16 bytes at a time, else lane-interleaved single elements
// (neighbouring threads read neighbouring elements).
template <bool VEC, int TPR>
__device__ __forceinline__ int col_of(int t, int i, int j) {
  return VEC ? (t + TPR * i) * 8 + j : (i * 8 + j) * TPR + t;
}

template <class T, bool VEC, int TPR>
__device__ __forceinline__ void load_chunk(const T* __restrict__ row, int cols, int t, int i, float (&v)[8]) {
  if (VEC) {
    const int c = (t + TPR * i) * 8;
    if (c < cols) {
      unpack8(ldg8(row + c), v);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = 0.f;
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int c = col_of<false, TPR>(t, i, j);
      v[j] = c < cols ? ldg1(row + c) : 0.f;
    }
  }
}
template <bool VEC, int TPR>
__device__ __forceinline__ void load_chunk8(const int8_t* __restrict__ codes, const uint8_t* __restrict__ exps, int cols,
                                            int t, int i, float (&v)[8]) {
  if (VEC) {
    const int c = (t + TPR * i) * 8;
    if (c < cols) {
      const uint2 q = __ldg(reinterpret_cast<const uint2*>(codes + c));
      const float s = act8_scale(__ldg(exps + (c >> 5)));
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = act8_value(j < 4 ? q.x : q.y, j & 3, s);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = 0.f;
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int c = col_of<false, TPR>(t, i, j);
      v[j] = c < cols ? fmul((float)codes[c], act8_scale(__ldg(exps + (c >> 5)))) : 0.f;
    }
  }
}
template <class T, bool VEC, int TPR>
__device__ __forceinline__ void load_param(const void* p, int f32, int vec, int cols, int t, int i, float (&v)[8]) {
  if (VEC && vec) {
    if (f32)
      load_chunk<float, true, TPR>((const float*)p, cols, t, i, v);
    else
      load_chunk<T, true, TPR>((const T*)p, cols, t, i, v);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int c = col_of<VEC, TPR>(t, i, j);
      v[j] = c >= cols ? 0.f : f32 ? __ldg((const float*)p + c) : ldg1((const T*)p + c);
    }
  }
}
template <class T, bool VEC, int TPR>
__device__ __forceinline__ void store_chunk(T* __restrict__ row, int cols, int t, int i, const float (&v)[8]) {
  if (VEC) {
    const int c = (t + TPR * i) * 8;
    if (c < cols) stg8(row + c, v);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int c = col_of<false, TPR>(t, i, j);
      if (c < cols) row[c] = Elem<T>::from_f(v[j]);
    }
  }
}

// Sums of a and b over the TPR threads of a row (a block is one row for
// TPR > 32; the trailing barrier lets the scratch be used again).
template <int TPR>
__device__ __forceinline__ void row_sum2(float& a, float& b, float* scratch) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    a += __shfl_xor_sync(0xffffffffu, a, o);
    b += __shfl_xor_sync(0xffffffffu, b, o);
  }
  if (TPR > 32) {
    constexpr int W = TPR / 32;
    const int w = threadIdx.x >> 5, l = threadIdx.x & 31;
    if (l == 0) {
      scratch[w] = a;
      scratch[32 + w] = b;
    }
    __syncthreads();
    a = l < W ? scratch[l] : 0.f;
    b = l < W ? scratch[32 + l] : 0.f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      a += __shfl_xor_sync(0xffffffffu, a, o);
      b += __shfl_xor_sync(0xffffffffu, b, o);
    }
    __syncthreads();
  }
}

// 8-bit checkpoint of chunk i of a row: a block of 32 columns is four
// neighbouring threads' chunks (VEC) or the same element of a warp's lanes.
template <class T, bool VEC, int TPR>
__device__ __forceinline__ void store_act8(int8_t* __restrict__ codes, uint8_t* __restrict__ exps, int cols, int t, int i,
                                           const float (&v)[8], bool live) {
  if (VEC) {
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) top = max(top, __float_as_uint(v[j]) & 0x7FFFFFFFu);
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
    const uint32_t byte = act8_exponent(top, act8_floor<T>());
    const float inv = act8_inverse(byte);
    const int c = (t + TPR * i) * 8;
    if (!live || c >= cols) return;
    const bool nan = byte == kAct8Nan;
    *reinterpret_cast<uint2*>(codes + c) =
        make_uint2(act8_codes4(v[0], v[1], v[2], v[3], inv, nan), act8_codes4(v[4], v[5], v[6], v[7], inv, nan));
    if ((t & 3) == 0) exps[c >> 5] = (uint8_t)byte;
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint32_t top = __reduce_max_sync(0xffffffffu, __float_as_uint(v[j]) & 0x7FFFFFFFu);
      const uint32_t byte = act8_exponent(top, act8_floor<T>());
      const int c = col_of<false, TPR>(t, i, j);
      if (live && c < cols) {
        codes[c] = (int8_t)act8_code(v[j], act8_inverse(byte), byte == kAct8Nan);
        if ((t & 31) == 0) exps[c >> 5] = (uint8_t)byte;
      }
    }
  }
}

template <int TPR>
__host__ __device__ constexpr int block_threads() { return TPR == 32 ? 256 : TPR; }

template <class T, bool VEC, int TPR, int NB>
__global__ void __launch_bounds__(block_threads<TPR>()) forward_kernel(Args a) {
  constexpr int RPB = block_threads<TPR>() / TPR;
  __shared__ float scratch[64];
  const int t = threadIdx.x % TPR;
  const float inv_d = 1.f / (float)a.cols;
  for (long long row0 = (long long)blockIdx.x * RPB; row0 < a.rows; row0 += (long long)gridDim.x * RPB) {
    const long long row = row0 + threadIdx.x / TPR;
    const bool live = row < a.rows;
    if (TPR == 32 && !live) return;  // whole warps
    const T* src = (const T*)a.x + row * a.ldx;
    float v[NB][8];
    float s = 0.f, zero = 0.f;
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      load_chunk<T, VEC, TPR>(src, a.cols, t, i, v[i]);
#pragma unroll
      for (int j = 0; j < 8; ++j) s += v[i][j];
    }
    row_sum2<TPR>(s, zero, scratch);
    const float mean = s * inv_d;
    float q = 0.f;
#pragma unroll
    for (int i = 0; i < NB; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float u = col_of<VEC, TPR>(t, i, j) < a.cols ? v[i][j] - mean : 0.f;
        q = fmaf(u, u, q);
      }
    row_sum2<TPR>(q, zero, scratch);
    const float rstd = 1.f / sqrtf(q * inv_d + a.eps);
    if (t == 0) {
      if (a.mean) a.mean[row] = mean;
      if (a.rstd) a.rstd[row] = rstd;
    }
    if (a.codes_out) {
#pragma unroll
      for (int i = 0; i < NB; ++i)
        store_act8<T, VEC, TPR>(a.codes_out + row * a.cols, a.exps_out + row * act8_blocks(a.cols), a.cols, t, i, v[i], true);
    }
    T* dst = (T*)a.out + row * a.ldo;
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      float w[8], b[8], y[8];
      if (a.weight) load_param<T, VEC, TPR>(a.weight, a.w_f32, a.w_vec, a.cols, t, i, w);
      if (a.bias) load_param<T, VEC, TPR>(a.bias, a.w_f32, a.w_vec, a.cols, t, i, b);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        float h = (v[i][j] - mean) * rstd;
        if (a.weight) h *= w[j];
        if (a.bias) h += b[j];
        y[j] = h;
      }
      store_chunk<T, VEC, TPR>(dst, a.cols, t, i, y);
    }
  }
}

template <class T, bool SRC8, bool VEC, int TPR, int NB>
__global__ void __launch_bounds__(block_threads<TPR>()) backward_kernel(Args a) {
  constexpr int THREADS = block_threads<TPR>();
  constexpr int RPB = THREADS / TPR;
  __shared__ float scratch[RPB > 1 ? RPB * 256 : 64];
  const int t = threadIdx.x % TPR;
  const float inv_d = 1.f / (float)a.cols;
  float dw[NB][8], db[NB][8];
#pragma unroll
  for (int i = 0; i < NB; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) dw[i][j] = db[i][j] = 0.f;
  for (long long row0 = (long long)blockIdx.x * RPB; row0 < a.rows; row0 += (long long)gridDim.x * RPB) {
    const long long row = row0 + threadIdx.x / TPR;
    if (TPR == 32 && row >= a.rows) break;  // whole warps; no block barrier in the loop
    const float mean = __ldg(a.mean + row), rstd = __ldg(a.rstd + row);
    float xh[NB][8], g[NB][8];
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      if (SRC8)
        load_chunk8<VEC, TPR>(a.codes + row * a.cols, a.exps + row * act8_blocks(a.cols), a.cols, t, i, xh[i]);
      else
        load_chunk<T, VEC, TPR>((const T*)a.x + row * a.ldx, a.cols, t, i, xh[i]);
      load_chunk<T, VEC, TPR>((const T*)a.dy + row * a.ldy, a.cols, t, i, g[i]);
    }
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      float w[8];
      if (a.weight) load_param<T, VEC, TPR>(a.weight, a.w_f32, a.w_vec, a.cols, t, i, w);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (col_of<VEC, TPR>(t, i, j) < a.cols) {
          const float h = (xh[i][j] - mean) * rstd, d = g[i][j];
          dw[i][j] = fmaf(d, h, dw[i][j]);
          db[i][j] += d;
          const float gg = a.weight ? d * w[j] : d;
          s1 += gg;
          s2 = fmaf(gg, h, s2);
          xh[i][j] = h;
          g[i][j] = gg;
        }
      }
    }
    row_sum2<TPR>(s1, s2, scratch);
    const float m1 = s1 * inv_d, m2 = s2 * inv_d;
    T* dst = (T*)a.out + row * a.ldo;
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      float d[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) d[j] = rstd * (g[i][j] - m1 - xh[i][j] * m2);
      store_chunk<T, VEC, TPR>(dst, a.cols, t, i, d);
    }
  }
  if (!a.part) return;
  float* part = a.part + (size_t)blockIdx.x * 2 * a.cols;
  if (RPB == 1) {
#pragma unroll
    for (int i = 0; i < NB; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int c = col_of<VEC, TPR>(t, i, j);
        if (c < a.cols) {
          part[c] = dw[i][j];
          part[a.cols + c] = db[i][j];
        }
      }
  } else {
    // the block's warps hold the same columns of different rows: one chunk of
    // 256 columns at a time through shared memory, added in warp order
    const int w = threadIdx.x / TPR;
#pragma unroll
    for (int i = 0; i < NB; ++i)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        __syncthreads();
#pragma unroll
        for (int j = 0; j < 8; ++j) scratch[w * 256 + j * 32 + t] = k ? db[i][j] : dw[i][j];
        __syncthreads();
        float s = 0.f;
#pragma unroll
        for (int r = 0; r < RPB; ++r) s += scratch[r * 256 + threadIdx.x];
        const int c = col_of<VEC, TPR>(threadIdx.x & 31, i, threadIdx.x >> 5);
        if (c < a.cols) part[(size_t)k * a.cols + c] = s;
      }
  }
}

// out_k[c] = sum over p of part[p][k][c]: 32 strands of p per column, each in
// order, then the strands in order.
template <class W>
__global__ void __launch_bounds__(1024) column_sum_kernel(const float* __restrict__ part, int parts, int sets, int cols,
                                                          W* __restrict__ out0, W* __restrict__ out1) {
  __shared__ float s[32][33];
  const int lx = threadIdx.x & 31, ly = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lx, k = blockIdx.y;
  W* out = k ? out1 : out0;
  if (!out) return;
  float v = 0.f;
  if (c < cols) {
#pragma unroll 8
    for (int p = ly; p < parts; p += 32) v += __ldg(part + ((size_t)p * sets + k) * cols + c);
  }
  s[ly][lx] = v;
  __syncthreads();
  v = s[lx][ly];  // a warp per column
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_down_sync(0xffffffffu, v, o);
  if (lx == 0 && blockIdx.x * 32 + ly < cols) out[blockIdx.x * 32 + ly] = Elem<W>::from_f(v);
}

// Rows longer than kMaxFused: one block per row, the row read once per pass.
template <class T>
__device__ __forceinline__ float load_any(const void* p, int f32, long long i) {
  return f32 ? __ldg((const float*)p + i) : ldg1((const T*)p + i);
}
template <class T, bool SRC8>
__device__ __forceinline__ float load_x(const Args& a, long long row, int c) {
  if (SRC8)
    return fmul((float)a.codes[row * a.cols + c], act8_scale(__ldg(a.exps + row * act8_blocks(a.cols) + (c >> 5))));
  return ldg1((const T*)a.x + row * a.ldx + c);
}
template <class T>
__global__ void __launch_bounds__(1024) forward_long_kernel(Args a) {
  __shared__ float scratch[64];
  const long long row = blockIdx.x;
  const float inv_d = 1.f / (float)a.cols;
  float s = 0.f, zero = 0.f;
  for (int c = threadIdx.x; c < a.cols; c += 1024) s += load_x<T, false>(a, row, c);
  row_sum2<1024>(s, zero, scratch);
  const float mean = s * inv_d;
  float q = 0.f;
  for (int c = threadIdx.x; c < a.cols; c += 1024) {
    const float u = load_x<T, false>(a, row, c) - mean;
    q = fmaf(u, u, q);
  }
  row_sum2<1024>(q, zero, scratch);
  const float rstd = 1.f / sqrtf(q * inv_d + a.eps);
  if (threadIdx.x == 0) {
    if (a.mean) a.mean[row] = mean;
    if (a.rstd) a.rstd[row] = rstd;
  }
  for (int c0 = 0; c0 < a.cols; c0 += 1024) {  // whole warps for the checkpoint's maxima
    const int c = c0 + threadIdx.x;
    const float x = c < a.cols ? load_x<T, false>(a, row, c) : 0.f;
    if (a.codes_out) {
      const uint32_t top = __reduce_max_sync(0xffffffffu, __float_as_uint(x) & 0x7FFFFFFFu);
      const uint32_t byte = act8_exponent(top, act8_floor<T>());
      if (c < a.cols) {
        a.codes_out[row * a.cols + c] = (int8_t)act8_code(x, act8_inverse(byte), byte == kAct8Nan);
        if ((threadIdx.x & 31) == 0) a.exps_out[row * act8_blocks(a.cols) + (c >> 5)] = (uint8_t)byte;
      }
    }
    if (c < a.cols) {
      float h = (x - mean) * rstd;
      if (a.weight) h *= load_any<T>(a.weight, a.w_f32, c);
      if (a.bias) h += load_any<T>(a.bias, a.w_f32, c);
      ((T*)a.out)[row * a.ldo + c] = Elem<T>::from_f(h);
    }
  }
}
template <class T, bool SRC8>
__global__ void __launch_bounds__(1024) backward_long_kernel(Args a) {
  __shared__ float scratch[64];
  const long long row = blockIdx.x;
  const float inv_d = 1.f / (float)a.cols, mean = a.mean[row], rstd = a.rstd[row];
  const T* dy = (const T*)a.dy + row * a.ldy;
  float s1 = 0.f, s2 = 0.f;
  for (int c = threadIdx.x; c < a.cols; c += 1024) {
    const float h = (load_x<T, SRC8>(a, row, c) - mean) * rstd;
    float g = ldg1(dy + c);
    if (a.weight) g *= load_any<T>(a.weight, a.w_f32, c);
    s1 += g;
    s2 = fmaf(g, h, s2);
  }
  row_sum2<1024>(s1, s2, scratch);
  const float m1 = s1 * inv_d, m2 = s2 * inv_d;
  for (int c = threadIdx.x; c < a.cols; c += 1024) {
    const float h = (load_x<T, SRC8>(a, row, c) - mean) * rstd;
    float g = ldg1(dy + c);
    if (a.weight) g *= load_any<T>(a.weight, a.w_f32, c);
    ((T*)a.out)[row * a.ldo + c] = Elem<T>::from_f(rstd * (g - m1 - h * m2));
  }
}
// dw and db of long rows: a thread per column over the rows of its block row.
template <class T, bool SRC8>
__global__ void __launch_bounds__(256) weight_grad_long_kernel(Args a) {
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= a.cols) return;
  float dw = 0.f, db = 0.f;
  for (long long row = blockIdx.y; row < a.rows; row += gridDim.y) {
    const float d = ldg1((const T*)a.dy + row * a.ldy + c);
    dw = fmaf(d, (load_x<T, SRC8>(a, row, c) - a.mean[row]) * a.rstd[row], dw);
    db += d;
  }
  float* part = a.part + (size_t)blockIdx.y * 2 * a.cols;
  part[c] = dw;
  part[a.cols + c] = db;
}

struct Shape {
  int tpr, nb;
};
// Threads and chunks of eight columns per thread that hold a row.
static Shape shape_for(int cols) {
  const int chunks = cdiv(cols, 8);
  if (chunks <= 128) return {32, chunks <= 32 ? 1 : chunks <= 64 ? 2 : 4};
  if (chunks <= 256) return {128, 2};
  if (chunks <= 512) return {256, 2};
  if (chunks <= 1024) return {512, 2};
  return {512, 4};
}
// Blocks of the backward pass: enough to fill the SMs, and no more partial
// rows of dw and db than that.
static int backward_blocks(long long rows, int cols) {
  if (cols > kMaxFused) return (int)(rows < 16 ? rows : 16);
  const Shape s = shape_for(cols);
  const int rpb = s.tpr == 32 ? 8 : 1;
  const long long want = (rows + rpb - 1) / rpb;
  const int per_sm = s.tpr <= 128 ? 4 : s.tpr == 256 ? 2 : 1;
  return (int)(want < 148LL * per_sm ? want : 148LL * per_sm);
}

template <class F>
static void with_shape(Shape s, F&& f) {
#define SCMP_SHAPE(T_, N_) \
  if (s.tpr == T_ && s.nb == N_) return f(std::integral_constant<int, T_>{}, std::integral_constant<int, N_>{});
  SCMP_SHAPE(32, 1) SCMP_SHAPE(32, 2) SCMP_SHAPE(32, 4) SCMP_SHAPE(128, 2) SCMP_SHAPE(256, 2) SCMP_SHAPE(512, 2)
  SCMP_SHAPE(512, 4)
#undef SCMP_SHAPE
}

static cudaError_t launch_forward(const Args& a, int dtype, bool vec, cudaStream_t st) {
  with_dtype(dtype, [&](auto* tag) {
    using T = std::remove_pointer_t<decltype(tag)>;
    if (a.cols > kMaxFused) {
      forward_long_kernel<T><<<(unsigned)a.rows, 1024, 0, st>>>(a);
      return;
    }
    with_shape(shape_for(a.cols), [&](auto tpr, auto nb) {
      constexpr int TPR = decltype(tpr)::value, NB = decltype(nb)::value, TH = block_threads<TPR>();
      const long long blocks = (a.rows + TH / TPR - 1) / (TH / TPR);
      const int grid = (int)(blocks < (1 << 30) ? blocks : 1 << 30);
      if (vec)
        forward_kernel<T, true, TPR, NB><<<grid, TH, 0, st>>>(a);
      else
        forward_kernel<T, false, TPR, NB><<<grid, TH, 0, st>>>(a);
    });
  });
  count_launch();
  return cudaGetLastError();
}

static cudaError_t launch_backward(const Args& a, int dtype, bool vec, int blocks, cudaStream_t st) {
  with_dtype(dtype, [&](auto* tag) {
    using T = std::remove_pointer_t<decltype(tag)>;
    auto go = [&](auto src8) {
      constexpr bool S8 = decltype(src8)::value;
      if (a.cols > kMaxFused) {
        backward_long_kernel<T, S8><<<(unsigned)a.rows, 1024, 0, st>>>(a);
        if (a.part) {
          weight_grad_long_kernel<T, S8><<<dim3(cdiv(a.cols, 256), blocks), 256, 0, st>>>(a);
          count_launch();
        }
        return;
      }
      with_shape(shape_for(a.cols), [&](auto tpr, auto nb) {
        constexpr int TPR = decltype(tpr)::value, NB = decltype(nb)::value, TH = block_threads<TPR>();
        if (vec)
          backward_kernel<T, S8, true, TPR, NB><<<blocks, TH, 0, st>>>(a);
        else
          backward_kernel<T, S8, false, TPR, NB><<<blocks, TH, 0, st>>>(a);
      });
    };
    if (a.codes)
      go(std::true_type{});
    else
      go(std::false_type{});
  });
  count_launch();
  return cudaGetLastError();
}

static int check_shape(const char* who, int dtype, int wdtype, long long rows, int cols) {
  const std::string w(who);
  if (!dtype_ok(dtype)) return fail(SCMP_ERR_INVALID_ARG, w + ": unknown dtype");
  if (wdtype != dtype && wdtype != SCMP_F32) return fail(SCMP_ERR_INVALID_ARG, w + ": weight and bias are float32 or x's type");
  if (rows < 0 || rows >= (1LL << 31) || cols < 1) return fail(SCMP_ERR_INVALID_ARG, w + ": bad shape (0 <= rows < 2^31, cols >= 1)");
  return SCMP_OK;
}

}  // namespace ln

cudaError_t launch_column_sum(const float* part, int parts, int sets, int cols, int dtype, void* out0, void* out1,
                                     cudaStream_t st) {
  with_dtype(dtype, [&](auto* tag) {
    using W = std::remove_pointer_t<decltype(tag)>;
    ln::column_sum_kernel<W><<<dim3(cdiv(cols, 32), sets), 1024, 0, st>>>(part, parts, sets, cols, (W*)out0, (W*)out1);
  });
  count_launch();
  return cudaGetLastError();
}

}  // namespace scmp

using namespace scmp;

extern "C" {

int scmp_layer_norm_forward(const void* x, int dtype, long long rows, int cols, long long ldx, const void* weight,
                            const void* bias, int wdtype, float eps, void* y, float* mean, float* rstd, int8_t* codes,
                            uint8_t* exps, void* stream) {
  if (int e = ln::check_shape("layer_norm_forward", dtype, wdtype, rows, cols)) return e;
  if (ldx < cols) return fail(SCMP_ERR_INVALID_ARG, "layer_norm_forward: ldx < cols");
  if (!(eps >= 0.f)) return fail(SCMP_ERR_INVALID_ARG, "layer_norm_forward: eps must be >= 0");
  if (rows == 0) return SCMP_OK;
  if (!x || !y || !codes != !exps) return fail(SCMP_ERR_INVALID_ARG, "layer_norm_forward: null pointer");
  ln::Args a{};
  a.rows = rows; a.cols = cols; a.ldx = ldx; a.ldo = cols; a.eps = eps;
  a.x = x; a.weight = weight; a.bias = bias; a.w_f32 = wdtype == SCMP_F32;
  a.w_vec = aligned16(weight) && aligned16(bias);
  a.out = y; a.mean = mean; a.rstd = rstd; a.codes_out = codes; a.exps_out = exps;
  const size_t es = dtype_size(dtype);
  const bool vec = cols % 8 == 0 && rows_aligned16(x, ldx, es) && aligned16(y) &&
                   (reinterpret_cast<uintptr_t>(codes) & 7) == 0;
  SCMP_CUDA(ln::launch_forward(a, dtype, vec, (cudaStream_t)stream), "layer_norm_forward");
  return SCMP_OK;
}

int scmp_layer_norm_backward_workspace_size(long long rows, int cols, size_t* bytes) {
  if (rows < 0 || rows >= (1LL << 31) || cols < 1 || !bytes)
    return fail(SCMP_ERR_INVALID_ARG, "layer_norm_backward_workspace_size: bad arguments");
  *bytes = (size_t)ln::backward_blocks(rows, cols) * 2 * cols * sizeof(float);
  return SCMP_OK;
}

int scmp_layer_norm_backward(const void* dy, long long lddy, const void* x, long long ldx, const int8_t* codes,
                             const uint8_t* exps, int dtype, long long rows, int cols, const float* mean,
                             const float* rstd, const void* weight, int wdtype, void* dx, void* dweight, void* dbias,
                             void* workspace, size_t workspace_bytes, void* stream) {
  if (int e = ln::check_shape("layer_norm_backward", dtype, wdtype, rows, cols)) return e;
  if (lddy < cols || (x && ldx < cols)) return fail(SCMP_ERR_INVALID_ARG, "layer_norm_backward: row pitch < cols");
  const cudaStream_t st = (cudaStream_t)stream;
  if (rows == 0) {
    if (dweight) SCMP_CUDA(cudaMemsetAsync(dweight, 0, cols * dtype_size(wdtype), st), "layer_norm_backward");
    if (dbias) SCMP_CUDA(cudaMemsetAsync(dbias, 0, cols * dtype_size(wdtype), st), "layer_norm_backward");
    return SCMP_OK;
  }
  if (!x == !codes || !codes != !exps)
    return fail(SCMP_ERR_INVALID_ARG, "layer_norm_backward: give x, or codes and exps");
  if (!dy || !mean || !rstd || !dx) return fail(SCMP_ERR_INVALID_ARG, "layer_norm_backward: null pointer");
  const int blocks = ln::backward_blocks(rows, cols);
  const bool sums = dweight || dbias;
  if (sums && (!workspace || workspace_bytes < (size_t)blocks * 2 * cols * sizeof(float)))
    return fail(SCMP_ERR_WORKSPACE, "layer_norm_backward: workspace missing or too small");
  ln::Args a{};
  a.rows = rows; a.cols = cols; a.ldx = ldx; a.ldy = lddy; a.ldo = cols;
  a.x = x; a.codes = codes; a.exps = exps; a.dy = dy; a.weight = weight; a.w_f32 = wdtype == SCMP_F32;
  a.w_vec = aligned16(weight);
  a.out = dx; a.mean = const_cast<float*>(mean); a.rstd = const_cast<float*>(rstd);
  a.part = sums ? (float*)workspace : nullptr;
  const size_t es = dtype_size(dtype);
  const bool vec = cols % 8 == 0 && rows_aligned16(dy, lddy, es) && aligned16(dx) &&
                   (x ? rows_aligned16(x, ldx, es) : (reinterpret_cast<uintptr_t>(codes) & 7) == 0);
  SCMP_CUDA(ln::launch_backward(a, dtype, vec, blocks, st), "layer_norm_backward");
  if (sums)
    SCMP_CUDA(launch_column_sum(a.part, blocks, 2, cols, wdtype, dweight, dbias, st), "layer_norm_backward: column sums");
  return SCMP_OK;
}

}  // extern "C"
