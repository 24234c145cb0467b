// The exact linear layer's C entry points, and the pass over dy that its
// gradients share.
#include "linear.cuh"
#include "status.cuh"

namespace scmp {
namespace lin {

// dpre = dy * act'(pre) and its column sums. A thread owns eight columns (VEC)
// or every 32nd of eight groups, over the rows of its block; the block's eight
// row groups are added in order into one partial row.
struct DpreArgs {
  const void* dy;
  const void* pre;
  const int8_t* codes;
  const uint8_t* exps;
  long long rows, ldy, ldp;
  int cols, act;
  void* dpre;   // (rows, cols), or null (no activation: dy itself is dpre)
  float* part;  // (gridDim.y, cols), or null
};
template <class T, bool VEC>
__global__ void __launch_bounds__(256) dpre_kernel(DpreArgs a) {
  __shared__ float s[8][256];
  const int lane = threadIdx.x & 31, group = threadIdx.x >> 5;
  const int c0 = blockIdx.x * 256;
  float sum[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) sum[j] = 0.f;
  for (long long row = (long long)blockIdx.y * 8 + group; row < a.rows; row += (long long)gridDim.y * 8) {
    const T* dy = (const T*)a.dy + row * a.ldy;
    float d[8], p[8];
    const int cv = c0 + lane * 8;
    if (VEC) {
      if (cv < a.cols) {
        unpack8(ldg8(dy + cv), d);
        if (a.act != SCMP_ACT_NONE) {
          if (a.codes) {
            const uint2 q = __ldg(reinterpret_cast<const uint2*>(a.codes + row * a.cols + cv));
            const float sc = act8_scale(__ldg(a.exps + row * act8_blocks(a.cols) + (cv >> 5)));
#pragma unroll
            for (int j = 0; j < 8; ++j) p[j] = fmul((float)(int8_t)((j < 4 ? q.x : q.y) >> (8 * (j & 3))), sc);
          } else {
            unpack8(ldg8((const T*)a.pre + row * a.ldp + cv), p);
          }
#pragma unroll
          for (int j = 0; j < 8; ++j) d[j] *= act_grad(a.act, p[j]);
        }
        if (a.dpre) stg8((T*)a.dpre + row * a.cols + cv, d);
#pragma unroll
        for (int j = 0; j < 8; ++j) sum[j] += d[j];
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int c = c0 + j * 32 + lane;
        if (c >= a.cols) continue;
        float v = ldg1(dy + c);
        if (a.act != SCMP_ACT_NONE) {
          const float q = a.codes ? fmul((float)a.codes[row * a.cols + c], act8_scale(a.exps[row * act8_blocks(a.cols) + (c >> 5)]))
                                  : ldg1((const T*)a.pre + row * a.ldp + c);
          v *= act_grad(a.act, q);
        }
        if (a.dpre) ((T*)a.dpre)[row * a.cols + c] = Elem<T>::from_f(v);
        sum[j] += v;
      }
    }
  }
  if (!a.part) return;
#pragma unroll
  for (int j = 0; j < 8; ++j) s[group][VEC ? lane * 8 + j : j * 32 + lane] = sum[j];
  __syncthreads();
  float v = 0.f;
#pragma unroll
  for (int g = 0; g < 8; ++g) v += s[g][threadIdx.x];
  if (c0 + threadIdx.x < a.cols) a.part[(size_t)blockIdx.y * a.cols + c0 + threadIdx.x] = v;
}
static int dpre_row_blocks(long long rows, int cols) {
  const int cb = cdiv(cols, 256);
  const long long want = (rows + 7) / 8;
  const int most = cdiv(148 * 4, cb);
  return (int)(want < most ? (want > 0 ? want : 1) : most);
}
static cudaError_t launch_dpre(const DpreArgs& a, int dtype, int row_blocks, cudaStream_t st) {
  const size_t es = dtype_size(dtype);
  const bool vec = a.cols % 8 == 0 && rows_aligned16(a.dy, a.ldy, es) &&
                   (a.act == SCMP_ACT_NONE || (a.codes ? (reinterpret_cast<uintptr_t>(a.codes) & 7) == 0 : rows_aligned16(a.pre, a.ldp, es)));
  with_dtype(dtype, [&](auto* tag) {
    using T = std::remove_pointer_t<decltype(tag)>;
    const dim3 grid(cdiv(a.cols, 256), row_blocks);
    if (vec)
      dpre_kernel<T, true><<<grid, 256, 0, st>>>(a);
    else
      dpre_kernel<T, false><<<grid, 256, 0, st>>>(a);
  });
  count_launch();
  return cudaGetLastError();
}

struct Carve {
  char* base;
  size_t off = 0;
  template <class U>
  U* take(size_t count) {
    off = (off + 255) & ~size_t(255);
    U* p = base ? reinterpret_cast<U*>(base + off) : nullptr;
    off += count * sizeof(U);
    return p;
  }
};
struct BackwardPlan {
  char* dpre;   // dpre in the tensors' type (with an activation)
  char* x;      // x unpacked from its checkpoint
  float* part;  // column sums of dpre per block row
  int row_blocks;
};
static BackwardPlan plan_backward(Carve& c, int dtype, long long rows, int d, int m, int act, bool x8, bool with_bias) {
  const size_t es = dtype_size(dtype);
  BackwardPlan p{};
  p.row_blocks = dpre_row_blocks(rows, m);
  if (act != SCMP_ACT_NONE) p.dpre = c.take<char>(rows * m * es);
  if (x8) p.x = c.take<char>(rows * d * es);
  if (with_bias) p.part = c.take<float>((size_t)p.row_blocks * m);
  return p;
}

static int check_shape(const char* who, int dtype, long long rows, int d, int m, int act) {
  const std::string w(who);
  if (!dtype_ok(dtype)) return fail(SCMP_ERR_INVALID_ARG, w + ": unknown dtype");
  if (rows < 0 || rows > 2147480000LL || d < 1 || m < 1 || d > 2147480000 || m > 2147480000)
    return fail(SCMP_ERR_INVALID_ARG, w + ": bad shape (rows >= 0, d, m >= 1, all below 2^31)");
  if (act < SCMP_ACT_NONE || act > SCMP_ACT_SILU) return fail(SCMP_ERR_INVALID_ARG, w + ": unknown activation");
  return SCMP_OK;
}

}  // namespace lin
}  // namespace scmp

using namespace scmp;

extern "C" {

int scmp_linear_forward_workspace_size(int dtype, long long rows, int d, int m, size_t* bytes) {
  if (int e = lin::check_shape("linear_forward_workspace_size", dtype, rows, d, m, 0)) return e;
  if (!bytes) return fail(SCMP_ERR_INVALID_ARG, "linear_forward_workspace_size: null pointer");
  *bytes = 0;
  return SCMP_OK;
}

int scmp_linear_forward(const void* x, long long ldx, const void* weight, long long ldw, const void* bias, int bias_dtype,
                        const void* residual, long long ldr, int dtype, long long rows, int d, int m, int activation,
                        void* y, void* pre, int8_t* pre_codes, uint8_t* pre_exps, void* workspace,
                        size_t workspace_bytes, void* stream) {
  if (int e = lin::check_shape("linear_forward", dtype, rows, d, m, activation)) return e;
  if (bias && bias_dtype != dtype && bias_dtype != SCMP_F32)
    return fail(SCMP_ERR_INVALID_ARG, "linear_forward: bias is float32 or x's type");
  if (ldx < d || ldw < d || (residual && ldr < m)) return fail(SCMP_ERR_INVALID_ARG, "linear_forward: row pitch too small");
  if (rows == 0) return SCMP_OK;
  if (!x || !weight || !y || !pre_codes != !pre_exps) return fail(SCMP_ERR_INVALID_ARG, "linear_forward: null pointer");
  lin::Product p{x, weight, ldx, 1, ldw, 1, (int)rows, m, d};
  lin::Epilogue e{bias, bias_dtype == SCMP_F32, residual, ldr, activation, y, m, pre, pre_codes, pre_exps};
  SCMP_CUDA(lin::launch_gemm(p, e, dtype, (cudaStream_t)stream), "linear_forward");
  return SCMP_OK;
}

int scmp_linear_backward_workspace_size(int dtype, long long rows, int d, int m, int activation, int x_packed,
                                        int with_bias, size_t* bytes) {
  if (int e = lin::check_shape("linear_backward_workspace_size", dtype, rows, d, m, activation)) return e;
  if (!bytes) return fail(SCMP_ERR_INVALID_ARG, "linear_backward_workspace_size: null pointer");
  lin::Carve c{nullptr};
  lin::plan_backward(c, dtype, rows, d, m, activation, x_packed != 0, with_bias != 0);
  *bytes = c.off;
  return SCMP_OK;
}

int scmp_linear_backward(const void* dy, long long lddy, const void* x, long long ldx, const int8_t* x_codes,
                         const uint8_t* x_exps, const void* weight, long long ldw, const void* pre, long long ldpre,
                         const int8_t* pre_codes, const uint8_t* pre_exps, int dtype, long long rows, int d, int m,
                         int activation, void* dx, void* dweight, void* dbias, int bias_dtype, void* workspace,
                         size_t workspace_bytes, void* stream) {
  if (int e = lin::check_shape("linear_backward", dtype, rows, d, m, activation)) return e;
  const cudaStream_t st = (cudaStream_t)stream;
  const size_t es = dtype_size(dtype);
  if (dbias && bias_dtype != dtype && bias_dtype != SCMP_F32)
    return fail(SCMP_ERR_INVALID_ARG, "linear_backward: the bias is float32 or dy's type");
  if (rows == 0) {
    if (dweight) SCMP_CUDA(cudaMemsetAsync(dweight, 0, (size_t)m * d * es, st), "linear_backward");
    if (dbias) SCMP_CUDA(cudaMemsetAsync(dbias, 0, (size_t)m * dtype_size(bias_dtype), st), "linear_backward");
    return SCMP_OK;
  }
  if (!dy || lddy < m || (dx && (!weight || ldw < d)) || (dweight && !x == !x_codes) || !x_codes != !x_exps || (x && ldx < d))
    return fail(SCMP_ERR_INVALID_ARG, "linear_backward: give dy, weight (for dx) and x or its codes and exps (for dweight), at pitches that hold a row");
  const bool act = activation != SCMP_ACT_NONE;
  if (act && (!pre == !pre_codes || !pre_codes != !pre_exps || (pre && ldpre < m)))
    return fail(SCMP_ERR_INVALID_ARG, "linear_backward: an activation's gradient needs pre, or its codes and exps");
  lin::Carve c{(char*)workspace};
  const lin::BackwardPlan w = lin::plan_backward(c, dtype, rows, d, m, activation, x_codes != nullptr, dbias != nullptr);
  if (c.off && (!workspace || workspace_bytes < c.off)) return fail(SCMP_ERR_WORKSPACE, "linear_backward: workspace missing or too small");
  const void* g = dy;
  long long ldg = lddy;
  if (act || dbias) {
    lin::DpreArgs a{dy, pre, pre_codes, pre_exps, rows, lddy, ldpre, m, activation, act ? w.dpre : nullptr, w.part};
    SCMP_CUDA(lin::launch_dpre(a, dtype, w.row_blocks, st), "linear_backward: activation");
    if (dbias)
      SCMP_CUDA(launch_column_sum(w.part, w.row_blocks, 1, m, bias_dtype, dbias, nullptr, st), "linear_backward: bias");
    if (act) { g = w.dpre; ldg = m; }
  }
  if (dx) {
    lin::Product p{g, weight, ldg, 1, 1, ldw, (int)rows, d, m};
    lin::Epilogue e{};
    e.out = dx;
    e.ldo = d;
    SCMP_CUDA(lin::launch_gemm(p, e, dtype, st), "linear_backward: dx");
  }
  if (dweight) {
    const void* xs = x;
    long long lx = ldx;
    if (x_codes) {
      SCMP_CUDA(launch_act8_unpack(x_codes, x_exps, rows, d, w.x, dtype, st), "linear_backward: unpack");
      xs = w.x;
      lx = d;
    }
    lin::Product p{g, xs, 1, ldg, 1, lx, m, d, (int)rows};
    lin::Epilogue e{};
    e.out = dweight;
    e.ldo = d;
    SCMP_CUDA(lin::launch_gemm(p, e, dtype, st), "linear_backward: dweight");
  }
  return SCMP_OK;
}

}  // extern "C"
