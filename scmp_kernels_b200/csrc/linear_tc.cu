// Matrix product of the linear layer on the tensor cores:
//   C(i, j) = sum over k of A(i, k) * B(j, k), float32 accumulators.
//
// A cluster of two CTAs owns a 256 x BN output tile (tcgen05.mma,
// cta_group::2): each CTA holds 128 rows of A and half of B's rows, so every
// operand byte in shared memory serves a tile twice as wide as one SM could
// hold. Operands come by TMA in 64-deep k blocks, 128-byte swizzled, either
// k-contiguous (x, w in the forward pass) or with the tile's axis contiguous (w
// for dx; dpre and x for dw), so no operand is transposed in memory. One warp
// loads, one thread of the leading CTA issues the MMAs, eight warps run the
// epilogue of a tile while the MMAs of the next fill the other half of tensor
// memory. Persistent grid, one cluster per SM pair.
//
// float32 operands: a float is the exact sum of three bfloat16 (its leading 8
// bits, the next 8, the last 8), kept as three planes; the product runs as the
// six plane pairs whose product can reach float32's last bit, smallest first,
// in the same loop over k blocks. Dropped pairs are below 2^-24 of |a||b|.
//
// Few output tiles for the SMs: the k blocks are split over several clusters,
// which leave float32 partial tiles that a second kernel adds in order and
// runs the epilogue on.
//
// Every wait is bounded (common.cuh): on a timeout the kernel records
// SCMP_ERR_TIMEOUT and all roles leave.
#include <cuda.h>

#include "linear.cuh"
#include "status.cuh"

namespace scmp {
namespace lin {

constexpr int KB = 64;            // k values per block: one 128-byte swizzled row
constexpr int EPI_WARPS = 8;
constexpr int TC_THREADS = 128 + 32 * EPI_WARPS;
constexpr int ACC_COLS = 256;     // tensor-memory columns between the two accumulators
constexpr int MAX_SEGMENTS = 6;

template <int BN>
struct Cfg {
  static constexpr int A_BYTES = 128 * KB * 2;
  static constexpr int B_BYTES = BN / 2 * KB * 2;
  static constexpr int STAGE = A_BYTES + B_BYTES;
  static constexpr int STAGES = BN == 256 ? 6 : 8;
  static constexpr int STG = EPI_WARPS * 4096;  // 32 rows x 128 bytes per epilogue warp
  static constexpr int BIAS = EPI_WARPS * 128;
  static constexpr int SMEM = STAGES * STAGE + STG + BIAS + 256 + 1024;
};

struct TcArgs {
  int m, n;              // output rows and columns
  int kblocks;           // k blocks of one plane pair
  int segments;          // plane pairs
  uint8_t pa[MAX_SEGMENTS], pb[MAX_SEGMENTS];
  int tiles_m, tiles_n, splits;
  int f16;               // operands are float16, else bfloat16
  int vec_out, vec_res, vec_pre, vec_codes;  // rows can be accessed 16 bytes at a time
  float* partial;        // (splits, m, n), or null
  Epilogue e;
};

__device__ __forceinline__ uint64_t desc_base(uint32_t lbo_bytes) {
  // version 1, 128-byte swizzle; 1024 bytes between 8-row (8-k) groups
  return ((uint64_t)(lbo_bytes >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) | ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
__device__ __forceinline__ void mma_f16_pair(uint32_t tmem, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem), "l"(a), "l"(b), "r"(idesc), "r"(acc)
      : "memory");
}
// Arrive on the barrier at this offset in both CTAs once all MMAs so far are done.
__device__ __forceinline__ void commit_pair(uint32_t bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar),
      "h"((uint16_t)0x3)
      : "memory");
}
__device__ __forceinline__ uint32_t leader_addr(uint32_t addr) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(addr));
  return r;
}
__device__ __forceinline__ void arrive_cluster(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void expect_tx(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
// A box of the tensor into this CTA's shared memory; the bytes count on the
// leading CTA's barrier.
__device__ __forceinline__ void tma_load(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t leader_bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::
          "r"(dst),
      "l"(map), "r"(x), "r"(y), "r"(z), "r"(leader_bar)
      : "memory");
}
__device__ __forceinline__ void tc_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_ld32(uint32_t addr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(addr));
}

template <class F>
__device__ __forceinline__ void act_each(float (&v)[32], F&& f) {
#pragma unroll
  for (int j = 0; j < 32; ++j) v[j] = f(v[j]);
}
__device__ __forceinline__ void act_values(int act, float (&v)[32]) {
  if (act == SCMP_ACT_RELU) act_each(v, [](float x) { return act_value(SCMP_ACT_RELU, x); });
  if (act == SCMP_ACT_GELU) act_each(v, [](float x) { return act_value(SCMP_ACT_GELU, x); });
  if (act == SCMP_ACT_GELU_TANH) act_each(v, [](float x) { return act_value(SCMP_ACT_GELU_TANH, x); });
  if (act == SCMP_ACT_SILU) act_each(v, [](float x) { return act_value(SCMP_ACT_SILU, x); });
}

// A warp's 32 rows x 32 columns between registers (a row per lane) and memory,
// through a 4 KB staging area: 16-byte pieces, the piece index of a row
// exclusive-ored so that neither side has bank conflicts; memory is accessed in
// whole row segments of 64 (16-bit) or 128 bytes.
template <class T>
struct Stage {
  static constexpr int PIECES = 32 * sizeof(T) / 16;  // 16-byte pieces per row: 4 or 8
  static constexpr int PER = 16 / sizeof(T);          // values per piece
  static __device__ __forceinline__ int slot(int row, int piece) {
    return row * PIECES + (piece ^ (PIECES == 4 ? (row >> 1) & 3 : row & 7));
  }
  static __device__ __forceinline__ void put_row(uint4* s, int lane, const float (&v)[32]) {
#pragma unroll
    for (int p = 0; p < PIECES; ++p) {
      uint4 q;
      T* e = reinterpret_cast<T*>(&q);
#pragma unroll
      for (int i = 0; i < PER; ++i) e[i] = Elem<T>::from_f(v[p * PER + i]);
      s[slot(lane, p)] = q;
    }
  }
  static __device__ __forceinline__ void add_row(const uint4* s, int lane, float (&v)[32]) {
#pragma unroll
    for (int p = 0; p < PIECES; ++p) {
      const uint4 q = s[slot(lane, p)];
      const T* e = reinterpret_cast<const T*>(&q);
#pragma unroll
      for (int i = 0; i < PER; ++i) v[p * PER + i] += Elem<T>::to_f(e[i]);
    }
  }
  // staging -> rows row0.. of a matrix, columns col0..col0+31
  static __device__ __forceinline__ void store(const uint4* s, int lane, T* base, long long ld, long long row0, int rows,
                                               int col0, int cols, bool vec) {
    if (vec && col0 + 32 <= cols) {
#pragma unroll
      for (int i = 0; i < PIECES; ++i) {
        const int row = i * (32 / PIECES) + lane / PIECES, p = lane % PIECES;
        if (row < rows) *reinterpret_cast<uint4*>(base + (row0 + row) * ld + col0 + p * PER) = s[slot(row, p)];
      }
    } else {
      const int c = lane;
      for (int row = 0; row < rows; ++row) {
        const T e = reinterpret_cast<const T*>(s + slot(row, c / PER))[c % PER];
        if (col0 + c < cols) base[(row0 + row) * ld + col0 + c] = e;
      }
    }
  }
  static __device__ __forceinline__ void load(uint4* s, int lane, const T* base, long long ld, long long row0, int rows,
                                              int col0, int cols, bool vec) {
    if (vec && col0 + 32 <= cols) {
#pragma unroll
      for (int i = 0; i < PIECES; ++i) {
        const int row = i * (32 / PIECES) + lane / PIECES, p = lane % PIECES;
        if (row < rows) s[slot(row, p)] = __ldg(reinterpret_cast<const uint4*>(base + (row0 + row) * ld + col0 + p * PER));
      }
    } else {
      const int c = lane;
      for (int row = 0; row < rows; ++row)
        reinterpret_cast<T*>(s + slot(row, c / PER))[c % PER] = col0 + c < cols ? base[(row0 + row) * ld + col0 + c] : T(0.f);
    }
  }
};

// Bias, checkpoint, activation, residual and stores of a warp's 32 x 32 piece
// (a row per lane in v).
template <class T, bool FULL>
__device__ __forceinline__ void finish_piece(const TcArgs& g, float (&v)[32], uint4* stg, float* bias_s, int lane,
                                             long long row0, int rows, int col0) {
  using S = Stage<T>;
  const Epilogue& e = g.e;
  if (FULL) {
    if (e.bias) {
      const int c = col0 + lane;
      bias_s[lane] = c >= g.n ? 0.f : e.bias_f32 ? __ldg((const float*)e.bias + c) : ldg1((const T*)e.bias + c);
      __syncwarp();
#pragma unroll
      for (int p = 0; p < 8; ++p) {
        const float4 b = reinterpret_cast<const float4*>(bias_s)[p];
        v[4 * p] += b.x;
        v[4 * p + 1] += b.y;
        v[4 * p + 2] += b.z;
        v[4 * p + 3] += b.w;
      }
    }
    if (e.pre) {
      S::put_row(stg, lane, v);
      __syncwarp();
      S::store(stg, lane, (T*)e.pre, g.n, row0, rows, col0, g.n, g.vec_pre);
      __syncwarp();
    }
    if (e.codes) {
      // the lane's 32 columns are one block of the checkpoint (columns past n count as zeros)
      uint32_t top = 0;
#pragma unroll
      for (int j = 0; j < 32; ++j) top = max(top, col0 + j < g.n ? __float_as_uint(v[j]) & 0x7FFFFFFFu : 0u);
      const uint32_t byte = act8_exponent(top, act8_floor<T>());
      const float inv = act8_inverse(byte);
      uint32_t w[8];
#pragma unroll
      for (int p = 0; p < 8; ++p) {
        w[p] = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) w[p] |= (uint32_t)(act8_code(v[4 * p + i], inv, byte == kAct8Nan) & 0xFF) << (8 * i);
      }
      if (lane < rows) {
        int8_t* dst = e.codes + (row0 + lane) * g.n + col0;
        if (g.vec_codes && col0 + 32 <= g.n) {
          reinterpret_cast<uint4*>(dst)[0] = make_uint4(w[0], w[1], w[2], w[3]);
          reinterpret_cast<uint4*>(dst)[1] = make_uint4(w[4], w[5], w[6], w[7]);
        } else {
#pragma unroll
          for (int j = 0; j < 32; ++j)
            if (col0 + j < g.n) dst[j] = (int8_t)(w[j >> 2] >> (8 * (j & 3)));
        }
        e.exps[(row0 + lane) * act8_blocks(g.n) + (col0 >> 5)] = (uint8_t)byte;
      }
    }
    act_values(e.act, v);
    if (e.residual) {
      S::load(stg, lane, (const T*)e.residual, e.ldr, row0, rows, col0, g.n, g.vec_res);
      __syncwarp();
      S::add_row(stg, lane, v);
      __syncwarp();
    }
  }
  S::put_row(stg, lane, v);
  __syncwarp();
  S::store(stg, lane, (T*)e.out, e.ldo, row0, rows, col0, g.n, g.vec_out);
  __syncwarp();
}

template <class T, bool A_MN, bool B_MN, int BN, bool FULL>
__global__ void __launch_bounds__(TC_THREADS, 1)
    gemm_tc_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                   const __grid_constant__ TcArgs g) {
  using C = Cfg<BN>;
  constexpr int NST = C::STAGES;
  extern __shared__ char smem_raw[];
  char* base = reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t sbase = smem_u32(base);
  char* tail = base + NST * C::STAGE + C::STG + C::BIAS;
  const uint32_t bars = smem_u32(tail);
  volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(tail + 8 * (2 * NST + 5));
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tail + 8 * (2 * NST + 5) + 4);
  auto full = [&](int s) { return bars + 8u * s; };
  auto empty = [&](int s) { return bars + 8u * (NST + s); };
  auto accf = [&](int b) { return bars + 8u * (2 * NST + b); };
  auto acce = [&](int b) { return bars + 8u * (2 * NST + 2 + b); };
  const uint32_t drain = bars + 8u * (2 * NST + 4);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint32_t rank;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  const int cluster = blockIdx.x >> 1, clusters = gridDim.x >> 1;

  if (warp == 1 && lane == 0) {
    for (int s = 0; s < NST; ++s) {
      mbar_init(full(s), 1);
      mbar_init(empty(s), 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(accf(b), 1);
      mbar_init(acce(b), 2 * EPI_WARPS);
    }
    mbar_init(drain, 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 2) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32((const void*)tmem_slot)),
                 "r"(512) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  if (warp == 0 && lane == 0) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(&map_a) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&map_b) : "memory");
  }
  tc_before();
  __syncthreads();
  cluster_sync();
  tc_after();
  const uint32_t tmem = *tmem_slot;

  const int tiles = g.tiles_m * g.tiles_n, items = tiles * g.splits, total_kb = g.kblocks * g.segments;
  // Tiles in bands of eight tile rows, column after column within a band, so
  // that the clusters running at a time share A's and B's rows in L2.
  auto place = [&](int item, int& tm, int& tn, int& k0, int& k1) {
    const int split = item / tiles, t = item - split * tiles;
    const int band = t / (8 * g.tiles_n), r = t - band * 8 * g.tiles_n;
    const int h = min(8, g.tiles_m - band * 8);
    tn = r / h;
    tm = band * 8 + r - tn * h;
    k0 = (int)((long long)total_kb * split / g.splits);
    k1 = (int)((long long)total_kb * (split + 1) / g.splits);
    return split;
  };

  if (warp == 0) {
    if (lane == 0) {
      uint32_t it = 0;
      bool ok = true;
      for (int item = cluster; item < items && ok; item += clusters) {
        int tm, tn, k0, k1;
        place(item, tm, tn, k0, k1);
        const int i0 = tm * 256 + (int)rank * 128, j0 = tn * BN + (int)rank * (BN / 2);
        int seg = k0 / g.kblocks, kb = k0 - seg * g.kblocks;
        for (int k = k0; k < k1; ++k, ++it) {
          const int s = it % NST;
          if (!mbar_wait(empty(s), ((it / NST) & 1) ^ 1, abort_flag, 20)) {
            ok = false;
            break;
          }
          const uint32_t a = sbase + s * C::STAGE, b = a + C::A_BYTES;
          const uint32_t lbar = leader_addr(full(s));
          if (rank == 0) expect_tx(full(s), 2 * C::STAGE);
          const int x = kb * KB, pa = g.pa[seg], pb = g.pb[seg];
          if (A_MN) {
            tma_load(a, &map_a, i0, x, pa, lbar);
            tma_load(a + 8192, &map_a, i0 + 64, x, pa, lbar);
          } else {
            tma_load(a, &map_a, x, i0, pa, lbar);
          }
          if (B_MN) {
            tma_load(b, &map_b, j0, x, pb, lbar);
            if (BN == 256) tma_load(b + 8192, &map_b, j0 + 64, x, pb, lbar);
          } else {
            tma_load(b, &map_b, x, j0, pb, lbar);
          }
          if (++kb == g.kblocks) {
            kb = 0;
            ++seg;
          }
        }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    if (rank == 0 && lane == 0) {
      // float32 accumulator, both operands of one 16-bit type, M = 256 over the pair
      const uint32_t ab = g.f16 ? 0u : 1u;
      const uint32_t idesc = (1u << 4) | (ab << 7) | (ab << 10) | ((A_MN ? 1u : 0u) << 15) | ((B_MN ? 1u : 0u) << 16) |
                             ((uint32_t)(BN >> 3) << 17) | (16u << 24);
      const uint64_t ad0 = desc_base(A_MN ? 8192 : 16), bd0 = desc_base(B_MN ? 8192 : 16);
      uint32_t it = 0, n_acc = 0;
      bool ok = true;
      for (int item = cluster; item < items && ok; item += clusters, ++n_acc) {
        int tm, tn, k0, k1;
        place(item, tm, tn, k0, k1);
        const int buf = n_acc & 1;
        if (!mbar_wait(acce(buf), ((n_acc >> 1) & 1) ^ 1, abort_flag, 21)) break;
        tc_after();
        const uint32_t acc = tmem + buf * ACC_COLS;
        for (int k = k0; k < k1; ++k, ++it) {
          const int s = it % NST;
          if (!mbar_wait(full(s), (it / NST) & 1, abort_flag, 22)) {
            ok = false;
            break;
          }
          tc_after();
          const uint32_t a = sbase + s * C::STAGE, b = a + C::A_BYTES;
          const uint64_t ad = ad0 | ((a >> 4) & 0x3FFF), bd = bd0 | ((b >> 4) & 0x3FFF);
#pragma unroll
          for (int q = 0; q < KB / 16; ++q)  // 16 k values: 32 bytes along a row, or two 8-k groups
            mma_f16_pair(acc, ad + q * (A_MN ? 128 : 2), bd + q * (B_MN ? 128 : 2), idesc, (k > k0 || q > 0) ? 1u : 0u);
          commit_pair(empty(s));
        }
        commit_pair(accf(buf));
      }
      // no MMA is in flight when tensor memory is freed
      asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(drain) : "memory");
      int none = 0;
      mbar_wait(drain, 0, &none, 23);
    }
    __syncwarp();
  } else if (warp >= 4) {
    const int ew = warp - 4, quad = ew & 3, half = ew >> 2;
    uint4* stg = reinterpret_cast<uint4*>(base + NST * C::STAGE + ew * 4096);
    float* bias_s = reinterpret_cast<float*>(base + NST * C::STAGE + C::STG + ew * 128);
    uint32_t n_acc = 0;
    for (int item = cluster; item < items; item += clusters, ++n_acc) {
      int tm, tn, k0, k1;
      const int split = place(item, tm, tn, k0, k1);
      const int buf = n_acc & 1;
      if (!mbar_wait(accf(buf), (n_acc >> 1) & 1, abort_flag, 24)) break;
      tc_after();
      const long long row0 = (long long)tm * 256 + rank * 128 + quad * 32;
      const int rows = (int)(g.m - row0 < 32 ? (g.m > row0 ? g.m - row0 : 0) : 32);
#pragma unroll 1
      for (int c = 0; c < BN / 64; ++c) {
        const int tc = half * (BN / 2) + c * 32, col0 = tn * BN + tc;
        uint32_t r[32];
        tmem_ld32(tmem + ((uint32_t)(quad * 32) << 16) + buf * ACC_COLS + tc, r);
        asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
        if (c == BN / 64 - 1) {  // the accumulator is read: the next tile's MMAs may overwrite it
          tc_before();
          __syncwarp();
          if (lane == 0) arrive_cluster(leader_addr(acce(buf)));
        }
        if (rows == 0 || col0 >= g.n) continue;
        float v[32];
#pragma unroll
        for (int j = 0; j < 32; ++j) v[j] = __uint_as_float(r[j]);
        if (g.partial) {
          Stage<float>::put_row(stg, lane, v);
          __syncwarp();
          Stage<float>::store(stg, lane, g.partial + (size_t)split * g.m * g.n, g.n, row0, rows, col0, g.n, g.n % 4 == 0);
          __syncwarp();
        } else {
          finish_piece<T, FULL>(g, v, stg, bias_s, lane, row0, rows, col0);
        }
      }
    }
  }
  if (*abort_flag) {
    // a wait gave up: let the copies in flight land before shared memory goes
    const long long t0 = clock64();
    while (clock64() - t0 < 2000000) {
    }
  }
  tc_before();
  __syncthreads();
  cluster_sync();
  if (warp == 2) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
}

// Adds the partial products in order and runs the epilogue: a lane per column
// (32 columns are one block of an 8-bit checkpoint), JOIN_ROWS rows per warp at
// a time so that their loads overlap.
constexpr int JOIN_ROWS = 4;
template <class T, bool FULL>
__global__ void __launch_bounds__(256) join_kernel(const __grid_constant__ TcArgs g) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long row0 = ((long long)blockIdx.y * 8 + warp) * JOIN_ROWS;
  const int col = blockIdx.x * 32 + lane;
  const bool live = col < g.n;
  const Epilogue& e = g.e;
  float v[JOIN_ROWS];
#pragma unroll
  for (int r = 0; r < JOIN_ROWS; ++r) v[r] = 0.f;
#pragma unroll 4
  for (int s = 0; s < g.splits; ++s) {
    const float* p = g.partial + ((size_t)s * g.m + row0) * g.n + col;
#pragma unroll
    for (int r = 0; r < JOIN_ROWS; ++r)
      if (live && row0 + r < g.m) v[r] += __ldg(p + (size_t)r * g.n);
  }
  const float bias = FULL && e.bias && live ? (e.bias_f32 ? __ldg((const float*)e.bias + col) : ldg1((const T*)e.bias + col)) : 0.f;
#pragma unroll
  for (int r = 0; r < JOIN_ROWS; ++r) {
    const long long row = row0 + r;
    if (row >= g.m) break;  // whole warps
    float y = v[r];
    if (FULL) {
      y += bias;
      if (e.pre && live) ((T*)e.pre)[row * g.n + col] = Elem<T>::from_f(y);
      if (e.codes) {
        const uint32_t byte = act8_exponent(__reduce_max_sync(0xffffffffu, live ? __float_as_uint(y) & 0x7FFFFFFFu : 0u), act8_floor<T>());
        if (live) e.codes[row * g.n + col] = (int8_t)act8_code(y, act8_inverse(byte), byte == kAct8Nan);
        if (lane == 0) e.exps[row * act8_blocks(g.n) + blockIdx.x] = (uint8_t)byte;
      }
      y = act_value(e.act, y);
      if (e.residual && live) y += ldg1((const T*)e.residual + row * e.ldr + col);
    }
    if (live) ((T*)e.out)[row * e.ldo + col] = Elem<T>::from_f(y);
  }
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
// An operand as TMA reads it: `planes` matrices of `outer` rows of `inner`
// 16-bit values at a pitch of ld values (a multiple of eight), 16-byte aligned.
// mn: the tile's axis is the inner one (else k is).
struct Operand {
  const void* p;
  long long inner, outer, ld;
  int planes;
  bool mn;
};

using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                 const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                 CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
static EncodeTiled encode_tiled() {
  static const EncodeTiled fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      p = nullptr;
    return (EncodeTiled)p;
  }();
  return fn;
}
static bool make_map(CUtensorMap* map, const Operand& o, bool f16, int tile_rows) {
  const cuuint64_t dims[3] = {(cuuint64_t)o.inner, (cuuint64_t)o.outer, (cuuint64_t)o.planes};
  const cuuint64_t strides[2] = {(cuuint64_t)o.ld * 2, (cuuint64_t)o.ld * 2 * o.outer};
  const cuuint32_t box[3] = {64, (cuuint32_t)(o.mn ? KB : tile_rows), 1}, one[3] = {1, 1, 1};
  return encode_tiled()(map, f16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3,
                        const_cast<void*>(o.p), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Tile width and number of k splits of a product.
struct Schedule {
  int bn, splits;
};
// Least estimated time, in SM clocks: waves of tiles over 74 SM pairs; a k block
// takes 560 clocks for 256 columns and 440 for 128 (32 and 24 KB per SM, at the
// 55 to 58 bytes per clock that L2 delivers to an SM: measured 566 and 444 on
// 4096 x 4096 x 11008); 2500 per tile that nothing hides; for a split product
// the partial tiles' way through L2 and a second launch.
static Schedule schedule_for(long long m, int n, long long kblocks) {
  Schedule best{256, 1};
  double least = 1e300;
  const long long pairs = 74;
  for (int bn : {256, 128}) {
    const long long tiles = ((m + 255) / 256) * ((n + bn - 1) / bn);
    for (int s = 1; s <= 16 && (s == 1 || kblocks / s >= 4); ++s) {
      const long long waves = (tiles * s + pairs - 1) / pairs;
      double t = waves * ((kblocks + s - 1) / s * (bn == 256 ? 560.0 : 440.0) + 2500.0);
      if (s > 1) t += 5000.0 + (double)m * n * (s + 1) * 4 / 2500.0;
      if (t < least) {
        least = t;
        best = {bn, s};
      }
    }
  }
  return best;
}
static int plane_pairs(int planes_a, int planes_b) { return planes_a == 1 ? planes_b : planes_b == 1 ? planes_a : 6; }
static size_t partial_bytes(long long m, int n, long long kblocks) {
  const Schedule s = schedule_for(m, n, kblocks);
  return s.splits > 1 ? (size_t)s.splits * m * n * sizeof(float) : 0;
}

template <class T, bool A_MN, bool B_MN, int BN, bool FULL>
static cudaError_t launch_tc_t(const CUtensorMap& ma, const CUtensorMap& mb, const TcArgs& g, cudaStream_t st) {
  auto kern = gemm_tc_kernel<T, A_MN, B_MN, BN, FULL>;
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg<BN>::SMEM);
  if (e != cudaSuccess) return e;
  const long long items = (long long)g.tiles_m * g.tiles_n * g.splits;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(2 * (items < 74 ? items : 74)), 1, 1);
  cfg.blockDim = dim3(TC_THREADS, 1, 1);
  cfg.dynamicSmemBytes = Cfg<BN>::SMEM;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = 2;
  at[0].val.clusterDim.y = 1;
  at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  e = cudaLaunchKernelEx(&cfg, kern, ma, mb, g);
  count_launch();
  if (e == cudaSuccess && g.splits > 1) {
    join_kernel<T, FULL><<<dim3(cdiv(g.n, 32), (unsigned)((g.m + 8LL * JOIN_ROWS - 1) / (8 * JOIN_ROWS))), 256, 0, st>>>(g);
    count_launch();
    e = cudaGetLastError();
  }
  return e;
}

// dtype: of the result and the epilogue's tensors; operands of a float32
// product are bfloat16 planes. partial: partial_bytes() of workspace.
static cudaError_t launch_tc(const Operand& a, const Operand& b, long long m, int n, long long k, const Epilogue& e, int dtype,
                             float* partial, cudaStream_t st) {
  if (!encode_tiled()) return cudaErrorNotSupported;
  TcArgs g{};
  g.m = (int)m;
  g.n = n;
  g.kblocks = (int)((k + KB - 1) / KB);
  g.segments = plane_pairs(a.planes, b.planes);
  static const uint8_t six_a[6] = {2, 0, 1, 1, 0, 0}, six_b[6] = {0, 2, 1, 0, 1, 0};
  for (int s = 0; s < g.segments; ++s) {
    g.pa[s] = b.planes == 1 ? g.segments - 1 - s : a.planes == 1 ? 0 : six_a[s];
    g.pb[s] = a.planes == 1 ? g.segments - 1 - s : b.planes == 1 ? 0 : six_b[s];
  }
  const Schedule sc = schedule_for(m, n, (long long)g.kblocks * g.segments);
  g.tiles_m = (int)((m + 255) / 256);
  g.tiles_n = cdiv(n, sc.bn);
  g.splits = sc.splits;
  g.f16 = dtype == SCMP_F16;
  g.partial = sc.splits > 1 ? partial : nullptr;
  g.e = e;
  const size_t es = dtype_size(dtype);
  g.vec_out = rows_aligned16(e.out, e.ldo, es);
  g.vec_res = rows_aligned16(e.residual, e.ldr, es);
  g.vec_pre = rows_aligned16(e.pre, n, es);
  g.vec_codes = aligned16(e.codes) && n % 16 == 0;
  CUtensorMap ma, mb;
  if (!make_map(&ma, a, g.f16, 128) || !make_map(&mb, b, g.f16, sc.bn / 2)) return cudaErrorInvalidValue;
  return with_dtype(dtype, [&](auto* tag) {
    using T = std::remove_pointer_t<decltype(tag)>;
    if (!a.mn && !b.mn)
      return sc.bn == 256 ? launch_tc_t<T, false, false, 256, true>(ma, mb, g, st) : launch_tc_t<T, false, false, 128, true>(ma, mb, g, st);
    if (!a.mn)
      return sc.bn == 256 ? launch_tc_t<T, false, true, 256, false>(ma, mb, g, st) : launch_tc_t<T, false, true, 128, false>(ma, mb, g, st);
    return sc.bn == 256 ? launch_tc_t<T, true, true, 256, false>(ma, mb, g, st) : launch_tc_t<T, true, true, 128, false>(ma, mb, g, st);
  });
}

// ---------------------------------------------------------------------------
// operands that TMA cannot read in place
// ---------------------------------------------------------------------------
// Rows at a 16-byte pitch; a float32 matrix as three bfloat16 planes (split3).
template <class T>
__global__ void __launch_bounds__(256) restage_kernel(const T* __restrict__ x, long long rows, int cols, long long ld,
                                                      uint16_t* __restrict__ out, long long ldo, bool vec) {
  const int oct = cdiv(cols, 8);
  const long long total = rows * oct, plane = rows * ldo;
  for (long long t = (long long)blockIdx.x * 256 + threadIdx.x; t < total; t += (long long)gridDim.x * 256) {
    const long long row = t / oct;
    const int c = (int)(t - row * oct) * 8;
    const T* src = x + row * ld + c;
    uint16_t* dst = out + row * ldo + c;
    if constexpr (sizeof(T) == 2) {
      uint16_t v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = c + i < cols ? __ldg(reinterpret_cast<const unsigned short*>(src) + i) : 0;
      *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(v);
    } else {
      float v[8];
      if (vec && c + 8 <= cols) {
        unpack8(ldg8(src), v);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = c + i < cols ? ldg1(src + i) : 0.f;
      }
      uint32_t w[3][4];
#pragma unroll
      for (int i = 0; i < 8; i += 2) {
        uint32_t lo[3], hi[3];
        split3(v[i], lo);
        split3(v[i + 1], hi);
#pragma unroll
        for (int p = 0; p < 3; ++p) w[p][i >> 1] = lo[p] | (hi[p] << 16);
      }
#pragma unroll
      for (int p = 0; p < 3; ++p) *reinterpret_cast<uint4*>(dst + p * plane) = make_uint4(w[p][0], w[p][1], w[p][2], w[p][3]);
    }
  }
}
static long long pitch_of(int cols) { return (cols + 7) / 8 * 8LL; }
static cudaError_t launch_restage(const void* x, long long rows, int cols, long long ld, int dtype, void* out, cudaStream_t st) {
  const long long items = rows * cdiv(cols, 8);
  const int grid = (int)((items + 255) / 256 < 148 * 8 ? (items + 255) / 256 : 148 * 8);
  if (dtype == SCMP_F32)
    restage_kernel<float><<<grid, 256, 0, st>>>((const float*)x, rows, cols, ld, (uint16_t*)out, pitch_of(cols), rows_aligned16(x, ld, 4));
  else
    restage_kernel<__half><<<grid, 256, 0, st>>>((const __half*)x, rows, cols, ld, (uint16_t*)out, pitch_of(cols), false);
  count_launch();
  return cudaGetLastError();
}

}  // namespace lin
}  // namespace scmp
