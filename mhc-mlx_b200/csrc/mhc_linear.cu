// Linear layer with its epilogue, and its gradients, in bf16 or fp16:
//
//   z = x W^T + b,  y = act(z) + residual
//   dz = dy act'(z),  dx = dz W,  dW = dz^T x,  db = sum over rows of dz
//
// x [M, K], W [N, K], y [M, N].  All three products are one tcgen05 GEMM
// D[m, n] = sum_r A[m, r] B[n, r] whose operands may be stored with the
// reduction along their rows or down their columns (W in dx; both in dW), fp32
// accumulators in tensor memory, bias, activation and residual applied as
// they are read back: z never makes a round trip through memory, unless the
// backward will want it: then it is written in fp32 beside y.  In the operands'
// type it would take half the room, but move a slope by up to 0.3 of the type's
// rounding of dy, most where the slope goes through 0.
//
// k_gemm: one CTA an SM walks 128 x BN output tiles (BN 256, 128 or 64 by the
// number of tiles):
//   warp 0      TMA: slices of 64 along the reduction, 128-byte swizzled, into a
//               ring that fills shared memory;
//   warp 1      four MMAs of 128 x BN x 16 a slice into one of two accumulators;
//   warps 2-9   read the other accumulator back and apply the epilogue while the
//               next tile's products run.  A thread holds a row of the tile;
//               32 rows x 64 columns at a time go through 4 KB of shared memory
//               of the warp's own, and from there as one TMA store (or, where
//               the output's rows are not on 16-byte boundaries, row by row with
//               the lanes along it): stores straight from registers touch 32
//               rows an instruction.
// Every wait is bounded: on one that runs out the CTA writes NaN into its
// remaining tiles and returns.
//
// Few rows (M <= 16) are bound by reading W once: k_few_rows, 16 rows of W to
// a block, its eight warps splitting K, with warp-level MMAs (a tensor-memory
// tile would be empty but for 1/8 of it).  Operands whose rows do not begin on
// 16-byte boundaries, which TMA cannot read, are copied to padded rows first.
//
// Measured, bf16, 8192 rows, 4096 to 11008, bias and SiLU: y and z 551 us,
// dz 122, db 7, dx 477, dW 521 us (1.34 to 1.55 PFLOP/s, 0.82 to 0.95 of what a
// library product reaches in a burst).  One after the other they take 2.0 ms
// rather than these 1.68: the products draw the power limit.  Pairs of CTAs
// sharing 256 x 256 tiles, with half the operand traffic, were no faster (551,
// 515, 550 us where single ones took 537, 493, 538).  One token of 4096 x 4096 by
// launches in a row: 7.7 us with the weights from HBM (12 layers' in turn, 33.6 MB
// each, 4.4 TB/s), 4.8 us where L2 holds them.
#include <math_constants.h>

#include "mhc_internal.h"
#include "mhc_tcgen05.cuh"

namespace mhc {
namespace {

enum Act { kNone = 0, kRelu = 1, kSilu = 2, kGelu = 3 };

// The fast exponential and quotient: off by some 2^-20 where |z| is ordinary, far
// below the 16-bit rounding of what comes of them.
template <int ACT>
__device__ __forceinline__ float act_of(float z) {
  if constexpr (ACT == kRelu) return z < 0.f ? 0.f : z;  // keeps NaN
  if constexpr (ACT == kSilu) return __fdividef(z, 1.0f + __expf(-z));
  if constexpr (ACT == kGelu) return 0.5f * z * (1.0f + erff(z * 0.70710678118654752f));
  return z;
}
template <int ACT>
__device__ __forceinline__ float act_slope(float z) {
  if constexpr (ACT == kRelu) return z > 0.f ? 1.f : (z == z ? 0.f : z);
  if constexpr (ACT == kSilu) {
    const float q = __fdividef(1.0f, 1.0f + __expf(-z));
    return q * (1.0f + z * (1.0f - q));
  }
  if constexpr (ACT == kGelu)
    return 0.5f * (1.0f + erff(z * 0.70710678118654752f)) +
           z * 0.39894228040143268f * __expf(-0.5f * z * z);
  return 1.f;
}

// ------------------------------------------------------------------- GEMM --
constexpr int kBM = 128, kBK = 64;
constexpr int kThreads = 320;

template <int BN>
struct Ring {
  static constexpr int kA = kBM * kBK * 2, kB = BN * kBK * 2, kStage = kA + kB;
  static constexpr int kStages = BN == 256 ? 4 : BN == 128 ? 6 : 8;
  static constexpr int kOut = 8 * 4096;  // the epilogue warps' stages
  static constexpr int kBytes = kStages * kStage + kOut + 1024;  // + alignment slack
  static_assert(kBytes <= 226 * 1024, "shared memory");
};

template <typename T>
struct Epilogue {
  const T* bias;      // [N], nullable
  const T* residual;  // [M][ldr], nullable
  float* z;           // [M][ldz], nullable
  T* d;               // [M][ldd]
  int64_t ldr, ldz, ldd;
  int M, N;
  int wide_res, wide_d;  // 16-byte accesses are possible
};

// Up to 8 consecutive values from p as fp32, 0 past n.
template <typename T>
__device__ __forceinline__ void read8(const T* p, bool wide, int n, float (&o)[8]) {
  if (wide && n >= 8) {
    unpack16<T, 8>(__ldg(reinterpret_cast<const uint4*>(p)), o);
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) o[k] = k < n ? to_f(p[k]) : 0.f;
  }
}
// Eight fp32 values rounded to T.
template <typename T>
__device__ __forceinline__ uint4 pack8(const float (&v)[8]) {
  return make_uint4(pack2_16<T>(v[0], v[1]), pack2_16<T>(v[2], v[3]), pack2_16<T>(v[4], v[5]),
                    pack2_16<T>(v[6], v[7]));
}
// A warp's stage: 32 rows of 64 values, 128 bytes a row, 16-byte chunks swizzled
// by the row as TMA does it.
__device__ __forceinline__ uint4* chunk_of(uint8_t* stage, int row, int chunk) {
  return reinterpret_cast<uint4*>(stage + row * 128 + ((chunk ^ (row & 7)) << 4));
}
__device__ __forceinline__ uint32_t* pair_of(uint8_t* stage, int row, int pair) {
  return reinterpret_cast<uint32_t*>(stage + row * 128 + (((pair >> 2) ^ (row & 7)) << 4) + (pair & 3) * 4);
}
// Rows of a matrix <-> the stage, lanes along the row: two values a lane.
template <typename T>
__device__ __forceinline__ void rows_out(T* p, int64_t ld, uint8_t* stage, int lane, int rows, int cols) {
  const int c = 2 * lane;
  for (int i = 0; i < rows; ++i) {
    const uint32_t v = *pair_of(stage, i, lane);
    uint16_t* q = reinterpret_cast<uint16_t*>(p + i * ld + c);
    if (c + 1 < cols && (reinterpret_cast<uintptr_t>(q) & 3u) == 0) {
      *reinterpret_cast<uint32_t*>(q) = v;
    } else {
      if (c < cols) q[0] = (uint16_t)v;
      if (c + 1 < cols) q[1] = (uint16_t)(v >> 16);
    }
  }
}
template <typename T>
__device__ __forceinline__ void rows_in(const T* p, int64_t ld, uint8_t* stage, int lane, int rows, int cols) {
  const int c = 2 * lane;
#pragma unroll 8
  for (int i = 0; i < rows; ++i) {
    const uint16_t* q = reinterpret_cast<const uint16_t*>(p + i * ld + c);
    uint32_t v = 0;
    if (c + 1 < cols && (reinterpret_cast<uintptr_t>(q) & 3u) == 0) {
      v = *reinterpret_cast<const uint32_t*>(q);
    } else {
      if (c < cols) v = q[0];
      if (c + 1 < cols) v |= (uint32_t)q[1] << 16;
    }
    *pair_of(stage, i, lane) = v;
  }
}
__device__ __forceinline__ void tma_store_2d(const CUtensorMap* map, const void* src, int x, int y) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%1, %2}], [%3];\n" ::"l"(
                   reinterpret_cast<uint64_t>(map)),
               "r"(x), "r"(y), "r"(smem_u32(src))
               : "memory");
  asm volatile("cp.async.bulk.commit_group;\n" ::: "memory");
}
__device__ __forceinline__ void tma_store_read() {  // the stages of this thread's stores are free
  asm volatile("cp.async.bulk.wait_group.read 0;\n" ::: "memory");
}

// Tiles in groups of up to kGroupM rows of tiles, each group column by column:
// the tiles at work at one time share a few panels of both operands in L2.
constexpr int kGroupM = 12;
__device__ __forceinline__ void tile_at(int t, int tm, int tn, int& m, int& n) {
  const int per = kGroupM * tn, g = t / per, r = t - g * per;
  const int rows = min(kGroupM, tm - g * kGroupM);
  n = r / rows;
  m = g * kGroupM + (r - n * rows);
}

template <typename T, int BN, bool AT, bool BT, int ACT>
__global__ void __launch_bounds__(kThreads, 1)
k_gemm(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
       const __grid_constant__ CUtensorMap map_d, const __grid_constant__ CUtensorMap map_z,
       const Epilogue<T> ep, int slices, int tm, int tn) {
  using L = Ring<BN>;
  constexpr int S = L::kStages;
  constexpr uint32_t kCols = 2 * BN;
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t full[S], empty[S], acc_full[2], acc_empty[2];
  __shared__ uint32_t s_tmem;
  __shared__ int s_abort;
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~uintptr_t(1023));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int tiles = tm * tn;
  volatile int* abort_flag = &s_abort;
  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&acc_full[b], 1);
      mbar_init(&acc_empty[b], 8);
    }
    s_abort = 0;
    mbar_init_fence();
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(
                     smem_u32(&s_tmem)),
                 "r"(kCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s_tmem;

  if (warp == 0) {
    // ---------------------------------------------------------------- TMA --
    if (lane == 0) {
      int it = 0;
      for (int t = blockIdx.x; t < tiles && !*abort_flag; t += gridDim.x) {
        int m, n;
        tile_at(t, tm, tn, m, n);
        for (int k = 0; k < slices; ++k, ++it) {
          const int s = it % S;
          if (!wait_or_abort(&empty[s], ((unsigned)(it / S) & 1u) ^ 1u, abort_flag)) {
            s_abort = 1;
            break;
          }
          uint8_t* a = smem + s * L::kStage;
          uint8_t* b = a + L::kA;
          mbar_arrive_expect_tx(&full[s], (unsigned)L::kStage);
          // reduction-major operands come as 64 x 64 blocks: [block][64 of the
          // reduction][128 bytes]; the others as one box of rows
          if constexpr (AT) {
            for (int j = 0; j < kBM / 64; ++j) tma_2d(a + j * 8192, &map_a, m * kBM + j * 64, k * kBK, &full[s]);
          } else {
            tma_2d(a, &map_a, k * kBK, m * kBM, &full[s]);
          }
          if constexpr (BT) {
            for (int j = 0; j < BN / 64; ++j) tma_2d(b + j * 8192, &map_b, n * BN + j * 64, k * kBK, &full[s]);
          } else {
            tma_2d(b, &map_b, k * kBK, n * BN, &full[s]);
          }
        }
      }
      // copies in flight land before the CTA's shared memory goes away: the MMAs have
      // waited for them, unless some wait has run out (this loop may have ended before)
      for (int i = it - S < 0 ? 0 : it - S; i < it; ++i) (void)mbar_wait(&full[i % S], (unsigned)(i / S) & 1u);
    }
  } else if (warp == 1) {
    // ---------------------------------------------------------------- MMA --
    if (lane == 0) {
      constexpr uint32_t ab = std::is_same<T, bf16>::value ? 1u : 0u;
      constexpr uint32_t idesc = f16_idesc(ab, BT ? 1u : 0u, kBM, BN, AT ? 1u : 0u);
      int it = 0, i = 0;
      for (int t = blockIdx.x; t < tiles; t += gridDim.x, ++i) {
        const int buf = i & 1;
        bool ok = wait_or_abort(&acc_empty[buf], ((unsigned)(i >> 1) & 1u) ^ 1u, abort_flag);
        tc_fence_after();
        for (int k = 0; ok && k < slices; ++k, ++it) {
          const int s = it % S;
          ok = wait_or_abort(&full[s], (unsigned)(it / S) & 1u, abort_flag);
          if (!ok) break;
          tc_fence_after();
          const uint32_t a0 = smem_u32(smem + s * L::kStage), b0 = a0 + L::kA;
#pragma unroll
          for (int kk = 0; kk < kBK / 16; ++kk) {
            // 16 of the reduction: 32 bytes along a row, or two groups of 8 rows
            const uint64_t ad = AT ? sw128_desc(a0 + kk * 2048, 8192, 1024) : sw128_desc(a0 + kk * 32, 16, 1024);
            const uint64_t bd = BT ? sw128_desc(b0 + kk * 2048, 8192, 1024) : sw128_desc(b0 + kk * 32, 16, 1024);
            umma_f16(tmem + buf * BN, ad, bd, idesc, (k | kk) != 0 ? 1u : 0u);
          }
          umma_commit(&empty[s]);
        }
        umma_commit(&acc_full[buf]);  // also after an abort: marks the issued MMAs' completion
        if (!ok) {
          s_abort = 1;
          // they still read shared memory and write the accumulators that are freed below
          (void)mbar_wait(&acc_full[buf], (unsigned)(i >> 1) & 1u);
          break;
        }
      }
    }
  } else {
    // ----------------------------------------------------------- epilogue --
    // TMEM lanes 32 sp ..; half of the columns (of 64 in all: the first half all)
    const int sp = warp & 3, half = (warp - 2) >> 2;
    const int c0 = BN == 64 ? (half ? 64 : 0) : half * (BN / 2), c1 = BN == 64 ? 64 : c0 + BN / 2;
    uint8_t* stage = smem + S * L::kStage + (warp - 2) * 4096;
    int i = 0;
    bool ok = true;
    for (int t = blockIdx.x; t < tiles; t += gridDim.x, ++i) {
      const int buf = i & 1;
      int m, n;
      tile_at(t, tm, tn, m, n);
      const int row0 = m * kBM + sp * 32, rows = min(32, ep.M - row0);
      // what does not hang on the products comes while they run: the bias, and the
      // residual (its first 64 columns into the stage, or all of it into L2)
      float bias[4] = {};  // of columns c0 + lane, + 32, + 64, + 96
      if (ep.bias) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int c = c0 + 32 * k + lane;
          if (c < c1 && n * BN + c < ep.N) bias[k] = to_f(ep.bias[n * BN + c]);
        }
      }
      if (ep.residual && rows > 0) {
        if (!ep.wide_res) {
          if (lane == 0) tma_store_read();
          __syncwarp();
          if (c0 < c1) rows_in(ep.residual + (int64_t)row0 * ep.ldr + n * BN + c0, ep.ldr, stage, lane, rows, ep.N - n * BN - c0);
        } else if (lane < rows) {
          for (int c = n * BN + c0; c < n * BN + c1 && c < ep.N; c += 64)
            asm volatile("prefetch.global.L2 [%0];" ::"l"(ep.residual + (int64_t)(row0 + lane) * ep.ldr + c));
        }
      }
      __syncwarp();
      if (ok) ok = __all_sync(0xffffffffu, wait_or_abort(&acc_full[buf], (unsigned)(i >> 1) & 1u, abort_flag) && !*abort_flag);
      tc_fence_after();
#pragma unroll 1
      for (int c = c0; c < c1; c += 64) {
        const int col = n * BN + c, cols = min(64, ep.N - col);
        if (rows <= 0 || cols <= 0) break;
        // 32 of the 64 columns (half h), with the bias
        const auto read_acc = [&](int h, float (&v)[32]) {
          uint32_t r[32];
          if (ok) tmem_ld32(tmem + ((uint32_t)(sp * 32) << 16) + (uint32_t)(buf * BN + c + 32 * h), r);
          const float bl = c == c0 ? (h ? bias[1] : bias[0]) : (h ? bias[3] : bias[2]);
#pragma unroll
          for (int e = 0; e < 32; ++e) v[e] = ok ? __uint_as_float(r[e]) : CUDART_NAN_F;
          if (ep.bias) {
#pragma unroll
            for (int e = 0; e < 32; ++e) v[e] += __shfl_sync(0xffffffffu, bl, e);
          }
        };
        const bool staged = ep.residual != nullptr && !ep.wide_res;
        if (!staged || c != c0) {
          if (lane == 0) tma_store_read();
          __syncwarp();
        }
        if (staged && c != c0) {
          rows_in(ep.residual + (int64_t)row0 * ep.ldr + col, ep.ldr, stage, lane, rows, cols);
          __syncwarp();
        }
#pragma unroll 1
        for (int h = 0; h < 2; ++h) {
          float a[32];
          read_acc(h, a);
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const int e0 = 32 * h + 8 * q;
            float v[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = act_of<ACT>(a[8 * q + e]);
            uint4* at = chunk_of(stage, lane, 4 * h + q);
            if (ep.residual) {
              float b[8];
              if (staged) unpack16<T, 8>(*at, b);
              else read8(ep.residual + (int64_t)(row0 + lane) * ep.ldr + col + e0, 1, lane < rows ? cols - e0 : 0, b);
#pragma unroll
              for (int e = 0; e < 8; ++e) v[e] += b[e];
            }
            *at = pack8<T>(v);
          }
        }
        if (ep.wide_d) {
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) tma_store_2d(&map_d, stage, col, row0);
        } else {
          __syncwarp();
          rows_out(ep.d + (int64_t)row0 * ep.ldd + col, ep.ldd, stage, lane, rows, cols);
          __syncwarp();
        }
        // z where it is wanted: the accumulator is read again, 32 columns fill the stage
#pragma unroll 1
        for (int h = 0; ep.z && 32 * h < cols && h < 2; ++h) {
          float a[32];
          read_acc(h, a);
          if (lane == 0) tma_store_read();
          __syncwarp();
#pragma unroll
          for (int q = 0; q < 8; ++q)
            *chunk_of(stage, lane, q) = make_uint4(__float_as_uint(a[4 * q]), __float_as_uint(a[4 * q + 1]),
                                                   __float_as_uint(a[4 * q + 2]), __float_as_uint(a[4 * q + 3]));
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) tma_store_2d(&map_z, stage, col + 32 * h, row0);
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];\n" ::"r"(smem_u32(&acc_empty[buf])) : "memory");
    }
    if (lane == 0) tma_store_read();
  }
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem), "r"(kCols) : "memory");
  }
}

// --------------------------------------------------------------- few rows --
// Eight values at row + k (0 past K), whatever the row's alignment: the two
// 16-byte granules that hold them, shifted into place.  Both hold values of
// this row, so neither leaves the memory that the tensor lies in.
__device__ __forceinline__ uint4 eight_at(const uint16_t* row, int k, int K) {
  if (k + 8 > K) {
    uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (k + e < K) w[e >> 1] |= (uint32_t)row[k + e] << (16 * (e & 1));
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
  const uintptr_t at = reinterpret_cast<uintptr_t>(row + k);
  const uint4* g = reinterpret_cast<const uint4*>(at & ~(uintptr_t)15);
  const uint4 a = __ldg(g);
  const int off = (int)(at & 15);
  if (off == 0) return a;
  const uint4 b = __ldg(g + 1);
  uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
  if (off & 8) {
#pragma unroll
    for (int i = 0; i < 6; ++i) w[i] = w[i + 2];
  }
  if (off & 4) {
#pragma unroll
    for (int i = 0; i < 5; ++i) w[i] = w[i + 1];
  }
  const int sh = 8 * (off & 2);
  return make_uint4(__funnelshift_r(w[0], w[1], sh), __funnelshift_r(w[1], w[2], sh),
                    __funnelshift_r(w[2], w[3], sh), __funnelshift_r(w[3], w[4], sh));
}

// y^T tile of 16 features x 8 MT tokens: D = W x^T with m16n8k16 MMAs.  A lane's
// fragments are 8 consecutive k of two rows of W and of MT rows of x (16 bytes
// each): the MMA's own order of k is permuted, alike for both operands.  The
// warps take every eighth slice of 32 k; their sums meet in shared memory, in
// order.
template <typename T, int MT, int ACT, bool ALIGNED>
__global__ void __launch_bounds__(256, 2)
k_few_rows(const T* __restrict__ x, int64_t ldx, const T* __restrict__ w, int64_t ldw,
           const Epilogue<T> ep, int K) {
  constexpr int kU = MT == 1 ? 8 : 4;  // slices in flight
  __shared__ float part[8][16][8 * MT + 1];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int r = lane >> 2, q = lane & 3;
  const int n0 = blockIdx.x * 16;
  const T* w0 = w + (int64_t)min(n0 + r, ep.N - 1) * ldw;  // rows past N: any row, not stored
  const T* w1 = w + (int64_t)min(n0 + r + 8, ep.N - 1) * ldw;
  const auto get = [&](const T* row, int k) -> uint4 {
    if constexpr (ALIGNED) return k < K ? __ldg(reinterpret_cast<const uint4*>(row + k)) : make_uint4(0, 0, 0, 0);
    else return eight_at(reinterpret_cast<const uint16_t*>(row), k, K);
  };
  float acc[MT][4];
#pragma unroll
  for (int j = 0; j < MT; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[j][e] = 0.f;
  for (int k0 = warp * 32; k0 < K; k0 += kU * 256) {
    uint4 a[kU], b[kU], c[kU][MT];
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      const int k = k0 + u * 256 + 8 * q;
      a[u] = get(w0, k);
      b[u] = get(w1, k);
#pragma unroll
      for (int j = 0; j < MT; ++j)
        c[u][j] = r + 8 * j < ep.M ? get(x + (int64_t)(r + 8 * j) * ldx, k) : make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      const unsigned lo[4] = {a[u].x, b[u].x, a[u].y, b[u].y}, hi[4] = {a[u].z, b[u].z, a[u].w, b[u].w};
#pragma unroll
      for (int j = 0; j < MT; ++j) {
        mma_16816<T>(acc[j], lo, c[u][j].x, c[u][j].y);
        mma_16816<T>(acc[j], hi, c[u][j].z, c[u][j].w);
      }
    }
  }
#pragma unroll
  for (int j = 0; j < MT; ++j) {
    part[warp][r][8 * j + 2 * q] = acc[j][0];
    part[warp][r][8 * j + 2 * q + 1] = acc[j][1];
    part[warp][r + 8][8 * j + 2 * q] = acc[j][2];
    part[warp][r + 8][8 * j + 2 * q + 1] = acc[j][3];
  }
  __syncthreads();
  for (int i = threadIdx.x; i < 16 * 8 * MT; i += 256) {
    const int f = i & 15, tok = i >> 4, n = n0 + f;
    if (tok >= ep.M || n >= ep.N) continue;
    float v = 0.f;
#pragma unroll
    for (int p = 0; p < 8; ++p) v += part[p][f][tok];
    if (ep.bias) v += to_f(ep.bias[n]);
    if (ep.z) ep.z[(int64_t)tok * ep.ldz + n] = v;
    v = act_of<ACT>(v);
    if (ep.residual) v += to_f(ep.residual[(int64_t)tok * ep.ldr + n]);
    ep.d[(int64_t)tok * ep.ldd + n] = from_f<T>(v);
  }
}

// ------------------------------------------------------- dz, db, padded rows --
// dz = dy act'(z) for a tile of `per` rows x 256 columns (8 a thread), and the
// tile's column sums.  dz may be null (no activation, rows as TMA wants them).
template <typename T, int ACT>
__global__ void __launch_bounds__(256)
k_act_grad(const T* __restrict__ dy, int64_t ldy, const float* __restrict__ z, int64_t ldz,
           T* __restrict__ dz, int64_t lddz, float* __restrict__ part, int64_t M, int N, int per, int wide_dy) {
  __shared__ float red[8][256];
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const int col = blockIdx.x * 256 + tx * 8, left = N - col;
  const int64_t m0 = (int64_t)blockIdx.y * per, m1 = m0 + per < M ? m0 + per : M;
  float sum[8] = {};
  if (left > 0) {
    for (int64_t m = m0 + ty; m < m1; m += 8) {
      float d[8];
      read8(dy + m * ldy + col, wide_dy, left, d);
      if constexpr (ACT != kNone) {
        float v[8];
        load_vec<float, 8>(z + m * ldz + col, v);  // z's rows are padded to 8
#pragma unroll
        for (int e = 0; e < 8; ++e) d[e] *= act_slope<ACT>(v[e]);
        if (left < 8) {
#pragma unroll
          for (int e = 0; e < 8; ++e) d[e] = e < left ? d[e] : 0.f;  // what lies in z's padding is nothing
        }
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) sum[e] += d[e];
      if (dz) store_vec<T, 8, false>(dz + m * lddz + col, d);
    }
  }
  if (!part) return;
#pragma unroll
  for (int e = 0; e < 8; ++e) red[ty][tx * 8 + e] = sum[e];
  __syncthreads();
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c < N) {
    float s = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) s += red[k][threadIdx.x];
    part[(int64_t)blockIdx.y * N + c] = s;
  }
}
template <typename T>
__global__ void __launch_bounds__(256)
k_bias_sum(const float* __restrict__ part, int rows, int N, T* __restrict__ db) {
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= N) return;
  float s = 0.f;
  for (int r = 0; r < rows; ++r) s += part[(int64_t)r * N + c];
  db[c] = from_f<T>(s);
}
// Rows of `cols` values at stride ld -> rows padded with zeros to ldp: one or two
// matrices in a launch.
template <typename T>
struct Pad {
  const T* src;
  T* dst;
  int64_t ld, ldp, rows;
  int cols;
};
template <typename T>
__global__ void __launch_bounds__(256)
k_pad(const Pad<T> a, const Pad<T> b) {
  const int64_t na = a.rows * (a.ldp / 8), total = na + b.rows * (b.ldp / 8);
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const Pad<T>& p = i < na ? a : b;
    const int64_t j = i < na ? i : i - na, per = p.ldp / 8, m = j / per;
    const int c = (int)(j - m * per) * 8;
    float v[8];
    read8(p.src + m * p.ld + c, false, p.cols - c, v);
    store_vec<T, 8, false>(p.dst + m * p.ldp + c, v);
  }
}

// ------------------------------------------------------------------- host --
bool tma_rows(const void* p, int64_t ld) { return aligned16(p) && ld % 8 == 0; }
int64_t up8(int64_t v) { return (v + 7) / 8 * 8; }
size_t up256(size_t v) { return (v + 255) / 256 * 256; }
size_t padded_bytes(int64_t rows, int64_t cols) { return up256((size_t)rows * (size_t)up8(cols) * 2); }

// A bump allocator over the caller's workspace.
struct Space {
  char* p;
  char* end;
  void* take(size_t n) {
    char* q = p;
    p += up256(n);
    return p <= end ? q : nullptr;
  }
};
int no_space(const char* fn) {
  return set_error(MHC_ERR_WORKSPACE, "%s: workspace smaller than its *_workspace_bytes()", fn);
}

struct Matrix {  // rows x cols values, rows ld apart
  const void* p;
  int64_t rows, cols, ld;
};
// The matrices (either may be null) with rows that TMA can read: padded copies
// where they are not.
template <typename T>
int for_tma(const char* fn, Matrix* a, Matrix* b, Space& ws, cudaStream_t st) {
  Pad<T> p[2] = {};
  int64_t work = 0;
  int n = 0;
  for (Matrix* m : {a, b}) {
    if (!m || tma_rows(m->p, m->ld)) continue;
    void* q = ws.take(padded_bytes(m->rows, m->cols));
    if (!q) return no_space(fn);
    const int64_t ldp = up8(m->cols);
    p[n++] = {static_cast<const T*>(m->p), static_cast<T*>(q), m->ld, ldp, m->rows, (int)m->cols};
    work += m->rows * (ldp / 8);
    m->p = q;
    m->ld = ldp;
  }
  if (n == 0) return MHC_OK;
  int64_t blocks = (work + 255) / 256;
  if (blocks > (int64_t)sm_count() * 16) blocks = (int64_t)sm_count() * 16;
  k_pad<T><<<(unsigned)blocks, 256, 0, st>>>(p[0], p[1]);
  return check_launch(fn);
}

template <typename T, int BN, bool AT, bool BT, int ACT>
int run_gemm(const char* fn, const Matrix& a, const Matrix& b, const Epilogue<T>& ep, int64_t red,
             cudaStream_t st) {
  CUtensorMap ma, mb;
  const CUtensorMapDataType dt =
      std::is_same<T, bf16>::value ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  int r = make_tensor_map(fn, &ma, dt, a.p, (uint64_t)a.cols, (uint64_t)a.rows, (uint64_t)a.ld * 2, 64,
                          AT ? 64 : kBM, CU_TENSOR_MAP_SWIZZLE_128B);
  if (r != MHC_OK) return r;
  r = make_tensor_map(fn, &mb, dt, b.p, (uint64_t)b.cols, (uint64_t)b.rows, (uint64_t)b.ld * 2, 64,
                      BT ? 64 : BN, CU_TENSOR_MAP_SWIZZLE_128B);
  if (r != MHC_OK) return r;
  // outputs: 64 columns (z: 32) x 32 rows a store; a map that is not used is the operand's
  CUtensorMap md = ma, mz = ma;
  if (ep.wide_d) {
    r = make_tensor_map(fn, &md, dt, ep.d, (uint64_t)ep.N, (uint64_t)ep.M, (uint64_t)ep.ldd * 2, 64, 32,
                        CU_TENSOR_MAP_SWIZZLE_128B);
    if (r != MHC_OK) return r;
  }
  if (ep.z) {
    r = make_tensor_map(fn, &mz, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, ep.z, (uint64_t)ep.N, (uint64_t)ep.M,
                        (uint64_t)ep.ldz * 4, 32, 32, CU_TENSOR_MAP_SWIZZLE_128B);
    if (r != MHC_OK) return r;
  }
  const auto kern = k_gemm<T, BN, AT, BT, ACT>;
  const cudaError_t e = allow_dyn_smem(kern, Ring<BN>::kBytes);
  if (e != cudaSuccess) return set_error(MHC_ERR_CUDA, "%s: %s", fn, cudaGetErrorString(e));
  const int tm = (ep.M + kBM - 1) / kBM, tn = (ep.N + BN - 1) / BN;
  if ((int64_t)tm * tn > 0x7fffffff - 65536)
    return set_error(MHC_ERR_UNSUPPORTED, "%s: %d x %d outputs are too many", fn, ep.M, ep.N);
  const int grid = tm * tn < sm_count() ? tm * tn : sm_count();
  kern<<<grid, kThreads, Ring<BN>::kBytes, st>>>(ma, mb, md, mz, ep, (int)((red + kBK - 1) / kBK), tm, tn);
  return check_launch(fn);
}
// The tile width with the least time by waves of tiles: a 128 x 256 tile takes
// about 1, a 128 x 128 one 0.55 and a 128 x 64 one 0.33 (the narrow ones read the
// A operand more often from shared memory).
int tile_width(int64_t M, int64_t N) {
  const int64_t sms = sm_count(), tm = (M + kBM - 1) / kBM;
  const int width[3] = {256, 128, 64};
  const double cost[3] = {1.0, 0.55, 0.33};
  int best = 256;
  double least = 1e300;
  for (int i = 0; i < 3; ++i) {
    const int64_t tiles = tm * ((N + width[i] - 1) / width[i]);
    const double t = (double)((tiles + sms - 1) / sms) * cost[i];
    if (t < least) {
      least = t;
      best = width[i];
    }
  }
  return best;
}
template <typename T, bool AT, bool BT, int ACT>
int gemm(const char* fn, const Matrix& a, const Matrix& b, const Epilogue<T>& ep, int64_t red,
         cudaStream_t st) {
  const int bn = tile_width(ep.M, ep.N);
  if (bn == 256) return run_gemm<T, 256, AT, BT, ACT>(fn, a, b, ep, red, st);
  if (bn == 128) return run_gemm<T, 128, AT, BT, ACT>(fn, a, b, ep, red, st);
  return run_gemm<T, 64, AT, BT, ACT>(fn, a, b, ep, red, st);
}

constexpr int kFewRows = 16;
// Rows to a block of k_act_grad: 128, fewer (down to 16) while there are not two
// blocks an SM, more where they would be more than a grid's second axis takes.
int rows_per(int64_t M, int64_t N) {
  constexpr int64_t kMost = 65535;
  if (M > 128 * kMost) return (int)up8((M + kMost - 1) / kMost);
  int per = 128;
  while (per > 16 && (M + per - 1) / per * ((N + 255) / 256) < 2 * (int64_t)sm_count()) per /= 2;
  return per;
}

template <typename T>
Epilogue<T> epilogue(void* d, int64_t ldd, int64_t M, int64_t N) {
  Epilogue<T> ep = {};
  ep.d = static_cast<T*>(d);
  ep.ldd = ldd;
  ep.M = (int)M;
  ep.N = (int)N;
  ep.wide_d = tma_rows(d, ldd);
  return ep;
}

template <typename T, int ACT>
int forward(const LinearArg& l, cudaStream_t st) {
  const char* fn = "mhc_linear_fwd";
  Epilogue<T> ep = epilogue<T>(l.y, l.ldy, l.M, l.N);
  ep.bias = static_cast<const T*>(l.bias);
  ep.residual = static_cast<const T*>(l.residual);
  ep.ldr = l.ldr;
  ep.z = static_cast<float*>(l.z);
  ep.ldz = l.ldz;
  ep.wide_res = tma_rows(l.residual, l.ldr);
  if (l.M <= kFewRows) {
    const bool aligned = tma_rows(l.x, l.ldx) && tma_rows(l.w, l.ldw) && l.K % 8 == 0;
    const unsigned grid = (unsigned)((l.N + 15) / 16);
    const T *x = static_cast<const T*>(l.x), *w = static_cast<const T*>(l.w);
    const int K = (int)l.K;
    if (l.M <= 8) {
      if (aligned) k_few_rows<T, 1, ACT, true><<<grid, 256, 0, st>>>(x, l.ldx, w, l.ldw, ep, K);
      else k_few_rows<T, 1, ACT, false><<<grid, 256, 0, st>>>(x, l.ldx, w, l.ldw, ep, K);
    } else {
      if (aligned) k_few_rows<T, 2, ACT, true><<<grid, 256, 0, st>>>(x, l.ldx, w, l.ldw, ep, K);
      else k_few_rows<T, 2, ACT, false><<<grid, 256, 0, st>>>(x, l.ldx, w, l.ldw, ep, K);
    }
    return check_launch(fn);
  }
  Space ws = {static_cast<char*>(l.workspace), static_cast<char*>(l.workspace) + l.workspace_bytes};
  Matrix a = {l.x, l.M, l.K, l.ldx}, b = {l.w, l.N, l.K, l.ldw};
  const int r = for_tma<T>(fn, &a, &b, ws, st);
  return r != MHC_OK ? r : gemm<T, false, false, ACT>(fn, a, b, ep, l.K, st);
}

template <typename T, int ACT>
int backward(const LinearGradArg& l, cudaStream_t st) {
  const char* fn = "mhc_linear_bwd";
  Space ws = {static_cast<char*>(l.workspace), static_cast<char*>(l.workspace) + l.workspace_bytes};
  Matrix dz = {l.dy, l.M, l.N, l.ldy};
  const bool products = l.dx || l.dw;
  const bool own = products && (ACT != kNone || !tma_rows(l.dy, l.ldy));
  if (own || l.dbias) {
    void* q = nullptr;
    if (own) {
      q = ws.take(padded_bytes(l.M, l.N));
      if (!q) return no_space(fn);
    }
    const int per = rows_per(l.M, l.N);
    const int64_t parts = (l.M + per - 1) / per;
    float* part = nullptr;
    if (l.dbias) {
      part = static_cast<float*>(ws.take((size_t)parts * (size_t)l.N * sizeof(float)));
      if (!part) return no_space(fn);
    }
    const dim3 grid((unsigned)((l.N + 255) / 256), (unsigned)parts);
    k_act_grad<T, ACT><<<grid, 256, 0, st>>>(static_cast<const T*>(l.dy), l.ldy, static_cast<const float*>(l.z),
                                             l.ldz, static_cast<T*>(q), up8(l.N), part, l.M, (int)l.N, per,
                                             tma_rows(l.dy, l.ldy));
    int r = check_launch(fn);
    if (r != MHC_OK) return r;
    if (part) {
      k_bias_sum<T><<<(unsigned)((l.N + 255) / 256), 256, 0, st>>>(part, (int)parts, (int)l.N,
                                                                   static_cast<T*>(l.dbias));
      r = check_launch(fn);
      if (r != MHC_OK) return r;
    }
    if (own) dz = {q, l.M, l.N, up8(l.N)};
  }
  Matrix w = {l.w, l.N, l.K, l.ldw}, x = {l.x, l.M, l.K, l.ldx};
  int r = for_tma<T>(fn, l.dx ? &w : nullptr, l.dw ? &x : nullptr, ws, st);
  if (r == MHC_OK && l.dx)  // dx[m, k] = sum_n dz[m, n] W[n, k]
    r = gemm<T, false, true, kNone>(fn, dz, w, epilogue<T>(l.dx, l.lddx, l.M, l.K), l.N, st);
  if (r == MHC_OK && l.dw)  // dW[n, k] = sum_m dz[m, n] x[m, k]
    r = gemm<T, true, true, kNone>(fn, dz, x, epilogue<T>(l.dw, l.lddw, l.N, l.K), l.M, st);
  return r;
}

#define MHC_BY_ACT(F, T, l, st)                 \
  switch ((l).act) {                            \
    case kNone: return F<T, kNone>(l, st);      \
    case kRelu: return F<T, kRelu>(l, st);      \
    case kSilu: return F<T, kSilu>(l, st);      \
    default: return F<T, kGelu>(l, st);         \
  }

}  // namespace

size_t linear_fwd_ws_bytes(const void* x, int64_t ldx, const void* w, int64_t ldw, int64_t M,
                           int64_t N, int64_t K) {
  if (M <= kFewRows) return 0;
  return (tma_rows(x, ldx) ? 0 : padded_bytes(M, K)) + (tma_rows(w, ldw) ? 0 : padded_bytes(N, K));
}
size_t linear_bwd_ws_bytes(const LinearGradArg& l) {
  size_t n = 0;
  if ((l.dx || l.dw) && (l.act != kNone || !tma_rows(l.dy, l.ldy))) n += padded_bytes(l.M, l.N);
  if (l.dbias) {
    const int per = rows_per(l.M, l.N);
    n += up256((size_t)((l.M + per - 1) / per) * (size_t)l.N * sizeof(float));
  }
  if (l.dx && !tma_rows(l.w, l.ldw)) n += padded_bytes(l.N, l.K);
  if (l.dw && !tma_rows(l.x, l.ldx)) n += padded_bytes(l.M, l.K);
  return n;
}
int launch_linear_fwd(const LinearArg& l, cudaStream_t st) {
  if (l.dtype == MHC_BF16) { MHC_BY_ACT(forward, bf16, l, st) }
  MHC_BY_ACT(forward, f16, l, st)
}
int launch_linear_bwd(const LinearGradArg& l, cudaStream_t st) {
  if (l.dtype == MHC_BF16) { MHC_BY_ACT(backward, bf16, l, st) }
  MHC_BY_ACT(backward, f16, l, st)
}

}  // namespace mhc
