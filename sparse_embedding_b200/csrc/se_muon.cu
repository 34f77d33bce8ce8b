// The Muon update of dense matrices: momentum, the orthogonalisation of the
// update by Newton-Schulz products, and the step of the weights. It has no
// counterpart in the reference, whose optimizers work on embedding rows.
//
// For an update U (m x n; taken as its transpose where m > n, so that s <= w
// are its sides), X_0 = U / (|U|_F + eps) and, a given number of times,
//   A = X X^T,   X <- a X + (b A + c A A) X
// with (a, b, c) = (3.4445, -4.7750, 2.0315), which drives every singular
// value of X into about [0.68, 1.2].
//
// Number formats. The products run on the tensor cores with f16 operands and
// fp32 sums. Every matrix is kept S = 2^13 times its value: entries of X and A
// are at most 1.25^2, those of B = b A + c A A at most 2.9, so S of each fits
// f16 (65,504) and values down to 2^-27 of the largest keep all 11 bits.
//  * X is a pair hi + lo of f16 (22 bits). Rounding X itself to 11 bits would
//    add noise to every direction, which the iteration amplifies like the small
//    singular values (a^5 = 485 times); the pair enters a X in the epilogue,
//    so it costs no matrix instruction.
//  * The diagonals of A and of B are kept apart in fp32, and the matrices hold
//    zeros there: near the end A is close to the identity, and its rounding
//    would be the largest error left. With A = D + O:  A A = O O + D O + O D + D D.
//  * bf16 outputs: products of the hi parts alone. fp32 and f16 outputs:
//    hi hi + hi lo + lo hi, three times the matrix work, for errors of fp32's order.
// Against 64 bits, for the matrices of the tests: 0.1 % at most from the single
// products (below bf16's own 0.17 % rounding), about 2e-6 from the triple ones.
//
// A and A A are symmetric: only tiles that touch the lower triangle are
// computed, and an element below the diagonal is written to both places by the
// thread that holds it.

#include <algorithm>
#include <cstring>

#include "se_dense.hpp"
#include "se_tcgen05.cuh"

namespace se_gpu {

namespace {

constexpr float kNsA = 3.4445f, kNsB = -4.7750f, kNsC = 2.0315f;
constexpr float kScale = 8192.0f;  // S
constexpr int kTileK = 64;         // k-values of a stage: one 128-byte swizzle row

// ---------------------------------------------------------------------------
// Momentum, norm, and the scaled update X_0
// ---------------------------------------------------------------------------

struct Strided {  // a batch of matrices with contiguous rows
  const void *p;
  int64_t batch, row;
};

constexpr int kNormParts = 128;  // blocks (and partial sums) per matrix, at most

// Element (i, j) of matrix z as fp32, for a type given at run time.
__device__ __forceinline__ float strided_at(const Strided &s, int type, int64_t z, int64_t i, int64_t j) {
  const int64_t at = z * s.batch + i * s.row + j;
  if (type == SE_FLOAT32) return static_cast<const float *>(s.p)[at];
  if (type == SE_FLOAT16) return __half2float(static_cast<const __half *>(s.p)[at]);
  return __bfloat162float(static_cast<const __nv_bfloat16 *>(s.p)[at]);
}

struct UpdateArgs {
  Strided grad;      // the update itself (orthogonalize), or the gradient
  int grad_type;
  Strided momentum;  // fp32; p null: the update is grad
  float beta;
  int nesterov;
  int64_t m, n;
};

// U from the gradient and the momentum after its update.
__device__ __forceinline__ float update_of(const UpdateArgs &a, float g, float mom) {
  return a.nesterov ? __fmaf_rn(a.beta, mom, g) : mom;
}

// M <- beta M + G, and this block's part of |U|^2 (fp64: squares of fp32
// values neither overflow nor vanish there).
__global__ void __launch_bounds__(256)
k_muon_momentum(UpdateArgs a, double *__restrict__ parts) {
  __shared__ double red[8];
  const int64_t z = blockIdx.y, count = a.m * a.n;
  double sum = 0.0;
  for (int64_t e = int64_t(blockIdx.x) * blockDim.x + threadIdx.x; e < count; e += int64_t(gridDim.x) * blockDim.x) {
    const int64_t i = e / a.n, j = e - i * a.n;
    float u = strided_at(a.grad, a.grad_type, z, i, j);
    if (a.momentum.p) {
      float *mp = const_cast<float *>(static_cast<const float *>(a.momentum.p)) + z * a.momentum.batch + i * a.momentum.row + j;
      const float mom = __fmaf_rn(a.beta, *mp, u);
      *mp = mom;
      u = update_of(a, u, mom);
    }
    sum += double(u) * double(u);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    sum = 0.0;
#pragma unroll
    for (int i = 0; i < 8; ++i) sum += red[i];
    parts[z * kNormParts + blockIdx.x] = sum;
  }
}

// X_0 = S U / (|U| + eps) as hi + lo, s x w (transposed where m > n): 32 x 32
// tiles through shared memory, so that both sides are read and written by rows.
__global__ void __launch_bounds__(256)
k_muon_scale(UpdateArgs a, const double *__restrict__ parts, int nparts, float eps, bool transposed,
             __half *__restrict__ hi, __half *__restrict__ lo, int64_t ld, int64_t batch_stride) {
  __shared__ float tile[32][33];
  __shared__ double factor;  // fp64: 1 / |U| of a tiny update passes fp32's range
  const int64_t z = blockIdx.z;
  pdl_wait();
  if (threadIdx.x < 32) {
    double sum = 0.0;
    for (int k = threadIdx.x; k < nparts; k += 32) sum += parts[z * kNormParts + k];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (threadIdx.x == 0) factor = double(kScale) / (sqrt(sum) + double(eps));
  }
  __syncthreads();
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const int64_t tiles_j = (a.n + 31) / 32, tiles = tiles_j * ((a.m + 31) / 32);
  for (int64_t t = blockIdx.x; t < tiles; t += gridDim.x) {
    const int64_t i0 = t / tiles_j * 32, j0 = (t - t / tiles_j * tiles_j) * 32;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int64_t i = i0 + ty + 8 * k, j = j0 + tx;
      if (i < a.m && j < a.n) {
        float u = strided_at(a.grad, a.grad_type, z, i, j);
        if (a.momentum.p)
          u = update_of(a, u, static_cast<const float *>(a.momentum.p)[z * a.momentum.batch + i * a.momentum.row + j]);
        tile[ty + 8 * k][tx] = float(double(u) * factor);
      }
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int64_t r = (transposed ? j0 : i0) + ty + 8 * k, c = (transposed ? i0 : j0) + tx;
      if (r < (transposed ? a.n : a.m) && c < (transposed ? a.m : a.n)) {
        const float v = transposed ? tile[tx][ty + 8 * k] : tile[ty + 8 * k][tx];
        const __half h = __float2half_rn(v);
        const int64_t at = z * batch_stride + r * ld + c;
        hi[at] = h;
        lo[at] = __float2half_rn(v - __half2float(h));
      }
    }
    __syncthreads();
  }
}

// ---------------------------------------------------------------------------
// The products
// ---------------------------------------------------------------------------

enum Product {
  kGram,    // A = X X^T
  kSquare,  // B = b A + c A A
  kApply,   // X' = a X + B X
  kFinish,  // the last X', as the call's result
};

struct Pair {  // a matrix as hi + lo
  __half *hi, *lo;
  int64_t ld, batch;
};

// What the last product does with O = X'.
struct FinishArgs {
  void *out;  // O itself, or the weights W <- keep W - rate O
  int type, update, transposed;
  int64_t row, batch;
  float keep, rate;
};

struct ProductArgs {
  CUtensorMap a_hi, a_lo, b_hi, b_lo;  // the operands
  int rows, cols, kblocks, batch;
  int tiles_i, tiles_j, tiles;         // of one matrix
  Pair in;                             // kSquare: A, kApply and kFinish: X
  Pair out;
  const float *diag_in;                // kSquare: A's diagonal, kApply and kFinish: B's
  float *diag_out;                     // kGram: A's (scaled by S), kSquare: B's (not scaled)
  FinishArgs fin;
  uint32_t *status;
};

constexpr int kEpilogueWarps = 8;
constexpr int kFlush = 4;  // k-blocks of a SPLIT accumulation between two flushes

template <int CG, int BN>
struct Layout {
  static constexpr int kA = 128 * 128;             // bytes of a CTA's A tile: 128 rows of 64 values
  static constexpr int kB = (BN / CG) * 128;       // and of its part of the B tile
  static constexpr int kStage = kA + kB;
  static constexpr int kStages = CG == 2 ? 6 : BN == 256 ? 4 : BN == 128 ? 6 : 8;
  static constexpr int kStaging = 32 * 33;         // floats of an epilogue warp's staging tile
  static constexpr int kBytes = kStages * kStage + kEpilogueWarps * kStaging * 4 + 1024;  // 1,024: tile alignment
};

// Tile t: matrix, first row, first column. The symmetric products list only
// tiles that reach the lower triangle, row of tiles by row of tiles.
template <int MODE, int TM, int BN>
__device__ __forceinline__ void tile_at(const ProductArgs &g, int t, int &z, int &row, int &col) {
  z = t / g.tiles;
  t -= z * g.tiles;
  if constexpr (MODE == kGram || MODE == kSquare) {
    int i = 0;
    for (;; ++i) {
      const int in_row = min((i * TM + TM - 1) / BN + 1, g.tiles_j);
      if (t < in_row) break;
      t -= in_row;
    }
    row = i * TM;
    col = t * BN;
  } else {
    const int i = t / g.tiles_j;
    row = i * TM;
    col = (t - i * g.tiles_j) * BN;
  }
}

__device__ __forceinline__ __half2 half2_at(const __half *p, int64_t at) {
  return *reinterpret_cast<const __half2 *>(p + at);
}
__device__ __forceinline__ void put_half2(const Pair &p, int64_t at, float f0, float f1, bool split) {
  const __half2 h = __floats2half2_rn(f0, f1);
  *reinterpret_cast<__half2 *>(p.hi + at) = h;
  if (split) {
    const float2 b = __half22float2(h);
    *reinterpret_cast<__half2 *>(p.lo + at) = __floats2half2_rn(f0 - b.x, f1 - b.y);
  }
}
__device__ __forceinline__ float load_typed(const void *p, int type, int64_t at) {
  if (type == SE_FLOAT32) return static_cast<const float *>(p)[at];
  if (type == SE_FLOAT16) return __half2float(static_cast<const __half *>(p)[at]);
  return __bfloat162float(static_cast<const __nv_bfloat16 *>(p)[at]);
}
__device__ __forceinline__ void store_typed(void *p, int type, int64_t at, float v) {
  if (type == SE_FLOAT32) static_cast<float *>(p)[at] = v;
  else if (type == SE_FLOAT16) static_cast<__half *>(p)[at] = __float2half_rn(v);
  else static_cast<__nv_bfloat16 *>(p)[at] = __float2bfloat16_rn(v);
}

// The epilogue of a 32 x 32 block of the accumulator, staged by the warp in
// `tile` (row stride 33). Everything else of the block is read and written two
// rows at a time, 16 lanes of two values each, so that global accesses are
// whole 32-byte sectors and shared-memory ones free of conflicts. All loads
// of a block are issued before its first store. Rows are r0 .. r0 + 31,
// columns c0 .. c0 + 31, both multiples of 32; storage reaches past the last
// column to a multiple of 64, so columns need no guard.
template <int MODE, bool SPLIT>
__device__ __forceinline__ void finish_block(const ProductArgs &g, float *tile, int z, int r0, int c0, float dr_lane) {
  const int lane = int(threadIdx.x) & 31, up = lane >> 4, pair = (lane & 15) * 2;
  constexpr bool kReadsIn = MODE != kGram, kInLo = MODE == kApply || MODE == kFinish || SPLIT;
  constexpr int kAtOnce = SPLIT ? 8 : 16;  // loads in flight; SPLIT needs registers for its sums
  __half2 xh[kReadsIn ? kAtOnce : 1], xl[kReadsIn && kInLo ? kAtOnce : 1];
  auto load = [&](int i0) {
    if constexpr (kReadsIn) {
#pragma unroll
      for (int i = 0; i < kAtOnce; ++i) {
        const int r = r0 + 2 * (i0 + i) + up;
        const int64_t at = int64_t(z) * g.in.batch + int64_t(r) * g.in.ld + c0 + pair;
        const bool in = r < g.rows;
        xh[i] = in ? half2_at(g.in.hi, at) : __half2();
        if constexpr (kInLo) xl[i] = in ? half2_at(g.in.lo, at) : __half2();
      }
    }
  };
  if constexpr (MODE == kGram || MODE == kSquare) {
    const bool diagonal = r0 == c0;
    float dc0 = 0.0f, dc1 = 0.0f;
    if constexpr (MODE == kSquare) {
      const float *d = g.diag_in + int64_t(z) * g.rows;
      dc0 = c0 + pair < g.cols ? d[c0 + pair] : 0.0f;
      dc1 = c0 + pair + 1 < g.cols ? d[c0 + pair + 1] : 0.0f;
    }
#pragma unroll 1
    for (int i0 = 0; i0 < 16; i0 += kAtOnce) {
    load(i0);
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      const int rr = 2 * (i0 + i) + up, r = r0 + rr;
      // a diagonal block takes its lower triangle on both sides
      const bool swap0 = diagonal && pair > rr, swap1 = diagonal && pair + 1 > rr;
      float f0 = tile[swap0 ? pair * 33 + rr : rr * 33 + pair];
      float f1 = tile[swap1 ? (pair + 1) * 33 + rr : rr * 33 + pair + 1];
      const bool d0 = diagonal && pair == rr, d1 = diagonal && pair + 1 == rr;
      if constexpr (MODE == kGram) {
        f0 *= 1.0f / kScale;
        f1 *= 1.0f / kScale;
      } else {
        const float dr = __shfl_sync(0xffffffffu, dr_lane, rr);
        float2 x = __half22float2(xh[i]);
        if constexpr (SPLIT) {
          const float2 l = __half22float2(xl[i]);
          x.x += l.x;
          x.y += l.y;
        }
        // off the diagonal (A A)_rc = acc + (D_r + D_c) O_rc, on it acc + D_r^2
        const float a0 = d0 ? dr : x.x, a1 = d1 ? dr : x.y;
        f0 = __fmaf_rn(kNsC / kScale, __fmaf_rn(d0 ? dr : dr + dc0, a0, f0), kNsB * a0);
        f1 = __fmaf_rn(kNsC / kScale, __fmaf_rn(d1 ? dr : dr + dc1, a1, f1), kNsB * a1);
      }
      if (d0 || d1) {
        if (r < g.rows) g.diag_out[int64_t(z) * g.rows + r] = (d0 ? f0 : f1) * (MODE == kSquare ? 1.0f / kScale : 1.0f);
        if (d0) f0 = 0.0f;
        else f1 = 0.0f;
      }
      if (r < g.rows) put_half2(g.out, int64_t(z) * g.out.batch + int64_t(r) * g.out.ld + c0 + pair, f0, f1, SPLIT);
      if (!diagonal) {
        tile[rr * 33 + pair] = f0;
        tile[rr * 33 + pair + 1] = f1;
      }
    }
    }
    if (!diagonal) {  // the mirror: rows c0 .., columns r0 ..
      __syncwarp();
#pragma unroll 4
      for (int i = 0; i < 16; ++i) {
        const int cc = 2 * i + up;
        put_half2(g.out, int64_t(z) * g.out.batch + int64_t(c0 + cc) * g.out.ld + r0 + pair, tile[pair * 33 + cc],
                  tile[(pair + 1) * 33 + cc], SPLIT);
      }
    }
  } else {
#pragma unroll 1
    for (int i0 = 0; i0 < 16; i0 += kAtOnce) {
    load(i0);
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      const int rr = 2 * (i0 + i) + up, r = r0 + rr;
      const float f = kNsA + __shfl_sync(0xffffffffu, dr_lane, rr);
      const float2 h = __half22float2(xh[i]), l = __half22float2(xl[i]);
      const float f0 = __fmaf_rn(f, h.x + l.x, tile[rr * 33 + pair] * (1.0f / kScale));
      const float f1 = __fmaf_rn(f, h.y + l.y, tile[rr * 33 + pair + 1] * (1.0f / kScale));
      if constexpr (MODE == kApply) {
        if (r < g.rows) put_half2(g.out, int64_t(z) * g.out.batch + int64_t(r) * g.out.ld + c0 + pair, f0, f1, true);
      } else {
        tile[rr * 33 + pair] = f0;
        tile[rr * 33 + pair + 1] = f1;
      }
    }
    }
    if constexpr (MODE == kFinish) {
      // by rows of the result, whichever way it lies: lane = its column
      __syncwarp();
      const FinishArgs &f = g.fin;
      const int across = f.transposed ? r0 : c0, along = f.transposed ? c0 : r0;
      const bool in = across + lane < (f.transposed ? g.rows : g.cols);
      const int most = min(32, (f.transposed ? g.cols : g.rows) - along);
      const int64_t base = int64_t(z) * f.batch + int64_t(along) * f.row + across + lane;
#pragma unroll 1
      for (int e0 = 0; e0 < most; e0 += 8) {
        float w[8];
        if (f.update) {
#pragma unroll
          for (int e = 0; e < 8; ++e) w[e] = in && e0 + e < most ? load_typed(f.out, f.type, base + (e0 + e) * f.row) : 0.0f;
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          float o = tile[f.transposed ? lane * 33 + e0 + e : (e0 + e) * 33 + lane] * (1.0f / kScale);
          if (f.update) o = __fmaf_rn(-f.rate, o, f.keep * w[e]);
          if (in && e0 + e < most) store_typed(f.out, f.type, base + (e0 + e) * f.row, o);
        }
      }
    }
  }
}

// One product over persistent tiles of (128 CG) x BN. Warp 0 loads operand
// stages by TMA, warp 1 issues the matrix instructions, warps 4-11 turn finished
// accumulators into the result while the next tile is computed (two
// accumulators of BN columns in tensor memory; each epilogue warp has 32 rows
// and every second block of 32 columns). Bound by the tensor cores for large
// sides (each stage is 4 instructions of M x BN x 16).
//
// SPLIT: the three products of hi and lo parts. The tensor core cuts its fp32
// sums off instead of rounding them, which over thousands of k-values costs
// more than the lo parts bring (measured: 3e-5 at 4,096), so a sum runs over
// kFlush k-blocks only and the epilogue warps add those up in registers.
template <int MODE, int CG, int BN, bool SPLIT>
__global__ void __launch_bounds__(128 + 32 * kEpilogueWarps, 1) k_ns_product(const __grid_constant__ ProductArgs g) {
  using L = Layout<CG, BN>;
  constexpr int kStages = L::kStages, kTM = 128 * CG, kBlocks = BN / 64;  // kBlocks: column blocks of an epilogue warp
  constexpr bool kBMN = MODE == kApply || MODE == kFinish;                // B operand is X itself: n-contiguous
  extern __shared__ uint8_t raw[];
  __shared__ uint64_t full[kStages], empty[kStages], acc_full[2], acc_empty[2], drained;
  __shared__ uint32_t tmem_base;
  __shared__ volatile uint32_t given_up;
  uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = CG == 2 ? cluster_rank() : 0u;
  const int unit = int(blockIdx.x) / CG, units = int(gridDim.x) / CG;
  const int total = g.tiles * g.batch;
  const int kb = g.kblocks * (SPLIT ? 3 : 1);
  const int per_sum = SPLIT ? kFlush : kb, sums = (kb + per_sum - 1) / per_sum;

  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&acc_full[i], 1);
      mbar_init(&acc_empty[i], kEpilogueWarps * CG);
    }
    mbar_init(&drained, 1);
    given_up = 0u;
    prefetch_map(&g.a_hi);
    prefetch_map(&g.b_hi);
  }
  if (warp == 2) tmem_alloc<CG>(&tmem_base, 2 * BN);
  tmem_fence_before();
  __syncthreads();
  if constexpr (CG == 2) cluster_sync_all();
  tmem_fence_after();
  const uint32_t tmem = tmem_base;
  pdl_trigger();
  pdl_wait();

  uint32_t issued = 0;  // stages loaded (warp 0)
  if (warp == 0) {
    if (elect_one()) {
      bool go = true;
      for (int t = unit; go && t < total; t += units) {
        int z, row, col;
        tile_at<MODE, kTM, BN>(g, t, z, row, col);
        row += int(rank) * 128;
        col += int(rank) * (BN / CG);
        for (int k = 0; k < kb; ++k) {
          const uint32_t st = issued % kStages, use = issued / kStages;
          if (!wait_or_give_up(&empty[st], (use & 1u) ^ 1u, &given_up)) {
            go = false;
            break;
          }
          // hi lo, lo hi, hi hi
          const int seg = SPLIT ? k / g.kblocks : 2, k0 = (SPLIT ? k - seg * g.kblocks : k) * kTileK;
          const CUtensorMap *ma = seg == 1 ? &g.a_lo : &g.a_hi, *mb = seg == 0 ? &g.b_lo : &g.b_hi;
          uint8_t *a = smem + st * L::kStage, *b = a + L::kA;
          uint32_t bar = smem_u32(&full[st]);
          if constexpr (CG == 2) bar = mapa(bar, 0);
          if (rank == 0) mbar_arrive_expect_tx(&full[st], CG * L::kStage);
          tma_load<CG>(a, ma, k0, row, z, bar);
          if constexpr (kBMN) {
#pragma unroll
            for (int q = 0; q < BN / CG / 64; ++q) tma_load<CG>(b + q * 8192, mb, col + q * 64, k0, z, bar);
          } else {
            tma_load<CG>(b, mb, k0, col, z, bar);
          }
          ++issued;
        }
      }
      // the stages' last uses: no arrival is outstanding when the CTA ends
      for (uint32_t i = issued > kStages ? issued - kStages : 0; go && i < issued; ++i)
        go = wait_or_give_up(&empty[i % kStages], (i / kStages) & 1u, &given_up);
    }
  } else if (warp == 1 && rank == 0) {
    if (elect_one()) {
      constexpr uint32_t kDesc = mma_desc(kTM, BN, kBMN);
      uint32_t used = 0, filled = 0;
      bool go = true;
      for (int t = unit; go && t < total; t += units) {
        for (int k = 0; go && k < kb; ++filled) {
          const uint32_t acc = filled & 1u;
          if (!wait_or_give_up(&acc_empty[acc], ((filled >> 1) & 1u) ^ 1u, &given_up)) {
            go = false;
            break;
          }
          tmem_fence_after();
          const int first = k, last = min(kb, k + per_sum);
          for (; k < last; ++k, ++used) {
            const uint32_t st = used % kStages;
            if (!wait_or_give_up(&full[st], (used / kStages) & 1u, &given_up)) {
              go = false;
              break;
            }
            tmem_fence_after();
            const uint32_t a = smem_u32(smem + st * L::kStage), b = a + L::kA;
            const uint64_t da = operand_desc(a, 16), db = operand_desc(b, kBMN ? 8192 : 16);
#pragma unroll
            for (int q = 0; q < kTileK / 16; ++q)  // 16 k-values: 32 bytes along a K-major row, 16 rows when MN-major
              mma_f16<CG>(tmem + acc * BN, da + q * (32 >> 4), db + q * ((kBMN ? 2048 : 32) >> 4), kDesc,
                          k > first || q > 0);
            mma_commit<CG>(&empty[st]);
          }
          if (go) mma_commit<CG>(&acc_full[acc]);
        }
      }
    }
  } else if (warp >= 4) {
    const int quad = warp & 3, side = (warp - 4) >> 2;
    float *tile = reinterpret_cast<float *>(smem + kStages * L::kStage) + (warp - 4) * L::kStaging;
    uint32_t filled = 0;
    bool go = true;
    for (int t = unit; t < total; t += units) {
      int z, row, col;
      tile_at<MODE, kTM, BN>(g, t, z, row, col);
      const int r0 = row + int(rank) * 128 + quad * 32;
      float dr = 0.0f;
      if (MODE != kGram && r0 + lane < g.rows) dr = g.diag_in[int64_t(z) * g.rows + r0 + lane];
      auto block = [&](int b) { return col + (2 * b + side) * 32; };
      auto wanted = [&](int c0) {
        return r0 < g.rows && c0 < g.cols && (MODE == kApply || MODE == kFinish || c0 <= r0);
      };
      auto address = [&](uint32_t acc, int b) {
        return tmem + acc * BN + uint32_t((2 * b + side) * 32) + (uint32_t(quad * 32) << 16);
      };
      auto stage = [&](const float (&v)[32]) {
        __syncwarp();
#pragma unroll
        for (int e = 0; e < 32; ++e) tile[lane * 33 + e] = v[e];
        __syncwarp();
      };
      auto take = [&](uint32_t acc) {  // an accumulator is full; false: gave up
        const bool ok = wait_or_give_up(&acc_full[acc], (filled >> 1) & 1u, &given_up);
        go = __all_sync(0xffffffffu, ok);
        tmem_fence_after();
        return go;
      };
      auto give = [&](uint32_t acc) {
        tmem_fence_before();
        __syncwarp();
        if (lane == 0) {
          uint32_t bar = smem_u32(&acc_empty[acc]);
          if constexpr (CG == 2) bar = mapa(bar, 0);
          mbar_arrive_cluster(bar);
        }
        ++filled;
      };
      if constexpr (SPLIT) {
        float v[kBlocks][32];
        for (int s = 0; s < sums; ++s) {
          const uint32_t acc = filled & 1u;
          if (!take(acc)) break;
#pragma unroll
          for (int b = 0; b < kBlocks; ++b) {
            float f[32];
            tmem_load32(address(acc, b), f);
#pragma unroll
            for (int e = 0; e < 32; ++e) v[b][e] = s == 0 ? f[e] : v[b][e] + f[e];
          }
          give(acc);
        }
        if (!go) break;
#pragma unroll
        for (int b = 0; b < kBlocks; ++b) {
          if (!wanted(block(b))) continue;
          stage(v[b]);
          finish_block<MODE, SPLIT>(g, tile, z, r0, block(b), dr);
        }
      } else {
        const uint32_t acc = filled & 1u;
        if (!take(acc)) break;
#pragma unroll 1
        for (int b = 0; b < kBlocks; ++b) {
          if (!wanted(block(b))) break;
          float v[32];
          __syncwarp();
          tmem_load32(address(acc, b), v);
          stage(v);
          finish_block<MODE, SPLIT>(g, tile, z, r0, block(b), dr);
        }
        give(acc);
      }
    }
  }

  __syncwarp();
  if (given_up) {
    // Leave nothing in flight: the loads that warp 0 issued and the matrix
    // instructions of warp 1; then report.
    if (warp == 1 && rank == 0 && elect_one()) {
      mma_commit<CG>(&drained);
      wait_for(&drained, 0u, nullptr);
    }
    if (warp == 0 && rank == 0) {
      const uint32_t last = __reduce_max_sync(0xffffffffu, issued);
      for (uint32_t i = last > kStages ? last - kStages : 0; i < last; ++i)
        wait_for(&full[i % kStages], (i / kStages) & 1u, nullptr);
    }
    if (threadIdx.x == 0) {
      *reinterpret_cast<volatile uint32_t *>(g.status) = 1u;
      __threadfence_system();
    }
  }
  tmem_fence_before();
  __syncthreads();
  if constexpr (CG == 2) cluster_sync_all();
  if (warp == 2) tmem_free<CG>(tmem, 2 * BN);
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------

// A word in host memory that a product sets when a wait gave up; the next call
// on the device reads it without waiting for the GPU.
uint32_t *ns_status(int device) {
  static std::mutex mu;
  static std::map<int, uint32_t *> known;
  std::lock_guard<std::mutex> lock(mu);
  auto it = known.find(device);
  if (it != known.end()) return it->second;
  // an allocation is allowed while another stream, or this one, is being captured
  cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
  cuda_check(cudaThreadExchangeStreamCaptureMode(&mode), "cudaThreadExchangeStreamCaptureMode");
  void *p = nullptr;
  const cudaError_t e = cudaHostAlloc(&p, sizeof(uint32_t), cudaHostAllocMapped | cudaHostAllocPortable);
  cudaThreadExchangeStreamCaptureMode(&mode);
  cuda_check(e, "cudaHostAlloc");
  *static_cast<volatile uint32_t *>(p) = 0u;
  return known[device] = static_cast<uint32_t *>(p);
}

using EncodeTiled = decltype(&cuTensorMapEncodeTiled);
EncodeTiled encode_tiled() {
  static EncodeTiled fn = [] {
    void *p = nullptr;
    cudaDriverEntryPointQueryResult found{};
    cuda_check(cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &found),
               "cudaGetDriverEntryPointByVersion");
    if (p == nullptr || found != cudaDriverEntryPointSuccess)
      throw Error(SE_ERR_CUDA, "the driver has no cuTensorMapEncodeTiled");
    return reinterpret_cast<EncodeTiled>(p);
  }();
  return fn;
}

// Boxes of 64 columns x `box` rows of a batch of rows x cols f16 matrices.
CUtensorMap matrix_map(const __half *p, int64_t rows, int64_t cols, int64_t ld, int64_t batch, int box) {
  CUtensorMap map;
  const cuuint64_t dims[3] = {cuuint64_t(cols), cuuint64_t(rows), cuuint64_t(batch)};
  const cuuint64_t strides[2] = {cuuint64_t(ld) * 2, cuuint64_t(ld) * 2 * cuuint64_t(rows)};
  const cuuint32_t boxes[3] = {64, cuuint32_t(box), 1}, steps[3] = {1, 1, 1};
  const CUresult r = encode_tiled()(&map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<__half *>(p), dims, strides,
                                    boxes, steps, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                                    CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) throw Error(SE_ERR_CUDA, "cuTensorMapEncodeTiled: error " + std::to_string(int(r)));
  return map;
}

// The workspace of a call: X twice (a product reads one and writes the other),
// A, B, their diagonals, and the partial norms.
struct Space {
  double *parts;
  Pair x[2], a, b;
  float *diag_a, *diag_b;
  size_t bytes;
};

Space muon_space(void *base, int64_t batch, int64_t s, int64_t w, bool split) {
  Space sp{};
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t here = at;
    at += (bytes + 255) & ~size_t(255);
    return static_cast<uint8_t *>(base) + here;
  };
  const int64_t ldx = (w + 63) / 64 * 64, lda = (s + 63) / 64 * 64;
  auto pair = [&](int64_t ld, bool lo) {
    Pair p{};
    p.ld = ld;
    p.batch = s * ld;
    p.hi = reinterpret_cast<__half *>(take(size_t(batch) * s * ld * 2));
    p.lo = lo ? reinterpret_cast<__half *>(take(size_t(batch) * s * ld * 2)) : p.hi;
    return p;
  };
  sp.parts = reinterpret_cast<double *>(take(size_t(batch) * kNormParts * sizeof(double)));
  sp.x[0] = pair(ldx, true);
  sp.x[1] = pair(ldx, true);
  sp.a = pair(lda, split);
  sp.b = pair(lda, split);
  sp.diag_a = reinterpret_cast<float *>(take(size_t(batch) * s * sizeof(float)));
  sp.diag_b = reinterpret_cast<float *>(take(size_t(batch) * s * sizeof(float)));
  sp.bytes = at;
  return sp;
}

bool split_products(int32_t out_type) { return out_type != SE_BFLOAT16; }

template <int MODE, int CG, int BN, bool SPLIT>
void launch_product(ProductArgs &g, int sms, cudaStream_t st) {
  using L = Layout<CG, BN>;
  auto *kernel = k_ns_product<MODE, CG, BN, SPLIT>;
  allow_dynamic_smem(kernel, L::kBytes);
  const int64_t units = std::min<int64_t>(int64_t(g.tiles) * g.batch, sms / CG);
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(unsigned(units * CG));
  cfg.blockDim = dim3(128 + 32 * kEpilogueWarps);
  cfg.dynamicSmemBytes = L::kBytes;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = CG;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = CG == 2 ? 2 : 1;
  cuda_check(cudaLaunchKernelEx(&cfg, kernel, g), "k_ns_product");
  launched("k_ns_product");
}

int64_t product_tiles(bool symmetric, int64_t rows, int64_t cols, int tm, int bn, int64_t &ti, int64_t &tj) {
  ti = (rows + tm - 1) / tm;
  tj = (cols + bn - 1) / bn;
  if (!symmetric) return ti * tj;
  int64_t n = 0;
  for (int64_t i = 0; i < ti; ++i) n += std::min<int64_t>((i * tm + tm - 1) / bn + 1, tj);
  return n;
}

// One product of `op_a` (rows x depth) and `op_b` (K-major: cols x depth;
// for X itself depth x cols).
template <int MODE>
void product(ProductArgs &g, const Pair &op_a, const Pair &op_b, int64_t rows, int64_t cols, int64_t depth,
             int64_t batch, bool split, int sms, cudaStream_t st) {
  constexpr bool kSym = MODE == kGram || MODE == kSquare, kBMN = !kSym;
  g.rows = int(rows);
  g.cols = int(cols);
  g.kblocks = int((depth + kTileK - 1) / kTileK);
  g.batch = int(batch);
  int64_t ti = 0, tj = 0;
  auto go = [&](auto cg, auto bn, auto sp) {
    constexpr int CG = decltype(cg)::value, BN = decltype(bn)::value;
    constexpr bool kSplit = decltype(sp)::value;
    const int64_t tiles = product_tiles(kSym, rows, cols, 128 * CG, BN, ti, tj);
    if (tiles * batch > 0x7fffffff) throw std::invalid_argument("batch x m x n is too large");
    g.tiles_i = int(ti);
    g.tiles_j = int(tj);
    g.tiles = int(tiles);
    const int box_b = kBMN ? 64 : BN / CG;
    auto map_b = [&](const __half *p) {
      return kBMN ? matrix_map(p, depth, cols, op_b.ld, batch, box_b) : matrix_map(p, cols, depth, op_b.ld, batch, box_b);
    };
    g.a_hi = matrix_map(op_a.hi, rows, depth, op_a.ld, batch, 128);
    g.b_hi = map_b(op_b.hi);
    if (kSplit) {
      g.a_lo = matrix_map(op_a.lo, rows, depth, op_a.ld, batch, 128);
      g.b_lo = map_b(op_b.lo);
    }
    launch_product<MODE, CG, BN, kSplit>(g, sms, st);
  };
  using std::integral_constant;
  const bool wide = product_tiles(kSym, rows, cols, 128, 256, ti, tj) * batch >= sms;
  const bool medium = product_tiles(kSym, rows, cols, 128, 128, ti, tj) * batch >= sms / 2;
  const integral_constant<int, 1> one{};
  if (split) {
    if (medium) go(one, integral_constant<int, 128>{}, std::true_type{});
    else go(one, integral_constant<int, 64>{}, std::true_type{});
  } else if (wide) {
    go(one, integral_constant<int, 256>{}, std::false_type{});
  } else if (medium) {
    go(one, integral_constant<int, 128>{}, std::false_type{});
  } else {
    go(one, integral_constant<int, 64>{}, std::false_type{});
  }
}

// The orthogonalised update of `u` into `fin`.
void orthogonalise(const UpdateArgs &u, int64_t batch, int steps, float eps, bool split, FinishArgs fin, void *workspace,
                   size_t workspace_bytes, int device, cudaStream_t st) {
  const bool transposed = u.m > u.n;
  const int64_t s = std::min(u.m, u.n), w = std::max(u.m, u.n);
  Space sp = muon_space(workspace, batch, s, w, split);
  if (workspace_bytes < sp.bytes) throw std::invalid_argument("workspace is smaller than se_muon_workspace asks for");
  const int sms = sm_count(device);
  uint32_t *status = ns_status(device);
  if (*static_cast<volatile uint32_t *>(status) != 0u) {
    *static_cast<volatile uint32_t *>(status) = 0u;
    throw Error(SE_ERR_RUNTIME, "an earlier orthogonalisation on cuda:" + std::to_string(device) +
                                    " gave up waiting for its copies; its results are not valid");
  }
  const int64_t count = u.m * u.n;
  const int nparts = int(std::min<int64_t>(kNormParts, (count + 1023) / 1024));
  k_muon_momentum<<<dim3(unsigned(nparts), unsigned(batch)), 256, 0, st>>>(u, sp.parts);
  launched("k_muon_momentum");
  {
    const int64_t tiles = ((u.m + 31) / 32) * ((u.n + 31) / 32);
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(unsigned(std::min<int64_t>(tiles, 1024)), 1, unsigned(batch));
    cfg.blockDim = dim3(256);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    cuda_check(cudaLaunchKernelEx(&cfg, k_muon_scale, u, static_cast<const double *>(sp.parts), nparts, eps, transposed,
                                  sp.x[0].hi, sp.x[0].lo, sp.x[0].ld, sp.x[0].batch),
               "k_muon_scale");
    launched("k_muon_scale");
  }
  fin.transposed = transposed;
  for (int k = 0; k < steps; ++k) {
    const Pair &x = sp.x[k & 1], &next = sp.x[(k & 1) ^ 1];
    ProductArgs g{};
    g.status = status;
    g.out = sp.a;
    g.diag_out = sp.diag_a;
    product<kGram>(g, x, x, s, s, w, batch, split, sms, st);
    g.in = sp.a;
    g.out = sp.b;
    g.diag_in = sp.diag_a;
    g.diag_out = sp.diag_b;
    product<kSquare>(g, sp.a, sp.a, s, s, s, batch, split, sms, st);
    g.in = x;
    g.out = next;
    g.diag_in = sp.diag_b;
    g.diag_out = nullptr;
    g.fin = fin;
    if (k + 1 < steps) product<kApply>(g, sp.b, x, s, w, s, batch, split, sms, st);
    else product<kFinish>(g, sp.b, x, s, w, s, batch, split, sms, st);
  }
}

void check_matrices(size_t batch, int64_t m, int64_t n, int32_t steps, float eps) {
  if (m < 0 || n < 0 || m > (1 << 20) || n > (1 << 20)) throw std::invalid_argument("m and n must be in [0, 2^20]");
  if (batch > 65535) throw std::invalid_argument("batch must be at most 65535");
  if (steps < 1 || steps > 100) throw std::invalid_argument("steps must be in [1, 100]");
  if (!(eps >= 0.0f) || !std::isfinite(eps)) throw std::invalid_argument("eps must be finite and non-negative");
}

void check_strides(const char *what, size_t batch, int64_t m, int64_t n, int64_t bs, int64_t rs) {
  if ((m > 1 && rs < n) || (batch > 1 && bs < (m - 1) * std::max(rs, n) + n))
    throw std::invalid_argument(std::string(what) + "'s rows or matrices overlap");
}

}  // namespace

}  // namespace se_gpu

using namespace se_gpu;

extern "C" int se_muon_workspace(int32_t out_dtype, size_t batch, int64_t m, int64_t n, size_t *bytes) {
  return guarded([&] {
    check_value_dtype(out_dtype, "out_dtype");
    check_matrices(batch, m, n, 1, 0.0f);
    if (bytes == nullptr) throw std::invalid_argument("bytes is null");
    *bytes = batch == 0 || m == 0 || n == 0
                 ? 0
                 : muon_space(nullptr, int64_t(batch), std::min(m, n), std::max(m, n), split_products(out_dtype)).bytes;
  });
}

extern "C" int se_orthogonalize(int32_t dtype, const void *update, size_t batch, int64_t m, int64_t n,
                                int64_t batch_stride, int64_t row_stride, int32_t steps, float eps, void *out,
                                void *workspace, size_t workspace_bytes, int32_t device, void *stream) {
  return guarded([&] {
    check_value_dtype(dtype, "dtype");
    check_matrices(batch, m, n, steps, eps);
    if (batch == 0 || m == 0 || n == 0) return;
    check_strides("update", batch, m, n, batch_stride, row_stride);
    DeviceGuard dg(device);
    check_device_ptr(update, device, "update");
    check_device_ptr(out, device, "out");
    check_device_ptr(workspace, device, "workspace");
    if (reinterpret_cast<uintptr_t>(workspace) % 256 != 0) throw std::invalid_argument("workspace must be 256-byte aligned");
    UpdateArgs u{};
    u.grad = {update, batch_stride, row_stride};
    u.grad_type = dtype;
    u.m = m;
    u.n = n;
    FinishArgs fin{};
    fin.out = out;
    fin.type = dtype;
    fin.row = n;
    fin.batch = m * n;
    orthogonalise(u, int64_t(batch), steps, eps, split_products(dtype), fin, workspace, workspace_bytes, device,
                  static_cast<cudaStream_t>(stream));
  });
}

extern "C" int se_muon_step(int32_t weight_dtype, int32_t grad_dtype, void *weight, int64_t weight_batch_stride,
                            int64_t weight_row_stride, const void *grad, int64_t grad_batch_stride,
                            int64_t grad_row_stride, float *momentum, int64_t momentum_batch_stride,
                            int64_t momentum_row_stride, size_t batch, int64_t m, int64_t n, double lr, double beta,
                            double weight_decay, double scale, int32_t nesterov, int32_t steps, float eps,
                            void *workspace, size_t workspace_bytes, int32_t device, void *stream) {
  return guarded([&] {
    check_value_dtype(weight_dtype, "weight_dtype");
    check_value_dtype(grad_dtype, "grad_dtype");
    check_matrices(batch, m, n, steps, eps);
    if (!std::isfinite(lr) || !std::isfinite(beta) || !std::isfinite(weight_decay) || !std::isfinite(scale))
      throw std::invalid_argument("lr, beta, weight_decay and scale must be finite");
    if (beta < 0.0 || beta >= 1.0) throw std::invalid_argument("beta must be in [0, 1)");
    if (batch == 0 || m == 0 || n == 0) return;
    check_strides("weight", batch, m, n, weight_batch_stride, weight_row_stride);
    check_strides("grad", batch, m, n, grad_batch_stride, grad_row_stride);
    check_strides("momentum", batch, m, n, momentum_batch_stride, momentum_row_stride);
    DeviceGuard dg(device);
    check_device_ptr(weight, device, "weight");
    check_device_ptr(grad, device, "grad");
    check_device_ptr(momentum, device, "momentum");
    check_device_ptr(workspace, device, "workspace");
    if (reinterpret_cast<uintptr_t>(workspace) % 256 != 0) throw std::invalid_argument("workspace must be 256-byte aligned");
    UpdateArgs u{};
    u.grad = {grad, grad_batch_stride, grad_row_stride};
    u.grad_type = grad_dtype;
    u.momentum = {momentum, momentum_batch_stride, momentum_row_stride};
    u.beta = float(beta);
    u.nesterov = nesterov != 0;
    u.m = m;
    u.n = n;
    FinishArgs fin{};
    fin.out = weight;
    fin.type = weight_dtype;
    fin.update = 1;
    fin.row = weight_row_stride;
    fin.batch = weight_batch_stride;
    fin.keep = float(1.0 - lr * weight_decay);
    fin.rate = float(lr * scale);
    orthogonalise(u, int64_t(batch), steps, eps, split_products(weight_dtype), fin, workspace, workspace_bytes, device,
                  static_cast<cudaStream_t>(stream));
  });
}
