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
//  * bf16 outputs: products of the hi parts alone, unless the caller asks for
//    full ones. fp32 and f16 outputs, and bf16 ones then: hi hi + hi lo + lo hi,
//    three times the matrix work, for errors of fp32's order.
// Against 64 bits, for gradient-like matrices: 0.03 to 0.1 % from the single
// products (bf16's own rounding is 0.17 %), 0.5e-6 to 1.3e-6 from the triple ones
// (fp32 operations in place of them: 0.7e-6 to 3e-6). With 1 to 8 directions far
// above the rest, where noise is magnified most, the triple products' error is
// 0.2 to 0.9 of that of fp32 operations (100 x 200 to 2048 x 1024); X in fp32
// beside the pair would take a tenth off it, for a third more of the workspace.
//
// A and A A are symmetric: only tiles that touch the lower triangle are
// computed, and an element below the diagonal is written to both places by the
// thread that holds it.

#include <algorithm>
#include <iterator>
#include <type_traits>

#include "se_dense.hpp"
#include "se_tcgen05.cuh"

namespace se_gpu {

namespace {

constexpr float kNsA = 3.4445f, kNsB = -4.7750f, kNsC = 2.0315f;
constexpr float kScale = 8192.0f;  // S
constexpr int kTileK = 64;         // k-values of a stage: one 128-byte swizzle row

struct BF16Full : BF16 {};  // bf16 results of full products: any result type but BF16 has three for one

// ---------------------------------------------------------------------------
// Momentum, norm, and the scaled update X_0
// ---------------------------------------------------------------------------

struct Strided {  // a batch of matrices with contiguous rows
  const void *p;
  int64_t batch, row;
};

constexpr int kNormParts = 512;  // blocks (and partial sums) per matrix, at most
constexpr int kSpan = 2048;      // values of a row that a block takes at a time, 8 per thread

struct UpdateArgs {
  Strided grad;      // the update itself (orthogonalize), or the gradient
  Strided momentum;  // fp32; p null: the update is grad
  float beta;
  int nesterov;
  int64_t m, n;
  int vec;           // rows of both start at 16-byte boundaries, n is a multiple of 8
};

// Eight consecutive values, or with vec = 0 eight that are `step` apart, the first `count`.
template <class V>
__device__ __forceinline__ void load_eight(const typename V::T *p, bool vec, int step, int count, float (&f)[8]) {
  using T = typename V::T;
  if (vec) {
    constexpr int kPer = 16 / sizeof(T);
    uint4 raw[8 / kPer];
#pragma unroll
    for (int i = 0; i < 8 / kPer; ++i) raw[i] = count > 0 ? reinterpret_cast<const uint4 *>(p)[i] : make_uint4(0u, 0u, 0u, 0u);
    const T *v = reinterpret_cast<const T *>(raw);
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = V::load(v[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = i < count ? V::load(p[i * step]) : 0.0f;
  }
}

// U from the gradient and the momentum after its update.
__device__ __forceinline__ float update_of(const UpdateArgs &a, float g, float mom) {
  return a.nesterov ? __fmaf_rn(a.beta, mom, g) : mom;
}

// Adds eight squares to `sum` through an fp32 sum (a conversion to fp64 per value
// would take longer than the loads). True where that was not safe: fp32 squares
// may have overflowed or vanished, and the caller takes its sum again with
// wide_square_sum.
__device__ __forceinline__ bool square_sum(const float (&u)[8], double &sum) {
  float f = 0.0f, most = 0.0f;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    f = __fmaf_rn(u[e], u[e], f);
    most = fmaxf(most, fabsf(u[e]));
  }
  sum += double(f);
  return !(f > 1e-24f && f < 1e36f) && !(most == 0.0f && f == 0.0f);
}
__device__ __forceinline__ void wide_square_sum(const float (&u)[8], double &sum) {
#pragma unroll
  for (int e = 0; e < 8; ++e) sum = fma(double(u[e]), double(u[e]), sum);
}

// S / (|U| + eps) as a fraction and two powers of two: the factor itself may lie
// outside fp32's range.
struct Factor {
  float fraction, power0, power1;
  __device__ __forceinline__ float times(float u) const { return u * power0 * power1 * fraction; }
};
__device__ __forceinline__ Factor update_factor(double sum, float eps) {
  const double f = double(kScale) / (sqrt(sum) + double(eps));
  Factor r;
  if (!(f > 0.0) || f > 1.7e308) {  // a sum that is infinite, no number, or zero with eps = 0
    r.fraction = float(f);
    r.power0 = r.power1 = 1.0f;
    return r;
  }
  int k;
  r.fraction = float(frexp(f, &k));  // [0.5, 1]
  const int half = k / 2;
  r.power0 = ldexpf(1.0f, half);
  r.power1 = ldexpf(1.0f, k - half);
  return r;
}

// M <- beta M + G, and this block's part of |U|^2. Zeroes the counters of the
// launch that follows. Bound by HBM: a matrix without gaps is taken as one row, and
// every thread has 8 values of each array in flight (8 x 1024 x 2048 bf16 31 us,
// 5.4 TB/s).
template <class V, bool MOM>
__global__ void __launch_bounds__(256)
k_muon_momentum(UpdateArgs a, double *__restrict__ parts, uint32_t *__restrict__ counters, int64_t ncounters) {
  __shared__ double red[8];
  const int64_t z = blockIdx.y;
  if (z == 0) {
    for (int64_t e = int64_t(blockIdx.x) * blockDim.x + threadIdx.x; e < ncounters; e += int64_t(gridDim.x) * blockDim.x)
      counters[e] = 0u;
  }
  const bool dense = a.grad.row == a.n && (!MOM || a.momentum.row == a.n);
  const int64_t rows = dense ? 1 : a.m, len = dense ? a.m * a.n : a.n;
  const int64_t spans = (len + kSpan - 1) / kSpan;
  const int step = a.vec ? 1 : 256;
  double sum = 0.0;
  bool unsafe = false;
  auto place = [&](int64_t t, int64_t &i, int64_t &j) {
    i = t / spans;
    j = (t - i * spans) * kSpan + threadIdx.x * (a.vec ? 8 : 1);
    return j >= len ? 0 : int(min(int64_t(8), (len - j + step - 1) / step));
  };
  for (int64_t t = blockIdx.x; t < rows * spans; t += gridDim.x) {
    int64_t i, j;
    const int count = place(t, i, j);
    float g[8];
    load_eight<V>(static_cast<const typename V::T *>(a.grad.p) + z * a.grad.batch + i * a.grad.row + j, a.vec, step, count, g);
    if constexpr (MOM) {
      float *mp = const_cast<float *>(static_cast<const float *>(a.momentum.p)) + z * a.momentum.batch + i * a.momentum.row + j;
      float mom[8];
      load_eight<F32>(mp, a.vec, step, count, mom);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        mom[e] = __fmaf_rn(a.beta, mom[e], g[e]);
        g[e] = update_of(a, g[e], mom[e]);
      }
      if (a.vec) {
        if (count > 0) {
          reinterpret_cast<float4 *>(mp)[0] = make_float4(mom[0], mom[1], mom[2], mom[3]);
          reinterpret_cast<float4 *>(mp)[1] = make_float4(mom[4], mom[5], mom[6], mom[7]);
        }
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (e < count) mp[e * step] = mom[e];
      }
    }
    unsafe |= square_sum(g, sum);
  }
  if (__syncthreads_or(unsafe)) {
    sum = 0.0;
    for (int64_t t = blockIdx.x; t < rows * spans; t += gridDim.x) {
      int64_t i, j;
      const int count = place(t, i, j);
      float g[8], mom[8];
      load_eight<V>(static_cast<const typename V::T *>(a.grad.p) + z * a.grad.batch + i * a.grad.row + j, a.vec, step, count, g);
      if constexpr (MOM) {
        load_eight<F32>(static_cast<const float *>(a.momentum.p) + z * a.momentum.batch + i * a.momentum.row + j, a.vec, step,
                        count, mom);
#pragma unroll
        for (int e = 0; e < 8; ++e) g[e] = update_of(a, g[e], mom[e]);
      }
      wide_square_sum(g, sum);
    }
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

// Eight values of X as hi + lo, 16 bytes each.
__device__ __forceinline__ void put_eight(__half *hi, __half *lo, const float (&f)[8]) {
  uint4 h, l;
  __half2 *hh = reinterpret_cast<__half2 *>(&h), *ll = reinterpret_cast<__half2 *>(&l);
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    hh[e] = __floats2half2_rn(f[2 * e], f[2 * e + 1]);
    const float2 b = __half22float2(hh[e]);
    ll[e] = __floats2half2_rn(f[2 * e] - b.x, f[2 * e + 1] - b.y);
  }
  *reinterpret_cast<uint4 *>(hi) = h;
  *reinterpret_cast<uint4 *>(lo) = l;
}

// X_0 = S U / (|U| + eps) as hi + lo, s x w (transposed where m > n): along the
// rows in 16-byte vectors, or, where the sides are exchanged or the layout has
// no vectors, in tiles of 64 x 64 values, 16 per thread, through shared memory,
// so that both are read and written by rows. X's storage reaches
// to a multiple of 64 columns, so its rows are written in whole vectors. Bound
// by HBM (8 x 1024 x 2048 bf16 31 us, 5.5 TB/s).
template <class V, bool MOM>
__global__ void __launch_bounds__(256)
k_muon_scale(UpdateArgs a, const double *__restrict__ parts, int nparts, float eps, bool transposed,
             __half *__restrict__ hi, __half *__restrict__ lo, int64_t ld, int64_t batch_stride) {
  __shared__ float tile[64][65];
  __shared__ Factor factor;
  const int64_t z = blockIdx.z;
  pdl_wait();
  if (threadIdx.x < 32) {
    double sum = 0.0;
    for (int k = threadIdx.x; k < nparts; k += 32) sum += parts[z * kNormParts + k];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (threadIdx.x == 0) factor = update_factor(sum, eps);
  }
  __syncthreads();
  const Factor k = factor;
  if (a.vec && !transposed) {  // along the rows: as many threads per row as it has eights, up to the block
    int shift = 0;
    while (shift < 8 && (int64_t(8) << shift) < a.n) ++shift;
    const int lanes = 1 << shift, sub = threadIdx.x & (lanes - 1);
    const int64_t each = blockDim.x >> shift;
    for (int64_t i = blockIdx.x * each + (threadIdx.x >> shift); i < a.m; i += gridDim.x * each) {
#pragma unroll 2
      for (int64_t j = sub * 8; j < a.n; j += lanes * 8) {
        float u[8];
        load_eight<V>(static_cast<const typename V::T *>(a.grad.p) + z * a.grad.batch + i * a.grad.row + j, true, 1, 8, u);
        if constexpr (MOM) {
          float mom[8];
          load_eight<F32>(static_cast<const float *>(a.momentum.p) + z * a.momentum.batch + i * a.momentum.row + j, true, 1, 8,
                          mom);
#pragma unroll
          for (int e = 0; e < 8; ++e) u[e] = update_of(a, u[e], mom[e]);
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) u[e] = k.times(u[e]);
        put_eight(hi + z * batch_stride + i * ld + j, lo + z * batch_stride + i * ld + j, u);
      }
    }
    return;
  }
  const int row = threadIdx.x >> 3, at = threadIdx.x & 7;  // 8 threads of 8 values per row, rows `row` and `row` + 32
  const int step = a.vec ? 1 : 8, first = a.vec ? at * 8 : at;
  const int64_t tiles_j = (a.n + 63) / 64, tiles = tiles_j * ((a.m + 63) / 64);
  for (int64_t t = blockIdx.x; t < tiles; t += gridDim.x) {
    const int64_t i0 = t / tiles_j * 64, j0 = (t - t / tiles_j * tiles_j) * 64;
    float u[2][8];
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const int64_t i = i0 + row + 32 * q, j = j0 + first;
      const int count = i >= a.m || j >= a.n ? 0 : int(min(int64_t(8), (a.n - j + step - 1) / step));
      load_eight<V>(static_cast<const typename V::T *>(a.grad.p) + z * a.grad.batch + i * a.grad.row + j, a.vec, step, count,
                    u[q]);
      if constexpr (MOM) {
        float mom[8];
        load_eight<F32>(static_cast<const float *>(a.momentum.p) + z * a.momentum.batch + i * a.momentum.row + j, a.vec, step,
                        count, mom);
#pragma unroll
        for (int e = 0; e < 8; ++e) u[q][e] = update_of(a, u[q][e], mom[e]);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) u[q][e] = k.times(u[q][e]);
    }
#pragma unroll
    for (int q = 0; q < 2; ++q) {
#pragma unroll
      for (int e = 0; e < 8; ++e) tile[row + 32 * q][first + e * step] = u[q][e];
    }
    __syncthreads();
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const int r = row + 32 * q, c = at * 8;
#pragma unroll
      for (int e = 0; e < 8; ++e) u[q][e] = transposed ? tile[c + e][r] : tile[r][c + e];
      const int64_t rr = (transposed ? j0 : i0) + r, cc = (transposed ? i0 : j0) + c;
      if (rr < (transposed ? a.n : a.m)) put_eight(hi + z * batch_stride + rr * ld + cc, lo + z * batch_stride + rr * ld + cc, u[q]);
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
  int vec;    // four values of a row at a time: whole 8 or 16 bytes
  int64_t row, batch;
  float keep, rate;
};

// How one kind of product is cut up: tiles of the result, each over `parts`
// parts of the k-values.
struct Cut {
  int rows, cols, kblocks;
  int tiles_j, tiles;  // of one matrix
  int parts;
};

struct NsArgs {
  CUtensorMap x_hi[2], x_lo[2], a_hi, a_lo, b_hi, b_lo;  // boxes of 64 x 64
  Cut gram, square, apply;
  int batch, steps;
  Pair x[2], a, b;
  float *diag_a, *diag_b;  // A's diagonal (scaled by S), B's (not scaled)
  int64_t diag_ld;         // of the next matrix's
  float *partial;          // gram.parts > 1: partial sums of its blocks, [block][part][32][32]
  uint32_t *arrived;       // and how many parts of a block are there
  uint32_t *barrier;       // blocks that finished a product
  uint32_t *failed;        // set when a wait gave up: X is not the result
  FinishArgs fin;
  long long limit;
  uint32_t *status;
};

constexpr int kEpilogueWarps = 8;
constexpr int kThreads = 128 + 32 * kEpilogueWarps;
constexpr int kFlush = 4;  // k-blocks of a SPLIT accumulation between two flushes

// Shared memory of a CTA: operand stages, then the epilogue warps' staging
// tiles.
//
// SPLIT has hi and lo parts of both operands in a stage, B's one below the
// other: A_hi times both is one instruction of N = 128, which takes no longer
// than N = 64 (75 clocks: A is read from shared memory either way), and A_lo B_hi
// adds to the half of A_hi B_lo: two thirds of the instructions and of the loads
// of the three products one after another (1000 x 517 fp32: 188 -> 159 us). At
// N = 128 an instruction of twice the width takes twice as long, so its tiles
// are 128 x 64 always. (Wider ones with three products one after another, us,
// 128 x 64 and the best of 128 x 128 and pairs: 1024 x 1024 fp32 181 and 286,
// 2560 x 2560 1,210 and 1,393, 4096 x 4096 5,056 and 4,985, 6144 x 6144 18,070
// and 17,408: too little and too rarely for kernels of their own.)
template <int CG, int BN, bool SPLIT>
struct Layout {
  static_assert(!SPLIT || (CG == 1 && BN == 64), "the tile of three products");
  static constexpr int kA = 128 * 128 * (SPLIT ? 2 : 1);        // bytes of a CTA's A tile: 128 rows of 64 values
  static constexpr int kB = (BN / CG) * 128 * (SPLIT ? 2 : 1);  // and of its part of the B tile
  static constexpr int kStage = kA + kB;
  static constexpr int kColumns = SPLIT ? 2 * BN : BN;          // of an accumulator
  static constexpr int kStaging = 32 * 32;                      // floats of a warp
  static constexpr int kStagingBytes = kEpilogueWarps * kStaging * 4;
  static constexpr int kRoom = 232448 - 1024 - 512 - kStagingBytes;  // 1,024: tile alignment; 512: static variables
  static constexpr int kStages = kRoom / kStage < 8 ? kRoom / kStage : 8;
  static constexpr int kBytes = kStages * kStage + kStagingBytes + 1024;
};

// Tile t of a matrix: its first row and column. The symmetric products list
// only tiles that reach the lower triangle, row of tiles by row of tiles.
template <int MODE, int TM, int BN>
__device__ __forceinline__ void tile_at(const Cut &c, int t, int &row, int &col) {
  if constexpr (MODE == kGram || MODE == kSquare) {
    int i = 0;
    for (;; ++i) {
      const int in_row = min((i * TM + TM - 1) / BN + 1, c.tiles_j);
      if (t < in_row) break;
      t -= in_row;
    }
    row = i * TM;
    col = t * BN;
  } else {
    const int i = t / c.tiles_j;
    row = i * TM;
    col = (t - i * c.tiles_j) * BN;
  }
}

// Place of (r, c) in a staging tile: groups of four values of a row are moved
// about by the row, so that a warp's 16-byte accesses along rows and its 4-byte
// accesses down four rows at a time meet no bank twice.
__device__ __forceinline__ int tile_place(int r, int c) {
  return r * 32 + ((((c >> 2) ^ r ^ (r >> 2)) & 7) << 2) + (c & 3);
}

// Four f16 values that other blocks may have written during the launch: from L2.
__device__ __forceinline__ uint2 load_four(const __half *p) { return __ldcg(reinterpret_cast<const uint2 *>(p)); }
__device__ __forceinline__ float4 open_four(uint2 v) {
  const float2 a = __half22float2(*reinterpret_cast<__half2 *>(&v.x)), b = __half22float2(*reinterpret_cast<__half2 *>(&v.y));
  return make_float4(a.x, a.y, b.x, b.y);
}
// Four values as hi, and with `split` lo, at the same offset of both.
__device__ __forceinline__ void put_four(__half *hi, __half *lo, const float4 &f, bool split) {
  const __half2 a = __floats2half2_rn(f.x, f.y), b = __floats2half2_rn(f.z, f.w);
  *reinterpret_cast<uint2 *>(hi) =
      make_uint2(*reinterpret_cast<const unsigned *>(&a), *reinterpret_cast<const unsigned *>(&b));
  if (split) {
    const float2 ra = __half22float2(a), rb = __half22float2(b);
    const __half2 c = __floats2half2_rn(f.x - ra.x, f.y - ra.y), d = __floats2half2_rn(f.z - rb.x, f.w - rb.y);
    *reinterpret_cast<uint2 *>(lo) =
        make_uint2(*reinterpret_cast<const unsigned *>(&c), *reinterpret_cast<const unsigned *>(&d));
  }
}
// Four consecutive values of the result's type as one store where its rows allow
// that (`vec`), else the first `count` one by one.
template <class OUT>
__device__ __forceinline__ void store_four(typename OUT::T *p, const float4 &f, bool vec, int count) {
  using T = typename OUT::T;
  using Raw = std::conditional_t<sizeof(T) == 4, uint4, uint2>;
  const T v[4] = {OUT::store(f.x), OUT::store(f.y), OUT::store(f.z), OUT::store(f.w)};
  if (vec) {
    if (count > 0) *reinterpret_cast<Raw *>(p) = *reinterpret_cast<const Raw *>(v);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (e < count) p[e] = v[e];
  }
}

// Where a block of O lies in the result: this lane's first four values, the rows
// of the result below it (every fourth), and how many of the four there are.
template <class OUT>
struct FinishBlock {
  typename OUT::T *at;
  int turns, count;
  __device__ __forceinline__ FinishBlock(const NsArgs &g, int z, int r0, int c0) {
    const int lane = int(threadIdx.x) & 31, up = lane >> 3, four = (lane & 7) * 4;
    const FinishArgs &f = g.fin;
    const int row = f.transposed ? c0 : r0, col = f.transposed ? r0 : c0;
    const int rows = f.transposed ? g.apply.cols : g.apply.rows, cols = f.transposed ? g.apply.rows : g.apply.cols;
    at = static_cast<typename OUT::T *>(f.out) + int64_t(z) * f.batch + int64_t(row + up) * f.row + col + four;
    turns = (min(32, rows - row) - up + 3) >> 2;
    count = max(0, min(4, cols - col - four));
  }
};

// What the epilogue of a 32 x 32 block reads besides the accumulator: A (kSquare)
// or X (kApply, kFinish), and A's diagonal over the columns. A warp asks for it
// before it waits for the accumulator, or while it still works on the block
// before, so that the latency is hidden.
template <int MODE, class OUT>
struct BlockInput {
  static constexpr bool kLo = MODE == kApply || MODE == kFinish || !std::is_same_v<OUT, BF16>;
  uint2 hi[8], lo[8];
  float4 diag;
  __device__ __forceinline__ void load(const NsArgs &g, int step, int z, int r0, int c0) {
    if constexpr (MODE != kGram) {
      const int lane = int(threadIdx.x) & 31, up = lane >> 3, four = (lane & 7) * 4;
      const Pair &in = MODE == kSquare ? g.a : g.x[step & 1];
      const int turns = (min(32, g.apply.rows - r0) - up + 3) >> 2;
      const int64_t from = int64_t(z) * in.batch + int64_t(r0 + up) * in.ld + c0 + four;
      const __half *h = in.hi + from, *l = in.lo + from;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        hi[i] = i < turns ? load_four(h) : make_uint2(0u, 0u);
        if constexpr (kLo) lo[i] = i < turns ? load_four(l) : make_uint2(0u, 0u);
        h += 4 * in.ld;
        l += 4 * in.ld;
      }
      if constexpr (MODE == kSquare)  // padded like the columns
        diag = __ldcg(reinterpret_cast<const float4 *>(g.diag_a + int64_t(z) * g.diag_ld + c0 + four));
    }
  }
};

// The epilogue of a 32 x 32 block of the accumulator, staged by the warp in
// `tile`. A turn handles four rows, eight lanes of four values each: global
// accesses are whole 32-byte sectors, and the code is short (a block's
// instructions run once, so that their fetches would cost more than the work:
// an unrolled first version took 4,300 to 8,000 clocks a block). `next` is
// called where the block's input has been used. Rows are r0 .. r0 + 31,
// columns c0 .. c0 + 31, both multiples of 32; storage reaches past the last
// column to a multiple of 64, so columns need no guard.
template <int MODE, class OUT, class Next>
__device__ __forceinline__ void finish_block(const NsArgs &g, int step, float *tile, int z, int r0, int c0,
                                             float dr_lane, const BlockInput<MODE, OUT> &input, Next &&next) {
  constexpr bool kSym = MODE == kGram || MODE == kSquare;
  constexpr bool kInLo = BlockInput<MODE, OUT>::kLo, SPLIT = !std::is_same_v<OUT, BF16>;
  const int lane = int(threadIdx.x) & 31, up = lane >> 3, four = (lane & 7) * 4;
  const int rows = g.apply.rows;
  const Pair &out = MODE == kGram ? g.a : MODE == kSquare ? g.b : g.x[(step & 1) ^ 1];
  const int turns = (min(32, rows - r0) - up + 3) >> 2;  // this lane's rows: r0 + up, r0 + up + 4, ...
  auto down = [&](int c) {  // four rows of column c
    return make_float4(tile[tile_place(four, c)], tile[tile_place(four + 1, c)], tile[tile_place(four + 2, c)],
                       tile[tile_place(four + 3, c)]);
  };
  const bool diagonal = kSym && r0 == c0;
  if (diagonal) {
    // The diagonal's value goes to its vector: (A A)_rr = acc + D_r^2. (Both
    // triangles of the block are written as they were summed; they differ by
    // the order of fp32 additions at most.)
    const float acc = tile[tile_place(lane, lane)];
    if (r0 + lane < rows) {
      const int64_t at = int64_t(z) * g.diag_ld + r0 + lane;
      if constexpr (MODE == kGram) g.diag_a[at] = acc * (1.0f / kScale);
      else g.diag_b[at] = __fmaf_rn(kNsC / kScale, __fmaf_rn(dr_lane, dr_lane, acc), kNsB * dr_lane) * (1.0f / kScale);
    }
    __syncwarp();
  }
  // Reads of the staged block before its writes: in turn, each would wait for the other.
  float4 v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = *reinterpret_cast<const float4 *>(tile + tile_place(4 * i + up, four));
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int rr = 4 * i + up;
    float4 &f = v[i];
    if constexpr (MODE == kGram) {
      f.x *= 1.0f / kScale;
      f.y *= 1.0f / kScale;
      f.z *= 1.0f / kScale;
      f.w *= 1.0f / kScale;
    } else {
      float4 x = open_four(input.hi[i]);
      if constexpr (kInLo) {
        const float4 l = open_four(input.lo[i]);
        x.x += l.x;
        x.y += l.y;
        x.z += l.z;
        x.w += l.w;
      }
      const float dr = __shfl_sync(0xffffffffu, dr_lane, rr);
      if constexpr (MODE == kSquare) {  // off the diagonal (A A)_rc = acc + (D_r + D_c) O_rc
        f.x = __fmaf_rn(kNsC / kScale, __fmaf_rn(dr + input.diag.x, x.x, f.x), kNsB * x.x);
        f.y = __fmaf_rn(kNsC / kScale, __fmaf_rn(dr + input.diag.y, x.y, f.y), kNsB * x.y);
        f.z = __fmaf_rn(kNsC / kScale, __fmaf_rn(dr + input.diag.z, x.z, f.z), kNsB * x.z);
        f.w = __fmaf_rn(kNsC / kScale, __fmaf_rn(dr + input.diag.w, x.w, f.w), kNsB * x.w);
      } else {
        const float k = kNsA + dr;
        f.x = __fmaf_rn(k, x.x, f.x * (1.0f / kScale));
        f.y = __fmaf_rn(k, x.y, f.y * (1.0f / kScale));
        f.z = __fmaf_rn(k, x.z, f.z * (1.0f / kScale));
        f.w = __fmaf_rn(k, x.w, f.w * (1.0f / kScale));
      }
    }
    if (diagonal) {
      if (rr == four) f.x = 0.0f;
      if (rr == four + 1) f.y = 0.0f;
      if (rr == four + 2) f.z = 0.0f;
      if (rr == four + 3) f.w = 0.0f;
    }
  }
  if constexpr (MODE == kFinish) {
    const FinishArgs &fin = g.fin;
    const FinishBlock<OUT> to(g, z, r0, c0);
    if (fin.transposed) {
#pragma unroll
      for (int i = 0; i < 8; ++i) *reinterpret_cast<float4 *>(tile + tile_place(4 * i + up, four)) = v[i];
      __syncwarp();
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = down(4 * i + up);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float4 &f = v[i];
      f = make_float4(f.x * (1.0f / kScale), f.y * (1.0f / kScale), f.z * (1.0f / kScale), f.w * (1.0f / kScale));
    }
    next();
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < to.turns) store_four<OUT>(to.at + int64_t(4 * i) * fin.row, v[i], fin.vec, to.count);
    return;
  }
  next();
  if constexpr (MODE != kFinish) {
    const int64_t to = int64_t(z) * out.batch + int64_t(r0 + up) * out.ld + c0 + four;
    __half *oh = out.hi + to, *ol = out.lo + to;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (i < turns) put_four(oh, ol, v[i], kInLo);
      oh += 4 * out.ld;
      ol += 4 * out.ld;
    }
  }
  if constexpr (kSym) {
    if (!diagonal) {  // the mirror: rows c0 .., columns r0 ..
      __syncwarp();
#pragma unroll
      for (int i = 0; i < 8; ++i) *reinterpret_cast<float4 *>(tile + tile_place(4 * i + up, four)) = v[i];
      __syncwarp();
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = down(4 * i + up);
      const int64_t to = int64_t(z) * out.batch + int64_t(c0 + up) * out.ld + r0 + four;
      __half *oh = out.hi + to, *ol = out.lo + to;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        put_four(oh, ol, v[i], SPLIT);
        oh += 4 * out.ld;
        ol += 4 * out.ld;
      }
    }
  }
}

// Parts of a sum: each leaves its block in `partial` (leave_part), and the warp
// whose part arrives last (last_part) adds all of them in their order into
// `tile` (join_parts). `block` numbers the blocks of all tiles.
__device__ __forceinline__ float4 *staged_four(float *tile, int i) {
  const int lane = int(threadIdx.x) & 31;
  return reinterpret_cast<float4 *>(tile + tile_place(4 * i + (lane >> 3), (lane & 7) * 4));
}
__device__ __forceinline__ void leave_part(const NsArgs &g, float *tile, int64_t block, int part) {
  float4 *mine = reinterpret_cast<float4 *>(g.partial + (block * g.gram.parts + part) * 1024) + (threadIdx.x & 31);
#pragma unroll
  for (int i = 0; i < 8; ++i) __stcg(mine + 32 * i, *staged_four(tile, i));
}
__device__ __forceinline__ bool last_part(const NsArgs &g, uint32_t *arrived) {
  __threadfence();
  __syncwarp();
  uint32_t before = 0;
  if ((threadIdx.x & 31) == 0) before = atomicAdd(arrived, 1u);
  before = __shfl_sync(0xffffffffu, before, 0);
  if (before != uint32_t(g.gram.parts - 1)) return false;
  __threadfence();
  if ((threadIdx.x & 31) == 0) *arrived = 0u;  // for the next step
  return true;
}
__device__ __forceinline__ void join_parts(const NsArgs &g, float *tile, int64_t block) {
  const int parts = g.gram.parts;
  const float4 *all = reinterpret_cast<const float4 *>(g.partial + block * parts * 1024) + (threadIdx.x & 31);
  float4 sum[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) sum[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 2
  for (int p = 0; p < parts; ++p) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float4 f = __ldcg(all + p * 256 + 32 * i);
      sum[i].x += f.x;
      sum[i].y += f.y;
      sum[i].z += f.z;
      sum[i].w += f.w;
    }
  }
  __syncwarp();
#pragma unroll
  for (int i = 0; i < 8; ++i) *staged_four(tile, i) = sum[i];
  __syncwarp();
}

// A ring of N buffers: the one in turn and how often the ring went round (its
// parity is the phase to wait for).
template <uint32_t N>
struct Ring {
  uint32_t at = 0, parity = 0;
  __device__ __forceinline__ void advance() {
    if (++at == N) {
      at = 0;
      parity ^= 1u;
    }
  }
};

// What a thread carries from product to product: where its role stands in the
// operand stages and in the accumulators, and the stages it has loaded.
template <uint32_t STAGES>
struct Progress {
  Ring<STAGES> stage;
  Ring<2> sum;
  uint32_t loaded = 0;
};

struct Shared {  // of a CTA
  uint64_t full[8], empty[8], acc_full[2], acc_empty[2], drained;
  uint32_t tmem;
  volatile uint32_t given_up;
};

// One product, all tiles of this unit (a CTA, or with CG = 2 a pair of them).
// Warp 0 loads operand stages by TMA, warp 1 issues the matrix instructions,
// warps 4-11 turn finished accumulators into the result while the next one is
// computed (two accumulators of BN columns in tensor memory; each epilogue
// warp has 32 rows of one half of the columns).
//
// SPLIT: the three products of hi and lo parts. The tensor core cuts its fp32
// sums off instead of rounding them, which over thousands of k-values costs
// more than the lo parts bring (measured: 3e-5 at 4,096), so a sum runs over
// kFlush k-blocks only and the epilogue warps add those up in registers.
template <int MODE, int CG, int BN, class OUT>
__device__ __forceinline__ void run_product(const NsArgs &g, const Cut &c, int step, Shared &sh, uint8_t *smem,
                                            uint32_t rank, Progress<Layout<CG, BN, !std::is_same_v<OUT, BF16>>::kStages> &at) {
  constexpr bool SPLIT = !std::is_same_v<OUT, BF16>;
  using L = Layout<CG, BN, SPLIT>;
  constexpr int kTM = 128 * CG, kBlocks = BN / 64;          // kBlocks: column blocks of an epilogue warp
  constexpr bool kBMN = MODE == kApply || MODE == kFinish;  // the B operand is X itself: n-contiguous
  constexpr uint32_t kStages = L::kStages;
  const int warp = int(threadIdx.x) >> 5, lane = int(threadIdx.x) & 31;
  const int unit = int(blockIdx.x) / CG, units = int(gridDim.x) / CG;
  const int parts = MODE == kGram ? c.parts : 1;
  const int total = c.tiles * parts * g.batch;
  // the k-blocks of part p
  auto k_from = [&](int p) { return MODE == kGram ? int(int64_t(c.kblocks) * p / parts) : p * c.kblocks; };
  auto sum_end = [&](int k, int last) { return SPLIT ? min(last, k + kFlush) : last; };

  if (warp == 0) {
    if (elect_one()) {
      const CUtensorMap *xh = &g.x_hi[step & 1], *xl = &g.x_lo[step & 1];
      const CUtensorMap *ah = MODE == kGram ? xh : MODE == kSquare ? &g.a_hi : &g.b_hi;
      const CUtensorMap *al = MODE == kGram ? xl : MODE == kSquare ? &g.a_lo : &g.b_lo;
      const CUtensorMap *bh = MODE == kSquare ? &g.a_hi : xh, *bl = MODE == kSquare ? &g.a_lo : xl;
      bool go = true;
      for (int t = unit; go && t < total; t += units) {
        const int zt = t / parts, z = zt / c.tiles, part = t - zt * parts;
        int row, col;
        tile_at<MODE, kTM, BN>(c, zt - z * c.tiles, row, col);
        row += int(rank) * 128;
        col += int(rank) * (BN / CG);
        for (int k = k_from(part), last = k_from(part + 1); k < last; ++k) {
          const uint32_t st = at.stage.at;
          if (!wait_or_give_up<true>(&sh.empty[st], at.stage.parity ^ 1u, &sh.given_up, g.limit)) {
            go = false;
            break;
          }
          const int k0 = k * kTileK;
          uint8_t *a = smem + st * L::kStage, *b = a + L::kA;
          uint32_t bar = smem_u32(&sh.full[st]);
          if constexpr (CG == 2) bar = mapa(bar, 0);
          if (rank == 0) mbar_arrive_expect_tx(&sh.full[st], CG * L::kStage);
#pragma unroll
          for (int q = 0; q < 2; ++q) tma_load<CG>(a + q * 8192, ah, k0, row + q * 64, z, bar);
#pragma unroll
          for (int q = 0; q < BN / CG / 64; ++q) {
            if constexpr (kBMN) tma_load<CG>(b + q * 8192, bh, col + q * 64, k0, z, bar);
            else tma_load<CG>(b + q * 8192, bh, k0, col + q * 64, z, bar);
          }
          if constexpr (SPLIT) {
#pragma unroll
            for (int q = 0; q < 2; ++q) tma_load<CG>(a + 16384 + q * 8192, al, k0, row + q * 64, z, bar);
            if constexpr (kBMN) tma_load<CG>(b + 8192, bl, col, k0, z, bar);
            else tma_load<CG>(b + 8192, bl, k0, col, z, bar);
          }
          at.stage.advance();
          ++at.loaded;
        }
      }
    }
    __syncwarp();
  } else if (warp == 1 && rank == 0) {
    if (elect_one()) {
      // One elected thread, so that operands of the matrix instructions are known
      // to be uniform: chosen as lane 0, with the descriptors computed for each
      // instruction, the thread needed 560 to 620 clocks a stage whatever the
      // tile (now 515 at 128 x 256, 305 at 128 x 128; the arithmetic takes 512
      // and 256).
      constexpr uint32_t kDesc = mma_desc(kTM, L::kColumns, kBMN), kLoDesc = mma_desc(kTM, BN, kBMN);
      constexpr uint32_t kStepA = 32 >> 4, kStepB = (kBMN ? 2048 : 32) >> 4;  // 16 k-values: along a row, or 16 rows
      const uint32_t first_a = smem_u32(smem), tmem = sh.tmem;
      const uint64_t desc_a = operand_desc(first_a, 16), desc_b = operand_desc(first_a + L::kA, kBMN ? 8192 : 16);
      bool go = true;
      for (int t = unit; go && t < total; t += units) {
        const int part = parts > 1 ? t % parts : 0, last = k_from(part + 1);
        for (int k = k_from(part); go && k < last; at.sum.advance()) {
          const uint32_t acc = tmem + at.sum.at * L::kColumns;
          if (!wait_or_give_up<true>(&sh.acc_empty[at.sum.at], at.sum.parity ^ 1u, &sh.given_up, g.limit)) {
            go = false;
            break;
          }
          tmem_fence_after();
          const int end = sum_end(k, last);
          bool add = false;
          for (; k < end; ++k) {
            const uint32_t st = at.stage.at;
            if (!wait_or_give_up<true>(&sh.full[st], at.stage.parity, &sh.given_up, g.limit)) {
              go = false;
              break;
            }
            tmem_fence_after();
            const uint64_t da = desc_a + st * (L::kStage >> 4), db = desc_b + st * (L::kStage >> 4);
            mma_f16<CG>(acc, da, db, kDesc, add);
            add = true;
#pragma unroll
            for (int q = 1; q < kTileK / 16; ++q) mma_f16<CG>(acc, da + q * kStepA, db + q * kStepB, kDesc, true);
            if constexpr (SPLIT) {
#pragma unroll
              for (int q = 0; q < kTileK / 16; ++q)
                mma_f16<CG>(acc + BN, da + (16384 >> 4) + q * kStepA, db + q * kStepB, kLoDesc, true);
            }
            mma_commit<CG>(&sh.empty[st]);
            at.stage.advance();
          }
          if (go) mma_commit<CG>(&sh.acc_full[at.sum.at]);
        }
      }
    }
    __syncwarp();
  } else if (warp >= 4) {
    const int quad = warp & 3, side = (warp - 4) >> 2;
    float *tile = reinterpret_cast<float *>(smem + kStages * L::kStage) + (warp - 4) * L::kStaging;
    const uint32_t tmem = sh.tmem + (uint32_t(quad * 32) << 16) + uint32_t(side * kBlocks * 32);
    bool go = true;
    auto take = [&] {  // the accumulator in turn is full; false: gave up
      go = __all_sync(0xffffffffu, wait_or_give_up<true>(&sh.acc_full[at.sum.at], at.sum.parity, &sh.given_up, g.limit));
      tmem_fence_after();
      return go;
    };
    auto give = [&] {
      tmem_fence_before();
      __syncwarp();
      if (lane == 0) {
        uint32_t bar = smem_u32(&sh.acc_empty[at.sum.at]);
        if constexpr (CG == 2) bar = mapa(bar, 0);
        mbar_arrive_cluster(bar);
      }
      at.sum.advance();
    };
    for (int t = unit; go && t < total; t += units) {
      const int zt = t / parts, z = zt / c.tiles, part = t - zt * parts;
      int row, col;
      tile_at<MODE, kTM, BN>(c, zt - z * c.tiles, row, col);
      const int r0 = row + int(rank) * 128 + quad * 32;
      float dr = 0.0f;
      if (MODE != kGram && r0 + lane < c.rows)
        dr = __ldcg((MODE == kSquare ? g.diag_a : g.diag_b) + int64_t(z) * g.diag_ld + r0 + lane);
      auto column = [&](int b) { return col + (side * kBlocks + b) * 32; };
      auto wanted = [&](int b) {
        return b < kBlocks && r0 < c.rows && column(b) < c.cols && (kBMN || column(b) <= r0);
      };
      BlockInput<MODE, OUT> input;
      auto ask = [&](int b) {
        if (wanted(b)) input.load(g, step, z, r0, column(b));
      };
      if constexpr (!SPLIT) ask(0);
      auto stage = [&](float *to, const float(&v)[32]) {
#pragma unroll
        for (int e = 0; e < 32; e += 4)
          *reinterpret_cast<float4 *>(to + tile_place(lane, e)) = make_float4(v[e], v[e + 1], v[e + 2], v[e + 3]);
      };
      auto finish = [&](int b) {
        finish_block<MODE, OUT>(g, step, tile, z, r0, column(b), dr, input, [&] { ask(b + 1); });
      };
      // in parts: this warp's place among the warps of all tiles, and its blocks
      const int64_t place = (int64_t(zt) * CG + rank) * kEpilogueWarps + warp - 4;
      const bool in_parts = MODE == kGram && parts > 1;
      if constexpr (SPLIT) {
        float v[32] = {};
        for (int k = k_from(part), last = k_from(part + 1); k < last; k = sum_end(k, last)) {
          if (!take()) break;
#pragma unroll
          for (int part_of = 0; part_of < 2; ++part_of) {  // hi hi, then hi lo + lo hi
            float f[32];
            tmem_load32(tmem + at.sum.at * L::kColumns + uint32_t(part_of * BN), f);
#pragma unroll
            for (int e = 0; e < 32; ++e) v[e] += f[e];
          }
          give();
        }
        if (!go) break;
        if (!wanted(0)) continue;
        __syncwarp();
        stage(tile, v);
        __syncwarp();
        if (in_parts) {
          leave_part(g, tile, place, part);
          if (!last_part(g, g.arrived + place)) continue;
          join_parts(g, tile, place);
        }
        ask(0);  // not earlier: the sums fill the registers
        finish(0);
      } else {
        if (!take()) break;
#pragma unroll 1
        for (int b = 0; b < kBlocks; ++b) {
          if (!wanted(b)) break;
          float v[32];
          __syncwarp();
          tmem_load32(tmem + at.sum.at * L::kColumns + uint32_t(b * 32), v);
          stage(tile, v);
          __syncwarp();
          if (in_parts) leave_part(g, tile, place * kBlocks + b, part);
          else finish(b);
        }
        give();
        if (in_parts && wanted(0) && last_part(g, g.arrived + place)) {
#pragma unroll 1
          for (int b = 0; b < kBlocks && wanted(b); ++b) {
            join_parts(g, tile, place * kBlocks + b);
            finish(b);
          }
        }
      }
    }
    asm volatile("fence.proxy.async.global;" ::: "memory");  // what this thread stored, for every block's TMA
  }
}

// All blocks have finished the product (their stores are visible to every
// block's loads); false: a wait gave up somewhere.
__device__ __forceinline__ bool grid_wait(uint32_t *barrier, uint32_t target, Shared &sh, long long limit) {
  __syncthreads();
  if (gridDim.x > 1) {
    if (threadIdx.x == 0) {
      asm volatile("red.release.gpu.global.add.u32 [%0], 1;" ::"l"(barrier) : "memory");
      const long long start = clock64();
      for (uint32_t n = 0;; ++n) {
        uint32_t seen;
        asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(seen) : "l"(barrier) : "memory");
        if (seen >= target) break;
        if (sh.given_up || n >= kWaitTries || clock64() - start > limit) {
          sh.given_up = 1u;
          break;
        }
      }
    }
    __syncthreads();
  }
  return sh.given_up == 0u;
}

// The whole iteration in one cooperative launch: 3 products a step, a barrier
// over the grid after each (about 2,500 clocks). One launch per product took 81
// us of host time and 10 us each at 1000 x 517; now a call takes 20 us of it.
// What bounds it: large sides the tensor cores at the power limit (4096 x 4096
// bf16 1,310 to 1,390 us in calls one after another, 1.0 PFLOP/s of the 1.37e12
// counted operations, 1,170 on a card that rested; of each product 70 of 85
// thousand clocks are instructions, the rest its last epilogue and the
// barrier); 1,000 the chain of a product's stages, epilogue and barrier, 12 to
// 20 thousand clocks, mostly latency (1000 x 517 fp32 151 us).
template <int CG, int BN, class OUT>
__global__ void __launch_bounds__(kThreads, 1) k_newton_schulz(const __grid_constant__ NsArgs g) {
  using L = Layout<CG, BN, !std::is_same_v<OUT, BF16>>;
  extern __shared__ uint8_t raw[];
  __shared__ Shared sh;
  uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  const int warp = int(threadIdx.x) >> 5;
  const uint32_t rank = CG == 2 ? cluster_rank() : 0u;
  if (threadIdx.x == 0) {
    for (int i = 0; i < L::kStages; ++i) {
      mbar_init(&sh.full[i], 1);
      mbar_init(&sh.empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sh.acc_full[i], 1);
      mbar_init(&sh.acc_empty[i], kEpilogueWarps * CG);
    }
    mbar_init(&sh.drained, 1);
    sh.given_up = 0u;
  }
  if (warp == 2) tmem_alloc<CG>(&sh.tmem, 2 * L::kColumns);
  tmem_fence_before();
  __syncthreads();
  if constexpr (CG == 2) cluster_sync_all();
  tmem_fence_after();

  Progress<L::kStages> at;
  uint32_t target = 0;
  for (int step = 0; step < g.steps; ++step) {
    run_product<kGram, CG, BN, OUT>(g, g.gram, step, sh, smem, rank, at);
    if (!grid_wait(g.barrier, target += gridDim.x, sh, g.limit)) break;
    run_product<kSquare, CG, BN, OUT>(g, g.square, step, sh, smem, rank, at);
    if (!grid_wait(g.barrier, target += gridDim.x, sh, g.limit)) break;
    if (step + 1 == g.steps && !g.fin.update) {
      run_product<kFinish, CG, BN, OUT>(g, g.apply, step, sh, smem, rank, at);
      break;
    }
    run_product<kApply, CG, BN, OUT>(g, g.apply, step, sh, smem, rank, at);
    if (step + 1 == g.steps) break;
    if (!grid_wait(g.barrier, target += gridDim.x, sh, g.limit)) break;
  }

  // No arrival or copy is outstanding when the CTA ends: the stages' last uses
  // have been read, or, where a wait gave up, the copies have landed and the
  // matrix instructions are done. Then that is reported.
  __syncthreads();
  const bool failed = sh.given_up != 0u;
  const uint32_t issued = __reduce_max_sync(0xffffffffu, at.loaded);
  const long long end = clock64() + kDrainClocks;
  if (warp == 0 && (!failed || rank == 0)) {
    for (uint32_t i = issued > L::kStages ? issued - L::kStages : 0; i < issued; ++i)
      wait_until(failed ? &sh.full[i % L::kStages] : &sh.empty[i % L::kStages], (i / L::kStages) & 1u, end);
  }
  if (failed) {
    // A pair's barrier counts the loads of both CTAs and completes no more where
    // they loaded different numbers of stages: they wait a hundred times a load's latency.
    while (CG == 2 && end - clock64() > kDrainClocks - 200000) {
    }
    if (warp == 1 && rank == 0) {
      if (elect_one()) {  // the thread that issued the instructions
        mma_commit<CG>(&sh.drained);
        wait_until(&sh.drained, 0u, end);
      }
      __syncwarp();
    }
    if (threadIdx.x == 0) {
      *reinterpret_cast<volatile uint32_t *>(g.failed) = 1u;
      *reinterpret_cast<volatile uint32_t *>(g.status) = 1u;
      __threadfence_system();
    }
  }
  tmem_fence_before();
  __syncthreads();
  if constexpr (CG == 2) cluster_sync_all();
  if (warp == 2) tmem_free<CG>(sh.tmem, 2 * L::kColumns);
}

// W <- keep W - rate O for O = (hi + lo) / S, a kernel of its own: the last
// product's epilogue would load and store 64-byte pieces of the weights' lines,
// and such a store waits long for its line when another piece of it is being
// loaded (8 x 1024 x 2048 bf16: that product took 152,000 to 203,000 clocks for
// 83,000 without weights; this kernel takes a quarter of the difference). Along
// the rows in vectors, or through shared memory in tiles of 64 x 64, as
// k_muon_scale. Bound by HBM (8 x 1024 x 2048 bf16 29 us, 4.7 TB/s). Where the
// products gave up, the weights stay as they were.
template <class W>
__global__ void __launch_bounds__(256)
k_muon_weights(const __half *__restrict__ hi, const __half *__restrict__ lo, int64_t ld, int64_t batch_stride, int64_t m,
               int64_t n, int vec, FinishArgs f, const uint32_t *__restrict__ failed) {
  __shared__ float tile[64][65];
  using T = typename W::T;
  const int64_t z = blockIdx.z;
  T *w = static_cast<T *>(f.out) + z * f.batch;
  hi += z * batch_stride;
  lo += z * batch_stride;
  const float rate = f.rate * (1.0f / kScale);
  pdl_wait();
  if (__ldcg(failed) != 0u) return;
  auto open = [&](int64_t at, float (&o)[8]) {  // eight values of O, not yet divided by S
    const uint4 h = *reinterpret_cast<const uint4 *>(hi + at), l = *reinterpret_cast<const uint4 *>(lo + at);
    const __half2 *hh = reinterpret_cast<const __half2 *>(&h), *ll = reinterpret_cast<const __half2 *>(&l);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float2 x = __half22float2(hh[e]), y = __half22float2(ll[e]);
      o[2 * e] = x.x + y.x;
      o[2 * e + 1] = x.y + y.y;
    }
  };
  if (vec && !f.transposed) {
    int shift = 0;
    while (shift < 8 && (int64_t(8) << shift) < n) ++shift;
    const int lanes = 1 << shift, sub = threadIdx.x & (lanes - 1);
    const int64_t each = blockDim.x >> shift;
    for (int64_t i = blockIdx.x * each + (threadIdx.x >> shift); i < m; i += gridDim.x * each) {
#pragma unroll 2
      for (int64_t j = sub * 8; j < n; j += lanes * 8) {
        float o[8], old[8];
        open(i * ld + j, o);
        T *at = w + i * f.row + j;
        load_eight<W>(at, true, 1, 8, old);
        constexpr int kPer = 16 / sizeof(T);
        uint4 raw[8 / kPer];
        T *v = reinterpret_cast<T *>(raw);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = W::store(__fmaf_rn(-rate, o[e], f.keep * old[e]));
#pragma unroll
        for (int e = 0; e < 8 / kPer; ++e) reinterpret_cast<uint4 *>(at)[e] = raw[e];
      }
    }
    return;
  }
  // tiles of W; X is read along its own rows
  const int row = threadIdx.x >> 3, eight = (threadIdx.x & 7) * 8;
  const int64_t tiles_j = (n + 63) / 64, tiles = tiles_j * ((m + 63) / 64);
  for (int64_t t = blockIdx.x; t < tiles; t += gridDim.x) {
    const int64_t i0 = t / tiles_j * 64, j0 = (t - t / tiles_j * tiles_j) * 64;
    const int64_t r0 = f.transposed ? j0 : i0, c0 = f.transposed ? i0 : j0, rows = f.transposed ? n : m;
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const int r = row + 32 * q;
      float o[8] = {};
      if (r0 + r < rows) open((r0 + r) * ld + c0 + eight, o);  // X's storage reaches past its columns to a multiple of 64
#pragma unroll
      for (int e = 0; e < 8; ++e) tile[r][eight + e] = o[e];
    }
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    float old[8][2];  // all loads before the first store
#pragma unroll
    for (int q = 0; q < 8; ++q) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int64_t i = i0 + warp + 8 * q, j = j0 + lane + 32 * h;
        old[q][h] = i < m && j < n ? W::load(w[i * f.row + j]) : 0.0f;
      }
    }
    __syncthreads();
#pragma unroll
    for (int q = 0; q < 8; ++q) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int i = warp + 8 * q, j = lane + 32 * h;
        if (i0 + i < m && j0 + j < n)
          w[(i0 + i) * f.row + j0 + j] = W::store(__fmaf_rn(-rate, f.transposed ? tile[j][i] : tile[i][j], f.keep * old[q][h]));
      }
    }
    __syncthreads();
  }
}

// ---------------------------------------------------------------------------
// Small matrices: one CTA each, everything on chip
// ---------------------------------------------------------------------------

constexpr int kSmallSide = 128, kSmallWide = 256;  // the largest s and w of the kernel below
constexpr int kSmallTile = 128 * 128;              // bytes: 128 rows of 64 values
constexpr bool on_chip(int64_t s, int64_t w) { return s <= kSmallSide && w <= kSmallWide; }

// Place (in values) of (r, c) in a matrix of 64-column tiles of 128 rows with
// 128-byte swizzle: what the matrix instructions read, K-major as rows of
// columns, or MN-major as rows of k.
__device__ __forceinline__ int small_place(int r, int c) {
  return (c >> 6) * (kSmallTile / 2) + r * 64 + ((((c >> 3) ^ r) & 7) << 3) + (c & 7);
}

__device__ __forceinline__ void open_eight(const uint4 &v, float (&f)[8]) {
  const __half2 *h = reinterpret_cast<const __half2 *>(&v);
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float2 t = __half22float2(h[e]);
    f[2 * e] = t.x;
    f[2 * e + 1] = t.y;
  }
}

// The whole call for a matrix with s <= 128 and w <= 128 (SIDES = 4) or 256
// (SIDES = 2): momentum, norm, all products and the result in one CTA. A thread
// owns every SIDES-th block of 32 columns of a row: its values of X and of A
// stay in its registers in fp32, and only their f16 operand parts go to shared
// memory, in the layout of the matrix instructions (X serves as a K-major
// operand of X X^T and, the same bytes, as the MN-major one of B X). Between two products there is only a
// barrier of the CTA, where the kernel for large matrices passes through L2
// and a barrier of the grid (128 x 64 bf16: 64 us there with its launches, 24 us
// here; 128 x 256 43 us, 64 matrices of 64 x 64 19 us).
// Bound by the instructions of one SM and the latency of 3 products a step;
// with X and A in shared memory as f16 pairs, unpacked and packed again in
// every epilogue, it took 33 us at 128 x 64 and 70 at 128 x 256.
//
// SPLIT: hi hi into one accumulator (at most 16 instructions, as between two
// flushes there), the lo products into another, 2^-11 of it in size, whose cut
// sums do not matter.
template <class V, class W, bool MOM, int SIDES>
__global__ void __launch_bounds__(128 * SIDES)
k_newton_schulz_small(UpdateArgs a, int s, int w, int transposed, int steps, float eps, FinishArgs fin,
                      uint32_t tmem_columns, long long limit, uint32_t *status) {
  constexpr bool SPLIT = !std::is_same_v<W, BF16>;  // as split_products says
  constexpr int kThreads = 128 * SIDES, kWarps = 4 * SIDES;
  constexpr int kX = SIDES == 2 ? 4 : 1, kA = 4 / SIDES;  // blocks of X and of A that a thread owns
  extern __shared__ uint8_t raw[];
  __shared__ __align__(16) float diag[kSmallSide];
  __shared__ double red[kWarps];
  __shared__ Factor factor;
  __shared__ uint64_t done;
  __shared__ uint32_t tmem_base;
  __shared__ volatile uint32_t given_up;
  __half *xh = reinterpret_cast<__half *>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  const int xtiles = (w + 63) >> 6, stiles = (s + 63) >> 6;
  __half *xl = xh + xtiles * (kSmallTile / 2), *ah = xl + xtiles * (kSmallTile / 2), *al = ah + stiles * (kSmallTile / 2);
  const int tid = int(threadIdx.x), warp = tid >> 5, lane = tid & 31;
  const int64_t z = blockIdx.x;

  if (tid == 0) {
    mbar_init(&done, 1);
    given_up = 0u;
  }
  if (warp == 0) tmem_alloc<1>(&tmem_base, tmem_columns);
  {
    const int n16 = (2 * xtiles + (SPLIT ? 2 : 1) * stiles) * (kSmallTile / 16);
    for (int i = tid; i < n16; i += kThreads) reinterpret_cast<uint4 *>(xh)[i] = make_uint4(0u, 0u, 0u, 0u);
  }
  if (tid < kSmallSide) diag[tid] = 0.0f;

  // U, its norm, X_0: eight values of a row per thread, a power of two of threads per row
  const int m = int(a.m), n = int(a.n);
  int shift = 0;
  while ((8 << shift) < n) ++shift;
  const int i0 = tid >> shift, rows = kThreads >> shift, j = (tid & ((1 << shift) - 1)) * 8, count = max(0, min(8, n - j));
  auto load_update = [&](int i, float (&u)[8], float (&mom)[8]) {
    load_eight<V>(static_cast<const typename V::T *>(a.grad.p) + z * a.grad.batch + i * a.grad.row + j, a.vec, 1, count, u);
    if constexpr (MOM)
      load_eight<F32>(static_cast<const float *>(a.momentum.p) + z * a.momentum.batch + i * a.momentum.row + j, a.vec, 1,
                      count, mom);
  };
  double sum = 0.0;
  bool unsafe = false;
#pragma unroll 2
  for (int i = i0; i < m; i += rows) {
    float u[8], mom[8];
    load_update(i, u, mom);
    if constexpr (MOM) {
      float *mp = const_cast<float *>(static_cast<const float *>(a.momentum.p)) + z * a.momentum.batch + i * a.momentum.row + j;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        mom[e] = __fmaf_rn(a.beta, mom[e], u[e]);
        u[e] = update_of(a, u[e], mom[e]);
      }
      if (a.vec) {
        if (count > 0) {
          reinterpret_cast<float4 *>(mp)[0] = make_float4(mom[0], mom[1], mom[2], mom[3]);
          reinterpret_cast<float4 *>(mp)[1] = make_float4(mom[4], mom[5], mom[6], mom[7]);
        }
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (e < count) mp[e] = mom[e];
      }
    }
    unsafe |= square_sum(u, sum);
  }
  if (__syncthreads_or(unsafe)) {
    sum = 0.0;
    for (int i = i0; i < m; i += rows) {
      float u[8], mom[8];
      load_update(i, u, mom);
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if constexpr (MOM) u[e] = update_of(a, u[e], mom[e]);
      wide_square_sum(u, sum);
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (lane == 0) red[warp] = sum;
  __syncthreads();
  if (tid == 0) {
    sum = 0.0;
#pragma unroll
    for (int i = 0; i < kWarps; ++i) sum += red[i];
    factor = update_factor(sum, eps);
  }
  tmem_fence_before();
  __syncthreads();
  tmem_fence_after();
  const uint32_t tmem = tmem_base;
  const Factor k0 = factor;
#pragma unroll 2
  for (int i = i0; i < m; i += rows) {
    float u[8], mom[8];
    load_update(i, u, mom);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if constexpr (MOM) u[e] = update_of(a, u[e], mom[e]);
      u[e] = e < count ? k0.times(u[e]) : 0.0f;
    }
    if (!transposed) {
      if (count > 0) put_eight(xh + small_place(i, j), xl + small_place(i, j), u);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if (e < count) {
          const __half h = __float2half_rn(u[e]);
          xh[small_place(j + e, i)] = h;
          xl[small_place(j + e, i)] = __float2half_rn(u[e] - __half2float(h));
        }
      }
    }
  }

  // A product: the operands written so far become visible to the tensor core,
  // one thread issues its instructions, all wait. False: gave up.
  const uint32_t sx = smem_u32(xh), sxl = smem_u32(xl), sa = smem_u32(ah), sal = smem_u32(al);
  uint32_t parity = 0;
  auto multiply = [&](uint32_t pa, uint32_t pal, uint32_t pb, uint32_t pbl, bool b_mn, int width, int depth) {
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    tmem_fence_before();
    __syncthreads();
    if (warp == 0 && elect_one()) {
      tmem_fence_after();
      const int wide = (width + 15) & ~15, chunks = (depth + 15) >> 4;
      const uint32_t desc = mma_desc(128, wide, b_mn);
      const uint32_t extra = tmem + tmem_columns / 2;  // the lo products' accumulator
      auto go = [&](uint32_t acc, uint32_t x, uint32_t y, bool add) {
        const uint64_t da = operand_desc(x, 16), db = operand_desc(y, b_mn ? kSmallTile : 16);
        for (int q = 0; q < chunks; ++q) {
          const uint32_t along = (q >> 2) * (kSmallTile >> 4) + (q & 3) * (32 >> 4);
          mma_f16<1>(acc, da + along, db + (b_mn ? q * (2048 >> 4) : along), desc, add || q > 0);
        }
      };
      go(tmem, pa, pb, false);
      if constexpr (SPLIT) {
        go(extra, pa, pbl, false);
        go(extra, pal, pb, true);
      }
      mma_commit<1>(&done);
    }
    __syncwarp();
    const bool ok = wait_or_give_up<false>(&done, parity, &given_up, limit);
    parity ^= 1u;
    const bool all = __syncthreads_and(ok) != 0;
    tmem_fence_after();
    return all;
  };
  const int quad = warp & 3, side = warp >> 2, r = quad * 32 + lane;
  const bool mine = quad * 32 < s;  // rows beyond s hold zeros throughout
  const int s16 = (s + 15) & ~15, w16 = (w + 15) & ~15;
  auto column = [&](int b) { return (b * SIDES + side) * 32; };
  auto sums = [&](int c0, float (&v)[32]) {
    __syncwarp();
    tmem_load32(tmem + (uint32_t(quad * 32) << 16) + uint32_t(c0), v);
    if constexpr (SPLIT) {
      float l[32];
      tmem_load32(tmem + (uint32_t(quad * 32) << 16) + tmem_columns / 2 + uint32_t(c0), l);
#pragma unroll
      for (int e = 0; e < 32; ++e) v[e] += l[e];
    }
  };
  // a block of the thread's row as operand parts, as far as the products' widths reach
  auto put_block = [&](__half *hi, __half *lo, int c0, int end, const float (&f)[32]) {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      if (c0 + 8 * q < end) {
        const int at = small_place(r, c0 + 8 * q);
        uint4 h;
        __half2 *hh = reinterpret_cast<__half2 *>(&h);
#pragma unroll
        for (int e = 0; e < 4; ++e) hh[e] = __floats2half2_rn(f[8 * q + 2 * e], f[8 * q + 2 * e + 1]);
        *reinterpret_cast<uint4 *>(hi + at) = h;
        if constexpr (SPLIT) {
          uint4 l;
          __half2 *ll = reinterpret_cast<__half2 *>(&l);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float2 back = __half22float2(hh[e]);
            ll[e] = __floats2half2_rn(f[8 * q + 2 * e] - back.x, f[8 * q + 2 * e + 1] - back.y);
          }
          *reinterpret_cast<uint4 *>(lo + at) = l;
        }
      }
    }
  };

  // this lane's element of a diagonal block, which becomes zero
  auto on_diagonal = [&](float (&f)[32]) {
    float d = 0.0f;
#pragma unroll
    for (int e = 0; e < 32; ++e) {
      d = e == lane ? f[e] : d;
      f[e] = e == lane ? 0.0f : f[e];
    }
    return d;
  };

  float x[kX][32], o[kA][32];
  __syncthreads();
#pragma unroll
  for (int b = 0; b < kX; ++b) {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      float h[8] = {}, l[8] = {};
      if (mine && column(b) + 8 * q < w16) {
        const int at = small_place(r, column(b) + 8 * q);
        open_eight(*reinterpret_cast<const uint4 *>(xh + at), h);
        open_eight(*reinterpret_cast<const uint4 *>(xl + at), l);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) x[b][8 * q + e] = h[e] + l[e];
    }
  }

  bool ok = true;
  for (int step = 0; step < steps; ++step) {
    // A = X X^T, its diagonal D apart: off it, O
    if (!(ok = multiply(sx, sxl, sx, sxl, false, s, w))) break;
    if (mine) {
#pragma unroll
      for (int b = 0; b < kA; ++b) {
        const int c0 = column(b);
        if (c0 >= s) break;
        sums(c0, o[b]);
#pragma unroll
        for (int e = 0; e < 32; ++e) o[b][e] *= 1.0f / kScale;
        if (c0 == quad * 32) {
          const float d = on_diagonal(o[b]);
          if (r < s) diag[r] = d;
        }
        put_block(ah, al, c0, s16, o[b]);
      }
    }
    // B = b A + c A A, in A's place: (A A)_rc = (O O)_rc + (D_r + D_c) O_rc, on the diagonal (O O)_rr + D_r^2
    if (!(ok = multiply(sa, sal, sa, sal, false, s, s))) break;
    float k = kNsA;
    if (mine) {
      const float dr = diag[r];
#pragma unroll
      for (int b = 0; b < kA; ++b) {
        const int c0 = column(b);
        if (c0 >= s) break;
        float v[32];
        sums(c0, v);
        if (c0 == quad * 32)
          k = __fmaf_rn(kNsC / kScale, __fmaf_rn(dr, dr, on_diagonal(v)), kNsB * dr) * (1.0f / kScale);
#pragma unroll
        for (int e = 0; e < 32; e += 4) {
          const float4 dc = *reinterpret_cast<const float4 *>(diag + c0 + e);
          v[e] = __fmaf_rn(kNsC / kScale, __fmaf_rn(dr + dc.x, o[b][e], v[e]), kNsB * o[b][e]);
          v[e + 1] = __fmaf_rn(kNsC / kScale, __fmaf_rn(dr + dc.y, o[b][e + 1], v[e + 1]), kNsB * o[b][e + 1]);
          v[e + 2] = __fmaf_rn(kNsC / kScale, __fmaf_rn(dr + dc.z, o[b][e + 2], v[e + 2]), kNsB * o[b][e + 2]);
          v[e + 3] = __fmaf_rn(kNsC / kScale, __fmaf_rn(dr + dc.w, o[b][e + 3], v[e + 3]), kNsB * o[b][e + 3]);
        }
        if (c0 == quad * 32) on_diagonal(v);
        put_block(ah, al, c0, s16, v);
      }
    }
    __syncthreads();  // every thread has read D: B's diagonal takes its place
    if (mine && quad % SIDES == side && r < s) diag[r] = k;  // the warp whose block holds these rows' diagonal
    // X = (a + diag B) X + B X
    if (!(ok = multiply(sa, sal, sx, sxl, true, w, s))) break;
    if (mine) {
      k = kNsA + diag[r];
#pragma unroll
      for (int b = 0; b < kX; ++b) {
        const int c0 = column(b);
        if (c0 >= w) break;
        float v[32];
        sums(c0, v);
#pragma unroll
        for (int e = 0; e < 32; ++e) x[b][e] = __fmaf_rn(k, x[b][e], v[e] * (1.0f / kScale));
        put_block(xh, xl, c0, w16, x[b]);
      }
    }
  }
  __syncthreads();
  if (!ok) {
    if (tid == 0) {
      wait_until(&done, parity ^ 1u, clock64() + kDrainClocks);
      *reinterpret_cast<volatile uint32_t *>(status) = 1u;
      __threadfence_system();
    }
  } else {
    // O through shared memory (X's operands are no longer needed), then in the call's own order
    float *out = reinterpret_cast<float *>(xh);
    const int ld = xtiles * 64;
    auto place = [&](int rr, int c) { return rr * ld + ((((c >> 2) ^ rr) & 7) << 2 | (c & 3)) + (c & ~31); };
    if (mine) {
#pragma unroll
      for (int b = 0; b < kX; ++b) {
        if (column(b) >= w) break;
#pragma unroll
        for (int e = 0; e < 32; e += 4)
          *reinterpret_cast<float4 *>(out + place(r, column(b) + e)) =
              make_float4(x[b][e], x[b][e + 1], x[b][e + 2], x[b][e + 3]);
      }
    }
    __syncthreads();
    typename W::T *to = static_cast<typename W::T *>(fin.out) + z * fin.batch;
    for (int i = warp; i < m; i += kWarps) {
#pragma unroll 2
      for (int c = lane; c < n; c += 32) {
        typename W::T *at = to + int64_t(i) * fin.row + c;
        float f = out[transposed ? place(c, i) : place(i, c)] * (1.0f / kScale);
        if constexpr (MOM) f = __fmaf_rn(-fin.rate, f, fin.keep * W::load(*at));
        *at = W::store(f);
      }
    }
  }
  tmem_fence_before();
  __syncthreads();
  if (warp == 0) tmem_free<1>(tmem, tmem_columns);
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------

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

// Boxes of 64 x 64 of a batch of rows x cols f16 matrices.
CUtensorMap matrix_map(const __half *p, int64_t rows, int64_t cols, int64_t ld, int64_t batch) {
  CUtensorMap map;
  const cuuint64_t dims[3] = {cuuint64_t(cols), cuuint64_t(rows), cuuint64_t(batch)};
  const cuuint64_t strides[2] = {cuuint64_t(ld) * 2, cuuint64_t(ld) * 2 * cuuint64_t(rows)};
  const cuuint32_t boxes[3] = {64, 64, 1}, steps[3] = {1, 1, 1};
  const CUresult r = encode_tiled()(&map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<__half *>(p), dims, strides,
                                    boxes, steps, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                                    CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) throw Error(SE_ERR_CUDA, "cuTensorMapEncodeTiled: error " + std::to_string(int(r)));
  return map;
}

// A type argument, its flag taken off, and whether the products are full.
struct ResultType {
  int32_t type;
  bool split;
};
ResultType result_type(int32_t t, const char *what) {
  const int32_t type = t & ~SE_FULL_PRODUCTS;
  check_value_dtype(type, what);
  return {type, t != SE_BFLOAT16};
}
template <class F> void dispatch_result(int32_t type, bool split, F &&f) {
  if (type == SE_BFLOAT16 && split) f(BF16Full{});
  else dispatch_value(type, f);
}

int64_t tile_count(bool symmetric, int64_t rows, int64_t cols, int tm, int bn) {
  const int64_t ti = (rows + tm - 1) / tm, tj = (cols + bn - 1) / bn;
  if (!symmetric) return ti * tj;
  int64_t n = 0;
  for (int64_t i = 0; i < ti; ++i) n += std::min<int64_t>((i * tm + tm - 1) / bn + 1, tj);
  return n;
}

// The tile of a call (the same for its three products): 128 cg x bn, cg = 2 by
// a pair of blocks; and in how many parts the k-values of X X^T are cut.
constexpr int kUnits = 148;  // blocks that run at once
struct Plan {
  int cg, bn, parts;
};

// The form with the least estimated time of a step. A product takes, for each
// round of tiles over the units, its k-blocks times the clocks of a stage, and
// at its end the last epilogue and the barrier. Both were measured for each
// form (clocks) and are rounded here; the estimate mostly orders the forms as
// their times do, e.g. bf16 (us) at 4096 x 4096 1x64 2341, 1x128 1534, 1x256
// 1384, 2x128 1356, 2x256 1344; at 2048 x 2048 300, 245, 331, 236, 331; at 1024 x
// 1024 111, 145, 218, 147, 218. Three products have one form, and only their
// parts are chosen. (kUnits, not the device's multiprocessors: the workspace is
// asked for without a device, and a launch never takes more blocks than run at once.)
Plan plan_for(int64_t batch, int64_t s, int64_t w, bool split) {
  struct Form {
    int cg, bn, stage, end;
  };
  constexpr Form single[] = {{1, 64, 330, 8000}, {1, 128, 420, 11000}, {2, 128, 400, 11000}, {1, 256, 600, 20000}, {2, 256, 560, 20000}};
  constexpr Form three[] = {{1, 64, 650, 12000}};
  constexpr int kJoin = 8000;  // clocks to add up parts
  Plan best{};
  int64_t least = 0;
  for (const Form *at = split ? three : single, *last = split ? std::end(three) : std::end(single); at != last; ++at) {
    const Form &f = *at;
    const int64_t stage = f.stage, units = kUnits / f.cg;
    auto rounds = [&](int64_t tiles) { return (tiles + units - 1) / units; };
    const int64_t sym = tile_count(true, s, s, 128 * f.cg, f.bn) * batch;
    const int64_t app = tile_count(false, s, w, 128 * f.cg, f.bn) * batch;
    const int64_t kw = (w + kTileK - 1) / kTileK, ks = (s + kTileK - 1) / kTileK;
    // a part saves stages, of at least 5,000 clocks each
    const int64_t parts =
        kw * stage < 2 * kJoin ? 1 : std::max<int64_t>(1, std::min<int64_t>(units / sym, kw * stage / 5000));
    const int64_t clocks = (rounds(sym * parts) * ((kw + parts - 1) / parts) + rounds(sym) * ks + rounds(app) * ks) * stage +
                           (parts > 1 ? kJoin : 0) + 3 * f.end;
    if (least == 0 || clocks < least) {
      least = clocks;
      best = Plan{f.cg, f.bn, int(parts)};
    }
  }
  return best;
}

// The workspace of a call: X twice (a product reads one and writes the other),
// A, B, their diagonals, the partial norms, the partial sums of X X^T, and the
// counters (zeroed by the first kernel).
struct Space {
  double *norms;
  Pair x[2], a, b;
  float *diag_a, *diag_b, *partial;
  uint32_t *counters;  // the barrier, the failure word, then one per block of X X^T
  int64_t ncounters;
  size_t bytes;
};

Space muon_space(void *base, int64_t batch, int64_t s, int64_t w, bool split) {
  const Plan p = plan_for(batch, s, w, split);
  Space sp{};
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t here = at;
    at += (bytes + 255) & ~size_t(255);
    return static_cast<uint8_t *>(base) + here;
  };
  const int64_t ldx = (w + 63) / 64 * 64, lda = (s + 63) / 64 * 64;
  auto pair = [&](int64_t ld, bool lo) {
    Pair q{};
    q.ld = ld;
    q.batch = s * ld;
    q.hi = reinterpret_cast<__half *>(take(size_t(batch) * s * ld * 2));
    q.lo = lo ? reinterpret_cast<__half *>(take(size_t(batch) * s * ld * 2)) : q.hi;
    return q;
  };
  sp.norms = reinterpret_cast<double *>(take(size_t(batch) * kNormParts * sizeof(double)));
  sp.x[0] = pair(ldx, true);
  sp.x[1] = pair(ldx, true);
  sp.a = pair(lda, split);
  sp.b = pair(lda, split);
  sp.diag_a = reinterpret_cast<float *>(take(size_t(batch) * lda * sizeof(float)));
  sp.diag_b = reinterpret_cast<float *>(take(size_t(batch) * lda * sizeof(float)));
  const int64_t values = p.parts > 1 ? tile_count(true, s, s, 128 * p.cg, p.bn) * batch * 128 * p.cg * p.bn : 0;
  sp.partial = reinterpret_cast<float *>(take(size_t(values) * p.parts * sizeof(float)));
  sp.ncounters = 2 + values / 1024;  // (at least one per warp of a tile)
  sp.counters = reinterpret_cast<uint32_t *>(take(size_t(sp.ncounters) * sizeof(uint32_t)));
  sp.bytes = at;
  return sp;
}

// Pairs of blocks that run at once (asked once per device and kernel).
template <class... KArgs>
int64_t resident_clusters(void (*kernel)(KArgs...), int device, const cudaLaunchConfig_t &cfg) {
  static std::mutex mu;
  static std::map<std::pair<const void *, int>, int> known;
  const auto key = std::make_pair(reinterpret_cast<const void *>(kernel), device);
  std::lock_guard<std::mutex> lock(mu);
  auto it = known.find(key);
  if (it != known.end()) return it->second;
  cudaLaunchConfig_t ask = cfg;
  cudaLaunchAttribute cluster = cfg.attrs[1];
  ask.attrs = &cluster;
  ask.numAttrs = 1;
  int n = 0;
  cuda_check(cudaOccupancyMaxActiveClusters(&n, kernel, &ask), "cluster occupancy");
  if (n < 1) throw Error(SE_ERR_CUDA, "no pair of blocks fits the device");
  return known[key] = n;
}

// A kernel of 256 threads that waits (pdl_wait) for the one before it.
template <class... KArgs, class... Args>
void launch_after(void (*kernel)(KArgs...), dim3 grid, cudaStream_t st, Args... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(256);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cuda_check(cudaLaunchKernelEx(&cfg, kernel, args...), "cudaLaunchKernelEx");
}

template <int CG, int BN, class OUT>
void launch_newton_schulz(const NsArgs &g, int64_t units, int device, cudaStream_t st) {
  const int sms = sm_count(device);
  using L = Layout<CG, BN, !std::is_same_v<OUT, BF16>>;
  auto *kernel = k_newton_schulz<CG, BN, OUT>;
  allow_dynamic_smem(kernel, L::kBytes);
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(unsigned(sms / CG * CG));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = L::kBytes;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeCooperative;  // the blocks wait for one another
  attr[0].val.cooperative = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = CG;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = CG == 2 ? 2 : 1;
  const int64_t at_once = CG == 2 ? resident_clusters(kernel, device, cfg) : sms;
  cfg.gridDim = dim3(unsigned(std::min(units, at_once) * CG));
  cuda_check(cudaLaunchKernelEx(&cfg, kernel, g), "k_newton_schulz");
  launched("k_newton_schulz");
}

// The orthogonalised update of `u` into `fin`.
void orthogonalise(UpdateArgs u, int grad_type, int64_t batch, int steps, float eps, bool split, FinishArgs fin, void *workspace,
                   size_t workspace_bytes, int device, cudaStream_t st) {
  const size_t gb = value_bytes(grad_type);
  u.vec = u.n % 8 == 0 && aligned16(u.grad.p) && u.grad.row * gb % 16 == 0 && (batch == 1 || u.grad.batch * gb % 16 == 0) &&
          (u.momentum.p == nullptr ||
           (aligned16(u.momentum.p) && u.momentum.row % 4 == 0 && (batch == 1 || u.momentum.batch % 4 == 0)));
  const bool transposed = u.m > u.n;
  const int64_t s = std::min(u.m, u.n), w = std::max(u.m, u.n);
  NsArgs g{};
  g.status = WaitWords::get().of(device, st);
  g.limit = wait_limit();
  fin.transposed = transposed;
  const size_t ob = value_bytes(fin.type);
  fin.vec = u.n % 4 == 0 && reinterpret_cast<uintptr_t>(fin.out) % (4 * ob) == 0 && fin.row % 4 == 0 &&
            (batch == 1 || fin.batch % 4 == 0);
  if (on_chip(s, w)) {
    const int xtiles = int((w + 63) / 64), stiles = int((s + 63) / 64);
    const size_t smem = size_t(2 * xtiles + (split ? 2 : 1) * stiles) * kSmallTile + 1024;
    const uint32_t columns = (w > 128 ? 256 : 128) * (split ? 2 : 1);
    auto launch = [&](auto grad, auto out, auto mom) {
      auto start = [&](auto sides) {
        auto *kernel = k_newton_schulz_small<decltype(grad), decltype(out), decltype(mom)::value, decltype(sides)::value>;
        allow_dynamic_smem(kernel, smem);
        kernel<<<unsigned(batch), 128 * decltype(sides)::value, smem, st>>>(u, int(s), int(w), int(transposed), steps, eps,
                                                                            fin, columns, g.limit, g.status);
      };
      if (w > 128) start(std::integral_constant<int, 2>{});
      else start(std::integral_constant<int, 4>{});
    };
    dispatch_result(fin.type, split, [&](auto out) {
      using Grad = std::conditional_t<std::is_same_v<decltype(out), BF16Full>, BF16, decltype(out)>;
      if (!fin.update) launch(Grad{}, out, std::false_type{});  // an update and its result have one type
      else if (grad_type == fin.type) launch(Grad{}, out, std::true_type{});
      else launch(F32{}, out, std::true_type{});
    });
    launched("k_newton_schulz_small");
    return;
  }
  check_device_ptr(workspace, device, "workspace");
  if (reinterpret_cast<uintptr_t>(workspace) % 256 != 0) throw std::invalid_argument("workspace must be 256-byte aligned");
  const Plan plan = plan_for(batch, s, w, split);
  const Space sp = muon_space(workspace, batch, s, w, split);
  if (workspace_bytes < sp.bytes) throw std::invalid_argument("workspace is smaller than se_muon_workspace asks for");
  const int tm = 128 * plan.cg;
  auto cut = [&](bool symmetric, int64_t cols, int64_t depth, int parts) {
    const int64_t tiles = tile_count(symmetric, s, cols, tm, plan.bn);
    if (tiles * parts * batch > 0x7fffffff) throw std::invalid_argument("batch x m x n is too large");
    return Cut{int(s), int(cols), int((depth + kTileK - 1) / kTileK), int((cols + plan.bn - 1) / plan.bn), int(tiles), parts};
  };
  g.gram = cut(true, s, w, plan.parts);
  g.square = cut(true, s, s, 1);
  g.apply = cut(false, w, s, 1);
  const int sms = sm_count(device);
  const bool dense = u.grad.row == u.n && (u.momentum.p == nullptr || u.momentum.row == u.n);
  const int64_t spans = dense ? (u.m * u.n + kSpan - 1) / kSpan : u.m * ((u.n + kSpan - 1) / kSpan);
  const int nparts = int(std::min<int64_t>(std::min<int64_t>(kNormParts, spans), std::max<int64_t>(1, 4 * sms / batch)));
  const int64_t tiles64 = ((u.m + 63) / 64) * ((u.n + 63) / 64);
  dispatch_value(grad_type, [&](auto tag) {
    using V = decltype(tag);
    auto go = [&](auto mom) {
      constexpr bool kMom = decltype(mom)::value;
      k_muon_momentum<V, kMom><<<dim3(unsigned(nparts), unsigned(batch)), 256, 0, st>>>(u, sp.norms, sp.counters, sp.ncounters);
      launched("k_muon_momentum");
      launch_after(k_muon_scale<V, kMom>, dim3(unsigned(std::min<int64_t>(tiles64, 8 * sms)), 1, unsigned(batch)), st, u,
                   static_cast<const double *>(sp.norms), nparts, eps, transposed, sp.x[0].hi, sp.x[0].lo, sp.x[0].ld,
                   sp.x[0].batch);
      launched("k_muon_scale");
    };
    if (u.momentum.p) go(std::true_type{});
    else go(std::false_type{});
  });

  for (int k = 0; k < 2; ++k) {
    g.x[k] = sp.x[k];
    g.x_hi[k] = matrix_map(sp.x[k].hi, s, w, sp.x[k].ld, batch);
    if (split) g.x_lo[k] = matrix_map(sp.x[k].lo, s, w, sp.x[k].ld, batch);
  }
  g.a = sp.a;
  g.b = sp.b;
  g.a_hi = matrix_map(sp.a.hi, s, s, sp.a.ld, batch);
  g.b_hi = matrix_map(sp.b.hi, s, s, sp.b.ld, batch);
  if (split) {
    g.a_lo = matrix_map(sp.a.lo, s, s, sp.a.ld, batch);
    g.b_lo = matrix_map(sp.b.lo, s, s, sp.b.ld, batch);
  }
  g.batch = int(batch);
  g.steps = steps;
  g.diag_a = sp.diag_a;
  g.diag_b = sp.diag_b;
  g.diag_ld = sp.a.ld;
  g.partial = sp.partial;
  g.barrier = sp.counters;
  g.failed = sp.counters + 1;
  g.arrived = sp.counters + 2;
  g.fin = fin;
  const int64_t units = std::max<int64_t>(int64_t(g.gram.tiles) * plan.parts, g.apply.tiles) * batch;
  const int form = plan.cg * 1000 + plan.bn;
  dispatch_result(fin.type, split, [&](auto out) {
    using OUT = decltype(out);
    if constexpr (std::is_same_v<OUT, BF16>) {  // wider tiles: single products only
      switch (form) {
        case 1128: return launch_newton_schulz<1, 128, OUT>(g, units, device, st);
        case 2128: return launch_newton_schulz<2, 128, OUT>(g, units, device, st);
        case 1256: return launch_newton_schulz<1, 256, OUT>(g, units, device, st);
        case 2256: return launch_newton_schulz<2, 256, OUT>(g, units, device, st);
        default: break;
      }
    }
    launch_newton_schulz<1, 64, OUT>(g, units, device, st);
  });
  if (!fin.update) return;
  dispatch_value(fin.type, [&](auto out) {
    const Pair &o = sp.x[steps & 1];
    const int vec = u.n % 8 == 0 && aligned16(fin.out) && fin.row * ob % 16 == 0 && (batch == 1 || fin.batch * ob % 16 == 0);
    const int64_t blocks = vec && !transposed ? (u.m * ((u.n + 7) / 8) + 255) / 256 : tiles64;
    launch_after(k_muon_weights<decltype(out)>, dim3(unsigned(std::min<int64_t>(blocks, 8 * sms)), 1, unsigned(batch)), st,
                 static_cast<const __half *>(o.hi), static_cast<const __half *>(o.lo), o.ld, o.batch, u.m, u.n, vec, fin,
                 static_cast<const uint32_t *>(g.failed));
  });
  launched("k_muon_weights");
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
    const ResultType out = result_type(out_dtype, "out_dtype");
    check_matrices(batch, m, n, 1, 0.0f);
    if (bytes == nullptr) throw std::invalid_argument("bytes is null");
    // Matrices on chip use none: the answer is one matrix's, whatever the batch,
    // so that it still tells calls with something to do from empty ones.
    if (on_chip(std::min(m, n), std::max(m, n))) batch = std::min<size_t>(batch, 1);
    *bytes = batch == 0 || m == 0 || n == 0
                 ? 0
                 : muon_space(nullptr, int64_t(batch), std::min(m, n), std::max(m, n), out.split).bytes;
  });
}

extern "C" int se_orthogonalize(int32_t dtype, const void *update, size_t batch, int64_t m, int64_t n,
                                int64_t batch_stride, int64_t row_stride, int32_t steps, float eps, void *out,
                                void *workspace, size_t workspace_bytes, int32_t device, void *stream) {
  return guarded([&] {
    const ResultType result = result_type(dtype, "dtype");
    check_matrices(batch, m, n, steps, eps);
    if (batch == 0 || m == 0 || n == 0) return;
    check_strides("update", batch, m, n, batch_stride, row_stride);
    DeviceGuard dg(device);
    check_device_ptr(update, device, "update");
    check_device_ptr(out, device, "out");
    UpdateArgs u{};
    u.grad = {update, batch_stride, row_stride};
    u.m = m;
    u.n = n;
    FinishArgs fin{};
    fin.out = out;
    fin.type = result.type;
    fin.row = n;
    fin.batch = m * n;
    orthogonalise(u, result.type, int64_t(batch), steps, eps, result.split, fin, workspace, workspace_bytes, device,
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
    const ResultType result = result_type(weight_dtype, "weight_dtype");
    check_value_dtype(grad_dtype, "grad_dtype");
    if (grad_dtype != result.type && grad_dtype != SE_FLOAT32)
      throw std::invalid_argument("grad_dtype must be weight_dtype or float32");
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
    UpdateArgs u{};
    u.grad = {grad, grad_batch_stride, grad_row_stride};
    u.momentum = {momentum, momentum_batch_stride, momentum_row_stride};
    u.beta = float(beta);
    u.nesterov = nesterov != 0;
    u.m = m;
    u.n = n;
    FinishArgs fin{};
    fin.out = weight;
    fin.type = result.type;
    fin.update = 1;
    fin.row = weight_row_stride;
    fin.batch = weight_batch_stride;
    fin.keep = float(1.0 - lr * weight_decay);
    fin.rate = float(lr * scale);
    orthogonalise(u, grad_dtype, int64_t(batch), steps, eps, result.split, fin, workspace, workspace_bytes, device,
                  static_cast<cudaStream_t>(stream));
  });
}
