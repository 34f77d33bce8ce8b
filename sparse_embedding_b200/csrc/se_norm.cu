// Layer normalisation of rows (pooled bags, looked-up rows, hidden rows) and
// its backward pass. It has no counterpart in the reference, whose users
// normalise the rows outside the store.
//
// For a row x of D values with weight w and bias b:
//   mean = sum x / D,  var = sum (x - mean)^2 / D,  r = 1 / sqrt(var + eps)
//   y = (x - mean) r w + b
// and for the gradient g of y, with h = (x - mean) r and q = g w:
//   dx = r (q - sum q / D - h (sum q h) / D)
//   dw = sum over rows of g h,   db = sum over rows of g
//
// Both passes are bound by HBM: the forward reads x and writes y, the
// backward reads x and g and writes dx. Every row is therefore read once,
// into registers, by `lanes` threads (a part of a warp, or a whole block for
// long rows); the variance is taken from the registers around the mean, not
// as a difference of two sums. All sums are fp32; y, dx, dw and db are rounded
// once, to the type they are stored in. A block keeps its share of the
// columns over all the rows it visits, so w and b are loaded once per thread
// and the sums of dw and db stay in registers until the block's end; the
// blocks' sums go to the caller's workspace and a second kernel adds them in
// block order, so equal calls give equal bits.

#include <algorithm>
#include <type_traits>

#include "se_common.cuh"
#include "se_dense.hpp"
#include "se_tcgen05.cuh"

namespace se_gpu {

namespace {

constexpr int kNormNarrowThreads = 256;  // block of the kernels with several rows per block
// A block per row: its most threads, of 16 values each, so that rows of up to
// 8,192 values fit the registers in every layout (the backward holds three fp32
// values per column besides the row).
constexpr int kNormWideThreads = 512;
// Rows at a time there. Forward: 16-bit rows of 4,096 take 105 us at two and 95
// at four (32,768 rows); backward: 156 at one and 171 at two (registers). Single
// values, 33,538 bf16 rows of 2,001: forward 89 us at one and 78 at two (115 with
// 8 values a thread), backward 131 at one and 183 at two.
constexpr __host__ __device__ int norm_wide_rows(int vec, bool gather, bool backward) {
  return gather ? (backward ? 1 : 2) : backward ? 1 : vec == 8 ? 4 : 2;
}

// VEC values of a row for one thread: 16 consecutive bytes, or, where the layout
// has no such vectors (GATHER), every `step`-th value from the thread's first,
// `count` of them, so that a warp's accesses are consecutive.
template <class V, int VEC, bool GATHER>
struct Pack {
  using T = typename V::T;
  struct Values {
    T v[VEC];
  };
  using Raw = std::conditional_t<GATHER, Values, uint4>;
  static_assert(GATHER || VEC * sizeof(T) == 16, "a vector is 16 bytes");
  // Values that every thread has whatever the row's length, by norm_shape's
  // choice of VEC and lanes: no test of their columns. Lanes are the least power
  // of two with VEC values each, so the row fills more than half of them (VEC
  // 8 to 32: dim > VEC / 2 lanes); VEC 4 takes rows from one value on. Over a
  // block lanes < dim / 16 + 32 and dim > 1,024, so 8 of 16 as well.
  static constexpr int kSure = !GATHER ? 0 : VEC == 4 ? 1 : VEC / 2;
  static __device__ __forceinline__ Raw zeros() {
    if constexpr (GATHER) {
      Values r;
#pragma unroll
      for (int i = 0; i < VEC; ++i) r.v[i] = V::store(0.0f);
      return r;
    } else {
      return make_uint4(0u, 0u, 0u, 0u);
    }
  }
  // of a row that is there; zeros behind its `count` values
  static __device__ __forceinline__ Raw load(const T *p, int step, int count) {
    if constexpr (GATHER) {
      Values r;
#pragma unroll
      for (int i = 0; i < VEC; ++i) r.v[i] = i < kSure || i < count ? p[i * step] : V::store(0.0f);
      return r;
    } else {
      return count > 0 ? *reinterpret_cast<const uint4 *>(p) : make_uint4(0u, 0u, 0u, 0u);
    }
  }
  static __device__ __forceinline__ void open(const Raw &r, float (&f)[VEC]) {
    const T *v = reinterpret_cast<const T *>(&r);
#pragma unroll
    for (int i = 0; i < VEC; ++i) f[i] = V::load(v[i]);
  }
  static __device__ __forceinline__ void store(T *p, const float (&f)[VEC], int step, int count) {
    if constexpr (GATHER) {
#pragma unroll
      for (int i = 0; i < VEC; ++i)
        if (i < kSure || i < count) p[i * step] = V::store(f[i]);
    } else if (count > 0) {
      uint4 r;
      T *v = reinterpret_cast<T *>(&r);
#pragma unroll
      for (int i = 0; i < VEC; ++i) v[i] = V::store(f[i]);
      *reinterpret_cast<uint4 *>(p) = r;
    }
  }
  // Column of value i of a thread's vector v, and how many values that has.
  static __device__ __forceinline__ int column(int v, int lane, int lanes, int i) {
    return GATHER ? lane + i * lanes : (v * lanes + lane) * VEC + i;
  }
  static __device__ __forceinline__ int count(int v, int lane, int lanes, int dim) {
    if constexpr (GATHER) return max(0, min(VEC, (dim - lane + lanes - 1) / lanes));
    else return (v * lanes + lane) * VEC < dim ? VEC : 0;
  }
};

// Value i of a weight or bias in its own type; `missing` where there is none.
__device__ __forceinline__ float param_at(const void *p, int type, int64_t i, float missing) {
  if (p == nullptr) return missing;
  if (type == SE_FLOAT32) return static_cast<const float *>(p)[i];
  if (type == SE_FLOAT16) return __half2float(static_cast<const __half *>(p)[i]);
  return __bfloat162float(static_cast<const __nv_bfloat16 *>(p)[i]);
}
__device__ __forceinline__ void param_put(void *p, int type, int64_t i, float f) {
  if (type == SE_FLOAT32) static_cast<float *>(p)[i] = f;
  else if (type == SE_FLOAT16) static_cast<__half *>(p)[i] = __float2half_rn(f);
  else static_cast<__nv_bfloat16 *>(p)[i] = __float2bfloat16_rn(f);
}

// Two fp32 operations in one instruction, where a vector has pairs.
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 r;
  asm("{\n .reg .b64 x, y, z;\n mov.b64 x, {%2, %3};\n mov.b64 y, {%4, %5};\n add.rn.f32x2 z, x, y;\n mov.b64 {%0, %1}, z;\n}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 r;
  asm("{\n .reg .b64 x, y, z;\n mov.b64 x, {%2, %3};\n mov.b64 y, {%4, %5};\n mul.rn.f32x2 z, x, y;\n mov.b64 {%0, %1}, z;\n}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 r;
  asm("{\n .reg .b64 x, y, z, w;\n mov.b64 x, {%2, %3};\n mov.b64 y, {%4, %5};\n mov.b64 z, {%6, %7};\n"
      " fma.rn.f32x2 w, x, y, z;\n mov.b64 {%0, %1}, w;\n}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return r;
}
// o = a + b, a b, a b + c on vectors; `all` is a value for every element.
template <int N> __device__ __forceinline__ void vadd(float (&o)[N], const float (&a)[N], const float (&b)[N]) {
  if constexpr (N == 1) o[0] = a[0] + b[0];
  else
#pragma unroll
    for (int i = 0; i < N; i += 2) {
      const float2 r = add2({a[i], a[i + 1]}, {b[i], b[i + 1]});
      o[i] = r.x;
      o[i + 1] = r.y;
    }
}
template <int N> __device__ __forceinline__ void vmul(float (&o)[N], const float (&a)[N], const float (&b)[N]) {
  if constexpr (N == 1) o[0] = a[0] * b[0];
  else
#pragma unroll
    for (int i = 0; i < N; i += 2) {
      const float2 r = mul2({a[i], a[i + 1]}, {b[i], b[i + 1]});
      o[i] = r.x;
      o[i + 1] = r.y;
    }
}
template <int N>
__device__ __forceinline__ void vfma(float (&o)[N], const float (&a)[N], const float (&b)[N], const float (&c)[N]) {
  if constexpr (N == 1) o[0] = __fmaf_rn(a[0], b[0], c[0]);
  else
#pragma unroll
    for (int i = 0; i < N; i += 2) {
      const float2 r = fma2({a[i], a[i + 1]}, {b[i], b[i + 1]}, {c[i], c[i + 1]});
      o[i] = r.x;
      o[i + 1] = r.y;
    }
}
template <int N> struct All {
  float v[N];
  __device__ __forceinline__ explicit All(float f) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = f;
  }
};
template <int N> __device__ __forceinline__ float vsum(const float (&a)[N]) {
  if constexpr (N == 1) {
    return a[0];
  } else if constexpr (N == 2) {
    return a[0] + a[1];
  } else {
    float h[N / 2];
#pragma unroll
    for (int i = 0; i < N / 2; i += 2) {
      const float2 r = add2({a[i], a[i + 1]}, {a[N / 2 + i], a[N / 2 + i + 1]});
      h[i] = r.x;
      h[i + 1] = r.y;
    }
    return vsum(h);
  }
}

// Sums of N values over the threads of a row, in every one of them.
//
// Within a warp's part (`lanes` threads), N > 1 rows at a time: in the first
// steps a thread gives away half of the values it holds and adds to the other
// half, until it holds one; the rest are plain xor steps on that one, and the
// sums go back by one shuffle each (N = 4 over 32 lanes: 10 shuffles for 20).
// For a whole block (WIDE) an exchange through shared memory follows.
// Successive exchanges alternate between two buffers, so one barrier each is
// enough: a buffer is written again only after the next exchange's barrier.
template <int N, bool WIDE>
struct RowSum {
  static_assert(N == 1 || N == 2 || N == 4, "a power of two");
  int lanes;
  float (*buf)[32][4];  // [2][32][4]
  int phase = 0;
  __device__ __forceinline__ void operator()(float (&v)[N]) { vote<false>(v, false); }
  // WIDE: the exchange's barrier also tells whether any thread's flag is set.
  template <bool VOTE = true>
  __device__ __forceinline__ bool vote(float (&v)[N], bool flag) {
    bool any = false;
    const int lane = int(threadIdx.x) & 31, part = lanes < 32 ? lanes : 32;
    constexpr unsigned kAll = 0xffffffffu;
    if (N == 1 || part < N) {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        if (o < part) {
#pragma unroll
          for (int i = 0; i < N; ++i) v[i] += __shfl_xor_sync(kAll, v[i], o);
        }
      }
    } else {
      const int half = part >> 1, quarter = part >> 2;
      float one;
      int rest;
      if constexpr (N == 4) {
        const bool up = lane & half, upper = lane & quarter;
        const float a = (up ? v[2] : v[0]) + __shfl_xor_sync(kAll, up ? v[0] : v[2], half);
        const float b = (up ? v[3] : v[1]) + __shfl_xor_sync(kAll, up ? v[1] : v[3], half);
        one = (upper ? b : a) + __shfl_xor_sync(kAll, upper ? a : b, quarter);
        rest = quarter;
      } else {
        const bool up = lane & half;
        one = (up ? v[N - 1] : v[0]) + __shfl_xor_sync(kAll, up ? v[0] : v[N - 1], half);
        rest = half;
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1)
        if (o < rest) one += __shfl_xor_sync(kAll, one, o);
      const int first = lane & ~(part - 1);
#pragma unroll
      for (int i = 0; i < N; ++i)
        v[i] = __shfl_sync(kAll, one, first + (N == 4 ? (i >> 1) * half + (i & 1) * quarter : i * half));
    }
    if constexpr (WIDE) {
      const int warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
      if (lane == 0) {
#pragma unroll
        for (int i = 0; i < N; ++i) buf[phase][warp][i] = v[i];
      }
      if constexpr (VOTE) any = __syncthreads_or(flag) != 0;
      else __syncthreads();
      const bool whole = (warps & (warps - 1)) == 0;  // a power of two: every lane's steps see all warps
      const int from = whole ? lane & (warps - 1) : lane;
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = from < warps ? buf[phase][from][i] : 0.0f;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        if (o < warps) {
#pragma unroll
          for (int i = 0; i < N; ++i) v[i] += __shfl_xor_sync(kAll, v[i], o);
        }
      }
      if (!whole) {  // lane 0's saw all
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = __shfl_sync(kAll, v[i], 0);
      }
      phase ^= 1;
    }
    return any;
  }
};

// Waits for `count` copies from stage `at` on, and reports that a wait gave up.
static __device__ __noinline__ void let_land(uint64_t *bars, int at, uint32_t parity, int stages, int count, uint32_t *status) {
  const long long end = clock64() + kDrainClocks;
  for (int i = 0; i < count; ++i) {
    wait_until(&bars[at], parity, end);
    if (++at == stages) {
      at = 0;
      parity ^= 1u;
    }
  }
  *reinterpret_cast<volatile uint32_t *>(status) = 1u;
  __threadfence_system();
}

// Tiles of rows on their way through shared memory, by bulk copies (one per
// tile where the rows have no gaps, else one per row) into a ring of buffers of
// `rows` rows for each of N arrays. The loads of a block are so several tiles
// deep, whatever registers its threads have left. A buffer's tile is ready when
// its barrier completes a phase; a wait that gives up makes the block leave.
//
// A bulk copy moves whole 16-byte units. Where rows do not start and end at
// such (ALIGNED false), the units that hold a row's first and last bytes are
// copied whole and the row is found inside; those of the matrix's first and
// last row reach past it (no row here is shorter than a unit), so the tiles
// with these two rows are not copied: the threads read them in place.
constexpr int kNormStages = 8;
template <class T, int N, bool ALIGNED>
struct RowRing {
  const T *src[N];
  int64_t stride[N];
  int64_t rows_total, step;  // rows of the matrix, rows between two tiles of this block
  int rows, dim, stages;
  uint8_t *buf;
  uint64_t *bars;
  volatile uint32_t *given_up;
  long long limit;
  int at = 0;
  uint32_t parity = 0;

  // bytes of a row in a buffer; rows without gaps lie there without gaps too
  static __host__ __device__ size_t pitch(int64_t dim) {
    return ALIGNED ? size_t(dim) * sizeof(T) : ((size_t(dim) * sizeof(T) + 15) & ~size_t(15)) + 16;
  }
  __device__ __forceinline__ uint8_t *buffer(int stage, int n) const {
    return buf + size_t(stage * N + n) * rows * pitch(dim);
  }
  __device__ __forceinline__ bool covers(int64_t base) const {
    return ALIGNED || (base > 0 && base + rows < rows_total);
  }
  // Row r of the tile in turn, which `covers` it.
  __device__ __forceinline__ const T *row(int n, int r, int64_t base) const {
    const uint8_t *b = buffer(at, n);
    if constexpr (ALIGNED) return reinterpret_cast<const T *>(b) + r * dim;
    // the address modulo 16, for which 32 bits are enough
    const bool dense = stride[n] == dim;
    const uint32_t at_row = uint32_t(base) + (dense ? 0u : uint32_t(r));
    const uint32_t from = uint32_t(reinterpret_cast<uintptr_t>(src[n])) + at_row * uint32_t(stride[n] * sizeof(T));
    return reinterpret_cast<const T *>(b + uint32_t(r) * uint32_t(dense ? dim * sizeof(T) : pitch(dim)) + (from & 15));
  }
  __device__ __forceinline__ static uint32_t units(const T *from, int64_t values, const uint8_t *&first) {
    const uintptr_t a = reinterpret_cast<uintptr_t>(from), e = a + size_t(values) * sizeof(T);
    first = reinterpret_cast<const uint8_t *>(a & ~uintptr_t(15));
    return uint32_t(((e + 15) & ~uintptr_t(15)) - (a & ~uintptr_t(15)));
  }
  __device__ __forceinline__ void fill(int stage, int64_t base) const {  // one thread
    const int64_t left = rows_total - base;
    const int count = int(left < rows ? left : rows);
    if (count <= 0) return;
    if (!covers(base)) {
      mbar_arrive_expect_tx(&bars[stage], 0);
      return;
    }
    uint32_t bytes = 0;
    const uint8_t *first;
#pragma unroll
    for (int n = 0; n < N; ++n) {
      if (stride[n] == dim) bytes += units(src[n] + base * stride[n], int64_t(count) * dim, first);
      else
        for (int r = 0; r < count; ++r) bytes += units(src[n] + (base + r) * stride[n], dim, first);
    }
    mbar_arrive_expect_tx(&bars[stage], bytes);
#pragma unroll
    for (int n = 0; n < N; ++n) {
      if (stride[n] == dim) {
        bytes = units(src[n] + base * stride[n], int64_t(count) * dim, first);
        bulk_copy_g2s(buffer(stage, n), first, bytes, &bars[stage]);
      } else {
        for (int r = 0; r < count; ++r) {
          bytes = units(src[n] + (base + r) * stride[n], dim, first);
          bulk_copy_g2s(buffer(stage, n) + r * pitch(dim), first, bytes, &bars[stage]);
        }
      }
    }
  }
  __device__ __forceinline__ void start(int64_t base) {
    if (threadIdx.x == 0) {
      for (int i = 0; i < stages; ++i) mbar_init(&bars[i], 1);
      *given_up = 0u;
      for (int i = 0; i < stages; ++i) fill(i, base + i * step);
    }
    __syncthreads();
  }
  __device__ __forceinline__ bool ready() const { return wait_or_give_up<N == 1>(&bars[at], parity, given_up, limit); }
  // The tile has been read by all threads: refill its buffer. Each thread has
  // passed fence_proxy_async_smem after its reads and then a barrier of the block
  // (that of its row's sum, where the block has one row at a time). The
  // barrier alone does not hold a copy back: a read that waits in the memory
  // pipe, behind stores that HBM holds up, comes after the copy (a warp's part of
  // one row in about 400,000 was a later row's, 32,768 x 4,096 bf16 backward).
  __device__ __forceinline__ void next(int64_t base) {
    if (threadIdx.x == 0) fill(at, base + stages * step);
    if (++at == stages) {
      at = 0;
      parity ^= 1u;
    }
  }
  // After a wait that gave up: the copies still in flight.
  __device__ __forceinline__ void drain(int64_t base, uint32_t *status) const {
    if (threadIdx.x == 0) {
      const int64_t tiles = (rows_total - base + step - 1) / step;
      let_land(bars, at, parity, stages, int(tiles < stages ? tiles : stages), status);
    }
  }
};

// Rows held in registers: `lanes` threads per row (a power of two up to 32, or
// with WIDE the block), NV vectors of VEC values per thread, U rows at a time
// (their loads are in flight together). Vectors are bound by HBM and, in short
// 16-bit rows, by instructions between load and store (212,992 x 128 fp32 41 us,
// 5.3 TB/s; 262,144 x 256 bf16 49 us, 5.5; 32,768 x 4,096 bf16 89 us, 6.0);
// single values by their loads, stores and tests (65,536 x 517 fp32 46 us, 5.9;
// 2^25 bf16 values in rows of 33 58 us, 2.3).
template <class V, int VEC, int NV, int U, bool WIDE, bool GATHER, bool RING, int LANES>
__global__ void __launch_bounds__(WIDE ? kNormWideThreads : kNormNarrowThreads,
                                  !WIDE && (GATHER ? VEC <= 8 : NV == 1) ? 3 : 1)
k_norm_forward(const typename V::T *__restrict__ x, int64_t x_stride, int64_t rows, int dim,
               const void *__restrict__ weight, const void *__restrict__ bias, int ptype, float eps,
               typename V::T *__restrict__ y, float *__restrict__ mean_out, float *__restrict__ rstd_out, int lanes_of_row,
               int stages, uint32_t *status, long long limit) {
  using P = Pack<V, VEC, GATHER>;
  using T = typename V::T;
  __shared__ float red[2][32][4];
  __shared__ uint64_t bars[kNormStages];
  __shared__ volatile uint32_t given_up;
  extern __shared__ __align__(128) uint8_t raw_smem[];
  const int lanes = LANES > 0 ? LANES : lanes_of_row;
  const int lane = WIDE ? int(threadIdx.x) : int(threadIdx.x) & (lanes - 1);
  const int group = WIDE ? 0 : int(threadIdx.x) / lanes;
  const int groups = WIDE ? 1 : int(blockDim.x) / lanes;
  float w[NV][VEC], b[NV][VEC];
#pragma unroll
  for (int v = 0; v < NV; ++v) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      const int c = P::column(v, lane, lanes, i);
      w[v][i] = c < dim ? param_at(weight, ptype, c, 1.0f) : 0.0f;
      b[v][i] = c < dim ? param_at(bias, ptype, c, 0.0f) : 0.0f;
    }
  }
  RowSum<U, WIDE> sum{lanes, red};
  const float inv = 1.0f / float(dim);
  const int64_t first = int64_t(blockIdx.x) * groups * U, step = int64_t(gridDim.x) * groups * U;
  RowRing<T, 1, !GATHER> ring{{x}, {x_stride}, rows, step, groups * U, dim, stages, raw_smem, bars, &given_up, limit};
  if (RING) ring.start(first);
  for (int64_t base = first; base < rows; base += step) {
    typename P::Raw raw[U][NV];
    const bool ok = !RING || ring.ready(), copied = RING && ring.covers(base);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t row = base + group * U + u;
      const T *staged = RING ? ring.row(0, group * U + u, base) : nullptr;
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        const int c = P::column(v, lane, lanes, 0), n = P::count(v, lane, lanes, dim);
        if (GATHER ? !copied && row >= rows : row >= rows) raw[u][v] = P::zeros();
        else if (copied) raw[u][v] = P::load(staged + c, lanes, n);
        else raw[u][v] = P::load(x + row * x_stride + c, lanes, n);
      }
    }
    if constexpr (RING && !WIDE) {
      fence_proxy_async_smem();
      if (__syncthreads_or(!ok)) {
        ring.drain(base, status);
        return;
      }
      ring.next(base);
    }
    // values beyond the row are zeros, and zeros again after the mean is taken off
    float f[U][NV][VEC], m[U], s[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float t[VEC];
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        P::open(raw[u][v], f[u][v]);
        if (v == 0) P::open(raw[u][0], t);
        else vadd(t, t, f[u][v]);
      }
      m[u] = vsum(t);
    }
    if constexpr (WIDE) {
      fence_proxy_async_smem();
      if (sum.vote(m, !ok)) {
        ring.drain(base, status);
        return;
      }
      ring.next(base);
    } else {
      sum(m);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      m[u] *= inv;
      const All<VEC> minus(-m[u]);
      float t[VEC];
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        const int n = P::count(v, lane, lanes, dim);
        if (GATHER || n > 0) vadd(f[u][v], f[u][v], minus.v);
        if (GATHER) {
#pragma unroll
          for (int i = P::kSure; i < VEC; ++i) f[u][v][i] = i < n ? f[u][v][i] : 0.0f;
        }
        if (v == 0) vmul(t, f[u][v], f[u][v]);
        else vfma(t, f[u][v], f[u][v], t);
      }
      s[u] = vsum(t);
    }
    sum(s);
#pragma unroll
    for (int u = 0; u < U; ++u) s[u] = __fmaf_rn(s[u], inv, eps);
    if constexpr (U == 1) {
      s[0] = 1.0f / sqrtf(s[0]);
    } else {  // a thread takes the root and the quotient of one of the rows (part of a row of `lanes` >= U threads)
      if (lanes < U) {
#pragma unroll
        for (int u = 0; u < U; ++u) s[u] = 1.0f / sqrtf(s[u]);
      } else {
        float one = s[0];
#pragma unroll
        for (int u = 1; u < U; ++u) one = (lane & (U - 1)) == u ? s[u] : one;
        one = 1.0f / sqrtf(one);
        const int from = (int(threadIdx.x) & 31) & ~(U - 1);
#pragma unroll
        for (int u = 0; u < U; ++u) s[u] = __shfl_sync(0xffffffffu, one, from + u);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t row = base + group * U + u;
      if (row >= rows) continue;
      if (lane == 0) {
        if (mean_out) mean_out[row] = m[u];
        if (rstd_out) rstd_out[row] = s[u];
      }
      const All<VEC> r(s[u]);
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        vmul(f[u][v], f[u][v], r.v);
        vfma(f[u][v], f[u][v], w[v], b[v]);
        P::store(y + row * dim + P::column(v, lane, lanes, 0), f[u][v], lanes, P::count(v, lane, lanes, dim));
      }
    }
  }
}

// A long sum of one thread: pieces of kPiece values, 64 pieces, and those, so
// that a chain of fp32 adds is short for any row or column (2^30 / 512 values: 64 +
// 64 + 512 adds; one after another, equal values may lose half a step of the sum each).
constexpr int kPiece = 64;
struct LongSum {
  float mid = 0.0f, sum = 0.0f;
  uint32_t n = 0;
  __device__ __forceinline__ void add(float piece) {
    mid += piece;
    if ((++n & 63u) == 0u) {
      sum += mid;
      mid = 0.0f;
    }
  }
  __device__ __forceinline__ float total() const { return sum + mid; }
};
// f(first, end) for pieces of the block's part of a row: a thread's columns are every blockDim-th from `first` on.
template <class F> __device__ __forceinline__ void row_pieces(int64_t dim, F &&f) {
  const int64_t step = int64_t(kPiece) * blockDim.x;
  for (int64_t base = 0; base < dim; base += step) f(base + threadIdx.x, min(dim, base + step));
}

// Rows longer than a block's registers: three passes over the row (the second
// and third out of L2, which bounds them: 3,355 x 20,001 fp32 252 us, 2.1 TB/s of
// what HBM has to move). Loops unrolled by eight: the piece's loop alone has one
// load in flight (402 us).
template <class V>
__global__ void __launch_bounds__(512)
k_norm_forward_long(const typename V::T *__restrict__ x, int64_t x_stride, int64_t rows, int64_t dim,
                    const void *__restrict__ weight, const void *__restrict__ bias, int ptype, float eps,
                    typename V::T *__restrict__ y, float *__restrict__ mean_out, float *__restrict__ rstd_out) {
  __shared__ float red[2][32][4];
  RowSum<1, true> sum{32, red};
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    const typename V::T *xr = x + row * x_stride;
    LongSum total, squares;
    row_pieces(dim, [&](int64_t c, int64_t end) {
      float f = 0.0f;
#pragma unroll 8
      for (; c < end; c += blockDim.x) f += V::load(xr[c]);
      total.add(f);
    });
    float m[1] = {total.total()};
    sum(m);
    m[0] /= float(dim);
    row_pieces(dim, [&](int64_t c, int64_t end) {
      float f = 0.0f;
#pragma unroll 8
      for (; c < end; c += blockDim.x) {
        const float d = V::load(xr[c]) - m[0];
        f = __fmaf_rn(d, d, f);
      }
      squares.add(f);
    });
    float s[1] = {squares.total()};
    sum(s);
    const float r = 1.0f / sqrtf(s[0] / float(dim) + eps);
    if (threadIdx.x == 0) {
      if (mean_out) mean_out[row] = m[0];
      if (rstd_out) rstd_out[row] = r;
    }
    for (int64_t c = threadIdx.x; c < dim; c += blockDim.x)
      y[row * dim + c] = V::store(__fmaf_rn((V::load(xr[c]) - m[0]) * r, param_at(weight, ptype, c, 1.0f),
                                            param_at(bias, ptype, c, 0.0f)));
  }
}

// Backward of rows held in registers (layout as k_norm_forward). partial:
// [gridDim.x][2][dim] fp32, this block's sums of g h and of g per column
// (null: no weight gradients wanted). Bound by HBM at vectors in a part of a
// warp (with the column kernel 212,992 x 128 fp32 56 us, 5.9 TB/s), by a block
// barrier a row at 16 warps an SM where a block takes one (32,768 x 4,096 bf16
// 147 us, 5.5; with a barrier of its own for the refill 170; the sums' registers
// allow no more), by instructions at single values (65,536 x 517
// fp32 84 us, 4.8; 9,973 x 1,037 bf16 34 us, 28 without the column kernel, 2.2).
template <class V, int VEC, int NV, int U, bool WIDE, bool GATHER, bool RING, int LANES>
__global__ void __launch_bounds__(WIDE ? kNormWideThreads : kNormNarrowThreads,
                                  !WIDE && (GATHER ? VEC <= 16 : NV <= 2) ? 2 : 1)
k_norm_backward(const typename V::T *__restrict__ grad, int64_t g_stride, const typename V::T *__restrict__ x,
                int64_t x_stride, int64_t rows, int dim, const float *__restrict__ mean,
                const float *__restrict__ rstd, const void *__restrict__ weight, int ptype,
                typename V::T *__restrict__ dx, float *__restrict__ partial, int lanes_of_row, int stages,
                long long limit, uint32_t *status) {
  using P = Pack<V, VEC, GATHER>;
  using T = typename V::T;
  __shared__ float red[2][32][4];
  __shared__ uint64_t bars[kNormStages];
  __shared__ volatile uint32_t given_up;
  extern __shared__ __align__(128) uint8_t raw_smem[];  // the ring; at the end, narrow: [warps][dim] fp32
  const int lanes = LANES > 0 ? LANES : lanes_of_row;
  const int lane = WIDE ? int(threadIdx.x) : int(threadIdx.x) & (lanes - 1);
  const int group = WIDE ? 0 : int(threadIdx.x) / lanes;
  const int groups = WIDE ? 1 : int(blockDim.x) / lanes;
  float w[NV][VEC], dw[NV][VEC], db[NV][VEC];
#pragma unroll
  for (int v = 0; v < NV; ++v) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      const int c = P::column(v, lane, lanes, i);
      w[v][i] = c < dim ? param_at(weight, ptype, c, 1.0f) : 0.0f;
      dw[v][i] = 0.0f;
      db[v][i] = 0.0f;
    }
  }
  RowSum<WIDE ? 2 * U : U, WIDE> sum{lanes, red};
  const float inv = 1.0f / float(dim);
  const int64_t first = int64_t(blockIdx.x) * groups * U, step = int64_t(gridDim.x) * groups * U;
  RowRing<T, 2, !GATHER> ring{{x, grad}, {x_stride, g_stride}, rows, step, groups * U, dim,
                              stages,    raw_smem,             bars, &given_up, limit};
  if (RING) ring.start(first);
  float next_m[U], next_r[U];  // a tile's statistics are asked for a tile ahead
  auto ask = [&](int64_t at) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t row = at + group * U + u;
      next_m[u] = row < rows ? mean[row] : 0.0f;
      next_r[u] = row < rows ? rstd[row] : 0.0f;
    }
  };
  ask(first);
  for (int64_t base = first; base < rows; base += step) {
    typename P::Raw xr[U][NV], gr[U][NV];
    float m[U], r[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      m[u] = next_m[u];
      r[u] = next_r[u];
    }
    ask(base + step);
    const bool ok = !RING || ring.ready(), copied = RING && ring.covers(base);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t row = base + group * U + u;
      const T *xs = RING ? ring.row(0, group * U + u, base) : nullptr;
      const T *gs = RING ? ring.row(1, group * U + u, base) : nullptr;
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        const int c = P::column(v, lane, lanes, 0), n = P::count(v, lane, lanes, dim);
        if (GATHER ? !copied && row >= rows : row >= rows) {
          xr[u][v] = gr[u][v] = P::zeros();
        } else if (copied) {
          xr[u][v] = P::load(xs + c, lanes, n);
          gr[u][v] = P::load(gs + c, lanes, n);
        } else {
          xr[u][v] = P::load(x + row * x_stride + c, lanes, n);
          gr[u][v] = P::load(grad + row * g_stride + c, lanes, n);
        }
      }
    }
    if constexpr (RING && !WIDE && GATHER) {
      fence_proxy_async_smem();
      if (__syncthreads_or(!ok)) {
        ring.drain(base, status);
        return;
      }
      ring.next(base);
    }
    // h = (x - m) r, as the formula has it: x r - m r would save an instruction a
    // pair, but m r, rounded by itself, puts |m| r 2^-24 on every h of the row (dw
    // 2e-5 off where the mean is 1,000 deviations; 3e-8 so).
    // Rows and columns beyond the matrix have r, g and w zero: they add nothing.
    float s0[U], s1[U], both[2 * U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const All<VEC> rr(r[u]), minus(-m[u]);
      float t0[VEC], t1[VEC];
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        float h[VEC], g[VEC], q[VEC];
        P::open(xr[u][v], h);
        P::open(gr[u][v], g);
        vadd(h, h, minus.v);
        vmul(h, h, rr.v);
        vmul(q, g, w[v]);
        if (v == 0) {
          vmul(t0, g, w[v]);
          vmul(t1, q, h);
        } else {
          vadd(t0, t0, q);
          vfma(t1, q, h, t1);
        }
        vfma(dw[v], g, h, dw[v]);
        vadd(db[v], db[v], g);
      }
      s0[u] = vsum(t0);
      s1[u] = vsum(t1);
    }
    if constexpr (WIDE) {  // one exchange for both
#pragma unroll
      for (int u = 0; u < U; ++u) {
        both[2 * u] = s0[u];
        both[2 * u + 1] = s1[u];
      }
      fence_proxy_async_smem();
      if (sum.vote(both, !ok)) {
        ring.drain(base, status);
        return;
      }
      ring.next(base);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        s0[u] = both[2 * u];
        s1[u] = both[2 * u + 1];
      }
    } else {
      sum(s0);
      sum(s1);
      // Vectors wait for their reads here, where the sums did already (100,000 x 512
      // bf16 100 us before the sums, 72 behind them); single values before the sums,
      // whose registers their refill would wait for (60,000 x 1,001 bf16 81 and 91 us).
      if constexpr (RING && !GATHER) {
        fence_proxy_async_smem();
        if (__syncthreads_or(!ok)) {
          ring.drain(base, status);
          return;
        }
        ring.next(base);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t row = base + group * U + u;
      if (row >= rows) continue;
      const All<VEC> rr(r[u]), minus(-m[u]), c0(-r[u] * (s0[u] * inv)), c1(-r[u] * (s1[u] * inv));
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        float h[VEC], g[VEC];
        P::open(xr[u][v], h);
        P::open(gr[u][v], g);
        vadd(h, h, minus.v);
        vmul(h, h, rr.v);
        vmul(g, g, w[v]);
        vfma(g, g, rr.v, c0.v);  // r q - r sum q / D - h r sum(q h) / D
        vfma(g, h, c1.v, g);
        P::store(dx + row * dim + P::column(v, lane, lanes, 0), g, lanes, P::count(v, lane, lanes, dim));
      }
    }
  }
  pdl_trigger();  // the column kernel's blocks may come as this grid's leave
  if (partial == nullptr) return;
  float *out = partial + int64_t(blockIdx.x) * 2 * dim;
  if constexpr (WIDE) {
#pragma unroll
    for (int v = 0; v < NV; ++v) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const int c = P::column(v, lane, lanes, i);
        if (c < dim) {
          out[c] = dw[v][i];
          out[dim + c] = db[v][i];
        }
      }
    }
  } else {
    // the warp's row groups by shuffles, then the block's warps in warp order
    float *cols = reinterpret_cast<float *>(raw_smem);
    __syncthreads();
    const int warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
#pragma unroll
      for (int v = 0; v < NV; ++v) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          float f = k == 0 ? dw[v][i] : db[v][i];
#pragma unroll
          for (int o = 16; o > 0; o >>= 1) {
            if (o >= lanes) f += __shfl_xor_sync(0xffffffffu, f, o);
          }
          const int c = P::column(v, lane, lanes, i);
          if ((threadIdx.x & 31) < unsigned(lanes) && c < dim) cols[warp * dim + c] = f;
        }
      }
      __syncthreads();
      for (int c = threadIdx.x; c < dim; c += blockDim.x) {
        float f = 0.0f;
        for (int i = 0; i < warps; ++i) f += cols[i * dim + c];
        out[k * dim + c] = f;
      }
      __syncthreads();
    }
  }
}

template <class V>
__global__ void __launch_bounds__(512)
k_norm_backward_long(const typename V::T *__restrict__ grad, int64_t g_stride, const typename V::T *__restrict__ x,
                     int64_t x_stride, int64_t rows, int64_t dim, const float *__restrict__ mean,
                     const float *__restrict__ rstd, const void *__restrict__ weight, int ptype,
                     typename V::T *__restrict__ dx) {
  __shared__ float red[2][32][4];
  RowSum<2, true> sum{32, red};
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    const typename V::T *xr = x + row * x_stride, *gr = grad + row * g_stride;
    const float m = mean[row], r = rstd[row];
    LongSum t0, t1;
    row_pieces(dim, [&](int64_t c, int64_t end) {
      float f0 = 0.0f, f1 = 0.0f;
      for (; c < end; c += blockDim.x) {
        const float q = V::load(gr[c]) * param_at(weight, ptype, c, 1.0f);
        f0 += q;
        f1 = __fmaf_rn(q, (V::load(xr[c]) - m) * r, f1);
      }
      t0.add(f0);
      t1.add(f1);
    });
    float s[2] = {t0.total(), t1.total()};
    sum(s);
    s[0] /= float(dim);
    s[1] /= float(dim);
    for (int64_t c = threadIdx.x; c < dim; c += blockDim.x) {
      const float q = V::load(gr[c]) * param_at(weight, ptype, c, 1.0f);
      dx[row * dim + c] = V::store(r * (q - s[0] - (V::load(xr[c]) - m) * r * s[1]));
    }
  }
}

// Column sums of long rows: a thread per column and split of the rows, loads
// along the rows (3,355 x 20,001 fp32 128 us, 4.2 TB/s).
template <class V>
__global__ void __launch_bounds__(256)
k_norm_columns_long(const typename V::T *__restrict__ grad, int64_t g_stride, const typename V::T *__restrict__ x,
                    int64_t x_stride, int64_t rows, int64_t dim, const float *__restrict__ mean,
                    const float *__restrict__ rstd, float *__restrict__ partial) {
  const int64_t c = int64_t(blockIdx.x) * blockDim.x + threadIdx.x;
  if (c >= dim) return;
  const int64_t each = (rows + gridDim.y - 1) / gridDim.y;
  const int64_t first = blockIdx.y * each, last = first + each < rows ? first + each : rows;
  LongSum dw, db;
  for (int64_t base = first; base < last; base += kPiece) {
    const int64_t end = min(last, base + kPiece);
    float fw = 0.0f, fb = 0.0f;
    for (int64_t row = base; row < end; ++row) {
      const float g = V::load(grad[row * g_stride + c]);
      fw = __fmaf_rn(g, (V::load(x[row * x_stride + c]) - mean[row]) * rstd[row], fw);
      fb += g;
    }
    dw.add(fw);
    db.add(fb);
  }
  partial[int64_t(blockIdx.y) * 2 * dim + c] = dw.total();
  partial[int64_t(blockIdx.y) * 2 * dim + dim + c] = db.total();
}

// dw and db: the blocks' sums of each column, added in a fixed order (each of
// the 32 threads of a column takes every 32nd block, then the 32 in order).
// Launch and latency bound it: 3.6 us for 128 columns, 8.7 for 4,096.
__global__ void __launch_bounds__(1024)
k_norm_columns(const float *__restrict__ partial, int64_t blocks, int64_t dim, void *__restrict__ dweight,
               void *__restrict__ dbias, int ptype) {
  __shared__ float part[32][33];
  const int lane = threadIdx.x & 31, strip = threadIdx.x >> 5;
  const int64_t c = int64_t(blockIdx.x) * 32 + lane;
  pdl_wait();
  LongSum sum;
  if (c < 2 * dim) {
    for (int64_t base = 0; base < blocks; base += 32 * kPiece) {
      const int count = int(min(blocks - base, int64_t(32 * kPiece)));
      const float *from = partial + base * 2 * dim;
      float f = 0.0f;
#pragma unroll 8
      for (int k = strip; k < count; k += 32) f += __ldcg(from + int64_t(k) * 2 * dim + c);
      sum.add(f);
    }
  }
  part[strip][lane] = sum.total();
  __syncthreads();
  if (strip == 0 && c < 2 * dim) {
    float f = 0.0f;
#pragma unroll
    for (int k = 0; k < 32; ++k) f += part[k][lane];
    if (c < dim) {
      if (dweight) param_put(dweight, ptype, c, f);
    } else if (dbias) {
      param_put(dbias, ptype, c - dim, f);
    }
  }
}

constexpr int kNormLongSplits = 64;

// A launch of the register kernels: their blocks, buffers and shared memory.
struct NormLaunch {
  int blocks, stages;
  size_t smem;
};

// How a call's rows are laid over threads.
struct NormShape {
  bool vec;    // 16-byte vectors
  bool wide;   // a block per row
  bool ring;   // through shared memory
  bool longer; // rows beyond a block's registers
  int nv, lanes, threads, unroll;
};

// Rows of up to 256 values without 16-byte layout, and vectors of up to 64 loads
// with gaps, are read in place: a copy for each such row is too many copies, and
// without gaps copying gains nothing there. 2^25 values, forward, copied and in
// place: fp32 rows of 64 with a gap of 8 78 and 49 us, of 8 with a gap of 8 407
// and 74, bf16 rows of 33 106 and 88; in place loses at longer rows (517 fp32
// values with a gap of 8, 110 and 118).
//
// Single values: 8 a thread where the row fits a part of a warp (33 bf16 values
// 88 us with 4 a thread, 66 with 8, 81 with 16), more only for longer rows.
NormShape norm_shape(int64_t dim, size_t value_size, bool aligned, bool gaps, bool backward) {
  NormShape s{};
  const int per = int(16 / value_size);
  s.vec = aligned && dim % per == 0;
  const int64_t n = s.vec ? dim / per : dim;  // loads per row
  s.threads = kNormNarrowThreads;
  if (s.vec ? n <= 128 : n <= 1024) {
    if (s.vec) {
      s.nv = n <= 32 ? 1 : n <= 64 ? 2 : 4;
      s.unroll = 4 / s.nv;
      s.ring = !gaps || s.nv > 2;
    } else {
      s.nv = n <= 32 ? 4 : n <= 256 ? 8 : n <= 512 ? 16 : 32;
      s.unroll = s.nv <= 8 ? 2 : 1;
      s.ring = s.nv > 8;
    }
    const int64_t lanes = s.vec ? n : (n + s.nv - 1) / s.nv;
    s.lanes = 1;
    while (s.lanes < lanes && s.lanes < 32) s.lanes *= 2;
    return s;
  }
  s.nv = s.vec ? 16 / per : 16;
  s.unroll = norm_wide_rows(per, !s.vec, backward);
  s.wide = s.ring = true;
  const int64_t threads = (n + s.nv - 1) / s.nv;
  s.longer = threads > kNormWideThreads;
  s.threads = int(std::min<int64_t>(kNormWideThreads, (threads + 31) / 32 * 32));
  s.lanes = s.threads;
  return s;
}

// Most blocks of the register kernels: `sms` x 1,024 threads. More
// blocks would add sums to the workspace and to the second kernel.
int norm_blocks(int64_t rows, const NormShape &s, int sms) {
  const int64_t per_block = int64_t(s.threads / s.lanes) * s.unroll;
  const int64_t need = (rows + per_block - 1) / per_block;
  return int(std::max<int64_t>(1, std::min<int64_t>(need, int64_t(sms) * (1024 / s.threads))));
}

// Rows of one launch of the backward with column sums: a thread of the fewest
// blocks (one per multiprocessor) adds 512 rows, so that its fp32 chain is short;
// more rows take more launches, whose sums lie side by side in the workspace.
int64_t norm_chunk(const NormShape &s, int sms) { return int64_t(sms) * (s.threads / s.lanes) * 512; }

// Most blocks' sums that a call leaves.
int64_t norm_partials(int64_t rows, const NormShape &s, int sms) {
  if (s.longer) return std::min<int64_t>(rows, kNormLongSplits);
  const int64_t chunk = norm_chunk(s, sms), whole = rows / chunk, rest = rows - whole * chunk;
  return whole * norm_blocks(chunk, s, sms) + (rest > 0 ? norm_blocks(rest, s, sms) : 0);
}

// The ring of a block takes at most 48 KB per array (two blocks of the backward,
// four of the forward on an SM, with 128 KB or more of loads in flight there),
// and the grid is what runs at once.
template <class K>
NormLaunch norm_launch(K *kernel, const NormShape &s, int64_t rows, int64_t dim, size_t value_size, int arrays,
                       int device, size_t least_smem) {
  const int sms = sm_count(device);
  NormLaunch l{};
  const int64_t tile_rows = int64_t(s.threads / s.lanes) * s.unroll;
  const size_t row = s.vec ? size_t(dim) * value_size : ((size_t(dim) * value_size + 15) & ~size_t(15)) + 16;
  const size_t tile = size_t(tile_rows) * row * arrays;
  l.stages = s.ring ? int(std::max<size_t>(2, std::min<size_t>(kNormStages, size_t(49152) * arrays / tile))) : 0;
  l.smem = std::max(tile * l.stages, least_smem);
  allow_dynamic_smem(kernel, l.smem);
  l.blocks = std::min(norm_blocks(rows, s, sms), sms * resident_blocks(kernel, device, s.threads, l.smem));
  return l;
}

// f with the kernel's constants: values per load, loads per thread, rows at a
// time, a block per row, values one by one, rows through shared memory,
// threads of a row (0: a variable; as a constant it makes the columns of single
// values immediate offsets: rows of 65 fp32 values 69 -> 54 us forward, 116 -> 85
// backward; and saves vectors the tests in the row sums: 262,144 x 256 bf16
// forward 52 -> 49, 65,536 x 64 fp32 backward 15.1 -> 13.4; in place, 256 bf16
// values with a gap of 8, backward 52 -> 44, forward 30 -> 33, so not there. 8
// threads lose by it: 524,288 x 64 bf16 forward 28.1 -> 29.8, backward 38.8 -> 41.2).
template <class V, bool BACKWARD, class F>
void with_norm_shape(const NormShape &s, F &&f) {
  constexpr int kVec = int(16 / sizeof(typename V::T));
  const std::false_type no{};
  const std::true_type yes{};
  using std::integral_constant;
  const integral_constant<int, kVec> vec{};
  const integral_constant<int, 1> one{};
  const integral_constant<int, 2> two{};
  const integral_constant<int, 4> four{};
  const integral_constant<int, 0> any{};
  const integral_constant<int, 32> all{};
  const integral_constant<int, 16> sixteen{};
  if (s.vec) {
    const integral_constant<int, norm_wide_rows(kVec, false, BACKWARD)> wide_rows{};
    if (s.wide) f(vec, integral_constant<int, 16 / kVec>{}, wide_rows, yes, no, yes, any);
    else if (s.nv == 4) f(vec, four, one, no, no, yes, all);
    else if (s.nv == 2 && s.ring) f(vec, two, two, no, no, yes, all);
    else if (s.nv == 2) f(vec, two, two, no, no, no, all);
    else if (s.ring && s.lanes == 32) f(vec, one, four, no, no, yes, all);
    else if (s.ring && s.lanes == 16) f(vec, one, four, no, no, yes, sixteen);
    else if (s.ring) f(vec, one, four, no, no, yes, any);
    else if (BACKWARD && s.lanes == 32) f(vec, one, four, no, no, no, all);
    else f(vec, one, four, no, no, no, any);
  } else {
    const integral_constant<int, 8> eight{};
    if (s.wide) f(sixteen, one, integral_constant<int, norm_wide_rows(kVec, true, BACKWARD)>{}, yes, yes, yes, any);
    else if (s.nv == 4) f(four, one, two, no, yes, no, any);
    else if (s.nv == 8 && s.lanes == 8) f(eight, one, two, no, yes, no, eight);
    else if (s.nv == 8 && s.lanes == 16) f(eight, one, two, no, yes, no, sixteen);
    else if (s.nv == 8) f(eight, one, two, no, yes, no, all);
    else if (s.nv == 16) f(sixteen, one, one, no, yes, yes, all);
    else f(integral_constant<int, 32>{}, one, one, no, yes, yes, all);
  }
}

void check_norm(int32_t value_dtype, int32_t param_dtype, size_t rows, int64_t dim) {
  check_value_dtype(value_dtype, "value_dtype");
  check_value_dtype(param_dtype, "param_dtype");
  if (dim <= 0) throw std::invalid_argument("dim must be > 0");
  if (dim > (int64_t(1) << 30)) throw std::invalid_argument("dim must be at most 2^30");
  if (rows > (size_t(1) << 40)) throw std::invalid_argument("rows must be at most 2^40");
}

}  // namespace

}  // namespace se_gpu

using namespace se_gpu;

extern "C" int se_set_wait_limit(uint64_t clocks) {
  return guarded([&] {
    if (clocks > uint64_t(kWaitClocks)) throw std::invalid_argument("clocks must be at most 8e9");
    wait_limit() = clocks == 0 ? kWaitClocks : (long long)(clocks);
  });
}

extern "C" int se_check_waits(int32_t device) {
  return guarded([&] { WaitWords::get().check(device); });
}

extern "C" int se_layer_norm(int32_t value_dtype, int32_t param_dtype, const void *x, size_t rows, int64_t dim,
                             int64_t x_stride, const void *weight, const void *bias, float eps, void *y,
                             float *mean_out, float *rstd_out, int32_t device, void *stream) {
  return guarded([&] {
    check_norm(value_dtype, param_dtype, rows, dim);
    if (!(eps >= 0.0f) || !std::isfinite(eps)) throw std::invalid_argument("eps must be finite and non-negative");
    if (rows == 0) return;
    if (x_stride < dim && rows > 1) throw std::invalid_argument("x_stride must be at least dim");
    DeviceGuard dg(device);
    check_device_ptr(x, device, "x");
    check_device_ptr(y, device, "y");
    check_device_ptr(weight, device, "weight", true);
    check_device_ptr(bias, device, "bias", true);
    check_device_ptr(mean_out, device, "mean", true);
    check_device_ptr(rstd_out, device, "rstd", true);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const int sms = sm_count(device);
    uint32_t *status = WaitWords::get().of(device, st);
    const size_t vb = value_bytes(value_dtype);
    const NormShape s = norm_shape(dim, vb, aligned16(x) && aligned16(y) && (rows == 1 || x_stride * vb % 16 == 0),
                                   rows > 1 && x_stride != dim, false);
    dispatch_value(value_dtype, [&](auto tag) {
      using V = decltype(tag);
      using T = typename V::T;
      const T *xp = static_cast<const T *>(x);
      T *yp = static_cast<T *>(y);
      if (s.longer) {
        const unsigned grid = unsigned(std::min<size_t>(rows, size_t(sms) * 4));
        k_norm_forward_long<V><<<grid, 512, 0, st>>>(xp, x_stride, int64_t(rows), dim, weight, bias, param_dtype, eps,
                                                     yp, mean_out, rstd_out);
        launched("k_norm_forward_long");
        return;
      }
      with_norm_shape<V, false>(s, [&](auto vec, auto nv, auto u, auto wide, auto gather, auto ring, auto lanes) {
        auto *kernel = k_norm_forward<V, decltype(vec)::value, decltype(nv)::value, decltype(u)::value,
                                      decltype(wide)::value, decltype(gather)::value, decltype(ring)::value,
                                      decltype(lanes)::value>;
        const NormLaunch l = norm_launch(kernel, s, int64_t(rows), dim, vb, 1, device, 0);
        kernel<<<l.blocks, s.threads, l.smem, st>>>(xp, x_stride, int64_t(rows), int(dim), weight, bias, param_dtype, eps,
                                                    yp, mean_out, rstd_out, s.lanes, l.stages, status, wait_limit().load());
      });
      launched("k_norm_forward");
    });
  });
}

extern "C" int se_layer_norm_backward_workspace(size_t rows, int64_t dim, int32_t device, size_t *bytes) {
  return guarded([&] {
    check_norm(SE_FLOAT32, SE_FLOAT32, rows, dim);
    if (bytes == nullptr) throw std::invalid_argument("bytes is null");
    // Enough for every type and alignment of the same rows and dim.
    const int sms = sm_count(device);
    int64_t blocks = 1;
    for (const size_t vb : {size_t(2), size_t(4)}) {
      for (const bool aligned : {false, true}) {
        const NormShape s = norm_shape(dim, vb, aligned, false, true);
        blocks = std::max(blocks, norm_partials(int64_t(rows), s, sms));
      }
    }
    *bytes = size_t(blocks) * 2 * size_t(dim) * sizeof(float);
  });
}

extern "C" int se_layer_norm_backward(int32_t value_dtype, int32_t param_dtype, const void *grad, int64_t grad_stride,
                                      const void *x, int64_t x_stride, size_t rows, int64_t dim, const float *mean,
                                      const float *rstd, const void *weight, void *dx, void *dweight, void *dbias,
                                      void *workspace, size_t workspace_bytes, int32_t device, void *stream) {
  return guarded([&] {
    check_norm(value_dtype, param_dtype, rows, dim);
    if (rows > 1 && (x_stride < dim || grad_stride < dim))
      throw std::invalid_argument("x_stride and grad_stride must be at least dim");
    DeviceGuard dg(device);
    check_device_ptr(weight, device, "weight", true);
    check_device_ptr(dweight, device, "dweight", true);
    check_device_ptr(dbias, device, "dbias", true);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const int sms = sm_count(device);
    uint32_t *status = WaitWords::get().of(device, st);
    const bool sums = dweight != nullptr || dbias != nullptr;
    int64_t blocks = 0;
    float *partial = nullptr;
    if (rows > 0) {
      check_device_ptr(grad, device, "grad");
      check_device_ptr(x, device, "x");
      check_device_ptr(mean, device, "mean");
      check_device_ptr(rstd, device, "rstd");
      check_device_ptr(dx, device, "dx");
      const size_t vb = value_bytes(value_dtype);
      const NormShape s = norm_shape(dim, vb, aligned16(x) && aligned16(grad) && aligned16(dx) &&
                                                  (rows == 1 || (x_stride * vb % 16 == 0 && grad_stride * vb % 16 == 0)),
                                     rows > 1 && (x_stride != dim || grad_stride != dim), true);
      blocks = norm_partials(int64_t(rows), s, sms);
      if (sums) {
        check_device_ptr(workspace, device, "workspace");
        if (reinterpret_cast<uintptr_t>(workspace) % 4 != 0 ||
            workspace_bytes < size_t(blocks) * 2 * size_t(dim) * sizeof(float))
          throw std::invalid_argument("workspace is smaller than se_layer_norm_backward_workspace asks for");
        partial = static_cast<float *>(workspace);
      }
      dispatch_value(value_dtype, [&](auto tag) {
        using V = decltype(tag);
        using T = typename V::T;
        const T *xp = static_cast<const T *>(x), *gp = static_cast<const T *>(grad);
        T *dxp = static_cast<T *>(dx);
        if (s.longer) {
          const unsigned grid = unsigned(std::min<size_t>(rows, size_t(sms) * 4));
          k_norm_backward_long<V><<<grid, 512, 0, st>>>(gp, grad_stride, xp, x_stride, int64_t(rows), dim, mean, rstd,
                                                        weight, param_dtype, dxp);
          launched("k_norm_backward_long");
          if (sums) {
            const dim3 cgrid(unsigned((dim + 255) / 256), unsigned(blocks));
            k_norm_columns_long<V><<<cgrid, 256, 0, st>>>(gp, grad_stride, xp, x_stride, int64_t(rows), dim, mean,
                                                          rstd, partial);
            launched("k_norm_columns_long");
          }
          return;
        }
        with_norm_shape<V, true>(s, [&](auto vec, auto nv, auto u, auto wide, auto gather, auto ring, auto lanes) {
          auto *kernel = k_norm_backward<V, decltype(vec)::value, decltype(nv)::value, decltype(u)::value,
                                         decltype(wide)::value, decltype(gather)::value, decltype(ring)::value,
                                         decltype(lanes)::value>;
          const size_t cols = s.wide || !sums ? 0 : size_t(s.threads / 32) * size_t(dim) * sizeof(float);
          const int64_t all = int64_t(rows), chunk = sums ? norm_chunk(s, sms) : all;
          blocks = 0;
          for (int64_t row = 0; row < all; row += chunk) {
            const int64_t count = std::min(chunk, all - row);
            const NormLaunch l = norm_launch(kernel, s, count, dim, vb, 2, device, cols);
            kernel<<<l.blocks, s.threads, l.smem, st>>>(gp + row * grad_stride, grad_stride, xp + row * x_stride, x_stride, count,
                                                        int(dim), mean + row, rstd + row, weight, param_dtype, dxp + row * dim,
                                                        sums ? partial + blocks * 2 * dim : nullptr, s.lanes, l.stages,
                                                        wait_limit().load(), status);
            launched("k_norm_backward");
            blocks += l.blocks;
          }
        });
      });
    }
    if (sums) {
      pdl(k_norm_columns, unsigned((2 * dim + 31) / 32), 1024, 0, st, static_cast<const float *>(partial), blocks, dim,
          dweight, dbias, int(param_dtype));
      count_launch();
    }
  });
}
