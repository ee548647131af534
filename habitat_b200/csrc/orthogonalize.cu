// Updates of weight matrices made nearly orthogonal by Newton-Schulz steps:
//   X = G / (|G|_F + eps);   `steps` times:  A = X X^T,  B = a I + b A + c A^2,  X <- B X
// (on G^T where G has more rows than columns), which drives all singular values towards one while the singular vectors
// stay.  Three products per step on the tensor cores (dense_gemm.cuh); A and B are symmetric, so only tiles that reach their lower
// triangle are computed and the rest is mirrored: s^2 l + s^3 + 2 s^2 l operations per step for sides s <= l.
//
// Numbers.  Operands are half precision (11 bits, against bfloat16's 8, at the same rate) scaled by powers of two: X, A and B by
// 2^8, which keeps entries of matrices with a norm near one far from the subnormal numbers, and G, for the first step,
// so that its Frobenius norm is in [2^13, 2^14).  The exact factor 1 / (|G| + eps) enters the first step's results in
// float32, so a 16-bit G is multiplied unrounded.  Sums are float32, the norm float64.  With `split` every operand is a
// pair of half-precision matrices, high and low parts (22 bits), and a product three (hi hi + hi lo + lo hi), which is what
// updates of all types get unless the caller asks for less.  Without, an operand is one (11 bits): 8192 x 4096 bfloat16 results
// are then 1.94e-3 off a 64-bit computation (1.66e-3 with pairs, all of it their own rounding), in a third of the MMAs.
//
// Sides.  All steps of an update with a shorter side of up to 128 run in one launch of one cluster, which keeps X on chip, and
// with one of up to 32 in float64 on the Gram matrix alone (orthogonalize_small.cuh); larger ones take three launches per step.
#include <atomic>
#include <cmath>
#include <type_traits>

#include "dense_gemm.cuh"
#include "dense_host.h"

namespace dense {
namespace {

constexpr float kScale = 256.0f;          // of stored X, A and B
constexpr int kNormThreads = 256;
constexpr int kMostPartials = 256;
constexpr int kNormBlocks = 592;           // over all matrices: four per SM of 148
constexpr int kSideBlocks = 2;            // blocks of 64 columns per CTA that a cluster is made wider for

template <typename T>
__device__ __forceinline__ float element(const void* base, int64_t at) { return static_cast<float>(static_cast<const T*>(base)[at]); }
__device__ __forceinline__ float load_element(const void* base, int type, int64_t at) {
  return type == kF32 ? element<float>(base, at) : type == kBF16 ? element<__nv_bfloat16>(base, at) : element<__half>(base, at);
}

struct Source {
  const void* base;
  int64_t ld, batch_stride;
  int32_t type, rows, cols;
};

// Eight elements from a 16-byte boundary on.
__device__ __forceinline__ void load_eight(const void* base, int type, int64_t at, float (&x)[8]) {
  if (type == kF32) {
    const float4* from = reinterpret_cast<const float4*>(static_cast<const float*>(base) + at);
    const float4 a = from[0], b = from[1];
    x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
    x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
    return;
  }
  const uint4 v = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(base) + at);
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = type == kBF16 ? make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xFFFF0000u))
                                   : __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
    x[2 * i] = f.x;
    x[2 * i + 1] = f.y;
  }
}

}  // namespace
}  // namespace dense

#include "orthogonalize_small.cuh"

namespace dense {
namespace {

// Sums of squares of G's elements, one per block.  `eights`: rows follow one another and are read in pieces of eight elements
// (figures below).
__global__ void __launch_bounds__(kNormThreads) norm_kernel(Source g, int eights, double* partials) {
  __shared__ double scratch[kNormThreads / 32];
  hb_grid_dependency_wait();
  const int64_t base = blockIdx.y * g.batch_stride;
  const int64_t n = static_cast<int64_t>(g.rows) * g.cols;
  double sum = 0.0;
  if (eights) {
    const int64_t step = static_cast<int64_t>(gridDim.x) * kNormThreads;
#pragma unroll 2
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * kNormThreads + threadIdx.x; i < n / 8; i += step) {
      float x[8];
      load_eight(g.base, g.type, base + 8 * i, x);
      double even = 0.0, odd = 0.0;
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        even = fma(static_cast<double>(x[e]), static_cast<double>(x[e]), even);
        odd = fma(static_cast<double>(x[e + 1]), static_cast<double>(x[e + 1]), odd);
      }
      sum += even + odd;
    }
    if (blockIdx.x == 0 && threadIdx.x < n % 8) {
      const double x = load_element(g.base, g.type, base + n - 1 - threadIdx.x);
      sum += x * x;
    }
  } else if (g.ld == g.cols) {
#pragma unroll 4
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * kNormThreads + threadIdx.x; i < n; i += static_cast<int64_t>(gridDim.x) * kNormThreads) {
      const double x = load_element(g.base, g.type, base + i);
      sum += x * x;
    }
  } else {
    for (int64_t r = blockIdx.x; r < g.rows; r += gridDim.x)
      for (int64_t i = threadIdx.x; i < g.cols; i += kNormThreads) {
        const double x = load_element(g.base, g.type, base + r * g.ld + i);
        sum += x * x;
      }
  }
#pragma unroll
  for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, d);
  if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < kNormThreads / 32; ++i) sum += scratch[i];
    partials[blockIdx.y * gridDim.x + blockIdx.x] = sum;
  }
}

// G as half-precision operands: X0 [s][l] = G p (or G^T p), p the power of two that brings its norm to [2^13, 2^14); the
// block at the origin leaves 1 / ((norm + eps) p), NaN where the norm is not finite.
struct Planes {
  __half* hi;
  int64_t ld, batch_stride, low;   // low: elements from a high part to its low part, 0 without
};
// p, worked out by every block.
__device__ __forceinline__ float operand_power(const double* partials, int n_partials, int batch, double eps, bool leaves_factor, float* factor,
                                               float* power) {
  if (threadIdx.x < 32) {
    double sum = 0.0;
#pragma unroll 4
    for (int i = static_cast<int>(threadIdx.x); i < n_partials; i += 32) sum += partials[static_cast<int64_t>(batch) * n_partials + i];
#pragma unroll
    for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, d);
    if (threadIdx.x == 0) {
      const double norm = sqrt(sum);
      const bool fine = norm < static_cast<double>(INFINITY);
      const int e = fine && norm > 0.0 ? max(-149, min(127, 13 - ilogb(norm))) : 0;
      *power = static_cast<float>(ldexp(1.0, e));
      if (leaves_factor) factor[batch] = fine ? static_cast<float>(1.0 / ((norm + eps) * ldexp(1.0, e))) : __int_as_float(0x7FFFFFFF);
    }
  }
  __syncthreads();
  return *power;
}

// G that is not transposed, its rows on 16-byte boundaries: pieces of eight elements.  Eight 1024 x 1024 float32 matrices, cold: the
// norms 10.5 us and this 12.4, 14.7 and 24.2 one element at a time (34 MB read are 5 us, 34 more written 10).
__global__ void __launch_bounds__(256) operand_rows_kernel(Source g, const double* partials, int n_partials, double eps, Planes x, float* factor) {
  __shared__ float power;
  hb_grid_dependency_wait();
  const int batch = blockIdx.y;
  const float p = operand_power(partials, n_partials, batch, eps, blockIdx.x == 0, factor, &power);
  const int64_t base = batch * g.batch_stride;
  const int per_row = (g.cols + 7) / 8;
  const int64_t n = static_cast<int64_t>(per_row) * g.rows, step = static_cast<int64_t>(gridDim.x) * 256;
#pragma unroll 2
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < n; i += step) {
    const int64_t r = n <= 0x7FFFFFFF ? static_cast<int64_t>(static_cast<int>(i) / per_row) : i / per_row;
    const int c = static_cast<int>(i - r * per_row) * 8;
    float v[8];
    if (c + 8 <= g.cols) {
      load_eight(g.base, g.type, base + r * g.ld + c, v);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = c + e < g.cols ? load_element(g.base, g.type, base + r * g.ld + c + e) : 0.0f;
    }
    uint32_t hi[4], lo[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float2 f = make_float2(v[2 * e] * p, v[2 * e + 1] * p);
      hi[e] = pack_f16(f.x, f.y);
      const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&hi[e]));
      lo[e] = pack_f16(f.x - h.x, f.y - h.y);
    }
    // X's rows are a multiple of 64 elements apart
    __half* to = x.hi + batch * x.batch_stride + r * x.ld + c;
    *reinterpret_cast<uint4*>(to) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
    if (x.low) *reinterpret_cast<uint4*>(to + x.low) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
  }
}

__global__ void __launch_bounds__(256) operand_kernel(Source g, const double* partials, int n_partials, double eps, int flip, Planes x,
                                                      float* factor) {
  __shared__ float tile[32][33];
  __shared__ float power;
  hb_grid_dependency_wait();
  const int batch = blockIdx.z;
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const float p = operand_power(partials, n_partials, batch, eps, blockIdx.x == 0 && blockIdx.y == 0, factor, &power);
  const int64_t base = batch * g.batch_stride;
  const int s = flip ? g.cols : g.rows, l = flip ? g.rows : g.cols;
  const int r0 = blockIdx.y * 32, c0 = blockIdx.x * 32;   // in X
#pragma unroll
  for (int i = 0; i < 32; i += 8) {
    // read along G's rows
    const int gr = (flip ? c0 : r0) + ty + i, gc = (flip ? r0 : c0) + tx;
    tile[ty + i][tx] = gr < g.rows && gc < g.cols ? load_element(g.base, g.type, base + static_cast<int64_t>(gr) * g.ld + gc) * p : 0.0f;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 32; i += 8) {
    const int r = r0 + ty + i, c = c0 + tx;
    if (r >= s || c >= l) continue;
    const float v = flip ? tile[tx][ty + i] : tile[ty + i][tx];
    __half* at = x.hi + batch * x.batch_stride + static_cast<int64_t>(r) * x.ld + c;
    const __half hi = __float2half_rn(v);
    *at = hi;
    if (x.low) at[x.low] = __float2half_rn(v - __half2float(hi));
  }
}

// Calls work(chunk, values) for the 32-column chunks of a warp's part: as they leave the accumulators, or, with kSplit (one chunk),
// from the sums behind the last accumulation.
template <int BN, bool kSplit, class Release, class Work>
__device__ __forceinline__ void for_chunks(const EpiContext& c, Block& sums, Release release, Work work) {
  constexpr int kChunks = Shape<BN>::kCols / 32;
  if constexpr (kSplit) {
    static_assert(kChunks == 1, "sums of 64 columns do not fit the registers");
    load_block(c.tmem, [&](int j, int i, float2 x) {
      sums[j][i] = c.first ? x : make_float2(sums[j][i].x + x.x, sums[j][i].y + x.y);
    });
    release();
    if (c.last) work(0, sums);
  } else {
#pragma unroll 1
    for (int chunk = 0; chunk < kChunks; ++chunk) {
      Block v;
      load_block(c.tmem + chunk * 32, [&](int j, int i, float2 x) { v[j][i] = x; });
      if (chunk == kChunks - 1) release();
      work(chunk, v);
    }
  }
}

// A block as half-precision operands at `to` (rows of `ld`) and, with rows and columns exchanged, at `turned`, and with kSplit what
// that leaves, `low` elements behind.
template <bool kSplit>
__device__ __forceinline__ void store_operands(Block& v, __half* to, __half* turned, int64_t ld, int64_t low, int rows_left, int turned_left, uint8_t* staging, int lane) {
#pragma unroll
  for (int part = 0; part < (kSplit ? 2 : 1); ++part) {
    uint32_t w[4][4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        w[j][i] = pack_f16(v[j][i].x, v[j][i].y);
        if (kSplit && part == 0) {
          const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[j][i]));
          v[j][i] = make_float2(v[j][i].x - f.x, v[j][i].y - f.y);
        }
      }
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t x[4] = {w[0][i], w[1][i], w[2][i], w[3][i]};
      store_fragment(smem_u32(staging), i, x, lane);
    }
    __syncwarp();
    store_staged(staging, reinterpret_cast<uint16_t*>(to + part * low), ld, 16, rows_left, 32, lane);
    if (turned) {
      __syncwarp();
#pragma unroll
      for (int j = 0; j < 4; ++j) store_fragment_turned(smem_u32(staging), j, w[j], lane);
      __syncwarp();
      store_staged(staging, reinterpret_cast<uint16_t*>(turned + part * low), ld, 16, turned_left, 32, lane);
    }
  }
}

// Whether 32 x 32 results of a symmetric product from (row0, n0) on are this tile's to store, and their mirror image with them:
// inside the matrix; of tiles of 128 columns, whose blocks lie on either side of the diagonal, all but the upper halves
// of those on it, of others what is not above it.
template <int BN>
__device__ __forceinline__ bool needed(int row0, int n0, int M) {
  return row0 < M && n0 < M && (n0 <= row0 || (BN == kCtaRows && n0 / kCtaRows != row0 / kCtaRows));
}

// What a symmetric product becomes: A = X X^T, or B = a I + b A + c A^2.
struct Symmetric {
  Planes out;
  Planes a;               // of B: A; else hi is null
  const float* factor;    // of the first A: X = X0 * factor; else null
  float scale;            // of the accumulators
  float on_a, on_diagonal;
};
__device__ __forceinline__ float symmetric_scale(const Symmetric& e, int batch) {
  float scale = e.scale;
  if (e.factor) {
    const float f = __ldg(e.factor + batch);
    scale *= f;
    scale *= f;
  }
  return scale;
}

// Symmetric products with few tiles and a long K are split along it; the shares go to memory as they are, tile by tile, and
// symmetric_sum_kernel adds them.
template <bool kLow>
struct ShareOut {
  static constexpr bool kSplit = kLow;
  static constexpr bool kInt8 = false, kMnMajorB = false;
  static constexpr int kClusterCtas = 0, kShares = 1;
  struct Params {
    float* shares;          // [tile and split][256][BN]
  };
  template <int BN>
  static __device__ __forceinline__ void fetch(const Params&, const Product&, const EpiContext&, int, int) {}
  template <int BN>
  static __device__ __forceinline__ void begin(const Params&, const Product&, const EpiContext&, Block&) {}
  template <int BN, class Release>
  static __device__ __forceinline__ void drain(const Params& ep, const Product&, const EpiContext& c, Block& sums, Release release) {
    for_chunks<BN, kSplit>(c, sums, release, [&](int chunk, Block& v) {
      float* to = ep.shares + (static_cast<int64_t>(c.t) * kPairRows + static_cast<int>(c.rank & 1u) * kCtaRows + c.row + (c.lane >> 2)) * BN +
                  c.part * Shape<BN>::kCols + 32 * chunk + 2 * (c.lane & 3);
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) *reinterpret_cast<float2*>(to + 8 * i * BN + 8 * j) = v[j][i];
    });
  }
};

template <int BN>
__global__ void __launch_bounds__(256) symmetric_sum_kernel(const __grid_constant__ Product p, const __grid_constant__ Symmetric e, const float* shares) {
  __shared__ float turned[32][33];
  hb_grid_dependency_wait();
  constexpr int kAcross = BN / 32, kPieces = kPairRows / 32 * kAcross;
  const int t = static_cast<int>(blockIdx.x) / kPieces, piece = static_cast<int>(blockIdx.x) % kPieces;
  // tile t of all batches, as with one split
  Product one = p;
  one.splits = 1;
  const Tile tile = tile_of<BN>(one, t);
  const int down = piece / kAcross * 32;
  const int row0 = down < kCtaRows ? tile.m0 + down : tile.m1 + down - kCtaRows, n0 = tile.n0 + piece % kAcross * 32;
  if (!needed<BN>(row0, n0, p.M)) return;
  const int tx = static_cast<int>(threadIdx.x) & 31, ty = static_cast<int>(threadIdx.x) >> 5;
  const int in_batch = t - tile.batch * p.per_batch;
  const float scale = symmetric_scale(e, tile.batch);
  __half* out = e.out.hi + tile.batch * e.out.batch_stride;
  // A's values and up to eight shares of each of four rows are on their way at once (one after the other, 25 shares of 150 x 150
  // results took 20 us; five steps of a 150 x 8000 update 192 us, 161 so); they are added in their order
  float a[4], sums[4] = {};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = row0 + ty + 8 * i, c = n0 + tx;
    a[i] = 0.0f;
    if (e.a.hi && r < p.M && c < p.M) {
      const __half* at = e.a.hi + tile.batch * e.a.batch_stride + static_cast<int64_t>(r) * e.a.ld + c;
      a[i] = __half2float(*at);
      if (e.a.low) a[i] += __half2float(at[e.a.low]);
    }
  }
  const int64_t share = static_cast<int64_t>(p.per_batch) * kPairRows * BN;
  const float* from = shares + tile.batch * p.splits * share + (static_cast<int64_t>(in_batch) * kPairRows + down + ty) * BN + piece % kAcross * 32 + tx;
  constexpr int kAtOnce = 8;
  for (int k0 = 0; k0 < p.splits; k0 += kAtOnce) {
    float x[kAtOnce][4];
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i) x[k][i] = k0 + k < p.splits ? from[(k0 + k) * share + 8 * i * BN] : 0.0f;
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i) sums[i] += x[k][i];
  }
#pragma unroll
  for (int i = 0; i < 32; i += 8) {
    const int r = row0 + ty + i, c = n0 + tx;
    const float v = fmaf(e.on_a, a[i / 8], sums[i / 8] * scale) + (e.a.hi && r == c ? e.on_diagonal : 0.0f);
    if (r < p.M && c < p.M && (n0 != row0 || c <= r)) {
      const __half hi = __float2half_rn(v);
      __half* to = out + static_cast<int64_t>(r) * e.out.ld + c;
      *to = hi;
      if (e.out.low) to[e.out.low] = __float2half_rn(v - __half2float(hi));
    }
    turned[ty + i][tx] = v;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 32; i += 8) {
    const int c = n0 + ty + i, r = row0 + tx;
    if (r >= p.M || c >= p.M || (n0 == row0 && c >= r)) continue;
    const float v = turned[tx][ty + i];
    const __half hi = __float2half_rn(v);
    __half* to = out + static_cast<int64_t>(c) * e.out.ld + r;
    *to = hi;
    if (e.out.low) to[e.out.low] = __float2half_rn(v - __half2float(hi));
  }
}

// Symmetric results: A = X X^T, or B = a I + b A + c A^2, as half-precision operands (kSplit: high and low parts).
template <bool kLow, int kPairs>
struct SymmetricOut {
  static constexpr bool kSplit = kLow;
  static constexpr bool kInt8 = false, kMnMajorB = false;
  static constexpr int kClusterCtas = 0, kShares = kPairs;
  using Params = Symmetric;
  template <int BN>
  static __device__ __forceinline__ void fetch(const Params&, const Product&, const EpiContext&, int, int) {}
  // b A + a I of the 32 x 32 results from (row0, n0) on.
  static __device__ __forceinline__ void other_terms(const Params& ep, const Product& p, const EpiContext& c, int row0, int n0, Block& v) {
    const int r = c.lane >> 2, n = 2 * (c.lane & 3);
    const __half* at = ep.a.hi + c.batch * ep.a.batch_stride + static_cast<int64_t>(row0 + r) * ep.a.ld + n0 + n;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const bool there = row0 + r + 8 * i < p.M;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float2 f = make_float2(0.0f, 0.0f);
        if (there) {
          f = __half22float2(*reinterpret_cast<const __half2*>(at + 8 * i * ep.a.ld + 8 * j));
          if (kSplit) {
            const float2 g = __half22float2(*reinterpret_cast<const __half2*>(at + ep.a.low + 8 * i * ep.a.ld + 8 * j));
            f = make_float2(f.x + g.x, f.y + g.y);      // 22 bits
          }
        }
        v[j][i] = make_float2(ep.on_a * f.x, ep.on_a * f.y);
      }
    }
    if (n0 == row0) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (n == r) v[j][j].x += ep.on_diagonal;
        if (n + 1 == r) v[j][j].y += ep.on_diagonal;
      }
    }
  }
  // The other terms are where the sums begin, read while the first slots are on their way: behind the last accumulation they took
  // 2,900 cycles of latency (five steps of a 200 x 200 float32 update 114 us, 103 so).
  template <int BN>
  static __device__ __forceinline__ void begin(const Params& ep, const Product& p, EpiContext& c, Block& sums) {
    c.scale = symmetric_scale(ep, c.batch);
    expect_shares<BN, SymmetricOut>(c);
    if (Shape<BN>::kCols > 32) return;
    if (ep.a.hi && needed<BN>(c.row0, c.n0, p.M) && (kShares == 1 || c.part % kShares == static_cast<int>(c.rank >> 1))) {
      other_terms(ep, p, c, c.row0, c.n0, sums);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) sums[j][i] = make_float2(0.0f, 0.0f);
    }
  }
  template <int BN, class Release>
  static __device__ __forceinline__ void drain(const Params& ep, const Product& p, const EpiContext& c, Block& sums, Release release) {
    auto store = [&](int n0, Block& v) {
      if (!needed<BN>(c.row0, n0, p.M)) return;
      // and those off the diagonal to their mirror image
      __half* base = ep.out.hi + c.batch * ep.out.batch_stride;
      store_operands<kSplit>(v, base + static_cast<int64_t>(c.row0) * ep.out.ld + n0,
                             n0 != c.row0 ? base + static_cast<int64_t>(n0) * ep.out.ld + c.row0 : nullptr, ep.out.ld, ep.out.low, p.M - c.row0,
                             p.M - n0, c.tail->staging + c.warp * kStageOutBytes, c.lane);
    };
    constexpr int kChunks = Shape<BN>::kCols / 32;
    if constexpr (kChunks == 1) {
      load_block(c.tmem, [&](int j, int i, float2 x) {
        sums[j][i] = make_float2(fmaf(c.scale, x.x, sums[j][i].x), fmaf(c.scale, x.y, sums[j][i].y));
      });
      release();
      if (kSplit && !c.last) return;
      if constexpr (kShares > 1)
        if (!join_shares<BN, SymmetricOut>(p, c, sums)) return;
      store(c.n0, sums);
    } else {
      static_assert(!kSplit, "sums of 64 columns do not fit the registers");
#pragma unroll 1
      for (int chunk = 0; chunk < kChunks; ++chunk) {
        const int n0 = c.n0 + chunk * 32;
        Block v = {};
        if (ep.a.hi && needed<BN>(c.row0, n0, p.M)) other_terms(ep, p, c, c.row0, n0, v);
        load_block(c.tmem + chunk * 32, [&](int j, int i, float2 x) {
          v[j][i] = make_float2(fmaf(c.scale, x.x, v[j][i].x), fmaf(c.scale, x.y, v[j][i].y));
        });
        if (chunk == kChunks - 1) release();
        store(n0, v);
      }
    }
  }
};

// X <- B X as operands of the next step, or as the result.
struct Step {
  Planes x;               // the next X; hi null: the result
  Out out;
  int32_t flip;           // the result is transposed
  const float* factor;    // of the first step
  float scale;
};
template <bool kLow, int kPairs>
struct UpdateOut {
  static constexpr bool kSplit = kLow;
  static constexpr bool kInt8 = false, kMnMajorB = true;
  static constexpr int kClusterCtas = 0, kShares = kPairs;
  using Params = Step;
  template <int BN>
  static __device__ __forceinline__ void fetch(const Params&, const Product&, const EpiContext&, int, int) {}
  template <int BN>
  static __device__ __forceinline__ void begin(const Params&, const Product&, const EpiContext& c, Block&) {
    expect_shares<BN, UpdateOut>(c);
  }
  template <int BN, class Release>
  static __device__ __forceinline__ void drain(const Params& ep, const Product& p, const EpiContext& c, Block& sums, Release release) {
    const int row0 = c.row0;
    const float scale = ep.factor ? ep.scale * __ldg(ep.factor + c.batch) : ep.scale;
    uint8_t* staging = c.tail->staging + c.warp * kStageOutBytes;
    for_chunks<BN, kSplit>(c, sums, release, [&](int chunk, Block& v) {
      if constexpr (kShares > 1)
        if (!join_shares<BN, UpdateOut>(p, c, v)) return;
      const int n0 = c.n0 + chunk * 32;
      if (n0 >= p.N || row0 >= p.M) return;
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) v[j][i] = make_float2(v[j][i].x * scale, v[j][i].y * scale);
      if (ep.x.hi) {
        store_operands<kSplit>(v, ep.x.hi + c.batch * ep.x.batch_stride + static_cast<int64_t>(row0) * ep.x.ld + n0, nullptr, ep.x.ld, ep.x.low, p.M - row0, 0,
                               staging, c.lane);
        return;
      }
      // rows and columns of the result from here on
      const int64_t first = c.batch * ep.out.batch_stride + (ep.flip ? static_cast<int64_t>(n0) * ep.out.ld + row0 : static_cast<int64_t>(row0) * ep.out.ld + n0);
      const int rows_left = p.M - row0, cols_left = p.N - n0;
      if (ep.out.type == kF32) {
        const int r = c.lane >> 2, n = 2 * (c.lane & 3);
        float* to = static_cast<float*>(ep.out.base) + first;
        const int64_t down = ep.flip ? 1 : ep.out.ld, across = ep.flip ? ep.out.ld : 1;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (8 * i + r >= rows_left) continue;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            float* at = to + (8 * i + r) * down + (8 * j + n) * across;
            if (!ep.flip && ep.out.vec >= 8 && 8 * j + n + 1 < cols_left) {
              *reinterpret_cast<float2*>(at) = v[j][i];
            } else {
              if (8 * j + n < cols_left) at[0] = v[j][i].x;
              if (8 * j + n + 1 < cols_left) at[across] = v[j][i].y;
            }
          }
        }
        return;
      }
      __syncwarp();
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        uint32_t w[4];
#pragma unroll
        for (int l = 0; l < 4; ++l) {
          const float2 x = ep.flip ? v[k][l] : v[l][k];
          w[l] = ep.out.type == kBF16 ? pack_bf16(x.x, x.y) : pack_f16(x.x, x.y);
        }
        if (ep.flip) store_fragment_turned(smem_u32(staging), k, w, c.lane);
        else store_fragment(smem_u32(staging), k, w, c.lane);
      }
      __syncwarp();
      store_staged(staging, static_cast<uint16_t*>(ep.out.base) + first, ep.out.ld, ep.out.vec, ep.flip ? cols_left : rows_left,
                   ep.flip ? rows_left : cols_left, c.lane);
    });
  }
};

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
int64_t up(int64_t x, int64_t m) { return (x + m - 1) / m * m; }

// Tiles of a symmetric product: with 128 columns two blocks each, else those whose columns begin before their rows end.
int64_t lower_tiles(int64_t s, int bn) {
  if (bn == kCtaRows) return two_block_tiles((s + kCtaRows - 1) / kCtaRows);
  const int64_t tm = (s + kPairRows - 1) / kPairRows, tn = (s + bn - 1) / bn, per = kPairRows / bn;
  int64_t n = 0;
  for (int64_t i = 0; i < tm; ++i) n += (i + 1) * per < tn ? (i + 1) * per : tn;
  return n;
}

constexpr int kMostPairs = 128;

// Times in units of 240 cycles: a slot of operands with low parts takes 4, of others 1, a second launch that adds shares from
// memory about 55, and sums that the pairs of a cluster exchange 15 and 7 (fitted to updates of 200 x 200 to 1024 x 1024).
constexpr int kSecondLaunch = 55;
int64_t slot_time(int64_t slots, bool split) { return slots * (split ? 4 : 1); }

// How many ways K of a symmetric product is split, the shares added by a second launch: as many as there are SM pairs for the
// tiles, of at least four slots; one unless that saves more than the launch takes.
int splits_of(int64_t batch, int64_t s, int64_t K, bool split, int pairs) {
  const int64_t tiles = batch * lower_tiles(s, 128), slots = (K + 63) / 64;
  int64_t n = pairs / tiles;
  if (n > slots / 4) n = slots / 4;
  if (n < 2) return 1;
  const int64_t each = (slots + n - 1) / n;
  if (slot_time(slots - each, split) < kSecondLaunch) return 1;
  return static_cast<int>((slots + each - 1) / each);      // none without slots
}

struct Layout {
  int64_t s, l, sp, lp;           // sides, and the pitches of rows of them
  int64_t x_bytes, a_bytes;       // one buffer of X, of A or B (all batches and planes)
  int64_t shares;                 // of products that are split along K
  int64_t total;
};
Layout layout_of(int64_t batch, int64_t rows, int64_t cols, bool split) {
  Layout r{};
  r.s = rows < cols ? rows : cols;
  r.l = rows < cols ? cols : rows;
  r.sp = up(r.s, 64);
  r.lp = up(r.l, 64);
  const int64_t planes = split ? 2 : 1;
  r.x_bytes = up(batch * planes * r.s * r.lp * 2, 256);
  r.a_bytes = up(batch * planes * r.s * r.sp * 2, 256);
  // of both symmetric products, for as many SM pairs as a GPU may have: with fewer there are no more splits
  if (batch > 0 && r.s > 0) {
    const int64_t tiles = batch * lower_tiles(r.s, 128);
    for (const int64_t K : {r.l, r.s}) {
      const int64_t n = splits_of(batch, r.s, K, split, kMostPairs), bytes = n > 1 ? tiles * n * kPairRows * 128 * 4 : 0;
      if (bytes > r.shares) r.shares = bytes;
    }
  }
  r.total = 2 * r.x_bytes + 2 * r.a_bytes + up(batch * 4, 256) + up(batch * kMostPartials * 8, 256) + r.shares;
  return r;
}

// Clusters of a product that the current GPU holds.
template <int BN, class Epi>
hb_status clusters_held(int* n) {
  static std::atomic<int> held[64];
  return max_clusters(gemm_kernel<BN, Epi>, 2 * Epi::kShares, Shape<BN>::kThreads, Ring<BN, Epi>::kSmem, held, n);
}

template <int BN, class Epi>
hb_status launch(Product p, const typename Epi::Params& ep, cudaStream_t s, Product* as_launched = nullptr) {
  int held = 0;
  auto kernel = gemm_kernel<BN, Epi>;
  if (const hb_status st = clusters_held<BN, Epi>(&held)) return st;
  p.tiles_m = static_cast<int32_t>((p.M + kPairRows - 1) / kPairRows);
  p.tiles_n = static_cast<int32_t>((p.N + BN - 1) / BN);
  const int64_t tiles = p.lower ? lower_tiles(p.M, BN) : static_cast<int64_t>(p.tiles_m) * p.tiles_n;
  if (tiles * p.batches * p.splits * kTileGroup > 0x7FFFFFFF) {
    hb::set_error("hb_orthogonalize: too large for one launch");
    return HB_ERR_TOO_LARGE;
  }
  set_tiles(&p, tiles);
  // pairs that share a tile have one each
  const int clusters = p.num_tiles < held || Epi::kShares > 1 ? p.num_tiles : held;
  HB_CUDA_TRY(launch_clusters(kernel, clusters, 2 * Epi::kShares, Shape<BN>::kThreads, Ring<BN, Epi>::kSmem, s, p, ep));
  if (as_launched) *as_launched = p;
  return HB_OK;
}

// How many pairs of a cluster share K of a product with `tiles` tiles of 128 columns: as many as make it shortest, where all its
// clusters run at once and every pair has a slot.  `alone`: what it takes otherwise.  (Five steps of a 777 x 1000 half-precision
// update, with the sums of all products exchanged or added by second launches: 159 and 213 us; 1024 x 1024 float32 176 and 220.)
int shares_of(int64_t tiles, int64_t K, bool split, const int (&held)[5], int64_t alone) {
  const int64_t slots = (K + 63) / 64;
  int best = 1;
  for (const int n : {2, 4}) {
    const int64_t each = (slots + n - 1) / n, cost = slot_time(each, split) + (split ? 15 : 7);
    if (tiles > held[n] || (n - 1) * each >= slots || cost >= alone) continue;
    alone = cost;
    best = n;
  }
  return best;
}

// The cluster that holds a matrix whose shorter side is at most 128: its CTAs, and blocks of 64 columns per CTA; 0 when it
// does not fit.
struct SidePlan {
  int ctas, blocks, R;
};
SidePlan side_plan(int64_t rows, int64_t cols, bool split) {
  const int64_t s = rows < cols ? rows : cols, l = rows < cols ? cols : rows;
  SidePlan r{0, 0, static_cast<int>(up(s, 16))};
  if (s < 1 || s > kSideRows || l > (1 << 20)) return r;
  const int64_t n = (l + kSideColumns - 1) / kSideColumns;
  for (const int ctas : {1, 2, 4, 8, 16}) {
    const int blocks = static_cast<int>((n + ctas - 1) / ctas);
    if (side_layout(r.R, blocks, split).total + 1024 > kSideSmem || (blocks > kSideBlocks && ctas < 16)) continue;
    r.ctas = ctas;
    r.blocks = blocks;
    break;
  }
  return r;
}

// The widest clusters of `kernel` (its shared memory `smem`) that the current GPU holds: 16, or 8 which every one does.
template <typename... KArgs>
hb_status widest_cluster(void (*kernel)(KArgs...), int threads, int smem, std::atomic<int>* held, std::atomic<int>* widest, int* out) {
  int dev = 0, n = 0;
  HB_CUDA_TRY(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64) {
    hb::set_error("device ordinal %d out of range", dev);
    return HB_ERR_UNSUPPORTED;
  }
  if (widest[dev].load() == 0) {
    HB_CUDA_TRY(cudaFuncSetAttribute(reinterpret_cast<const void*>(kernel), cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    const bool wide = max_clusters(kernel, 16, threads, smem, held, &n) == HB_OK;
    if (!wide) {
      cudaGetLastError();
      if (const hb_status st = max_clusters(kernel, 8, threads, smem, held, &n)) return st;
    }
    widest[dev].store(wide ? 16 : 8);
  }
  *out = widest[dev].load();
  return HB_OK;
}

// Matrices with a shorter side of at most 32: CTAs of a cluster, columns of each, shared memory; ctas 0 when they do not fit.
struct GramPlan {
  int ctas, columns, smem;
};
GramPlan gram_plan(int64_t s, int64_t l, int widest) {
  GramPlan r{0, 0, 0};
  if (s < 1 || s > kGramSide) return r;
  const int S = static_cast<int>(up(s, 8));
  for (int ctas = 1; ctas <= widest; ctas *= 2) {
    const int64_t columns = (l + ctas - 1) / ctas, smem = gram_smem(S, columns);
    if (smem > kSideSmem || (columns > 128 && ctas < widest)) continue;
    r.ctas = ctas;
    r.columns = static_cast<int>(columns);
    r.smem = static_cast<int>(smem);
    break;
  }
  return r;
}

// How many steps the recurrence of gram_side_kernel may take between two looks at X: what rounding leaves in A, 2^-53 of its norm by
// up to 32 terms, grows by the largest slope of t (a + b t + c t^2)^2 (at 0: a^2) per step, and has to be below 2^-24 when the last
// factor is made from it.  top: the largest eigenvalue of A.  The slope is of degree four: 64 points find its size.
int gram_stretch(double a, double b, double c, double top, int steps) {
  double slope = 1.0;
  for (int i = 0; i <= 64; ++i) {
    const double t = top * i / 64, y = a + t * (b + c * t);
    slope = std::fmax(slope, std::fabs(y * (y + 2.0 * t * (b + 2.0 * c * t))));
  }
  const double most = slope > 1.0 ? 24.0 / std::log2(slope) : steps;
  return most < steps ? 1 + static_cast<int>(most) : steps;
}

template <bool kSplit>
hb_status launch_side(const SidePlan& plan, int64_t batch, const SideParams& p, bool* launched, cudaStream_t s) {
  static std::atomic<int> held[64];
  static std::atomic<int> widest[64];
  auto kernel = small_side_kernel<kSplit>;
  int most = 0;
  if (const hb_status st = widest_cluster(kernel, kSideThreads, kSideSmem, held, widest, &most)) return st;
  if (plan.ctas > most || batch * plan.ctas > 0x7FFFFFFF) return HB_OK;
  HB_CUDA_TRY(launch_clusters(kernel, static_cast<int>(batch), plan.ctas, kSideThreads, kSideSmem, s, p));
  *launched = true;
  return HB_OK;
}

}  // namespace
}  // namespace dense

extern "C" int64_t hb_orthogonalize_workspace_bytes(int64_t batch, int64_t rows, int64_t cols, int32_t split) {
  if (batch < 0 || rows < 0 || cols < 0) return -1;
  return dense::layout_of(batch, rows, cols, split != 0).total;
}

extern "C" hb_status hb_orthogonalize(const void* update, int32_t type, int64_t batch, int64_t rows, int64_t cols, int64_t pitch,
                                      int64_t batch_stride, int32_t steps, const double* coefficients, double eps, int32_t split, void* out,
                                      int64_t out_pitch, int64_t out_batch_stride, void* workspace, int64_t workspace_bytes, void* stream) {
  using namespace dense;
  const char* name = "hb_orthogonalize";
  if (batch < 0 || rows < 0 || cols < 0 || type < HB_F32 || type > HB_F16 || pitch < cols || out_pitch < cols || steps < 1 || steps > 100 ||
      !coefficients || !(eps >= 0.0) || !std::isfinite(eps)) {
    hb::set_error("%s: sizes must not be negative, pitches at least cols, steps 1 to 100, eps finite and not negative", name);
    return HB_ERR_INVALID_ARGUMENT;
  }
  const double a = coefficients[0], b = coefficients[1], c = coefficients[2];
  // The largest singular value any step can leave, from at most one on: the maximum of |x (a + b x^2 + c x^4)| over what the
  // step before can leave; and the largest of B.  Stored operands are scaled by 2^8 and end at 65,504; A has the squares.
  double most = 1.0, most_b = 0.0, widest = 1.0;      // widest: the largest before any step
  for (int i = 0; i < steps && most <= 12.0 && most_b <= 250.0; ++i) {
    widest = std::fmax(widest, most);
    const double top = most * most;
    double next = 0.0;
    auto look = [&](double t) {          // t = x^2
      if (!(t >= 0.0 && t <= top)) return;
      const double y = std::fabs(a + t * (b + c * t)), x = std::sqrt(t);
      most_b = y <= 1e9 ? std::fmax(most_b, y) : 1e9;
      next = std::fmax(next, x * y);
    };
    // the ends, the factor's extremum, and those of x times it: a + 3 b t + 5 c t^2 = 0
    look(0.0);
    look(top);
    look(-b / (2.0 * c));
    const double root = std::sqrt(9.0 * b * b - 20.0 * a * c);
    look((-3.0 * b + root) / (10.0 * c));
    look((-3.0 * b - root) / (10.0 * c));
    look(-a / (3.0 * b));
    most = next * 1.001;
  }
  if (!(most <= 12.0) || !(most_b <= 250.0)) {
    hb::set_error("%s: with these coefficients the singular values grow beyond 12, or a factor beyond 250", name);
    return HB_ERR_INVALID_ARGUMENT;
  }
  int32_t* status = nullptr;
  if (const hb_status st = begin_call(name, &status)) return st;
  if (batch == 0 || rows == 0 || cols == 0) return HB_OK;
  if (!update || !out || !starts_on(update, bytes_of(type)) || !starts_on(out, bytes_of(type))) {
    hb::set_error("%s: NULL argument, or one that does not start on a boundary of its type", name);
    return HB_ERR_INVALID_ARGUMENT;
  }
  if (rows > (1 << 24) || cols > (1 << 24) || batch > 65535 || batch * 2 > 0x7FFFFFFF) {
    hb::set_error("%s: at most 65,535 matrices of sides up to 2^24", name);
    return HB_ERR_TOO_LARGE;
  }
  const Layout lay = layout_of(batch, rows, cols, split != 0);
  if (!workspace || workspace_bytes < lay.total || reinterpret_cast<uintptr_t>(workspace) % 256) {
    hb::set_error("%s: the workspace has to have %lld bytes, on a 256-byte boundary", name, static_cast<long long>(lay.total));
    return HB_ERR_INVALID_ARGUMENT;
  }
  const int flip = rows > cols ? 1 : 0;
  const Source g{update, pitch, batch_stride, type, static_cast<int32_t>(rows), static_cast<int32_t>(cols)};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  {
    const int64_t s = rows < cols ? rows : cols, l = rows < cols ? cols : rows;
    bool launched = false;
    auto gram = [&](auto size) -> hb_status {
      constexpr int S = decltype(size)::value;
      static std::atomic<int> held[64], held_width[64];
      int ctas = 0;
      if (const hb_status e = widest_cluster(gram_side_kernel<S>, kGramThreads, kSideSmem, held, held_width, &ctas)) return e;
      const GramPlan plan = gram_plan(s, l, ctas);
      if (!plan.ctas || batch * plan.ctas > 0x7FFFFFFF) return HB_OK;
      const GramParams p{g, Out{out, out_pitch, out_batch_stride, type, 0}, static_cast<int32_t>(s), static_cast<int32_t>(l), plan.columns, flip, steps,
                         gram_stretch(a, b, c, widest * widest, steps), a, b, c, eps};
      HB_CUDA_TRY(launch_clusters(gram_side_kernel<S>, static_cast<int>(batch), plan.ctas, kGramThreads, plan.smem, st, p));
      launched = true;
      return HB_OK;
    };
    hb_status e = HB_OK;
    if (s <= 8) e = gram(std::integral_constant<int, 8>{});
    else if (s <= 16) e = gram(std::integral_constant<int, 16>{});
    else if (s <= 24) e = gram(std::integral_constant<int, 24>{});
    else if (s <= 32) e = gram(std::integral_constant<int, 32>{});
    if (e != HB_OK || launched) return e;
  }
  if (const SidePlan plan = side_plan(rows, cols, split != 0); plan.ctas) {
    SideParams p{};
    p.g = g;
    p.out = Out{out, out_pitch, out_batch_stride, type, row_alignment(out, out_pitch, batch > 1 ? out_batch_stride : 0, bytes_of(type))};
    p.s = static_cast<int32_t>(rows < cols ? rows : cols);
    p.l = static_cast<int32_t>(rows < cols ? cols : rows);
    p.R = plan.R;
    p.blocks = plan.blocks;
    p.flip = flip;
    p.eights = !flip && row_alignment(update, pitch, batch > 1 ? batch_stride : 0, bytes_of(type)) == 16 ? 1 : 0;
    p.steps = steps;
    p.a = static_cast<float>(a);
    p.b = static_cast<float>(b);
    p.c = static_cast<float>(c);
    p.eps = eps;
    p.status = status;
    bool launched = false;
    if (const hb_status e = split ? launch_side<true>(plan, batch, p, &launched, st) : launch_side<false>(plan, batch, p, &launched, st)) return e;
    if (launched) return HB_OK;
  }
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  __half* x[2] = {reinterpret_cast<__half*>(ws), reinterpret_cast<__half*>(ws + lay.x_bytes)};
  __half* A = reinterpret_cast<__half*>(ws + 2 * lay.x_bytes);
  __half* B = reinterpret_cast<__half*>(ws + 2 * lay.x_bytes + lay.a_bytes);
  float* factor = reinterpret_cast<float*>(ws + 2 * lay.x_bytes + 2 * lay.a_bytes);
  double* partials = reinterpret_cast<double*>(reinterpret_cast<uint8_t*>(factor) + up(batch * 4, 256));
  float* shares = reinterpret_cast<float*>(reinterpret_cast<uint8_t*>(partials) + up(batch * kMostPartials * 8, 256));
  const int64_t planes = split ? 2 : 1;
  const int64_t x_matrix = lay.s * lay.lp, a_matrix = lay.s * lay.sp;
  auto x_planes = [&](int i) { return Planes{x[i], lay.lp, x_matrix, split ? batch * x_matrix : 0}; };
  const Planes a_planes{A, lay.sp, a_matrix, split ? batch * a_matrix : 0}, b_planes{B, lay.sp, a_matrix, split ? batch * a_matrix : 0};

  int64_t n_partials = up(rows * cols, kNormThreads * 16) / (kNormThreads * 16);
  // (64 blocks at least, as far as there are elements for them)
  const int64_t wanted = batch * 64 < kNormBlocks ? kNormBlocks / batch : 64;
  if (n_partials > wanted) n_partials = wanted;
  if (n_partials > kMostPartials) n_partials = kMostPartials;
  const int64_t between = batch > 1 ? batch_stride : 0;
  const bool eights = row_alignment(update, pitch, between, bytes_of(type)) == 16;
  const bool flat = pitch == cols && row_alignment(update, 0, between, bytes_of(type)) == 16;
  HB_CUDA_TRY(hb::launch_overlapped(norm_kernel, dim3(static_cast<unsigned>(n_partials), static_cast<unsigned>(batch)), dim3(kNormThreads), 0, st,
                                    g, flat ? 1 : 0, partials));
  const dim3 grid(static_cast<unsigned>((lay.l + 31) / 32), static_cast<unsigned>((lay.s + 31) / 32), static_cast<unsigned>(batch));
  if (grid.y > 65535) {
    hb::set_error("%s: the shorter side is at most 2,097,120", name);
    return HB_ERR_TOO_LARGE;
  }
  if (eights && !flip) {
    int64_t blocks = (up(cols, 8) / 8 * rows + 255) / 256;
    const int64_t most_blocks = (2 * kNormBlocks + batch - 1) / batch;
    if (blocks > most_blocks) blocks = most_blocks;
    HB_CUDA_TRY(hb::launch_overlapped(operand_rows_kernel, dim3(static_cast<unsigned>(blocks), static_cast<unsigned>(batch)), dim3(256), 0, st, g,
                                      static_cast<const double*>(partials), static_cast<int>(n_partials), eps, x_planes(0), factor));
  } else {
    HB_CUDA_TRY(hb::launch_overlapped(operand_kernel, grid, dim3(256), 0, st, g, static_cast<const double*>(partials), static_cast<int>(n_partials),
                                      eps, flip, x_planes(0), factor));
  }

  int sms = 0;
  if (const hb_status e = sm_count(&sms)) return e;
  const int pairs = sms / 2 < kMostPairs ? sms / 2 : kMostPairs;
  auto sym_tiles = [&](int bn) { return batch * lower_tiles(lay.s, bn); };
  auto upd_tiles = [&](int bn) { return batch * ((lay.s + kPairRows - 1) / kPairRows) * ((lay.l + bn - 1) / bn); };
  // sums for 64 columns per epilogue lane, a tile of 256, do not fit its registers (8192 x 4096 float32: 13.1 ms)
  const int bn_sym = split ? tile_columns({128, 64}, pairs, sym_tiles) : tile_columns({256, 128, 64}, pairs, sym_tiles);
  const int bn_upd = split ? 128 : tile_columns({256, 128}, pairs, upd_tiles);
  // pairs of a cluster that share K: of X X^T, A A and B X
  int held[5] = {};
  if (const hb_status e = split ? clusters_held<128, SymmetricOut<true, 2>>(&held[2]) : clusters_held<128, SymmetricOut<false, 2>>(&held[2])) return e;
  if (const hb_status e = split ? clusters_held<128, SymmetricOut<true, 4>>(&held[4]) : clusters_held<128, SymmetricOut<false, 4>>(&held[4])) return e;
  auto symmetric_shares = [&](int64_t K) {
    const int64_t slots = (K + 63) / 64, each_way = splits_of(batch, lay.s, K, split != 0, pairs);
    const int64_t alone = each_way > 1 ? slot_time((slots + each_way - 1) / each_way, split != 0) + kSecondLaunch
                                       : slot_time(slots, split != 0) * (bn_sym == 64 ? 3 : 4) / 4;
    return shares_of(sym_tiles(128), K, split != 0, held, alone);
  };
  const int gram_shares = symmetric_shares(lay.l), poly_shares = symmetric_shares(lay.s);
  const int upd_shares = shares_of(upd_tiles(128), lay.s, split != 0, held, slot_time((lay.s + 63) / 64, split != 0) * (bn_upd == 256 ? 2 : 1));
  auto symmetric_columns = [&](int64_t K, int shares) { return shares > 1 || splits_of(batch, lay.s, K, split != 0, pairs) > 1 ? 128 : bn_sym; };
  CUtensorMap x_rows[2], x_cols[2], x_k[2], a_rows, a_cols, b_rows;
  for (int i = 0; i < (steps > 1 ? 2 : 1); ++i) {
    HB_CUDA_TRY(encode_planes(&x_rows[i], x[i], 2, lay.l, lay.s, batch * planes, lay.lp, x_matrix, kCtaRows));
    HB_CUDA_TRY(encode_planes(&x_cols[i], x[i], 2, lay.l, lay.s, batch * planes, lay.lp, x_matrix, symmetric_columns(lay.l, gram_shares) / 2));
    HB_CUDA_TRY(encode_planes(&x_k[i], x[i], 2, lay.l, lay.s, batch * planes, lay.lp, x_matrix, 64));
  }
  HB_CUDA_TRY(encode_planes(&a_rows, A, 2, lay.s, lay.s, batch * planes, lay.sp, a_matrix, kCtaRows));
  HB_CUDA_TRY(encode_planes(&a_cols, A, 2, lay.s, lay.s, batch * planes, lay.sp, a_matrix, symmetric_columns(lay.s, poly_shares) / 2));
  HB_CUDA_TRY(encode_planes(&b_rows, B, 2, lay.s, lay.s, batch * planes, lay.sp, a_matrix, kCtaRows));

  const int32_t out_vec = row_alignment(out, out_pitch, batch > 1 ? out_batch_stride : 0, type == HB_F32 ? 4 : 2);
  auto run = [&](auto is_split) -> hb_status {
    constexpr bool kSplit = decltype(is_split)::value;
    using Sym = SymmetricOut<kSplit, 1>;
    using Upd = UpdateOut<kSplit, 1>;
    auto product = [&](const CUtensorMap& ma, const CUtensorMap& mb, int64_t N, int64_t K) {
      Product p{};
      p.a = ma;
      p.b = mb;
      p.M = static_cast<int32_t>(lay.s);
      p.N = static_cast<int32_t>(N);
      p.kblocks = static_cast<int32_t>((K + 63) / 64);
      p.batches = static_cast<int32_t>(batch);
      p.splits = 1;
      p.status = status;
      return p;
    };
    auto symmetric = [&](const CUtensorMap& ma, const CUtensorMap& mb, int64_t K, int shares_of_k, const typename Sym::Params& ep) -> hb_status {
      Product p = product(ma, mb, lay.s, K);
      p.lower = 1;
      if (shares_of_k == 2) return launch<128, SymmetricOut<kSplit, 2>>(p, ep, st);
      if (shares_of_k == 4) return launch<128, SymmetricOut<kSplit, 4>>(p, ep, st);
      p.splits = splits_of(batch, lay.s, K, kSplit, pairs);
      if (p.splits > 1) {
        if (const hb_status e = launch<128, ShareOut<kSplit>>(p, {shares}, st, &p)) return e;
        HB_CUDA_TRY(hb::launch_overlapped(symmetric_sum_kernel<128>, dim3(static_cast<unsigned>(p.num_tiles / p.splits * (kPairRows / 32) * 4)), dim3(256), 0,
                                          st, p, ep, static_cast<const float*>(shares)));
        return HB_OK;
      }
      if constexpr (!kSplit)
        if (bn_sym == 256) return launch<256, Sym>(p, ep, st);
      return bn_sym == 128 ? launch<128, Sym>(p, ep, st) : launch<64, Sym>(p, ep, st);
    };
    for (int i = 0; i < steps; ++i) {
      const int from = i & 1, to = from ^ 1;
      const bool first = i == 0, last = i == steps - 1;
      const typename Sym::Params gram{a_planes, Planes{}, first ? factor : nullptr, first ? kScale : 1.0f / kScale, 0.0f, 0.0f};
      if (const hb_status e = symmetric(x_rows[from], x_cols[from], lay.l, gram_shares, gram)) return e;
      // B 2^8 = b (A 2^8) + (c / 2^8) (A 2^8)^2 + a 2^8 I
      const typename Sym::Params poly{b_planes, a_planes, nullptr, static_cast<float>(c / kScale), static_cast<float>(b), static_cast<float>(a * kScale)};
      if (const hb_status e = symmetric(a_rows, a_cols, lay.s, poly_shares, poly)) return e;
      // (B 2^8)(X 2^8 or X0) -> X 2^8, or X
      const float scale = (first ? 1.0f : 1.0f / kScale) * (last ? 1.0f : kScale) / kScale;
      const Step ep{last ? Planes{} : x_planes(to), Out{out, out_pitch, out_batch_stride, type, out_vec}, flip, first ? factor : nullptr, scale};
      const Product p = product(b_rows, x_k[from], lay.l, lay.s);
      hb_status e = HB_OK;
      if (upd_shares == 2) e = launch<128, UpdateOut<kSplit, 2>>(p, ep, st);
      else if (upd_shares == 4) e = launch<128, UpdateOut<kSplit, 4>>(p, ep, st);
      else if constexpr (kSplit) e = launch<128, Upd>(p, ep, st);
      else e = bn_upd == 256 ? launch<256, Upd>(p, ep, st) : launch<128, Upd>(p, ep, st);
      if (e) return e;
    }
    return HB_OK;
  };
  return split ? run(std::true_type{}) : run(std::false_type{});
}
