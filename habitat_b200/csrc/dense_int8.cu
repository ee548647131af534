// Dense layers in 8-bit integers: rows quantised with one scale each, products with one scale per row and per output
// channel, and the same with the result handed on as quantised rows.
//
// Definition (float32 arithmetic, every operation rounded to nearest): amax = max |x| of the row, q = rint(x * (127 / amax)),
// scale = amax / 127; y = (float(sum q w) * channel scale) * row scale + bias, then ReLU.  The integer sums are exact, so
// results do not depend on the order of the additions: all kernels here, and any other program that follows the
// definition, give the same bits.  Two exceptions to the formula: a row whose amax is below 2^-119 counts as zeros, since its scale would
// be a subnormal number of a few bits (and below 2^-121 127 / amax overflows); a row with an infinity or a NaN gets zeros and the
// scale NaN, so that its results are NaN and not finite numbers that look like some.
#include <atomic>
#include <cmath>
#include <type_traits>

#include "dense_gemm.cuh"
#include "dense_host.h"
#include "dense_quant.cuh"

namespace dense {
namespace {

constexpr int64_t kMostK = 131071;      // 128 * 128 * K stays below 2^31
constexpr int64_t kMostRows = 0x7FFFFF00;

// ---------------------------------------------------------------------------
// Quantisation
// ---------------------------------------------------------------------------
constexpr int kQuantThreads = 256;

// The largest value over the TPR threads that share a row, for all of them.
template <int TPR>
__device__ __forceinline__ float row_max(float v, float* scratch) {
#pragma unroll
  for (int d = 16; d; d >>= 1) v = max_nan(v, __shfl_xor_sync(0xFFFFFFFFu, v, d));
  if (TPR == 32) return v;
  if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
  __syncthreads();
  v = scratch[0];
#pragma unroll
  for (int i = 1; i < TPR / 32; ++i) v = max_nan(v, scratch[i]);
  return v;
}

// Bound by memory: a row is read once, into registers (TPR threads x VECS pieces of VB bytes: up to 4 KB with a warp per row,
// 32 KB with a block), and written from there.
template <typename T, int VB, int TPR, int VECS>
__global__ void __launch_bounds__(kQuantThreads)
quantize_vec_kernel(const T* __restrict__ x, int64_t rows, int cols, int64_t pitch, int8_t* __restrict__ q, int64_t q_pitch,
                    float* __restrict__ scales) {
  constexpr int kPer = VB / static_cast<int>(sizeof(T));
  using Piece = typename std::conditional<VB == 16, uint4, uint2>::type;
  using Bytes = typename std::conditional<kPer == 8, uint2, typename std::conditional<kPer == 4, uint32_t, uint16_t>::type>::type;
  __shared__ float scratch[kQuantThreads / 32];
  hb_grid_dependency_wait();
  const int64_t row = static_cast<int64_t>(blockIdx.x) * (kQuantThreads / TPR) + threadIdx.x / TPR;
  if (row >= rows) return;   // whole warps, and with TPR = 256 whole blocks
  const int t = static_cast<int>(threadIdx.x) % TPR;
  const T* xr = x + row * pitch;
  union {
    Piece u;
    T e[kPer];
  } v[VECS];
#pragma unroll
  for (int i = 0; i < VECS; ++i) {
    const int at = (i * TPR + t) * kPer;
    v[i].u = Piece{};
    if (at < cols) v[i].u = *reinterpret_cast<const Piece*>(xr + at);
  }
  float amax = 0.0f;
#pragma unroll
  for (int i = 0; i < VECS; ++i)
#pragma unroll
    for (int j = 0; j < kPer; ++j) amax = max_nan(amax, fabsf(to_float(v[i].e[j])));
  const RowScale s = row_scale(row_max<TPR>(amax, scratch));
  if (t == 0) scales[row] = s.scale;
  int8_t* qr = q + row * q_pitch;
#pragma unroll
  for (int i = 0; i < VECS; ++i) {
    const int at = (i * TPR + t) * kPer;
    uint32_t b[8];
#pragma unroll
    for (int j = 0; j < kPer; ++j) b[j] = s.bad ? 0 : quantized(to_float(v[i].e[j]), s.inverse);
    union {
      Bytes u;
      uint32_t w[2];
    } o;
    if constexpr (kPer == 2) {
      o.w[0] = __byte_perm(b[0], b[1], 0x0040);
    } else {
#pragma unroll
      for (int j = 0; j < kPer / 4; ++j) o.w[j] = low_bytes(b[4 * j], b[4 * j + 1], b[4 * j + 2], b[4 * j + 3]);
    }
    if (at < cols) *reinterpret_cast<Bytes*>(qr + at) = o.u;
  }
}

// Rows that start anywhere, or are longer than a block's registers: element by element, TPR threads per row with up to eight
// elements each in registers; longer rows are read twice (the second time from cache).
constexpr int kAnyElements = 8;
template <typename T, int TPR>
__global__ void __launch_bounds__(kQuantThreads)
quantize_any_kernel(const T* __restrict__ x, int64_t rows, int64_t cols, int64_t pitch, int8_t* __restrict__ q, int64_t q_pitch,
                    float* __restrict__ scales) {
  __shared__ float scratch[kQuantThreads / 32];
  hb_grid_dependency_wait();
  const int64_t row = static_cast<int64_t>(blockIdx.x) * (kQuantThreads / TPR) + threadIdx.x / TPR;
  if (row >= rows) return;
  const int t = static_cast<int>(threadIdx.x) % TPR;
  const T* xr = x + row * pitch;
  int8_t* qr = q + row * q_pitch;
  float amax = 0.0f;
  if (cols <= TPR * kAnyElements) {
    float v[kAnyElements];
#pragma unroll
    for (int i = 0; i < kAnyElements; ++i) v[i] = i * TPR + t < cols ? to_float(xr[i * TPR + t]) : 0.0f;
#pragma unroll
    for (int i = 0; i < kAnyElements; ++i) amax = max_nan(amax, fabsf(v[i]));
    const RowScale s = row_scale(row_max<TPR>(amax, scratch));
    if (t == 0) scales[row] = s.scale;
#pragma unroll
    for (int i = 0; i < kAnyElements; ++i)
      if (i * TPR + t < cols) qr[i * TPR + t] = s.bad ? 0 : static_cast<int8_t>(quantized(v[i], s.inverse));
    return;
  }
#pragma unroll 4
  for (int64_t i = t; i < cols; i += TPR) amax = max_nan(amax, fabsf(to_float(xr[i])));
  const RowScale s = row_scale(row_max<TPR>(amax, scratch));
  if (t == 0) scales[row] = s.scale;
#pragma unroll 4
  for (int64_t i = t; i < cols; i += TPR) qr[i] = s.bad ? 0 : static_cast<int8_t>(quantized(to_float(xr[i]), s.inverse));
}

template <typename T, int VB>
auto pick_vec(int64_t cols) -> decltype(&quantize_vec_kernel<T, VB, 32, 2>) {
  constexpr int64_t kPer = VB / sizeof(T);
  if (cols <= 32 * 2 * kPer) return quantize_vec_kernel<T, VB, 32, 2>;
  if (cols <= 32 * 4 * kPer) return quantize_vec_kernel<T, VB, 32, 4>;
  if (cols <= 32 * 8 * kPer) return quantize_vec_kernel<T, VB, 32, 8>;
  if (cols <= kQuantThreads * 2 * kPer) return quantize_vec_kernel<T, VB, kQuantThreads, 2>;
  if (cols <= kQuantThreads * 4 * kPer) return quantize_vec_kernel<T, VB, kQuantThreads, 4>;
  if (cols <= kQuantThreads * 8 * kPer) return quantize_vec_kernel<T, VB, kQuantThreads, 8>;
  return nullptr;
}

template <typename T>
cudaError_t launch_quantize(const void* x, int64_t rows, int64_t cols, int64_t pitch, int8_t* q, int64_t q_pitch, float* scales,
                            cudaStream_t s) {
  const T* xt = static_cast<const T*>(x);
  // pieces of 16 or 8 bytes that every row starts on and consists of
  auto whole = [&](int bytes) {
    const int64_t per = bytes / static_cast<int64_t>(sizeof(T));
    return reinterpret_cast<uintptr_t>(x) % bytes == 0 && (pitch % per == 0 || rows == 1) && cols % per == 0 &&
           reinterpret_cast<uintptr_t>(q) % per == 0 && (q_pitch % per == 0 || rows == 1);
  };
  auto vec = whole(16) ? pick_vec<T, 16>(cols) : whole(8) ? pick_vec<T, 8>(cols) : nullptr;
  if (vec) {
    const bool warp_row = cols <= 32 * 8 * (whole(16) ? 16 : 8) / static_cast<int64_t>(sizeof(T));
    const int64_t per = warp_row ? kQuantThreads / 32 : 1;
    return hb::launch_overlapped(vec, dim3(static_cast<unsigned>((rows + per - 1) / per)), dim3(kQuantThreads), 0, s, xt, rows,
                                 static_cast<int>(cols), pitch, q, q_pitch, scales);
  }
  // single elements: a warp per row while its registers hold one
  const bool warp_row = cols <= 32 * kAnyElements;
  const int64_t per = warp_row ? kQuantThreads / 32 : 1;
  return hb::launch_overlapped(warp_row ? quantize_any_kernel<T, 32> : quantize_any_kernel<T, kQuantThreads>,
                               dim3(static_cast<unsigned>((rows + per - 1) / per)), dim3(kQuantThreads), 0, s, xt, rows, cols, pitch, q,
                               q_pitch, scales);
}

struct LayerScales {
  const float* row;
  const float* channel;
  const float* bias;     // or null
  int32_t relu;
  float one;             // 1
};

}  // namespace
}  // namespace dense

#include "dense_few.cuh"

namespace dense {
namespace {

// Rows of bytes that start anywhere -> rows that start on 16 bytes (TMA reads nothing else), 16 bytes per thread; see load_piece.
__global__ void __launch_bounds__(256) align_rows_kernel(const int8_t* __restrict__ x, int rows, int K, int64_t pitch, int8_t* __restrict__ out,
                                                         int pieces) {
  hb_grid_dependency_wait();
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i >= static_cast<int64_t>(rows) * pieces) return;
  const int64_t r = i / pieces;
  const int k = static_cast<int>(i - r * pieces) * 16;
  reinterpret_cast<uint4*>(out)[i] = load_piece<false>(x + r * pitch, k, K);
}

// ---------------------------------------------------------------------------
// Epilogues
// ---------------------------------------------------------------------------

// A float from memory to shared memory, zero where there is none, without a register on the way: scales that were loaded a
// tile ahead into registers were spilled, which waits for them.
__device__ __forceinline__ void copy_float(const float* to, const float* from, bool there) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(smem_u32(to)), "l"(from), "r"(there ? 4 : 0) : "memory");
}
template <int BN>
__device__ __forceinline__ void fetch_scales(const LayerScales& s, const Product& p, const EpiContext& c, int row0, int n0, bool channels) {
  float* to = c.layer->scales[c.warp];
  if (channels) {
#pragma unroll
    for (int i = 0; i < Shape<BN>::kCols; i += 32) {
      const bool there = n0 + i + c.lane < p.N;
      const int n = there ? n0 + i + c.lane : 0;
      copy_float(to + i + c.lane, s.channel + n, there);
      copy_float(to + 64 + i + c.lane, (s.bias ? s.bias : s.channel) + n, there && s.bias);
    }
  }
  const bool there = row0 + c.lane < p.M;
  copy_float(to + 128 + c.lane, s.row + (there ? row0 + c.lane : 0), there);
}

// Two sums (mul2: two products).  A packed sum of packed products is merged into a multiply-add, which rounds once instead of twice,
// whatever the instructions' rounding says; y * one + b, with a one that only the host knows, is the rounded sum and stays as it is.
// (The epilogue is bound by its issue slots: with single sums and maxima quantised rows of 65,536 x 1024 x 1024 took 69 us,
// 63 so.)
__device__ __forceinline__ float2 add2(float2 a, float2 b, float one) {
  float2 r;
  asm("{\n\t.reg .b64 x, y, z, d;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%6, %6};\n\tmov.b64 z, {%4, %5};\n\tfma.rn.f32x2 d, x, y, z;\n\t"
      "mov.b64 {%0, %1}, d;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(one));
  return r;
}

// The warp's part of the tile as results before ReLU: v[j][i] are columns 8 j + 2 (lane mod 4) and the next of row 8 i + lane / 4.
template <int BN, class Release>
__device__ __forceinline__ void finish(const LayerScales& s, const Product& p, const EpiContext& c, float2 (&v)[Shape<BN>::kCols / 8][4],
                                       Release release) {
  constexpr int kCols = Shape<BN>::kCols;
  uint32_t acc[2][kCols / 2];
  load_fragment<kCols>(c.tmem, acc[0]);
  load_fragment<kCols>(c.tmem + (16u << 16), acc[1]);
  asm volatile("cp.async.wait_all;" ::: "memory");
  __syncwarp();
  const float* at = c.layer->scales[c.warp];
  const float2* sc = reinterpret_cast<const float2*>(at) + (c.lane & 3);
  float row[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) row[i] = at[128 + 8 * i + (c.lane >> 2)];
  tc_wait_ld();
  release();
#pragma unroll
  for (int j = 0; j < kCols / 8; ++j) {
    const float2 w = sc[4 * j], b = sc[32 + 4 * j];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t* a = &acc[i >> 1][4 * j + 2 * (i & 1)];
      const float2 x = make_float2(__int2float_rn(static_cast<int>(a[0])), __int2float_rn(static_cast<int>(a[1])));
      const float2 y = mul2(mul2(x, w), make_float2(row[i], row[i]));
      v[j][i] = add2(y, b, s.one);
    }
  }
  __syncwarp();
  if (c.next_row0 >= 0) fetch_scales<BN>(s, p, c, c.next_row0, c.next_n0, c.next_n0 != c.n0);
}

__device__ __forceinline__ float max3_abs(float a, float b, float c) {
  float r;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// Two results in 16 bits, with ReLU (NaN stays) in the conversion.
template <bool kRelu, bool kBf16>
__device__ __forceinline__ uint32_t pack_result(float2 x) {
  uint32_t r;
  if (!kRelu) return kBf16 ? pack_bf16(x.x, x.y) : pack_f16(x.x, x.y);
  if (kBf16) asm("cvt.rn.relu.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(x.y), "f"(x.x));
  else asm("cvt.rn.relu.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(x.y), "f"(x.x));
  return r;
}
template <bool kRelu, bool kBf16>
__device__ __forceinline__ void pack_results(const float2 (*v)[4], uint32_t (&w)[4][4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) w[i][j] = pack_result<kRelu, kBf16>(v[j][i]);
}

struct FloatOut {
  static constexpr bool kInt8 = true, kMnMajorB = false, kSplit = false;
  static constexpr int kClusterCtas = 0, kShares = 1;
  struct Params {
    LayerScales s;
    Out out;
  };
  template <int BN>
  static __device__ __forceinline__ void fetch(const Params& ep, const Product& p, const EpiContext& c, int row0, int n0) {
    fetch_scales<BN>(ep.s, p, c, row0, n0, true);
  }
  template <int BN>
  static __device__ __forceinline__ void begin(const Params&, const Product&, const EpiContext&, Block&) {}
  template <int BN, class Release>
  static __device__ __forceinline__ void drain(const Params& ep, const Product& p, const EpiContext& c, Block&, Release release) {
    constexpr int kBlocks = Shape<BN>::kCols / 8;
    float2 v[kBlocks][4];
    finish<BN>(ep.s, p, c, v, release);
    const int row0 = c.row0 + (c.lane >> 2);
    if (ep.out.type == kF32) {
      if (ep.s.relu) {
#pragma unroll
        for (int j = 0; j < kBlocks; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) v[j][i] = make_float2(relu_nan(v[j][i].x), relu_nan(v[j][i].y));
      }
      // four lanes fill a sector
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (row0 + 8 * i >= p.M) continue;
        float* to = static_cast<float*>(ep.out.base) + static_cast<int64_t>(row0 + 8 * i) * ep.out.ld + c.n0 + 2 * (c.lane & 3);
        const int left = p.N - c.n0 - 2 * (c.lane & 3);
        if (ep.out.vec >= 8) {
#pragma unroll
          for (int j = 0; j < kBlocks; ++j) {
            if (8 * j + 2 <= left) *reinterpret_cast<float2*>(to + 8 * j) = v[j][i];
            else if (8 * j < left) to[8 * j] = v[j][i].x;
          }
        } else {
#pragma unroll
          for (int j = 0; j < kBlocks; ++j) {
            if (8 * j < left) to[8 * j] = v[j][i].x;
            if (8 * j + 1 < left) to[8 * j + 1] = v[j][i].y;
          }
        }
      }
      return;
    }
    uint8_t* staging = c.tail->staging + c.warp * kStageOutBytes;
#pragma unroll
    for (int g = 0; g < kBlocks; g += 4) {         // 32 columns, 64 bytes, at a time
      uint32_t w[4][4];
      if (ep.out.type == kBF16) {
        if (ep.s.relu) pack_results<true, true>(v + g, w);
        else pack_results<false, true>(v + g, w);
      } else {
        if (ep.s.relu) pack_results<true, false>(v + g, w);
        else pack_results<false, false>(v + g, w);
      }
      __syncwarp();
#pragma unroll
      for (int i = 0; i < 4; ++i) store_fragment(smem_u32(staging), i, w[i], c.lane);
      __syncwarp();
      store_staged(staging, static_cast<uint16_t*>(ep.out.base) + static_cast<int64_t>(c.row0) * ep.out.ld + c.n0 + 8 * g, ep.out.ld, ep.out.vec,
                   p.M - c.row0, p.N - c.n0 - 8 * g, c.lane);
    }
  }
};

// The result as quantised rows.  The CTAs of a cluster hold whole rows between them (one pair per 256 columns): every lane
// keeps its 64 results in registers, a warp sends its rows' largest magnitudes to all CTAs of its row half through distributed
// shared memory (counted in bytes there: nobody waits for a store to be acknowledged), and quantises when the others' are
// there.  The accumulators are free before the exchange, so the next tile's MMAs run during it.
template <int kCtas>
struct QuantOut {
  static constexpr bool kInt8 = true, kMnMajorB = false, kSplit = false;
  static constexpr int kClusterCtas = kCtas, kShares = 1;
  struct Params {
    LayerScales s;
    int8_t* q;
    int64_t pitch;       // a multiple of 16, as is the address
    float* scales;
  };
  template <int BN>
  static __device__ __forceinline__ void fetch(const Params& ep, const Product& p, const EpiContext& c, int row0, int n0) {
    fetch_scales<BN>(ep.s, p, c, row0, n0, true);
  }
  template <int BN>
  static __device__ __forceinline__ void begin(const Params&, const Product&, const EpiContext& c, Block&) {
    if (c.part == 0 && c.lane == 0)
      mbar_expect_tx(smem_u32(&c.tail->exchange[c.n_tile & 1u][c.row >> 5]), kCtas / 2 * Shape<BN>::kParts * 32 * 4);
  }
  template <int BN, class Release>
  static __device__ __forceinline__ void drain(const Params& ep, const Product& p, const EpiContext& c, Block&, Release release) {
    constexpr int kBlocks = Shape<BN>::kCols / 8, kParts = Shape<BN>::kParts;
    float2 v[kBlocks][4];
    finish<BN>(ep.s, p, c, v, release);
    // the largest magnitude of each of the 32 rows; lane l goes on with row 8 (l mod 4) + l / 4
    float amax = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float m = 0.0f;
      if (ep.s.relu) {
#pragma unroll
        for (int j = 0; j < kBlocks; ++j) m = max3(m, v[j][i].x, v[j][i].y);
      } else {
#pragma unroll
        for (int j = 0; j < kBlocks; ++j) m = max3_abs(m, v[j][i].x, v[j][i].y);
      }
      m = max_nan(m, __shfl_xor_sync(0xFFFFFFFFu, m, 1));
      m = max_nan(m, __shfl_xor_sync(0xFFFFFFFFu, m, 2));
      if ((c.lane & 3) == i) amax = m;
    }
    const int mine = c.row + 8 * (c.lane & 3) + (c.lane >> 2);       // among the CTA's rows
    const uint32_t buf = c.n_tile & 1u, side = c.rank & 1u;
    const uint32_t bar = smem_u32(&c.tail->exchange[buf][c.row >> 5]);       // of the warps with the same 32 rows (one for all 128: 64 us, not 60.4)
    const uint32_t at = smem_u32(&c.layer->row_max[buf][c.rank >> 1][c.part][mine]);
#pragma unroll
    for (int i = 0; i < kCtas / 2; ++i) st_async_f32(map_to_cta(at, 2 * i + side), amax, map_to_cta(bar, 2 * i + side));
    if (!mbar_wait_cluster(bar, (c.n_tile >> 1) & 1u, &c.tail->abort, p.status, 0x541)) {
      *c.ok = false;
      return;
    }
#pragma unroll
    for (int i = 0; i < kCtas / 2; ++i)
#pragma unroll
      for (int j = 0; j < kParts; ++j) amax = max_nan(amax, c.layer->row_max[buf][i][j][mine]);
    const RowScale s = row_scale(amax);
    const int row = c.row0 + 8 * (c.lane & 3) + (c.lane >> 2);
    if (c.rank < 2 && c.part == 0 && row < p.M) ep.scales[row] = s.scale;
    const unsigned bad = __ballot_sync(0xFFFFFFFFu, s.bad);
    uint8_t* staging = c.tail->staging + c.warp * kStageOutBytes;
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int from = (c.lane & ~3) | i;                             // the lane that has row 8 i + lane / 4
      const float inverse = __shfl_sync(0xFFFFFFFFu, s.inverse, from);
      uint32_t w[4];                            // the lane's two columns of blocks 2 j and 2 j + 1
      if (ep.s.relu) {
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = quantized4<true>(v[2 * j][i], v[2 * j + 1][i], inverse);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = quantized4<false>(v[2 * j][i], v[2 * j + 1][i], inverse);
      }
      store_fragment(smem_u32(staging), i, w, c.lane);
    }
    __syncwarp();
    const int n = c.n0 + 16 * (c.lane & 3);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = c.row0 + 8 * i + (c.lane >> 2);
      if (r >= p.M) continue;
      const uint4 w = staged_row(staging, 8 * i + (c.lane >> 2), c.lane & 3);     // pairs of columns of two blocks in turn
      uint4 x = make_uint4(__byte_perm(w.x, w.y, 0x5410), __byte_perm(w.z, w.w, 0x5410), __byte_perm(w.x, w.y, 0x7632),
                           __byte_perm(w.z, w.w, 0x7632));
      if (bad >> ((c.lane & ~3) | i) & 1u) x = make_uint4(0, 0, 0, 0);
      int8_t* to = ep.q + static_cast<int64_t>(r) * ep.pitch + n;
      if (n + 16 <= p.N) {
        *reinterpret_cast<uint4*>(to) = x;
      } else {
        const uint32_t xs[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (n + e < p.N) to[e] = static_cast<int8_t>(xs[e >> 2] >> (8 * (e & 3)));
      }
    }
  }
};

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
int64_t round_up(int64_t x, int64_t m) { return (x + m - 1) / m * m; }
bool tma_rows(const void* p, int64_t pitch) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && pitch % 16 == 0; }

struct Operands {
  const int8_t* q;
  int64_t q_pitch;
  const int8_t* w;
  int64_t w_pitch;
};

hb_status check_product(const char* name, const int8_t* q, int64_t q_pitch, const float* q_scales, const int8_t* w, int64_t w_pitch,
                        const float* w_scales, const float* bias, int64_t M, int64_t N, int64_t K) {
  if (M < 0 || N < 0 || K < 1 || q_pitch < K || w_pitch < K) {
    hb::set_error("%s: M and N must not be negative, K at least 1, pitches at least K", name);
    return HB_ERR_INVALID_ARGUMENT;
  }
  if (M > kMostRows || N > kMostRows || K > kMostK) {
    hb::set_error("%s: K is at most 131071 (the sums are 32-bit integers), M and N below 2^31", name);
    return HB_ERR_TOO_LARGE;
  }
  if (M && N && (!q || !q_scales || !w || !w_scales)) {
    hb::set_error("%s: NULL argument", name);
    return HB_ERR_INVALID_ARGUMENT;
  }
  if (!starts_on(q_scales, 4) || !starts_on(w_scales, 4) || !starts_on(bias, 4)) {
    hb::set_error("%s: scales and biases start on 4-byte boundaries", name);
    return HB_ERR_INVALID_ARGUMENT;
  }
  return HB_OK;
}

int64_t align_bytes(int64_t rows, int64_t K, bool aligned) { return aligned ? 0 : round_up(rows * round_up(K, 16), 256); }

// Quantised results that take two launches, through float32 rows in memory: rows wider than a cluster of eight holds; few rows with
// so many columns that eight SMs cannot read the weights in the time (1 x 1024 x 8192: 20 us in one launch, 7 in two);
// and batches of up to two rounds of 256 rows, for which one cluster's SMs are the whole launch (127 x 1024 x 1024: 7.3 us in one
// launch, 6.7 in two; 127 x 1024 x 4096: 13.8 and 11.5; one after the other from the host both take 7.8 and 14.3, 12.5).
bool through_memory(int64_t M, int64_t N, int64_t K) { return N > 1024 || (M <= kFewRows ? K > 2048 : M <= 512); }

// Operands that TMA can read: as they are, or copied to the workspace.
hb_status align_operands(const char* name, Operands* o, int64_t M, int64_t N, int64_t K, uint8_t* workspace, int64_t workspace_bytes,
                         cudaStream_t s) {
  const bool q_ok = tma_rows(o->q, o->q_pitch), w_ok = tma_rows(o->w, o->w_pitch);
  const int64_t need = align_bytes(M, K, q_ok) + align_bytes(N, K, w_ok);
  if (need > 0 && (!workspace || workspace_bytes < need || reinterpret_cast<uintptr_t>(workspace) % 256)) {
    hb::set_error("%s: the workspace has to have %lld bytes, on a 256-byte boundary", name, static_cast<long long>(need));
    return HB_ERR_INVALID_ARGUMENT;
  }
  const int64_t pitch = round_up(K, 16);
  auto copy = [&](const int8_t** x, int64_t* x_pitch, int64_t rows) -> hb_status {
    const int64_t pieces = pitch / 16, blocks = (rows * pieces + 255) / 256;
    if (blocks > 0x7FFFFFFF) {
      hb::set_error("%s: too large to be copied to aligned rows", name);
      return HB_ERR_TOO_LARGE;
    }
    HB_CUDA_TRY(hb::launch_overlapped(align_rows_kernel, dim3(static_cast<unsigned>(blocks)), dim3(256), 0, s, *x, static_cast<int>(rows),
                                      static_cast<int>(K), *x_pitch, reinterpret_cast<int8_t*>(workspace), static_cast<int>(pieces)));
    *x = reinterpret_cast<const int8_t*>(workspace);
    *x_pitch = pitch;
    workspace += align_bytes(rows, K, false);
    return HB_OK;
  };
  if (!q_ok)
    if (const hb_status st = copy(&o->q, &o->q_pitch, M)) return st;
  if (!w_ok && M > kFewRows)       // few rows' kernel reads them as they are
    if (const hb_status st = copy(&o->w, &o->w_pitch, N)) return st;
  return HB_OK;
}

hb_status describe(Product* p, const Operands& o, int64_t M, int64_t N, int64_t K, int bn, int32_t* status) {
  HB_CUDA_TRY(encode_planes(&p->a, o.q, 1, K, M, 1, o.q_pitch, 0, kCtaRows));
  HB_CUDA_TRY(encode_planes(&p->b, o.w, 1, K, N, 1, o.w_pitch, 0, bn / 2));
  p->M = static_cast<int32_t>(M);
  p->N = static_cast<int32_t>(N);
  p->kblocks = static_cast<int32_t>((K + kSlotK - 1) / kSlotK);
  p->batches = 1;
  p->splits = 1;
  p->tiles_m = static_cast<int32_t>((M + kPairRows - 1) / kPairRows);
  p->tiles_n = static_cast<int32_t>((N + bn - 1) / bn);
  p->lower = 0;
  p->status = status;
  return HB_OK;
}

template <int BN>
hb_status launch_float(const Operands& o, int64_t M, int64_t N, int64_t K, const FloatOut::Params& ep, int32_t* status, cudaStream_t s) {
  static std::atomic<int> held[64];
  int pairs = 0;
  auto kernel = gemm_kernel<BN, FloatOut>;
  if (const hb_status st = max_clusters(kernel, 2, Shape<BN>::kThreads, Ring<BN, FloatOut>::kSmem, held, &pairs)) return st;
  Product p{};
  if (const hb_status st = describe(&p, o, M, N, K, BN, status)) return st;
  const int64_t tiles = static_cast<int64_t>(p.tiles_m) * p.tiles_n;
  if (tiles * kTileGroup > 0x7FFFFFFF) {
    hb::set_error("hb_int8_matmul: M x N too large for one launch");
    return HB_ERR_TOO_LARGE;
  }
  set_tiles(&p, tiles);
  const int clusters = p.num_tiles < pairs ? p.num_tiles : pairs;
  HB_CUDA_TRY(launch_clusters(kernel, clusters, 2, Shape<BN>::kThreads, Ring<BN, FloatOut>::kSmem, s, p, ep));
  return HB_OK;
}

template <int kCtas>
hb_status launch_quant(const Operands& o, int64_t M, int64_t N, int64_t K, const typename QuantOut<kCtas>::Params& ep, int32_t* status,
                       cudaStream_t s) {
  static std::atomic<int> held[64];
  int clusters = 0;
  auto kernel = gemm_kernel<256, QuantOut<kCtas>>;
  if (const hb_status st = max_clusters(kernel, kCtas, Shape<256>::kThreads, Ring<256, QuantOut<kCtas>>::kSmem, held, &clusters)) return st;
  Product p{};
  if (const hb_status st = describe(&p, o, M, N, K, 256, status)) return st;
  set_tiles(&p, p.tiles_m);
  if (p.num_tiles < clusters) clusters = p.num_tiles;
  HB_CUDA_TRY(launch_clusters(kernel, clusters, kCtas, Shape<256>::kThreads, Ring<256, QuantOut<kCtas>>::kSmem, s, p, ep));
  return HB_OK;
}

}  // namespace

hb_status sm_count(int* sms) {
  int dev = 0;
  HB_CUDA_TRY(cudaGetDevice(&dev));
  HB_CUDA_TRY(cudaDeviceGetAttribute(sms, cudaDevAttrMultiProcessorCount, dev));
  return HB_OK;
}

cudaError_t encode_planes(CUtensorMap* map, const void* base, int elem_bytes, int64_t cols, int64_t rows, int64_t planes, int64_t pitch,
                          int64_t plane_stride, int box_rows) {
  using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
  static std::atomic<void*> encode{nullptr};
  void* fn = encode.load();
  if (!fn) {
    cudaDriverEntryPointQueryResult found;
    const cudaError_t e = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &found);
    if (e != cudaSuccess) return e;
    if (!fn || found != cudaDriverEntryPointSuccess) return cudaErrorNotSupported;
    encode.store(fn);
  }
  const cuuint64_t dims[3] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows), static_cast<cuuint64_t>(planes)};
  // one plane: its stride is never used, but has to be a multiple of 16 bytes
  const cuuint64_t row_bytes = static_cast<cuuint64_t>(pitch) * elem_bytes;
  const cuuint64_t strides[2] = {row_bytes, planes > 1 ? static_cast<cuuint64_t>(plane_stride) * elem_bytes : row_bytes};
  const cuuint32_t box[3] = {static_cast<cuuint32_t>(128 / elem_bytes), static_cast<cuuint32_t>(box_rows), 1};
  const cuuint32_t elem[3] = {1, 1, 1};
  return reinterpret_cast<EncodeFn>(fn)(map, elem_bytes == 1 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3,
                                        const_cast<void*>(base), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
                                        CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS
             ? cudaSuccess
             : cudaErrorInvalidValue;
}

namespace {
std::mutex g_status_mu;
int32_t* g_status[64];
// Codes that the host has found in each GPU's word, and the last of them.  The word says nothing about whose launch it was, and whoever looks
// first takes it; so everyone who asks compares the count with the one they were last told of, host threads here
// (one more than that; 0: none yet), handles for themselves (hb_dense_failures).
std::atomic<int64_t> g_failures[64];
std::atomic<int32_t> g_code[64];
thread_local int64_t t_told[64];

hb_status status_word_of(int* dev, int32_t** word) {
  HB_CUDA_TRY(cudaGetDevice(dev));
  if (*dev < 0 || *dev >= 64) {
    hb::set_error("device ordinal %d out of range", *dev);
    return HB_ERR_UNSUPPORTED;
  }
  std::lock_guard<std::mutex> lock(g_status_mu);
  if (!g_status[*dev]) {
    void* p = nullptr;
    HB_CUDA_TRY(cudaHostAlloc(&p, 64, cudaHostAllocDefault));
    g_status[*dev] = static_cast<int32_t*>(p);
    *static_cast<volatile int32_t*>(g_status[*dev]) = 0;
  }
  *word = g_status[*dev];
  return HB_OK;
}

int64_t count_failures(int dev, int32_t* word) {
  if (*static_cast<volatile int32_t*>(word)) {
    if (const int32_t code = __atomic_exchange_n(word, 0, __ATOMIC_ACQ_REL)) {
      g_code[dev].store(code);
      g_failures[dev].fetch_add(1);
    }
  }
  return g_failures[dev].load();
}

// The last code where a launch has given up since this thread was last told, else 0.
int32_t news(int dev, int32_t* word) {
  int64_t& told = t_told[dev];
  if (told == 0) told = g_failures[dev].load() + 1;      // what others met before this thread's first call is theirs
  const int64_t now = count_failures(dev, word) + 1;
  if (now == told) return 0;
  told = now;
  return g_code[dev].load();
}
}  // namespace

hb_status begin_call(const char* name, int32_t** word) {
  int dev = 0;
  if (const hb_status st = status_word_of(&dev, word)) return st;
  if (const int32_t code = news(dev, *word)) {
    hb::set_error("%s: an earlier dense-layer launch gave up on a bounded wait (code 0x%x)", name, code);
    return HB_ERR_DEVICE_TIMEOUT;
  }
  return HB_OK;
}

hb_status dense_status(int32_t* code) {
  int dev = 0;
  int32_t* word = nullptr;
  if (const hb_status st = status_word_of(&dev, &word)) return st;
  HB_CUDA_TRY(cudaDeviceSynchronize());
  *code = news(dev, word);
  return HB_OK;
}

hb_status dense_failures(bool synchronise, int64_t* failures) {
  int dev = 0;
  int32_t* word = nullptr;
  if (const hb_status st = status_word_of(&dev, &word)) return st;
  if (synchronise) HB_CUDA_TRY(cudaDeviceSynchronize());
  *failures = count_failures(dev, word);
  return HB_OK;
}

hb_status inject_status(int32_t code) {
  int dev = 0;
  int32_t* word = nullptr;
  if (const hb_status st = status_word_of(&dev, &word)) return st;
  *static_cast<volatile int32_t*>(word) = code;
  return HB_OK;
}

}  // namespace dense

extern "C" hb_status hb_dense_status(int32_t* device_status) {
  if (!device_status) {
    hb::set_error("hb_dense_status: NULL argument");
    return HB_ERR_INVALID_ARGUMENT;
  }
  if (const hb_status st = dense::dense_status(device_status)) return st;
  if (*device_status) {
    hb::set_error("a dense-layer launch gave up on a bounded wait (code 0x%x)", *device_status);
    return HB_ERR_DEVICE_TIMEOUT;
  }
  return HB_OK;
}

extern "C" hb_status hb_dense_failures(int32_t synchronise, int64_t* failures) {
  if (!failures) {
    hb::set_error("hb_dense_failures: NULL argument");
    return HB_ERR_INVALID_ARGUMENT;
  }
  return dense::dense_failures(synchronise != 0, failures);
}

extern "C" hb_status hb_dense_inject_status(int32_t device_status) { return dense::inject_status(device_status); }

extern "C" hb_status hb_quantize_rows(const void* x, int32_t x_type, int64_t rows, int64_t cols, int64_t x_pitch, int8_t* q,
                                      int64_t q_pitch, float* scales, void* stream) {
  if (rows < 0 || cols < 1 || x_pitch < cols || q_pitch < cols || x_type < HB_F32 || x_type > HB_F16) {
    hb::set_error("hb_quantize_rows: rows must not be negative, cols at least 1, pitches at least cols");
    return HB_ERR_INVALID_ARGUMENT;
  }
  if (rows == 0) return HB_OK;
  if (!x || !q || !scales || !dense::starts_on(x, dense::bytes_of(x_type)) || !dense::starts_on(scales, 4)) {
    hb::set_error("hb_quantize_rows: NULL argument, or one that does not start on a boundary of its type");
    return HB_ERR_INVALID_ARGUMENT;
  }
  if (rows > dense::kMostRows) {
    hb::set_error("hb_quantize_rows: rows are below 2^31");
    return HB_ERR_TOO_LARGE;
  }
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  auto launch = x_type == HB_F32 ? dense::launch_quantize<float>
                                 : x_type == HB_BF16 ? dense::launch_quantize<__nv_bfloat16> : dense::launch_quantize<__half>;
  HB_CUDA_TRY(launch(x, rows, cols, x_pitch, q, q_pitch, scales, s));
  return HB_OK;
}

extern "C" int64_t hb_int8_workspace_bytes(const int8_t* q, int64_t q_pitch, const int8_t* w, int64_t w_pitch, int64_t M, int64_t N,
                                           int64_t K, int32_t quantized) {
  if (M < 0 || N < 0 || K < 1) return -1;
  int64_t bytes = dense::align_bytes(M, K, dense::tma_rows(q, q_pitch)) + dense::align_bytes(N, K, dense::tma_rows(w, w_pitch));
  if (quantized && dense::through_memory(M, N, K)) bytes += dense::round_up(M * dense::round_up(N, 4) * 4, 256);
  return bytes;
}

extern "C" hb_status hb_int8_matmul(const int8_t* q, int64_t q_pitch, const float* q_scales, const int8_t* w, int64_t w_pitch,
                                    const float* w_scales, const float* bias, int32_t relu, int64_t M, int64_t N, int64_t K, void* out,
                                    int32_t out_type, int64_t out_pitch, void* workspace, int64_t workspace_bytes, void* stream) {
  using namespace dense;
  const char* name = "hb_int8_matmul";
  if (const hb_status st = check_product(name, q, q_pitch, q_scales, w, w_pitch, w_scales, bias, M, N, K)) return st;
  if (out_type < HB_F32 || out_type > HB_F16 || out_pitch < N || (M && N && !out) || !starts_on(out, bytes_of(out_type))) {
    hb::set_error("%s: out has to be given, on a boundary of its type (0 to 2), with a pitch of at least N", name);
    return HB_ERR_INVALID_ARGUMENT;
  }
  int32_t* status = nullptr;
  if (const hb_status st = begin_call(name, &status)) return st;
  if (M == 0 || N == 0) return HB_OK;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  Operands o{q, q_pitch, w, w_pitch};
  if (const hb_status st = align_operands(name, &o, M, N, K, static_cast<uint8_t*>(workspace), workspace_bytes, s)) return st;
  FloatOut::Params ep{{q_scales, w_scales, bias, relu ? 1 : 0, 1.0f}, {out, out_pitch, 0, out_type, 0}};
  ep.out.vec = row_alignment(out, out_pitch, 0, out_type == HB_F32 ? 4 : 2);
  if (M <= kFewRows) {
    FewParams few{o.q, o.w, o.q_pitch, o.w_pitch, ep.s, static_cast<int32_t>(M), static_cast<int32_t>(N), static_cast<int32_t>(K), ep.out, nullptr, 0,
                  nullptr};
    return launch_few(few, s);
  }
  int sms = 0;
  if (const hb_status st = sm_count(&sms)) return st;
  switch (tile_columns({256, 128, 64}, sms / 2, [&](int bn) { return ((M + kPairRows - 1) / kPairRows) * ((N + bn - 1) / bn); })) {
    case 256: return launch_float<256>(o, M, N, K, ep, status, s);
    case 128: return launch_float<128>(o, M, N, K, ep, status, s);
    default: return launch_float<64>(o, M, N, K, ep, status, s);
  }
}

extern "C" hb_status hb_int8_matmul_quantized(const int8_t* q, int64_t q_pitch, const float* q_scales, const int8_t* w, int64_t w_pitch,
                                              const float* w_scales, const float* bias, int32_t relu, int64_t M, int64_t N, int64_t K,
                                              int8_t* out, int64_t out_pitch, float* out_scales, void* workspace, int64_t workspace_bytes,
                                              void* stream) {
  using namespace dense;
  const char* name = "hb_int8_matmul_quantized";
  if (const hb_status st = check_product(name, q, q_pitch, q_scales, w, w_pitch, w_scales, bias, M, N, K)) return st;
  if (M && (N < 1 || !out || !out_scales || !tma_rows(out, out_pitch) || out_pitch < N || !starts_on(out_scales, 4))) {
    hb::set_error("%s: out and out_scales have to be given, N at least 1, out's rows on 16-byte boundaries", name);
    return HB_ERR_INVALID_ARGUMENT;
  }
  int32_t* status = nullptr;
  if (const hb_status st = begin_call(name, &status)) return st;
  if (M == 0) return HB_OK;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  Operands o{q, q_pitch, w, w_pitch};
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  if (through_memory(M, N, K)) {
    const int64_t pitch = round_up(N, 4), bytes = round_up(M * pitch * 4, 256);
    const int64_t before = align_bytes(M, K, tma_rows(q, q_pitch)) + align_bytes(N, K, tma_rows(w, w_pitch));
    if (!ws || workspace_bytes < before + bytes || reinterpret_cast<uintptr_t>(ws) % 256) {
      hb::set_error("%s: the workspace has to have %lld bytes, on a 256-byte boundary", name, static_cast<long long>(before + bytes));
      return HB_ERR_INVALID_ARGUMENT;
    }
    float* y = reinterpret_cast<float*>(ws + before);
    if (const hb_status st = hb_int8_matmul(q, q_pitch, q_scales, w, w_pitch, w_scales, bias, relu, M, N, K, y, HB_F32, pitch, ws, before, stream))
      return st;
    return hb_quantize_rows(y, HB_F32, M, N, pitch, out, out_pitch, out_scales, stream);
  }
  if (const hb_status st = align_operands(name, &o, M, N, K, ws, workspace_bytes, s)) return st;
  const LayerScales scales{q_scales, w_scales, bias, relu ? 1 : 0, 1.0f};
  if (M <= kFewRows) {
    FewParams few{o.q, o.w, o.q_pitch, o.w_pitch, scales, static_cast<int32_t>(M), static_cast<int32_t>(N), static_cast<int32_t>(K), Out{}, out,
                  out_pitch, out_scales};
    return launch_few(few, s);
  }
  switch ((N + 255) / 256) {
    case 1: return launch_quant<2>(o, M, N, K, {scales, out, out_pitch, out_scales}, status, s);
    case 2: return launch_quant<4>(o, M, N, K, {scales, out, out_pitch, out_scales}, status, s);
    case 3: return launch_quant<6>(o, M, N, K, {scales, out, out_pitch, out_scales}, status, s);
    default: return launch_quant<8>(o, M, N, K, {scales, out, out_pitch, out_scales}, status, s);
  }
}
