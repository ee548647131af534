// The two ends of runtime predictors with 8-bit hidden layers: queries -> quantised rows behind fc1, and fc2 of quantised rows.
#include "dense_host.h"
#include "dense_quant.cuh"

namespace dense {
namespace {

constexpr int kInputThreads = 256;       // four features each: up to 1,024
constexpr int kInputQueries = 8;         // at a time
constexpr int kInputDevices = 256;

__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 r;
  asm("{\n\t.reg .b64 x, y, z, d;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 z, {%6, %7};\n\tfma.rn.f32x2 d, x, y, z;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return r;
}

// fc1 has at most 12 inputs: a thread keeps the weights of its four features in registers and walks over queries, eight between
// barriers, while the next eight are loaded and normalised.  12 multiply-adds per result on the ordinary cores, in pairs, are
// 11 us for 65,536 queries of 12 inputs, and the rows' 67 MB 10 us; 73 us measured.  What is left is what happens
// around the barrier, at which the largest value of a query crosses all eight warps before its first byte can be written: four queries at
// a time take 83 us, one CTA per SM 91, and three CTAs of fewer registers, four queries at a time, 87.
__global__ void __launch_bounds__(kInputThreads, 2)
mlp_input_kernel(const float* __restrict__ features, int n_op_feat, const uint8_t* __restrict__ device_row, const double* __restrict__ device_features,
                 int n_dev, const double* __restrict__ mu, const double* __restrict__ sigma, const float* __restrict__ w, const float* __restrict__ b,
                 int64_t Q, int width, int8_t* __restrict__ q, int64_t q_pitch, float* __restrict__ scales) {
  __shared__ __align__(16) float x[2][kInputQueries][kMaxInFeat];
  __shared__ __align__(16) float peak[2][kInputQueries][kInputThreads / 32];
  static_assert(kInputQueries == 8 && kInputThreads == 256, "eight queries by eight warps");
  __shared__ float devices[kInputDevices][4];                 // normalised
  const int tid = static_cast<int>(threadIdx.x), warp = tid >> 5, lane = tid & 31;
  const int inputs = n_op_feat + 4;
  hb_grid_dependency_wait();
  float2 wr[2][kMaxInFeat], br[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int f = 4 * tid + 2 * i;
    br[i] = make_float2(f < width ? b[f] : 0.0f, f + 1 < width ? b[f + 1] : 0.0f);
#pragma unroll
    for (int c = 0; c < kMaxInFeat; ++c)
      wr[i][c] = make_float2(f < width && c < inputs ? w[f * inputs + c] : 0.0f, f + 1 < width && c < inputs ? w[(f + 1) * inputs + c] : 0.0f);
  }
  for (int e = tid; e < 4 * n_dev; e += kInputThreads) {
    const int c = n_op_feat + (e & 3);
    devices[e >> 2][e & 3] = static_cast<float>((device_features[e] - mu[c]) / sigma[c]);
  }
  // thread e of the first 96 brings input e mod 12 of query e / 12
  const int mine_k = tid / kMaxInFeat, mine_c = tid - mine_k * kMaxInFeat;
  const bool brings = tid < kInputQueries * kMaxInFeat && mine_c < inputs;
  const double mine_mu = brings ? mu[mine_c] : 0.0, mine_sigma = brings ? sigma[mine_c] : 1.0;
  float raw = 0.0f;
  int row = 0;
  auto request = [&](int64_t q0) {
    if (!brings || q0 + mine_k >= Q) return;
    if (mine_c < n_op_feat) raw = features[(q0 + mine_k) * n_op_feat + mine_c];
    else row = device_row[q0 + mine_k];
  };
  auto put = [&](int buf) {
    if (!brings) return;
    x[buf][mine_k][mine_c] = mine_c < n_op_feat ? static_cast<float>((static_cast<double>(raw) - mine_mu) / mine_sigma)
                                                : devices[row < n_dev ? row : n_dev - 1][mine_c - n_op_feat];
  };
  const int64_t step = static_cast<int64_t>(gridDim.x) * kInputQueries;
  int64_t q0 = static_cast<int64_t>(blockIdx.x) * kInputQueries;
  request(q0);
  __syncthreads();                       // the devices
  put(0);
  __syncthreads();
  for (int buf = 0; q0 < Q; q0 += step, buf ^= 1) {
    request(q0 + step);
    float2 y[kInputQueries][2];
    float tops[kInputQueries];
#pragma unroll
    for (int k = 0; k < kInputQueries; ++k) {
      y[k][0] = br[0];
      y[k][1] = br[1];
      float xs[kMaxInFeat];
#pragma unroll
      for (int c = 0; c < kMaxInFeat; c += 4) {
        const float4 v = *reinterpret_cast<const float4*>(&x[buf][k][c]);
        xs[c] = v.x; xs[c + 1] = v.y; xs[c + 2] = v.z; xs[c + 3] = v.w;
      }
#pragma unroll
      for (int c = 0; c < kMaxInFeat; ++c) {
        if (c < inputs) {
          const float2 vv = make_float2(xs[c], xs[c]);
          y[k][0] = fma2(wr[0][c], vv, y[k][0]);
          y[k][1] = fma2(wr[1][c], vv, y[k][1]);
        }
      }
      // (ReLU: in the maxima, which begin at 0, and in the conversion below)
      tops[k] = max3(max3(0.0f, y[k][0].x, y[k][0].y), y[k][1].x, y[k][1].y);
    }
    // the warp's largest value of each query: halves of the queries over pairs of lanes, then what is left over all
#pragma unroll
    for (int n = kInputQueries / 2, d = 16; n; n /= 2, d /= 2) {
      const bool upper = (lane & d) != 0;
#pragma unroll
      for (int i = 0; i < n; ++i) {
        const float keep = upper ? tops[i + n] : tops[i], send = upper ? tops[i] : tops[i + n];
        tops[i] = max_nan(keep, __shfl_xor_sync(0xFFFFFFFFu, send, d));
      }
    }
    tops[0] = max_nan(tops[0], __shfl_xor_sync(0xFFFFFFFFu, tops[0], 2));
    tops[0] = max_nan(tops[0], __shfl_xor_sync(0xFFFFFFFFu, tops[0], 1));
    if ((lane & 3) == 0) peak[buf][lane >> 2][warp] = tops[0];      // lane bits 4, 3, 2 are the query's
    put(buf ^ 1);
    __syncthreads();
    // lane k mod 8 works out query k's scale for its warp
    const float4 lo = *reinterpret_cast<const float4*>(peak[buf][lane & 7]), hi = *reinterpret_cast<const float4*>(&peak[buf][lane & 7][4]);
    const float amax = max_nan(max_nan(max_nan(lo.x, lo.y), max_nan(lo.z, lo.w)), max_nan(max_nan(hi.x, hi.y), max_nan(hi.z, hi.w)));
    const RowScale s = row_scale(amax);
    if (tid < kInputQueries && q0 + tid < Q) scales[q0 + tid] = s.scale;
    const unsigned bad = __ballot_sync(0xFFFFFFFFu, s.bad);
#pragma unroll
    for (int k = 0; k < kInputQueries; ++k) {
      const float inverse = __shfl_sync(0xFFFFFFFFu, s.inverse, k);
      if (q0 + k >= Q) break;
      const uint32_t word = bad >> k & 1u ? 0 : quantized4<true>(y[k][0], y[k][1], inverse);
      int8_t* to = q + (q0 + k) * q_pitch + 4 * tid;
      if (4 * tid + 4 <= width) {
        *reinterpret_cast<uint32_t*>(to) = word;
      } else {
        for (int i = 0; 4 * tid + i < width; ++i) to[i] = static_cast<int8_t>(word >> (8 * i));
      }
    }
  }
}

// Byte i of a word of signed bytes whose signs are flipped, as a float: behind the exponent of 2^23 it counts from 128 on.  (The
// conversion instruction takes bytes at an eighth of this rate: 28 us.)
constexpr uint32_t kFlip = 0x80808080u;
__device__ __forceinline__ float byte_value(uint32_t word, int i) {
  return __uint_as_float(__byte_perm(word, 0x4B000000u, 0x7540u + i)) - 8388736.0f;
}

// A warp per row; a lane's 32 weights stay in registers.  65,536 rows of 1,024 features are 67 MB, 10 us; 22 us measured, about
// three instructions per byte.  The sum goes over the lanes as a fixed tree.
__global__ void __launch_bounds__(256)
mlp_output_kernel(const int8_t* __restrict__ q, int64_t q_pitch, const float* __restrict__ scales, const float* __restrict__ w, const float* __restrict__ b,
                  int64_t Q, int width, float* __restrict__ out) {
  const int lane = static_cast<int>(threadIdx.x) & 31;
  hb_grid_dependency_wait();
  float wr[32];
#pragma unroll
  for (int i = 0; i < 32; ++i) {
    const int f = (i >> 4) * 512 + 16 * lane + (i & 15);
    wr[i] = f < width ? w[f] : 0.0f;
  }
  const float bias = b[0];
  constexpr int kRows = 4;               // on their way at a time
  for (int64_t row = ((static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) >> 5) * kRows; row < Q; row += static_cast<int64_t>(gridDim.x) * 8 * kRows) {
    uint32_t ws[kRows][2][4];
#pragma unroll
    for (int r = 0; r < kRows; ++r)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        // the row's pitch is a multiple of 16; what lies behind its end has no weight, and is not read where nothing of the row is
        const int f = h * 512 + 16 * lane;
        const int8_t* at = q + (row + r) * q_pitch + f;
        uint4 v = make_uint4(0, 0, 0, 0);
        if (row + r < Q) {
          if (f + 16 <= width) {
            v = __ldg(reinterpret_cast<const uint4*>(at));
          } else if (f < width) {
            uint32_t t[4] = {0, 0, 0, 0};
#pragma unroll
            for (int i = 0; i < 16; ++i)
              if (f + i < width) t[i >> 2] |= static_cast<uint32_t>(static_cast<uint8_t>(at[i])) << (8 * (i & 3));
            v = make_uint4(t[0], t[1], t[2], t[3]);
          }
        }
        ws[r][h][0] = v.x ^ kFlip; ws[r][h][1] = v.y ^ kFlip; ws[r][h][2] = v.z ^ kFlip; ws[r][h][3] = v.w ^ kFlip;
      }
    float sums[kRows] = {};
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < 16; ++i)
#pragma unroll
        for (int r = 0; r < kRows; ++r)
          sums[r] = fmaf(byte_value(ws[r][h][i >> 2], i & 3), wr[16 * h + i], sums[r]);
#pragma unroll
    for (int d = 16; d; d >>= 1)
#pragma unroll
      for (int r = 0; r < kRows; ++r) sums[r] += __shfl_xor_sync(0xFFFFFFFFu, sums[r], d);
#pragma unroll
    for (int r = 0; r < kRows; ++r)
      if (lane == r && row + r < Q) out[row + r] = fmaf(sums[r], scales[row + r], bias);
  }
}

}  // namespace
}  // namespace dense

extern "C" hb_status hb_int8_mlp_input(const float* op_features, int32_t n_op_features, const uint8_t* device_row, const double* device_features,
                                       int32_t n_device_rows, const double* mu, const double* sigma, const float* w, const float* b, int64_t Q,
                                       int32_t width, int8_t* q, int64_t q_pitch, float* scales, void* stream) {
  if (Q < 0 || n_op_features < 1 || n_op_features + 4 > kMaxInFeat || width < 1 || width > 1024 || n_device_rows < 1 ||
      n_device_rows > dense::kInputDevices) {
    hb::set_error("hb_int8_mlp_input: 1 <= F <= 8, 1 <= width <= 1024, 1 to 256 device rows");
    return HB_ERR_UNSUPPORTED;
  }
  if (Q == 0) return HB_OK;
  if (!op_features || !device_row || !device_features || !mu || !sigma || !w || !b || !q || !scales || q_pitch < width || q_pitch % 16 ||
      reinterpret_cast<uintptr_t>(q) % 16) {
    hb::set_error("hb_int8_mlp_input: NULL argument, or rows of q that do not start on 16-byte boundaries");
    return HB_ERR_INVALID_ARGUMENT;
  }
  int sms = 0;
  if (const hb_status st = dense::sm_count(&sms)) return st;
  const int64_t rounds = (Q + dense::kInputQueries - 1) / dense::kInputQueries;
  const int64_t blocks = rounds < 2 * sms ? rounds : 2 * sms;
  HB_CUDA_TRY(hb::launch_overlapped(dense::mlp_input_kernel, dim3(static_cast<unsigned>(blocks)), dim3(dense::kInputThreads), 0,
                                    static_cast<cudaStream_t>(stream), op_features, n_op_features, device_row, device_features, n_device_rows, mu, sigma,
                                    w, b, Q, width, q, q_pitch, scales));
  return HB_OK;
}

extern "C" hb_status hb_int8_mlp_output(const int8_t* q, int64_t q_pitch, const float* scales, const float* w, const float* b, int64_t Q, int32_t width,
                                        float* out, void* stream) {
  if (Q < 0 || width < 1 || width > 1024) {
    hb::set_error("hb_int8_mlp_output: 1 <= width <= 1024");
    return HB_ERR_UNSUPPORTED;
  }
  if (Q == 0) return HB_OK;
  if (!q || !scales || !w || !b || !out || !dense::starts_on(out, 4) || q_pitch < width || q_pitch % 16 || reinterpret_cast<uintptr_t>(q) % 16) {
    hb::set_error("hb_int8_mlp_output: NULL argument, or rows of q that do not start on 16-byte boundaries");
    return HB_ERR_INVALID_ARGUMENT;
  }
  int sms = 0;
  if (const hb_status st = dense::sm_count(&sms)) return st;
  const int64_t blocks = (Q + 31) / 32 < 4 * sms ? (Q + 31) / 32 : 4 * sms;
  HB_CUDA_TRY(hb::launch_overlapped(dense::mlp_output_kernel, dim3(static_cast<unsigned>(blocks)), dim3(256), 0, static_cast<cudaStream_t>(stream), q, q_pitch,
                                    scales, w, b, Q, width, out));
  return HB_OK;
}
