// The two ends of runtime predictors with 8-bit hidden layers: queries -> quantised rows behind fc1, and fc2 of quantised rows.
#include "dense_host.h"
#include "dense_quant.cuh"

namespace dense {
namespace {

constexpr int kInputThreads = 256;       // four features each: up to 1,024
constexpr int kInputQueries = 8;         // at a time

// fc1 has at most 12 inputs: a thread keeps the weights of its four features in registers and walks over queries, eight between
// barriers.  12 multiply-adds per result on the ordinary cores are 22 us for 65,536 queries, and the rows' 67 MB 10 us.
__global__ void __launch_bounds__(kInputThreads)
mlp_input_kernel(const float* __restrict__ features, int n_op_feat, const uint8_t* __restrict__ device_row, const double* __restrict__ device_features,
                 int n_dev, const double* __restrict__ mu, const double* __restrict__ sigma, const float* __restrict__ w, const float* __restrict__ b,
                 int64_t Q, int width, int8_t* __restrict__ q, int64_t q_pitch, float* __restrict__ scales) {
  __shared__ float x[kInputQueries][kMaxInFeat];
  __shared__ float peak[kInputThreads / 32][kInputQueries];
  const int tid = static_cast<int>(threadIdx.x), warp = tid >> 5, lane = tid & 31;
  const int inputs = n_op_feat + 4;
  hb_grid_dependency_wait();
  float wr[4][kMaxInFeat], br[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int f = 4 * tid + i;
    br[i] = f < width ? b[f] : 0.0f;
#pragma unroll
    for (int c = 0; c < kMaxInFeat; ++c) wr[i][c] = f < width && c < inputs ? w[f * inputs + c] : 0.0f;
  }
  for (int64_t q0 = static_cast<int64_t>(blockIdx.x) * kInputQueries; q0 < Q; q0 += static_cast<int64_t>(gridDim.x) * kInputQueries) {
    __syncthreads();                     // the last queries' x and peak have been read
    for (int e = tid; e < kInputQueries * kMaxInFeat; e += kInputThreads) {
      const int k = e / kMaxInFeat, c = e - k * kMaxInFeat;
      float v = 0.0f;
      if (q0 + k < Q && c < inputs) {
        int row = device_row[q0 + k];
        row = row < n_dev ? row : n_dev - 1;
        const double y = c < n_op_feat ? static_cast<double>(features[(q0 + k) * n_op_feat + c]) : device_features[row * 4 + c - n_op_feat];
        v = static_cast<float>((y - mu[c]) / sigma[c]);
      }
      x[k][c] = v;
    }
    __syncthreads();
    float y[kInputQueries][4];
#pragma unroll
    for (int k = 0; k < kInputQueries; ++k) {
#pragma unroll
      for (int i = 0; i < 4; ++i) y[k][i] = br[i];
#pragma unroll
      for (int c = 0; c < kMaxInFeat; ++c) {
        const float v = x[k][c];
        if (c < inputs) {
#pragma unroll
          for (int i = 0; i < 4; ++i) y[k][i] = fmaf(wr[i][c], v, y[k][i]);
        }
      }
      float m = 0.0f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        y[k][i] = relu_nan(y[k][i]);
        m = max_nan(m, y[k][i]);
      }
#pragma unroll
      for (int d = 16; d; d >>= 1) m = max_nan(m, __shfl_xor_sync(0xFFFFFFFFu, m, d));
      if (lane == 0) peak[warp][k] = m;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kInputQueries; ++k) {
      if (q0 + k >= Q) break;
      float m = peak[0][k];
#pragma unroll
      for (int i = 1; i < kInputThreads / 32; ++i) m = max_nan(m, peak[i][k]);
      const RowScale s = row_scale(m);
      if (tid == 0) scales[q0 + k] = s.scale;
      const uint32_t word = s.bad ? 0 : low_bytes(quantized(y[k][0], s.inverse), quantized(y[k][1], s.inverse), quantized(y[k][2], s.inverse), quantized(y[k][3], s.inverse));
      int8_t* to = q + (q0 + k) * q_pitch + 4 * tid;
      if (4 * tid + 4 <= width) {
        *reinterpret_cast<uint32_t*>(to) = word;
      } else {
        for (int i = 0; 4 * tid + i < width; ++i) to[i] = static_cast<int8_t>(word >> (8 * i));
      }
    }
  }
}

// A warp per row, bound by the rows' bytes; a lane's 32 weights stay in registers.  The sum goes over the lanes as a fixed tree.
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
  for (int64_t row = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) >> 5; row < Q; row += static_cast<int64_t>(gridDim.x) * 8) {
    float sum = 0.0f;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int f = h * 512 + 16 * lane;
      // the row's pitch is a multiple of 16; what lies behind its end has no weight, and is not read where nothing of the row is
      if (f >= width) continue;
      const int8_t* at = q + row * q_pitch + f;
      uint32_t ws[4] = {0, 0, 0, 0};
      if (f + 16 <= width) {
        const uint4 v = __ldg(reinterpret_cast<const uint4*>(at));
        ws[0] = v.x; ws[1] = v.y; ws[2] = v.z; ws[3] = v.w;
      } else {
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (f + i < width) ws[i >> 2] |= static_cast<uint32_t>(static_cast<uint8_t>(at[i])) << (8 * (i & 3));
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) sum = fmaf(static_cast<float>(static_cast<int8_t>(ws[i >> 2] >> (8 * (i & 3)))), wr[16 * h + i], sum);
    }
#pragma unroll
    for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, d);
    if (lane == 0) out[row] = fmaf(sum, scales[row], bias);
  }
}

}  // namespace
}  // namespace dense

extern "C" hb_status hb_int8_mlp_input(const float* op_features, int32_t n_op_features, const uint8_t* device_row, const double* device_features,
                                       int32_t n_device_rows, const double* mu, const double* sigma, const float* w, const float* b, int64_t Q,
                                       int32_t width, int8_t* q, int64_t q_pitch, float* scales, void* stream) {
  if (Q < 0 || n_op_features < 1 || n_op_features + 4 > kMaxInFeat || width < 1 || width > 1024 || n_device_rows < 1) {
    hb::set_error("hb_int8_mlp_input: 1 <= F <= 8, 1 <= width <= 1024, at least one device row");
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
  if (!q || !scales || !w || !b || !out || q_pitch < width || q_pitch % 16 || reinterpret_cast<uintptr_t>(q) % 16) {
    hb::set_error("hb_int8_mlp_output: NULL argument, or rows of q that do not start on 16-byte boundaries");
    return HB_ERR_INVALID_ARGUMENT;
  }
  int sms = 0;
  if (const hb_status st = dense::sm_count(&sms)) return st;
  const int64_t blocks = (Q + 7) / 8 < 8 * sms ? (Q + 7) / 8 : 8 * sms;
  HB_CUDA_TRY(hb::launch_overlapped(dense::mlp_output_kernel, dim3(static_cast<unsigned>(blocks)), dim3(256), 0, static_cast<cudaStream_t>(stream), q, q_pitch,
                                    scales, w, b, Q, width, out));
  return HB_OK;
}
