// 8-bit products of few rows (tokens), bound by the weights' bytes and by latency: mma.sync tiles of 16 channels x 8 rows
// straight from memory, no shared memory in between.
//
// A lane loads 16 bytes of a channel's row (four lanes 64 bytes) and the same bytes of a token's; which of the 64 values of K an
// MMA takes for its k-th does not matter as long as both operands agree, so the two MMAs of a piece take the lanes' words
// 0, 1 and 2, 3.  Warps of a block share its channels and split K; their 32-bit sums are added in shared memory, exactly.
// 8 x 8192 x 8192: 27 us with tiles of 256 rows, whose slots are mostly empty rows.
#pragma once

#include "dense_gemm.cuh"
#include "dense_host.h"
#include "dense_quant.cuh"

namespace dense {
namespace {

constexpr int kFewRows = 16;             // the most rows that come here
constexpr int kFewAhead = 4;             // pieces of 64 values that a warp has on their way

struct FewParams {
  const int8_t* q;
  const int8_t* w;
  int64_t q_pitch, w_pitch;
  LayerScales s;
  int32_t M, N, K;
  Out out;                               // results
  int8_t* out_q;                         // or quantised rows
  int64_t out_pitch;
  float* out_scales;
};

__device__ __forceinline__ void mma_s8(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// 16 bytes of a row from byte k on, zeros from K on; no word that has none of the row's bytes is read.  Rows that start
// anywhere come in whole words and are shifted.
template <bool kAligned>
__device__ __forceinline__ uint4 load_piece(const int8_t* row, int k, int K) {
  if (k >= K) return make_uint4(0, 0, 0, 0);
  if (kAligned ? k + 16 <= K : k + 20 <= K) {
    if (kAligned) return __ldg(reinterpret_cast<const uint4*>(row + k));
    const uintptr_t at = reinterpret_cast<uintptr_t>(row + k);
    const uint32_t* words = reinterpret_cast<const uint32_t*>(at & ~static_cast<uintptr_t>(3));
    const uint32_t shift = static_cast<uint32_t>(at & 3u) * 8u;
    uint32_t w[5];
#pragma unroll
    for (int i = 0; i < 5; ++i) w[i] = __ldg(words + i);
    return make_uint4(__funnelshift_r(w[0], w[1], shift), __funnelshift_r(w[1], w[2], shift), __funnelshift_r(w[2], w[3], shift),
                      __funnelshift_r(w[3], w[4], shift));
  }
  uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll 1
  for (int i = 0; i < 16 && k + i < K; ++i) {
    const uint32_t byte = static_cast<uint32_t>(static_cast<uint8_t>(row[k + i])) << (8 * (i & 3));
    if (i < 4) w[0] |= byte;
    else if (i < 8) w[1] |= byte;
    else if (i < 12) w[2] |= byte;
    else w[3] |= byte;
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// kAligned: the channels' rows start on 16 bytes (the tokens' always do).  kTiles: groups of eight rows; kChannels: tiles of 16 channels per block; kSplits: warps that share a tile's K.  kQuant: a cluster has
// all channels and the result leaves as quantised rows.
template <int kTiles, int kChannels, int kSplits, bool kQuant, bool kAligned>
__global__ void __launch_bounds__(32 * kChannels * kSplits, kChannels == 1 && kTiles == 1 ? 4 : 1) few_rows_kernel(const __grid_constant__ FewParams p) {
  constexpr int kWarps = kChannels * kSplits, kRows = 8 * kTiles;
  __shared__ int sums[kSplits > 1 ? kWarps : 1][kTiles][4][32];
  __shared__ float peak[8][kRows];           // largest magnitudes of each CTA of the cluster
  __shared__ float warp_peak[kChannels][kRows];
  const int tid = static_cast<int>(threadIdx.x), warp = tid >> 5, lane = tid & 31;
  const int tile = warp % kChannels, split = warp / kChannels;
  const int g = lane >> 2, t = lane & 3;
  const int n0 = (static_cast<int>(blockIdx.x) * kChannels + tile) * 16;
  if (kQuant) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");      // "runs": waited for before its memory is written to
  hb_grid_dependency_wait();

  const int8_t* wr[2] = {p.w + static_cast<int64_t>(min(n0 + g, p.N - 1)) * p.w_pitch, p.w + static_cast<int64_t>(min(n0 + g + 8, p.N - 1)) * p.w_pitch};
  const int8_t* qr[kTiles];
#pragma unroll
  for (int i = 0; i < kTiles; ++i) qr[i] = p.q + static_cast<int64_t>(min(8 * i + g, p.M - 1)) * p.q_pitch;
  int acc[kTiles][4] = {};
  const int pieces = (p.K + 63) / 64;
  for (int p0 = split * kFewAhead; p0 < pieces; p0 += kSplits * kFewAhead) {
    uint4 a[kFewAhead][2], b[kFewAhead][kTiles];
#pragma unroll
    for (int j = 0; j < kFewAhead; ++j) {
      const int k = 64 * (p0 + j) + 16 * t;
#pragma unroll
      for (int i = 0; i < 2; ++i) a[j][i] = load_piece<kAligned>(wr[i], k, p.K);
#pragma unroll
      for (int i = 0; i < kTiles; ++i) b[j][i] = load_piece<true>(qr[i], k, p.K);
    }
#pragma unroll
    for (int j = 0; j < kFewAhead; ++j)
#pragma unroll
      for (int i = 0; i < kTiles; ++i) {
        mma_s8(acc[i], a[j][0].x, a[j][1].x, a[j][0].y, a[j][1].y, b[j][i].x, b[j][i].y);
        mma_s8(acc[i], a[j][0].z, a[j][1].z, a[j][0].w, a[j][1].w, b[j][i].z, b[j][i].w);
      }
  }
  if (kSplits > 1) {
#pragma unroll
    for (int i = 0; i < kTiles; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) sums[warp][i][j][lane] = acc[i][j];
    __syncthreads();
    if (split == 0) {
#pragma unroll
      for (int k = 1; k < kSplits; ++k)
#pragma unroll
        for (int i = 0; i < kTiles; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[i][j] += sums[k * kChannels + tile][i][j][lane];
    }
  }
  // acc[i][j]: channel n0 + g + 8 (j / 2), row 8 i + 2 t + j mod 2
  float v[kTiles][4];
  if (split == 0) {
    float w[2], b[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int n = n0 + g + 8 * h;
      w[h] = n < p.N ? __ldg(p.s.channel + n) : 0.0f;
      b[h] = n < p.N && p.s.bias ? __ldg(p.s.bias + n) : 0.0f;
    }
#pragma unroll
    for (int i = 0; i < kTiles; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int m = 8 * i + 2 * t + (j & 1), n = n0 + g + 8 * (j >> 1);
        const float rs = m < p.M ? __ldg(p.s.row + m) : 0.0f;
        float y = __fadd_rn(__fmul_rn(__fmul_rn(__int2float_rn(acc[i][j]), w[j >> 1]), rs), b[j >> 1]);
        if (p.s.relu) y = relu_nan(y);
        v[i][j] = y;
        if (!kQuant && m < p.M && n < p.N) {
          const int64_t at = m * p.out.ld + n;
          if (p.out.type == kF32) static_cast<float*>(p.out.base)[at] = y;
          else if (p.out.type == kBF16) static_cast<__nv_bfloat16*>(p.out.base)[at] = __float2bfloat16_rn(y);
          else static_cast<__half*>(p.out.base)[at] = __float2half_rn(y);
        }
      }
  }
  if (!kQuant) return;
  // ---- the rows' largest magnitudes over all channels of the cluster ----
  if (split == 0) {
#pragma unroll
    for (int i = 0; i < kTiles; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float m = n0 + g < p.N ? fabsf(v[i][j]) : 0.0f;
        m = max_nan(m, n0 + g + 8 < p.N ? fabsf(v[i][j + 2]) : 0.0f);
#pragma unroll
        for (int d = 4; d < 32; d *= 2) m = max_nan(m, __shfl_xor_sync(0xFFFFFFFFu, m, d));
        if (g == 0) warp_peak[tile][8 * i + 2 * t + j] = m;
      }
  }
  __syncthreads();
  uint32_t ctas, rank = cluster_ctarank();
  asm volatile("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(ctas));
  asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
  if (tid < kRows) {
    float m = 0.0f;
#pragma unroll
    for (int i = 0; i < kChannels; ++i) m = max_nan(m, warp_peak[i][tid]);
    for (uint32_t i = 0; i < ctas; ++i) st_cluster_f32(map_to_cta(smem_u32(&peak[rank][tid]), i), m);
  }
  __syncwarp();
  cluster_sync_all();
  if (split == 0) {
#pragma unroll
    for (int i = 0; i < kTiles; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int m = 8 * i + 2 * t + j;
        float top = 0.0f;
        for (uint32_t k = 0; k < ctas; ++k) top = max_nan(top, peak[k][m]);
        const RowScale s = row_scale(top);
        if (m >= p.M) continue;
        if (rank == 0 && tile == 0 && g == 0) p.out_scales[m] = s.scale;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int n = n0 + g + 8 * h;
          if (n < p.N) p.out_q[m * p.out_pitch + n] = s.bad ? 0 : static_cast<int8_t>(quantized(v[i][j + 2 * h], s.inverse));
        }
      }
  }
}

constexpr int kFewClusterChannels = 8;     // tiles of 16 channels per CTA of a cluster

template <int kTiles, bool kAligned>
cudaError_t launch_few_as(const FewParams& p, cudaStream_t s) {
  if (p.out_q) {
    const int ctas = (p.N + 16 * kFewClusterChannels - 1) / (16 * kFewClusterChannels);       // at most eight: N <= 1024
    return launch_clusters(few_rows_kernel<kTiles, kFewClusterChannels, 2, true, kAligned>, 1, ctas, 32 * kFewClusterChannels * 2, 0, s, p);
  }
  return hb::launch_overlapped(few_rows_kernel<kTiles, 1, 8, false, kAligned>, dim3(static_cast<unsigned>((p.N + 15) / 16)), dim3(256), 0, s, p);
}

hb_status launch_few(const FewParams& p, cudaStream_t s) {
  const bool aligned = reinterpret_cast<uintptr_t>(p.w) % 16 == 0 && p.w_pitch % 16 == 0;
  const cudaError_t e = p.M <= 8 ? (aligned ? launch_few_as<1, true>(p, s) : launch_few_as<1, false>(p, s))
                                 : (aligned ? launch_few_as<2, true>(p, s) : launch_few_as<2, false>(p, s));
  if (e != cudaSuccess) return hb::cuda_fail(e, "few_rows_kernel");
  return HB_OK;
}

}  // namespace
}  // namespace dense
