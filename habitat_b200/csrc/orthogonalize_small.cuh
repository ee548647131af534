// Newton-Schulz steps of matrices whose shorter side is at most 128, in one launch: a cluster per matrix keeps X in shared
// memory, columns spread over its CTAs, for all steps.
//
// A step on tiles in memory is three launches of a few microseconds each whatever the size; here it is two barriers of
// the cluster.  Per step each CTA multiplies its columns to a share of A = X X^T, the shares are added slice by slice through
// distributed shared memory (in the order of the ranks) and the sums handed to every CTA, which works out A^2 and
// B = a I + b A + c A^2 for itself and replaces its columns by B X.  X lies as blocks of 64 columns, R rows of 128 bytes with
// the 128-byte swizzle: K-major for A (K = columns) and MN-major for B X (N = columns) with the same bytes.
//
// An MMA has 128 rows; of X, A and B only R (s rounded up to 16) are stored, so it reads into what lies behind.  Rows of D
// from R on are whatever that gives and are not read.
#pragma once

#include "dense_gemm.cuh"
#include "dense_host.h"

namespace dense {
namespace {

constexpr int kSideThreads = 256;
constexpr int kSideRows = 128;                 // the longest shorter side
constexpr int kSideSmem = 232448;              // all of an SM's, so that no two of these blocks share its tensor memory
constexpr int kSideColumns = 64;               // per block of X

struct SideTail {
  uint64_t done;
  uint32_t tmem;
  int abort;
  double sums[16];
  double warp_sums[kSideThreads / 32];
};

struct SideParams {
  Source g;
  Out out;
  int32_t s, l, R, blocks, flip, steps;   // blocks: of 64 columns, per CTA
  float a, b, c;
  double eps;
  int32_t* status;
};

// Bytes in front of the tail: X, the operands A then B, what an MMA reads behind them, the share of A.
struct SideLayout {
  int block, x, operand, share, total;
};
__host__ __device__ inline SideLayout side_layout(int R, int blocks, bool split) {
  SideLayout r;
  const int planes = split ? 2 : 1;
  r.block = R * 128;
  r.x = 0;
  r.operand = planes * blocks * r.block;
  // behind the last block up to 128 - R more rows are read
  const int operand_end = r.operand + planes * ((R + 63) / 64) * r.block;
  r.share = operand_end;
  const int share_end = r.share + R * (R + 4) * 4, read_end = operand_end + (kSideRows - R) * 128;
  r.total = ((share_end > read_end ? share_end : read_end) + 1023) / 1024 * 1024 + 1024;
  return r;
}

__device__ __forceinline__ void mma_one(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void commit_one(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ float4 ld_cluster_f4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ void st_cluster_u4(uint32_t addr, uint4 v) {
  asm volatile("st.shared::cluster.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
__device__ __forceinline__ void st_cluster_f64(uint32_t addr, double v) {
  asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(addr), "d"(v) : "memory");
}
__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t n;
  asm volatile("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(n));
  return n;
}

// Byte of element (row, column 0 .. 63) in a block.
__device__ __forceinline__ uint32_t block_at(int row, int col) {
  return static_cast<uint32_t>(row * 128 + ((((col >> 3) ^ row) & 7) << 4) + ((col & 7) << 1));
}

// Eight values in half precision, and what that leaves.
__device__ __forceinline__ uint4 halves(float (&v)[8]) {
  uint4 r;
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __half2 h = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
    w[i] = *reinterpret_cast<const uint32_t*>(&h);
    const float2 f = __half22float2(h);
    v[2 * i] -= f.x;
    v[2 * i + 1] -= f.y;
  }
  r.x = w[0]; r.y = w[1]; r.z = w[2]; r.w = w[3];
  return r;
}

template <bool kSplit>
__global__ void __launch_bounds__(kSideThreads, 1) small_side_kernel(const __grid_constant__ SideParams p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  const SideLayout lay = side_layout(p.R, p.blocks, kSplit);
  SideTail* tail = reinterpret_cast<SideTail*>(base + lay.total - 1024);
  const int tid = static_cast<int>(threadIdx.x), warp = tid >> 5, lane = tid & 31;
  const int rank = static_cast<int>(cluster_ctarank()), ctas = static_cast<int>(cluster_size());
  const int matrix = static_cast<int>(blockIdx.x) / ctas;
  const int R = p.R, nb = p.blocks;
  const int x_low = nb * lay.block;                       // from a high block of X to its low one
  const int k_blocks = (R + 63) / 64, op_low = k_blocks * lay.block;
  volatile int* abort_flag = &tail->abort;
  const uint32_t bar = smem_u32(&tail->done);
  uint32_t phase = 0;

  if (tid == 0) {
    mbar_init(bar, 1);
    tail->abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tail->tmem)), "r"(512u) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  for (int i = tid; i < (kSplit ? 2 : 1) * nb * lay.block / 16; i += kSideThreads)
    reinterpret_cast<uint4*>(base)[i] = make_uint4(0, 0, 0, 0);
  hb_grid_dependency_wait();

  // ---- the norm ----
  const int64_t g0 = matrix * p.g.batch_stride;
  const int c0 = rank * nb * kSideColumns;                              // this CTA's columns of X
  const int cols = min(max(p.l - c0, 0), nb * kSideColumns);
  const int n_el = p.s * cols;
  // walks the elements along G's rows: work(row of X, column of this CTA, value)
  auto for_elements = [&](auto work) {
    const int inner = p.flip ? p.s : cols;
    if (inner >= 32) {
      const int outer = p.flip ? cols : p.s;
      for (int o = warp; o < outer; o += kSideThreads / 32) {
        const int64_t row = g0 + static_cast<int64_t>(p.flip ? c0 + o : o) * p.g.ld + (p.flip ? 0 : c0);
#pragma unroll 4
        for (int i = lane; i < inner; i += 32) {
          const float x = load_element(p.g.base, p.g.type, row + i);
          if (p.flip) work(i, o, x);
          else work(o, i, x);
        }
      }
    } else {
#pragma unroll 4
      for (int e = tid; e < n_el; e += kSideThreads) {
        const int o = e / inner, i = e - o * inner;
        const float x = load_element(p.g.base, p.g.type, g0 + static_cast<int64_t>(p.flip ? c0 + o : o) * p.g.ld + (p.flip ? 0 : c0) + i);
        if (p.flip) work(i, o, x);
        else work(o, i, x);
      }
    }
  };
  double sum = 0.0;
  for_elements([&](int, int, float x) { sum += static_cast<double>(x) * x; });
#pragma unroll
  for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, d);
  if (lane == 0) tail->warp_sums[warp] = sum;
  __syncthreads();
  cluster_sync_all();       // all CTAs run, and their barriers are set up
  if (tid < ctas) {
    double t = 0.0;
    for (int i = 0; i < kSideThreads / 32; ++i) t += tail->warp_sums[i];
    st_cluster_f64(map_to_cta(smem_u32(&tail->sums[rank]), static_cast<uint32_t>(tid)), t);
  }
  cluster_sync_all();
  double total = 0.0;
  for (int i = 0; i < ctas; ++i) total += tail->sums[i];
  const double norm = sqrt(total);
  const bool fine = norm < static_cast<double>(INFINITY);
  const int e = fine && norm > 0.0 ? max(-149, min(127, 13 - ilogb(norm))) : 0;
  const float power = static_cast<float>(ldexp(1.0, e));
  const float factor = fine ? static_cast<float>(1.0 / ((norm + p.eps) * ldexp(1.0, e))) : __int_as_float(0x7FFFFFFF);

  // ---- X0 = G 2^e ----
  for_elements([&](int r, int c, float x) {
    const float v = x * power;
    uint8_t* at = base + (c >> 6) * lay.block + block_at(r, c & 63);
    const __half hi = __float2half_rn(v);
    *reinterpret_cast<__half*>(at) = hi;
    if (kSplit) *reinterpret_cast<__half*>(at + x_low) = __float2half_rn(v - __half2float(hi));
  });
  fence_proxy_async();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tail->tmem;
  const uint32_t sb = smem_u32(base);

  constexpr uint64_t kDesc = (static_cast<uint64_t>(1024 >> 4) << 32) | (static_cast<uint64_t>(1) << 46) | (static_cast<uint64_t>(2) << 61);
  const uint64_t desc_k = kDesc | (static_cast<uint64_t>(1) << 16);
  const uint64_t desc_mn = kDesc | (static_cast<uint64_t>(lay.block >> 4) << 16);       // slabs of 64 columns are a block apart
  constexpr uint32_t idesc0 = (1u << 4) | (static_cast<uint32_t>(kSideRows >> 4) << 24);
  const uint32_t idesc_sym = idesc0 | (static_cast<uint32_t>(R >> 3) << 17);
  auto desc = [&](uint64_t hi, int at) { return hi | (((sb + static_cast<uint32_t>(at)) & 0x3FFFF) >> 4); };
  // waits for the MMAs that were committed last; a wait that runs out is recorded and the rest of the launch goes on without
  auto finished = [&] {
    mbar_wait(bar, phase, abort_flag, p.status, 0x551);
    phase ^= 1u;
    tc_fence_after();
  };
  const int quad = warp & 3, part = warp >> 2, row = quad * 32 + lane;
  const bool rows_here = quad * 32 < R;                                    // warps beyond have no rows of D
  const uint32_t lanes = tmem + (static_cast<uint32_t>(quad * 32) << 16);
  // sums of two blocks' products at most per accumulator (see kGrouped); without low parts one takes all
  const int groups = kSplit ? (nb + 1) / 2 : 1, per_group = kSplit ? 2 : nb;

  for (int step = 0; step < p.steps; ++step) {
    const bool first = step == 0, last = step == p.steps - 1;
    // ---- this CTA's share of A ----
    if (warp == 0 && elect_one()) {
      for (int gr = 0; gr < groups; ++gr) {
        uint32_t more = 0;
        // the small products first: what an addition cuts off goes by the sum's size
        for (int seg = kSplit ? 0 : 2; seg < 3; ++seg)
          for (int b = gr * per_group; b < min(nb, (gr + 1) * per_group); ++b) {
            const int at = b * lay.block;
            for (int k = 0; k < 4; ++k, more = 1)
              mma_one(tmem + gr * R, desc(desc_k, at + (seg == 1 ? x_low : 0) + 32 * k), desc(desc_k, at + (seg == 0 ? x_low : 0) + 32 * k),
                      idesc_sym, more);
          }
      }
      commit_one(bar);
    }
    __syncwarp();
    finished();
    {
      float scale = first ? kScale : 1.0f / kScale;
      if (first) {
        scale *= factor;
        scale *= factor;
      }
      if (rows_here) {
        for (int j = part; j < R / 16; j += 2) {
          __syncwarp();
          float v[16];
          tc_ld16(lanes + j * 16, v);
          for (int gr = 1; gr < groups; ++gr) {
            float w[16];
            tc_ld16(lanes + gr * R + j * 16, w);
#pragma unroll
            for (int i = 0; i < 16; ++i) v[i] += w[i];
          }
          if (row < R) {
            float* at = reinterpret_cast<float*>(base + lay.share) + row * (R + 4) + j * 16;
#pragma unroll
            for (int i = 0; i < 4; ++i)
              *reinterpret_cast<float4*>(at + 4 * i) = make_float4(v[4 * i] * scale, v[4 * i + 1] * scale, v[4 * i + 2] * scale, v[4 * i + 3] * scale);
          }
        }
      }
      tc_fence_before();
    }
    __syncwarp();
    cluster_sync_all();
    // ---- A: pieces of eight columns, each added up by one thread of the cluster and handed to all CTAs ----
    {
      const int pieces = R * R / 8, per_row = R / 8;
      for (int u = rank * kSideThreads + tid; u < pieces; u += ctas * kSideThreads) {
        const int r = u / per_row, c = (u - r * per_row) * 8;
        const uint32_t at = sb + lay.share + (r * (R + 4) + c) * 4;
        float v[8] = {};
        for (int i = 0; i < ctas; ++i) {
          const uint32_t from = map_to_cta(at, static_cast<uint32_t>(i));
          const float4 x = ld_cluster_f4(from), y = ld_cluster_f4(from + 16);
          v[0] += x.x; v[1] += x.y; v[2] += x.z; v[3] += x.w;
          v[4] += y.x; v[5] += y.y; v[6] += y.z; v[7] += y.w;
        }
        const uint32_t to = sb + lay.operand + (c >> 6) * lay.block + block_at(r, c & 63);
        const uint4 hi = halves(v);
        for (int i = 0; i < ctas; ++i) st_cluster_u4(map_to_cta(to, static_cast<uint32_t>(i)), hi);
        if (kSplit) {
          const uint4 lo = halves(v);
          for (int i = 0; i < ctas; ++i) st_cluster_u4(map_to_cta(to + op_low, static_cast<uint32_t>(i)), lo);
        }
      }
      asm volatile("fence.proxy.async;" ::: "memory");
    }
    __syncwarp();
    cluster_sync_all();
    // ---- B = a I + b A + c A^2, in A's place ----
    asm volatile("fence.proxy.async;" ::: "memory");
    tc_fence_after();
    if (warp == 0 && elect_one()) {
      uint32_t more = 0;
      for (int seg = kSplit ? 0 : 2; seg < 3; ++seg)
        for (int k = 0; k < R / 16; ++k, more = 1) {
          const int at = lay.operand + (k >> 2) * lay.block + 32 * (k & 3);
          mma_one(tmem, desc(desc_k, at + (seg == 1 ? op_low : 0)), desc(desc_k, at + (seg == 0 ? op_low : 0)), idesc_sym, more);
        }
      commit_one(bar);
    }
    __syncwarp();
    finished();
    if (rows_here) {
      for (int j = part; j < R / 16; j += 2) {
        __syncwarp();
        float v[16];
        tc_ld16(lanes + j * 16, v);
        if (row < R) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int c = j * 16 + 8 * h;
            uint8_t* at = base + lay.operand + (c >> 6) * lay.block + block_at(row, c & 63);
            float a8[8];
            auto add = [&](const uint8_t* from, bool low) {
              const uint4 x = *reinterpret_cast<const uint4*>(from);
              const uint32_t xs[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&xs[i]));
                a8[2 * i] = low ? a8[2 * i] + f.x : f.x;
                a8[2 * i + 1] = low ? a8[2 * i + 1] + f.y : f.y;
              }
            };
            add(at, false);
            if (kSplit) add(at + op_low, true);
            float w[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              w[i] = fmaf(p.b, a8[i], p.c / kScale * v[8 * h + i]);
              if (c + i == row) w[i] += p.a * kScale;
            }
            *reinterpret_cast<uint4*>(at) = halves(w);
            if (kSplit) *reinterpret_cast<uint4*>(at + op_low) = halves(w);
          }
        }
      }
    }
    fence_proxy_async();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    // ---- X <- B X, up to eight blocks at a time ----
    const float scale = (first ? factor : 1.0f / kScale) * (last ? 1.0f : kScale) / kScale;
    for (int b0 = 0; b0 < nb; b0 += 8) {
      const int b1 = min(nb, b0 + 8);
      if (warp == 0 && elect_one()) {
        for (int b = b0; b < b1; b += 4) {
          const int n = min(4, b1 - b);
          const uint32_t idesc = idesc0 | (1u << 16) | (static_cast<uint32_t>(n * kSideColumns >> 3) << 17);
          uint32_t more = 0;
          for (int seg = kSplit ? 0 : 2; seg < 3; ++seg)
            for (int k = 0; k < R / 16; ++k, more = 1) {
              const int at = lay.operand + (k >> 2) * lay.block + 32 * (k & 3) + (seg == 1 ? op_low : 0);
              mma_one(tmem + (b - b0) * kSideColumns, desc(desc_k, at), desc(desc_mn, b * lay.block + (seg == 0 ? x_low : 0) + k * 2048), idesc,
                      more);
            }
        }
        commit_one(bar);
      }
      __syncwarp();
      finished();
      if (rows_here) {
        for (int j = part; j < (b1 - b0) * (kSideColumns / 16); j += 2) {
          __syncwarp();
          float v[16];
          tc_ld16(lanes + j * 16, v);
#pragma unroll
          for (int i = 0; i < 16; ++i) v[i] *= scale;
          const int c = b0 * kSideColumns + j * 16;           // column of this CTA
          if (!last) {
            if (row < R) {
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                uint8_t* at = base + (c >> 6) * lay.block + block_at(row, (c & 63) + 8 * h);
                float w[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) w[i] = v[8 * h + i];
                *reinterpret_cast<uint4*>(at) = halves(w);
                if (kSplit) *reinterpret_cast<uint4*>(at + x_low) = halves(w);
              }
            }
          } else if (row < p.s) {
            const int64_t m0 = matrix * p.out.batch_stride;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              if (c + i >= cols) break;
              const int64_t to = m0 + (p.flip ? static_cast<int64_t>(c0 + c + i) * p.out.ld + row : static_cast<int64_t>(row) * p.out.ld + c0 + c + i);
              if (p.out.type == kF32) static_cast<float*>(p.out.base)[to] = v[i];
              else if (p.out.type == kBF16) static_cast<__nv_bfloat16*>(p.out.base)[to] = __float2bfloat16_rn(v[i]);
              else static_cast<__half*>(p.out.base)[to] = __float2half_rn(v[i]);
            }
          }
        }
      }
      fence_proxy_async();
      tc_fence_before();
      __syncthreads();
      tc_fence_after();
    }
  }

  // ---- teardown ----
  if (*abort_flag && tid == 0)
    for (const long long t0 = clock64(); clock64() - t0 < 1000000;) {}
  __syncthreads();
  cluster_sync_all();       // no CTA leaves while another may still reach its memory
  if (warp == 0) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
  }
}

}  // namespace
}  // namespace dense
