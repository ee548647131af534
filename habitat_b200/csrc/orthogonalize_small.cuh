// Newton-Schulz steps of matrices whose shorter side is at most 128, in one launch: a cluster per matrix keeps X in shared
// memory, columns spread over its CTAs, for all steps.
//
// A step on tiles in memory is three launches of a few microseconds each whatever the size; here it is two barriers and
// one exchange within the cluster.  Per step each CTA multiplies its columns to a share of A = X X^T, the shares are added slice by slice through
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

constexpr int kSideThreads = 512;              // a warp has every fourth 16 columns (every second with 256: 64 x 64 bfloat16 25 us, 19 so)
constexpr int kSideParts = kSideThreads / 128; // of the columns
constexpr int kSideRows = 128;                 // the longest shorter side
constexpr int kSideSmem = 232448;              // all of an SM's, so that no two of these blocks share its tensor memory
constexpr int kSideColumns = 64;               // per block of X

struct SideTail {
  uint64_t done, arrived;
  uint32_t tmem;
  int abort;
  double sums[16];
  double warp_sums[kSideThreads / 32];
};

struct SideParams {
  Source g;
  Out out;
  int32_t s, l, R, blocks, flip, steps;   // blocks: of 64 columns, per CTA
  int32_t eights;                         // G's rows start on 16-byte boundaries and are X's
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

// This CTA's rows of A, from r0 on, from the shares of all CTAs (added in the order of the ranks), as operands.  All loads of a
// piece are on their way at once: one after the other they took 9 us a step with eight CTAs and 128 rows.
template <bool kSplit, int kCtas>
__device__ __forceinline__ void add_shares(uint32_t share, uint32_t operand, int block, int low, int R, int r0, int rows, int tid) {
  const int per_row = R / 4, pieces = rows * per_row;
  for (int u = tid; u < pieces; u += kSideThreads) {
    const int r = r0 + u / per_row, c = (u - u / per_row * per_row) * 4;
    const uint32_t at = share + (r * (R + 4) + c) * 4;
    float4 x[kCtas];
#pragma unroll
    for (int i = 0; i < kCtas; ++i) x[i] = ld_cluster_f4(map_to_cta(at, static_cast<uint32_t>(i)));
    float4 v = x[0];
#pragma unroll
    for (int i = 1; i < kCtas; ++i) {
      v.x += x[i].x; v.y += x[i].y; v.z += x[i].z; v.w += x[i].w;
    }
    const uint32_t to = operand + (c >> 6) * block + block_at(r, c & 63);
    const uint32_t h0 = pack_f16(v.x, v.y), h1 = pack_f16(v.z, v.w);
    const float2 f0 = __half22float2(*reinterpret_cast<const __half2*>(&h0)), f1 = __half22float2(*reinterpret_cast<const __half2*>(&h1));
    asm volatile("st.shared.v2.b32 [%0], {%1, %2};" ::"r"(to), "r"(h0), "r"(h1) : "memory");
    if (kSplit)
      asm volatile("st.shared.v2.b32 [%0], {%1, %2};" ::"r"(to + low), "r"(pack_f16(v.x - f0.x, v.y - f0.y)), "r"(pack_f16(v.z - f1.x, v.w - f1.y))
                   : "memory");
  }
}
// Bytes of this CTA's shared memory to the same place in another's, counted on a barrier there.
__device__ __forceinline__ void push(uint32_t at, uint32_t bytes, uint32_t bar, uint32_t rank) {
  asm volatile("cp.async.bulk.shared::cluster.shared::cta.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(map_to_cta(at, rank)), "r"(at),
               "r"(bytes), "r"(map_to_cta(bar, rank))
               : "memory");
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
  const uint32_t arrived = smem_u32(&tail->arrived);
  // the rows of A that this CTA adds up
  const int slice0 = min(R, rank * ((R + ctas - 1) / ctas)), slice = min(R, slice0 + (R + ctas - 1) / ctas) - slice0;
  uint32_t phase = 0;

  if (tid == 0) {
    mbar_init(bar, 1);
    mbar_init(arrived, 1);
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
  // Eight columns of a row per thread: kept as they are in the 32 bytes that their high and low parts will take; without low parts
  // there are 16, which take 16-bit updates, and float32 ones are read again.
  const int per_row = (cols + 7) / 8, units = p.s * per_row;
  auto unit_at = [&](int u, int& r, int& c) {
    if (p.flip) {
      c = u / p.s;
      r = u - c * p.s;
    } else {
      r = u / per_row;
      c = u - r * per_row;
    }
    c *= 8;
    return base + (c >> 6) * lay.block + block_at(r, c & 63);
  };
  auto load_unit = [&](int r, int c, float (&v)[8]) {
    const int64_t from = g0 + (p.flip ? static_cast<int64_t>(c0 + c) * p.g.ld + r : static_cast<int64_t>(r) * p.g.ld + c0 + c);
    const int64_t step = p.flip ? p.g.ld : 1;
    if (p.eights && c + 8 <= cols) {
      load_eight(p.g.base, p.g.type, from, v);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = c + i < cols ? load_element(p.g.base, p.g.type, from + i * step) : 0.0f;
    }
  };
  double sum = 0.0;
#pragma unroll 2
  for (int u = tid; u < units; u += kSideThreads) {
    int r, c;
    uint8_t* at = unit_at(u, r, c);
    float v[8];
    load_unit(r, c, v);
    double some[2] = {};
#pragma unroll
    for (int i = 0; i < 8; ++i) some[i & 1] = fma(static_cast<double>(v[i]), static_cast<double>(v[i]), some[i & 1]);
    sum += some[0] + some[1];
    if (kSplit) {
      *reinterpret_cast<float4*>(at) = make_float4(v[0], v[1], v[2], v[3]);
      *reinterpret_cast<float4*>(at + x_low) = make_float4(v[4], v[5], v[6], v[7]);
    } else if (p.g.type == kBF16) {
      *reinterpret_cast<uint4*>(at) = make_uint4(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7]));
    } else if (p.g.type == kF16) {
      *reinterpret_cast<uint4*>(at) = make_uint4(pack_f16(v[0], v[1]), pack_f16(v[2], v[3]), pack_f16(v[4], v[5]), pack_f16(v[6], v[7]));
    }
  }
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
  for (int u = tid; u < units; u += kSideThreads) {
    int r, c;
    uint8_t* at = unit_at(u, r, c);
    float v[8];
    if (kSplit) {
      const float4 x = *reinterpret_cast<const float4*>(at), y = *reinterpret_cast<const float4*>(at + x_low);
      v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w; v[4] = y.x; v[5] = y.y; v[6] = y.z; v[7] = y.w;
    } else if (p.g.type == kF32) {
      load_unit(r, c, v);
    } else {
      const uint4 x = *reinterpret_cast<const uint4*>(at);
      const uint32_t xs[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 f = p.g.type == kBF16 ? make_float2(__uint_as_float(xs[i] << 16), __uint_as_float(xs[i] & 0xFFFF0000u))
                                           : __half22float2(*reinterpret_cast<const __half2*>(&xs[i]));
        v[2 * i] = f.x;
        v[2 * i + 1] = f.y;
      }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] *= power;
    *reinterpret_cast<uint4*>(at) = halves(v);
    if (kSplit) *reinterpret_cast<uint4*>(at + x_low) = halves(v);
  }
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
  // With low parts an accumulator takes 32 of K, small products first, and the accumulators are added here, rounded to nearest: the
  // tensor core cuts what does not fit its sums (see gemm_kernel).  128 x 1024 float32 updates, results off the 64-bit ones (float32
  // operations 1.5e-6) and time: 4.4e-6 and 68 us with 128 of K in each and all of A A and B X in one, 2.7e-6 and 71 with 64, 1.8e-6 and 75 so.
  // Without low parts one takes all.
  constexpr int kGroupSteps = kSplit ? 2 : 1 << 20;                        // of 16 of K
  const int k_steps = R / 16, groups = kSplit ? (k_steps + kGroupSteps - 1) / kGroupSteps : 1;       // of A A and B X: at most 4 of 128 columns
  const int round_steps = kSplit ? 512 / R * kGroupSteps : nb * 4;         // of X X^T, as many as there are accumulators for
  const int round_blocks = 8 / groups;                                     // of B X

  for (int step = 0; step < p.steps; ++step) {
    const bool first = step == 0, last = step == p.steps - 1;
    // ---- this CTA's share of A ----
    float shares[kSideRows / 16 / kSideParts][16];                         // 16 columns of chunks part, part + kSideParts, ...
    for (int k0 = 0; k0 < nb * 4; k0 += round_steps) {
      const int k1 = min(nb * 4, k0 + round_steps);
      if (warp == 0 && elect_one()) {
        for (int from = k0, gr = 0; from < k1; ++gr) {
          const int to = kSplit ? min(k1, from + kGroupSteps) : k1;
          uint32_t more = 0;
          // the small products first: what an addition cuts off goes by the sum's size
          for (int seg = kSplit ? 0 : 2; seg < 3; ++seg)
            for (int k = from; k < to; ++k, more = 1) {
              const int at = (k >> 2) * lay.block + 32 * (k & 3);
              mma_one(tmem + gr * R, desc(desc_k, at + (seg == 1 ? x_low : 0)), desc(desc_k, at + (seg == 0 ? x_low : 0)), idesc_sym, more);
            }
          from = to;
        }
        commit_one(bar);
      }
      __syncwarp();
      finished();
      if (rows_here) {
#pragma unroll
        for (int i = 0; i < kSideRows / 16 / kSideParts; ++i) {
          const int j = part + i * kSideParts;
          if (j >= R / 16) break;
          __syncwarp();
          if (k0 == 0) tc_ld16(lanes + j * 16, shares[i]);
          for (int gr = k0 == 0 ? 1 : 0; kSplit && gr * kGroupSteps < k1 - k0; ++gr) {
            float w[16];
            tc_ld16(lanes + gr * R + j * 16, w);
#pragma unroll
            for (int e = 0; e < 16; ++e) shares[i][e] += w[e];
          }
        }
      }
      if (k1 < nb * 4) {           // the accumulators are used again
        tc_fence_before();
        __syncthreads();
        tc_fence_after();
      }
    }
    {
      float scale = first ? kScale : 1.0f / kScale;
      if (first) {
        scale *= factor;
        scale *= factor;
      }
      if (rows_here) {
#pragma unroll
        for (int i = 0; i < kSideRows / 16 / kSideParts; ++i) {
          const int j = part + i * kSideParts;
          if (j >= R / 16) break;
          const float (&v)[16] = shares[i];
          if (row < R && ctas == 1) {
            // the share is A
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const int c = j * 16 + 8 * h;
              uint8_t* at = base + lay.operand + (c >> 6) * lay.block + block_at(row, c & 63);
              float w[8];
#pragma unroll
              for (int e = 0; e < 8; ++e) w[e] = v[8 * h + e] * scale;
              *reinterpret_cast<uint4*>(at) = halves(w);
              if (kSplit) *reinterpret_cast<uint4*>(at + op_low) = halves(w);
            }
          } else if (row < R) {
            float* at = reinterpret_cast<float*>(base + lay.share) + row * (R + 4) + j * 16;
#pragma unroll
            for (int e = 0; e < 16; e += 4)
              *reinterpret_cast<float4*>(at + e) = make_float4(v[e] * scale, v[e + 1] * scale, v[e + 2] * scale, v[e + 3] * scale);
          }
        }
      }
      tc_fence_before();
    }
    // ---- A: a slice of rows added up by each CTA, whole rows copied to the others (written piece by piece into all shared
    // memories, with longer accumulations than now: 64 x 1024 float32 43.6 us, 37.9 so; 100 x 4000 91.5 and 82.5) ----
    if (ctas > 1) {
      if (tid == 0) mbar_expect_tx(arrived, static_cast<uint32_t>((kSplit ? 2 : 1) * k_blocks * (R - slice) * 128));
      __syncwarp();
      cluster_sync_all();
      switch (ctas) {
        case 2: add_shares<kSplit, 2>(sb + lay.share, sb + lay.operand, lay.block, op_low, R, slice0, slice, tid); break;
        case 4: add_shares<kSplit, 4>(sb + lay.share, sb + lay.operand, lay.block, op_low, R, slice0, slice, tid); break;
        case 8: add_shares<kSplit, 8>(sb + lay.share, sb + lay.operand, lay.block, op_low, R, slice0, slice, tid); break;
        default: add_shares<kSplit, 16>(sb + lay.share, sb + lay.operand, lay.block, op_low, R, slice0, slice, tid); break;
      }
      fence_proxy_async();
      __syncthreads();
      if (tid < ctas && tid != rank && slice > 0)
        for (int i = 0; i < (kSplit ? 2 : 1) * k_blocks; ++i)
          push(sb + lay.operand + i * lay.block + slice0 * 128, static_cast<uint32_t>(slice * 128), arrived, static_cast<uint32_t>(tid));
      __syncwarp();
      mbar_wait_cluster(arrived, static_cast<uint32_t>(step & 1), abort_flag, p.status, 0x552);
      __syncwarp();
      asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");      // "have all rows": B may take the place of what was copied
    } else {
      fence_proxy_async();
      __syncthreads();
    }
    // ---- B = a I + b A + c A^2, in A's place ----
    asm volatile("fence.proxy.async;" ::: "memory");
    tc_fence_after();
    if (warp == 0 && elect_one()) {
      for (int gr = 0; gr < groups; ++gr) {
        uint32_t more = 0;
        const int k0 = gr * kGroupSteps, k1 = kSplit ? min(k_steps, k0 + kGroupSteps) : k_steps;
        for (int seg = kSplit ? 0 : 2; seg < 3; ++seg)
          for (int k = k0; k < k1; ++k, more = 1) {
            const int at = lay.operand + (k >> 2) * lay.block + 32 * (k & 3);
            mma_one(tmem + gr * R, desc(desc_k, at + (seg == 1 ? op_low : 0)), desc(desc_k, at + (seg == 0 ? op_low : 0)), idesc_sym, more);
          }
      }
      commit_one(bar);
    }
    __syncwarp();
    finished();
    __syncwarp();
    if (ctas > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    if (rows_here) {
      for (int j = part; j < R / 16; j += kSideParts) {
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
    // ---- X <- B X, up to eight blocks at a time (with low parts: accumulators) ----
    const float scale = (first ? factor : 1.0f / kScale) * (last ? 1.0f : kScale) / kScale;
    for (int b0 = 0; b0 < nb; b0 += round_blocks) {
      const int b1 = min(nb, b0 + round_blocks);
      if (warp == 0 && elect_one()) {
        for (int gr = 0; gr < groups; ++gr) {
          const int k0 = gr * kGroupSteps, k1 = kSplit ? min(k_steps, k0 + kGroupSteps) : k_steps;
          for (int b = b0; b < b1; b += 4) {
            const int n = min(4, b1 - b);
            const uint32_t idesc = idesc0 | (1u << 16) | (static_cast<uint32_t>(n * kSideColumns >> 3) << 17);
            uint32_t more = 0;
            for (int seg = kSplit ? 0 : 2; seg < 3; ++seg)
              for (int k = k0; k < k1; ++k, more = 1) {
                const int at = lay.operand + (k >> 2) * lay.block + 32 * (k & 3) + (seg == 1 ? op_low : 0);
                mma_one(tmem + (gr * round_blocks + b - b0) * kSideColumns, desc(desc_k, at),
                        desc(desc_mn, b * lay.block + (seg == 0 ? x_low : 0) + k * 2048), idesc, more);
              }
          }
        }
        commit_one(bar);
      }
      __syncwarp();
      finished();
      if (rows_here) {
        for (int j = part; j < (b1 - b0) * (kSideColumns / 16); j += kSideParts) {
          __syncwarp();
          float v[16];
          tc_ld16(lanes + j * 16, v);
          for (int gr = 1; gr < groups; ++gr) {
            float w[16];
            tc_ld16(lanes + gr * round_blocks * kSideColumns + j * 16, w);
#pragma unroll
            for (int i = 0; i < 16; ++i) v[i] += w[i];
          }
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
            if (p.out.vec >= (p.out.type == kF32 ? 16 : 4) && !p.flip && c + 16 <= cols) {
              const int64_t to = m0 + static_cast<int64_t>(row) * p.out.ld + c0 + c;
              if (p.out.type == kF32) {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                  reinterpret_cast<float4*>(static_cast<float*>(p.out.base) + to)[i] = make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
              } else {
                uint32_t w[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) w[i] = p.out.type == kBF16 ? pack_bf16(v[2 * i], v[2 * i + 1]) : pack_f16(v[2 * i], v[2 * i + 1]);
                uint16_t* at = static_cast<uint16_t*>(p.out.base) + to;
                if (p.out.vec == 16) {
#pragma unroll
                  for (int i = 0; i < 2; ++i) reinterpret_cast<uint4*>(at)[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
                } else if (p.out.vec == 8) {
#pragma unroll
                  for (int i = 0; i < 4; ++i) reinterpret_cast<uint2*>(at)[i] = make_uint2(w[2 * i], w[2 * i + 1]);
                } else {
#pragma unroll
                  for (int i = 0; i < 8; ++i) reinterpret_cast<uint32_t*>(at)[i] = w[i];
                }
              }
              continue;
            }
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

// ---------------------------------------------------------------------------
// Shorter side at most 32: everything but the two ends happens on s x s matrices.  All factors B are polynomials of the first
// A = X0 X0^T and commute, so with P the product of the B so far, X = P X0 and the next A is A B^2.  X is read once,
// multiplied to A0 (whose trace is the squared norm), and once more, from shared memory, to P X0.  What that costs is precision:
// A has the squares of the singular values, and P amplifies small ones by up to a^steps; so it is done in float64 on the
// ordinary cores (64 multiply-adds per cycle and SM: 32^3 of them take 512 cycles), and rounded once at the end.
// What rounding leaves in A where an eigenvalue should be zero grows by about a^2 per step, and may be negative, which X X^T cannot
// be and a + b A + c A^2 does not bring back.  So after `stretch` steps, before that is 2^-24 (seven steps with the default
// coefficients), X <- P X is formed and its A is what the next steps begin with.
// 1024 x 12: 47 us as steps on the tensor cores (two cluster barriers and three dependent rounds of MMAs each).
constexpr int kGramSide = 32;
constexpr int kGramThreads = 256;

struct GramParams {
  Source g;
  Out out;
  int32_t s, l, columns, flip, steps, stretch;       // columns: of X, per CTA; stretch: steps between two looks at X
  double a, b, c, eps;
};

constexpr int kGramPitch = kGramSide + 2;                     // rows of doubles start on 16 bytes, eight of them in different banks
constexpr int kGramMatrix = kGramSide * kGramPitch;           // doubles
constexpr int kGramFixed = (5 * kGramMatrix + kGramThreads * 16) * 8;
inline int64_t gram_smem(int S, int64_t columns) { return kGramFixed + columns * (S + 2) * 8; }

__device__ __forceinline__ double2 ld_cluster_d2(uint32_t addr) {
  double2 v;
  asm volatile("ld.shared::cluster.v2.f64 {%0, %1}, [%2];" : "=d"(v.x), "=d"(v.y) : "r"(addr) : "memory");
  return v;
}

// S: s rounded up to a multiple of eight, so that loops over it are unrolled (loads of a whole row on their way at once).
template <int S>
__global__ void __launch_bounds__(kGramThreads) gram_side_kernel(const __grid_constant__ GramParams p) {
  extern __shared__ double smem_d[];
  const int tid = static_cast<int>(threadIdx.x), lane = tid & 31, warp = tid >> 5;
  const int rank = static_cast<int>(cluster_ctarank()), ctas = static_cast<int>(cluster_size());
  const int matrix = static_cast<int>(blockIdx.x) / ctas;
  const int s = p.s;
  constexpr int kX = S + 2, kPitch = kGramPitch;
  double* part = smem_d;                               // sums of threads; [16][256]
  double* share = part + kGramThreads * 16;            // this CTA's share of A
  double* A = share + kGramMatrix;
  double* B = A + kGramMatrix;
  double* P = B + kGramMatrix;                         // and the next one behind it
  double* T = part;                                    // the threads' sums are used up by then
  double* x = share + 5 * kGramMatrix;                 // [column][kX]
  hb_grid_dependency_wait();

  // ---- this CTA's columns of X ----
  const int c0 = rank * p.columns, cols = min(max(p.l - c0, 0), p.columns);
  const int64_t g0 = matrix * p.g.batch_stride;
  if (p.flip) {
    // rows of G are columns of X
#pragma unroll 8
    for (int e = tid; e < cols * S; e += kGramThreads) {
      const int c = e / S, r = e - c * S;
      x[c * kX + r] = r < s ? static_cast<double>(load_element(p.g.base, p.g.type, g0 + static_cast<int64_t>(c0 + c) * p.g.ld + r)) : 0.0;
    }
  } else {
#pragma unroll
    for (int r0 = 0; r0 < S; r0 += kGramThreads / 32) {
      const int r = r0 + warp;
#pragma unroll 4
      for (int c = lane; c < cols; c += 32)
        x[c * kX + r] = r < s ? static_cast<double>(load_element(p.g.base, p.g.type, g0 + static_cast<int64_t>(r) * p.g.ld + c0 + c)) : 0.0;
    }
  }
  __syncthreads();

  constexpr int kSide = S / 4, kTiles = kSide * kSide, kSlices = kGramThreads / kTiles;
  double scale = 0.0;                                  // what X is still to be multiplied by
  const double* F = nullptr;                           // and its factor
  for (int done = 0;;) {
    // ---- its share of A: 4 x 4 elements per thread and slice of the columns ----
    {
      double v[16] = {};
      const int tile = tid % kTiles, slice = tid / kTiles;
      if (slice < kSlices) {
        const int i0 = tile / kSide * 4, j0 = tile % kSide * 4;
#pragma unroll 2
        for (int c = slice; c < cols; c += kSlices) {
          const double* xc = x + c * kX;
          double xi[4], xj[4];
#pragma unroll
          for (int k = 0; k < 4; k += 2) {
            const double2 a = *reinterpret_cast<const double2*>(xc + i0 + k), b = *reinterpret_cast<const double2*>(xc + j0 + k);
            xi[k] = a.x; xi[k + 1] = a.y; xj[k] = b.x; xj[k + 1] = b.y;
          }
#pragma unroll
          for (int k = 0; k < 16; ++k) v[k] = fma(xi[k >> 2], xj[k & 3], v[k]);
        }
      }
#pragma unroll
      for (int k = 0; k < 16; ++k) part[k * kGramThreads + tid] = v[k];
    }
    __syncthreads();
    for (int e = tid; e < kTiles * 16; e += kGramThreads) {
      const int tile = e % kTiles, k = e / kTiles;
      double sum = 0.0;
#pragma unroll 8
      for (int i = 0; i < kSlices; ++i) sum += part[k * kGramThreads + i * kTiles + tile];
      share[(tile / kSide * 4 + (k >> 2)) * S + tile % kSide * 4 + (k & 3)] = sum;
    }
    cluster_sync_all();
    // ---- A: the shares of all CTAs, in the order of the ranks ----
    for (int e = 2 * tid; e < S * S; e += 2 * kGramThreads) {
      const uint32_t at = smem_u32(share + e);
      double2 sum = make_double2(0.0, 0.0);
#pragma unroll 8
      for (int i = 0; i < ctas; ++i) {
        const double2 y = ld_cluster_d2(map_to_cta(at, static_cast<uint32_t>(i)));
        sum.x += y.x;
        sum.y += y.y;
      }
      A[e / S * kPitch + e % S] = sum.x;
      A[e / S * kPitch + e % S + 1] = sum.y;
    }
    __syncthreads();
    if (done == 0) {
      double trace = lane < S ? A[lane * kPitch + lane] : 0.0;       // every warp for itself, in the same order
#pragma unroll
      for (int d = 16; d; d >>= 1) trace += __shfl_xor_sync(0xFFFFFFFFu, trace, d);
      const double norm = sqrt(trace);
      scale = norm < static_cast<double>(INFINITY) ? 1.0 / (norm + p.eps) : __longlong_as_double(0x7FFFFFFFFFFFFFFFll);
    }

    // ---- P = the product of the steps' factors: kRows x 2 elements of each matrix per thread ----
    // All matrices are symmetric (polynomials of A), so rows of the left one are read as columns, two doubles at a time.  With
    // four rows three loads feed eight multiply-adds, what shared memory and the float64 pipe do in the same time; up to 16 x 16
    // latency counts and two rows keep more threads busy.
    constexpr int kRows = S <= 16 ? 2 : 4, kHalf = S / 2, kBatch = S <= 16 ? 8 : 4;
    const int r4 = tid / kHalf * kRows, c2 = tid % kHalf * 2;
    const bool mine = r4 < S;
    using Part = double[kRows][2];
    auto product = [&](const double* u, const double* v, Part& o) {
#pragma unroll
      for (int i = 0; i < kRows; ++i) o[i][0] = o[i][1] = 0.0;
      if (!mine) return;
#pragma unroll
      for (int k0 = 0; k0 < S; k0 += kBatch) {
        double2 us[kBatch][kRows / 2], w[kBatch];
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {
#pragma unroll
          for (int i = 0; i < kRows / 2; ++i) us[k][i] = *reinterpret_cast<const double2*>(u + (k0 + k) * kPitch + r4 + 2 * i);
          w[k] = *reinterpret_cast<const double2*>(v + (k0 + k) * kPitch + c2);
        }
#pragma unroll
        for (int k = 0; k < kBatch; ++k)
#pragma unroll
          for (int i = 0; i < kRows / 2; ++i) {
            o[2 * i][0] = fma(us[k][i].x, w[k].x, o[2 * i][0]);
            o[2 * i][1] = fma(us[k][i].x, w[k].y, o[2 * i][1]);
            o[2 * i + 1][0] = fma(us[k][i].y, w[k].x, o[2 * i + 1][0]);
            o[2 * i + 1][1] = fma(us[k][i].y, w[k].y, o[2 * i + 1][1]);
          }
      }
    };
    auto put = [&](double* to, const Part& o) {
      if (!mine) return;
#pragma unroll
      for (int i = 0; i < kRows; ++i) *reinterpret_cast<double2*>(to + (r4 + i) * kPitch + c2) = make_double2(o[i][0], o[i][1]);
    };
    auto at = [&](int i, int j) { return (r4 + i) * kPitch + c2 + j; };
    __syncthreads();
    if (mine) {
#pragma unroll
      for (int i = 0; i < kRows; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) A[at(i, j)] *= scale * scale;
    }
    __syncthreads();
    int now = 0;
    const int steps = min(p.stretch, p.steps - done);
    for (int step = 0; step < steps; ++step) {
      const bool last = step == steps - 1;
      Part o;
      product(A, A, o);
      if (mine) {
#pragma unroll
        for (int i = 0; i < kRows; ++i)
#pragma unroll
          for (int j = 0; j < 2; ++j) o[i][j] = fma(p.c, o[i][j], fma(p.b, A[at(i, j)], r4 + i == c2 + j ? p.a : 0.0));
      }
      put(B, o);
      if (step == 0) put(P, o);
      __syncthreads();
      if (step > 0) {
        product(B, P + now, o);
        now = kGramMatrix - now;
        put(P + now, o);
      }
      if (!last) {
        product(B, A, o);
        put(T, o);
      }
      __syncthreads();
      if (!last) {
        product(T, B, o);
        put(A, o);
        __syncthreads();
      }
    }
    F = P + now;
    done += steps;
    if (done >= p.steps) break;

    // ---- X <- P X, a column per thread ----
    cluster_sync_all();       // all have read the shares
    for (int c = tid; c < cols; c += kGramThreads) {
      double* xc = x + c * kX;
      double2 v[S / 2];
#pragma unroll
      for (int k = 0; k < S / 2; ++k) v[k] = *reinterpret_cast<const double2*>(xc + 2 * k);
#pragma unroll 1
      for (int r = 0; r < S; r += 2) {
        double2 sum = make_double2(0.0, 0.0);
#pragma unroll
        for (int k = 0; k < S; ++k) {
          const double2 f = *reinterpret_cast<const double2*>(F + k * kPitch + r);
          sum.x = fma(f.x, k & 1 ? v[k >> 1].y : v[k >> 1].x, sum.x);
          sum.y = fma(f.y, k & 1 ? v[k >> 1].y : v[k >> 1].x, sum.y);
        }
        *reinterpret_cast<double2*>(xc + r) = make_double2(sum.x * scale, sum.y * scale);
      }
    }
    scale = 1.0;
    __syncthreads();
  }

  // ---- the result, P X: some rows of one or two columns per lane, lanes over the columns ----
  const int64_t o0 = matrix * p.out.batch_stride;
  auto store = [&](int r, int c, double v) {
    const int64_t to = o0 + (p.flip ? static_cast<int64_t>(c0 + c) * p.out.ld + r : static_cast<int64_t>(r) * p.out.ld + c0 + c);
    const float f = static_cast<float>(v * scale);
    if (p.out.type == kF32) static_cast<float*>(p.out.base)[to] = f;
    else if (p.out.type == kBF16) static_cast<__nv_bfloat16*>(p.out.base)[to] = __float2bfloat16_rn(f);
    else static_cast<__half*>(p.out.base)[to] = __float2half_rn(f);
  };
  constexpr int kOutRows = S <= 16 ? 4 : 8, kOutCols = S <= 16 ? 1 : 2;
  const int chunks = (cols + 32 * kOutCols - 1) / (32 * kOutCols);
  for (int item = warp; item < S / kOutRows * chunks; item += kGramThreads / 32) {
    const int r = item % (S / kOutRows) * kOutRows, c = item / (S / kOutRows) * 32 * kOutCols + lane;
    if (r >= s) continue;
    const double* xs[kOutCols];
#pragma unroll
    for (int j = 0; j < kOutCols; ++j) xs[j] = x + min(c + 32 * j, cols - 1) * kX;      // columns beyond the last read it again
    double v[kOutRows][kOutCols] = {};
#pragma unroll 4
    for (int k = 0; k < S; k += 2) {
      double2 y[kOutCols];
#pragma unroll
      for (int j = 0; j < kOutCols; ++j) y[j] = *reinterpret_cast<const double2*>(xs[j] + k);
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < kOutRows; i += 2) {
          const double2 f = *reinterpret_cast<const double2*>(F + (k + h) * kPitch + r + i);
#pragma unroll
          for (int j = 0; j < kOutCols; ++j) {
            v[i][j] = fma(f.x, h ? y[j].y : y[j].x, v[i][j]);
            v[i + 1][j] = fma(f.y, h ? y[j].y : y[j].x, v[i + 1][j]);
          }
        }
    }
#pragma unroll
    for (int i = 0; i < kOutRows; ++i) {
      if (r + i >= s) break;
#pragma unroll
      for (int j = 0; j < kOutCols; ++j)
        if (c + 32 * j < cols) store(r + i, c + 32 * j, v[i][j]);
    }
  }
  cluster_sync_all();       // no CTA leaves while another may still read its share
}

}  // namespace
}  // namespace dense
