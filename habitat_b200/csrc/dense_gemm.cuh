// The matrix product behind the dense-layer operators (dense_int8.cu, orthogonalize.cu): D = A B^T on two-SM pairs.
//
// A pair of CTAs (cta_group::2) computes tiles of 256 x BN: each CTA brings its 128 rows of A and its BN / 2 rows of B
// into a ring of 128-byte-wide slots by TMA (128-byte swizzle, no multicast), the even CTA's elected lane issues the MMAs for
// both, and the accumulators (32-bit) lie in TMEM two to four times, so that the epilogue warps of each CTA drain one tile
// while the next one is multiplied.  Per slot the pair moves 2 (128 + BN / 2) x 128 bytes for 4 MMAs; with BN = 256 that is 64
// bytes per clock and SM, half of what two separate SMs with 128 x 256 tiles would need of L2.  A slot is 128 bytes of K
// whatever the type, 128 8-bit integers or 64 half-precision values, so both share the ring and the issue loop.
#pragma once

#include <cuda_fp16.h>

#include <initializer_list>

#include "mlp_common.cuh"

namespace dense {

constexpr int kPairRows = 256;             // rows of a pair's tile
constexpr int kCtaRows = 128;
constexpr int kSlotK = 128;                // bytes of K per slot
constexpr int kEpiWarp0 = 4;               // warps: 0 TMA, 1 MMA, 2 TMEM, 3 none, from 4 on epilogue
constexpr int kMostEpiWarps = 16;
constexpr int kStageOutBytes = 32 * 64;    // an epilogue warp's staging: 32 rows x 64 bytes

enum OutType : int32_t { kF32 = 0, kBF16 = 1, kF16 = 2 };

// What goes by the tile's width alone.
template <int BN>
struct Shape {
  static constexpr int kBRows = BN / 2;                               // rows of B (columns of D) per CTA
  static constexpr int kAccs = BN == 256 ? 2 : 4;                     // accumulators
  static constexpr int kTmemCols = kAccs * BN;
  // Epilogue warps: what they do per tile is a chain of loads and conversions that two warps per scheduler cannot fill (28 %
  // of the issue slots, 12,600 cycles per tile of 256 x 256 against 4,096 of MMAs at K = 1,024).
  static constexpr int kEpiWarps = BN == 64 ? 8 : 16;
  static constexpr int kThreads = 32 * (kEpiWarp0 + kEpiWarps);
  static constexpr int kParts = kEpiWarps / 4;       // of the columns
  static constexpr int kCols = BN / kParts;          // a warp's: 64, 32, 32
};

// Shared memory behind the ring: staging, barriers; 8-bit layers: scales and row maxima of the cluster's CTAs.
struct Tail {
  uint8_t staging[kMostEpiWarps * kStageOutBytes];
  uint64_t full[8], empty[8], acc_full[4], acc_empty[4], exchange[2][4], drain;
  uint32_t tmem;
  int abort;
};
struct LayerTail {
  float scales[kMostEpiWarps][160];        // an epilogue warp's: 64 channel scales, 64 biases, 32 row scales
  float row_max[2][4][4][kCtaRows];
};

// The ring.  kSplit: a slot has the high and the low parts of both operands.
template <int BN, class Epi>
struct Ring {
  static constexpr int kOperands = (kCtaRows + Shape<BN>::kBRows) * kSlotK;     // per CTA
  static constexpr int kSlotBytes = kOperands * (Epi::kSplit ? 2 : 1);
  static constexpr int kSlots = Epi::kShares > 1 ? (Epi::kSplit ? 3 : 6) : Epi::kSplit ? (BN == 256 ? 3 : 4) : Epi::kInt8 ? (BN == 256 ? 5 : BN == 128 ? 6 : 8) : BN == 256 ? 6 : 8;
  // what the other pairs of a cluster send of a tile: their sums of this CTA's part of the columns
  static constexpr int kShareBytes = (Epi::kShares - 1) * (kCtaRows * BN / Epi::kShares) * 4;
  static constexpr int kSmem = kSlots * kSlotBytes + kShareBytes + static_cast<int>(sizeof(Tail)) + (Epi::kInt8 ? static_cast<int>(sizeof(LayerTail)) : 0) + 1024;
  static_assert(kSmem <= 232448, "more than a block may have");
};

// What a launch multiplies: `batches` products of M x N with kblocks slots of K each.  With Epi::kSplit the operands are pairs of
// planes, high and low parts (the low ones lie `batches` matrices behind), and the sum is hi lo + lo hi + hi hi: a slot has
// four operands for three products.
struct Product {
  CUtensorMap a, b;        // [matrices][rows][K], boxes of 128 (a) and BN / 2 (b) rows x 128 bytes; b K-major or MN-major
  int32_t M, N, kblocks, batches;
  int32_t splits;          // of K: every tile is made that many times, with a share of the slots each
  int32_t tiles_m, tiles_n, num_tiles;   // num_tiles: over all batches
  int32_t lower;           // 1: D is symmetric, each pair of mirrored blocks is computed once
  int32_t per_batch;       // tiles of a batch, and its and a tile group's reciprocal (set_tiles)
  uint32_t per_batch_inv, per_group_inv;
  int32_t* status;
};

constexpr int kTileGroup = 8;      // row blocks that tiles go through together

struct Tile {
  int batch, m0, m1, n0, split;      // m0, m1: first rows of the two CTAs
};

// n / d and, in n, the remainder, for 0 <= n < 2^31.  m is 2^32 / d rounded down (reciprocal_of): the estimate is at most two too
// small.
__device__ __forceinline__ int divide(int& n, int d, uint32_t m) {
  int q = static_cast<int>(__umulhi(static_cast<uint32_t>(n), m));
  n -= q * d;
  while (n >= d) {
    n -= d;
    ++q;
  }
  return q;
}
inline uint32_t reciprocal_of(int64_t d) { return d <= 1 ? 0xFFFFFFFFu : static_cast<uint32_t>((int64_t{1} << 32) / d); }

inline void set_tiles(Product* p, int64_t per_batch) {
  p->per_batch = static_cast<int32_t>(per_batch);
  p->num_tiles = static_cast<int32_t>(per_batch * p->batches * p->splits);
  p->per_batch_inv = reciprocal_of(per_batch);
  p->per_group_inv = reciprocal_of(static_cast<int64_t>(kTileGroup) * p->tiles_n);
}

// Tiles of a symmetric result of n x n blocks of 128, each with two blocks of one column: a pair's CTAs share columns, not rows.
// Of a block and its mirror image one is needed, n (n + 1) / 2 in all; a column c has those of rows c to n - 1, and every
// other column an odd number.  Two such columns, c and c + 2, help each other out: block (c + 2, c) is computed as its mirror
// image (c, c + 2), which leaves both with an even number, and at most one tile in all is half empty.  (Neighbouring rows in
// every pair: 20 tiles for n = 8, not 18, so eight matrices of 1024 x 1024 take a third round of 74 pairs: five float32 steps, call
// after call, 758 us, 678 so.)
// With r = n - 1 - c the columns r = 4 g to 4 g + 3 have 2 g + 1, 2 g + 1, 2 g + 1 and 2 g + 2 tiles, all before them
// 4 g^2 + g.
__host__ __device__ __forceinline__ int64_t two_block_tiles(int64_t n) {
  const int64_t g = n / 4;
  return 4 * g * g + g + n % 4 * (2 * g + 1);
}
// The rows of blocks and the column of tile t; a row of n where there is none.
__host__ __device__ __forceinline__ void two_block_tile(int n, int t, int* row0, int* row1, int* column) {
  int g = static_cast<int>((sqrtf(16.0f * static_cast<float>(t) + 1.0f) - 1.0f) * 0.125f);
  while (4 * g * g + g > t) --g;
  while (4 * (g + 1) * (g + 1) + g + 1 <= t) ++g;
  const int wide = 2 * g + 1;
  int k = t - 4 * g * g - g, turn = 0;
  while (turn < 3 && k >= wide) {
    k -= wide;
    ++turn;
  }
  const int c = n - 1 - 4 * g - turn;
  *column = c;
  int r = c + 2 * k;                          // rows c, c + 1, ...
  if (turn == 0) r -= 1;                      // c - 2, c, c + 1, ...
  if (turn == 2 && k > 0) r += 1;             // c, c + 1, c + 3, ...
  *row0 = turn == 0 && k == 0 ? (c >= 2 ? c - 2 : n) : r;
  *row1 = r + 1;
}

// Tile `t` of a launch.  Full products go through groups of eight row blocks, column by column, so that the tiles in
// flight share rows and columns in L2.
template <int BN>
__device__ __forceinline__ Tile tile_of(const Product& p, int t) {
  Tile r;
  r.batch = divide(t, p.per_batch, p.per_batch_inv);
  r.split = 0;
  if (p.splits > 1) {
    r.split = r.batch % p.splits;
    r.batch /= p.splits;
  }
  int mt, nt;
  if (BN == kCtaRows && p.lower) {
    two_block_tile(p.tiles_n, t, &mt, &r.m1, &nt);
    r.m0 = mt * kCtaRows;
    r.m1 *= kCtaRows;
    r.n0 = nt * BN;
    return r;
  }
  if (p.lower) {
    constexpr int kPer = kPairRows / BN;
    mt = 0;
    nt = t;
    for (;;) {
      const int row = min((mt + 1) * kPer, p.tiles_n);
      if (nt < row) break;
      nt -= row;
      ++mt;
    }
  } else {
    const int g = divide(t, kTileGroup * p.tiles_n, p.per_group_inv);
    const int rows = min(kTileGroup, p.tiles_m - g * kTileGroup);
    nt = rows == kTileGroup ? t / kTileGroup : t / rows;
    mt = g * kTileGroup + t - nt * rows;
  }
  r.m0 = mt * kPairRows;
  r.m1 = r.m0 + kCtaRows;
  r.n0 = nt * BN;
  return r;
}

__device__ __forceinline__ void tma_3d_2sm(uint32_t dst, const CUtensorMap* map, int32_t x, int32_t y, int32_t z,
                                           uint32_t cluster_mbar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes "
      "[%0], [%1, {%3, %4, %5}], [%2];"
      ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(cluster_mbar), "r"(x), "r"(y), "r"(z)
      : "memory");
}
// Commits to the barriers of both CTAs of the pair; `pair` is its index in the cluster.
__device__ __forceinline__ void commit_pair(uint32_t bar, uint32_t pair) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar),
      "h"(static_cast<uint16_t>(3u << (2 * pair)))
      : "memory");
}
template <bool I8>
__device__ __forceinline__ void mma_pair(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  if (I8)
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
        "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
        "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
}
// "Read out": nothing but tensor memory is handed over, so the arrival need not wait for this thread's stores to memory, as
// one with release semantics in the cluster does.
__device__ __forceinline__ void arrive_remote_relaxed(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}
// A value for another CTA's shared memory, counted in bytes on a barrier there.
__device__ __forceinline__ void st_async_f32(uint32_t cluster_addr, float v, uint32_t cluster_mbar) {
  asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.b32 [%0], %1, [%2];" ::"r"(cluster_addr),
               "r"(__float_as_uint(v)), "r"(cluster_mbar)
               : "memory");
}
// Accumulators are read as 16 x 256-bit fragments: of 16 rows lane l gets rows l / 4 and l / 4 + 8, and of every eight
// columns 2 (l mod 4) and the next.  A lane then has 4 rows and a quarter of its warp's columns; with whole rows per lane
// (32 x 32 bits) every lane loads the scale and bias of every column from shared memory, which the MMAs' operands go
// through as well (65,536 x 1024 x 1024: quantised rows 84 us, 67 without those loads).
template <int COLS>
__device__ __forceinline__ void load_fragment(uint32_t taddr, uint32_t* r);
template <>
__device__ __forceinline__ void load_fragment<64>(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.16x256b.x8.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
}
template <>
__device__ __forceinline__ void load_fragment<32>(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.16x256b.x4.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}

__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
// max(x, 0) that keeps NaN
__device__ __forceinline__ float relu_nan(float x) { return max_nan(x, 0.0f); }

__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
  const __nv_bfloat162 p = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&p);
}
__device__ __forceinline__ uint32_t pack_f16(float a, float b) {
  const __half2 p = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&p);
}

// Where results go: rows of `ld` elements, matrices `batch_stride` elements apart; `vec`: the bytes, up to 16, that every row
// starts on a multiple of.
struct Out {
  void* base;
  int64_t ld, batch_stride;
  int32_t type;
  int32_t vec;
};

inline int32_t row_alignment(const void* base, int64_t ld, int64_t batch_stride, int elem_bytes) {
  const uint64_t x = static_cast<uint64_t>(reinterpret_cast<uintptr_t>(base)) | static_cast<uint64_t>(ld * elem_bytes) |
                     static_cast<uint64_t>(batch_stride * elem_bytes) | 16u;
  return static_cast<int32_t>(x & (~x + 1));
}

// Fragments to rows: stores four 8 x 8 matrices of 16-bit elements, w[j] to the 16-byte column j of rows 8 i .. 8 i + 7 of a
// warp's staging (64 bytes per row, columns permuted by the row so that eight rows fill all banks); and the 16 bytes of row
// r and column c.
__device__ __forceinline__ void store_fragment(uint32_t staging, int i, const uint32_t (&w)[4], int lane) {
  const int r = 8 * i + (lane & 7), j = lane >> 3;
  asm volatile("stmatrix.sync.aligned.m8n8.x4.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(staging + r * 64 + ((j ^ ((r >> 1) & 3)) << 4)),
               "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3])
               : "memory");
}
__device__ __forceinline__ uint4 staged_row(const uint8_t* staging, int r, int c) {
  return *reinterpret_cast<const uint4*>(staging + r * 64 + ((c ^ ((r >> 1) & 3)) << 4));
}
// The same with rows and columns exchanged: w[i] to the 16-byte column i of rows 8 j .. 8 j + 7, which are columns of the results.
__device__ __forceinline__ void store_fragment_turned(uint32_t staging, int j, const uint32_t (&w)[4], int lane) {
  const int r = 8 * j + (lane & 7), i = lane >> 3;
  asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(staging + r * 64 + ((i ^ ((r >> 1) & 3)) << 4)),
               "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3])
               : "memory");
}
// A warp's staging of 32 x 32 16-bit elements to rows of `ld` elements from `to` on, of which rows_left and cols_left are there.
__device__ __forceinline__ void store_staged(const uint8_t* staging, uint16_t* to, int64_t ld, int vec, int rows_left, int cols_left, int lane) {
  if (vec >= 4) {
    const int n = 8 * (lane & 3);
    uint16_t* at = to + (lane >> 2) * ld + n;
#pragma unroll
    for (int i = 0; i < 4; ++i, at += 8 * ld) {
      if (8 * i + (lane >> 2) >= rows_left) continue;
      const uint4 x = staged_row(staging, 8 * i + (lane >> 2), lane & 3);
      const uint32_t xs[4] = {x.x, x.y, x.z, x.w};
      if (n + 8 > cols_left) {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (n + e < cols_left) at[e] = static_cast<uint16_t>(xs[e >> 1] >> (16 * (e & 1)));
      } else if (vec == 16) {
        *reinterpret_cast<uint4*>(at) = x;
      } else if (vec == 8) {
        reinterpret_cast<uint2*>(at)[0] = make_uint2(x.x, x.y);
        reinterpret_cast<uint2*>(at)[1] = make_uint2(x.z, x.w);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) reinterpret_cast<uint32_t*>(at)[e] = xs[e];
      }
    }
  } else if (lane < cols_left) {
    // rows that start on any element: a row of 32 at a time
#pragma unroll 8
    for (int r = 0; r < 32; ++r)
      if (r < rows_left)
        to[r * ld + lane] = *reinterpret_cast<const uint16_t*>(staging + r * 64 + (((lane >> 3) ^ ((r >> 1) & 3)) << 4) + 2 * (lane & 7));
  }
}

// What a tile's epilogue may use.
struct EpiContext {
  Tail* tail;
  LayerTail* layer;       // 8-bit layers'
  uint32_t tmem;          // this warp's lanes and first column of its part of the tile
  int warp, lane, part;   // epilogue warp, its part of the columns
  int row;                // the warp's first row among the CTA's 128
  int row0, n0;           // its first row and the first column of its part, in the matrix
  int batch, t;           // and the tile's number
  uint32_t n_tile;        // how many tiles the CTA has drained before
  bool first, last;       // accumulation of the tile (kSplit)
  float scale;            // a policy's
  uint32_t rank;          // in the cluster
  int next_row0, next_n0; // of the next tile; next_row0 < 0: there is none
  bool* ok;
};

// 32 columns of a warp's part as float fragments: v[j][i] are columns 8 j + 2 (lane mod 4) and the next of row 8 i + lane / 4.
using Block = float2[4][4];
template <class Use>
__device__ __forceinline__ void load_block(uint32_t tmem, Use use) {
  uint32_t acc[2][16];
  load_fragment<32>(tmem, acc[0]);
  load_fragment<32>(tmem + (16u << 16), acc[1]);
  tc_wait_ld();
#pragma unroll
  for (int j = 0; j < 4; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) use(j, i, make_float2(__uint_as_float(acc[i >> 1][4 * j + 2 * (i & 1)]), __uint_as_float(acc[i >> 1][4 * j + 2 * (i & 1) + 1])));
}

// The width of a tile whose rounds take least.  A round of MMAs takes 64 cycles per 16 values of K (32 in 8 bits) for up to
// 128 columns and 128 for 256, and its epilogue and start about as long as 24 columns and a quarter of its own.
template <class Count>
inline int tile_columns(std::initializer_list<int> widths, int pairs, Count tiles) {
  int best = 0;
  int64_t least = INT64_MAX;
  for (const int bn : widths) {
    const int64_t cost = (tiles(bn) + pairs - 1) / pairs * (4 * (bn > 128 ? bn : 128) + bn + 96);
    if (cost < least) {
      least = cost;
      best = bn;
    }
  }
  return best;
}

// Sums of a tile whose K is split over the kShares pairs of a cluster: every warp but one sends its 32 x 32 sums to the same warp
// of the pair that finishes these columns, which adds them in the order of the pairs.  False: they are another pair's.
template <int BN, class Epi>
__device__ __forceinline__ bool join_shares(const Product& p, const EpiContext& c, Block& sums) {
  constexpr int S = Epi::kShares;
  static_assert(Shape<BN>::kCols == 32 && Shape<BN>::kParts % S == 0, "a block per warp, parts for every pair");
  const int mine = static_cast<int>(c.rank >> 1), owner = c.part % S;
  const uint32_t bar = smem_u32(&c.tail->exchange[0][0]);
  const uint32_t at = smem_u32(c.tail) - Ring<BN, Epi>::kShareBytes + ((c.part / S * 4 + (c.row >> 5)) * (S - 1)) * 4096 + c.lane * 16;
  if (mine != owner) {
    const uint32_t there = 2 * owner + (c.rank & 1u);
    const uint32_t to = map_to_cta(at + (mine - (mine > owner ? 1 : 0)) * 4096, there), to_bar = map_to_cta(bar, there);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const float2 x = sums[k >> 1][2 * (k & 1)], y = sums[k >> 1][2 * (k & 1) + 1];
      st_async_v4(to + 512 * k, __float_as_uint(x.x), __float_as_uint(x.y), __float_as_uint(y.x), __float_as_uint(y.y), to_bar);
    }
    return false;
  }
  if (!mbar_wait_cluster(bar, 0, &c.tail->abort, p.status, 0x542)) {
    *c.ok = false;
    return false;
  }
#pragma unroll
  for (int from = 0; from < S - 1; ++from)
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      float4 v;
      asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(at + from * 4096 + 512 * k) : "memory");
      float2& x = sums[k >> 1][2 * (k & 1)];
      float2& y = sums[k >> 1][2 * (k & 1) + 1];
      x = make_float2(x.x + v.x, x.y + v.y);
      y = make_float2(y.x + v.z, y.y + v.w);
    }
  return true;
}

// What this CTA will be sent.
template <int BN, class Epi>
__device__ __forceinline__ void expect_shares(const EpiContext& c) {
  if (Epi::kShares > 1 && c.warp == 0 && c.lane == 0) mbar_expect_tx(smem_u32(&c.tail->exchange[0][0]), Ring<BN, Epi>::kShareBytes);
}

// The kernel.  Epilogue: a policy with `Params`, static kInt8, kMnMajorB, kSplit, kClusterCtas (0: pairs by themselves; else the CTAs of a
// cluster that share rows, one pair per BN columns), kShares (above 1: the pairs of a cluster share K, a tile per cluster) and
//   static void begin(const Params&, const Product&, EpiContext&, sums)         before a tile's accumulators are waited for
//   static void fetch(const Params&, const Product&, EpiContext&, row0, n0)     requests what a tile's results need, a tile ahead
//   static void drain(const Params&, const Product&, EpiContext&, sums, release)   calls release() once the accumulators are read, and,
//                                                                                  where it has used what fetch() brought, requests the next tile's
// kSplit: the tensor core adds 16 products of K at a time to its float32 sums and cuts what does not fit, which over long K is
// off by as many units as there are additions, all to the same side (1024 x 1024 float32 updates: 3.7e-5).  So every
// slot has an accumulation of its own, the small products of high and low parts first, and drain() adds them in
// registers (sums), rounded to nearest (2.1e-6); it acts on the last one.
template <int BN, class Epi>
__global__ void __launch_bounds__(Shape<BN>::kThreads, 1)
gemm_kernel(const __grid_constant__ Product p, const __grid_constant__ typename Epi::Params ep) {
  using S = Shape<BN>;
  using R = Ring<BN, Epi>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  Tail* tail = reinterpret_cast<Tail*>(ring + R::kSlots * R::kSlotBytes + R::kShareBytes);
  const int warp = static_cast<int>(threadIdx.x >> 5), lane = static_cast<int>(threadIdx.x & 31);
  const uint32_t rank = cluster_ctarank();
  const uint32_t side = rank & 1u, pair = rank >> 1;
  const uint32_t leader = rank & ~1u;
  constexpr int kCluster = Epi::kClusterCtas ? Epi::kClusterCtas : 2 * Epi::kShares;
  volatile int* abort_flag = &tail->abort;
  const uint32_t full = smem_u32(tail->full), empty = smem_u32(tail->empty), acc_full = smem_u32(tail->acc_full),
                 acc_empty = smem_u32(tail->acc_empty);

  if (threadIdx.x == 32) {
    for (int s = 0; s < R::kSlots; ++s) {
      mbar_init(full + 8 * s, 1);       // the leader's: its producer's expect_tx; both CTAs' copies count there
      mbar_init(empty + 8 * s, 1);
    }
    for (int s = 0; s < S::kAccs; ++s) {
      mbar_init(acc_full + 8 * s, 1);
      mbar_init(acc_empty + 8 * s, 2 * S::kEpiWarps);
    }
    for (int s = 0; s < 8; ++s) mbar_init(smem_u32(&tail->exchange[0][0]) + 8 * s, 1);
    mbar_init(smem_u32(&tail->drain), 1);
    tail->abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 2) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tail->tmem)),
                 "r"(static_cast<uint32_t>(S::kTmemCols))
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  if (threadIdx.x == 0) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&p.a)) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&p.b)) : "memory");
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();
  tc_fence_after();
  hb_grid_dependency_wait();   // the set-up above overlaps the end of the launch before it on the stream
  const uint32_t tmem = tail->tmem;

  // a tile of the list per cluster; where it shares rows, its pairs take neighbouring columns
  const int workers = static_cast<int>(gridDim.x) / kCluster;
  const int worker = static_cast<int>(blockIdx.x) / kCluster;
  auto locate = [&](int t) {
    if (Epi::kClusterCtas) return Tile{0, t * kPairRows, t * kPairRows + kCtaRows, static_cast<int>(pair) * BN, 0};
    Tile r = tile_of<BN>(p, t);
    if (Epi::kShares > 1) r.split = static_cast<int>(pair);
    return r;
  };
  // slots of K of a share, and where it begins
  const int splits = Epi::kShares > 1 ? Epi::kShares : p.splits;
  const int most_kb = splits > 1 ? (p.kblocks + splits - 1) / splits : p.kblocks;
  auto slots_of = [&](int split) { return splits > 1 ? max(0, min(most_kb, p.kblocks - split * most_kb)) : most_kb; };

  if (warp == 0) {
    // ------------------------------ copies ------------------------------
    if (lane == 0) {
      const uint32_t ring_addr = smem_u32(ring);
      uint32_t s = 0, ph = 1;
      bool ok = true;
      for (int t = worker; t < p.num_tiles && ok; t += workers) {
        const Tile tile = locate(t);
        const int kb0 = tile.split * most_kb, kb1 = kb0 + slots_of(tile.split);
        const int m = side ? tile.m1 : tile.m0, n = tile.n0 + static_cast<int>(side) * S::kBRows;
        for (int kb = kb0; kb < kb1; ++kb) {
          ok = mbar_wait(empty + 8 * s, ph, abort_flag, p.status, 0x511);
          if (!ok) break;
          const uint32_t bar = map_to_cta(full + 8 * s, leader);
          if (side == 0) mbar_expect_tx(full + 8 * s, 2 * R::kSlotBytes);
          constexpr int kElems = Epi::kInt8 ? kSlotK : kSlotK / 2;
#pragma unroll
          for (int part = 0; part < (Epi::kSplit ? 2 : 1); ++part) {
            const uint32_t dst = ring_addr + s * R::kSlotBytes + part * R::kOperands;
            const int z = tile.batch + part * p.batches;
            tma_3d_2sm(dst, &p.a, kb * kElems, m, z, bar);
            if (Epi::kMnMajorB) {
              // [64 rows of K][64 columns] per slab
#pragma unroll
              for (int j = 0; j < S::kBRows / 64; ++j)
                tma_3d_2sm(dst + kCtaRows * kSlotK + j * 8192, &p.b, n + 64 * j, kb * kElems, z, bar);
            } else {
              tma_3d_2sm(dst + kCtaRows * kSlotK, &p.b, kb * kElems, n, z, bar);
            }
          }
          if (++s == R::kSlots) { s = 0; ph ^= 1u; }
        }
      }
    }
  } else if (warp == 1) {
    // ------------------------------ MMAs (leader) ------------------------------
    if (side == 0 && elect_one()) {
      // D: 32-bit integers (2) or float (1); A and B: signed 8-bit (1) or f16 (0); B MN-major: bit 16; N, M
      constexpr uint32_t idesc = (Epi::kInt8 ? (2u << 4) | (1u << 7) | (1u << 10) : (1u << 4)) |
                                 (Epi::kMnMajorB ? 1u << 16 : 0u) | (static_cast<uint32_t>(BN >> 3) << 17) |
                                 (static_cast<uint32_t>(kPairRows >> 4) << 24);
      // 8 rows of a swizzle atom are 1,024 bytes; MN-major: slabs of 64 columns are 8 KB apart
      constexpr uint64_t kDesc = (static_cast<uint64_t>(1024 >> 4) << 32) | (static_cast<uint64_t>(1) << 46) |
                                 (static_cast<uint64_t>(2) << 61);
      constexpr uint64_t a_hi = kDesc | (static_cast<uint64_t>(1) << 16);
      constexpr uint64_t b_hi = kDesc | (static_cast<uint64_t>(Epi::kMnMajorB ? 8192 >> 4 : 1) << 16);
      constexpr uint32_t b_step = Epi::kMnMajorB ? 2048 >> 4 : 32 >> 4;
      const uint32_t a0 = (smem_u32(ring) & 0x3FFFF) >> 4;
      uint32_t s = 0, ph = 0, n = 0;
      bool ok = true;
      for (int t = worker; t < p.num_tiles && ok; t += workers) {
        const int slots = slots_of(splits > 1 ? locate(t).split : 0);
        for (int kb = 0; kb < slots && ok;) {
          const uint32_t st = n % S::kAccs, turn = n / S::kAccs & 1u;
          ++n;
          ok = mbar_wait(acc_empty + 8 * st, turn ^ 1u, abort_flag, p.status, 0x521);
          tc_fence_after();
          const uint32_t d = tmem + st * BN;
          uint32_t more = 0;
          for (const int end = Epi::kSplit ? kb + 1 : slots; kb < end && ok; ++kb) {
            ok = mbar_wait(full + 8 * s, ph, abort_flag, p.status, 0x522);
            if (!ok) break;
            tc_fence_after();
            const uint32_t a_lo = a0 + s * (R::kSlotBytes >> 4);
            const uint32_t b_lo = a_lo + (kCtaRows * kSlotK >> 4);
            constexpr uint32_t kLow = R::kOperands >> 4;      // from a high part to its low one
            if (Epi::kSplit) {
#pragma unroll
              for (int k = 0; k < 4; ++k) mma_pair<Epi::kInt8>(d, a_hi | (a_lo + 2 * k), b_hi | (b_lo + kLow + b_step * k), idesc, k ? 1u : 0u);
#pragma unroll
              for (int k = 0; k < 4; ++k) mma_pair<Epi::kInt8>(d, a_hi | (a_lo + kLow + 2 * k), b_hi | (b_lo + b_step * k), idesc, 1u);
              more = 1;
            }
#pragma unroll
            for (int k = 0; k < 4; ++k, more = 1) mma_pair<Epi::kInt8>(d, a_hi | (a_lo + 2 * k), b_hi | (b_lo + b_step * k), idesc, more);
            commit_pair(empty + 8 * s, pair);
            if (++s == R::kSlots) { s = 0; ph ^= 1u; }
          }
          if (ok) commit_pair(acc_full + 8 * st, pair);
        }
      }
    }
  } else if (warp >= kEpiWarp0) {
    // ------------------------------ epilogue ------------------------------
    const int w = warp - kEpiWarp0;
    const int quad = warp & 3;
    bool ok = true;
    EpiContext c;
    c.tail = tail; c.layer = reinterpret_cast<LayerTail*>(tail + 1); c.warp = w; c.lane = lane; c.part = w >> 2; c.row = quad * 32; c.rank = rank; c.ok = &ok;
    uint32_t n = 0;
    const uint32_t acc_empty_leader = map_to_cta(acc_empty, leader);
    Block sums;
    c.n_tile = 0;
    Tile tile{}, next{};
    auto look_ahead = [&](int t) {
      c.next_row0 = -1;
      if (t >= p.num_tiles) return;
      next = locate(t);
      c.next_row0 = (side ? next.m1 : next.m0) + c.row;
      c.next_n0 = next.n0 + c.part * S::kCols;
    };
    look_ahead(worker);
    if (c.next_row0 >= 0) Epi::template fetch<BN>(ep, p, c, c.next_row0, c.next_n0);
    for (int t = worker; t < p.num_tiles && ok; t += workers, ++c.n_tile) {
      tile = next;
      c.row0 = c.next_row0;
      c.n0 = c.next_n0;
      c.batch = tile.batch;
      look_ahead(t + workers);
      Epi::template begin<BN>(ep, p, c, sums);
      c.t = t;
      const int rounds = Epi::kSplit ? slots_of(tile.split) : 1;
      for (int i = 0; i < rounds && ok; ++i, ++n) {
        const uint32_t st = n % S::kAccs, turn = n / S::kAccs & 1u;
        c.tmem = tmem + (static_cast<uint32_t>(quad * 32) << 16) + st * BN + static_cast<uint32_t>(c.part * S::kCols);
        c.first = i == 0;
        c.last = i == rounds - 1;
        if (!mbar_wait(acc_full + 8 * st, turn, abort_flag, p.status, 0x531)) { ok = false; break; }
        tc_fence_after();
        Epi::template drain<BN>(ep, p, c, sums, [&] {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) {
            if (side == 0) mbar_arrive(acc_empty + 8 * st);
            else arrive_remote_relaxed(acc_empty_leader + 8 * st);
          }
        });
      }
    }
  }

  // ------------------------------ teardown ------------------------------
  tc_fence_before();
  __syncthreads();
  if (*abort_flag) {
    // given up: wait, within limits, for MMAs and copies in flight
    if (side == 0 && warp == 1 && elect_one()) {
      commit_pair(smem_u32(&tail->drain), pair);
      const long long t0 = clock64();
      while (!mbar_try_wait_cluster(smem_u32(&tail->drain), 0) && clock64() - t0 <= kWaitCycles) {}
    }
    if (threadIdx.x == 0)
      for (const long long t0 = clock64(); clock64() - t0 < 1000000;) {}
    __syncthreads();
  }
  cluster_sync_all();   // no CTA leaves while another may still touch its memory
  if (warp == 2) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem),
                 "r"(static_cast<uint32_t>(S::kTmemCols))
                 : "memory");
  }
}

}  // namespace dense
