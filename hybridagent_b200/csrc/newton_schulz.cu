// Newton-Schulz orthogonalisation of a batch of equal-shaped matrices (sm_100a).
//
// One step, with m = min(rows, cols) and n = max(rows, cols) (X is m x n, or its transpose):
//     A = X X^T            (m x m, symmetric)
//     B = b A + c A A      (m x m, symmetric)
//     X <- a X + B X
// Every product runs on tcgen05 with fp16 operands and fp32 accumulators.  fp16 and not bf16: all
// values are bounded (singular values stay below about 1.2), so its range suffices with fixed
// power-of-two scales, and its three more bits cut the rounding error of the result eightfold.
//
// Rounding X itself is what a strongly graded spectrum is sensitive to: the rounding noise of the
// leading directions is full-rank and is amplified as much as the small singular values (485-fold
// in five steps).  So X is kept as a high and a low fp16 plane (22 bits) until the steps that are left multiply by
// no more than kPlainGain: in all but the last two of the usual steps, however many there are.  With a low plane in the
// first three steps only, 300 x 400 of rank 4 was off by 8e-3 after six steps, 0.1 after eight and 1.1 after ten; now by 3e-3,
// 6e-3 and 6e-2, which is what the accumulators cut off (2^-21 of X in a step), multiplied by 3.44 in every later step.
// The products read the high plane only: with a on B's diagonal a step is (a I + B) X, and its
// epilogue adds a * low in fp32 (what B does to the low plane touches only the few leading
// directions).  Against 64-bit results (rank-16 plus 5 % noise, 1024 x 1024, rounded to bf16): 2.1e-3
// relative, of which 1.7e-3 is the final rounding; one fp16 plane gives 2.1e-2, bf16 operands 1.6e-1.
//
// The diagonals of G and of the factors keep what their rounding takes, in fp32 (diagonal_at below).  Where all
// singular values are alike, as in a matrix much longer than wide, these matrices are close to multiples of I, their
// diagonals round in the same direction, and the later steps amplify that up to fourfold: 383 x 14575, normal
// elements, is 2.95e-3 off without and 1.78e-3 with it (rounded to bf16).  It costs 3 us of the 116 of 48 of
// 256 x 512 and under 1 % of large batches.
//
// Two steps can run as one product with X: with Q1 = a I + b G + c G^2 (G = X X^T), the Gram matrix
// after the step is G' = Q1 G Q1, Q2 follows from G', and X <- (Q2 Q1) X.  That replaces 2 (3 m^2 n + m^3)
// operations by 3 m^2 n + 7 m^3.  All of these are polynomials of G and commute, but once rounded they do not: Q1 G
// and Q2 Q1 are not symmetric and are formed in full.  Mirroring one half of them puts their commutators, as large as the
// roundings, into directions that X has not, where the steps multiply them: 2.3e-2 instead of 5.2e-3 for a matrix
// 4096 x 12288 of rank 32.  Q1 (Q1 G)^T is symmetric up to the rounding of Q1 G.  See pairs() for where steps
// are merged and what that costs in accuracy.
//
// All products of all steps of all shapes run in one persistent launch, one CTA per SM, one or two CTAs to a
// tile: a step of a small matrix takes a few microseconds, less than what three launches cost.  The work is a list of
// jobs (a stage, that is one product, of all matrices of one shape), whose tiles the CTAs take in turn; a tile
// waits until all tiles of the previous stage of its matrix are stored (a counter per matrix in global memory), so
// matrices need not wait for one another and a job's last tiles run beside the next one's first.  Jobs of several
// shapes alternate, so that one shape's tiles fill the time in which another's results travel.  A job waits only for
// jobs before it in the list, and the launch is cooperative: all CTAs are resident, so the waits end.
//
// In a CTA, warp 0 feeds a ring of 128-byte-swizzled operand tiles by TMA, one thread of warp 1 issues the
// MMAs, and eight epilogue warps read the accumulators from one of two TMEM buffers while the next tile
// is multiplied.  Results leave in blocks of 128 x 32 through a second ring: warp 2 fetches a block's addend
// into it, four epilogue warps (one for each quarter of the TMEM lanes; two such groups take turns) replace it by
// the result, and a store warp for each group moves it out by TMA, which clips the edges, and raises the
// matrix's counter after its last block of a tile.  Fetching, storing and signalling take long, so none is left
// to the epilogue warps: products with small K are bound by the epilogue.  Tall matrices (rows > cols) are not
// transposed: both operand layouts (K contiguous, or M/N contiguous) are read by the MMA as they lie.
//
// Measured, from call to result: 4096 x 4096 1.25 ms, 1.1 PFLOP/s executed (symmetric tiles once), and 4096 x 12288 2.2 to
// 2.5 ms, where the chip's power holds fp16 products of 4096 and 8192 in torch at 1.24 and 1.34; two of 17408 x 5120 11.2 ms;
// 128 of 704 x 2816 3.2 to 3.8 ms, bound by the traffic of X's planes, 0.51 GB each, and by 704 in tiles of 256; 48 of
// 256 x 512 122 us and 8 of 1024 x 256 105 us, bound by the way from one stage to the next (load, products, epilogue, store,
// counter: 4 to 8 us).
#include <cuda.h>

#include <algorithm>
#include <cmath>

#include "ha_common.cuh"
#include "newton_schulz.cuh"
#include "umma.cuh"

namespace ha {
namespace {

constexpr int kBM = 128;           // rows of a CTA's part of a tile: the TMEM lanes
constexpr int kBK = 64;            // K elements of a ring slot: one 128-byte swizzle row
constexpr int kGemmThreads = 416;  // operands, MMA, addends, stores; eight epilogue warps; stores
constexpr int kPreciseSteps = 3;   // with a low plane of X in any case
constexpr double kPlainGain = 12;  // of the steps that a single plane's rounding may go through (3.4445^2 is 11.9)
constexpr int kHalf = kBM * kBK * 2;  // bytes of one operand's part of a slot
constexpr int kSlot = 2 * kHalf;
constexpr int kSlots = 5;
constexpr int kBlockCols = 32;
constexpr int kBlock = kBM * kBlockCols * 2;  // bytes of an epilogue block
constexpr int kBlocks = 4;                    // in the ring, each with room for a second result
// Gram matrices along more than 32768 are added up in parts of that.  The matrix unit cuts its sums off instead of rounding
// them, about 2^-24 of the sum at each of K / 16 additions, always downwards: 160 x 524288 was off by 6.1e-3, 160 x 2097152 by
// 2.3e-2.  A part's accumulators are added in fp32 to what the parts before left in the X plane that is free then.
constexpr int kPartBlocks = 32768 / kBK;
constexpr int kGemmSmem = kSlots * kSlot + kBlocks * 2 * kBlock + 1024;  // + alignment

// What becomes of the accumulators (times `scale`):
//   kSquare     stored, of square matrices; with the mirrored tile where the stage says so (tiles on and above
//               the diagonal run)
//   kPoly       the same after adding add * addend and `diag` on the diagonal
//   kPrecise    added to add * low, stored as high and low plane
//   kPlain      stored
//   kFinal      stored as bf16
enum Epilogue { kSquare, kPoly, kPrecise, kPlain, kFinal };

// Tensor maps of a run: per buffer, the boxes it is read and written in.
enum Map {
  kMapXk = 0,       // + 0, 1: X planes, 64 x 128 operand tiles, K contiguous
  kMapXmn = 2,      // + 0, 1: X planes, 64 x 64 operand tiles, M / N contiguous
  kMapXout = 4,     // + 0, 1: X planes, epilogue blocks
  kMapLow = 6,      // low plane, epilogue blocks
  kMapSq = 7,       // + 0 .. 2: square matrices, operand tiles
  kMapSqOut = 10,   // + 0 .. 2: epilogue blocks
  kMapSqMirror = 13,  // + 0 .. 2: mirrored blocks, 32 x 128
  kMapDst = 16,       // the caller's matrices, epilogue blocks
  kMaps = 17
};

struct Stage {
  int M, N, K;        // D is M x N
  int tiles_m, tiles_n, per_matrix;
  uint32_t before;    // a matrix's counter when its previous stage is stored
  int counter;        // of the shape's first matrix
  float scale, add, diag;
  uint8_t map_a, map_b, map_out, map_2, map_add;
  int8_t square_1, square_2, square_out;  // the square matrices read and written, or -1
  float4* diagonal;     // of the shape's square matrices: square i of matrix z at i * diagonal_all + z * diagonal_each
  int diagonal_each, diagonal_all;
  int8_t epilogue, m_fast, a_mn, b_mn, keep_low, by_column;  // *_mn: the operand's M / N index is the contiguous one
  int8_t mirror;        // D is symmetric
  int part;             // blocks of K that are accumulated at once
  float4* sums;         // of earlier parts: of matrix z at z * sums_each
  int64_t sums_each;
};
// A stage of all `count` matrices of its shape.
struct Job {
  uint16_t stage, count;
};

// Kernel parameters; small ones launch faster.
template <int SHAPES, int STAGES, int JOBS>
struct RunArgsOf {
  CUtensorMap map[SHAPES * kMaps];
  Stage stage[STAGES];
  Job job[JOBS];
  int jobs;
  uint32_t* counter;  // one for each matrix
  uint32_t* error;
  uint16_t* dst;      // the caller's matrices, if a stage writes them
  int64_t dst_elems;
};
constexpr int kMaxStages = 3 * HA_NS_MAX_STEPS + 2;  // of one shape
constexpr int kManyShapes = kNsShapes, kManyStages = kNsStages, kManyJobs = kNsStages;
using OneShape = RunArgsOf<1, kMaxStages, kMaxStages>;
using ManyShapes = RunArgsOf<kManyShapes, kManyStages, kManyJobs>;
static_assert(sizeof(ManyShapes) <= 32000, "kernel parameters");

__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float2 unpack_half2(uint32_t w) {
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}

struct TileAt {
  int z, i, j;  // matrix, tile row, tile column
};
// A square matrix's diagonal element q = r + e, r its fp16 value, as (r, e, e / r).  To first order and on the
// diagonal alone, a product gains e1 r2 + r1 e2 there.  In the product with X, row (tall: column) i should gain
// e x_i; it is scaled by 1 + e / r, which is the same for what the diagonal contributes.
__device__ __forceinline__ float4* diagonal_at(const Stage& g, int square, int z, int row) {
  return g.diagonal + int64_t(square) * g.diagonal_all + int64_t(z) * g.diagonal_each + row;
}
__device__ __forceinline__ float4 split_diagonal(float q) {
  const float r = __half2float(__float2half_rn(q)), e = q - r;
  const float f = __fdividef(e, r);  // at most half a step; more, or NaN, where r is subnormal or 0
  return make_float4(r, e, fabsf(f) <= 1.0f / 2048 ? f : 0.0f, 0.0f);
}
// Tile `t` of a job.  Mirrored stages: the tiles on and above the diagonal, column by column (above and not
// below: the last column's products are only as wide as it is, the last row's always 128 or 256 rows).
__device__ __forceinline__ TileAt tile_at(const Stage& g, int t) {
  TileAt a;
  a.z = t / g.per_matrix;
  const int r = t - a.z * g.per_matrix;
  if (g.mirror) {
    int i = int((sqrtf(8.0f * float(r) + 1.0f) - 1.0f) * 0.5f);
    while (i * (i + 1) / 2 > r) --i;
    while ((i + 1) * (i + 2) / 2 <= r) ++i;
    a.j = i;
    a.i = r - i * (i + 1) / 2;
  } else if (g.m_fast) {
    a.j = r / g.tiles_m;
    a.i = r - a.j * g.tiles_m;
  } else {
    a.i = r / g.tiles_n;
    a.j = r - a.i * g.tiles_n;
  }
  return a;
}
// A CTA's (or pair's) walk through the jobs: tiles `first`, `first` + `step`, .. of the whole list.
struct Walk {
  int first, step;
  int skew = 0;  // tiles of the jobs before, modulo `step`
  __device__ __forceinline__ int start() const { return first >= skew ? first - skew : first - skew + step; }
  __device__ __forceinline__ void pass(int tiles) { skew = (skew + tiles) % step; }
};

// Columns of a tile that reach into D, in whole blocks: N of its products.
template <int CG>
__device__ __forceinline__ int width_of(const Stage& g, const TileAt& at) {
  const int cols = g.N - at.j * (128 * CG);
  return cols >= 128 * CG ? 128 * CG : (cols + kBlockCols - 1) & ~(kBlockCols - 1);
}
// Blocks of a CTA's part of a tile: those that reach into D.
template <int CG>
__device__ __forceinline__ int blocks_of(const Stage& g, const TileAt& at, int rank) {
  if (at.i * (128 * CG) + rank * kBM >= g.M) return 0;
  return width_of<CG>(g, at) / kBlockCols;
}

struct Shared {
  uint64_t full[kSlots], empty[kSlots];       // operand slots: loaded; multiplied
  uint64_t acc_full[2], acc_empty[2];         // accumulators: complete; read
  uint64_t blk_full[kBlocks], blk_ready[kBlocks], blk_free[kBlocks];  // addend there; result there; stored
  uint32_t tmem;
  uint32_t granted;                           // tiles of this CTA whose previous stage is known to be stored
  volatile uint32_t stop;
};

// One of the eight epilogue warps, kept over all stages.
struct Warp {
  int lane, quarter, group, rank;
  Walk walk;
  uint32_t ring;           // shared memory: blocks, then their second results
  uint32_t tmem;           // its lanes of the accumulators
  uint32_t n, tile;        // blocks and tiles of this CTA so far
  uint32_t acc, acc_phase;
};

// An epilogue warp's accumulators are read: the next products may use them.
template <int CG>
__device__ __forceinline__ void release_accumulator(Shared& sh, uint32_t acc, int lane) {
  tc_fence_before();
  __syncwarp();
  if (lane == 0) {
    const uint32_t bar = smem_u32(&sh.acc_empty[acc]);
    if (CG == 2)
      mbar_arrive_cluster(cluster_map(bar, 0));
    else
      mbar_arrive(bar);
  }
}

// A tile whose products come in parts: adds up the accumulators of blocks k0, k0 + 2, .. in fp32, in `sums` (this lane's row
// of block k, eight pieces of four columns 128 apart, at 1024 k), and leaves the sum in the last part's.  A thread reads
// what it wrote itself.  (Not inline, and through TMEM: in the epilogue's code it cost every small matrix 2 to 4 us.)
template <int CG>
__device__ __noinline__ bool add_parts(Shared& sh, float4* sums, uint32_t tmem, uint32_t acc, uint32_t phase, int parts,
                                       int k0, int blocks, int lane) {
  for (int part = 1;; ++part) {
    if (!__all_sync(0xffffffffu, mbar_wait(smem_u32(&sh.acc_full[acc]), phase, &sh.stop))) return false;
    tc_fence_after();
#pragma unroll 1
    for (int k = k0; k < blocks; k += 2) {
      const uint32_t from = tmem + acc * (128 * CG) + k * kBlockCols;
      uint32_t v[32];
      tmem_ld32(from, v);
      tmem_ld_wait();
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        float4* at = sums + k * 1024 + j * 128;
        float4 x = make_float4(__uint_as_float(v[4 * j]), __uint_as_float(v[4 * j + 1]), __uint_as_float(v[4 * j + 2]),
                               __uint_as_float(v[4 * j + 3]));
        if (part > 1) {
          const float4 s = __ldcg(at);
          x.x += s.x, x.y += s.y, x.z += s.z, x.w += s.w;
        }
        if (part < parts) __stcg(at, x);
        v[4 * j] = __float_as_uint(x.x), v[4 * j + 1] = __float_as_uint(x.y);
        v[4 * j + 2] = __float_as_uint(x.z), v[4 * j + 3] = __float_as_uint(x.w);
      }
      if (part == parts) tmem_st32(from, v);
    }
    if (part == parts) {
      tmem_st_wait();
      asm volatile("fence.proxy.async;" ::: "memory");  // the next product with X writes the sums' plane by TMA
      return true;
    }
    release_accumulator<CG>(sh, acc, lane);
    acc ^= 1;
    phase ^= acc == 0;
  }
}

template <int CG, int EPI>
__device__ __forceinline__ bool epilogue(const Stage& g, const Job& job, Warp& w, Shared& sh) {
  constexpr bool kSym = EPI == kSquare || EPI == kPoly;
  constexpr bool kAdd = EPI == kPoly || EPI == kPrecise;
  constexpr int kTile = 128 * CG;
  const int lane = w.lane;
  const int mine = w.quarter * 32 + lane;                            // this lane's row of a block:
  const uint32_t row_at = mine * 64, key = (uint32_t(mine) >> 1) & 3;  // its 16-byte piece j lies at j ^ key
  const float add_scale = g.add;
  const int tiles = job.count * g.per_matrix;
  // Of the diagonals: (r, e) of this lane's row from both factors; factor of its row of X, or of its columns in
  // the group's blocks.
  float d[kSym ? 4 : 2 * CG];
  const int parts = EPI == kSquare ? (g.K - 1) / kBK / g.part + 1 : 1;
  auto fetch = [&](const TileAt& at, int k0) {
    if (!kSym && g.by_column) {
#pragma unroll
      for (int u = 0; u < 2 * CG; ++u) {
        const int col = at.j * kTile + (k0 + 2 * u) * kBlockCols + lane;
        d[u] = col < g.N ? __ldcg(&diagonal_at(g, g.square_1, at.z, col)->z) : 0.0f;
      }
    } else {
      const int row = at.i * kTile + w.rank * kBM + mine;
      if (kSym) {
        float4 a = make_float4(0.0f, 0.0f, 0.0f, 0.0f), b = a;
        if (row < g.M) {
          a = __ldcg(diagonal_at(g, g.square_1, at.z, row));
          b = __ldcg(diagonal_at(g, g.square_2, at.z, row));
        }
        d[0] = a.x, d[1] = a.y, d[2 * kSym] = b.x, d[3 * kSym] = b.y;
      } else {
        d[0] = row < g.M ? __ldcg(&diagonal_at(g, g.square_1, at.z, row)->z) : 0.0f;
      }
    }
  };
  auto wanted = [&](const TileAt& at) { return g.square_1 >= 0 && (!kSym || at.i == at.j); };
  bool fetched = false;
  for (int t = w.walk.start(); t < tiles; t += w.walk.step) {
    const TileAt at = tile_at(g, t);
    const int blocks = blocks_of<CG>(g, at, w.rank);
    const int row = at.i * kTile + w.rank * kBM + mine, k0 = int((w.n ^ uint32_t(w.group)) & 1);
    float scale = g.scale, diag = g.diag;
    __half2 by_column[CG];  // factors less 1
    ++w.tile;
    if (wanted(at)) {
      if (!fetched) {
        if (!granted_wait_warp(&sh.granted, w.tile, &sh.stop, lane)) return false;
        fetch(at, k0);
      }
      if (kSym) {
        diag += EPI == kPoly ? d[1] * (add_scale + 2.0f * scale * d[0])
                             : scale * (d[0] * d[3 * kSym] + d[1] * d[2 * kSym]);
      } else if (!g.by_column) {
        scale *= 1.0f + d[0];
      } else {
#pragma unroll
        for (int u = 0; u < CG; ++u) by_column[u] = __floats2half2_rn(d[2 * u], d[2 * u + 1]);
      }
    }
    // The next tile's, if it may be read already: loaded while this one is worked on.
    fetched = false;
    if (t + w.walk.step < tiles) {
      const TileAt next = tile_at(g, t + w.walk.step);
      if (wanted(next) && granted_to_warp(&sh.granted, w.tile + 1, lane)) {
        fetch(next, k0 ^ (blocks & 1));
        fetched = true;
      }
    }
    if (EPI == kSquare && parts > 1) {
      const int slot = ((t - at.z * g.per_matrix) * CG + w.rank) * (4 * CG);
      if (!add_parts<CG>(sh, g.sums + at.z * g.sums_each + int64_t(slot) * 1024 + mine, w.tmem, w.acc, w.acc_phase, parts, k0,
                         blocks, lane))
        return false;
      w.acc += parts - 1;  // the accumulators of the last part
      w.acc_phase ^= (w.acc >> 1) & 1;
      w.acc &= 1;
    }
    if (!__all_sync(0xffffffffu, mbar_wait(smem_u32(&sh.acc_full[w.acc]), w.acc_phase, &sh.stop))) return false;
    tc_fence_after();
    const uint32_t d = w.tmem + w.acc * kTile;
#pragma unroll 1
    for (int k = k0; k < blocks; k += 2) {
      const uint32_t b = (w.n + k) % kBlocks, phase = ((w.n + k) / kBlocks) & 1;
      const uint32_t block = w.ring + b * kBlock, second = block + kBlocks * kBlock;
      const int col = at.j * kTile + k * kBlockCols;
      uint32_t v[32];
      tmem_ld32(d + k * kBlockCols, v);
      if (!__all_sync(0xffffffffu, mbar_wait(smem_u32(&sh.blk_full[b]), phase, &sh.stop))) return false;
      uint32_t add[16];  // 32 packed addends
      if (kAdd) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                       : "=r"(add[4 * j]), "=r"(add[4 * j + 1]), "=r"(add[4 * j + 2]), "=r"(add[4 * j + 3])
                       : "r"(block + row_at + ((j ^ key) << 4))
                       : "memory");
      }
      tmem_ld_wait();
      if (!kSym && g.by_column) {
        const __half2 two = CG == 2 && k >= 4 ? by_column[CG - 1] : by_column[0];
        const float f = 1.0f + ((k & 2) ? __high2float(two) : __low2float(two));
#pragma unroll
        for (int j = 0; j < 32; ++j) v[j] = __float_as_uint(__uint_as_float(v[j]) * __shfl_sync(0xffffffffu, f, j));
      }
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        float x = __uint_as_float(v[2 * j]) * scale, y = __uint_as_float(v[2 * j + 1]) * scale;
        if (kAdd) {
          const float2 a = unpack_half2(add[j]);
          x = __fmaf_rn(add_scale, a.x, x);
          y = __fmaf_rn(add_scale, a.y, y);
        }
        v[2 * j] = __float_as_uint(x);
        v[2 * j + 1] = __float_as_uint(y);
      }
      if (kSym && col == row - lane && at.i == at.j) {  // lane l's element l is on the diagonal
        float mine = 0.0f;
#pragma unroll
        for (int j = 0; j < 32; ++j)
          if (j == lane) {
            mine = __uint_as_float(v[j]) + diag;
            v[j] = __float_as_uint(mine);
          }
        const float4 q = split_diagonal(mine);  // where a tile off the diagonal has its mirrored block
        asm volatile("st.shared.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(second + lane * 16), "f"(q.x), "f"(q.y),
                     "f"(q.z), "f"(q.w)
                     : "memory");
      }
      uint32_t out[16], low[16];  // 32 packed results
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const float x = __uint_as_float(v[2 * j]), y = __uint_as_float(v[2 * j + 1]);
        if (EPI == kFinal) {
          const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
          out[j] = *reinterpret_cast<const uint32_t*>(&h);
        } else {
          out[j] = pack_half2(x, y);
        }
        if (EPI == kPrecise) {
          const float2 a = unpack_half2(out[j]);
          low[j] = pack_half2((x - a.x) * kScaleLo, (y - a.y) * kScaleLo);
        }
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t* o = (EPI == kPrecise ? low : out) + 4 * j;
        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(block + row_at + ((j ^ key) << 4)), "r"(o[0]),
                     "r"(o[1]), "r"(o[2]), "r"(o[3])
                     : "memory");
        if (EPI == kPrecise)
          asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(second + row_at + ((j ^ key) << 4)),
                       "r"(out[4 * j]), "r"(out[4 * j + 1]), "r"(out[4 * j + 2]), "r"(out[4 * j + 3])
                       : "memory");
      }
      if (kSym && g.mirror && at.i != at.j) {
        // transposed, 32 rows of 128: lanes 2l and 2l + 1 exchange halves so that each writes two
        // neighbours of one row
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          const uint32_t other = __shfl_xor_sync(0xffffffffu, out[j], 1);
          const uint32_t o = (lane & 1) ? __byte_perm(other, out[j], 0x7632) : __byte_perm(out[j], other, 0x5410);
          asm volatile("st.shared.b32 [%0], %1;" ::"r"(second + (2 * j + (lane & 1)) * (2 * kBM) + w.quarter * 64 +
                                                       (lane >> 1) * 4),
                       "r"(o)
                       : "memory");
        }
      }
      fence_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&sh.blk_ready[b]));
    }
    w.n += blocks;
    release_accumulator<CG>(sh, w.acc, lane);
    if (++w.acc == 2) w.acc = 0, w.acc_phase ^= 1;
  }
  return true;
}

// Warp 2, one thread: a block's addend, or only the block itself, to the epilogue warps.
template <int CG, class Args>
__device__ __forceinline__ void feed_blocks(const Args& p, Shared& sh, uint32_t ring, Walk walk, int rank) {
  uint32_t n = 0, tile = 0;
  for (int q = 0; q < p.jobs; ++q) {
    const Job job = p.job[q];
    const Stage& g = p.stage[job.stage];
    const bool add = g.epilogue == kPoly || g.epilogue == kPrecise;
    const int tiles = job.count * g.per_matrix;
    for (int t = walk.start(); t < tiles; t += walk.step) {
      ++tile;
      const TileAt at = tile_at(g, t);
      const int blocks = blocks_of<CG>(g, at, rank);
      for (int k = 0; k < blocks; ++k, ++n) {
        const uint32_t b = n % kBlocks, full = smem_u32(&sh.blk_full[b]);
        if (!mbar_wait(smem_u32(&sh.blk_free[b]), ((n / kBlocks) & 1) ^ 1, &sh.stop)) return;
        if (!add) {
          mbar_arrive(full);
          continue;
        }
        if (k == 0 && !granted_wait(&sh.granted, tile, &sh.stop)) return;
        mbar_expect_tx(full, kBlock);
        tma_load_3d<1>(ring + b * kBlock, &p.map[g.map_add], full, at.j * (128 * CG) + k * kBlockCols,
                       at.i * (128 * CG) + rank * kBM, at.z);
      }
    }
    walk.pass(tiles);
  }
}

// Warps 3 and 12, one thread each: the blocks that one epilogue group finished, to memory; then the counter.
template <int CG, class Args>
__device__ __forceinline__ void store_blocks(const Args& p, Shared& sh, uint32_t ring, Walk walk, int rank,
                                             uint32_t group) {
  uint32_t n = 0, tile = 0;
  for (int q = 0; q < p.jobs; ++q) {
    const Job job = p.job[q];
    const Stage& g = p.stage[job.stage];
    const int tiles = job.count * g.per_matrix;
    for (int t = walk.start(); t < tiles; t += walk.step) {
      ++tile;
      const TileAt at = tile_at(g, t);
      const int blocks = blocks_of<CG>(g, at, rank), row = at.i * (128 * CG) + rank * kBM;
      const bool more = t + walk.step < tiles;
      const int k0 = int((n ^ group) & 1);
      uint32_t last = kBlocks;  // block of the store before, not yet handed back
      for (int k = k0; k < blocks; k += 2) {
        const uint32_t b = (n + k) % kBlocks, block = ring + b * kBlock, second = block + kBlocks * kBlock;
        const int col = at.j * (128 * CG) + k * kBlockCols;
        if (!mbar_wait(smem_u32(&sh.blk_ready[b]), ((n + k) / kBlocks) & 1, &sh.stop)) return;
        if (g.epilogue == kPrecise) {
          tma_store_3d(&p.map[g.map_out], second, col, row, at.z);
          if (g.keep_low) tma_store_3d(&p.map[g.map_2], block, col, row, at.z);
        } else {
          tma_store_3d(&p.map[g.map_out], block, col, row, at.z);
          if (at.i != at.j) {
            if (g.mirror) tma_store_3d(&p.map[g.map_2], second, row, col, at.z);
          } else if (g.square_out >= 0 && col >= row && col < row + kBM) {  // the block holds 32 diagonal elements
            bulk_store(diagonal_at(g, g.square_out, at.z, col), second, kBlockCols * sizeof(float4));
          }
        }
        tma_store_commit();
        // With more tiles to come a block is handed back as soon as it has been read: four of them are few
        // (3.6 ms against 4.0 for 128 of 704 x 2816).  In the last tile the next store goes first (100 us
        // against 103 for 8 of 1024 x 256).
        if (more) {
          tma_store_wait_read<0>();
          mbar_arrive(smem_u32(&sh.blk_free[b]));
        } else {
          if (last < kBlocks) {
            tma_store_wait_read<1>();
            mbar_arrive(smem_u32(&sh.blk_free[last]));
          }
          last = b;
        }
      }
      n += blocks;
      tma_store_wait_all();
      // A tile without blocks of this group must not be counted before its matrix's previous stage is stored:
      // the counter tells stages apart only as long as they are raised one after another.
      if (last < kBlocks) mbar_arrive(smem_u32(&sh.blk_free[last]));
      if (k0 >= blocks && !granted_wait(&sh.granted, tile, &sh.stop)) return;
      counter_raise(p.counter + g.counter + at.z);
    }
    walk.pass(tiles);
  }
}

// CG: CTAs of a tile (1: 128 x 128; 2: 256 x 256, each CTA with 128 rows of A and of D and half of the
// columns of B).
template <int CG, class Args>
__global__ void __launch_bounds__(kGemmThreads, 1) newton_schulz_kernel(const __grid_constant__ Args p) {
  constexpr int kTile = 128 * CG;         // rows and columns of a tile
  constexpr int kColumns = 2 * kTile;     // TMEM columns: two accumulators
  extern __shared__ uint8_t smem_raw[];
  __shared__ Shared sh;
  const uint32_t ring = (smem_u32(smem_raw) + 1023) & ~1023u;
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const uint32_t rank = CG == 2 ? cluster_rank() : 0;

  if (threadIdx.x == 0) {
    sh.stop = 0;
    sh.granted = 0;
    for (int i = 0; i < kSlots; ++i) {
      mbar_init(smem_u32(&sh.full[i]), 1);
      mbar_init(smem_u32(&sh.empty[i]), 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_u32(&sh.acc_full[i]), 1);
      mbar_init(smem_u32(&sh.acc_empty[i]), 8 * CG);
    }
    for (int i = 0; i < kBlocks; ++i) {
      mbar_init(smem_u32(&sh.blk_full[i]), 1);
      mbar_init(smem_u32(&sh.blk_ready[i]), 4);
      mbar_init(smem_u32(&sh.blk_free[i]), 1);
    }
    mbar_fence_init();
  }
  if (warp == 1) tmem_alloc<CG>(smem_u32(&sh.tmem), kColumns);
  tc_fence_before();
  if (CG == 2)
    cluster_sync();  // the pair's barriers exist before either CTA signals the other's
  else
    __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sh.tmem;
  Walk walk{int(blockIdx.x) / CG, int(gridDim.x) / CG};

  if (warp == 0) {
    if (elect_one()) {
      int slot = 0;
      uint32_t phase = 0, tile = 0;
      bool ok = true;
      for (int q = 0; q < p.jobs && ok; ++q) {
        const Job job = p.job[q];
        const Stage& g = p.stage[job.stage];
        const int tiles = job.count * g.per_matrix;
        const CUtensorMap *map_a = &p.map[g.map_a], *map_b = &p.map[g.map_b];
        const int kblocks = (g.K + kBK - 1) / kBK;
        const bool a_mn = g.a_mn, b_mn = g.b_mn;
        int ready = -1;
        for (int t = walk.start(); t < tiles && ok; t += walk.step) {
          const TileAt at = tile_at(g, t);
          if (at.z != ready) {
            ok = counter_wait(p.counter + g.counter + at.z, g.before, &sh.stop);
            if (!ok) break;
            ready = at.z;
          }
          grant(&sh.granted, ++tile);
          const int m0 = at.i * kTile + int(rank) * kBM;
          const int n0 = at.j * kTile + (CG == 2 ? int(rank) * (width_of<CG>(g, at) / 2) : 0);
          for (int kb = 0; kb < kblocks; ++kb) {
            ok = mbar_wait(smem_u32(&sh.empty[slot]), phase ^ 1, &sh.stop);
            if (!ok) break;
            uint32_t full = smem_u32(&sh.full[slot]);
            const uint32_t a = ring + slot * kSlot, b = a + kHalf;
            if (rank == 0) mbar_expect_tx(full, CG * kSlot);  // the first CTA's barrier counts both halves
            if (CG == 2) full = cluster_map(full, 0);
            if (a_mn) {
              tma_load_3d<CG>(a, map_a, full, m0, kb * kBK, at.z);
              tma_load_3d<CG>(a + 8192, map_a, full, m0 + 64, kb * kBK, at.z);
            } else {
              tma_load_3d<CG>(a, map_a, full, kb * kBK, m0, at.z);
            }
            if (b_mn) {
              tma_load_3d<CG>(b, map_b, full, n0, kb * kBK, at.z);
              tma_load_3d<CG>(b + 8192, map_b, full, n0 + 64, kb * kBK, at.z);
            } else {
              tma_load_3d<CG>(b, map_b, full, kb * kBK, n0, at.z);
            }
            if (++slot == kSlots) slot = 0, phase ^= 1;
          }
        }
        walk.pass(tiles);
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    if (rank == 0 && elect_one()) {
      int slot = 0;
      uint32_t phase = 0, acc = 0, acc_phase = 0;
      bool ok = true;
      for (int q = 0; q < p.jobs && ok; ++q) {
        const Job job = p.job[q];
        const Stage& g = p.stage[job.stage];
        const int tiles = job.count * g.per_matrix;
        const int kblocks = (g.K + kBK - 1) / kBK;
        const uint32_t lead_a = g.a_mn ? 8192 : 16, lead_b = g.b_mn ? 8192 : 16;
        const uint32_t next_a = g.a_mn ? kStepMN : kStepK, next_b = g.b_mn ? kStepMN : kStepK;
        for (int t = walk.start(); t < tiles && ok; t += walk.step) {
          const int width = g.N % kTile == 0 ? kTile : width_of<CG>(g, tile_at(g, t));
          const uint32_t idesc = f16_idesc(kTile, width, g.a_mn, g.b_mn);
          ok = mbar_wait(smem_u32(&sh.acc_empty[acc]), acc_phase ^ 1, &sh.stop);
          if (!ok) break;
          tc_fence_after();
          uint32_t d = tmem + acc * kTile;
          int in_part = 0;
          for (int kb = 0; kb < kblocks; ++kb) {
            if (in_part == g.part) {  // the next part, into the other accumulators
              mma_commit<CG>(smem_u32(&sh.acc_full[acc]));
              if (++acc == 2) acc = 0, acc_phase ^= 1;
              ok = mbar_wait(smem_u32(&sh.acc_empty[acc]), acc_phase ^ 1, &sh.stop);
              if (!ok) break;
              tc_fence_after();
              d = tmem + acc * kTile;
              in_part = 0;
            }
            ok = mbar_wait(smem_u32(&sh.full[slot]), phase, &sh.stop);
            if (!ok) break;
            tc_fence_after();
            const uint32_t a = ring + slot * kSlot, b = a + kHalf;
            const uint32_t da = smem_desc(a, lead_a), db = smem_desc(b, lead_b);
#pragma unroll
            for (int k = 0; k < kBK / 16; ++k)
              mma_f16<CG>(d, da + k * next_a, db + k * next_b, idesc, in_part > 0 || k > 0);
            ++in_part;
            mma_commit<CG>(smem_u32(&sh.empty[slot]));
            if (++slot == kSlots) slot = 0, phase ^= 1;
          }
          if (ok) mma_commit<CG>(smem_u32(&sh.acc_full[acc]));
          if (++acc == 2) acc = 0, acc_phase ^= 1;
        }
        walk.pass(tiles);
      }
    }
    __syncwarp();
  } else if (warp == 2) {
    if (lane == 0) feed_blocks<CG>(p, sh, ring + kSlots * kSlot, walk, int(rank));
    __syncwarp();
  } else if (warp == 3 || warp == 12) {
    if (lane == 0) {
      store_blocks<CG>(p, sh, ring + kSlots * kSlot, walk, int(rank), warp == 3 ? 0 : 1);
      tma_store_wait_all();
      if (p.dst != nullptr && any_gave_up(p.error)) sh.stop = 1;
    }
    __syncwarp();
  } else {
    Warp w{};
    w.lane = lane;
    w.quarter = warp & 3;  // the TMEM lanes this warp may read: 32 * quarter ..
    w.group = (warp - 4) >> 2;
    w.walk = walk;
    w.rank = int(rank);
    w.ring = ring + kSlots * kSlot;
    w.tmem = tmem + (uint32_t(w.quarter * 32) << 16);
    bool ok = true;
    for (int q = 0; q < p.jobs && ok; ++q) {
      const Job job = p.job[q];
      const Stage& g = p.stage[job.stage];
      switch (g.epilogue) {
        case kSquare: ok = epilogue<CG, kSquare>(g, job, w, sh); break;
        case kPoly: ok = epilogue<CG, kPoly>(g, job, w, sh); break;
        case kPrecise: ok = epilogue<CG, kPrecise>(g, job, w, sh); break;
        case kPlain: ok = epilogue<CG, kPlain>(g, job, w, sh); break;
        default: ok = epilogue<CG, kFinal>(g, job, w, sh); break;
      }
      w.walk.pass(job.count * g.per_matrix);
    }
  }
  __syncthreads();
  if (sh.stop) {  // a wait ran out: let copies and products in flight end before their memory is given up
    if (threadIdx.x == 0) gave_up(p.error);
    const uint64_t t0 = global_ns();
    while (global_ns() - t0 < 2000000) {
    }
    __syncthreads();
    if (p.dst != nullptr) fill_nan(p.dst, p.dst_elems, kGemmThreads);
    __syncthreads();
  }
  tc_fence_before();
  if (CG == 2) cluster_sync();  // neither CTA leaves while the other's products read or write its memory
  tc_fence_after();
  if (warp == 1) tmem_dealloc<CG>(tmem, kColumns);
}

// ---------------------------------------------------------------- host side
using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                 const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                 CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiled encode_tiled() {
  static EncodeTiled fn = [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      f = nullptr;
    return reinterpret_cast<EncodeTiled>(f);
  }();
  return fn;
}

// fp16 matrices, rows `ld` and matrices `plane` elements apart.
struct Operand {
  const __half* base;
  int64_t rows, cols, ld, plane;
};

// `n` of them, read or written in box_cols x box_rows pieces.
int make_map(CUtensorMap* map, const Operand& x, int64_t n, int box_cols, int box_rows, CUtensorMapSwizzle swizzle) {
  const EncodeTiled fn = encode_tiled();
  if (fn == nullptr) return fail(HA_ERR_CUDA, "cuTensorMapEncodeTiled is not available");
  const cuuint64_t dims[3] = {cuuint64_t(x.cols), cuuint64_t(x.rows), cuuint64_t(n)};
  const cuuint64_t strides[2] = {cuuint64_t(x.ld) * 2, cuuint64_t(x.plane) * 2};
  const cuuint32_t box[3] = {cuuint32_t(box_cols), cuuint32_t(box_rows), 1};
  const cuuint32_t step[3] = {1, 1, 1};
  const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<__half*>(x.base), dims, strides, box, step,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS)
    return fail(HA_ERR_CUDA, "cuTensorMapEncodeTiled: error %d for %lld x %lld x %lld", int(r), (long long)n,
                (long long)x.rows, (long long)x.cols);
  return HA_OK;
}

int sm_count(int* out) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess ||
      cudaDeviceGetAttribute(out, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
    return check_launch("ns_run (device query)");
  return HA_OK;
}

// How many of the leading pairs of steps, (0, 1) and (2, 3), run as one product with X.  Each saves 3 m^2 (n - m)
// operations, costs 2 m^3 and a stage, and moves X's planes once less.
// Speed, in us without / with: first pair, n = 1.5 m, 204 of 256 x 384 347 / 329, 51 of 512 x 768 331 / 320, 33 of
// 640 x 960 382 / 379, 2048 x 3072 288 / 296; n = 2 m, 10 of 1024 x 2048 430 / 414, 4096 x 8192 2109 / 2040; two matrices alone
// take 2 to 4 us more.  Second pair, n = 2 m, 25 of 640 x 1280 359 / 356, 10 of 1024 x 2048 414 / 411, 2048 x 4096 343 / 339,
// 4096 x 8192 2040 / 1933; n = 2.5 m, 20 of 640 x 1600 351 / 333, 4096 x 10240 2371 / 2286.
// Relative error against 64-bit results with none / the first / both (1.66e-3 is rounding them to bf16): normal
// elements, 640 x 1920 1.81 / 1.81 / 2.19e-3, but both 2.33e-3 at 512 x 1280: hence 640; rank 32, 1024 x 4096 3.05 / 3.08 / 4.92e-3;
// rank 1 3.76 / 4.08 / 4.68e-3.
int pairs(int64_t m, int64_t n, const float* coef, int steps) {
  int count = 0;
  double top = 1.0;  // bound of the singular values before step s
  for (int s = 0; s + 2 <= steps && s < 4; s += 2) {
    const bool worth = s == 0 ? m >= 256 && (n >= m * 2 || (m <= 512 && n * 2 >= m * 3))
                              : m >= 640 && (n * 2 >= m * 5 || (m >= 2048 && n >= m * 2));
    const double between = ns_growth(coef + 3 * s, top);
    // both factors' product has to fit the planes like each of them
    if (!worth || ns_factor(coef + 3 * s, top) * ns_factor(coef + 3 * s + 3, between) > kMaxFactor) break;
    top = ns_growth(coef + 3 * s + 3, between);
    ++count;
  }
  return count;
}

int make_maps(const NsBatch& b, CUtensorMap* maps) {
  int rc = HA_OK;
  auto map = [&](int to, const Operand& x, int cols, int rows, CUtensorMapSwizzle swizzle) {
    if (rc == HA_OK) rc = make_map(&maps[to], x, b.n, cols, rows, swizzle);
  };
  auto operand = [&](int to, const Operand& x, int rows) { map(to, x, 64, rows, CU_TENSOR_MAP_SWIZZLE_128B); };
  auto block = [&](int to, const Operand& x) { map(to, x, kBlockCols, kBM, CU_TENSOR_MAP_SWIZZLE_64B); };
  for (int i = 0; i < 2; ++i) {
    const Operand x{b.hi[i], b.rows, b.cols, b.ld_x, b.plane_x};
    operand(kMapXk + i, x, 128);
    operand(kMapXmn + i, x, 64);
    block(kMapXout + i, x);
  }
  if (b.dst != nullptr)
    block(kMapDst, Operand{reinterpret_cast<const __half*>(b.dst), b.rows, b.cols, b.cols, b.rows * b.cols});
  block(kMapLow, Operand{b.lo, b.rows, b.cols, b.ld_x, b.plane_x});
  for (int i = 0; i < 3; ++i) {
    const Operand q{b.square[i], b.m, b.m, b.ld_g, b.plane_g};
    operand(kMapSq + i, q, 128);
    block(kMapSqOut + i, q);
    map(kMapSqMirror + i, q, kBM, kBlockCols, CU_TENSOR_MAP_SWIZZLE_NONE);
  }
  return rc;
}

// The stages of a shape, whose maps start at `map0` and counters at `counter`; returns their number.
int make_stages(NsBatch* shape, const float* coef, int steps, int map0, int counter, Stage* stages) {
  const NsBatch& b = *shape;
  int count = 0;
  const bool tall = b.rows > b.cols;
  const int m = int(b.m), n = int(tall ? b.rows : b.cols);
  auto add = [&](Epilogue e, int M, int N, int K) {
    Stage& g = stages[count++];
    g = Stage{};
    g.counter = counter;
    g.epilogue = int8_t(e);
    g.M = M, g.N = N, g.K = K;
    g.square_1 = g.square_2 = g.square_out = -1;
    g.diagonal = b.diagonal[0];
    g.diagonal_each = int(b.m_pad);
    g.diagonal_all = int(b.m_pad * b.n);
    return &g;
  };
  // x y^T of square matrices x and y; `mirror`: it is symmetric
  auto multiply = [&](Epilogue e, int x, int y, int to, bool mirror) {
    Stage* g = add(e, m, m, m);
    g->mirror = mirror;
    g->map_a = uint8_t(map0 + kMapSq + x);
    g->map_b = uint8_t(map0 + kMapSq + y);
    g->map_out = uint8_t(map0 + kMapSqOut + to);
    g->map_2 = uint8_t(map0 + kMapSqMirror + to);
    g->map_add = uint8_t(map0 + kMapSqOut + x);
    g->square_1 = int8_t(x);
    g->square_2 = int8_t(y);
    g->square_out = int8_t(to);
    g->scale = 1.0f / kScaleG;
    return g;
  };
  auto factor = [&](int gram, int to, const float* c) {  // c0 I + c1 G + c2 G G
    Stage* g = multiply(kPoly, gram, gram, to, true);
    g->scale = c[2] / kScaleG;
    g->add = c[1];
    g->diag = c[0] * kScaleG;
  };
  const int merged = pairs(m, n, coef, steps);
  double left[HA_NS_MAX_STEPS + 1], top = 1.0;  // what steps s .. multiply by at most
  for (int s = 0; s < steps; ++s) {
    left[s] = ns_factor(coef + 3 * s, top);
    top = ns_growth(coef + 3 * s, top);
  }
  left[steps] = 1.0;
  for (int s = steps; s-- > 0;) left[s] = left[s + 1] * (left[s] > 1.0 ? left[s] : 1.0);
  auto low_before = [&](int s) { return s < steps && (s < kPreciseSteps || left[s] > kPlainGain); };
  int cur = 0;
  for (int s = 0; s < steps;) {
    const bool pair = s < 2 * merged;
    const float* c = coef + 3 * s;
    Stage* g = add(kSquare, m, m, n);
    g->mirror = true;
    g->a_mn = g->b_mn = tall;
    g->sums = reinterpret_cast<float4*>(b.hi[cur ^ 1]);  // (the products that read it are done)
    g->sums_each = b.plane_x * 2 / int64_t(sizeof(float4));
    g->map_a = g->map_b = uint8_t(map0 + (tall ? kMapXmn : kMapXk) + cur);
    g->map_out = uint8_t(map0 + kMapSqOut);
    g->map_2 = uint8_t(map0 + kMapSqMirror);
    g->square_out = 0;
    g->scale = kScaleG / (kScaleX * kScaleX);
    factor(0, 1, c);
    if (pair) {
      multiply(kSquare, 1, 0, 2, false);  // Q1 G
      multiply(kSquare, 1, 2, 0, true);   // G' = Q1 (Q1 G)^T
      factor(0, 2, c + 3);
      multiply(kSquare, 2, 1, 0, false);  // Q2 Q1
    }
    const int q = pair ? 0 : 1;
    g = add(low_before(s) ? kPrecise : kPlain, int(b.rows), int(b.cols), m);
    g->b_mn = !tall;
    g->by_column = tall;
    g->square_1 = int8_t(q);
    g->map_a = uint8_t(map0 + (tall ? kMapXk + cur : kMapSq + q));
    g->map_b = uint8_t(map0 + (tall ? kMapSq + q : kMapXmn + cur));
    cur ^= 1;
    g->map_out = uint8_t(map0 + kMapXout + cur);
    g->map_2 = g->map_add = uint8_t(map0 + kMapLow);  // rewritten in place, block by block
    g->scale = 1.0f / kScaleG;
    g->add = (pair ? c[0] * c[3] : c[0]) / kScaleLo;
    s += pair ? 2 : 1;
    g->keep_low = low_before(s);  // the next step reads it
  }
  Stage& last = stages[count - 1];
  shape->out = cur;
  shape->rounded = b.bf16 && last.epilogue == kPlain;
  if (shape->rounded) {
    last.epilogue = kFinal;
    last.scale /= kScaleX;
    if (b.dst != nullptr) {
      last.map_out = uint8_t(map0 + kMapDst);
      shape->out = -1;
    }
  }
  return count;
}

// Cuts a shape's stages into tiles; adds its share of the chip's time, in cycles, to *work, and the time
// that it would take alone to *alone.  False if there are too many tiles.
//
// The tile is 256 x 256 on a CTA pair or 128 x 128 on one CTA.  The large one reads half the operand bytes per product:
// measured, 64 of K take 600 cycles of a pair's tile and 500 of the small one, a quarter of it, which waits
// for its operands.  But a stage of large tiles takes 16 thousand cycles from its first load to its last counter
// beside that, of small ones 8 thousand, unless there are tiles to fill the wait, and few large tiles leave
// SMs idle: small / large in us, 16 x 512 x 512: 122 / 157; 1 x 2048 x 2048: 218 / 265; 19 x 1152 x 1600:
// 1181 / 1006; 13 x 1920 x 1536: 1514 / 1129.
bool cut(Stage* stages, int count, int64_t batch, int cg, int workers, double* work, double* alone) {
  const int tile = 128 * cg;
  uint32_t before = 0;
  for (int s = 0; s < count; ++s) {
    Stage& g = stages[s];
    g.tiles_m = (g.M + tile - 1) / tile;
    g.tiles_n = (g.N + tile - 1) / tile;
    const int64_t per = g.mirror ? int64_t(g.tiles_m) * (g.tiles_m + 1) / 2 : int64_t(g.tiles_m) * g.tiles_n;
    if (per * batch > 0x3fffffff || before > 0x7fffffff) return false;
    g.per_matrix = int(per);
    g.m_fast = g.tiles_m <= g.tiles_n;  // the shorter side first: its operand panels stay in L2
    g.before = before;
    // (a Gram matrix too large for the free plane is nearly as wide as long: no sum of that one's side is long)
    g.part = g.sums != nullptr && per * tile * tile * 4 <= g.sums_each * int64_t(sizeof(float4)) ? kPartBlocks : 0x7fffffff;
    before += uint32_t(per) * 2 * cg;   // both store warps of each of its CTAs
    const double tiles = double(per * batch), each = (cg == 1 ? 500.0 : 600.0) * ((g.K + kBK - 1) / kBK);
    const double wait = cg == 1 ? 8e3 : 16e3;
    const double spared = double(g.tiles_n * tile - g.N) / tile * double(g.tiles_m * batch);  // in the last column
    *work += each * (tiles - spared) / workers;
    *alone += each * double((per * batch + workers - 1) / workers) + (tiles > workers ? wait * workers / tiles : wait);
  }
  return true;
}

// The jobs of one shape in the order in which they run, each with the share of the shape's work before it.
struct Placed {
  Job job;
  double at;
};
int place(const Stage* stages, int first_stage, int count, const NsBatch& b, Placed* out) {
  int n = 0;
  double total = 0.0, done = 0.0;
  auto cost = [&](int s) { return double(stages[s].per_matrix) * ((stages[s].K + kBK - 1) / kBK); };
  for (int s = 0; s < count; ++s) total += cost(s);
  for (int s = 0; s < count; ++s) {
    out[n++] = Placed{Job{uint16_t(first_stage + s), uint16_t(b.n)}, done / total};
    done += cost(s);
  }
  return n;
}

template <int CG, class Args>
int launch(const Args& p, int sms, cudaStream_t st) {
  auto* kernel = newton_schulz_kernel<CG, Args>;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kGemmSmem) != cudaSuccess)
    return check_launch("newton_schulz_kernel (shared memory)");
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(unsigned(sms / CG * CG));
  cfg.blockDim = dim3(kGemmThreads);
  cfg.dynamicSmemBytes = kGemmSmem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeCooperative;
  attr[0].val.cooperative = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = CG;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = CG == 2 ? 2 : 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, p);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return fail(HA_ERR_CUDA, "newton_schulz_kernel: %s", cudaGetErrorString(e));
  }
  return HA_OK;
}

// One launch for `n` shapes.
template <class Args>
int run(NsBatch** shapes, int n, const float* coef, int steps, int sms, cudaStream_t st) {
  constexpr int kRoom = int(sizeof(Args::job) / sizeof(Job));
  static thread_local Args p;
  static thread_local Placed list[kRoom];
  int first[kManyShapes + 1] = {0};
  for (int i = 0; i < n; ++i) {
    if (int rc = make_maps(*shapes[i], p.map + i * kMaps)) return rc;
    const int counter = int(shapes[i]->counter - shapes[0]->counter);
    first[i + 1] = first[i] + make_stages(shapes[i], coef, steps, i * kMaps, counter, p.stage + first[i]);
  }
  auto cost = [&](int cg) {
    double work = 0.0, longest = 0.0;
    for (int i = 0; i < n; ++i) {
      double alone = 0.0;
      if (!cut(p.stage + first[i], first[i + 1] - first[i], shapes[i]->n, cg, sms / cg, &work, &alone)) return -1.0;
      if (alone > longest) longest = alone;
    }
    return work > longest ? work : longest;
  };
  const double two = cost(2), one = cost(1);
  if (one < 0) return fail(HA_ERR_INVALID, "Newton-Schulz products with too many tiles");
  const int cg = two < 0 || one <= two ? 1 : 2;
  if (cg == 2) cost(2);
  int jobs = 0;
  for (int i = 0; i < n; ++i)
    jobs += place(p.stage + first[i], first[i], first[i + 1] - first[i], *shapes[i], list + jobs);
  std::stable_sort(list, list + jobs, [](const Placed& a, const Placed& b) { return a.at < b.at; });
  for (int q = 0; q < jobs; ++q) p.job[q] = list[q].job;
  p.jobs = jobs;
  p.counter = shapes[0]->counter;
  p.error = shapes[0]->error;
  p.dst = n == 1 && shapes[0]->out < 0 ? shapes[0]->dst : nullptr;
  p.dst_elems = shapes[0]->n * shapes[0]->rows * shapes[0]->cols;
  return cg == 1 ? launch<1>(p, sms, st) : launch<2>(p, sms, st);
}

int64_t up(int64_t x, int64_t a) { return (x + a - 1) / a * a; }

}  // namespace

int ns_map(CUtensorMap* map, const __half* plane, const NsBatch& b, int box_cols, int box_rows) {
  return make_map(map, Operand{plane, b.rows, b.cols, b.ld_x, b.plane_x}, b.n, box_cols, box_rows,
                  CU_TENSOR_MAP_SWIZZLE_128B);
}

double ns_growth(const float* c, double s) {
  const double a = c[0], b = c[1], d = c[2];
  auto value = [&](double t) { return std::fabs(t * (a + t * t * (b + t * t * d))); };
  double top = value(s);
  auto consider = [&](double q) {  // q = t^2 where the derivative a + 3 b q + 5 d q^2 vanishes
    if (q > 0 && q < s * s && value(std::sqrt(q)) > top) top = value(std::sqrt(q));
  };
  if (d != 0) {
    const double disc = 9 * b * b - 20 * a * d;
    if (disc >= 0) {
      consider((-3 * b + std::sqrt(disc)) / (10 * d));
      consider((-3 * b - std::sqrt(disc)) / (10 * d));
    }
  } else if (b != 0) {
    consider(-a / (3 * b));
  }
  return top;
}

double ns_factor(const float* c, double s) {
  const double a = c[0], b = c[1], d = c[2], g = s * s;
  auto value = [&](double q) { return std::fabs(a + q * (b + q * d)); };
  double top = value(0) > value(g) ? value(0) : value(g);
  if (d != 0 && -b / (2 * d) > 0 && -b / (2 * d) < g && value(-b / (2 * d)) > top) top = value(-b / (2 * d));
  return top;
}

int64_t ns_bytes_per_matrix(int64_t rows, int64_t cols) {
  const int64_t m = rows < cols ? rows : cols;
  return up(rows * up(cols, 8) * 2, 256) * 3 + (up(m * up(m, 8) * 2, 256) + up(m, 32) * int64_t(sizeof(float4))) * 3;
}

void ns_carve(NsBatch* b, void* base) {
  b->m = b->rows < b->cols ? b->rows : b->cols;
  b->ld_x = up(b->cols, 8);
  b->ld_g = up(b->m, 8);
  b->plane_x = up(b->rows * b->ld_x * 2, 256) / 2;
  b->plane_g = up(b->m * b->ld_g * 2, 256) / 2;
  __half* p = static_cast<__half*>(base);
  b->hi[0] = p;
  b->hi[1] = b->hi[0] + b->n * b->plane_x;
  b->lo = b->hi[1] + b->n * b->plane_x;
  for (int i = 0; i < 3; ++i) b->square[i] = b->lo + b->n * b->plane_x + i * b->n * b->plane_g;
  b->m_pad = up(b->m, 32);
  float4* d = reinterpret_cast<float4*>(b->square[2] + b->n * b->plane_g);
  for (int i = 0; i < 3; ++i) b->diagonal[i] = d + i * b->n * b->m_pad;
}

int ns_stages(int steps) { return 3 * steps + 2; }

int ns_run(NsBatch* shapes, int n, const float* coef, int steps, cudaStream_t st) {
  int sms = 0;
  if (int rc = sm_count(&sms)) return rc;
  NsBatch* wide[kNsShapes];
  int count = 0;
  for (int i = 0; i < n; ++i) {
    if (narrow_fits(shapes[i].rows, shapes[i].cols, coef, steps)) {
      if (int rc = narrow_run(&shapes[i], coef, steps, sms, st)) return rc;
    } else {
      wide[count++] = &shapes[i];
    }
  }
  if (count == 0) return HA_OK;
  if (count == 1) return run<OneShape>(wide, 1, coef, steps, sms, st);
  return run<ManyShapes>(wide, count, coef, steps, sms, st);
}

}  // namespace ha
