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
// in five steps).  So the first kPreciseSteps steps keep X as a high and a low fp16 plane (22 bits).
// The products read the high plane only: with a on B's diagonal a step is (a I + B) X, and its
// epilogue adds a * low in fp32 (what B does to the low plane touches only the few leading
// directions).  Against 64-bit results (rank-16 plus 5 % noise, 1024 x 1024, rounded to bf16): 2.2e-3
// relative, of which 1.7e-3 is the final rounding; one fp16 plane gives 2.1e-2, bf16 operands 1.6e-1.
//
// Two steps can run as one product with X: with Q1 = a I + b G + c G^2 (G = X X^T), the Gram matrix
// after the step is G' = Q1 G Q1 (all three commute), Q2 follows from G', and X <- (Q2 Q1) X.  That
// replaces two products with X (6 m^2 n of 2 (3 m^2 n + m^3)) by one and three more symmetric ones:
// 3 m^2 n + 5 m^3.  See pairs() for where that is done and what it costs in accuracy.
//
// Kernel: persistent, one CTA per SM, one or two CTAs to a tile.  Warp 0 feeds a ring of 128-byte-swizzled operand tiles with
// TMA, one thread of warp 1 issues the MMAs, warps 2-5 read the accumulators from one of two TMEM
// buffers while the next tile is multiplied, and store 32 x 64 blocks by TMA, which clips the edges.
// Tall matrices (rows > cols) are not transposed: both operand layouts (K contiguous, or M/N
// contiguous) are read by the MMA as they lie.
#include <cuda.h>

#include <cmath>

#include "ha_common.cuh"
#include "newton_schulz.cuh"
#include "umma.cuh"

namespace ha {
namespace {

constexpr int kBM = 128;          // rows of a CTA's part of a tile: the TMEM lanes
constexpr int kBK = 64;           // K elements of a ring slot: one 128-byte swizzle row
constexpr int kGemmThreads = 192;  // producer warp, MMA warp, four epilogue warps
constexpr int kPreciseSteps = 3;
constexpr int kHalf = kBM * kBK * 2;      // bytes of one operand's part of a slot
constexpr int kSlot = 2 * kHalf;
constexpr int kBlock = 32 * 64 * 2;       // bytes of an epilogue block: 32 rows of 64 columns

// What becomes of the accumulators (times `scale`):
//   kSymmetric  stored, with the mirrored tile (D is symmetric; tiles on and below the diagonal run)
//   kPoly       the same after adding add * addend and `diag` on the diagonal
//   kPrecise    added to add * low / 2^11, stored as high and low plane
//   kPlain      stored
enum Epilogue { kSymmetric, kPoly, kPrecise, kPlain };

template <int EPI>
struct Layout {
  static constexpr bool kSym = EPI == kSymmetric || EPI == kPoly;
  static constexpr bool kAdd = EPI == kPoly || EPI == kPrecise;   // reads an addend by TMA, two blocks ahead
  static constexpr int kBlocks = kAdd ? 3 : (kSym ? 1 : 2);       // a warp's blocks, addend in, result out
  static constexpr int kSecond = EPI == kPlain ? 0 : 1;           // block of the mirrored tile or second plane
  static constexpr int kSlots = kAdd ? 5 : 6;
  static constexpr int kWarp = (kBlocks + kSecond) * kBlock;
  static constexpr int kSmem = kSlots * kSlot + 4 * kWarp + 1024;  // + alignment
};

struct GemmArgs {
  int M, N, K;                 // D is M x N
  int tiles_m, tiles_n;
  int per_matrix;              // tiles of one matrix (symmetric: those on and below the diagonal)
  int tiles;
  int m_fast;                  // consecutive tiles go down the rows
  float scale;                 // on the accumulator
  float add;                   // on the addend
  float diag;                  // added on the diagonal (kPoly)
  uint32_t* error;
};

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
// SYM: the tiles on and below the diagonal, row by row.
template <bool SYM>
__device__ __forceinline__ TileAt tile_at(const GemmArgs& p, int t) {
  TileAt a;
  a.z = t / p.per_matrix;
  const int r = t - a.z * p.per_matrix;
  if (SYM) {
    int i = int((sqrtf(8.0f * float(r) + 1.0f) - 1.0f) * 0.5f);
    while (i * (i + 1) / 2 > r) --i;
    while ((i + 1) * (i + 2) / 2 <= r) ++i;
    a.i = i;
    a.j = r - i * (i + 1) / 2;
  } else if (p.m_fast) {
    a.j = r / p.tiles_m;
    a.i = r - a.j * p.tiles_m;
  } else {
    a.i = r / p.tiles_n;
    a.j = r - a.i * p.tiles_n;
  }
  return a;
}

// The blocks of 32 x 64 outputs that an epilogue warp works, tile by tile; blocks outside D are left out.
template <int CG, bool SYM>
struct BlockCursor {
  int t, c0;       // tile, column in the tile
  int i, j, z;     // of tile t
  int row0;        // first row of the warp's blocks
  __device__ __forceinline__ void enter(const GemmArgs& p, int warp_row, int step) {
    for (; t < p.tiles; t += step) {
      const TileAt at = tile_at<SYM>(p, t);
      i = at.i, j = at.j, z = at.z;
      row0 = i * (128 * CG) + warp_row;
      if (row0 < p.M) break;
    }
    c0 = 0;
  }
  __device__ __forceinline__ int col0() const { return j * (128 * CG) + c0; }
  // Whether the next block belongs to another tile.
  __device__ __forceinline__ bool last(const GemmArgs& p) const {
    return c0 + 64 >= 128 * CG || col0() + 64 >= p.N;
  }
  __device__ __forceinline__ void next(const GemmArgs& p, int warp_row, int step) {
    if (last(p)) {
      t += step;
      enter(p, warp_row, step);
    } else {
      c0 += 64;
    }
  }
};

// A_MN / B_MN: the operand's M / N index is the contiguous one in memory.  CG: CTAs of a tile
// (1: 128 x 128; 2: 256 x 256, each CTA with 128 rows of A and of D and 128 columns of B).
template <int CG, bool A_MN, bool B_MN, int EPI>
__global__ void __launch_bounds__(kGemmThreads, 1)
    ns_gemm_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                   const __grid_constant__ CUtensorMap map_out, const __grid_constant__ CUtensorMap map_2,
                   const __grid_constant__ CUtensorMap map_add, GemmArgs p) {
  using L = Layout<EPI>;
  constexpr bool kSym = L::kSym;
  constexpr int kSlots = L::kSlots;
  constexpr int kTile = 128 * CG;         // rows and columns of a tile
  constexpr int kColumns = 2 * kTile;     // TMEM columns: two accumulators
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t bar_full[kSlots], bar_empty[kSlots], bar_acc_full[2], bar_acc_empty[2];
  __shared__ __align__(8) uint64_t bar_add[4][3];
  __shared__ uint32_t tmem_base_s;
  __shared__ volatile uint32_t stop;
  const uint32_t ring = (smem_u32(smem_raw) + 1023) & ~1023u;
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const uint32_t rank = CG == 2 ? cluster_rank() : 0;

  grid_launch_dependents();
  if (threadIdx.x == 0) {
    stop = 0;
    for (int i = 0; i < kSlots; ++i) {
      mbar_init(smem_u32(&bar_full[i]), 1);
      mbar_init(smem_u32(&bar_empty[i]), 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_u32(&bar_acc_full[i]), 1);
      mbar_init(smem_u32(&bar_acc_empty[i]), 4 * CG);
    }
    for (int i = 0; i < 12; ++i) mbar_init(smem_u32(&bar_add[i / 3][i % 3]), 1);
    mbar_fence_init();
    tma_prefetch_map(&map_a);
    tma_prefetch_map(&map_b);
    tma_prefetch_map(&map_out);
    if (L::kSecond) tma_prefetch_map(&map_2);
    if (L::kAdd) tma_prefetch_map(&map_add);
  }
  if (warp == 1) tmem_alloc<CG>(smem_u32(&tmem_base_s), kColumns);
  tc_fence_before();
  if (CG == 2)
    cluster_sync();  // the pair's barriers exist before either CTA signals the other's
  else
    __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_base_s;
  grid_wait();

  const int kblocks = (p.K + kBK - 1) / kBK;
  const int first = blockIdx.x / CG, step = gridDim.x / CG;

  if (warp == 0) {
    if (elect_one()) {
      int slot = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int t = first; t < p.tiles && ok; t += step) {
        const TileAt at = tile_at<kSym>(p, t);
        const int m0 = at.i * kTile + int(rank) * kBM, n0 = at.j * kTile + int(rank) * 128;
        for (int kb = 0; kb < kblocks; ++kb) {
          ok = mbar_wait(smem_u32(&bar_empty[slot]), phase ^ 1, &stop);
          if (!ok) break;
          uint32_t full = smem_u32(&bar_full[slot]);
          const uint32_t a = ring + slot * kSlot, b = a + kHalf;
          if (rank == 0) mbar_expect_tx(full, CG * kSlot);  // the first CTA's barrier counts both halves
          if (CG == 2) full = cluster_map(full, 0);
          if (A_MN) {
            tma_load_3d<CG>(a, &map_a, full, m0, kb * kBK, at.z);
            tma_load_3d<CG>(a + 8192, &map_a, full, m0 + 64, kb * kBK, at.z);
          } else {
            tma_load_3d<CG>(a, &map_a, full, kb * kBK, m0, at.z);
          }
          if (B_MN) {
            tma_load_3d<CG>(b, &map_b, full, n0, kb * kBK, at.z);
            tma_load_3d<CG>(b + 8192, &map_b, full, n0 + 64, kb * kBK, at.z);
          } else {
            tma_load_3d<CG>(b, &map_b, full, kb * kBK, n0, at.z);
          }
          if (++slot == kSlots) slot = 0, phase ^= 1;
        }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    if (rank == 0 && elect_one()) {
      constexpr uint32_t idesc = f16_idesc(kTile, kTile, A_MN, B_MN);
      int slot = 0;
      uint32_t phase = 0, acc = 0, acc_phase = 0;
      bool ok = true;
      for (int t = first; t < p.tiles && ok; t += step) {
        ok = mbar_wait(smem_u32(&bar_acc_empty[acc]), acc_phase ^ 1, &stop);
        if (!ok) break;
        tc_fence_after();
        const uint32_t d = tmem + acc * kTile;
        for (int kb = 0; kb < kblocks; ++kb) {
          ok = mbar_wait(smem_u32(&bar_full[slot]), phase, &stop);
          if (!ok) break;
          tc_fence_after();
          const uint32_t a = ring + slot * kSlot, b = a + kHalf;
          const uint64_t da = smem_desc(a, A_MN ? 8192 : 16, 1024), db = smem_desc(b, B_MN ? 8192 : 16, 1024);
#pragma unroll
          for (int k = 0; k < kBK / 16; ++k)  // descriptor addresses count 16-byte units
            mma_f16<CG>(d, da + k * (A_MN ? 128 : 2), db + k * (B_MN ? 128 : 2), idesc, kb > 0 || k > 0);
          mma_commit<CG>(smem_u32(&bar_empty[slot]));
          if (++slot == kSlots) slot = 0, phase ^= 1;
        }
        if (ok) mma_commit<CG>(smem_u32(&bar_acc_full[acc]));
        if (++acc == 2) acc = 0, acc_phase ^= 1;
      }
    }
    __syncwarp();
  } else {
    const int quarter = warp & 3;  // the TMEM lanes this warp may read: 32 * quarter ..
    const int warp_row = int(rank) * kBM + quarter * 32;
    const uint32_t blocks = ring + kSlots * kSlot + quarter * L::kWarp, second = blocks + L::kBlocks * kBlock;
    const uint32_t swizzled = lane * 128;  // this lane's row; its 16-byte piece j lies at j ^ (lane & 7)
    BlockCursor<CG, kSym> now{first}, ahead{first};
    now.enter(p, warp_row, step);
    ahead = now;
    uint32_t use = 0, use_phase = 0, fetch = 0;  // block of `now`, its barrier's phase, block of `ahead`
    auto fetch_addend = [&]() {  // by lane 0; the block's last store has been read
      if (ahead.t < p.tiles) {
        const uint32_t bar = smem_u32(&bar_add[quarter][fetch]);
        mbar_expect_tx(bar, kBlock);
        tma_load_3d<1>(blocks + fetch * kBlock, &map_add, bar, ahead.col0(), ahead.row0, ahead.z);
        ahead.next(p, warp_row, step);
      }
      if (++fetch == 3) fetch = 0;
    };
    if (L::kAdd && lane == 0) {
      fetch_addend();
      fetch_addend();
    }
    uint32_t acc = 0, acc_phase = 0;
    for (int t = first; t < p.tiles; t += step) {
      bool ok = mbar_wait(smem_u32(&bar_acc_full[acc]), acc_phase, &stop);
      if (!__all_sync(0xffffffffu, ok)) break;
      tc_fence_after();
      const uint32_t d = tmem + acc * kTile + (uint32_t(quarter * 32) << 16);
      while (now.t == t) {
        const int col0 = now.col0(), row0 = now.row0, row = row0 + lane;
        const bool last = now.last(p);
        const uint32_t block = blocks + use * kBlock;
        uint32_t v[2][32];
        tmem_ld32(d + now.c0, v[0]);
        tmem_ld32(d + now.c0 + 32, v[1]);
        uint32_t add[32];  // 64 packed addends
        if (L::kAdd) {
          ok = mbar_wait(smem_u32(&bar_add[quarter][use]), use_phase, &stop);
          if (!__all_sync(0xffffffffu, ok)) break;
#pragma unroll
          for (int j = 0; j < 8; ++j)
            asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                         : "=r"(add[4 * j]), "=r"(add[4 * j + 1]), "=r"(add[4 * j + 2]), "=r"(add[4 * j + 3])
                         : "r"(block + swizzled + ((j ^ (lane & 7)) << 4))
                         : "memory");
        }
        tmem_ld_wait();
        uint32_t out[32], low[32];  // 64 packed results
#pragma unroll
        for (int j = 0; j < 32; ++j) {
          float x = __uint_as_float(v[j / 16][2 * (j % 16)]) * p.scale;
          float y = __uint_as_float(v[j / 16][2 * (j % 16) + 1]) * p.scale;
          if (L::kAdd) {
            const float2 g = unpack_half2(add[j]);
            x = __fmaf_rn(p.add, g.x, x);
            y = __fmaf_rn(p.add, g.y, y);
          }
          if (EPI == kPoly) {
            if (col0 + 2 * j == row) x += p.diag;
            if (col0 + 2 * j + 1 == row) y += p.diag;
          }
          out[j] = pack_half2(x, y);
          if (EPI == kPrecise) {
            const float2 g = unpack_half2(out[j]);
            low[j] = pack_half2((x - g.x) * kScaleLo, (y - g.y) * kScaleLo);
          }
        }
        // Earlier stores of this warp have been read, so every block but this one is free: fetch two ahead.
        if (lane == 0) {
          tma_store_wait_read<L::kSecond ? 0 : 1>();
          if (L::kAdd) fetch_addend();
        }
        __syncwarp();
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const uint32_t* w = (EPI == kPrecise ? low : out) + 4 * j;
          asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(block + swizzled + ((j ^ (lane & 7)) << 4)),
                       "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3])
                       : "memory");
        }
        if (EPI == kPrecise) {
#pragma unroll
          for (int j = 0; j < 8; ++j)
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(second + swizzled + ((j ^ (lane & 7)) << 4)),
                         "r"(out[4 * j]), "r"(out[4 * j + 1]), "r"(out[4 * j + 2]), "r"(out[4 * j + 3])
                         : "memory");
        }
        if (kSym && now.i != now.j) {
          // the transposed block, 64 rows of 32: lanes 2l and 2l + 1 exchange halves so that each writes
          // two neighbours of one row
#pragma unroll
          for (int j = 0; j < 32; ++j) {
            const uint32_t other = __shfl_xor_sync(0xffffffffu, out[j], 1);
            const uint32_t w = (lane & 1) ? __byte_perm(other, out[j], 0x7632) : __byte_perm(out[j], other, 0x5410);
            asm volatile("st.shared.b32 [%0], %1;" ::"r"(second + (2 * j + (lane & 1)) * 64 + (lane >> 1) * 4), "r"(w)
                         : "memory");
          }
        }
        fence_async_smem();
        __syncwarp();
        if (lane == 0) {
          if (EPI == kPrecise) {
            tma_store_3d(&map_2, block, col0, row0, now.z);
            tma_store_3d(&map_out, second, col0, row0, now.z);
          } else {
            tma_store_3d(&map_out, block, col0, row0, now.z);
            if (kSym && now.i != now.j) tma_store_3d(&map_2, second, row0, col0, now.z);
          }
          tma_store_commit();
        }
        if (++use == L::kBlocks) use = 0, use_phase ^= 1;
        now.next(p, warp_row, step);
        if (last) break;
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        const uint32_t bar = smem_u32(&bar_acc_empty[acc]);
        if (CG == 2)
          mbar_arrive_cluster(cluster_map(bar, 0));
        else
          mbar_arrive(bar);
      }
      if (++acc == 2) acc = 0, acc_phase ^= 1;
    }
    if (lane == 0) tma_store_wait_all();
    __syncwarp();
  }
  __syncthreads();
  if (stop) {  // a wait ran out: let copies and products in flight end before their memory is given up
    if (threadIdx.x == 0) atomicExch(p.error, 1u);
    const uint64_t t0 = global_ns();
    while (global_ns() - t0 < 2000000) {
    }
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

// `n` of them, read or written in box_cols x box_rows pieces (128-byte rows swizzled).
int make_map(CUtensorMap* map, const Operand& x, int64_t n, int box_cols, int box_rows) {
  const EncodeTiled fn = encode_tiled();
  if (fn == nullptr) return fail(HA_ERR_CUDA, "cuTensorMapEncodeTiled is not available");
  const cuuint64_t dims[3] = {cuuint64_t(x.cols), cuuint64_t(x.rows), cuuint64_t(n)};
  const cuuint64_t strides[2] = {cuuint64_t(x.ld) * 2, cuuint64_t(x.plane) * 2};
  const cuuint32_t box[3] = {cuuint32_t(box_cols), cuuint32_t(box_rows), 1};
  const cuuint32_t step[3] = {1, 1, 1};
  const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<__half*>(x.base), dims, strides, box, step,
                        CU_TENSOR_MAP_INTERLEAVE_NONE,
                        box_cols == 64 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_NONE,
                        CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS)
    return fail(HA_ERR_CUDA, "cuTensorMapEncodeTiled: error %d for %lld x %lld x %lld", int(r), (long long)n,
                (long long)x.rows, (long long)x.cols);
  return HA_OK;
}

int64_t tiles_of(const GemmArgs& p, int64_t tile, bool symmetric) {
  const int64_t m = (p.M + tile - 1) / tile, n = (p.N + tile - 1) / tile;
  return symmetric ? m * (m + 1) / 2 : m * n;
}

// addend: G (kPoly), or the low plane, which kPrecise also rewrites in place, block by block.
template <int CG, bool A_MN, bool B_MN, int EPI>
int launch(const Operand& a, const Operand& b, const Operand& out, const Operand& addend, GemmArgs p, int64_t batch,
           int sms, cudaStream_t st) {
  using L = Layout<EPI>;
  constexpr bool kSym = L::kSym;
  constexpr int kTile = 128 * CG;
  CUtensorMap ma, mb, mo, m2, mx;
  int rc = make_map(&ma, a, batch, 64, A_MN ? 64 : kBM);
  if (rc == HA_OK) rc = make_map(&mb, b, batch, 64, B_MN ? 64 : 128);
  if (rc == HA_OK) rc = make_map(&mo, out, batch, 64, 32);
  if (rc == HA_OK && kSym) rc = make_map(&m2, out, batch, 32, 64);  // mirrored blocks
  if (rc == HA_OK && L::kAdd) rc = make_map(&mx, addend, batch, 64, 32);
  if (rc != HA_OK) return rc;
  if (!kSym) m2 = EPI == kPrecise ? mx : mo;
  if (!L::kAdd) mx = mo;
  p.tiles_m = (p.M + kTile - 1) / kTile;
  p.tiles_n = (p.N + kTile - 1) / kTile;
  const int64_t per = tiles_of(p, kTile, kSym);
  if (per * batch > 0x3fffffff) return fail(HA_ERR_INVALID, "Newton-Schulz product of %lld tiles", (long long)(per * batch));
  p.per_matrix = int(per);
  p.tiles = int(per * batch);
  p.m_fast = p.tiles_m <= p.tiles_n;  // the shorter side first: its operand panels stay in L2
  auto* kernel = ns_gemm_kernel<CG, A_MN, B_MN, EPI>;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kSmem) != cudaSuccess)
    return check_launch("ns_gemm_kernel (shared memory)");
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(unsigned(p.tiles < sms / CG ? p.tiles : sms / CG) * CG);
  cfg.blockDim = dim3(kGemmThreads);
  cfg.dynamicSmemBytes = L::kSmem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = CG;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  if (cudaLaunchKernelEx(&cfg, kernel, ma, mb, mo, m2, mx, p) != cudaSuccess) return check_launch("ns_gemm_kernel");
  return HA_OK;
}

// Picks the tile.  A 256 x 256 tile on a CTA pair reads half the operand bytes per product of a 128 x 128
// tile on one CTA and runs 1.35 times as fast where both fill the chip (2.75 against 3.70 ms for five
// steps of 4096 x 12288), but leaves SMs idle when there are few tiles and pads more.  An SM works
// two 128 x 128 units for each of its pair's tiles, so the rule compares rounds of work.
template <bool A_MN, bool B_MN, int EPI>
int product(const Operand& a, const Operand& b, const Operand& out, const Operand& addend, const GemmArgs& p,
            int64_t batch, int sms, cudaStream_t st) {
  constexpr bool kSym = Layout<EPI>::kSym;
  const int64_t one = (tiles_of(p, 128, kSym) * batch + sms - 1) / sms;
  const int64_t two = (tiles_of(p, 256, kSym) * batch + sms / 2 - 1) / (sms / 2);
  if (1.35 * double(one) <= 2.0 * double(two)) return launch<1, A_MN, B_MN, EPI>(a, b, out, addend, p, batch, sms, st);
  return launch<2, A_MN, B_MN, EPI>(a, b, out, addend, p, batch, sms, st);
}

int sm_count(int* out) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess ||
      cudaDeviceGetAttribute(out, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
    return check_launch("ns_run (device query)");
  return HA_OK;
}

// How many of the leading pairs of steps, (0, 1) and (2, 3), run as one product with X.  Each saves
// 3 m^2 (n - m) multiply-adds and costs a launch.  Relative error against 64-bit results (CPU model
// of these roundings, rounded to bf16; none / first / both): 1024 x 4096 normal 1.85 / 1.86 / 2.15e-3,
// 512 x 1536 2.16 / 2.18 / 2.57e-3, rank 16 plus 5 % noise 1024 x 4096 2.18 / 2.21 / 2.36e-3: the first
// pair costs nothing, the second little where m is large.
int pairs(int64_t m, int64_t n, const float* coef, int steps) {
  int count = 0;
  double top = 1.0;  // bound of the singular values before step s
  for (int s = 0; s + 2 <= steps && s < 4; s += 2) {
    const bool worth = s == 0 ? n * 2 >= m * 3 && m >= 256 : n >= m * 2 && m >= 640;
    const double between = ns_growth(coef + 3 * s, top);
    // both factors' product has to fit the planes like each of them
    if (!worth || ns_factor(coef + 3 * s, top) * ns_factor(coef + 3 * s + 3, between) > kMaxFactor) break;
    top = ns_growth(coef + 3 * s + 3, between);
    ++count;
  }
  return count;
}

int run_steps(const NsBatch& b, const float* coef, int steps, int* out, int sms, cudaStream_t st) {
  const bool tall = b.rows > b.cols;
  const int m = int(b.m), n = int(tall ? b.rows : b.cols);
  auto square = [&](int i) { return Operand{b.square[i], b.m, b.m, b.ld_g, b.plane_g}; };
  const Operand lo{b.lo, b.rows, b.cols, b.ld_x, b.plane_x};
  GemmArgs sym{};  // a symmetric m x m product of m x m matrices
  sym.error = b.error;
  sym.M = sym.N = sym.K = m;
  sym.scale = 1.0f / kScaleG;
  auto multiply = [&](int x, int y, int to) {  // of commuting symmetric matrices
    return product<false, false, kSymmetric>(square(x), square(y), square(to), square(to), sym, b.n, sms, st);
  };
  auto factor = [&](int gram, int to, const float* c) {  // c0 I + c1 G + c2 G G
    GemmArgs g = sym;
    g.scale = c[2] / kScaleG;
    g.add = c[1];
    g.diag = c[0] * kScaleG;
    return product<false, false, kPoly>(square(gram), square(gram), square(to), square(gram), g, b.n, sms, st);
  };
  const int merged = pairs(m, n, coef, steps);
  int cur = 0;
  for (int s = 0; s < steps;) {
    const bool pair = s < 2 * merged;
    const float* c = coef + 3 * s;
    const Operand x{b.hi[cur], b.rows, b.cols, b.ld_x, b.plane_x};
    const Operand y{b.hi[cur ^ 1], b.rows, b.cols, b.ld_x, b.plane_x};
    GemmArgs g = sym;
    g.K = n;
    g.scale = kScaleG / (kScaleX * kScaleX);
    int rc = tall ? product<true, true, kSymmetric>(x, x, square(0), square(0), g, b.n, sms, st)
                  : product<false, false, kSymmetric>(x, x, square(0), square(0), g, b.n, sms, st);
    if (rc == HA_OK) rc = factor(0, 1, c);
    if (pair) {
      if (rc == HA_OK) rc = multiply(0, 1, 2);
      if (rc == HA_OK) rc = multiply(2, 1, 0);  // G' = G Q1 Q1
      if (rc == HA_OK) rc = factor(0, 2, c + 3);
      if (rc == HA_OK) rc = multiply(2, 1, 0);  // Q2 Q1
    }
    if (rc != HA_OK) return rc;
    const Operand q = square(pair ? 0 : 1);
    g.M = int(b.rows);
    g.N = int(b.cols);
    g.K = m;
    g.scale = 1.0f / kScaleG;
    g.add = (pair ? c[0] * c[3] : c[0]) / kScaleLo;
    if (s < kPreciseSteps)
      rc = tall ? product<false, false, kPrecise>(x, q, y, lo, g, b.n, sms, st)
                : product<false, true, kPrecise>(q, x, y, lo, g, b.n, sms, st);
    else
      rc = tall ? product<false, false, kPlain>(x, q, y, lo, g, b.n, sms, st)
                : product<false, true, kPlain>(q, x, y, lo, g, b.n, sms, st);
    if (rc != HA_OK) return rc;
    cur ^= 1;
    s += pair ? 2 : 1;
  }
  *out = cur;
  return HA_OK;
}

int64_t up(int64_t x, int64_t a) { return (x + a - 1) / a * a; }

}  // namespace

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
  return up(rows * up(cols, 8) * 2, 256) * 3 + up(m * up(m, 8) * 2, 256) * 3;
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
}

int ns_run(const NsBatch& b, const float* coef, int steps, int* out, cudaStream_t st) {
  int sms = 0;
  if (int rc = sm_count(&sms)) return rc;
  return run_steps(b, coef, steps, out, sms, st);
}

}  // namespace ha
