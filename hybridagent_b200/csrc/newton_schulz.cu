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
// in five steps).  So the first kPreciseSteps steps keep X as a high and a low fp16 plane (22 bits):
// the products read the high plane only, and the epilogue adds a * (high + low) in fp32.  Later
// steps, where the spectrum is compressed, fold a into B's diagonal and read nothing more.
// Against 64-bit results (rank-16 plus 5 % noise, 1024 x 1024, rounded to bf16): 2.1e-3 relative,
// of which 1.7e-3 is the final rounding; one fp16 plane gives 2.1e-2, bf16 operands 1.6e-1.
//
// Kernel: persistent, one CTA per SM.  Warp 0 feeds a ring of 128-byte-swizzled operand tiles with
// TMA, one thread of warp 1 issues the MMAs, warps 2-5 read the accumulators from one of two TMEM
// buffers while the next tile is multiplied, and store 32 x 64 blocks by TMA, which clips the edges.
// Tall matrices (rows > cols) are not transposed: both operand layouts (K contiguous, or M/N
// contiguous) are read by the MMA as they lie.
#include <cuda.h>

#include "ha_common.cuh"
#include "newton_schulz.cuh"
#include "umma.cuh"

namespace ha {
namespace {

constexpr int kBM = 128;          // rows of a tile: the TMEM lanes of one CTA
constexpr int kBK = 64;           // K elements of a ring slot: one 128-byte swizzle row
constexpr int kGemmThreads = 192;  // producer warp, MMA warp, four epilogue warps
constexpr int kPreciseSteps = 3;

enum Epilogue { kGram, kPoly, kPrecise, kFolded };

struct GemmArgs {
  int M, N, K;                 // D is M x N
  int tiles_m, tiles_n, batch;
  float scale;                 // on the accumulator
  float add;                   // on the addend: b (kPoly), a (kPrecise)
  float diag;                  // added on the diagonal (kPoly)
  const __half* add_hi;        // kPoly: A; kPrecise: X high plane
  const __half* add_lo;        // kPrecise: X low plane
  int64_t add_ld, add_plane;
  uint32_t* error;
};

template <int BN>
struct Geometry {
  static constexpr int kTileA = kBM * kBK * 2;
  static constexpr int kTileB = BN * kBK * 2;
  static constexpr int kSlot = kTileA + kTileB;
  static constexpr int kSlots = BN == 256 ? 4 : 6;
  static constexpr int kStaging = 4 * 2 * 4096;  // four warps, two blocks of 32 x 64 fp16
  static constexpr int kSmem = kSlots * kSlot + kStaging + 1024;  // + alignment
  static constexpr int kColumns = 2 * BN;        // TMEM columns: two accumulators
};

__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float2 unpack_half2(uint32_t w) {
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}

// A_MN / B_MN: the operand's M / N index is the contiguous one in memory.
template <int BN, bool A_MN, bool B_MN, int EPI>
__global__ void __launch_bounds__(kGemmThreads, 1)
    ns_gemm_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                   const __grid_constant__ CUtensorMap map_hi, const __grid_constant__ CUtensorMap map_lo, GemmArgs p) {
  using G = Geometry<BN>;
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t bar_full[G::kSlots], bar_empty[G::kSlots], bar_acc_full[2], bar_acc_empty[2];
  __shared__ uint32_t tmem_base_s;
  __shared__ volatile uint32_t stop;
  const uint32_t ring = (smem_u32(smem_raw) + 1023) & ~1023u;
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    stop = 0;
    for (int i = 0; i < G::kSlots; ++i) {
      mbar_init(smem_u32(&bar_full[i]), 1);
      mbar_init(smem_u32(&bar_empty[i]), 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_u32(&bar_acc_full[i]), 1);
      mbar_init(smem_u32(&bar_acc_empty[i]), 4);
    }
    mbar_fence_init();
  }
  if (warp == 1) tmem_alloc(smem_u32(&tmem_base_s), G::kColumns);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_base_s;

  const int per_matrix = p.tiles_m * p.tiles_n;
  const int tiles = per_matrix * p.batch;
  const int kblocks = (p.K + kBK - 1) / kBK;

  if (warp == 0) {
    if (elect_one()) {
      tma_prefetch_map(&map_a);
      tma_prefetch_map(&map_b);
      int slot = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int t = blockIdx.x; t < tiles && ok; t += gridDim.x) {
        const int z = t / per_matrix, r = t - z * per_matrix;
        const int n0 = (r / p.tiles_m) * BN, m0 = (r % p.tiles_m) * kBM;
        for (int kb = 0; kb < kblocks; ++kb) {
          ok = mbar_wait(smem_u32(&bar_empty[slot]), phase ^ 1, &stop);
          if (!ok) break;
          const uint32_t full = smem_u32(&bar_full[slot]);
          const uint32_t a = ring + slot * G::kSlot, b = a + G::kTileA;
          mbar_expect_tx(full, G::kSlot);
          if (A_MN) {
#pragma unroll
            for (int j = 0; j < kBM / 64; ++j) tma_load_3d(a + j * 8192, &map_a, full, m0 + 64 * j, kb * kBK, z);
          } else {
            tma_load_3d(a, &map_a, full, kb * kBK, m0, z);
          }
          if (B_MN) {
#pragma unroll
            for (int j = 0; j < BN / 64; ++j) tma_load_3d(b + j * 8192, &map_b, full, n0 + 64 * j, kb * kBK, z);
          } else {
            tma_load_3d(b, &map_b, full, kb * kBK, n0, z);
          }
          if (++slot == G::kSlots) slot = 0, phase ^= 1;
        }
      }
    }
  } else if (warp == 1) {
    if (elect_one()) {
      constexpr uint32_t idesc = f16_idesc(kBM, BN, A_MN, B_MN);
      int slot = 0;
      uint32_t phase = 0, acc = 0, acc_phase = 0;
      bool ok = true;
      for (int t = blockIdx.x; t < tiles && ok; t += gridDim.x) {
        ok = mbar_wait(smem_u32(&bar_acc_empty[acc]), acc_phase ^ 1, &stop);
        if (!ok) break;
        tc_fence_after();
        const uint32_t d = tmem + acc * BN;
        for (int kb = 0; kb < kblocks; ++kb) {
          ok = mbar_wait(smem_u32(&bar_full[slot]), phase, &stop);
          if (!ok) break;
          tc_fence_after();
          const uint32_t a = ring + slot * G::kSlot, b = a + G::kTileA;
          const uint64_t da = smem_desc(a, A_MN ? 8192 : 16, 1024), db = smem_desc(b, B_MN ? 8192 : 16, 1024);
#pragma unroll
          for (int k = 0; k < kBK / 16; ++k)  // descriptor addresses count 16-byte units
            mma_f16(d, da + k * (A_MN ? 128 : 2), db + k * (B_MN ? 128 : 2), idesc, kb > 0 || k > 0);
          mma_commit(smem_u32(&bar_empty[slot]));
          if (++slot == G::kSlots) slot = 0, phase ^= 1;
        }
        if (ok) mma_commit(smem_u32(&bar_acc_full[acc]));
        if (++acc == 2) acc = 0, acc_phase ^= 1;
      }
    }
  } else {
    const int quarter = warp & 3;  // the TMEM lanes this warp may read: 32 * quarter ..
    const uint32_t staging = ring + G::kSlots * G::kSlot + quarter * 8192;
    uint32_t acc = 0, acc_phase = 0, block = 0;
    for (int t = blockIdx.x; t < tiles; t += gridDim.x) {
      const int z = t / per_matrix, r = t - z * per_matrix;
      const int n0 = (r / p.tiles_m) * BN, m0 = (r % p.tiles_m) * kBM;
      const int row0 = m0 + quarter * 32, row = row0 + lane;
      const bool ok = mbar_wait(smem_u32(&bar_acc_full[acc]), acc_phase, &stop);
      if (!__all_sync(0xffffffffu, ok)) break;
      tc_fence_after();
      const uint32_t d = tmem + acc * BN + (uint32_t(quarter * 32) << 16);
#pragma unroll 1
      for (int c0 = 0; c0 < BN; c0 += 64) {
        uint32_t hi[32], lo[32];  // 64 packed outputs
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t v[32];
          tmem_ld32(d + c0 + h * 32, v);
          uint4 ah[4] = {}, al[4] = {};  // the addend's 32 elements
          const int col = n0 + c0 + h * 32;
          if ((EPI == kPoly || EPI == kPrecise) && row < p.M) {
            const int64_t at = int64_t(z) * p.add_plane + int64_t(row) * p.add_ld + col;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              if (col + 8 * j < p.N) {
                ah[j] = *reinterpret_cast<const uint4*>(p.add_hi + at + 8 * j);
                if (EPI == kPrecise) al[j] = *reinterpret_cast<const uint4*>(p.add_lo + at + 8 * j);
              }
            }
          }
          tmem_ld_wait();
          const uint32_t* aw = reinterpret_cast<const uint32_t*>(ah);
          const uint32_t* lw = reinterpret_cast<const uint32_t*>(al);
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            float x = __uint_as_float(v[2 * j]) * p.scale, y = __uint_as_float(v[2 * j + 1]) * p.scale;
            if (EPI == kPoly) {
              const float2 g = unpack_half2(aw[j]);
              x = __fmaf_rn(p.add, g.x, x);
              y = __fmaf_rn(p.add, g.y, y);
              if (col + 2 * j == row) x += p.diag;
              if (col + 2 * j + 1 == row) y += p.diag;
            }
            if (EPI == kPrecise) {
              const float2 g = unpack_half2(aw[j]), l = unpack_half2(lw[j]);
              x = __fmaf_rn(p.add, __fmaf_rn(l.x, 1.0f / kScaleLo, g.x), x);
              y = __fmaf_rn(p.add, __fmaf_rn(l.y, 1.0f / kScaleLo, g.y), y);
            }
            hi[h * 16 + j] = pack_half2(x, y);
            if (EPI == kPrecise) {
              const float2 g = unpack_half2(hi[h * 16 + j]);
              lo[h * 16 + j] = pack_half2((x - g.x) * kScaleLo, (y - g.y) * kScaleLo);
            }
          }
        }
        // 32 rows of 128 bytes, 16-byte pieces swizzled by the row as the tensor map expects
        const bool inside = row0 < p.M && n0 + c0 < p.N;  // (uniform in the warp)
#pragma unroll
        for (int plane = 0; plane < (EPI == kPrecise ? 2 : 1); ++plane) {
          const uint32_t buf = staging + (block & 1) * 4096;
          if (lane == 0) tma_store_wait_read<1>();  // the store before last has read this block
          __syncwarp();
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const uint32_t* w = (plane == 0 ? hi : lo) + 4 * j;
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(buf + lane * 128 + ((j ^ (lane & 7)) << 4)),
                         "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3])
                         : "memory");
          }
          fence_async_smem();
          __syncwarp();
          if (lane == 0) {
            if (inside) tma_store_3d(plane == 0 ? &map_hi : &map_lo, buf, n0 + c0, row0, z);
            tma_store_commit();
          }
          ++block;
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&bar_acc_empty[acc]));
      if (++acc == 2) acc = 0, acc_phase ^= 1;
    }
    if (lane == 0) tma_store_wait_all();
  }
  __syncthreads();
  if (stop) {  // a wait ran out: let copies and products in flight end before their memory is given up
    if (threadIdx.x == 0) atomicExch(p.error, 1u);
    const uint64_t t0 = global_ns();
    while (global_ns() - t0 < 2000000) {
    }
    __syncthreads();
  }
  tc_fence_after();
  if (warp == 1) tmem_dealloc(tmem, G::kColumns);
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

// `n` matrices of rows x cols fp16 elements, rows `ld` apart, read or written in box_cols x box_rows
// pieces with the 128-byte swizzle.
int make_map(CUtensorMap* map, const __half* base, int64_t n, int64_t rows, int64_t cols, int64_t ld, int64_t plane,
             int box_cols, int box_rows) {
  const EncodeTiled fn = encode_tiled();
  if (fn == nullptr) return fail(HA_ERR_CUDA, "cuTensorMapEncodeTiled is not available");
  const cuuint64_t dims[3] = {cuuint64_t(cols), cuuint64_t(rows), cuuint64_t(n)};
  const cuuint64_t strides[2] = {cuuint64_t(ld) * 2, cuuint64_t(plane) * 2};
  const cuuint32_t box[3] = {cuuint32_t(box_cols), cuuint32_t(box_rows), 1};
  const cuuint32_t step[3] = {1, 1, 1};
  const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<__half*>(base), dims, strides, box, step,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS)
    return fail(HA_ERR_CUDA, "cuTensorMapEncodeTiled: error %d for %lld x %lld x %lld", int(r), (long long)n,
                (long long)rows, (long long)cols);
  return HA_OK;
}

struct Operand {
  const __half* base;
  int64_t rows, cols, ld, plane;
};

template <int BN, bool A_MN, bool B_MN, int EPI>
int launch(const Operand& a, const Operand& b, const Operand& out, const __half* out_lo, GemmArgs p, int sms,
           cudaStream_t st) {
  using G = Geometry<BN>;
  CUtensorMap ma, mb, mh, ml;
  int rc = make_map(&ma, a.base, p.batch, a.rows, a.cols, a.ld, a.plane, 64, A_MN ? 64 : kBM);
  if (rc == HA_OK) rc = make_map(&mb, b.base, p.batch, b.rows, b.cols, b.ld, b.plane, 64, B_MN ? 64 : BN);
  if (rc == HA_OK) rc = make_map(&mh, out.base, p.batch, out.rows, out.cols, out.ld, out.plane, 64, 32);
  if (rc == HA_OK)
    rc = make_map(&ml, out_lo != nullptr ? out_lo : out.base, p.batch, out.rows, out.cols, out.ld, out.plane, 64, 32);
  if (rc != HA_OK) return rc;
  p.tiles_m = (p.M + kBM - 1) / kBM;
  p.tiles_n = (p.N + BN - 1) / BN;
  const int64_t tiles = int64_t(p.tiles_m) * p.tiles_n * p.batch;
  if (tiles > 0x3fffffff) return fail(HA_ERR_INVALID, "Newton-Schulz product of %lld tiles", (long long)tiles);
  auto* kernel = ns_gemm_kernel<BN, A_MN, B_MN, EPI>;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, G::kSmem) != cudaSuccess)
    return check_launch("ns_gemm_kernel (shared memory)");
  const unsigned grid = unsigned(tiles < sms ? tiles : sms);
  kernel<<<grid, kGemmThreads, G::kSmem, st>>>(ma, mb, mh, ml, p);
  return check_launch("ns_gemm_kernel");
}

int sm_count(int* out) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess ||
      cudaDeviceGetAttribute(out, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
    return check_launch("ns_run (device query)");
  return HA_OK;
}

template <int BN>
int run_steps(const NsBatch& b, const float* coef, int steps, int* out, int sms, cudaStream_t st) {
  const bool tall = b.rows > b.cols;
  const int m = int(b.m), n = int(tall ? b.rows : b.cols);
  const Operand gram{b.gram, b.m, b.m, b.ld_g, b.plane_g}, poly{b.poly, b.m, b.m, b.ld_g, b.plane_g};
  int cur = 0;
  for (int s = 0; s < steps; ++s) {
    const float ca = coef[3 * s], cb = coef[3 * s + 1], cc = coef[3 * s + 2];
    const bool precise = s < kPreciseSteps;
    const Operand x{b.hi[cur], b.rows, b.cols, b.ld_x, b.plane_x};
    const Operand y{b.hi[cur ^ 1], b.rows, b.cols, b.ld_x, b.plane_x};
    GemmArgs g{};
    g.batch = int(b.n);
    g.error = b.error;
    g.M = g.N = m;
    g.K = n;
    g.scale = kScaleG / (kScaleX * kScaleX);
    int rc = tall ? launch<BN, true, true, kGram>(x, x, gram, nullptr, g, sms, st)
                  : launch<BN, false, false, kGram>(x, x, gram, nullptr, g, sms, st);
    if (rc != HA_OK) return rc;
    g.K = m;
    g.scale = cc / kScaleG;
    g.add = cb;
    g.diag = precise ? 0.0f : ca * kScaleG;
    g.add_hi = b.gram;
    g.add_ld = b.ld_g;
    g.add_plane = b.plane_g;
    rc = launch<BN, false, false, kPoly>(gram, gram, poly, nullptr, g, sms, st);
    if (rc != HA_OK) return rc;
    g.M = int(b.rows);
    g.N = int(b.cols);
    g.K = m;
    g.scale = 1.0f / kScaleG;
    g.add = ca;
    g.diag = 0.0f;
    g.add_hi = b.hi[cur];
    g.add_lo = b.lo;
    g.add_ld = b.ld_x;
    g.add_plane = b.plane_x;
    if (precise)  // the low plane is read and rewritten in place, each element by one thread
      rc = tall ? launch<BN, false, false, kPrecise>(x, poly, y, b.lo, g, sms, st)
                : launch<BN, false, true, kPrecise>(poly, x, y, b.lo, g, sms, st);
    else
      rc = tall ? launch<BN, false, false, kFolded>(x, poly, y, nullptr, g, sms, st)
                : launch<BN, false, true, kFolded>(poly, x, y, nullptr, g, sms, st);
    if (rc != HA_OK) return rc;
    cur ^= 1;
  }
  *out = cur;
  return HA_OK;
}

int64_t up(int64_t x, int64_t a) { return (x + a - 1) / a * a; }

}  // namespace

int64_t ns_bytes_per_matrix(int64_t rows, int64_t cols) {
  const int64_t m = rows < cols ? rows : cols;
  return up(rows * up(cols, 8) * 2, 256) * 3 + up(m * up(m, 8) * 2, 256) * 2;
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
  b->gram = b->lo + b->n * b->plane_x;
  b->poly = b->gram + b->n * b->plane_g;
}

int ns_run(const NsBatch& b, const float* coef, int steps, int* out, cudaStream_t st) {
  int sms = 0;
  if (int rc = sm_count(&sms)) return rc;
  return run_steps<256>(b, coef, steps, out, sms, st);
}

}  // namespace ha
