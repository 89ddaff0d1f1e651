// Newton-Schulz orthogonalisation of matrices whose shorter side is at most 128 (sm_100a).
//
// Routers, adapters and heads are a few rows by thousands of columns.  Their steps are too small to
// spread over the chip (a stage of the general kernel takes 3 us for next to no arithmetic), so the whole
// iteration runs inside one CTA, on the m x m side alone.  With G = X X^T and every
// factor Q = a I + b G + c G^2 a polynomial in G,
//     S <- Q S,   G <- Q G Q   (a few steps),   X <- S X,
// and X is read once for G and once for the product, for several steps.
//
// G loses what X's small singular values need if it is rounded to fp16: its noise is amplified by up to
// a^2 in every step.  So every matrix here is a sum of two fp16 planes, high and low, 22 bits, a product
// is three (high x high, high x low, low x high, added in fp32), and the steps are cut into parts over which
// that gain stays below kMaxGain; a part ends by forming X anew.  With the usual coefficients: three steps, then two.
//
// One cluster of 1 to 8 CTAs works on a matrix: each forms G of its columns (or rows, if tall) from the planes
// that the load kernel wrote, the partial sums are exchanged through distributed shared memory, every CTA runs the
// steps for itself (which needs no further exchange) and applies S to its columns.  All MMAs have 128 rows;
// N and K are m rounded up to 16, so small m costs little.
//
// Bound by the latency of the products on the m x m side, one after another.  Measured, whole calls: 64 x 96 33 us,
// 4 of 128 x 2816 87 us, 64 of 32 x 4096 171 us.
#include <cuda.h>

#include <cmath>

#include "ha_common.cuh"
#include "newton_schulz.cuh"
#include "umma.cuh"

namespace ha {
namespace {

constexpr int kThreadsN = 256;             // eight warps: TMEM lane quarter = warp % 4, column half = warp / 4
constexpr int kHalfPlane = 128 * 64 * 2;   // 128 rows of 64 fp16: one swizzled block
constexpr int kPlane = 2 * kHalfPlane;     // a 128 x 128 plane: columns 0..63, 64..127
constexpr int kMatrix = 2 * kPlane;        // high and low plane
constexpr int kOffS = 0, kOffG = kMatrix, kOffQ = 2 * kMatrix, kBytes = 3 * kMatrix + 2 * kHalfPlane;
constexpr int kSmemN = kBytes + 1024;
constexpr int kRing = 6;
// Pieces of X whose products are accumulated at once; the matrix unit cuts its sums off, which adds up (newton_schulz.cu):
// 16 x 16777216 was off by 1.5e-2 with all of a CTA's in one sum.
constexpr int kPartPieces = 256;
constexpr float kScaleN = 4096.0f;         // planes of G and Q hold 2^12 times theirs, low planes the remainder
constexpr float kScaleS = 32.0f;           // planes of S: its elements reach the product of all factors

struct NarrowArgs {
  CUtensorMap hi[2], lo;    // blocks of 64 columns x 128 rows (m rounded up to 16 of them if wide)
  CUtensorMap dst;          // the same of the caller's matrices, which take the result if `direct`
  int m, n;                 // shorter and longer side
  int tall, cluster, steps, bf16, direct;
  uint32_t ends;            // bit s: a part ends after step s
  float coef[3 * HA_NS_MAX_STEPS];
  uint32_t* error;
  uint16_t* out;            // the caller's matrices (`direct`)
  int64_t out_elems;
};

struct Bars {
  uint64_t full[kRing], empty[kRing], done[3];
};

// Byte of element (row, col) in a plane: 128-byte rows of 64 columns, 16-byte pieces swizzled by the row.
__device__ __forceinline__ uint32_t plane_at(int row, int col) {
  return uint32_t((col >> 6) * kHalfPlane + row * 128 + ((((col >> 3) & 7) ^ (row & 7)) << 4) + (col & 7) * 2);
}
__device__ __forceinline__ uint4 lds128(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(a)
               : "memory");
  return v;
}
__device__ __forceinline__ void sts128(uint32_t a, uint4 v) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(a), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
__device__ __forceinline__ float2 halves(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }

// Eight values of a row as high and low plane pieces.
__device__ __forceinline__ void store8(uint32_t matrix, int row, int col, const float (&x)[8]) {
  uint32_t h[4], l[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __half2 p = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
    const float2 f = __half22float2(p);
    const __half2 q = __floats2half2_rn(x[2 * i] - f.x, x[2 * i + 1] - f.y);
    h[i] = *reinterpret_cast<const uint32_t*>(&p);
    l[i] = *reinterpret_cast<const uint32_t*>(&q);
  }
  const uint32_t at = matrix + plane_at(row, col);
  sts128(at, make_uint4(h[0], h[1], h[2], h[3]));
  sts128(at + kPlane, make_uint4(l[0], l[1], l[2], l[3]));
}

// The 16-K slices of an operand: K-major blocks of 64 K, kHalfPlane apart, or M/N-major ones with a row for
// each K (blocks of 64 M / N, `lead` bytes apart).
template <bool MN>
__device__ __forceinline__ uint32_t slice(uint32_t desc, int ks) {
  return MN ? desc + ks * kStepMN : desc + (ks >> 2) * (kHalfPlane >> 4) + (ks & 3) * kStepK;
}
// D (+)= A B over `n` slices and the two smaller terms of both planes: into D too, or into `cross` (D + 128), where
// low planes are 2^11 larger.
template <bool A_MN, bool B_MN, bool CROSS>
__device__ __forceinline__ void split_mma(uint32_t d, uint32_t ah, uint32_t al, uint32_t bh, uint32_t bl,
                                          uint32_t idesc, int n, bool more) {
#pragma unroll 4
  for (int ks = 0; ks < n; ++ks) {
    const uint32_t a0 = slice<A_MN>(ah, ks), a1 = slice<A_MN>(al, ks);
    const uint32_t b0 = slice<B_MN>(bh, ks), b1 = slice<B_MN>(bl, ks);
    const bool add = more || ks > 0;
    mma_f16<1>(d, a0, b0, idesc, add);
    mma_f16<1>(CROSS ? d + 128 : d, a0, b1, idesc, CROSS ? add : true);
    mma_f16<1>(CROSS ? d + 128 : d, a1, b0, idesc, true);
  }
}

// Adds this warp's accumulators of one more part of a Gram matrix, those of high x high at `tmem` and of the cross terms 128
// columns further, to the sum of the parts before, 256 columns further; after the last part the sum takes their place.
// (Not inline: the code of a rare case cost small matrices 2 us.)
__device__ __noinline__ void add_part(uint32_t tmem, int c0, int np, bool first, bool last) {
#pragma unroll 1
  for (; c0 < np; c0 += 64) {
    uint32_t a[32], b[32];
    tmem_ld32(tmem + c0, a);
    tmem_ld32(tmem + 128 + c0, b);
    tmem_ld_wait();
#pragma unroll
    for (int j = 0; j < 32; ++j)
      a[j] = __float_as_uint(__fmaf_rn(__uint_as_float(b[j]), 1.0f / kScaleLo, __uint_as_float(a[j])));
    if (!first) {
      tmem_ld32(tmem + 256 + c0, b);
      tmem_ld_wait();
#pragma unroll
      for (int j = 0; j < 32; ++j) a[j] = __float_as_uint(__uint_as_float(a[j]) + __uint_as_float(b[j]));
    }
    tmem_st32(tmem + (last ? 0 : 256) + c0, a);
    if (last) {
#pragma unroll
      for (int j = 0; j < 32; ++j) b[j] = 0;
      tmem_st32(tmem + 128 + c0, b);
    }
  }
  tmem_st_wait();
}

__global__ void __launch_bounds__(kThreadsN, 1) narrow_kernel(const __grid_constant__ NarrowArgs p) {
  extern __shared__ uint8_t smem_raw[];
  __shared__ Bars bars;
  __shared__ uint32_t tmem_s;
  __shared__ volatile uint32_t stop;
  const uint32_t base = (smem_u32(smem_raw) + 1023) & ~1023u;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int quarter = warp & 3, half = warp >> 2;
  const int row = quarter * 32 + lane;  // this thread's row of every 128-row result
  const int rank = int(cluster_rank()), z = int(blockIdx.x) / p.cluster;
  const int np = (p.m + 15) & ~15;      // N and K of the square products

  if (threadIdx.x == 0) {
    stop = 0;
    for (int i = 0; i < kRing; ++i) {
      mbar_init(smem_u32(&bars.full[i]), 1);
      mbar_init(smem_u32(&bars.empty[i]), 1);
    }
    for (int i = 0; i < 3; ++i) mbar_init(smem_u32(&bars.done[i]), 1);
    mbar_fence_init();
    tma_prefetch_map(&p.hi[0]);
    tma_prefetch_map(&p.hi[1]);
    tma_prefetch_map(&p.lo);
  }
  if (warp == 0) tmem_alloc<1>(smem_u32(&tmem_s), 512);
  tc_fence_before();
  cluster_sync();
  tc_fence_after();
  grid_wait();  // the load kernel's planes
  const uint32_t tmem = tmem_s, lanes = tmem + (uint32_t(quarter * 32) << 16);
  uint32_t done_phase = 0;  // bit i: phase of bars.done[i]
  // Once a wait has run out the pieces that are left are left undone, in this part and in all that follow; the barriers of
  // the CTA and of the cluster are gone through all the same.
  bool ok = true;      // no wait of this thread has run out
  bool dead = false;   // one of the CTA's has, in an earlier part
  auto wait_done = [&](int i) {
    __syncwarp();
    ok &= mbar_wait<true>(smem_u32(&bars.done[i]), (done_phase >> i) & 1, &stop);
    __syncwarp();  // lanes leave the polling loop one by one; TMEM reads and barriers need the whole warp
    done_phase ^= 1u << i;
    tc_fence_after();
  };

  // This CTA's pieces of X: wide, 64 columns of all rows; tall, 128 rows of all columns.
  const int span = p.tall ? 128 : 64;
  const int nblk = p.tall ? (p.m + 63) / 64 : 1;  // 64-column blocks of a piece
  const int piece_bytes = p.tall ? 2 * nblk * kHalfPlane : 2 * np * 128;  // both planes
  const int pieces_all = (p.n + span - 1) / span;
  const int per_cta = (pieces_all + p.cluster - 1) / p.cluster;
  const int piece0 = rank * per_cta;
  const int pieces = max(0, min(per_cta, pieces_all - piece0));
  int plane = 0;             // high plane that holds X
  // Warp 0 issues copies and products: all its lanes follow, one elected lane acts (operands of MMAs are
  // uniform to the compiler that way; issued by `threadIdx.x == 0` each took 150 cycles).
  uint32_t full_phase = 0;   // phases of bars.full
  uint32_t emptied = 0;      // bit i: whether bars.empty[i] was committed to an odd number of times
  auto load_piece = [&](int i, uint32_t dst, uint32_t bar) {
    mbar_expect_tx(bar, piece_bytes);
    const int at = (piece0 + i) * span;
    for (int b = 0; b < nblk; ++b) {
      const int x = p.tall ? 64 * b : at, y = p.tall ? at : 0;
      tma_load_3d<1>(dst + b * kHalfPlane, &p.hi[plane], bar, x, y, z);
      tma_load_3d<1>(dst + piece_bytes / 2 + b * kHalfPlane, &p.lo, bar, x, y, z);
    }
  };

  auto wait_full = [&](int slot) {
    __syncwarp();
    ok &= mbar_wait<true>(smem_u32(&bars.full[slot]), (full_phase >> slot) & 1, &stop);
    __syncwarp();
    full_phase ^= 1u << slot;
    tc_fence_after();
  };

  for (int s0 = 0; s0 < p.steps;) {
  int s1 = s0 + 1;  // this part: steps s0 .. s1 - 1
  while (!((p.ends >> (s1 - 1)) & 1)) ++s1;
  // ---- G: high x high into columns 0.., the cross terms (2^11 larger) into columns 128..
  const int gram_slots = nblk == 2 ? 3 : kRing;
  const int gram_pieces = dead ? 0 : pieces;
  if (warp == 0)
    for (int i = 0; i < min(gram_pieces, gram_slots); ++i)
      if (elect_one()) load_piece(i, base + i * piece_bytes, smem_u32(&bars.full[i]));
  for (int from = 0;; from += kPartPieces) {
  const int to = min(from + kPartPieces, gram_pieces);
  if (warp == 0) {
    const uint32_t idesc = f16_idesc(128, np, p.tall, p.tall);
    const int ksteps = span / 16;
    for (int i = from; i < to; ++i) {
      const int slot = i % gram_slots;
      wait_full(slot);
      if (!__all_sync(0xffffffffu, ok)) break;
      const uint32_t hi = base + slot * piece_bytes, lo = hi + piece_bytes / 2;
      if (elect_one()) {
        const uint32_t h = smem_desc(hi, kHalfPlane), l = smem_desc(lo, kHalfPlane);
        if (p.tall)
          split_mma<true, true, true>(tmem, h, l, h, l, idesc, ksteps, i > from);
        else
          split_mma<false, false, true>(tmem, h, l, h, l, idesc, ksteps, i > from);
        mma_commit<1>(smem_u32(&bars.empty[slot]));
      }
      emptied ^= 1u << slot;
      if (i + gram_slots < gram_pieces) {
        __syncwarp();
        ok &= mbar_wait<true>(smem_u32(&bars.empty[slot]), ((emptied >> slot) & 1) ^ 1, &stop);
        __syncwarp();
        if (elect_one()) load_piece(i + gram_slots, base + slot * piece_bytes, smem_u32(&bars.full[slot]));
      }
    }
    if (elect_one()) mma_commit<1>(smem_u32(&bars.done[0]));
  }
  wait_done(0);
  if (gram_pieces > kPartPieces) add_part(lanes, half * 32, np, from == 0, to == gram_pieces);
  if (to == gram_pieces) break;
  tc_fence_before();
  __syncthreads();  // the accumulators are read
  tc_fence_after();
  }
  // 2^12 G as fp32, summed over the cluster, as planes into every CTA.
  {
    const uint32_t part = base + kOffS;  // 128 rows of 128 floats
    for (int c0 = half * 32; c0 < np; c0 += 64) {
      uint32_t a[32], b[32];
      tmem_ld32(lanes + c0, a);
      tmem_ld32(lanes + 128 + c0, b);
      tmem_ld_wait();
      float x[32];
#pragma unroll
      for (int j = 0; j < 32; ++j)
        x[j] = gram_pieces == 0 ? 0.0f
                           : __fmaf_rn(__uint_as_float(b[j]), 1.0f / kScaleLo, __uint_as_float(a[j])) *
                                 (kScaleN / (kScaleX * kScaleX));
      if (row < np) {
        if (p.cluster == 1) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float y[8] = {x[8 * j], x[8 * j + 1], x[8 * j + 2], x[8 * j + 3],
                                x[8 * j + 4], x[8 * j + 5], x[8 * j + 6], x[8 * j + 7]};
            store8(base + kOffG, row, c0 + 8 * j, y);
          }
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j)  // 16-byte pieces rotated by the row against bank conflicts
            sts128(part + row * 512 + ((((c0 >> 2) + j + row) & 31) << 4),
                   make_uint4(__float_as_uint(x[4 * j]), __float_as_uint(x[4 * j + 1]), __float_as_uint(x[4 * j + 2]),
                              __float_as_uint(x[4 * j + 3])));
        }
      }
    }
    tc_fence_before();
    if (p.cluster > 1) {
      __syncwarp();
      cluster_sync();
      const int mine = (np + p.cluster - 1) / p.cluster, r0 = rank * mine, r1 = min(np, r0 + mine);
      const int quads = np / 4;
      for (int e = threadIdx.x; e < (r1 - r0) * quads; e += kThreadsN) {
        const int r = r0 + e / quads, q = e % quads;
        float4 v[8], s = make_float4(0, 0, 0, 0);
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if (k < p.cluster)
            asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                         : "=f"(v[k].x), "=f"(v[k].y), "=f"(v[k].z), "=f"(v[k].w)
                         : "r"(cluster_map(part + r * 512 + (((q + r) & 31) << 4), k))
                         : "memory");
#pragma unroll
        for (int k = 0; k < 8; ++k)  // in rank order: the same sum in every run
          if (k < p.cluster) s.x += v[k].x, s.y += v[k].y, s.z += v[k].z, s.w += v[k].w;
        const __half2 h0 = __floats2half2_rn(s.x, s.y), h1 = __floats2half2_rn(s.z, s.w);
        const float2 f0 = __half22float2(h0), f1 = __half22float2(h1);
        const __half2 l0 = __floats2half2_rn(s.x - f0.x, s.y - f0.y), l1 = __floats2half2_rn(s.z - f1.x, s.w - f1.y);
        const uint32_t at = base + kOffG + plane_at(r, 4 * q);
#pragma unroll 1
        for (int k = 0; k < p.cluster; ++k) {
          asm volatile("st.shared::cluster.v2.b32 [%0], {%1, %2};" ::"r"(cluster_map(at, k)),
                       "r"(*reinterpret_cast<const uint32_t*>(&h0)), "r"(*reinterpret_cast<const uint32_t*>(&h1))
                       : "memory");
          asm volatile("st.shared::cluster.v2.b32 [%0], {%1, %2};" ::"r"(cluster_map(at + kPlane, k)),
                       "r"(*reinterpret_cast<const uint32_t*>(&l0)), "r"(*reinterpret_cast<const uint32_t*>(&l1))
                       : "memory");
        }
      }
      __syncwarp();
      cluster_sync();
    }
    fence_async_smem();
    __syncthreads();
    tc_fence_after();
  }

  // ---- the steps, in every CTA alike
  const uint32_t G = base + kOffG, Q = base + kOffQ, S = base + kOffS;
  const uint32_t square = f16_idesc(128, np, false, false);
  // D = x y, both planes; by one lane
  auto multiply = [&](uint32_t d, uint32_t x, uint32_t y, int bar) {
    split_mma<false, false, false>(d, smem_desc(x, 16), smem_desc(x + kPlane, 16), smem_desc(y, 16),
                                   smem_desc(y + kPlane, 16), square, np / 16, false);
    mma_commit<1>(smem_u32(&bars.done[bar]));
  };
  // the planes of `to` from accumulators (times `scale`)
  auto keep = [&](uint32_t d, float scale, uint32_t to) {
    for (int c0 = half * 32; c0 < np; c0 += 64) {
      uint32_t v[32];
      tmem_ld32(lanes + d + c0, v);
      tmem_ld_wait();
      if (row < np) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          float x[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) x[i] = __uint_as_float(v[8 * j + i]) * scale;
          store8(to, row, c0 + 8 * j, x);
        }
      }
    }
  };
  auto publish = [&]() {  // shared-memory planes to the MMAs, accumulators free for the next
    tc_fence_before();
    fence_async_smem();
    __syncthreads();
    tc_fence_after();
  };
  for (int s = s0; s < s1; ++s) {
    const float ca = p.coef[3 * s], cb = p.coef[3 * s + 1], cc = p.coef[3 * s + 2];
    if (warp == 0 && elect_one()) multiply(tmem, G, G, 0);
    wait_done(0);
    for (int c0 = half * 32; c0 < np; c0 += 64) {  // Q = ca I + cb G + cc G G
      uint32_t v[32];
      tmem_ld32(lanes + c0, v);
      tmem_ld_wait();
      if (row < np) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t at = G + plane_at(row, c0 + 8 * j);
          const uint4 h = lds128(at), l = lds128(at + kPlane);
          const uint32_t hw[4] = {h.x, h.y, h.z, h.w}, lw[4] = {l.x, l.y, l.z, l.w};
          float x[8];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float2 f = halves(hw[i]), g = halves(lw[i]);
            x[2 * i] = __fmaf_rn(cb, f.x + g.x, __uint_as_float(v[8 * j + 2 * i]) * (cc / kScaleN));
            x[2 * i + 1] = __fmaf_rn(cb, f.y + g.y, __uint_as_float(v[8 * j + 2 * i + 1]) * (cc / kScaleN));
          }
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (c0 + 8 * j + i == row) x[i] += ca * kScaleN;
          store8(Q, row, c0 + 8 * j, x);
          if (s == s0) {
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] *= kScaleS / kScaleN;
            store8(S, row, c0 + 8 * j, x);
          }
        }
      }
    }
    publish();
    const bool last = s + 1 == s1;
    if (warp == 0 && elect_one()) {
      if (!last) multiply(tmem + 128, G, Q, 1);
      if (s > s0) multiply(tmem + 256, Q, S, 2);
    }
    if (!last) {
      wait_done(1);
      keep(128, 1.0f / kScaleN, G);  // G Q in G's place: the product that read G is done
      publish();
      if (warp == 0 && elect_one()) multiply(tmem, G, Q, 0);
    }
    if (s > s0) {
      wait_done(2);
      keep(256, 1.0f / kScaleN, S);
    }
    if (!last) {
      wait_done(0);
      keep(0, 1.0f / kScaleN, G);
    }
    publish();
  }

  // ---- S X, piece by piece: accumulators of piece i in columns 256 (i % 2) .., cross term with the low
  // plane of X (2^11 larger) 128 columns further.  Planes of S stay; the ring takes the rest.
  const int stages = nblk == 2 ? 1 : 2;  // of results, high and low block
  const int slots = nblk == 2 ? 2 : min(kRing, 6 * kHalfPlane / piece_bytes);
  const uint32_t ring = base + kOffG, staging = base + kBytes - stages * 2 * kHalfPlane;
  const bool idle = quarter * 32 >= (p.tall ? 128 : np);            // no row of this warp is stored
  int stored = 0;
  const int todo = __syncthreads_or(int(stop)) ? 0 : pieces;
  const uint32_t idesc = p.tall ? f16_idesc(128, np, false, false) : f16_idesc(128, 64, false, true);
  const bool both = s1 < p.steps;  // X goes on: high and low plane
  const bool bf16 = p.bf16 && !both, direct = p.direct && !both;
  auto issue = [&](int i) {  // by warp 0: the products of piece i
    const int slot = i % slots;
    wait_full(slot);
    if (!elect_one()) return;
    const uint32_t hi = smem_desc(ring + slot * piece_bytes, kHalfPlane), lo = hi + (piece_bytes >> 5);
    const uint32_t sh = smem_desc(S, 16), sl = smem_desc(S + kPlane, 16), d = tmem + (i & 1) * 256;
#pragma unroll 4
    for (int ks = 0; ks < np / 16; ++ks) {
      const uint32_t s0 = slice<false>(sh, ks), s1 = slice<false>(sl, ks);
      if (p.tall) {
        const uint32_t x0 = slice<false>(hi, ks), x1 = slice<false>(lo, ks);
        mma_f16<1>(d, x0, s0, idesc, ks > 0);
        mma_f16<1>(d, x0, s1, idesc, true);
        mma_f16<1>(d + 128, x1, s0, idesc, ks > 0);
      } else {
        const uint32_t x0 = slice<true>(hi, ks), x1 = slice<true>(lo, ks);
        mma_f16<1>(d, s0, x0, idesc, ks > 0);
        mma_f16<1>(d, s1, x0, idesc, true);
        mma_f16<1>(d + 128, s0, x1, idesc, ks > 0);
      }
    }
    mma_commit<1>(smem_u32(&bars.done[i & 1]));
  };
  if (warp == 0) {
    for (int i = 0; i < min(todo, slots); ++i)
      if (elect_one()) load_piece(i, ring + i * piece_bytes, smem_u32(&bars.full[i]));
    if (todo > 0) issue(0);
  }
  for (int i = 0; i < todo; ++i) {
    if ((i & 31) == 31 && __syncthreads_or(int(stop))) break;  // (every time: 5 % of 64 of 32 x 4096)
    if (warp == 0 && i + 1 < todo) issue(i + 1);
    __syncwarp();
    wait_done(i & 1);
    if (warp == 0 && i + slots < todo && elect_one() && ok)  // piece i's slot has been read
      load_piece(i + slots, ring + (i % slots) * piece_bytes, smem_u32(&bars.full[i % slots]));
    for (int blk = 0; blk < nblk; ++blk, ++stored) {  // 64 columns at a time: 32 for each half of the warps
      if (stages == 1) {
        if (warp == 0 && elect_one()) tma_store_wait_read<0>();
        __syncthreads();  // the staging blocks are free
      }
      const uint32_t stage = staging + (stages == 2 ? (stored & 1) * 2 * kHalfPlane : 0);
      uint32_t a[32], b[32];
      const uint32_t from = lanes + (i & 1) * 256 + blk * 64 + half * 32;
      tmem_ld32(from, a);
      tmem_ld32(from + 128, b);
      tmem_ld_wait();
#pragma unroll
      for (int j = 0; j < 4 && !idle; ++j) {
        uint32_t h[4], l[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int e = 8 * j + 2 * k;
          auto value = [&](int i) {
            return __fmaf_rn(__uint_as_float(b[i]), 1.0f / kScaleLo, __uint_as_float(a[i])) * (1.0f / kScaleS);
          };
          const float x = value(e), y = value(e + 1);
          const __half2 q = __floats2half2_rn(x, y);
          const float2 f = __half22float2(q);
          const __half2 r = __floats2half2_rn((x - f.x) * kScaleLo, (y - f.y) * kScaleLo);
          h[k] = *reinterpret_cast<const uint32_t*>(&q);
          if (bf16) {
            const __nv_bfloat162 w = __floats2bfloat162_rn(x * (1.0f / kScaleX), y * (1.0f / kScaleX));
            h[k] = *reinterpret_cast<const uint32_t*>(&w);
          }
          l[k] = *reinterpret_cast<const uint32_t*>(&r);
        }
        const uint32_t at = stage + plane_at(row, half * 32 + 8 * j);
        sts128(at, make_uint4(h[0], h[1], h[2], h[3]));
        if (both) sts128(at + kHalfPlane, make_uint4(l[0], l[1], l[2], l[3]));
      }
      tc_fence_before();
      fence_async_smem();
      if (warp == 0 && elect_one()) tma_store_wait_read<0>();  // (the block before: free after the barrier)
      __syncthreads();
      if (warp == 0 && elect_one()) {
        tc_fence_after();
        const int at = (piece0 + i) * span, x = p.tall ? 64 * blk : at, y = p.tall ? at : 0;
        tma_store_3d(direct ? &p.dst : &p.hi[plane ^ 1], stage, x, y, z);
        if (both) tma_store_3d(&p.lo, stage + kHalfPlane, x, y, z);
        tma_store_commit();
      }
      __syncwarp();
    }
  }
  if (warp == 0 && elect_one()) {
    tma_store_wait_all();  // this CTA reads back only what it stored itself
    if (direct && any_gave_up(p.error)) stop = 1;
  }
  dead = __syncthreads_or(int(stop));
  plane ^= 1;
  s0 = s1;
  }
  if (dead) {  // a wait ran out: let copies and products in flight end before their memory is given up
    if (threadIdx.x == 0) gave_up(p.error);
    const uint64_t t0 = global_ns();
    while (global_ns() - t0 < 2000000) {
    }
    __syncthreads();
    if (p.direct) fill_nan(p.out, p.out_elems, kThreadsN);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 0) tmem_dealloc<1>(tmem, 512);
}

}  // namespace

// Cuts the steps into parts; false if some value would leave the planes' range.
static bool cut_parts(const float* coef, int steps, uint32_t* ends, int* parts) {
  constexpr double kMaxGain = 2000.0;  // of G's rounding noise, 2^-22, over a part
  double s = 1.0, product = 1.0;
  *ends = 0;
  *parts = 0;
  for (int i = 0; i < steps; ++i) {  // 2^12 times G, Q, G Q and 2^5 times S below 65504
    const float* c = coef + 3 * i;
    const double f = ns_factor(c, s), next = ns_growth(c, s);
    if (!(f <= 12.0 && s * s * f <= 12.0 && next * next <= 12.0)) return false;
    if (i > 0 && product * product * f * f > kMaxGain) {
      *ends |= 1u << (i - 1);
      ++*parts;
      product = 1.0;
    }
    product *= f;
    s = next;
  }
  *ends |= 1u << (steps - 1);
  ++*parts;
  return true;
}

bool narrow_fits(int64_t rows, int64_t cols, const float* coef, int steps) {
  uint32_t ends;
  int parts;
  return (rows < cols ? rows : cols) <= 128 && cut_parts(coef, steps, &ends, &parts);
}

int narrow_run(NsBatch* shape, const float* coef, int steps, int sms, cudaStream_t st) {
  const NsBatch& b = *shape;
  NarrowArgs p{};
  const int box = b.rows > b.cols ? 128 : (int(b.m) + 15) & ~15;
  int rc = ns_map(&p.hi[0], b.hi[0], b, 64, box), parts = 0;
  if (rc == HA_OK) rc = ns_map(&p.hi[1], b.hi[1], b, 64, box);
  if (rc == HA_OK) rc = ns_map(&p.lo, b.lo, b, 64, box);
  p.bf16 = shape->rounded = b.bf16;
  p.direct = b.bf16 && b.dst != nullptr;
  if (rc == HA_OK && p.direct) {
    NsBatch d = b;
    d.ld_x = b.cols;
    d.plane_x = b.rows * b.cols;
    rc = ns_map(&p.dst, reinterpret_cast<const __half*>(b.dst), d, 64, box);
  }
  if (rc != HA_OK) return rc;
  cut_parts(coef, steps, &p.ends, &parts);
  shape->out = p.direct ? -1 : parts & 1;
  p.out = b.dst;
  p.out_elems = b.n * b.rows * b.cols;
  p.tall = b.rows > b.cols;
  p.m = int(b.m);
  p.n = int(p.tall ? b.rows : b.cols);
  p.steps = steps;
  for (int i = 0; i < 3 * steps; ++i) p.coef[i] = coef[i];
  p.error = b.error;
  // More CTAs for a matrix while the chip has room for them and each still has two pieces.
  const int pieces = (p.n + (p.tall ? 127 : 63)) / (p.tall ? 128 : 64);
  p.cluster = 1;
  while (p.cluster < 8 && 2 * p.cluster * b.n <= sms && 4 * p.cluster <= pieces) p.cluster *= 2;
  if (cudaFuncSetAttribute(narrow_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemN) != cudaSuccess)
    return check_launch("narrow_kernel (shared memory)");
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(unsigned(b.n * p.cluster));
  cfg.blockDim = dim3(kThreadsN);
  cfg.dynamicSmemBytes = kSmemN;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = unsigned(p.cluster);
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, narrow_kernel, p);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return fail(HA_ERR_CUDA, "narrow_kernel: %s", cudaGetErrorString(e));
  }
  return HA_OK;
}

}  // namespace ha
