// Tensor-core plumbing of sm_100a: mbarriers with bounded waits, tiled TMA copies, and the
// tcgen05 matrix unit with its accumulators in TMEM.  Thin wrappers over PTX, one instruction
// each; the kernels that use them state the layouts.
#pragma once

#include <cuda.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "bounded_wait.h"

namespace ha {

__device__ __forceinline__ uint32_t smem_u32(const void* p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}

__device__ __forceinline__ uint64_t global_ns() {
  uint64_t t;
  asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t));
  return t;
}

// One lane of a converged warp, the same one every time.
__device__ __forceinline__ bool elect_one() {
  uint32_t pred;
  asm volatile(
      "{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.b32 %0, 1, 0, p;\n}\n"
      : "=r"(pred));
  return pred != 0;
}

// ---------------------------------------------------------------- mbarriers
__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void mbar_fence_init() {
  asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
}
__device__ __forceinline__ void mbar_expect_tx(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ bool mbar_try(uint32_t bar, uint32_t parity) {
  uint32_t done;
  asm volatile(
      "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n selp.b32 %0, 1, 0, p;\n}\n"
      : "=r"(done)
      : "r"(bar), "r"(parity), "r"(1000000)  // may sleep for up to a millisecond: polling warps slow the issuing one
      : "memory");
  return done != 0;
}

// The same barrier or buffer in another CTA of the cluster.
__device__ __forceinline__ uint32_t cluster_map(uint32_t addr, uint32_t rank) {
  uint32_t out;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(out) : "r"(addr), "r"(rank));
  return out;
}
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}

// Programmatic dependent launch: lets the next kernel of the stream, if it was launched for that, start its
// prologue; and waits there until the kernels before have finished and their writes are visible.
__device__ __forceinline__ void grid_launch_dependents() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}
__device__ __forceinline__ void grid_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// A bounded wait (bounded_wait.h).  No wait of a healthy launch comes near the limit: it is some hundred times the
// longest kernel; it turns a lost arrival into an error word instead of a GPU that never answers.
constexpr uint64_t kWaitNs = 4000000000ull;
template <bool EARLY = false>
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity, volatile uint32_t* stop) {
  return bounded_wait<EARLY>([&] { return mbar_try(bar, parity); }, [] { return global_ns(); }, stop, kWaitNs);
}

// The same for a counter in global memory that other CTAs of the launch raise: true once it has
// reached `want`, with everything they wrote before raising it visible, to TMA too.
__device__ __forceinline__ uint32_t load_acquire(const uint32_t* p) {
  uint32_t v;
  asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
  return v;
}
__device__ __forceinline__ bool counter_wait(const uint32_t* counter, uint32_t want, volatile uint32_t* stop) {
  if (!bounded_wait<false>([&] { return load_acquire(counter) >= want; }, [] { return global_ns(); }, stop, kWaitNs)) return false;
  asm volatile("fence.proxy.async;" ::: "memory");
  return true;
}
// What one thread of a CTA has waited for with counter_wait, passed on to another through shared memory.
__device__ __forceinline__ void grant(uint32_t* granted, uint32_t value) {
  asm volatile("st.release.cta.shared::cta.u32 [%0], %1;" ::"r"(smem_u32(granted)), "r"(value) : "memory");
}
__device__ __forceinline__ uint32_t granted_now(uint32_t* granted) {
  uint32_t v;
  asm volatile("ld.acquire.cta.shared::cta.u32 %0, [%1];" : "=r"(v) : "r"(smem_u32(granted)) : "memory");
  return v;
}
__device__ __forceinline__ bool granted_wait(uint32_t* granted, uint32_t want, volatile uint32_t* stop) {
  if (!bounded_wait<false>([&] { return granted_now(granted) >= want; }, [] { return global_ns(); }, stop, kWaitNs)) return false;
  asm volatile("fence.proxy.async;" ::: "memory");
  return true;
}
// The same for all lanes of a converged warp: lane 0 looks or waits, and what it has acquired is ordered before what the
// others read afterwards by __syncwarp() (a vote orders no memory).
__device__ __forceinline__ bool granted_to_warp(uint32_t* granted, uint32_t want, int lane) {
  const bool yes = __all_sync(0xffffffffu, lane != 0 || granted_now(granted) >= want);
  __syncwarp();
  return yes;
}
__device__ __forceinline__ bool granted_wait_warp(uint32_t* granted, uint32_t want, volatile uint32_t* stop, int lane) {
  const bool yes = __all_sync(0xffffffffu, lane != 0 || granted_wait(granted, want, stop));
  __syncwarp();
  return yes;
}
// Raises it after this thread's TMA stores, which have completed.
__device__ __forceinline__ void counter_raise(uint32_t* counter) {
  asm volatile("red.release.gpu.global.add.u32 [%0], 1;" ::"l"(counter) : "memory");
}

// ---------------------------------------------------------------- launches that gave up
// Whether a CTA of this launch, or of one before it, gave up, asked by a thread whose stores have completed.  Either the
// answer is yes, or those stores lie before whatever a CTA writes after gave_up(): so the result of a launch that all
// CTAs end with this, and with fill_nan() if it says yes, is NaN as a whole or right.
__device__ __forceinline__ bool any_gave_up(const uint32_t* error) {
  __threadfence();
  return load_acquire(error) != 0;
}
// One thread of a CTA that gave up.
__device__ __forceinline__ void gave_up(uint32_t* error) {
  atomicExch(error, 1u);
  __threadfence();
}
// All `threads` threads of a CTA, after a barrier; dst is 16-byte aligned, elems a multiple of 8.
__device__ __forceinline__ void fill_nan(uint16_t* dst, int64_t elems, int threads) {
  const uint4 nan = make_uint4(0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu);
  for (int64_t e = int64_t(threadIdx.x) * 8; e < elems; e += int64_t(threads) * 8) *reinterpret_cast<uint4*>(dst + e) = nan;
}

// ---------------------------------------------------------------- TMA
__device__ __forceinline__ void tma_prefetch_map(const CUtensorMap* map) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(map)) : "memory");
}
// CG = 2: `bar` may lie in the other CTA of the pair (a cluster address).
template <int CG>
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int x, int y, int z) {
  if constexpr (CG == 1) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], "
        "[%2];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y), "r"(z)
        : "memory");
  } else {
    asm volatile(
        "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, "
        "{%3, %4, %5}], [%2];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y), "r"(z)
        : "memory");
  }
}
__device__ __forceinline__ void tma_store_3d(const CUtensorMap* map, uint32_t src, int x, int y, int z) {
  asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.tile.bulk_group [%0, {%2, %3, %4}], [%1];" ::"l"(
                   reinterpret_cast<uint64_t>(map)),
               "r"(src), "r"(x), "r"(y), "r"(z)
               : "memory");
}
// Plain bytes; addresses and size are multiples of 16.
__device__ __forceinline__ void bulk_store(void* dst, uint32_t src, uint32_t bytes) {
  asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(
                   static_cast<uint64_t>(__cvta_generic_to_global(dst))),
               "r"(src), "r"(bytes)
               : "memory");
}
__device__ __forceinline__ void tma_store_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void tma_store_wait_read() {
  asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void tma_store_wait_all() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }
// Orders this thread's shared-memory writes before later TMA reads of them.
__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// ---------------------------------------------------------------- tcgen05
// CG = 2: one warp of each CTA of the pair; both get the same columns.
template <int CG>
__device__ __forceinline__ void tmem_alloc(uint32_t dst_smem, uint32_t columns) {
  if constexpr (CG == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(dst_smem), "r"(columns)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  } else {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(dst_smem), "r"(columns)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
  }
}
template <int CG>
__device__ __forceinline__ void tmem_dealloc(uint32_t addr, uint32_t columns) {
  if constexpr (CG == 1)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(addr), "r"(columns));
  else
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(addr), "r"(columns));
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// Shared-memory operand descriptor, 128-byte swizzle, tile start aligned to 1024 bytes.
//   K-major (rows of 64 K-elements = 128 bytes): 8-row groups 1024 bytes apart;
//     `lead` unused; the next 16 K-elements start 32 bytes further.
//   MN-major (rows of 64 MN-elements, one row per K-index): 8-K groups 1024 bytes apart,
//     64-element MN blocks `lead` bytes apart; the next 16 K-indices start 2048 bytes further.
// Only its low word varies (start address in 16-byte units, `lead`); the high word holds the 1024 bytes,
// the descriptor's version and the swizzle.  Stepping along K adds to the low word.
constexpr uint32_t kDescHigh = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t smem_desc(uint32_t addr, uint32_t lead) {
  return ((addr >> 4) & 0x3fff) | ((lead >> 4) << 16);  // (addresses hold the CTA's rank in a cluster above)
}
constexpr uint32_t kStepK = 32 >> 4, kStepMN = 2048 >> 4;  // the next 16 K-indices

// D[tmem] (+)= A * B, both operands 16-bit floats of the type in `idesc`, fp32 accumulators.  CG = 2:
// issued by the pair's first CTA; each CTA holds its half of A's rows, of B's columns and of D's rows.
// a, b: low words of the operands' descriptors.
template <int CG>
__device__ __forceinline__ void mma_f16(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, bool accumulate) {
  if constexpr (CG == 1) {
    asm volatile(
        "{\n .reg .pred p;\n .reg .b64 x, y;\n setp.ne.b32 p, %4, 0;\n mov.b64 x, {%1, %5};\n mov.b64 y, {%2, %5};\n"
        " tcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %3, p;\n}\n" ::"r"(d),
        "r"(a), "r"(b), "r"(idesc), "r"(uint32_t(accumulate)), "r"(kDescHigh)
        : "memory");
  } else {
    asm volatile(
        "{\n .reg .pred p;\n .reg .b64 x, y;\n setp.ne.b32 p, %4, 0;\n mov.b64 x, {%1, %5};\n mov.b64 y, {%2, %5};\n"
        " tcgen05.mma.cta_group::2.kind::f16 [%0], x, y, %3, p;\n}\n" ::"r"(d),
        "r"(a), "r"(b), "r"(idesc), "r"(uint32_t(accumulate)), "r"(kDescHigh)
        : "memory");
  }
}
// Arrives on `bar` (CG = 2: on that barrier of both CTAs) when every tcgen05.mma this thread issued
// so far has completed.
template <int CG>
__device__ __forceinline__ void mma_commit(uint32_t bar) {
  if constexpr (CG == 1)
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
  else
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar),
        "h"(uint16_t(3))
        : "memory");
}

// 32 lanes x 32 consecutive fp32 columns: lane l of the warp gets row l of its TMEM quarter.
__device__ __forceinline__ void tmem_ld32(uint32_t addr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(addr));
}
__device__ __forceinline__ void tmem_st32(uint32_t addr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
      "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(addr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
      "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
      "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }

// Instruction descriptor of kind::f16 with fp16 operands and fp32 accumulators; *_mn: that operand
// is MN-major.
__host__ __device__ constexpr uint32_t f16_idesc(int m, int n, bool a_mn, bool b_mn) {
  return (1u << 4) | (uint32_t(a_mn) << 15) | (uint32_t(b_mn) << 16) | (uint32_t(n >> 3) << 17) |
         (uint32_t(m >> 4) << 24);
}

}  // namespace ha
