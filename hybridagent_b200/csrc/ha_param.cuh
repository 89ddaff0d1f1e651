// Stores of updated parameter values, local and into the peers' packed parameter buffers, shared
// by the update kernels.
#pragma once

#include "ha_common.cuh"

namespace ha {

struct Peers {
  int n;
  int64_t delta[HA_MAX_PEERS];
};

// Four values rounded to a 16-bit DT, packed as one 8-byte word.
template <int DT>
__device__ __forceinline__ uint2 pack4(float4 x) {
  return make_uint2(uint32_t(Elem<DT>::narrow(x.x)) | (uint32_t(Elem<DT>::narrow(x.y)) << 16),
                    uint32_t(Elem<DT>::narrow(x.z)) | (uint32_t(Elem<DT>::narrow(x.w)) << 16));
}

// The same 8 bytes at `local` + e in every peer's copy of the packed parameter buffer.
__device__ __forceinline__ void push_raw4(const Peers& p, uint64_t local, int64_t e, uint2 w) {
#pragma unroll
  for (int q = 0; q < HA_MAX_PEERS; ++q) {  // constant indices keep delta[] in the parameter bank
    if (q >= p.n) break;
    __stcs(reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(local + p.delta[q]) + e), w);
  }
}

__device__ __forceinline__ void push_f32x4(const Peers& p, uint64_t local, int64_t e, float4 x) {
#pragma unroll
  for (int q = 0; q < HA_MAX_PEERS; ++q) {
    if (q >= p.n) break;
    store4_f32(reinterpret_cast<float*>(local + p.delta[q]), e, x);
  }
}

template <int DT>
__device__ __forceinline__ void push1(const Peers& p, uint64_t local, int64_t k, float x) {
#pragma unroll
  for (int q = 0; q < HA_MAX_PEERS; ++q) {
    if (q >= p.n) break;
    if constexpr (DT == HA_F32) {
      reinterpret_cast<float*>(local + p.delta[q])[k] = x;
    } else {
      reinterpret_cast<uint16_t*>(local + p.delta[q])[k] = Elem<DT>::narrow(x);
    }
  }
}

}  // namespace ha
