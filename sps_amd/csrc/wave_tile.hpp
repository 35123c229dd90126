// Tiles of 32 rows that a wave moves by itself, from global memory through its registers to LDS that no other wave
// reads: no barriers, so waves that split a long axis go each at their own pace.
#pragma once
#include "attn_tiles.hpp"

namespace sps {

// One wave's 32-row tile of D elements, in registers on its way from the cache to LDS: 16 bytes a lane and pass.
template <int D>
struct WaveTile {
  static constexpr int CPR = D / 8, RPP = 64 / CPR, PASSES = kBlock / RPP;
  static constexpr int RS = TileGeom<D>::RS;  // padded LDS rows
  u32x4_t v[PASSES];

  // `off`: the lane's piece of the first pass; nontemporal, since a cache row is read once.
  __device__ __forceinline__ void load(BufRsrc rs, uint32_t off, uint32_t row_bytes) {
#pragma unroll
    for (int p = 0; p < PASSES; ++p) v[p] = __builtin_amdgcn_raw_buffer_load_b128(rs, off + p * RPP * row_bytes, 0, 2);
  }
  __device__ __forceinline__ void store(uint16_t* tile, int lane) const {
#pragma unroll
    for (int p = 0; p < PASSES; ++p) lds_write_b128(tile + (p * RPP + lane / CPR) * RS + (lane % CPR) * 8, v[p]);
  }
};

// LDS operations of one wave run in order; this keeps the compiler, which sees one lane's addresses, from exchanging
// them where lanes read what others wrote.
__device__ __forceinline__ void wave_lds_order() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local");
  __builtin_amdgcn_wave_barrier();
}

}  // namespace sps
