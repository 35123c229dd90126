// Parts of the forms for few tiles: a workgroup has 32 rows (queries, or keys), its waves share the blocks they meet and
// join at the end.
#pragma once
#include "attn_scores.hpp"
#include "wave_tile.hpp"

namespace sps {

// Elements of a wave's LDS: two tiles, whose place 32 rows of fp32 accumulators take at the end.
template <int D>
constexpr int few_lds() {
  constexpr int tiles = 2 * kBlock * WaveTile<D>::RS, rows = 2 * kBlock * (D + 4);
  return tiles > rows ? tiles : rows;
}

// Zeroes the columns that pad rows of D = 16 in a wave's two tiles.
template <int D>
__device__ __forceinline__ void zero_pads(uint16_t* tiles, int lane) {
  if constexpr (TileGeom<D>::DPAD > D) {
    for (int i = lane; i < 2 * kBlock; i += 64) {
#pragma unroll
      for (int y = D; y < TileGeom<D>::DPAD; y += 8) lds_write_b128(tiles + i * WaveTile<D>::RS + y, u32x4_t{0u, 0u, 0u, 0u});
    }
  }
}

// A wave's accumulators (lane: row lane % 32) -> 32 rows of D + 4 floats in its LDS.
template <int D>
__device__ __forceinline__ void put_rows(float* rows, const f32x16_t (&acc)[TileGeom<D>::DC], int lane) {
  float* p = rows + (lane & 31) * (D + 4);
#pragma unroll
  for (int dc = 0; dc < TileGeom<D>::DC; ++dc) {
#pragma unroll
    for (int i4 = 0; i4 < 4; ++i4) {
      const int d = 32 * dc + 8 * i4 + 4 * (lane >> 5);
      const f32x4_t y = {acc[dc][4 * i4], acc[dc][4 * i4 + 1], acc[dc][4 * i4 + 2], acc[dc][4 * i4 + 3]};
      if (d < D) *reinterpret_cast<f32x4_t*>(p + d) = y;
    }
  }
}

// Sum over the waves, in their order, of weight(wave, row) times their rows (`stride` floats apart), rounded to 16 bits.
template <int D, class E, class Weight>
__device__ __forceinline__ void sum_rows(const float* rows, int stride, uint16_t* out, int64_t out_n, int n, int tid,
                                         Weight weight) {
  for (int i = tid; i < n * (D / 8); i += 256) {
    const int r = i / (D / 8), d = (i % (D / 8)) * 8;
    float y[8] = {};
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const float f = weight(w, r);
      const float* x = rows + w * stride + r * (D + 4) + d;
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = __builtin_fmaf(f, x[e], y[e]);
    }
    *reinterpret_cast<u32x4_t*>(out + r * out_n + d) =
        u32x4_t{E::pack2(y[0], y[1]), E::pack2(y[2], y[3]), E::pack2(y[4], y[5]), E::pack2(y[6], y[7])};
  }
}

}  // namespace sps
