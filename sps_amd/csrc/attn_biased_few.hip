// Forward attention with changed scores where there are few tiles: a workgroup has 32 queries (not 128), its four waves
// take every fourth block of their keys each, and join at the end.
//
// Scores, masks and softmax as in attn_fwd.hpp. Each wave moves its blocks by itself, through registers into tiles of
// its own, one block ahead, without barriers (wave_tile.hpp). A chain of latencies bounds such calls, and it is a
// quarter as long (few_tiles, attn_scores.hpp, has the rule and what both forms measured). Per block: the scores' instructions
// and two dependent product chains, ~1.2 us at one wave per SIMD.
#include "attn_few.hpp"

namespace sps {

template <int D>
constexpr int few_waves() { return D <= 64 ? 3 : D == 128 ? 2 : 1; }

template <int D, class E, class M>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(few_waves<D>(), 8))) void attn_few_kernel(
    const BiasedArgs a) {
  using W = WaveTile<D>;
  constexpr int DC = TileGeom<D>::DC, TE = kBlock * W::RS;
  constexpr int WE = few_lds<D>();
  __shared__ __attribute__((aligned(16))) uint16_t s_tile[kWaves][WE];
  __shared__ float s_m[kWaves][kBlock], s_l[kWaves][kBlock], s_f[kWaves][kBlock];

  MaskSpec m = a.m;
  m.family = FAMILY_FULL;
  const int tid = threadIdx.x, lane = tid & 63, wave = wave_uniform(tid >> 6);
  const int g = lane >> 5, c32 = lane & 31;
  // The last queries, which see the most keys, first.
  const int BH = a.B * a.H, rank = (int)(blockIdx.x / (unsigned)BH), bh = (int)blockIdx.x - rank * BH;
  const int b = bh / a.H, h = bh - b * a.H;
  const int q0 = ((m.N - 1) / kBlock - rank) * kBlock, qp = q0 + c32;
  const bool qvalid = qp < m.N;
  const RowView row = row_view(a, b);
  const Interval r0 = qvalid ? prefix_keys(qp, row.run_start(qp), row.run_end(qp, m.N), row_prefix(a, b))
                             : Interval{kEmptyLo, kEmptyHi};
  const WaveSpan span = wave_span_monotone(r0);
  const int64_t q_doc = (!row.mono && qvalid) ? load_doc(a, b, qp) : 0;
  const int b0 = wave_uniform(span.min_lo) / kBlock + wave, nb = wave_uniform(span.max_hi) / kBlock + 1;

  const BufRsrc k_src = head_rsrc<D>(a.k + b * a.sk.b + h * a.sk.h, a.sk.n, m.N);
  const BufRsrc v_src = head_rsrc<D>(a.v + b * a.sv.b + h * a.sv.h, a.sv.n, m.N);
  const uint32_t k_row = (uint32_t)(a.sk.n * 2), v_row = (uint32_t)(a.sv.n * 2);
  const uint32_t lane_row = (uint32_t)(lane / W::CPR), piece = (uint32_t)(lane % W::CPR) * 16u;
  W rk, rv;
  // Always: blocks past the last are never used, and the compiler can count the loads in flight.
  auto issue = [&](int i) {
    const uint32_t r = (uint32_t)(i * kBlock) + lane_row;
    rk.load(k_src, r * k_row + piece, k_row);
    rv.load(v_src, r * v_row + piece, v_row);
  };
  issue(b0);
  u32x4_t qf[D / 16];
  {
    const uint16_t* q = a.q + b * a.sq.b + h * a.sq.h + (int64_t)(qvalid ? qp : 0) * a.sq.n + 8 * g;
#pragma unroll
    for (int c = 0; c < D / 16; ++c) qf[c] = *reinterpret_cast<const u32x4_t*>(q + 16 * c);
  }
  const ScoreConsts consts = score_consts<M>(a, h);
  float* lut = nullptr;
  if constexpr (M::kBias) {
    lut = dynamic_lds();
    fill_lut<true>(a, h, lut, tid, 256);
    __syncthreads();
  }
  uint16_t *const kt = s_tile[wave], *const vt = kt + TE;
  zero_pads<D>(kt, lane);

  float m_run = -INFINITY, l_run[2] = {0.f, 0.f};
  f32x16_t acc[DC];
#pragma unroll
  for (int dc = 0; dc < DC; ++dc) acc[dc] = f32x16_t{};
  for (int i = b0; i < nb; i += kWaves) {
    rk.store(kt, lane);
    rv.store(vt, lane);
    issue(i + kWaves);
    wave_lds_order();
    const int t0 = i * kBlock;
    f32x16_t sc;
#pragma unroll
    for (int c = 0; c < D / 16; ++c)
      sc = E::mfma(lds_read_b128(kt + c32 * W::RS + 16 * c + 8 * g), qf[c], c == 0 ? f32x16_t{} : sc);
    qs_scores<M>(sc, consts, lut, qp, t0, g, block_kind(q0 - t0 - 31, consts.far), 0.f, [](int, float) {});
    if (row.mono) {
      if (classify_block(span, t0, true) != TILE_FULL) mask_partial<true>(sc, r0, span, t0, g, [] { return 0u; });
    } else {
      mask_partial<false>(sc, r0, span, t0, g, [&] { return qs_exact_bits(a, b, r0, STREAM_NATURAL, t0, g, q_doc); });
    }
    float mx = max3f(sc[0], sc[1], sc[2]);
#pragma unroll
    for (int e = 3; e < 15; e += 2) mx = max3f(mx, sc[e], sc[e + 1]);
    mx = half_max(__builtin_elementwise_maximum(mx, sc[15]));
    if (wave_any(mx > m_run)) {
      const float m_new = mx > m_run ? mx : m_run;
      const float alpha = mx > m_run ? fast_exp2(m_run - m_new) : 1.f;
      l_run[0] *= alpha;
      l_run[1] *= alpha;
#pragma unroll
      for (int dc = 0; dc < DC; ++dc) acc[dc] *= alpha;
      m_run = m_new;
    }
    const float negm = m_run == -INFINITY ? 0.f : -m_run;
    uint32_t pk[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float p0 = fast_exp2(sc[2 * e] + negm), p1 = fast_exp2(sc[2 * e + 1] + negm);
      pk[e] = E::pack2(p0, p1);
      if constexpr (M::kBias)
        l_run[e & 1] += p0 + p1;  // (of the unrounded weights: see attn_fwd.hpp)
      else
        l_run[e & 1] = E::sum2(pk[e], l_run[e & 1]);
    }
#pragma unroll
    for (int dc = 0; dc < DC; ++dc) {
#pragma unroll
      for (int kh = 0; kh < 2; ++kh) {
        const u32x4_t pf = {pk[4 * kh], pk[4 * kh + 1], pk[4 * kh + 2], pk[4 * kh + 3]};
        acc[dc] = E::mfma(lds_frag_tr(vt, W::RS, 16 * kh, 32 * dc, lane), pf, acc[dc]);
      }
    }
    wave_lds_order();
  }

  // The waves join: accumulators through their LDS, each wave's weight once per query.
  put_rows<D>(reinterpret_cast<float*>(s_tile[wave]), acc, lane);
  const float l = half_sum(l_run[0] + l_run[1]);
  if (g == 0) {
    s_m[wave][c32] = m_run;
    s_l[wave][c32] = l;
  }
  __syncthreads();
  const int queries = imin(kBlock, m.N - q0);
  if (tid < queries) {
    float top = -INFINITY, sum = 0.f, f[kWaves];
#pragma unroll
    for (int w = 0; w < kWaves; ++w) top = fmaxf(top, s_m[w][tid]);
    const float mu = top == -INFINITY ? 0.f : top;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      f[w] = fast_exp2(s_m[w][tid] - mu);
      sum = __builtin_fmaf(f[w], s_l[w][tid], sum);
    }
    const float inv = sum > 0.f ? __builtin_amdgcn_rcpf(sum) : 0.f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) s_f[w][tid] = f[w] * inv;
    a.lse[(int64_t)bh * m.N + q0 + tid] = sum > 0.f ? top + __log2f(sum) : -INFINITY;
  }
  __syncthreads();
  sum_rows<D, E>(reinterpret_cast<const float*>(s_tile[0]), WE / 2, a.out + b * a.sout.b + h * a.sout.h + (int64_t)q0 * a.sout.n,
                 a.sout.n, queries, tid, [&](int w, int r) { return s_f[w][r]; });
}

template <int D, class E, class M>
static hipError_t launch_m(const BiasedArgs& a, hipStream_t stream) {
  const int64_t nblocks = (int64_t)((a.m.N + kBlock - 1) / kBlock) * a.B * a.H;
  const size_t lds = M::kBias ? lut_len(a.far) * sizeof(float) : 0;
  hipLaunchKernelGGL((attn_few_kernel<D, E, M>), dim3((unsigned)nblocks), dim3(256), lds, stream, a);
  return hipGetLastError();
}

template <int D, class E>
static hipError_t launch_e(const BiasedArgs& a, hipStream_t stream) {
  const bool cap = a.cap2 != 0.f, bias = a.slopes || a.table;
  if (!cap) return launch_m<D, E, ChangedScores<false, true>>(a, stream);
  return bias ? launch_m<D, E, ChangedScores<true, true>>(a, stream) : launch_m<D, E, ChangedScores<true, false>>(a, stream);
}

hipError_t launch_biased_fwd_few(const BiasedArgs& a, int D, int is_f16, hipStream_t stream) {
#define SPS_CASE(DD) \
  case DD:           \
    return is_f16 ? launch_e<DD, ElemF16>(a, stream) : launch_e<DD, ElemBF16>(a, stream);
  switch (D) {
    SPS_CASE(16)
    SPS_CASE(32)
    SPS_CASE(64)
    SPS_CASE(128)
    SPS_CASE(256)
    default:
      return hipErrorInvalidValue;
  }
#undef SPS_CASE
}

}  // namespace sps
