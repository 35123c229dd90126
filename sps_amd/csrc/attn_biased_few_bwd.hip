// Backward attention with changed scores where there are few tiles: a workgroup has 32 queries (dQ) or 32 keys (dK, dV),
// its four waves take every fourth block of the others each, and join at the end (attn_biased_few.hip is the forward).
//
// Products, masks and seeds as in attn_bwd_dq.hpp and attn_bwd_dkdv.hpp; each wave moves its blocks by itself, one ahead
// (wave_tile.hpp). Bound by the chain of blocks' latencies, a quarter as long; few_tiles (attn_scores.hpp) has the rule
// and what both forms measured. The joins add the waves in their order: results do not depend on timing.
#include "attn_few.hpp"

namespace sps {

// Waves per SIMD. dQ at D = 128 holds Q, dO, the block ahead and the accumulators: at two waves it spills (8 heads of 512
// tokens, 20.8 against 12.4 us).
template <int D>
constexpr int few_dq_waves() { return D <= 32 ? 3 : D == 64 ? 2 : 1; }
template <int D>
constexpr int few_dkdv_waves() { return D <= 64 ? 2 : 1; }

// dQ, the seeds of the dK/dV pass, and with M::kTable the sums of the bias table's gradient.
template <int D, class E, class M>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(few_dq_waves<D>(), 8))) void attn_few_dq_kernel(
    const BiasedArgs a) {
  using W = WaveTile<D>;
  constexpr int DC = TileGeom<D>::DC, TE = kBlock * W::RS, WE = few_lds<D>();
  __shared__ __attribute__((aligned(16))) uint16_t s_tile[kWaves][WE];

  MaskSpec m = a.m;
  m.family = FAMILY_FULL;
  const int tid = threadIdx.x, lane = tid & 63, wave = wave_uniform(tid >> 6);
  const int g = lane >> 5, c32 = lane & 31;
  const int BH = a.B * a.H, rank = (int)(blockIdx.x / (unsigned)BH), bh = (int)blockIdx.x - rank * BH;
  const int b = bh / a.H, h = bh - b * a.H;
  const int tile = (m.N - 1) / kBlock - rank, q0 = tile * kBlock, qp = q0 + c32;  // the last, which see the most, first
  const bool qvalid = qp < m.N;
  const int qsafe = qvalid ? qp : 0;
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
  auto issue = [&](int i) {
    const uint32_t r = (uint32_t)(i * kBlock) + lane_row;
    rk.load(k_src, r * k_row + piece, k_row);
    rv.load(v_src, r * v_row + piece, v_row);
  };
  u32x4_t qf[D / 16], dof[D / 16];
  float delta;
  {
    const uint16_t* q = a.q + b * a.sq.b + h * a.sq.h + (int64_t)qsafe * a.sq.n + 8 * g;
    const uint16_t* dout = a.dO + b * a.sdo.b + h * a.sdo.h + (int64_t)qsafe * a.sdo.n + 8 * g;
    const uint16_t* o = a.o + b * a.so.b + h * a.so.h + (int64_t)qsafe * a.so.n + 8 * g;
    u32x4_t of[D / 16];
#pragma unroll
    for (int c = 0; c < D / 16; ++c) {
      qf[c] = *reinterpret_cast<const u32x4_t*>(q + 16 * c);
      dof[c] = *reinterpret_cast<const u32x4_t*>(dout + 16 * c);
      of[c] = *reinterpret_cast<const u32x4_t*>(o + 16 * c);
    }
    issue(b0);
    float part[2] = {0.f, 0.f};
#pragma unroll
    for (int c = 0; c < D / 16; ++c) {
#pragma unroll
      for (int j = 0; j < 4; ++j) part[j & 1] = E::dot2(of[c][j], dof[c][j], part[j & 1]);
    }
    delta = half_sum(part[0] + part[1]);
  }
  const float lse_raw = a.lse[(int64_t)bh * m.N + qsafe], lse = lse_raw == -INFINITY ? 0.f : lse_raw;
  if (qvalid && wave == 0 && g == 0) {
    float* seed = a.seeds + (int64_t)bh * 2 * m.N + qp;
    seed[0] = -lse;
    seed[m.N] = -delta;
  }
  const ScoreConsts consts = score_consts<M>(a, h);
  float* lut = nullptr;
  TableSums<M> sums;
  if constexpr (M::kBias) {
    lut = dynamic_lds();
    fill_lut<true>(a, h, lut, tid, 256);
    sums.init(a, lut + lut_len(a.far), tid, wave);
    __syncthreads();
  }
  uint16_t *const kt = s_tile[wave], *const vt = kt + TE;
  zero_pads<D>(kt, lane);

  f32x16_t acc[DC];
#pragma unroll
  for (int dc = 0; dc < DC; ++dc) acc[dc] = f32x16_t{};
  for (int i = b0; i < nb; i += kWaves) {
    rk.store(kt, lane);
    rv.store(vt, lane);
    issue(i + kWaves);
    wave_lds_order();
    const int t0 = i * kBlock;
    f32x16_t sc, dp = f32x16_t{} - delta;
#pragma unroll
    for (int c = 0; c < D / 16; ++c) {
      sc = E::mfma(lds_read_b128(kt + c32 * W::RS + 16 * c + 8 * g), qf[c], c == 0 ? f32x16_t{} : sc);
      dp = E::mfma(lds_read_b128(vt + c32 * W::RS + 16 * c + 8 * g), dof[c], dp);
    }
    const BlockKind kind = block_kind(q0 - t0 - 31, consts.far);
    f32x16_t fac;  // the cap's derivative, where dS is wanted without it too
    qs_scores<M>(sc, consts, lut, qp, t0, g, kind, -lse, [&](int e, float r) {
      if constexpr (M::kCap && M::kTable)
        fac[e] = cap_slope(r);
      else if constexpr (M::kCap)
        dp[e] *= cap_slope(r);
    });
    if (row.mono) {
      if (classify_block(span, t0, true) != TILE_FULL) mask_partial<true>(sc, r0, span, t0, g, [] { return 0u; });
    } else {
      mask_partial<false>(sc, r0, span, t0, g, [&] { return qs_exact_bits<2>(a, b, r0, STREAM_NATURAL, t0, g, q_doc); });
    }
#pragma unroll
    for (int e = 0; e < 16; ++e) dp[e] *= fast_exp2(sc[e]);
    if constexpr (M::kTable) {
      sums.add(dp, kind, q0, t0, lane);
      if constexpr (M::kCap) {
#pragma unroll
        for (int e = 0; e < 16; ++e) dp[e] *= fac[e];
      }
    }
    uint32_t dsk[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) dsk[e] = E::pack2(dp[2 * e], dp[2 * e + 1]);
#pragma unroll
    for (int dc = 0; dc < DC; ++dc) {
#pragma unroll
      for (int kh = 0; kh < 2; ++kh) {
        const u32x4_t df = {dsk[4 * kh], dsk[4 * kh + 1], dsk[4 * kh + 2], dsk[4 * kh + 3]};
        acc[dc] = E::mfma(lds_frag_tr(kt, W::RS, 16 * kh, 32 * dc, lane), df, acc[dc]);
      }
    }
    wave_lds_order();
  }

  if constexpr (M::kTable)
    sums.store(a, a.dtable_part + ((int64_t)bh * a.dtable_tiles + tile) * a.buckets, tid, lane);
  put_rows<D>(reinterpret_cast<float*>(s_tile[wave]), acc, lane);
  __syncthreads();
  sum_rows<D, E>(reinterpret_cast<const float*>(s_tile[0]), WE / 2, a.dq + b * a.sdq.b + h * a.sdq.h + (int64_t)q0 * a.sdq.n,
                 a.sdq.n, imin(kBlock, m.N - q0), tid, [&](int, int) { return a.sm_scale; });
}

// dK and dV.
template <int D, class E, class M>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(few_dkdv_waves<D>(), 8))) void attn_few_dkdv_kernel(
    const BiasedArgs a) {
  using W = WaveTile<D>;
  constexpr int DC = TileGeom<D>::DC, TE = kBlock * W::RS, WE = few_lds<D>();
  __shared__ __attribute__((aligned(16))) uint16_t s_tile[kWaves][WE];
  __shared__ __attribute__((aligned(16))) float s_seed[kWaves][2 * kBlock];  // of a block's queries: -LSE, -Delta

  MaskSpec m = a.m;
  m.family = FAMILY_FULL;
  const int tid = threadIdx.x, lane = tid & 63, wave = wave_uniform(tid >> 6);
  const int g = lane >> 5, c32 = lane & 31;
  const int BH = a.B * a.H, rank = (int)(blockIdx.x / (unsigned)BH), bh = (int)blockIdx.x - rank * BH;
  const int b = bh / a.H, h = bh - b * a.H;
  const int k0 = rank * kBlock, kp = k0 + c32;  // the first keys, which the most queries see, first
  const bool kvalid = kp < m.N;
  const int ksafe = kvalid ? kp : 0;
  const RowView row = row_view(a, b);
  const Interval r0 = kvalid ? prefix_queries(kp, row.run_start(kp), row.run_end(kp, m.N), row_prefix(a, b))
                             : Interval{kEmptyLo, kEmptyHi};
  const WaveSpan span = wave_span_monotone(r0);
  const int64_t k_doc = (!row.mono && kvalid) ? load_doc(a, b, kp) : 0;
  const int b0 = wave_uniform(span.min_lo) / kBlock + wave, nb = wave_uniform(span.max_hi) / kBlock + 1;

  const BufRsrc q_src = head_rsrc<D>(a.q + b * a.sq.b + h * a.sq.h, a.sq.n, m.N);
  const BufRsrc o_src = head_rsrc<D>(a.dO + b * a.sdo.b + h * a.sdo.h, a.sdo.n, m.N);
  const BufRsrc seed_src = make_rsrc(a.seeds + (int64_t)bh * 2 * m.N, (uint32_t)(2 * m.N * 4));
  const uint32_t q_row = (uint32_t)(a.sq.n * 2), o_row = (uint32_t)(a.sdo.n * 2);
  const uint32_t lane_row = (uint32_t)(lane / W::CPR), piece = (uint32_t)(lane % W::CPR) * 16u;
  W rq, ro;
  uint32_t rs;
  auto issue = [&](int i) {
    const uint32_t r = (uint32_t)(i * kBlock) + lane_row;
    rq.load(q_src, r * q_row + piece, q_row);
    ro.load(o_src, r * o_row + piece, o_row);
    rs = __builtin_amdgcn_raw_buffer_load_b32(seed_src, (uint32_t)((g * m.N + imin(i * kBlock + c32, m.N - 1)) * 4), 0, 0);
  };
  issue(b0);
  u32x4_t kf[D / 16], vf[D / 16];
  {
    const uint16_t* k = a.k + b * a.sk.b + h * a.sk.h + (int64_t)ksafe * a.sk.n + 8 * g;
    const uint16_t* v = a.v + b * a.sv.b + h * a.sv.h + (int64_t)ksafe * a.sv.n + 8 * g;
#pragma unroll
    for (int c = 0; c < D / 16; ++c) {
      kf[c] = *reinterpret_cast<const u32x4_t*>(k + 16 * c);
      vf[c] = *reinterpret_cast<const u32x4_t*>(v + 16 * c);
    }
  }
  const ScoreConsts consts = score_consts<M>(a, h);
  float* lut = nullptr;
  if constexpr (M::kBias) {
    lut = dynamic_lds();
    fill_lut<false>(a, h, lut, tid, 256);
    __syncthreads();
  }
  uint16_t *const qt = s_tile[wave], *const ot = qt + TE;
  float* const seed = s_seed[wave];
  zero_pads<D>(qt, lane);

  f32x16_t dk[DC], dv[DC];
#pragma unroll
  for (int dc = 0; dc < DC; ++dc) {
    dk[dc] = f32x16_t{};
    dv[dc] = f32x16_t{};
  }
  for (int i = b0; i < nb; i += kWaves) {
    rq.store(qt, lane);
    ro.store(ot, lane);
    seed[lane] = __builtin_bit_cast(float, rs);
    issue(i + kWaves);
    wave_lds_order();
    const int qc = i * kBlock;
    f32x16_t sc, dp;
    f32x4_t l4[4];
#pragma unroll
    for (int i4 = 0; i4 < 4; ++i4) {
      l4[i4] = *reinterpret_cast<const f32x4_t*>(seed + 8 * i4 + 4 * g);
      const f32x4_t d4 = *reinterpret_cast<const f32x4_t*>(seed + kBlock + 8 * i4 + 4 * g);
#pragma unroll
      for (int t = 0; t < 4; ++t) dp[4 * i4 + t] = d4[t];
    }
#pragma unroll
    for (int c = 0; c < D / 16; ++c) {
      sc = E::mfma(lds_read_b128(qt + c32 * W::RS + 16 * c + 8 * g), kf[c], c == 0 ? f32x16_t{} : sc);
      dp = E::mfma(lds_read_b128(ot + c32 * W::RS + 16 * c + 8 * g), vf[c], dp);
    }
    ks_scores<M>(sc, consts, lut, kp, qc, g, block_kind(qc - k0 - 31, consts.far), [&](int e) { return l4[e >> 2][e & 3]; },
                 [&](int e, float r) {
                   if constexpr (M::kCap) dp[e] *= cap_slope(r);
                 });
    if (row.mono) {
      if (classify_block(span, qc, true) != TILE_FULL) mask_partial<true>(sc, r0, span, qc, g, [] { return 0u; });
    } else {
      mask_partial<false>(sc, r0, span, qc, g, [&] { return ks_exact_bits<2>(a, b, r0.lo, r0.hi, qc, g, k_doc); });
    }
    uint32_t pk[8], dsk[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float p0 = fast_exp2(sc[2 * e]), p1 = fast_exp2(sc[2 * e + 1]);
      pk[e] = E::pack2(p0, p1);
      dsk[e] = E::pack2(p0 * dp[2 * e], p1 * dp[2 * e + 1]);
    }
#pragma unroll
    for (int dc = 0; dc < DC; ++dc) {
#pragma unroll
      for (int kh = 0; kh < 2; ++kh) {
        const u32x4_t pf = {pk[4 * kh], pk[4 * kh + 1], pk[4 * kh + 2], pk[4 * kh + 3]};
        const u32x4_t df = {dsk[4 * kh], dsk[4 * kh + 1], dsk[4 * kh + 2], dsk[4 * kh + 3]};
        dv[dc] = E::mfma(lds_frag_tr(ot, W::RS, 16 * kh, 32 * dc, lane), pf, dv[dc]);
        dk[dc] = E::mfma(lds_frag_tr(qt, W::RS, 16 * kh, 32 * dc, lane), df, dk[dc]);
      }
    }
    wave_lds_order();
  }

  const float* const rows = reinterpret_cast<const float*>(s_tile[0]);
  const int keys = imin(kBlock, m.N - k0);
  put_rows<D>(reinterpret_cast<float*>(s_tile[wave]), dk, lane);
  __syncthreads();
  sum_rows<D, E>(rows, WE / 2, a.dk + b * a.sdk.b + h * a.sdk.h + (int64_t)k0 * a.sdk.n, a.sdk.n, keys, tid,
                 [&](int, int) { return a.sm_scale; });
  __syncthreads();
  put_rows<D>(reinterpret_cast<float*>(s_tile[wave]), dv, lane);
  __syncthreads();
  sum_rows<D, E>(rows, WE / 2, a.dv + b * a.sdv.b + h * a.sdv.h + (int64_t)k0 * a.sdv.n, a.sdv.n, keys, tid,
                 [&](int, int) { return 1.f; });
}

template <int D, class E, class M>
static hipError_t launch_dq(const BiasedArgs& a, hipStream_t stream) {
  const int64_t nblocks = (int64_t)((a.m.N + kBlock - 1) / kBlock) * a.B * a.H;
  const size_t lds = M::kBias ? lut_len(a.far) * sizeof(float) * (M::kTable ? 1 + kTableCopies : 1) : 0;
  hipLaunchKernelGGL((attn_few_dq_kernel<D, E, M>), dim3((unsigned)nblocks), dim3(256), lds, stream, a);
  return hipGetLastError();
}

template <int D, class E, class M>
static hipError_t launch_dkdv(const BiasedArgs& a, hipStream_t stream) {
  const int64_t nblocks = (int64_t)((a.m.N + kBlock - 1) / kBlock) * a.B * a.H;
  const size_t lds = M::kBias ? lut_len(a.far) * sizeof(float) : 0;
  hipLaunchKernelGGL((attn_few_dkdv_kernel<D, E, M>), dim3((unsigned)nblocks), dim3(256), lds, stream, a);
  return hipGetLastError();
}

template <int D, class E>
static hipError_t launch_e(const BiasedArgs& a, int pass, hipStream_t stream) {
  const bool cap = a.cap2 != 0.f, bias = a.slopes || a.table;
  if (pass == FEW_DQ && a.dtable_part)
    return cap ? launch_dq<D, E, ChangedScores<true, true, true>>(a, stream)
               : launch_dq<D, E, ChangedScores<false, true, true>>(a, stream);
  auto launch = [&](auto m) {
    using M = decltype(m);
    if (pass == FEW_DQ) return launch_dq<D, E, M>(a, stream);
    return launch_dkdv<D, E, M>(a, stream);
  };
  if (!cap) return launch(ChangedScores<false, true>());
  return bias ? launch(ChangedScores<true, true>()) : launch(ChangedScores<true, false>());
}

hipError_t launch_biased_bwd_few(const BiasedArgs& a, int D, int is_f16, int pass, hipStream_t stream) {
#define SPS_CASE(DD) \
  case DD:           \
    return is_f16 ? launch_e<DD, ElemF16>(a, pass, stream) : launch_e<DD, ElemBF16>(a, pass, stream);
  switch (D) {
    SPS_CASE(16)
    SPS_CASE(32)
    SPS_CASE(64)
    SPS_CASE(128)
    default:
      return hipErrorInvalidValue;
  }
#undef SPS_CASE
}

}  // namespace sps
