// Forward attention with unchanged scores (attn_fwd.hpp has the kernel), and the forward's mask as bytes.
#include "attn_fwd.hpp"

namespace sps {

// Writes the visibility mask exactly as the query-stationary kernels (forward, dQ) evaluate it:
// same plan, same per-wave classification, same per-element tests and lane layout.
__global__ __launch_bounds__(256) void mask_dump_q_kernel(const AttnArgs a) {
  __shared__ int s_span[4 * kWaves];
  const MaskSpec m = a.m;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int g = lane >> 5, c32 = lane & 31;
  int b, h;
  TilePlan tp;
  q_workgroup(a, b, h, tp);
  const RowView row = row_view(a, b, tp.mono);
  const int qp = tp.tile * kTile + wave * kBlock + c32;
  const bool qvalid = qp < m.N;
  QState st;
  int run_start;
  if (q_begin(a, tp, row, qp, s_span, st, run_start)) q_lanes(m, qp, run_start, st);
  const QPlan& plan = st.plan;
  const bool exact = row.mono;
  const int64_t dq_doc = (!exact && qvalid) ? load_doc(a, b, qp) : 0;
  uint8_t* mrow = a.mask_out + ((int64_t)b * m.N + (qvalid ? qp : 0)) * m.N;
  const BlockMask bm = q_block_mask(st, exact);
  for (int i = 0; i < plan.count(); ++i) {
    const bool s0 = i < plan.n0;
    const int t0 = plan.first(i), stream = plan.stream(i);
    const WaveSpan ws = s0 ? st.w0 : st.w1;
    const Interval lr = s0 ? st.r0 : st.r1;
    const int cls = i < 128 ? mask_class(bm, i) : classify_block(ws, t0, exact);
    if (cls == TILE_SKIP || !qvalid) continue;
    uint32_t bits = 0xffffu;
    if (cls == TILE_PARTIAL) {
      f32x16_t z = {};
      auto exact_bits = [&] { return qs_exact_bits(a, b, lr, stream, t0, g, dq_doc); };
      if (exact)
        mask_partial<true>(z, lr, ws, t0, g, exact_bits);
      else
        mask_partial<false>(z, lr, ws, t0, g, exact_bits);
      bits = 0;
      for (int e = 0; e < 16; ++e) bits |= (uint32_t)(z[e] == 0.f) << e;
    }
    for (int e = 0; e < 16; ++e) {
      if ((bits >> e) & 1u) mrow[stream_pos(m, stream, t0 + acc_row(e, g))] = 1;
    }
  }
}

template <int D, class E>
static hipError_t launch_fwd_t(const AttnArgs& a, hipStream_t stream) {
  const int64_t nblocks = (int64_t)q_tiles(a.m.N) * a.B * a.H;
  if (nblocks == 0) return hipSuccess;
  if (a.m.family == FAMILY_FULL)
    hipLaunchKernelGGL((attn_fwd_kernel<D, E, fwd_waves_full<D>()>), dim3((unsigned)nblocks), dim3(256), 0, stream, a);
  else
    hipLaunchKernelGGL((attn_fwd_kernel<D, E, fwd_waves_sps<D>()>), dim3((unsigned)nblocks), dim3(256), 0, stream, a);
  return hipGetLastError();
}

hipError_t launch_attn_fwd(const AttnArgs& a, int D, int is_f16, hipStream_t stream) {
#define SPS_FWD_CASE(DD)                                                                      \
  case DD:                                                                                    \
    return is_f16 ? launch_fwd_t<DD, ElemF16>(a, stream) : launch_fwd_t<DD, ElemBF16>(a, stream);
  switch (D) {
    SPS_FWD_CASE(16)
    SPS_FWD_CASE(32)
    SPS_FWD_CASE(64)
    SPS_FWD_CASE(128)
    SPS_FWD_CASE(256)
    default:
      return hipErrorInvalidValue;
  }
#undef SPS_FWD_CASE
}

hipError_t launch_mask_dump_q(const AttnArgs& a, hipStream_t stream) {
  const int n = q_tiles(a.m.N) * a.B * a.H;
  if (n == 0) return hipSuccess;
  hipLaunchKernelGGL(mask_dump_q_kernel, dim3(n), dim3(256), 0, stream, a);
  return hipGetLastError();
}

}  // namespace sps
