// Backward attention, bf16/f16 MFMA, gfx950. Two deterministic passes, no atomics, as in the
// reference (_sps_bwd_dq_kernel / _sps_bwd_dkdv_kernel, triton_sps_flash_attention.py:272-488;
// reverse twins triton_reverse_sps_flash_attention.py:370-599; full triton_full_flash_attention.py:301-460):
//
//  1. dQ pass (query-stationary, the forward's plan and classification). Its prologue computes
//     Delta = rowsum(O * dO) for its own queries and stores it for pass 2 (this replaces the
//     reference's separate _attn_bwd_preprocess launch). Per 32-key block:
//       S^T = K Q^T, dP^T = V dO^T (K, V rows from LDS; Q, dO in registers),
//       P = exp2(S*scale2 - LSE) (one fp32 FMA per score, as the reference scales its fp32 scores:
//       triton_sps_flash_attention.py:471), dS = P (dP - Delta)   (lane-local LSE and Delta),
//       dQ^T += K^T dS^T  (K^T fragments via ds_read_b64_tr_b16).
//  2. dK/dV pass (key-stationary; head dims up to 64, attn_bwd_split.hip has the larger ones). A
//     workgroup owns 128 keys of one stream (natural, persistent or temporary), each wave 32 of them
//     held in registers; it walks the 32-query chunks of the union of its lanes' query intervals
//     (persistent keys: diagonal to document end; temporary keys: the w-token window):
//       S = Q K^T, dP = dO V^T (Q, dO rows from LDS; K, V in registers),
//       P = exp2(S*scale2 - LSE) (fp32 FMA per score, triton_sps_flash_attention.py:361),
//       dV^T += dO^T P, dK^T += Q^T dS (dO^T, Q^T fragments via ds_read_b64_tr_b16).
// Both passes consume their tiles in groups of four 32-row blocks (one barrier per group) through
// the run_groups pipeline: buffer loads one group ahead into registers, double-buffered LDS; with
// documents the first group's loads leave right after the workgroup's plan is read. dK and dQ are
// scaled by sm_scale at the end, as in the reference.
#include "attn_bwd_dkdv.hpp"

namespace sps {

// Writes the visibility mask exactly as the key-stationary dK/dV kernel evaluates it.
__global__ __launch_bounds__(256) void mask_dump_kv_kernel(const AttnArgs a) {
  __shared__ int s_span[2 * kWaves];
  const MaskSpec m = a.m;
  const int tid = threadIdx.x, lane = tid & 63;
  const int g = lane >> 5;
  int b, h;
  TilePlan tp;
  k_workgroup(a, b, h, tp);
  const RowView row = row_view(a, b, tp.mono);
  KState st;
  int run_end;
  if (k_begin(a, tp, row, s_span, st, run_end, tid >> 6)) k_lanes(m, run_end, st);
  const bool exact = row.mono;
  const int64_t dk_doc = (!exact && st.kvalid) ? load_doc(a, b, st.kp) : 0;
  const BlockMask bm = k_block_mask(st, exact);
  for (int i = 0; i < st.nc; ++i) {
    const int qc = (st.c0 + i) * kBlock;
    const int cls = i < 128 ? mask_class(bm, i) : classify_block(st.w, qc, exact);
    if (cls == TILE_SKIP || !st.kvalid) continue;
    uint32_t bits = 0xffffu;
    if (cls == TILE_PARTIAL) {
      f32x16_t z = {};
      auto exact_bits = [&] { return ks_exact_bits(a, b, st.kp, st.r.hi, qc, g, dk_doc); };
      if (exact)
        mask_partial<true>(z, st.r, st.w, qc, g, exact_bits);
      else
        mask_partial<false>(z, st.r, st.w, qc, g, exact_bits);
      bits = 0;
      for (int e = 0; e < 16; ++e) bits |= (uint32_t)(z[e] == 0.f) << e;
    }
    for (int e = 0; e < 16; ++e) {
      const int qp = qc + acc_row(e, g);
      if (((bits >> e) & 1u) && qp < m.N) a.mask_out[((int64_t)b * m.N + qp) * m.N + st.kp] = 1;
    }
  }
}

template <int D, class E>
static hipError_t launch_bwd_t(const AttnArgs& a, int passes, hipStream_t stream) {
  const int64_t nq = (int64_t)q_tiles(a.m.N) * a.B * a.H;
  const int64_t nk = (int64_t)k_tiles(a.m.family, a.m.N, a.m.P) * a.B * a.H;
  if ((passes & kBwdDq) && nq > 0) {
    const dim3 grid((unsigned)nq), block(256);
    if (D == 128 && dq_two_waves(a.m, nq))
      hipLaunchKernelGGL((attn_bwd_dq_kernel<D, E, D == 128 ? 2 : dq_waves<D>()>), grid, block, 0, stream, a);
    else
      hipLaunchKernelGGL((attn_bwd_dq_kernel<D, E>), grid, block, 0, stream, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  if ((passes & kBwdDkdv) && nk > 0) {
    // From D = 128 on a wave cannot hold K, V, dK and dV of 32 keys beside another wave: two share them.
    if constexpr (D >= 128) {
      return launch_attn_bwd_dkdv_split(a, D, std::is_same<E, ElemF16>::value, nk, stream);
    } else {
      hipLaunchKernelGGL((attn_bwd_dkdv_kernel<D, E>), dim3((unsigned)nk), dim3(256), 0, stream, a);
      return hipGetLastError();
    }
  }
  return hipSuccess;
}

hipError_t launch_attn_bwd(const AttnArgs& a, int D, int is_f16, int passes, hipStream_t stream) {
#define SPS_BWD_CASE(DD)                                                                                  \
  case DD:                                                                                                \
    return is_f16 ? launch_bwd_t<DD, ElemF16>(a, passes, stream) : launch_bwd_t<DD, ElemBF16>(a, passes, stream);
  switch (D) {
    SPS_BWD_CASE(16)
    SPS_BWD_CASE(32)
    SPS_BWD_CASE(64)
    SPS_BWD_CASE(128)
    SPS_BWD_CASE(256)
    default:
      return hipErrorInvalidValue;
  }
#undef SPS_BWD_CASE
}

hipError_t launch_mask_dump_q(const AttnArgs& a, hipStream_t stream);

hipError_t launch_mask_dump(const AttnArgs& a, int schedule, hipStream_t stream) {
  if (schedule == 0) return launch_mask_dump_q(a, stream);
  const int n = k_tiles(a.m.family, a.m.N, a.m.P) * a.B * a.H;
  if (n == 0) return hipSuccess;
  hipLaunchKernelGGL(mask_dump_kv_kernel, dim3(n), dim3(256), 0, stream, a);
  return hipGetLastError();
}

}  // namespace sps
