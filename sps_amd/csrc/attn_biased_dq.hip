// dQ pass with changed scores (attn_bwd_dq.hpp has the kernel, attn_scores.hpp the changes); with the gradient of the
// bias table: attn_biased_dq_table.hip.
#include "attn_bwd_dq.hpp"

namespace sps {

template <int D, class E, class M>
static hipError_t launch_m(const BiasedArgs& a, hipStream_t stream) {
  const int64_t nq = (int64_t)q_tiles(a.m.N) * a.B * a.H;
  if (nq == 0) return hipSuccess;
  const size_t lds = M::kBias ? lut_len(a.far) * sizeof(float) * (M::kTable ? 1 + kTableCopies : 1) : 0;
  const dim3 grid((unsigned)nq), block(256);
  if (D == 128 && dq_two_waves_changed(nq))
    hipLaunchKernelGGL((attn_bwd_dq_kernel<D, E, D == 128 ? 2 : dq_waves_changed<D, M>(), M>), grid, block, lds, stream, a);
  else
    hipLaunchKernelGGL((attn_bwd_dq_kernel<D, E, dq_waves_changed<D, M>(), M>), grid, block, lds, stream, a);
  return hipGetLastError();
}

template <int D, class E>
static hipError_t launch_e(const BiasedArgs& a, hipStream_t stream) {
  const bool cap = a.cap2 != 0.f, bias = a.slopes || a.table;
  if (!cap) return launch_m<D, E, ChangedScores<false, true>>(a, stream);
  return bias ? launch_m<D, E, ChangedScores<true, true>>(a, stream) : launch_m<D, E, ChangedScores<true, false>>(a, stream);
}

hipError_t launch_biased_dq(const BiasedArgs& a, int D, int is_f16, hipStream_t stream) {
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
