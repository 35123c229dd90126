// Forward attention with changed scores (attn_fwd.hpp has the kernel, attn_scores.hpp the changes).
#include "attn_fwd.hpp"

namespace sps {

template <int D, class E, class M>
static hipError_t launch_m(const BiasedArgs& a, hipStream_t stream) {
  const int64_t nblocks = (int64_t)q_tiles(a.m.N) * a.B * a.H;
  if (nblocks == 0) return hipSuccess;
  const size_t lds = M::kBias ? lut_len(a.far) * sizeof(float) : 0;
  hipLaunchKernelGGL((attn_fwd_kernel<D, E, fwd_waves_full<D>(), M>), dim3((unsigned)nblocks), dim3(256), lds, stream, a);
  return hipGetLastError();
}

template <int D, class E>
static hipError_t launch_e(const BiasedArgs& a, hipStream_t stream) {
  const bool cap = a.cap2 != 0.f, bias = a.slopes || a.table;
  // Uncapped scores without a bias (a prefix alone) take the biased form: its bias is 0.
  if (!cap) return launch_m<D, E, ChangedScores<false, true>>(a, stream);
  return bias ? launch_m<D, E, ChangedScores<true, true>>(a, stream) : launch_m<D, E, ChangedScores<true, false>>(a, stream);
}

hipError_t launch_biased_fwd(const BiasedArgs& a, int D, int is_f16, hipStream_t stream) {
  if (few_tiles(a, D)) return launch_biased_fwd_few(a, D, is_f16, stream);
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
