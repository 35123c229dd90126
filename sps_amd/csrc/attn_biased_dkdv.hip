// dK/dV pass with changed scores at head dims up to 64 (attn_bwd_dkdv.hpp has the kernel, attn_scores.hpp the changes).
#include "attn_bwd_dkdv.hpp"

namespace sps {

template <int D, class E, class M>
static hipError_t launch_m(const BiasedArgs& a, hipStream_t stream) {
  const int64_t nk = (int64_t)k_tiles(FAMILY_FULL, a.m.N, 0) * a.B * a.H;
  if (nk == 0) return hipSuccess;
  const size_t lds = M::kBias ? lut_len(a.far) * sizeof(float) : 0;
  hipLaunchKernelGGL((attn_bwd_dkdv_kernel<D, E, M>), dim3((unsigned)nk), dim3(256), lds, stream, a);
  return hipGetLastError();
}

template <int D, class E>
static hipError_t launch_e(const BiasedArgs& a, hipStream_t stream) {
  const bool cap = a.cap2 != 0.f, bias = a.slopes || a.table;
  if (!cap) return launch_m<D, E, ChangedScores<false, true>>(a, stream);
  return bias ? launch_m<D, E, ChangedScores<true, true>>(a, stream) : launch_m<D, E, ChangedScores<true, false>>(a, stream);
}

#define SPS_CASE(DD) \
  case DD:           \
    return is_f16 ? launch_e<DD, ElemF16>(a, stream) : launch_e<DD, ElemBF16>(a, stream);
hipError_t launch_biased_dkdv(const BiasedArgs& a, int D, int is_f16, hipStream_t stream) {
  switch (D) {
    SPS_CASE(16)
    SPS_CASE(32)
    SPS_CASE(64)
    default:
      return launch_biased_dkdv_wide(a, D, is_f16, stream);
  }
}
#undef SPS_CASE

}  // namespace sps
