// The dK/dV pass at head dims of 128 and 256 with unchanged scores (attn_bwd_split.hpp has the kernel).
#include "attn_bwd_split.hpp"

namespace sps {

hipError_t launch_attn_bwd_dkdv_split(const AttnArgs& a, int D, int is_f16, int64_t nblocks, hipStream_t stream) {
  const dim3 grid((unsigned)nblocks), block(kSplitThreads);
  if (D == 128) {
    if (is_f16)
      hipLaunchKernelGGL((attn_bwd_dkdv_split_kernel<128, ElemF16>), grid, block, 0, stream, a);
    else
      hipLaunchKernelGGL((attn_bwd_dkdv_split_kernel<128, ElemBF16>), grid, block, 0, stream, a);
  } else {
    if (is_f16)
      hipLaunchKernelGGL((attn_bwd_dkdv_split_kernel<256, ElemF16>), grid, block, 0, stream, a);
    else
      hipLaunchKernelGGL((attn_bwd_dkdv_split_kernel<256, ElemBF16>), grid, block, 0, stream, a);
  }
  return hipGetLastError();
}

}  // namespace sps
