// dQ pass with changed scores that also sums the gradient of the bias table (attn_bwd_dq.hpp has the kernel,
// attn_scores.hpp the changes and the sums), and the table's gradient from the query tiles' sums.
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
  return a.cap2 != 0.f ? launch_m<D, E, ChangedScores<true, true, true>>(a, stream)
                       : launch_m<D, E, ChangedScores<false, true, true>>(a, stream);
}

hipError_t launch_biased_dq_table(const BiasedArgs& a, int D, int is_f16, hipStream_t stream) {
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

// dTable[j, h] = sum over rows and query tiles of their sums, in a fixed order: one workgroup per head, its threads
// over the buckets and, where buckets leave threads over, over interleaved shares of the tiles. A few hundred KiB in
// all: bound by the latency of a launch.
__global__ __launch_bounds__(256) void table_gradient_kernel(const BiasedArgs a, void* out) {
  __shared__ float s_part[256];
  const int h = blockIdx.x, tid = threadIdx.x;
  const int tiles = a.dtable_tiles, nb = a.buckets, shares = 256 / nb;
  const int j = tid % nb, share = tid / nb;
  float s = 0.f;
  if (share < shares) {
    const int64_t row = (int64_t)tiles * nb;  // of one (batch row, head)
    for (int b = 0; b < a.B; ++b) {
      const float* p = a.dtable_part + ((int64_t)b * a.H + h) * row + j;
#pragma unroll 8
      for (int t = share; t < tiles; t += shares) s += p[(int64_t)t * nb];
    }
  }
  s_part[tid] = s;
  __syncthreads();
  if (tid >= nb) return;
  for (int i = 1; i < shares; ++i) s += s_part[i * nb + tid];
  const int64_t at = (int64_t)tid * a.H + h;
  if (a.table_dtype == 2)
    reinterpret_cast<float*>(out)[at] = s;
  else
    reinterpret_cast<uint16_t*>(out)[at] = (uint16_t)(a.table_dtype == 1 ? ElemF16::pack2(s, s) : ElemBF16::pack2(s, s));
}

hipError_t launch_table_gradient(const BiasedArgs& a, void* dtable, hipStream_t stream) {
  if (a.H == 0) return hipSuccess;
  hipLaunchKernelGGL(table_gradient_kernel, dim3(a.H), dim3(256), 0, stream, a, dtable);
  return hipGetLastError();
}

}  // namespace sps
