// Appends the accepted path of each sequence's drafts to its KV cache, gfx950: rows are copied as they are, and the
// lengths advance by the rows stored.
//
// One workgroup per sequence: its first wave finds the path (the set of the last accepted draft's ancestors; a draft's
// depth is its place on it), the workgroup copies the rows in 16-byte pieces, and after a barrier, when every length
// has been read, one thread per head (or one, where the heads share a length) advances it. Where each head has a
// length of its own, several workgroups share a sequence's heads, so that few sequences fill more of the chip.
// Bound by latency: the parents, the lengths, then one round of loads and stores (64 sequences x 16 heads, half of
// 64 drafts accepted, D = 64, 16.8 MB read and written: 6.2 us, 3.4 at a large copy's 4.9 TB/s; one sequence of 12 heads
// 3.8 us, a launch's latency).
#include "tree_kernels.hpp"

namespace sps {

constexpr int kCommitThreads = 512;

__global__ __launch_bounds__(kCommitThreads) void commit_kernel(const CommitArgs a) {
  __shared__ int s_path[kMaxDrafts];
  __shared__ int s_n;
  const int b = blockIdx.x, tid = threadIdx.x;
  const int per = (a.H + gridDim.y - 1) / gridDim.y, h0 = blockIdx.y * per, nh = imin(per, a.H - h0);
  if (nh <= 0) return;
  if (tid < 64) {
    const uint64_t set = ancestor_set(a.parents, a.parents_i64, b * a.parents_sb, a.T, tid);
    const int64_t last = a.last_i64 ? reinterpret_cast<const int64_t*>(a.last)[b]
                                    : (int64_t) reinterpret_cast<const int32_t*>(a.last)[b];
    const int x = last >= 0 && last < a.T ? (int)last : 0;
    uint64_t path = (uint64_t)__shfl((uint32_t)(set >> 32), x) << 32 | (uint32_t)__shfl((uint32_t)set, x);
    if (last < 0 || last >= a.T) path = 0;
    if ((path >> tid) & 1) s_path[__builtin_popcountll(path & ((1ull << tid) - 1))] = tid;
    if (tid == 0) s_n = __builtin_popcountll(path);
  }
  __syncthreads();
  const int n = s_n;
  if (n == 0) return;
  auto length = [&](int h) -> int64_t {
    return cache_len_load(a.len, b * a.len_sb + (a.len_per_head ? h * a.len_sh : 0), a.len_i64);
  };
  const int pieces = a.row_bytes / 16, total = nh * n * pieces;
  for (int i = tid; i < total; i += kCommitThreads) {
    const int p = i % pieces, r = i / pieces, j = r % n, h = h0 + r / n;
    const int64_t len = length(h);
    if (len < 0 || len >= a.storage - j) continue;
    const int64_t at = len + j;
    const int t = s_path[j];
    const u32x4_t kx = *reinterpret_cast<const u32x4_t*>(a.dk + b * a.dk_sb + t * a.dk_st + h * a.dk_sh + 16 * p);
    const u32x4_t vx = *reinterpret_cast<const u32x4_t*>(a.dv + b * a.dv_sb + t * a.dv_st + h * a.dv_sh + 16 * p);
    *reinterpret_cast<u32x4_t*>(a.k + b * a.ksb + h * a.ksh + at * a.kst + 16 * p) = kx;
    *reinterpret_cast<u32x4_t*>(a.v + b * a.vsb + h * a.vsh + at * a.vst + 16 * p) = vx;
  }
  __syncthreads();
  for (int i = tid; i < (a.len_per_head ? nh : 1); i += kCommitThreads) {
    const int64_t len = length(h0 + i);
    if (len < 0 || len >= a.storage) continue;
    const int64_t to = len < a.storage - n ? len + n : a.storage;
    cache_len_store(a.len, b * a.len_sb + (a.len_per_head ? (h0 + i) * a.len_sh : 0), a.len_i64, to);
  }
}

hipError_t launch_commit(const CommitArgs& a, hipStream_t stream) {
  if (a.B == 0 || a.H == 0 || a.T == 0) return hipSuccess;
  const int split = a.len_per_head ? imax(1, imin(a.H, 512 / imax(a.B, 1))) : 1;
  hipLaunchKernelGGL(commit_kernel, dim3(a.B, split), dim3(kCommitThreads), 0, stream, a);
  return hipGetLastError();
}

}  // namespace sps
