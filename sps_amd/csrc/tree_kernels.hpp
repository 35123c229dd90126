// Argument blocks, geometry and host launchers of the draft-tree kernels (tree.hip, commit_drafts.hip).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "attn_scores.hpp"
#include "decode_kernels.hpp"

namespace sps {

constexpr int kMaxDrafts = 64;

// Floats per partial record of one query: acc[D], max, sum, 2 pad.
constexpr int tree_record_floats(int D) { return D + 4; }

struct TreeSeg {
  const uint16_t* k;
  const uint16_t* v;
  int64_t ksb, ksh, kst, vsb, vsh, vst;
  const void* len;
  int len_i64, len_per_head;
  int scan;        // keys t >= scan are never read
  int chunk_base;  // first chunk of this segment
};

struct TreeArgs {
  int B, H, T, n_seg;
  TreeSeg seg[kMaxDecodeSegs];
  const uint16_t* q;  // [B, T, H, D], strides (b, t, h); drafts' keys and values likewise
  const uint16_t* dk;
  const uint16_t* dv;
  Strides3 sq, sdk, sdv;  // (b, h: head, n: draft)
  const void* parents;    // [B, T] int32 or int64 (unit stride along T), or null: a chain
  int parents_i64;
  int64_t parents_sb;
  float* part;   // [B H, max(n_chunks, 1), T, D + 4]: the chunks' records
  int n_chunks, chunk_keys;
  uint16_t* out;  // [B, T, H, D] contiguous
  int cap, bias;  // scores capped / biased
  BiasedArgs s;   // score fields (scale2, cap2, cap_in, slopes, table, ..., bucket)
};

hipError_t launch_tree(const TreeArgs& a, int D, int is_f16, hipStream_t stream);

// Keys per chunk and workgroup, from the sizes the host knows.
int tree_chunk_keys(int B, int H, int T, int n_seg, const int64_t* scan);
// Whether one workgroup takes all keys of a row and writes its outputs, without records and a merge.
bool tree_whole_rows(int B, int H, int T, int n_seg, const int64_t* scan);

struct CommitArgs {
  int B, H, T;
  int row_bytes;  // of one key or value
  char* k;
  char* v;
  int64_t ksb, ksh, kst, vsb, vsh, vst;  // byte strides
  int storage;
  void* len;  // [B, H] or [B]
  int len_i64, len_per_head;
  int64_t len_sb, len_sh;
  const char* dk;  // [B, T, H, D], byte strides (b, t, h)
  const char* dv;
  int64_t dk_sb, dk_st, dk_sh, dv_sb, dv_st, dv_sh;
  const void* parents;
  int parents_i64;
  int64_t parents_sb;
  const void* last;  // [B]
  int last_i64;
};
hipError_t launch_commit(const CommitArgs& a, hipStream_t stream);

// Draft `lane` (< T <= 64, one wave): the set of its ancestors and itself, 0 where it is no draft. A parent is -1 (the
// cached sequence's last token) or an earlier draft; what has any other parent, or descends from such a one, is no
// draft. Pointers double: after step i the set holds 2^(i + 1) generations.
__device__ __forceinline__ uint64_t ancestor_set(const void* parents, int i64, int64_t row, int T, int lane) {
  int64_t p = lane - 1;
  if (parents && lane < T)
    p = i64 ? reinterpret_cast<const int64_t*>(parents)[row + lane]
            : (int64_t) reinterpret_cast<const int32_t*>(parents)[row + lane];
  bool bad = lane >= T || p < -1 || p >= lane;
  uint64_t set = 1ull << lane;
  int up = bad || p < 0 ? lane : (int)p;  // a root points to itself
  for (int step = 1; step < T; step <<= 1) {
    const uint32_t lo = __shfl((uint32_t)set, up), hi = __shfl((uint32_t)(set >> 32), up);
    const int b = __shfl((int)bad, up);
    set |= (uint64_t)hi << 32 | lo;
    bad = bad || b;
    up = __shfl(up, up);
  }
  return bad ? 0 : set;
}

}  // namespace sps
