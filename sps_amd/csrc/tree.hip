// Attention of up to 64 drafted tokens per sequence (a tree, a chain, or one token) over up to 3 variable-length KV
// segments and the drafts' own ancestors, gfx950.
//
// Draft i sees every live key of the segments, its ancestors among the drafts and itself. The positions that a bias by
// distance uses run through the segments in their order; a draft's is the number of live keys plus its depth.
//
// Split over the keys: one workgroup per chunk of one segment, (sequence, head), and one for the drafts among
// themselves; each writes a partial record (accumulator, maximum, sum) per draft, and a second kernel merges them.
// The pass is bound by HBM: every key and value is read once, 4 D bytes against 4 D T products, so at T = 64 the
// matrix cores need a fifth of the time the bytes do. A workgroup stages groups of 32-key blocks by direct
// global -> LDS loads, one group ahead (head dims below 64: through registers); its four waves are the drafts' tiles
// of 32 (T > 32: two) times shares of the blocks. Products and softmax as the forward's (attn_fwd.hpp): S^T = K Q^T,
// a lane holds one draft, so maximum and sum are the lane's own. The buffer descriptors cover the chunk's live rows
// alone: rows past the live length read as zeros, whatever the cache holds there, and offsets stay small however long
// the cache.
#include "tree_kernels.hpp"

namespace sps {

__device__ __forceinline__ int tree_live(const TreeArgs& a, const TreeSeg& sg, int b, int h) {
  if (sg.scan == 0) return 0;
  const int64_t i = sg.len_per_head ? (int64_t)b * a.H + h : b;
  const int64_t n = sg.len_i64 ? reinterpret_cast<const int64_t*>(sg.len)[i]
                               : (int64_t) reinterpret_cast<const int32_t*>(sg.len)[i];
  return n < 0 ? 0 : n > sg.scan ? sg.scan : (int)n;
}

// Online softmax of one wave's 32 drafts.
template <int D>
struct TreeState {
  static constexpr int DC = TileGeom<D>::DC;
  float m, l;
  f32x16_t acc[DC];
};

template <int D, class E, int QT>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(D <= 64 ? 2 : 1, 8))) void tree_partial_kernel(
    const TreeArgs a) {
  using G = TileGeom<D>;
  constexpr int NB = tree_group(D);
  constexpr bool kDma = D >= 64;
  using DT = DmaTile<kDma ? D : 64, false>;
  constexpr int TE = kDma ? DT::ELEMS : G::ELEMS;
  constexpr int SHARES = 4 / QT;  // waves that share one tile's blocks
  constexpr int REC = tree_record_floats(D);
  // A wave's 32 x D accumulators pass through one of the four arrays at the end.
  constexpr int AE = NB * TE > 64 * (D + 2) ? NB * TE : 64 * (D + 2);
  __shared__ __attribute__((aligned(16))) uint16_t sK0[AE], sK1[AE], sV0[AE], sV1[AE];
  __shared__ uint64_t s_set[kMaxDrafts];
  __shared__ float s_ml[4][2][32];
  auto tK = [&](int buf, int y) -> uint16_t* { return (buf ? sK1 : sK0) + y * TE; };
  auto tV = [&](int buf, int y) -> uint16_t* { return (buf ? sV1 : sV0) + y * TE; };

  const int c = blockIdx.x, h = blockIdx.y, b = blockIdx.z;
  const int tid = threadIdx.x, lane = tid & 63, wave = wave_uniform(tid >> 6);
  const int g = lane >> 5, c32 = lane & 31;
  const int qt = wave % QT, share = wave / QT;
  const bool drafts = c == a.n_chunks;  // the drafts among themselves

  // The chunk: rows [0, rows) from k, v; `place`: the position of its first key, `past`: live keys of all segments.
  const uint16_t *k, *v;
  int64_t kst, vst;
  int rows, place = 0, past = 0;
  if (drafts) {
    k = a.dk + b * a.sdk.b + h * a.sdk.h;
    v = a.dv + b * a.sdv.b + h * a.sdv.h;
    kst = a.sdk.n;
    vst = a.sdv.n;
    rows = a.T;
  } else {
    int si = 0;
    while (si + 1 < a.n_seg && c >= a.seg[si + 1].chunk_base) ++si;
    const TreeSeg& sg = a.seg[si];
    const int t0 = (c - sg.chunk_base) * a.chunk_keys;
    const int live = tree_live(a, sg, b, h);
    rows = imin(live - t0, a.chunk_keys);
    if (rows <= 0) return;
    k = sg.k + b * sg.ksb + h * sg.ksh + t0 * sg.kst;
    v = sg.v + b * sg.vsb + h * sg.vsh + t0 * sg.vst;
    kst = sg.kst;
    vst = sg.vst;
    place = t0;
    if (a.bias) {
      for (int s = 0; s < a.n_seg; ++s) {
        const int n = s == si ? live : tree_live(a, a.seg[s], b, h);
        past += n;
        if (s < si) place += n;
      }
    }
  }
  rows = wave_uniform(rows);
  const int nb = (rows + kBlock - 1) / kBlock;

  const BufRsrc k_src = make_rsrc(k, (uint32_t)((int64_t)(rows - 1) * kst * 2 + D * 2));
  const BufRsrc v_src = make_rsrc(v, (uint32_t)((int64_t)(rows - 1) * vst * 2 + D * 2));
  const uint32_t k_blk = (uint32_t)(kBlock * kst * 2), v_blk = (uint32_t)(kBlock * vst * 2);
  const auto k_dma = DT::sources(tid, (uint32_t)(kst * 2));
  const auto v_dma = DT::sources(tid, (uint32_t)(vst * 2));
  constexpr uint32_t kOut = 0x80000000u;  // past every descriptor's range: zeros
  auto issue_dma = [&](int j, int buf) {
#pragma unroll
    for (int y = 0; y < NB; ++y) {
      const int i = NB * j + y;
      if (i < nb) {
        DT::load(k_src, (uint32_t)i * k_blk, k_dma, tK(buf, y), wave);
        DT::load(v_src, (uint32_t)i * v_blk, v_dma, tV(buf, y), wave);
      }
    }
  };
  TileRegs<D> rk[1][NB], rv[1][NB];
  const auto k_off = TileRegs<D>::offsets(tid, (uint32_t)(kst * 2));
  const auto v_off = TileRegs<D>::offsets(tid, (uint32_t)(vst * 2));
  auto issue_regs = [&](int j, int slot) {
#pragma unroll
    for (int y = 0; y < NB; ++y) {
      const int i = NB * j + y;
      rk[slot][y].load(k_src, i < nb ? (uint32_t)i * k_blk : kOut, k_off, tid);
      rv[slot][y].load(v_src, i < nb ? (uint32_t)i * v_blk : kOut, v_off, tid);
    }
  };
  auto put_regs = [&](int slot, int buf) {
#pragma unroll
    for (int y = 0; y < NB; ++y) {
      rk[slot][y].store(tK(buf, y), tid);
      rv[slot][y].store(tV(buf, y), tid);
    }
  };
  if constexpr (kDma) {
    issue_dma(0, 0);
  } else {
#pragma unroll
    for (int y = 0; y < NB; ++y) {
      zero_pad_cols<D>(tK(0, y), tid);
      zero_pad_cols<D>(tK(1, y), tid);
      zero_pad_cols<D>(tV(0, y), tid);
      zero_pad_cols<D>(tV(1, y), tid);
    }
  }

  // The lane's draft: its query (zeros past the last), and depth.
  const int qi = qt * 32 + c32;
  const bool qvalid = qi < a.T;
  u32x4_t qf[D / 16];
  {
    const uint16_t* row = a.q + b * a.sq.b + h * a.sq.h + (qvalid ? qi : 0) * a.sq.n;
#pragma unroll
    for (int x = 0; x < D / 16; ++x) {
      const u32x4_t z = {0u, 0u, 0u, 0u};
      qf[x] = qvalid ? *reinterpret_cast<const u32x4_t*>(row + 16 * x + 8 * g) : z;
    }
  }
  float* lut = nullptr;
  float slope2 = 0.f;
  if (a.bias) {
    // Table bias of distances 0 .. far (the last also of every greater one).
    lut = dynamic_lds();
    if (a.s.slopes) slope2 = a.s.slopes[h] * kLog2e;
    for (int n = tid; n <= a.s.far; n += 256) {
      float x = a.s.table ? table_entry(a.s, n < a.s.far ? a.s.bucket[n] : a.s.buckets - 1, h) : 0.f;
      lut[n] = x < kHidden ? -INFINITY : x * kLog2e;
    }
  }
  if (a.bias || drafts) {
    if (wave == 0) {
      const uint64_t set = ancestor_set(a.parents, a.parents_i64, b * a.parents_sb, a.T, lane);
      s_set[lane] = set;
    }
    __syncthreads();
  }
  const uint64_t own = a.bias || drafts ? s_set[qi] : 0;
  const int depth = own ? __builtin_popcountll(own) - 1 : 0;

  TreeState<D> st;
  st.m = -INFINITY;
  st.l = 0.f;
#pragma unroll
  for (int dc = 0; dc < G::DC; ++dc) st.acc[dc] = f32x16_t{};
  const float scale2 = a.s.scale2, cap2 = a.s.cap2, cap_in = a.s.cap_in;
  const int far = a.s.far;
  auto row_frag = [&](const uint16_t* tile, int x) {
    if constexpr (kDma)
      return lds_read_b128(tile + DT::frag(c32, g, x));
    else
      return lds_read_b128(tile + c32 * G::RS + 16 * x + 8 * g);
  };
  auto tr_frag = [&](const uint16_t* tile, int kh, int dc) {
    if constexpr (kDma)
      return DT::frag_tr(tile, 16 * kh, dc, lane);
    else
      return lds_frag_tr(tile, G::RS, 16 * kh, 32 * dc, lane);
  };
  auto block = [&](int i, uint16_t* kt, uint16_t* vt) {
    f32x16_t sc = E::mfma(row_frag(kt, 0), qf[0], f32x16_t{});
#pragma unroll
    for (int x = 1; x < D / 16; ++x) sc = E::mfma(row_frag(kt, x), qf[x], sc);
    if (a.cap) {
#pragma unroll
      for (int e = 0; e < 16; ++e)
        sc[e] = __builtin_fmaf(__builtin_amdgcn_rcpf(1.f + fast_exp2(sc[e] * cap_in)), -2.f * cap2, cap2);
    } else {
#pragma unroll
      for (int e = 0; e < 16; ++e) sc[e] *= scale2;
    }
    const int r0 = i * kBlock + 4 * g;  // the chunk's row of element 0
    if (drafts) {
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int j = r0 + acc_row0(e);
        const bool see = j < a.T && ((own >> j) & 1);
        if (a.bias) {
          const int n = imax(depth - (__builtin_popcountll(s_set[imin(j, kMaxDrafts - 1)]) - 1), 0);
          sc[e] += __builtin_fmaf(-slope2, (float)n, lut[imin(n, far)]);
        }
        sc[e] = see ? sc[e] : -INFINITY;
      }
    } else {
      if (a.bias) {
        const int d = past + depth - place - r0;  // distance of element 0
        // The smallest distance of the block, over lanes and rows: where it reaches `far` the table adds one value.
        if (past - place - i * kBlock - 31 >= far) {
          const float base = __builtin_fmaf(-slope2, (float)d, lut[far]);
#pragma unroll
          for (int e = 0; e < 16; ++e) sc[e] += __builtin_fmaf(slope2, (float)acc_row0(e), base);
        } else {
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const int n = imax(d - acc_row0(e), 0);  // (negative past the live rows, which are masked)
            sc[e] += __builtin_fmaf(-slope2, (float)n, lut[imin(n, far)]);
          }
        }
      }
      if (rows - i * kBlock < kBlock) {
#pragma unroll
        for (int e = 0; e < 16; ++e) sc[e] = r0 + acc_row0(e) < rows ? sc[e] : -INFINITY;
      }
    }
    float mx = max3f(sc[0], sc[1], sc[2]);
#pragma unroll
    for (int e = 3; e < 15; e += 2) mx = max3f(mx, sc[e], sc[e + 1]);
    mx = half_max(__builtin_elementwise_maximum(mx, sc[15]));
    if (wave_any(mx > st.m)) {
      const float m_new = mx > st.m ? mx : st.m;
      const float alpha = mx > st.m ? fast_exp2(st.m - m_new) : 1.f;
      st.l *= alpha;
#pragma unroll
      for (int dc = 0; dc < G::DC; ++dc) st.acc[dc] *= alpha;
      st.m = m_new;
    }
    const float negm = st.m == -INFINITY ? 0.f : -st.m;
    uint32_t pk[8];
    float sum = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float p0 = fast_exp2(sc[2 * e] + negm), p1 = fast_exp2(sc[2 * e + 1] + negm);
      pk[e] = E::pack2(p0, p1);
      sum += p0 + p1;
    }
    st.l += sum;
#pragma unroll
    for (int dc = 0; dc < G::DC; ++dc) {
#pragma unroll
      for (int kh = 0; kh < 2; ++kh) {
        const u32x4_t pf = {pk[4 * kh], pk[4 * kh + 1], pk[4 * kh + 2], pk[4 * kh + 3]};
        st.acc[dc] = E::mfma(tr_frag(vt, kh, dc), pf, st.acc[dc]);
      }
    }
  };
  auto body = [&](int j, int buf) {
    if (drafts) {
      // Rows that are no draft: zeros, so that whatever they hold stays out of the zero-weighted products.
      for (int x = tid; x < NB * kBlock; x += 256) {
        const int i = NB * j + x / kBlock, r = x % kBlock, t = i * kBlock + r;
        if (i < nb && !(t < a.T && s_set[t])) {
          uint16_t* vt = tV(buf, x / kBlock) + r * (kDma ? D : G::RS);
          for (int y = 0; y < D; y += 8) lds_write_b128(vt + y, u32x4_t{0u, 0u, 0u, 0u});
        }
      }
      __syncthreads();
    }
#pragma unroll
    for (int y = 0; y < NB; ++y) {
      if (y % SHARES != share) continue;
      const int i = NB * j + y;
      if (i < nb) block(i, tK(buf, y), tV(buf, y));
    }
  };
  if constexpr (kDma)
    run_groups_dma<NB, true>(nb, issue_dma, body);
  else
    run_groups<1, NB>(nb, issue_regs, put_regs, body);

  // The waves of a tile combine: accumulators through the staging arrays (one per wave), then one record per draft.
  uint16_t* const mine = wave == 0 ? sK0 : wave == 1 ? sK1 : wave == 2 ? sV0 : sV1;
  {
    float* p = reinterpret_cast<float*>(mine) + c32 * (D + 2);
#pragma unroll
    for (int dc = 0; dc < G::DC; ++dc) {
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int d = 32 * dc + 4 * g + acc_row0(e);
        if (d < D) p[d] = st.acc[dc][e];
      }
    }
    const float l = half_sum(st.l);
    if (g == 0) {
      s_ml[wave][0][c32] = st.m;
      s_ml[wave][1][c32] = l;
    }
  }
  __syncthreads();
  float* out = a.part + ((int64_t)(b * a.H + h) * (a.n_chunks + 1) + c) * a.T * REC;
  for (int x = tid; x < a.T * D; x += 256) {
    const int q = x / D, d = x % D, tile = q / 32, r = q % 32;
    float M = -INFINITY;
#pragma unroll
    for (int s = 0; s < SHARES; ++s) M = fmaxf(M, s_ml[s * QT + tile][0][r]);
    const float mu = M == -INFINITY ? 0.f : M;
    float A = 0.f, L = 0.f;
#pragma unroll
    for (int s = 0; s < SHARES; ++s) {
      const int w = s * QT + tile;
      const uint16_t* arr = w == 0 ? sK0 : w == 1 ? sK1 : w == 2 ? sV0 : sV1;
      const float f = fast_exp2(s_ml[w][0][r] - mu);
      A = __builtin_fmaf(f, reinterpret_cast<const float*>(arr)[r * (D + 2) + d], A);
      L = __builtin_fmaf(f, s_ml[w][1][r], L);
    }
    out[q * REC + d] = A;
    if (d == 0) {
      out[q * REC + D] = M;
      // A negative sum marks what is no draft.
      out[q * REC + D + 1] = drafts && !s_set[q] ? -1.f : L;
    }
  }
}

// One wave per (sequence, head, draft), four to a workgroup: merges the live chunks' records and the drafts' own.
template <int D, class E>
__global__ __launch_bounds__(256) void tree_merge_kernel(const TreeArgs a) {
  constexpr int REC = tree_record_floats(D);
  constexpr int DPL = (D + 63) / 64;
  const int h = blockIdx.y, b = blockIdx.z, lane = threadIdx.x & 63;
  const int qi = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (qi >= a.T) return;
  const int64_t stride = (int64_t)a.T * REC;
  const float* part = a.part + (int64_t)(b * a.H + h) * (a.n_chunks + 1) * stride + qi * REC;
  int nc[kMaxDecodeSegs], total = 1;  // (the drafts' own record is item 0)
  for (int s = 0; s < kMaxDecodeSegs; ++s) {
    nc[s] = s < a.n_seg ? (tree_live(a, a.seg[s], b, h) + a.chunk_keys - 1) / a.chunk_keys : 0;
    total += nc[s];
  }
  auto chunk_of = [&](int i) {
    if (i == 0) return a.n_chunks;
    i -= 1;
    for (int s = 0; s < a.n_seg; ++s) {
      if (i < nc[s]) return a.seg[s].chunk_base + i;
      i -= nc[s];
    }
    return a.n_chunks;
  };
  float M = -INFINITY;
  bool none = false;
  for (int i0 = 0; i0 < total; i0 += 64) {
    const int i = i0 + lane;
    if (i < total) {
      const float* r = part + chunk_of(i) * stride;
      M = fmaxf(M, r[D]);
      if (i == 0) none = r[D + 1] < 0.f;
    }
  }
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) M = fmaxf(M, __shfl_xor(M, o));
  none = __builtin_amdgcn_readfirstlane((int)none) != 0;
  const float mu = M == -INFINITY ? 0.f : M;
  float L = 0.f, A[DPL];
#pragma unroll
  for (int x = 0; x < DPL; ++x) A[x] = 0.f;
  for (int i0 = 0; i0 < total; i0 += 64) {
    const int i = imin(i0 + lane, total - 1), c = chunk_of(i);
    const float* r = part + c * stride;
    const float f = i0 + lane < total ? fast_exp2(r[D] - mu) : 0.f;
    L += f * r[D + 1];
    const int n = imin(64, total - i0);
    for (int j0 = 0; j0 < n; j0 += 8) {
      float x[8][DPL], fj[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const int j = imin(j0 + u, n - 1);
        fj[u] = j0 + u < n ? __shfl(f, j) : 0.f;
        const float* rj = part + __shfl(c, j) * stride;
#pragma unroll
        for (int y = 0; y < DPL; ++y) x[u][y] = D % 64 == 0 || lane + 64 * y < D ? rj[lane + 64 * y] : 0.f;
      }
#pragma unroll
      for (int u = 0; u < 8; ++u)
#pragma unroll
        for (int y = 0; y < DPL; ++y) A[y] = __builtin_fmaf(fj[u], x[u][y], A[y]);
    }
  }
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) L += __shfl_xor(L, o);
  const float inv = L > 0.f && !none ? 1.f / L : 0.f;
  uint16_t* row = a.out + (((int64_t)b * a.T + qi) * a.H + h) * D;
#pragma unroll
  for (int y = 0; y < DPL; ++y) {
    const int d = lane + 64 * y;
    const float o = none ? 0.f : A[y] * inv;
    if (D % 64 == 0 || d < D) row[d] = (uint16_t)E::pack2(o, o);
  }
}

int tree_chunk_keys(int B, int H, int D, int T, int n_seg, const int64_t* scan) {
  const int step = tree_group(D) * kBlock;
  int64_t keys = 0;
  for (int s = 0; s < n_seg; ++s) keys += scan[s];
  // Longer chunks write fewer records, shorter ones fill the chip.
  int chunk = 512;
  while (chunk > step && (int64_t)B * H * ((keys + chunk - 1) / chunk) < 1024) chunk /= 2;
  while (chunk < 4096 && (int64_t)B * H * ((keys + 2 * chunk - 1) / (2 * chunk)) >= 2048) chunk *= 2;
  return imax(chunk, step);
}

template <int D, class E>
static hipError_t launch_t(const TreeArgs& a, hipStream_t stream) {
  const dim3 grid(a.n_chunks + 1, a.H, a.B), block(256);
  const size_t lds = a.bias ? (a.s.far + 1) * sizeof(float) : 0;
  if (a.T <= 32)
    hipLaunchKernelGGL((tree_partial_kernel<D, E, 1>), grid, block, lds, stream, a);
  else
    hipLaunchKernelGGL((tree_partial_kernel<D, E, 2>), grid, block, lds, stream, a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL((tree_merge_kernel<D, E>), dim3((a.T + 3) / 4, a.H, a.B), block, 0, stream, a);
  return hipGetLastError();
}

hipError_t launch_tree(const TreeArgs& a, int D, int is_f16, hipStream_t stream) {
#define SPS_CASE(DD) \
  case DD:           \
    return is_f16 ? launch_t<DD, ElemF16>(a, stream) : launch_t<DD, ElemBF16>(a, stream);
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
