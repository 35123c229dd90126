// Attention of up to 64 drafted tokens per sequence (a tree, a chain, or one token) over up to 3 variable-length KV
// segments and the drafts' own ancestors, gfx950.
//
// Draft i sees every live key of the segments, its ancestors among the drafts and itself. The positions that a bias by
// distance uses run through the segments in their order; a draft's is the number of live keys plus its depth.
//
// Split over the keys: one workgroup per chunk of one segment and (sequence, head); the first chunk's also takes the
// drafts among themselves. Each writes a partial record (accumulator, maximum, sum) per draft, and a second kernel
// merges them; a row of a single chunk goes straight to the outputs (tree_whole_rows). The pass is bound by HBM: every key and value is read once, 4 D bytes against 4 D T products, so at
// T = 64 the matrix cores need a fifth of the time the bytes do. What counts is bytes in flight: a wave streams 32-key
// blocks of its own through registers, loading ahead, passes each through LDS tiles of its own into the layouts of the
// products, and meets the other waves only at the end. (Groups of blocks staged by direct global -> LDS loads with a
// barrier per group: 64 sequences x 16 heads of ~2300 keys, 16 drafts, D = 64, 124 us; now 96 us, 6.3 TB/s, and 89 us
// for one token.)
// Products and softmax as the forward's (attn_fwd.hpp): S^T = K Q^T, a lane holds one draft, so maximum and sum are the
// lane's own. The buffer descriptors cover the chunk's live rows alone: rows past the live length read as zeros,
// whatever the cache holds there, and offsets stay small however long the cache.
#include "tree_kernels.hpp"
#include "wave_tile.hpp"

namespace sps {

__device__ __forceinline__ int tree_live(const TreeArgs& a, const TreeSeg& sg, int b, int h) {
  if (sg.scan == 0) return 0;
  const int64_t i = sg.len_per_head ? (int64_t)b * a.H + h : b;
  const int64_t n = sg.len_i64 ? reinterpret_cast<const int64_t*>(sg.len)[i]
                               : (int64_t) reinterpret_cast<const int32_t*>(sg.len)[i];
  return n < 0 ? 0 : n > sg.scan ? sg.scan : (int)n;
}

// QW: tiles of 32 drafts a wave holds; TS: tiles that are split over the waves instead (D = 256, whose registers hold
// one: each block is then loaded by two waves). At D = 128 two tiles in one wave cost half the waves per SIMD and still
// win (32 x 8 rows of ~2300 keys, 64 drafts, 106 -> 92 us).
template <int D>
constexpr int tree_tiles_in_wave() { return D <= 128 ? 2 : 1; }
// Blocks a wave holds in registers, loaded ahead, and waves per SIMD. More waves with one block each beat fewer with
// several (64 x 16 rows, D = 64, one token, capped: three waves of one block 98 us, two of three 103, two of four 107).
template <int D, int QW>
constexpr int tree_stages() { return D == 128 && QW == 2 ? 2 : 1; }
template <int D, int QW>
constexpr int tree_waves() { return D <= 64 ? (QW == 1 ? 3 : 2) : D == 128 ? (QW == 1 ? 2 : 1) : 1; }

// CHANGED: scores are capped or biased.
template <int D, class E, int QW, int TS, bool CHANGED>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(tree_waves<D, QW>(), 8))) void tree_partial_kernel(
    const TreeArgs a) {
  using W = WaveTile<D>;
  constexpr int DC = TileGeom<D>::DC, S = tree_stages<D, QW>();
  constexpr int TE = kBlock * W::RS;
  constexpr int SHARES = 4 / TS;  // waves that share one tile's blocks
  constexpr int REC = tree_record_floats(D);
  // Per wave a tile of keys and one of values; at the end 32 x D accumulators.
  constexpr int AS = D + 4;  // floats per row of them
  constexpr int WE = 2 * TE > 64 * AS ? 2 * TE : 64 * AS;
  __shared__ __attribute__((aligned(16))) uint16_t s_tile[4][WE];
  __shared__ uint64_t s_set[kMaxDrafts];
  __shared__ float s_m[4][32], s_l[4][32], s_f[4][32];

  // Workgroups go round-robin to the XCDs: chunk by chunk over all rows, so that no XCD gets the same chunks (the first
  // are always live, the last seldom) of every row.
  const int c = (int)(blockIdx.x / (unsigned)(a.B * a.H)), bh = (int)blockIdx.x - c * a.B * a.H;
  const int b = bh / a.H, h = bh - b * a.H;
  const int tid = threadIdx.x, lane = tid & 63, wave = wave_uniform(tid >> 6);
  const int g = lane >> 5, c32 = lane & 31;
  const int tile0 = TS == 2 ? wave & 1 : 0, share = wave / TS;
  const bool first = c == 0;  // with the drafts among themselves
  const bool bias = CHANGED && a.bias;

  // The chunk's rows [0, rows); `place`: the position of its first key, `past`: live keys of all segments.
  const uint16_t *k = a.dk, *v = a.dv;
  int64_t kst = 0, vst = 0;
  int rows = 0, place = 0, past = 0;
  if (c < a.n_chunks) {
    int si = 0;
    while (si + 1 < a.n_seg && c >= a.seg[si + 1].chunk_base) ++si;
    const TreeSeg& sg = a.seg[si];
    const int t0 = (c - sg.chunk_base) * a.chunk_keys;
    const int live = tree_live(a, sg, b, h);
    rows = imax(imin(live - t0, a.chunk_keys), 0);
    if (rows == 0 && !first) return;
    k = sg.k + b * sg.ksb + h * sg.ksh + t0 * sg.kst;
    v = sg.v + b * sg.vsb + h * sg.vsh + t0 * sg.vst;
    kst = sg.kst;
    vst = sg.vst;
    place = t0;
    if (bias) {
      for (int s = 0; s < a.n_seg; ++s) {
        const int n = s == si ? live : tree_live(a, a.seg[s], b, h);
        past += n;
        if (s < si) place += n;
      }
    }
  }
  rows = wave_uniform(rows);
  const int nb = (rows + kBlock - 1) / kBlock;
  const int mine = nb > share ? (nb - share + SHARES - 1) / SHARES : 0;  // blocks share, share + SHARES, ...

  // The lane's drafts' queries (zeros past the last).
  u32x4_t qf[QW][D / 16];
#pragma unroll
  for (int x = 0; x < QW; ++x) {
    const int qi = (tile0 + x) * 32 + c32;
    const BufRsrc q_src = make_rsrc(a.q + b * a.sq.b + h * a.sq.h, (uint32_t)((int64_t)(a.T - 1) * a.sq.n * 2 + D * 2));
    // (a row past the last draft: past the range, whatever the rows' stride)
    const uint32_t at = qi < a.T ? (uint32_t)(qi * a.sq.n * 2) + 16 * g : 0x80000000u;
#pragma unroll
    for (int y = 0; y < D / 16; ++y) qf[x][y] = buf_load_b128(q_src, at + 32 * y);
  }
  // Every wave loads S blocks ahead, always: blocks past the last lie past the descriptors' range (or, with rows that
  // overlap, in it) and are never used, and the compiler can count the loads in flight.
  const BufRsrc k_src = make_rsrc(k, rows ? (uint32_t)((int64_t)(rows - 1) * kst * 2 + D * 2) : 0u);
  const BufRsrc v_src = make_rsrc(v, rows ? (uint32_t)((int64_t)(rows - 1) * vst * 2 + D * 2) : 0u);
  const uint32_t k_row = (uint32_t)(kst * 2), v_row = (uint32_t)(vst * 2);
  const uint32_t r0 = (uint32_t)(lane / W::CPR), piece = (uint32_t)(lane % W::CPR) * 16u;
  W rk[S], rv[S];
  auto issue = [&](int j, int s) {
    const uint32_t r = (uint32_t)((share + j * SHARES) * kBlock) + r0;
    rk[s].load(k_src, r * k_row + piece, k_row);
    rv[s].load(v_src, r * v_row + piece, v_row);
  };
#pragma unroll
  for (int s = 0; s < S; ++s) issue(s, s);

  float* lut = nullptr;
  float slope2 = 0.f;
  if (bias) {
    // Table bias of distances 0 .. far (the last also of every greater one).
    lut = dynamic_lds();
    if (a.s.slopes) slope2 = a.s.slopes[h] * kLog2e;
    for (int n = tid; n <= a.s.far; n += 256) {
      float x = a.s.table ? table_entry(a.s, n < a.s.far ? a.s.bucket[n] : a.s.buckets - 1, h) : 0.f;
      lut[n] = x < kHidden ? -INFINITY : x * kLog2e;
    }
  }
  if (bias || first) {
    if (wave == 0) s_set[lane] = ancestor_set(a.parents, a.parents_i64, b * a.parents_sb, a.T, lane);
    __syncthreads();
  }
  int depth[QW];
#pragma unroll
  for (int x = 0; x < QW; ++x)
    depth[x] = bias ? imax(__builtin_popcountll(s_set[(tile0 + x) * 32 + c32]) - 1, 0) : 0;

  float m_run[QW], l_run[QW];
  f32x16_t acc[QW][DC];
#pragma unroll
  for (int x = 0; x < QW; ++x) {
    m_run[x] = -INFINITY;
    l_run[x] = 0.f;
#pragma unroll
    for (int dc = 0; dc < DC; ++dc) acc[x][dc] = f32x16_t{};
  }
  const float scale2 = a.s.scale2, cap2 = a.s.cap2, cap_in = a.s.cap_in;
  const int far = a.s.far;
  uint16_t *const kt = s_tile[wave], *const vt = kt + TE;
  if constexpr (TileGeom<D>::DPAD > D) {
    for (int i = lane; i < 2 * kBlock; i += 64) {
      const u32x4_t z = {0u, 0u, 0u, 0u};
#pragma unroll
      for (int y = D; y < TileGeom<D>::DPAD; y += 8) lds_write_b128(kt + i * W::RS + y, z);
    }
  }

  // The staged block's products with the lane's drafts, change(scores, tile) of them (in the log2 domain, hidden ones
  // -inf), softmax, and the products with the values.
  auto block = [&](auto change) {
    f32x16_t sc[QW];
#pragma unroll
    for (int y = 0; y < D / 16; ++y) {
      const u32x4_t f = lds_read_b128(kt + c32 * W::RS + 16 * y + 8 * g);
#pragma unroll
      for (int x = 0; x < QW; ++x) sc[x] = E::mfma(f, qf[x][y], y == 0 ? f32x16_t{} : sc[x]);
    }
    uint32_t pk[QW][8];
#pragma unroll
    for (int x = 0; x < QW; ++x) {
      if (CHANGED && a.cap) {
#pragma unroll
        for (int e = 0; e < 16; ++e)
          sc[x][e] = __builtin_fmaf(__builtin_amdgcn_rcpf(1.f + fast_exp2(sc[x][e] * cap_in)), -2.f * cap2, cap2);
      } else {
#pragma unroll
        for (int e = 0; e < 16; ++e) sc[x][e] *= scale2;
      }
      change(sc[x], x);
      float mx = max3f(sc[x][0], sc[x][1], sc[x][2]);
#pragma unroll
      for (int e = 3; e < 15; e += 2) mx = max3f(mx, sc[x][e], sc[x][e + 1]);
      mx = half_max(__builtin_elementwise_maximum(mx, sc[x][15]));
      if (wave_any(mx > m_run[x])) {
        const float m_new = mx > m_run[x] ? mx : m_run[x];
        const float alpha = mx > m_run[x] ? fast_exp2(m_run[x] - m_new) : 1.f;
        l_run[x] *= alpha;
#pragma unroll
        for (int dc = 0; dc < DC; ++dc) acc[x][dc] *= alpha;
        m_run[x] = m_new;
      }
      const float negm = m_run[x] == -INFINITY ? 0.f : -m_run[x];
      float sum = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float p0 = fast_exp2(sc[x][2 * e] + negm), p1 = fast_exp2(sc[x][2 * e + 1] + negm);
        pk[x][e] = E::pack2(p0, p1);
        sum += p0 + p1;
      }
      l_run[x] += sum;
    }
#pragma unroll
    for (int dc = 0; dc < DC; ++dc) {
#pragma unroll
      for (int kh = 0; kh < 2; ++kh) {
        const u32x4_t f = lds_frag_tr(vt, W::RS, 16 * kh, 32 * dc, lane);
#pragma unroll
        for (int x = 0; x < QW; ++x) {
          const u32x4_t pf = {pk[x][4 * kh], pk[x][4 * kh + 1], pk[x][4 * kh + 2], pk[x][4 * kh + 3]};
          acc[x][dc] = E::mfma(f, pf, acc[x][dc]);
        }
      }
    }
  };
  // Bias of element e at distance n.
  auto add_bias = [&](float s, int n) { return s + __builtin_fmaf(-slope2, (float)n, lut[imin(n, far)]); };
  for (int j0 = 0; j0 < mine; j0 += S) {
#pragma unroll
    for (int s = 0; s < S; ++s) {
      const int j = j0 + s, i = share + j * SHARES;
      rk[s].store(kt, lane);
      rv[s].store(vt, lane);
      issue(j + S, s);
      wave_lds_order();
      if (j < mine) {
        const int t = i * kBlock + 4 * g;  // the chunk's row of element 0
        block([&](f32x16_t& sc, int x) {
          if (bias) {
            const int d = past + depth[x] - place - t;  // distance of element 0
            // The smallest distance of the block, over lanes and rows: where it reaches `far` the table adds one value.
            if (past - place - i * kBlock - 31 >= far) {
              const float base = __builtin_fmaf(-slope2, (float)d, lut[far]);
#pragma unroll
              for (int e = 0; e < 16; ++e) sc[e] += __builtin_fmaf(slope2, (float)acc_row0(e), base);
            } else {
#pragma unroll
              for (int e = 0; e < 16; ++e) sc[e] = add_bias(sc[e], imax(d - acc_row0(e), 0));  // (negative: past the live rows)
            }
          }
          if (rows - i * kBlock < kBlock) {
#pragma unroll
            for (int e = 0; e < 16; ++e) sc[e] = t + acc_row0(e) < rows ? sc[e] : -INFINITY;
          }
        });
      }
      wave_lds_order();
    }
  }
  if (first) {
    // The drafts among themselves: their last blocks to the waves with the fewest of the chunk's.
    const int i = SHARES - 1 - share;
    if (i * kBlock < a.T) {
      const BufRsrc dk_src = make_rsrc(a.dk + b * a.sdk.b + h * a.sdk.h, (uint32_t)((int64_t)(a.T - 1) * a.sdk.n * 2 + D * 2));
      const BufRsrc dv_src = make_rsrc(a.dv + b * a.sdv.b + h * a.sdv.h, (uint32_t)((int64_t)(a.T - 1) * a.sdv.n * 2 + D * 2));
      const uint32_t dk_row = (uint32_t)(a.sdk.n * 2), dv_row = (uint32_t)(a.sdv.n * 2), r = (uint32_t)(i * kBlock) + r0;
      rk[0].load(dk_src, r * dk_row + piece, dk_row);
      rv[0].load(dv_src, r * dv_row + piece, dv_row);
      rk[0].store(kt, lane);
      rv[0].store(vt, lane);
      wave_lds_order();
      // Rows that are no draft: zeros, so that whatever they hold stays out of the zero-weighted products.
      if (!s_set[i * kBlock + c32]) {
        for (int y = 8 * g; y < D; y += 16) lds_write_b128(vt + c32 * W::RS + y, u32x4_t{0u, 0u, 0u, 0u});
      }
      wave_lds_order();
      block([&](f32x16_t& sc, int x) {
        const uint64_t own = s_set[(tile0 + x) * 32 + c32];
        const int j0 = i * kBlock + 4 * g;
        if (bias) {
#pragma unroll
          for (int e = 0; e < 16; ++e)
            sc[e] = add_bias(sc[e], imax(depth[x] - (__builtin_popcountll(s_set[j0 + acc_row0(e)]) - 1), 0));
        }
#pragma unroll
        for (int e = 0; e < 16; ++e) sc[e] = (own >> (j0 + acc_row0(e))) & 1 ? sc[e] : -INFINITY;
      });
      wave_lds_order();
    }
  }

  // The waves combine, tile by tile: accumulators through the waves' LDS, each wave's weight once per draft, then one
  // record per draft, 16 bytes a thread; or, of a single chunk, the outputs.
  const bool whole = a.n_chunks <= 1;
  float* out = a.part + ((int64_t)bh * imax(a.n_chunks, 1) + c) * a.T * REC;
#pragma unroll
  for (int x = 0; x < QW; ++x) {
    if (x > 0) __syncthreads();
    float* p = reinterpret_cast<float*>(s_tile[wave]) + c32 * AS;
#pragma unroll
    for (int dc = 0; dc < DC; ++dc) {
#pragma unroll
      for (int i4 = 0; i4 < 4; ++i4) {
        const int d = 32 * dc + 8 * i4 + 4 * g;
        const f32x4_t y = {acc[x][dc][4 * i4], acc[x][dc][4 * i4 + 1], acc[x][dc][4 * i4 + 2], acc[x][dc][4 * i4 + 3]};
        if (d < D) *reinterpret_cast<f32x4_t*>(p + d) = y;
      }
    }
    const float l = half_sum(l_run[x]);
    if (g == 0) {
      s_m[wave][c32] = m_run[x];
      s_l[wave][c32] = l;
    }
    __syncthreads();
    const int q0 = x * 32, drafts = imin(a.T - q0, 32 * TS);  // (TS tiles at once)
    if (tid < drafts) {
      const int tile = tid / 32, r = tid % 32;
      float M = -INFINITY, L = 0.f;
#pragma unroll
      for (int s = 0; s < SHARES; ++s) M = fmaxf(M, s_m[s * TS + tile][r]);
      const float mu = M == -INFINITY ? 0.f : M;
#pragma unroll
      for (int s = 0; s < SHARES; ++s) {
        const float f = fast_exp2(s_m[s * TS + tile][r] - mu);
        s_f[s * TS + tile][r] = f;
        L = __builtin_fmaf(f, s_l[s * TS + tile][r], L);
      }
      if (whole) {
        const float inv = L > 0.f ? 1.f / L : 0.f;
#pragma unroll
        for (int s = 0; s < SHARES; ++s) s_f[s * TS + tile][r] *= inv;
      } else {
        out[(q0 + tid) * REC + D] = M;
        out[(q0 + tid) * REC + D + 1] = first && !s_set[q0 + tid] ? -1.f : L;  // a negative sum marks what is no draft
      }
    }
    __syncthreads();
    for (int i = tid; i < drafts * (D / 4); i += 256) {
      const int ql = i / (D / 4), d = (i % (D / 4)) * 4, tile = ql / 32, r = ql % 32;
      f32x4_t A = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int s = 0; s < SHARES; ++s) {
        const int w = s * TS + tile;
        const float f = s_f[w][r];
        const f32x4_t y = *reinterpret_cast<const f32x4_t*>(reinterpret_cast<const float*>(s_tile[w]) + r * AS + d);
#pragma unroll
        for (int e = 0; e < 4; ++e) A[e] = __builtin_fmaf(f, y[e], A[e]);
      }
      if (whole) {
        if (!s_set[q0 + ql]) A = f32x4_t{0.f, 0.f, 0.f, 0.f};
        *reinterpret_cast<u32x2_t*>(a.out + (((int64_t)b * a.T + q0 + ql) * a.H + h) * D + d) =
            u32x2_t{E::pack2(A[0], A[1]), E::pack2(A[2], A[3])};
      } else {
        *reinterpret_cast<f32x4_t*>(out + (q0 + ql) * REC + d) = A;
      }
    }
  }
}

// Merges the live chunks' records of every draft. A chain of latencies: lengths and the first records are loaded in one
// round trip (the records of chunks that turn out not to be live are dropped), D / 4 lanes a draft with 16 bytes each
// and no exchange between lanes. WIDE (many chunks): a whole workgroup per draft, its lane groups over the chunks.
template <int D, class E, bool WIDE>
__global__ __launch_bounds__(256) void tree_merge_kernel(const TreeArgs a) {
  constexpr int REC = tree_record_floats(D);
  constexpr int LPQ = D / 4, GROUPS = 256 / LPQ, AHEAD = 8;
  __shared__ float s_m[GROUPS], s_l[GROUPS];
  __shared__ __attribute__((aligned(16))) float s_a[GROUPS][D];
  const int tid = threadIdx.x, group = tid / LPQ, d0 = (tid % LPQ) * 4;
  const int64_t id = WIDE ? (int64_t)blockIdx.x : (int64_t)blockIdx.x * GROUPS + group;
  if (id >= (int64_t)a.B * a.H * a.T) return;  // (never where the workgroup meets below)
  const int bh = (int)(id / a.T), q = (int)(id - (int64_t)bh * a.T), b = bh / a.H, h = bh - b * a.H;
  const int chunks = imax(a.n_chunks, 1), step = WIDE ? GROUPS : 1, start = WIDE ? group : 0;
  const int64_t stride = (int64_t)a.T * REC;
  const float* part = a.part + (int64_t)bh * chunks * stride + q * REC;
  f32x4_t x[AHEAD];
  f32x2_t ml[AHEAD];
  auto load = [&](int u, int c) {
    const float* r = part + c * stride;
    x[u] = *reinterpret_cast<const f32x4_t*>(r + d0);
    ml[u] = *reinterpret_cast<const f32x2_t*>(r + D);
  };
#pragma unroll
  for (int u = 0; u < AHEAD; ++u) load(u, imin(start + u * step, chunks - 1));
  int nc[kMaxDecodeSegs];
#pragma unroll
  for (int s = 0; s < kMaxDecodeSegs; ++s)
    nc[s] = s < a.n_seg ? (tree_live(a, a.seg[s], b, h) + a.chunk_keys - 1) / a.chunk_keys : 0;
  auto live = [&](int c) {
    bool on = c == 0;  // (always has a record)
#pragma unroll
    for (int s = 0; s < kMaxDecodeSegs; ++s)
      on = on || (s < a.n_seg && c >= a.seg[s].chunk_base && c < a.seg[s].chunk_base + nc[s]);
    return on && c < chunks;
  };
  f32x4_t A = {0.f, 0.f, 0.f, 0.f};
  float M = -INFINITY, L = 0.f;
  bool none = false;
  for (int c0 = start; c0 < chunks; c0 += AHEAD * step) {
    bool on[AHEAD];
    float m_new = M;
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      const int c = c0 + u * step;
      on[u] = live(c);
      if (c0 != start && on[u]) load(u, c);
    }
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) m_new = on[u] ? fmaxf(m_new, ml[u][0]) : m_new;
    if (c0 == 0) none = ml[0][1] < 0.f;
    const float mu = m_new == -INFINITY ? 0.f : m_new, keep = fast_exp2(M - mu);
    A *= keep;
    L *= keep;
    M = m_new;
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      if (on[u]) {
        const float f = fast_exp2(ml[u][0] - mu);
#pragma unroll
        for (int e = 0; e < 4; ++e) A[e] = __builtin_fmaf(f, x[u][e], A[e]);
        L = __builtin_fmaf(f, ml[u][1], L);
      }
    }
  }
  if constexpr (WIDE) {
    *reinterpret_cast<f32x4_t*>(&s_a[group][d0]) = A;
    if (d0 == 0) {
      s_m[group] = M;
      s_l[group] = none ? -1.f : L;
    }
    __syncthreads();
    if (group > 0) return;
    none = s_l[0] < 0.f;
    M = -INFINITY;
    for (int i = 0; i < GROUPS; ++i) M = fmaxf(M, s_m[i]);
    const float mu = M == -INFINITY ? 0.f : M;
    A = f32x4_t{0.f, 0.f, 0.f, 0.f};
    L = 0.f;
    for (int i = 0; i < GROUPS; ++i) {
      const float f = fast_exp2(s_m[i] - mu);
      const f32x4_t y = *reinterpret_cast<const f32x4_t*>(&s_a[i][d0]);
#pragma unroll
      for (int e = 0; e < 4; ++e) A[e] = __builtin_fmaf(f, y[e], A[e]);
      L = __builtin_fmaf(f, s_l[i], L);
    }
  }
  const float inv = L > 0.f && !none ? 1.f / L : 0.f;
  if (none) A = f32x4_t{0.f, 0.f, 0.f, 0.f};
  uint16_t* row = a.out + (((int64_t)b * a.T + q) * a.H + h) * D + d0;
  *reinterpret_cast<u32x2_t*>(row) = u32x2_t{E::pack2(A[0] * inv, A[1] * inv), E::pack2(A[2] * inv, A[3] * inv)};
}

// Longer chunks write fewer records and meet fewer ends, shorter ones fill the chip (MI355X, us a call):
//  - up to 512 keys for one or two drafts, whose records are small: 16 x 12 rows of ~2300 keys, D = 64, 512 / 1024 keys
//    25.3 / 27.1; 64 x 16 rows 93.5 / 93.8.
//  - up to 1024 for up to eight (8 x 32 rows, D = 32, 1024 / 2048 keys 19.8 / 20.6), 2048 for more (64 x 16 rows, 16
//    drafts, 1024 / 2048 / 4096 keys 110.2 / 105.9 / 110.2; 64 drafts 147.9 / 137.1 / 141.9).
//  - shorter where that leaves fewer workgroups than CUs (12 rows of 4000 keys, 8 drafts, 128 / 256 / 512 keys 11.3 /
//    11.9 / 12.5; 16 rows of 16000 keys, D = 128, 61 drafts, 512 / 1024 / 2048 keys 45.5 / 39.2 / 48.8).
int tree_chunk_keys(int B, int H, int T, int n_seg, const int64_t* scan) {
  auto workgroups = [&](int chunk) {
    int64_t n = 0;
    for (int s = 0; s < n_seg; ++s) n += (scan[s] + chunk - 1) / chunk;
    return n * B * H;
  };
  int chunk = T <= 2 ? 512 : T <= 8 ? 1024 : 2048;
  while (chunk > 4 * kBlock && workgroups(chunk) < 256) chunk /= 2;
  return chunk;
}

// No merge, no second launch; the rows' lengths are not evened out. For keys in one segment (MI355X, us a call, chunks and
// merge / whole rows; live lengths 1/2 to 1 of the scan below 2048 keys, 1/8 to 1 from there):
//  - up to 512 keys always (16 rows, D = 64, one draft, 256 keys 8.8 / 5.5, 512 8.7 / 6.8; 32 rows, D = 128, 61 drafts,
//    512 17.7 / 16.9), 1024 from 128 rows (16 drafts 13.2 / 12.0; 32 rows, D = 128, one draft 11.0 / 14.0);
//  - from 256 rows 2048 (D = 128, one draft 37 / 31), which few drafts' calls no longer gain from beyond (4096: 59 / 60);
//  - with more than eight drafts 4096 (256 rows, D = 64, 16 drafts 32.0 / 32.0, 61 44 / 40; 1024 rows 113 / 108 and
//    147 / 124), and 8192 from 512 rows (16 drafts 114 / 112, 61 140 / 125).
bool tree_whole_rows(int B, int H, int T, int n_seg, const int64_t* scan) {
  const int64_t rows = (int64_t)B * H;
  int64_t keys = 0;
  for (int s = 0; s < n_seg; ++s) {
    if (keys && scan[s]) return false;
    keys += scan[s];
  }
  const int64_t most = rows < 128 ? 512 : rows < 256 ? 1024 : T <= 8 ? 2048 : rows < 512 ? 4096 : 8192;
  return keys <= most;
}

template <int D, class E, bool CHANGED>
static void launch_partial(const TreeArgs& a, hipStream_t stream) {
  const dim3 grid((unsigned)imax(a.n_chunks, 1) * a.B * a.H), block(256);
  const size_t lds = a.bias ? (a.s.far + 1) * sizeof(float) : 0;
  if (a.T <= 32)
    hipLaunchKernelGGL((tree_partial_kernel<D, E, 1, 1, CHANGED>), grid, block, lds, stream, a);
  else
    hipLaunchKernelGGL((tree_partial_kernel<D, E, tree_tiles_in_wave<D>(), 2 / tree_tiles_in_wave<D>(), CHANGED>), grid, block, lds, stream, a);
}

template <int D, class E>
static hipError_t launch_t(const TreeArgs& a, hipStream_t stream) {
  if (a.cap || a.bias)
    launch_partial<D, E, true>(a, stream);
  else
    launch_partial<D, E, false>(a, stream);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || a.n_chunks <= 1) return e;
  const int64_t drafts = (int64_t)a.B * a.H * a.T;
  constexpr int kGroups = 256 / (D / 4);
  // A lane group walks its chunks eight at a time; past that a workgroup shares them.
  if (a.n_chunks <= 8)
    hipLaunchKernelGGL((tree_merge_kernel<D, E, false>), dim3((unsigned)((drafts + kGroups - 1) / kGroups)), dim3(256), 0, stream, a);
  else
    hipLaunchKernelGGL((tree_merge_kernel<D, E, true>), dim3((unsigned)drafts), dim3(256), 0, stream, a);
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
