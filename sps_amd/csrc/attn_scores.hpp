// Scores changed between their product and the softmax: a tanh cap, a bias by distance, a prefix that every
// query sees. The attention kernels take one of these as a template parameter; PlainScores leaves them as they are.
//
// For query q and key k of head h, with x = sm_scale * (q . k) and n = max(q - k, 0):
//   s = cap * tanh(x / cap) [or x] - slope[h] * n [+ table[bucket(n), h]],
// in the log2 domain of the softmax (everything times log2 e). With r = 1 / (1 + exp2(2 log2(e) x / cap)):
//   cap * tanh(x / cap) = cap - 2 cap r,   d/dx = 1 - tanh^2 = 4 r (1 - r),
// one exponential and one reciprocal (both of the hardware, 1 ulp) per score; exp2 overflowing to infinity gives
// r = 0 and one flushed to zero r = 1, the two limits. The difference cap - 2 cap r carries an absolute error of
// about cap * 2^-23, in a score: below 1e-5 for caps up to 80.
//
// The bias depends on the distance alone, so a 32 x 32 block of pairs holds 63 of them. Three kinds of block:
//  - every distance at least `far`, the first of the last bucket (0 without a table): one linear function of
//    the distance, an FMA per score with constants of the lane and the accumulator row; one constant, in the FMA that
//    scales the scores, without slopes (B4 H16 N2048 D64 with a table, forward 64.6 -> 61.1 us, dK/dV 93.8 -> 89.4);
//  - every key at or past its query (only a prefix shows those): the bias of distance 0;
//  - the others: read from a table in LDS over the distances -kLutPad .. far + kLutPad, built once per workgroup;
//    the lanes of one read hold consecutive distances, so it meets no bank twice.
// Table entries below kHidden (the types' lowest values and -inf among them) hide their pairs.
//
// Rounded to the inputs' type, as with unchanged scores: P and dS for their products, and O, which the backward's
// Delta = rowsum(O * dO) is read from. A concentrated softmax feels the last most: dQ is off by 0.0024 (dense) to 0.0034
// (linear bias, short documents) of its norm in bf16, where its own rounding is 0.0017. Everything else is fp32.
#pragma once
#include "attn_tiles.hpp"

namespace sps {

constexpr int kMaxDistance = 512;    // largest distance a bucket may start at
constexpr float kMinCap = 0x1p-10f, kMaxCap = 0x1p20f;  // caps outside lose the scores to fp32's range or precision
constexpr int kMaxBuckets = 256;
constexpr int kLutPad = 64;          // a block's distances span 63, on either side of [0, far]
constexpr float kHidden = -16384.f;  // (their log-sum-exp would leave fp32 no bits for the scores)
constexpr float kLog2e = 1.4426950408889634f;

constexpr int kFewTiles = 256;       // at most so many tiles of 128 are few, at any head dim

struct BiasedArgs : AttnArgs {
  const void* prefix;  // [B] int32 or int64: leading positions of each row that all its queries see, or null
  int prefix_i64;
  float cap2;          // cap * log2(e)
  float cap_in;        // 2 log2(e) sm_scale / cap
  const float* slopes;  // [H], or null
  const void* table;    // [buckets, H] of table_dtype (0 bf16, 1 f16, 2 f32), strides table_sj, table_sh; or null
  int table_dtype;
  int64_t table_sj, table_sh;
  int buckets, far;     // far: first distance of the last bucket
  float* dtable_part;   // [B, H, dtable_tiles, buckets]: table gradient of each query tile (backward with a table)
  int dtable_tiles;
  uint8_t bucket[kMaxDistance];      // of the distances below far
  uint16_t first[kMaxBuckets];       // first distance of each bucket (of the next one that has any, where it has none)
};

struct PlainScores {
  static constexpr bool kOn = false, kCap = false, kBias = false, kTable = false;
  using Args = AttnArgs;
};

// CAP: capped scores; BIAS: a bias by distance; TABLE: the dQ pass also sums the gradient of the bias table.
template <bool CAP, bool BIAS, bool TABLE = false>
struct ChangedScores {
  static constexpr bool kOn = true, kCap = CAP, kBias = BIAS, kTable = TABLE;
  using Args = BiasedArgs;
};

// The visible prefix of row b, clamped to the row.
__device__ __forceinline__ int row_prefix(const BiasedArgs& a, int b) {
  if (!a.prefix) return 0;
  const int64_t n = a.prefix_i64 ? reinterpret_cast<const int64_t*>(a.prefix)[b]
                                 : (int64_t) reinterpret_cast<const int32_t*>(a.prefix)[b];
  return n < 0 ? 0 : n > a.m.N ? a.m.N : (int)n;
}

// Keys that query q sees and queries that see key k, for a document run [s, e] and a visible prefix. Both bounds of
// both never decrease with the position, as the schedule needs.
__device__ __forceinline__ Interval prefix_keys(int q, int s, int e, int prefix) {
  return Interval{s, imax(q, imin(prefix - 1, e))};
}
__device__ __forceinline__ Interval prefix_queries(int k, int s, int e, int prefix) {
  return Interval{k < prefix ? s : k, e};
}

// Start of a query-stationary (key-stationary) workgroup: q_begin (k_begin), or with a prefix, which the prepass's
// plans do not know, the plan from the lanes' intervals.
template <class M>
__device__ __forceinline__ bool q_start(const typename M::Args& a, const TilePlan& tp, const RowView& row, int b, int qp,
                                        int* s_span, QState& st, int& run_start) {
  if constexpr (M::kOn) {
    if (a.prefix) {
      run_start = 0;
      const int prefix = row_prefix(a, b);
      const bool in = qp < a.m.N;
      st.r0 = in ? prefix_keys(qp, row.run_start(qp), row.run_end(qp, a.m.N), prefix) : Interval{kEmptyLo, kEmptyHi};
      st.r1 = Interval{kEmptyLo, kEmptyHi};
      st.w0 = wave_span_monotone(st.r0);
      st.w1 = wave_span_monotone(st.r1);
      q_plan_from_spans(a.m, s_span, st);
      return false;
    }
  }
  return q_begin(a, tp, row, qp, s_span, st, run_start);
}

template <class M>
__device__ __forceinline__ bool k_start(const typename M::Args& a, const TilePlan& tp, const RowView& row, int b,
                                        int* s_span, KState& st, int& run_end, int wave) {
  if constexpr (M::kOn) {
    if (a.prefix) {
      run_end = 0;
      const int prefix = row_prefix(a, b);
      k_lane_key(a.m, tp.tile, st, wave);
      st.r = st.kvalid ? prefix_queries(st.kp, row.run_start(st.kp), row.run_end(st.kp, a.m.N), prefix)
                       : Interval{kEmptyLo, kEmptyHi};
      st.w = wave_span_monotone(st.r);
      k_plan_from_spans(s_span, st, wave);
      return false;
    }
  }
  return k_begin(a, tp, row, s_span, st, run_end, wave);
}

__device__ __forceinline__ float table_entry(const BiasedArgs& a, int j, int h) {
  const int64_t i = j * a.table_sj + h * a.table_sh;
  if (a.table_dtype == 2) return reinterpret_cast<const float*>(a.table)[i];
  const uint16_t x = reinterpret_cast<const uint16_t*>(a.table)[i];
  return a.table_dtype == 1 ? ElemF16::to_f32(x) : ElemBF16::to_f32(x);
}

// Distances the LDS table covers, and its bytes.
__host__ __device__ __forceinline__ int lut_len(int far) { return far + 2 * kLutPad; }

// Writes the LDS table: entry i (or, REVERSED, lut_len - 1 - i) holds the log2-domain bias of distance i - kLutPad.
// Read after the next barrier.
template <bool REVERSED>
__device__ __forceinline__ void fill_lut(const BiasedArgs& a, int h, float* lut, int tid, int threads) {
  const int len = lut_len(a.far);
  const float slope = a.slopes ? a.slopes[h] : 0.f;
  for (int i = tid; i < len; i += threads) {
    const int n = imax(i - kLutPad, 0);
    float v = 0.f;
    if (a.table) {
      v = table_entry(a, n < a.far ? a.bucket[n] : a.buckets - 1, h);
      if (v < kHidden) v = -INFINITY;
    }
    lut[REVERSED ? len - 1 - i : i] = __builtin_fmaf(-slope, (float)n, v) * kLog2e;
  }
}

// The launch's dynamic LDS: the table of the biases.
__device__ __forceinline__ float* dynamic_lds() {
  extern __shared__ __attribute__((aligned(16))) float s_dynamic[];
  return s_dynamic;
}

// Constants of a workgroup's head.
struct ScoreConsts {
  float scale2;         // sm_scale * log2 e
  float cap2, cap_in;
  float far2, slope2;   // bias of distance n >= far: far2 - slope2 * n
  bool sloped;          // there are slopes
  int far;
};

template <class M>
__device__ __forceinline__ ScoreConsts score_consts(const typename M::Args& a, int h) {
  ScoreConsts c = {a.scale2, 0.f, 0.f, 0.f, 0.f, false, 0};
  if constexpr (M::kCap) {
    c.cap2 = a.cap2;
    c.cap_in = a.cap_in;
  }
  if constexpr (M::kBias) {
    c.far = a.far;
    if (a.slopes) c.slope2 = a.slopes[h] * kLog2e;
    c.sloped = a.slopes != nullptr;
    if (a.table) {
      const float v = table_entry(a, a.buckets - 1, h);
      c.far2 = v < kHidden ? -INFINITY : v * kLog2e;
    }
  }
  return c;
}

// One raw product -> its score plus `add` (which holds cap2 where scores are capped); r of a capped score.
template <class M>
__device__ __forceinline__ float changed(float s, const ScoreConsts& c, float add, float& r) {
  if constexpr (M::kCap) {
    r = __builtin_amdgcn_rcpf(1.f + fast_exp2(s * c.cap_in));
    return __builtin_fmaf(r, -2.f * c.cap2, add);
  } else {
    return __builtin_fmaf(s, c.scale2, add);
  }
}

// Row of accumulator element e inside its lane half's rows.
constexpr int acc_row0(int e) { return 8 * (e >> 2) + (e & 3); }

// Distances of a block: BLOCK_FAR all at least far (and 0), BLOCK_AHEAD all 0, BLOCK_NEAR the others; d0: the
// smallest signed distance (query - key), 62 below the largest.
enum BlockKind : int { BLOCK_FAR, BLOCK_AHEAD, BLOCK_NEAR };
__device__ __forceinline__ BlockKind block_kind(int d0, int far) {
  return d0 >= far ? BLOCK_FAR : d0 + 62 <= 0 ? BLOCK_AHEAD : BLOCK_NEAR;
}

// Scores of a block in the query-stationary layout (lane: query q, element e: key t0 + 4 g + acc_row0(e)), each plus
// add0; `lut` is the reversed table. each(e, r): r of a capped score.
template <class M, class Each>
__device__ __forceinline__ void qs_scores(f32x16_t& sc, const ScoreConsts& c, const float* lut, int q, int t0, int g,
                                          BlockKind kind, float add0, Each each) {
  const float add = M::kCap ? add0 + c.cap2 : add0;
  auto all = [&](auto bias) {
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      float r = 0.f;
      sc[e] = changed<M>(sc[e], c, bias(e), r);
      each(e, r);
    }
  };
  if constexpr (!M::kBias) {
    all([&](int) { return add; });
  } else {
    const int d = q - t0 - 4 * g;  // distance of element 0
    if (kind == BLOCK_NEAR) {
      // Distance d - row sits at lut_len - 1 - (kLutPad + d - row).
      const float* p = lut + (lut_len(c.far) - 1 - kLutPad - d);
      all([&](int e) { return p[acc_row0(e)] + add; });
    } else if (kind == BLOCK_FAR && c.sloped) {
      const float base = __builtin_fmaf(-c.slope2, (float)d, c.far2 + add);
      all([&](int e) { return __builtin_fmaf(c.slope2, (float)acc_row0(e), base); });
    } else {
      const float base = (kind == BLOCK_FAR ? c.far2 : lut[lut_len(c.far) - 1 - kLutPad]) + add;
      all([&](int) { return base; });
    }
  }
}

// The same in the key-stationary layout (lane: key k, element e: query q0 + 4 g + acc_row0(e)), each plus add0(e);
// `lut` is the forward table.
template <class M, class Add, class Each>
__device__ __forceinline__ void ks_scores(f32x16_t& sc, const ScoreConsts& c, const float* lut, int k, int q0, int g,
                                          BlockKind kind, Add add0, Each each) {
  auto all = [&](auto bias) {
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      float r = 0.f;
      sc[e] = changed<M>(sc[e], c, bias(e) + add0(e), r);
      each(e, r);
    }
  };
  const float add = M::kCap ? c.cap2 : 0.f;
  if constexpr (!M::kBias) {
    all([&](int) { return add; });
  } else {
    const int d = q0 + 4 * g - k;  // distance of element 0
    if (kind == BLOCK_NEAR) {
      const float* p = lut + kLutPad + d;
      all([&](int e) { return p[acc_row0(e)] + add; });
    } else if (kind == BLOCK_FAR && c.sloped) {
      const float base = __builtin_fmaf(-c.slope2, (float)d, c.far2 + add);
      all([&](int e) { return __builtin_fmaf(-c.slope2, (float)acc_row0(e), base); });
    } else {
      const float base = (kind == BLOCK_FAR ? c.far2 : lut[kLutPad]) + add;
      all([&](int) { return base; });
    }
  }
}

// The cap's derivative from r.
__device__ __forceinline__ float cap_slope(float r) { return __builtin_fmaf(-4.f * r, r, 4.f * r); }

// Sums of dS by distance, for the gradient of the bias table (dQ pass: dTable[j, h] = sum of dS over the pairs of
// bucket j). The pairs of a near block fall on the 63 diagonals of the block, summed in registers: with the rows of
// the keys zero-padded to 64 lanes (columns in the upper half), each step moves the sums one lane down and adds the
// next row, so after 16 rows lane l holds the diagonal l - 32. Every wave adds them to sums of its own in LDS, which no
// other wave touches: the result does not depend on timing. (LDS additions of the single values take ~150 cycles an
// instruction: dQ, B4 H16 N2048 D64, 181 us against 85 with these.) Blocks of one bucket add up in a register of each
// lane.
constexpr int kTableCopies = kWaves;
template <class M>
struct TableSums {
  float* copy;  // the sums of this wave, by distance + kLutPad
  float* all;
  float far_sum, ahead_sum;
  int far;

  __device__ __forceinline__ void init(const BiasedArgs& a, float* lds, int tid, int wave) {
    if constexpr (M::kTable) {
      far = a.far;
      all = lds;
      copy = lds + wave * lut_len(far);
      far_sum = ahead_sum = 0.f;
      for (int i = tid; i < kTableCopies * lut_len(far); i += 256) lds[i] = 0.f;
    }
  }

  // One row more: the sums move one lane down.
  static __device__ __forceinline__ float next_row(float sums, uint32_t row) {
    const int moved = __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, sums), 0x130, 0xF, 0xF, true);  // wave_shl 1
    return __builtin_bit_cast(float, moved) + __builtin_bit_cast(float, row);
  }

  // q0: the wave's first query.
  __device__ __forceinline__ void add(const f32x16_t& ds, BlockKind kind, int q0, int t0, int lane) {
    if (kind == BLOCK_NEAR) {
      float sums[2];
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        // Rows 16 half + 15 .. 16 half: elements 8 half + 7 .. 8 half, whose lane halves hold rows 4 apart. Swapped
        // against zeros, an element becomes the two rows, each in the upper lanes with zeros below.
        uint32_t row[16];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float v = ds[8 * half + e];
          const auto r = __builtin_amdgcn_permlane32_swap(0u, __builtin_bit_cast(uint32_t, v), false, false);
          row[acc_row0(e)] = r[0];
          row[acc_row0(e) + 4] = r[1];
        }
        float s = __builtin_bit_cast(float, row[15]);
#pragma unroll
        for (int r = 14; r >= 0; --r) s = next_row(s, row[r]);
        sums[half] = s;
      }
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        float* p = copy + (kLutPad + q0 - t0 - 16 * half + lane - 32);
        if (lane > 16) *p += sums[half];  // (lanes 0 .. 16 hold no diagonal)
        // The next addition's addresses are other lanes' of this one: the wave's LDS operations run in order, and the
        // compiler, which sees one lane's addresses only, may not exchange them.
        asm volatile("" ::: "memory");
      }
    } else {
      float s[4] = {ds[0], ds[1], ds[2], ds[3]};
#pragma unroll
      for (int e = 4; e < 16; ++e) s[e & 3] += ds[e];
      const float t = (s[0] + s[1]) + (s[2] + s[3]);
      if (kind == BLOCK_FAR)
        far_sum += t;
      else
        ahead_sum += t;
    }
  }

  // The workgroup's sums by bucket, out[0 .. buckets - 1]: the copies of each distance, then each bucket's distances.
  __device__ __forceinline__ void store(const BiasedArgs& a, float* out, int tid, int lane) {
    const int len = lut_len(far);
    float f = half_sum(far_sum), z = half_sum(ahead_sum);
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      f += __shfl_xor(f, o);
      z += __shfl_xor(z, o);
    }
    __syncthreads();  // every wave's additions are done
    if (lane == 0) {
      copy[0] += z;        // distance -kLutPad: no pair's
      copy[len - 1] += f;  // distance far + kLutPad - 1: no pair's either
    }
    __syncthreads();
    for (int i = tid; i < len; i += 256) {
      float s = 0.f;
#pragma unroll
      for (int c = 0; c < kTableCopies; ++c) s += all[c * len + i];
      all[i] = s;
    }
    __syncthreads();
    // Bucket j holds a run of distances (the first also all at or below 0, the last all from `far` on).
    for (int j = tid; j < a.buckets; j += 256) {
      const int i0 = j == 0 ? 0 : kLutPad + a.first[j], i1 = j + 1 == a.buckets ? len : kLutPad + a.first[j + 1];
      float s = 0.f;
      for (int i = i0; i < i1; ++i) s += all[i];
      out[j] = s;
    }
  }
};

// Where tiles of 128 positions leave most of the chip idle, a workgroup has 32. Its traffic is four times as much, so it
// loses once the other form fills the CUs. Measured (us, capped, the other form against this; rows x heads x tokens):
//   D = 64   forward 1 x 8 x 512 13.6 / 7.4, 1 x 8 x 2048 42 / 21, 1 x 16 x 2048 (256 tiles) 43 / 28, 2 x 16 x 2048 (512)
//            46 / 50; dQ at the same 18.5 / 8.9, 55 / 23, 57 / 34; dK/dV 17.2 / 7.8, 58 / 24, 61 / 38, then 70 / 72
//   D = 128  forward 1 x 8 x 512 17.2 / 9.6, 2 x 16 x 512 (128) 17.6 / 12.0, 1 x 16 x 2048 (256) 55 / 50, 2 x 16 x 1024
//            (256) 31.1 / 31.5; dQ 26 / 12, 28 / 20, 93 / 72, 4 x 16 x 512 (256) 32 / 38; dK/dV 23 / 12, 25 / 20, 79 / 82
//   D = 256  forward 2 x 8 x 512 (64) 25.6 / 19.2, 2 x 16 x 512 (128) 27.3 / 28.7; the backward keeps to the other form,
//            whose wide tiles this one's registers do not hold
// With one block of 32 there is nothing to split (16 heads of 32 tokens, D = 128, biased, 6.0 against 6.7). Rows so far
// apart that offsets of 31 rows past the last would leave 32 bits take the other form.
inline bool few_tiles(const BiasedArgs& a, int D) {
  const int64_t far = 1 << 24;
  return (int64_t)q_tiles(a.m.N) * a.B * a.H <= (D <= 64 ? kFewTiles : D == 128 ? 128 : 64) && a.m.N > kBlock &&
         a.sq.n < far && a.sk.n < far && a.sv.n < far && a.sdo.n < far;
}

// Host launchers.
hipError_t launch_biased_fwd(const BiasedArgs& a, int D, int is_f16, hipStream_t stream);
hipError_t launch_biased_fwd_few(const BiasedArgs& a, int D, int is_f16, hipStream_t stream);
// The backward's passes where there are few tiles (head dims to 128); dQ with the table's sums where dtable_part is set.
enum FewPass : int { FEW_DQ, FEW_DKDV };
hipError_t launch_biased_bwd_few(const BiasedArgs& a, int D, int is_f16, int pass, hipStream_t stream);
hipError_t launch_biased_dq(const BiasedArgs& a, int D, int is_f16, hipStream_t stream);
hipError_t launch_biased_dq_table(const BiasedArgs& a, int D, int is_f16, hipStream_t stream);  // fills dtable_part
hipError_t launch_biased_dkdv(const BiasedArgs& a, int D, int is_f16, hipStream_t stream);
hipError_t launch_biased_dkdv_wide(const BiasedArgs& a, int D, int is_f16, hipStream_t stream);  // head dims 128, 256
// Table gradient [buckets, H] of table_dtype, contiguous, from the query tiles' sums.
hipError_t launch_table_gradient(const BiasedArgs& a, void* dtable, hipStream_t stream);

}  // namespace sps
