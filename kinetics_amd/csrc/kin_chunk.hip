// Attention of a chunk of new tokens over the paged cache: a ragged batch in which every sequence
// brings one token (decode), a few, or a whole prompt.
//
// Work decomposition: the rows of one (sequence, KV head) -- new tokens times the group's query
// heads -- are cut into tiles of 128; one workgroup of 4 waves owns a tile (and, where there are
// few tiles, one of several spans of its keys; merge_chunk_kernel joins the spans).
//   More than 32 rows: every wave owns 32 rows; 64 keys at a time are staged in LDS for all four
//     (two stages, filled by LDS-direct loads of the next tile while this one is used).
//   Up to 32 rows (decode): all waves hold the same rows and take every fourth block of 32 keys,
//     staged in LDS of their own without any barrier; their results are joined through LDS at the end.
//
// A block of 32 keys by 32 rows is  S^T = K Q^T  on v_mfma_f32_32x32x16: lane l holds row l % 32 and
// 16 of the 32 keys in its registers, so the softmax needs one exchange with lane ^ 32 and no LDS.
// O^T += V^T P^T wants P with 8 consecutive registers per lane as the matrix unit's operand; the
// registers hold the keys 4h + 0..3 and 8 + 4h + 0..3 (h = lane / 32) of every 16, and as the order in
// which keys are summed is free, V^T is read in that same order: ds_read_b64_tr_b16 hands a lane
// four keys of one column.  P never leaves the registers.  The running sum and maximum, and O, are fp32.
//
// The matrix unit takes P in the cache's element type.  With more than 32 rows a weight is rounded to it once (half a unit in the
// last place, as the result itself): a second element for what the rounding leaves makes half as many products again, 550 -> 750 us
// for 8192 tokens from nothing and 155 -> 219 for 2048 behind 30720, which the matrix unit bounds.  With up to 32 rows, where it waits for HBM,
// it gets both, and 2^-18 of a bfloat16 weight is left; the decode kernels keep fp32 (60 single tokens beside four prompts 129.2 -> 130.5 us).
//
// What bounds it, measured on MI355X: prompts the matrix unit (52 % busy) and the vector unit (50 %), which two waves a SIMD hardly overlap --
// 8192 tokens from nothing, 32 heads on 8 of 128, bf16: 550 us, 1.0 PFLOP/s; 2048 behind 30720, 4 heads on 1: 154 us, 0.86 PFLOP/s.
// Decode rows HBM: 60 single tokens of 301..8201 beside four prompts, 8 KV heads of 64, f16: 132 us.  Few rows the chain of
// dependent loads: 8 single tokens of 513..4097: 8 us and 4 for the join.
#include "kin_chunk.h"

namespace kin {

constexpr int kChunkRows = 128;     // rows of a workgroup's tile
constexpr int kChunkKeys = 64;      // keys of a staged tile
// Workgroups on a CU: the registers of a wave's outputs allow 3 with heads of 64 and 2 with heads of 128.
constexpr int chunk_wgs_per_cu(int head_dim) { return head_dim == kHeadDimSmall ? 3 : 2; }
// A weight is 2^(score - reference + up): the reference, the running maximum, is only moved when a score passes it by
// rescale_at.  bfloat16 has fp32's range.  float16 ends at 2^16 and in steps of 2^-24: with weights of up to 2^15, one of 2^-27 of the
// reference has all its bits and none above 2^-38 is lost (at 2^0, thousands of 2^-26 were in the sum but not in the result).
// Scores above 2^20 are too coarse for that: fp32 may take one above its reference by more than float16 has left.
constexpr float rescale_at(bool f16) { return f16 ? 2.f : 8.f; }
template <bool F16>
__device__ __forceinline__ float weight_up(float reference) {
  if constexpr (F16) return fabsf(reference) < 0x1p20f ? 13.f : 0.f;
  return 0.f;
}

struct ChunkAttnParams {
  ChunkParams c;
  uint16_t* out;   // [nnz, hq, D]
  float* lse;      // [nnz, hq] or null
  float* ws_o;     // [splits, nnz * hq, D] fp32, splits > 1 only
  float* ws_lse;   // [splits, nnz * hq] (log2 domain)
  int32_t* ws_count;  // [nnz * hq]: spans of this row's keys
  int slots;       // row tiles over all sequences, some of them empty
  int num_splits;  // most spans of one row tile's keys (the launch's second dimension)
  int span_narrow, span_wide;  // tiles of 64 keys in a span, for row tiles of up to 32 rows and for larger ones
};

typedef short shortx4 __attribute__((ext_vector_type(4)));
typedef unsigned short ushortx2 __attribute__((ext_vector_type(2)));

// First row tile of the sequence b whose rows start at e0: tiles are numbered so that every sequence has room for its rows
// whatever the others bring, without a scan: floor(e0 * group / 128) + b.
__device__ __forceinline__ int first_slot(const ChunkParams& p, int e0, int b) {
  return (int)((int64_t)e0 * p.group / kChunkRows) + b;
}
__device__ __forceinline__ int first_row(const ChunkParams& p, int b) { return min(max(p.q_indptr[b], 0), p.nnz); }
// The sequence that owns row tile `slot` -- the last one whose first tile is not behind it -- into sq; -1 if there is none.
__device__ __forceinline__ int seq_of_slot(const ChunkParams& p, int slot, ChunkSeq& sq) {
  const int lane = threadIdx.x & 63;
  if (p.batch <= 64) {  // one sequence per lane: everything about it in one round trip
    const int i = min(lane, p.batch - 1);
    const int e0 = first_row(p, i), e1 = p.q_indptr[i + 1], ps = p.page_indptr[i], pe = p.page_indptr[i + 1];
    const int last = p.last_page_len[i], prefix = p.prefix_lens ? p.prefix_lens[i] : 0;
    const int b = __popcll(__ballot(lane < p.batch && first_slot(p, e0, i) <= slot)) - 1;
    if (b < 0) return -1;
    sq = make_chunk_seq(p, __builtin_amdgcn_readlane(e0, b), __builtin_amdgcn_readlane(e1, b), __builtin_amdgcn_readlane(ps, b),
                        __builtin_amdgcn_readlane(pe, b), __builtin_amdgcn_readlane(last, b), __builtin_amdgcn_readlane(prefix, b));
    return b;
  }
  int lo = 0, n = p.batch;
  while (true) {  // 64 candidates per step
    const int step = (n + 63) >> 6;
    const int b = lo + lane * step;
    const bool ok = b < lo + n && first_slot(p, first_row(p, b), b) <= slot;
    const int count = __popcll(__ballot(ok));
    if (count == 0) return -1;
    const int next = lo + (count - 1) * step;
    n = min(step, lo + n - next);
    lo = next;
    if (step == 1) break;
  }
  lo = __builtin_amdgcn_readfirstlane(lo);
  sq = chunk_seq(p, lo);
  return lo;
}

// One wave's 32 rows: queries as a matrix operand, running softmax, output.
template <int HD>
struct WaveRows {
  uint4 q[HD / 16];
  floatx16 o[HD / 32];
  float m, l;       // running maximum (units of the raw product, or log2 with EXTRA) and this lane's part of the sum
  float up;         // its weights are larger by 2^up
  RowSpan span;
  float slope2;
  uint64_t pos_inf, neg_inf;  // bit e: output register e gets an infinity of that sign (both: NaN)
};

template <int HD>
__device__ __forceinline__ void load_rows(const ChunkParams& p, const ChunkSeq& s, int h, int r, bool valid, WaveRows<HD>& w) {
  const int lane = threadIdx.x & 63, half = lane >> 5;
  const int i = r / p.group, g = r - i * p.group;
  w.m = kNegInf;
  w.l = w.up = 0.f;
  w.pos_inf = w.neg_inf = 0;
#pragma unroll
  for (int t = 0; t < HD / 32; ++t)
#pragma unroll
    for (int e = 0; e < 16; ++e) w.o[t][e] = 0.f;
  w.span = row_span(p, s, i, valid);
  w.slope2 = (p.slopes && valid) ? p.slopes[h * p.group + g] * kLog2e : 0.f;
  const uint4* src = reinterpret_cast<const uint4*>(p.q + ((int64_t)(s.e0 + i) * p.hq + h * p.group + g) * HD);
#pragma unroll
  for (int k = 0; k < HD / 16; ++k) w.q[k] = valid ? src[2 * k + half] : uint4{0, 0, 0, 0};
}

// The 8 elements with zeros in place of the infinite and NaN ones.
template <bool F16>
__device__ __forceinline__ uint4 finite_only(const uint4& v) {
  const uint32_t e = F16 ? 0x7c00u : 0x7f80u;
  uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if ((w[i] & e) == e) w[i] &= 0xffff0000u;
    if (((w[i] >> 16) & e) == e) w[i] &= 0xffffu;
  }
  return uint4{w[0], w[1], w[2], w[3]};
}

// 32 * NSUB staged keys against the wave's rows.  k / v: the staged rows in LDS; slot0: token slot of the
// first key; masked: some key is not seen by some row; units: bit u = the 16 keys u come from a page
// of the cache.
template <int HD, bool F16, bool EXTRA, int NSUB, typename AfterK, typename BeforeV>
__device__ __forceinline__ void attend_block(const ChunkParams& p, WaveRows<HD>& w, const unsigned char* k, const unsigned char* v,
                                             int slot0, bool masked, uint32_t units, AfterK after_k, BeforeV before_v) {
  constexpr int kRowB = HD * 2;
  const int lane = threadIdx.x & 63, half = lane >> 5, col = lane & 31;
  floatx16 s[NSUB];
  // The wave that is at its products goes first on its SIMD (2048 behind 30720: 171 -> 166 us; with cap or bias it costs 3 %).
  if constexpr (!EXTRA) __builtin_amdgcn_s_setprio(1);
#pragma unroll
  for (int t = 0; t < NSUB; ++t) {
#pragma unroll
    for (int e = 0; e < 16; ++e) s[t][e] = 0.f;
#pragma unroll
    for (int kk = 0; kk < HD / 16; ++kk) {
      const uint4 a = *reinterpret_cast<const uint4*>(k + (t * 32 + col) * kRowB + (((2 * kk + half) ^ row_swizzle<HD>(col)) * 16));
      s[t] = mfma_32x32x16<F16>(a, w.q[kk], s[t]);
    }
  }
  if constexpr (!EXTRA) __builtin_amdgcn_s_setprio(0);
  after_k();
  float bias = 0.f;  // what all of this lane's scores still lack
  if constexpr (EXTRA) {
#pragma unroll
    for (int t = 0; t < NSUB; ++t) cap_scores<false>(p, s[t], [](int) { return 0.f; });
    if (p.slopes) {
      // Register e is key slot0 + 4 half + k(e).  Where every key lies in front of the wave's rows, -slope |p - j| is a part that
      // all of a lane's keys share and slope * k(e): one instruction per score.
      const float dist = (float)(w.span.hi - slot0 - 4 * half);
      if (!__ballot(w.span.hi >= 0 && w.span.hi < slot0 + 32 * NSUB - 1)) {
        bias = -w.slope2 * dist;
#pragma unroll
        for (int t = 0; t < NSUB; ++t)
#pragma unroll
          for (int e = 0; e < 16; ++e) s[t][e] = fmaf(w.slope2, (float)(t * 32 + acc_row(e, 0)), s[t][e]);
      } else {
#pragma unroll
        for (int t = 0; t < NSUB; ++t)
#pragma unroll
          for (int e = 0; e < 16; ++e) s[t][e] = fmaf(-w.slope2, fabsf(dist - (float)(t * 32 + acc_row(e, 0))), s[t][e]);
      }
    }
  }
  if (masked) {
#pragma unroll
    for (int t = 0; t < NSUB; ++t)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int slot = (units >> (2 * t + (e >> 3))) & 1 ? slot0 + t * 32 + acc_row(e, half) : 0x7fffffff;
        s[t][e] = row_sees(w.span, p.first_page_offset, slot) ? s[t][e] : kNegInf;
      }
  }
  const float c = EXTRA ? 1.f : p.scale_log2;
  float mt = kNegInf;
#pragma unroll
  for (int t = 0; t < NSUB; ++t)
#pragma unroll
    for (int e = 0; e < 16; ++e) mt = fmaxf(mt, s[t][e]);
  mt = max_halves(EXTRA ? mt + bias : mt);
  // The reference follows the scores only when they pass it by some way, so most blocks need no rescaling of O.
  const bool move = mt > w.m && !((mt - w.m) * c <= rescale_at(F16));
  if (__ballot(move)) {
    const float m_new = move ? mt : w.m, up = move ? weight_up<F16>(mt * c) : w.up;
    const float alpha = m_new == kNegInf ? 1.f : fast_exp2((w.m - m_new) * c + (up - w.up));
    w.m = m_new;
    w.up = up;
    w.l *= alpha;
#pragma unroll
    for (int t = 0; t < HD / 32; ++t)
#pragma unroll
      for (int e = 0; e < 16; ++e) w.o[t][e] *= alpha;
  }
  const float shift = (w.m == kNegInf ? 0.f : w.m * c) - w.up - (EXTRA ? bias : 0.f);
  // V^T: lane (16-lane group g = lane / 16 % 2, place q = lane % 16) asks for 4 columns of key row q / 4 and is handed
  // the 4 keys of column 16 g + q; two such reads make one operand (keys 4h.. and 8 + 4h..).
  const int q4 = (lane & 15) >> 2, cq = ((lane >> 4) & 1) * 2 + ((lane & 3) >> 1), lo8 = (lane & 1) * 8;
  auto read_v = [&](int t, int kk, int dt) -> uint4 {
    uint2 part[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int row = 8 * e + 4 * half + q4;
      const int chunk = (dt * 4 + cq) ^ row_swizzle<HD>(row);
      const unsigned char* a = v + (t * 32 + kk * 16 + row) * kRowB + chunk * 16 + lo8;
      const shortx4 r = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) shortx4*)(a));
      part[e] = __builtin_bit_cast(uint2, r);
    }
    return uint4{part[0].x, part[0].y, part[1].x, part[1].y};
  };
  // With the longer scores the first operands are read before the exponentials (capped, window 1024: 117 -> 107 us; without
  // cap or bias no difference).
  constexpr bool kEarlyValues = EXTRA && NSUB == 2;
  uint4 early[kEarlyValues ? HD / 32 : 1];
  if constexpr (kEarlyValues) {
#pragma unroll
    for (int dt = 0; dt < HD / 32; ++dt) early[dt] = read_v(0, 0, dt);
    __builtin_amdgcn_sched_barrier(0);
  }
  // Up to 32 rows: a weight as two elements, the second what the first one's rounding left.
  constexpr bool kTwoParts = NSUB == 1;
  uint4 pb[NSUB][2], pl[2];
#pragma unroll
  for (int t = 0; t < NSUB; ++t) {
    uint32_t d[8], r[8];
#pragma unroll
    for (int e = 0; e < 16; e += 2) {
      const float p0 = fast_exp2(fmaf(s[t][e], c, -shift)), p1 = fast_exp2(fmaf(s[t][e + 1], c, -shift));
      w.l += p0 + p1;
      d[e / 2] = pack2<F16>(p0, p1);
      if constexpr (kTwoParts) r[e / 2] = pack2<F16>(p0 - elem_lo<F16>(d[e / 2]), p1 - elem_hi<F16>(d[e / 2]));
    }
    pb[t][0] = uint4{d[0], d[1], d[2], d[3]};
    pb[t][1] = uint4{d[4], d[5], d[6], d[7]};
    if constexpr (kTwoParts) {
      pl[0] = uint4{r[0], r[1], r[2], r[3]};
      pl[1] = uint4{r[4], r[5], r[6], r[7]};
    }
  }
  before_v();
  if constexpr (!EXTRA) __builtin_amdgcn_s_setprio(1);
#pragma unroll
  for (int t = 0; t < NSUB; ++t)
#pragma unroll
    for (int kk = 0; kk < 2; ++kk)
#pragma unroll
      for (int dt = 0; dt < HD / 32; ++dt) {
        uint4 a;
        if constexpr (kEarlyValues) a = t == 0 && kk == 0 ? early[dt] : read_v(t, kk, dt);
        else a = read_v(t, kk, dt);
        w.o[dt] = mfma_32x32x16<F16>(a, pb[t][kk], w.o[dt]);
        if constexpr (kTwoParts) w.o[dt] = mfma_32x32x16<F16>(a, pl[kk], w.o[dt]);
      }
  if constexpr (!EXTRA) __builtin_amdgcn_s_setprio(0);
}

// A value that is not seen has weight 0, and 0 times an infinity would be NaN; so would be the sum of a weight's two parts
// times an infinity.  In the blocks where some row does not see some key, and in all blocks where weights have two
// parts, infinite and NaN values are therefore taken out of the staged rows: which elements of this
// lane's output they reach is kept as bits, and the result gets them at the end.
template <int HD, bool F16, int ROWS>
__device__ __forceinline__ bool rows_special(const unsigned char* v) {
  ushortx2 top = {0, 0};  // the largest magnitude bits of the even and of the odd elements
#pragma unroll
  for (int x = 0; x < ROWS * (HD / 8); x += 64) {
    const uint4 y = *reinterpret_cast<const uint4*>(v + (x + (threadIdx.x & 63)) * 16);
    const uint32_t w[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) top = __builtin_elementwise_max(top, __builtin_bit_cast(ushortx2, w[i] & 0x7fff7fffu));
  }
  return __ballot(max(top.x, top.y) >= (F16 ? 0x7c00 : 0x7f80)) != 0;
}
template <int HD, bool F16>
__device__ __forceinline__ void note_specials(WaveRows<HD>& w, const unsigned char* v, int keys, int slot0, uint32_t units, int first) {
  const int half = (threadIdx.x >> 5) & 1;
#pragma unroll 1
  for (int j = 0; j < keys; ++j) {
    const bool on = row_sees(w.span, first, slot0 + j) && ((units >> (j >> 4)) & 1);
#pragma unroll 1
    for (int x = 0; x < HD / 2; ++x) {  // element x % 16 of output tile x / 16
      const int d = (x >> 4) * 32 + acc_row(x & 15, half);
      const uint32_t bits = *reinterpret_cast<const uint16_t*>(v + j * HD * 2 + (((d >> 3) ^ row_swizzle<HD>(j & 15)) * 16) + (d & 7) * 2);
      const float y = elem_lo<F16>(bits);
      if (on && !(fabsf(y) < INFINITY)) {
        if (!(y < 0.f)) w.pos_inf |= 1ull << x;
        if (!(y > 0.f)) w.neg_inf |= 1ull << x;
      }
    }
  }
}
template <int HD, bool F16>
__device__ __forceinline__ void clear_specials(unsigned char* v, int rows) {
#pragma unroll 1
  for (int x = threadIdx.x & 63; x < rows * (HD / 8); x += 64) {
    uint4* at = reinterpret_cast<uint4*>(v + x * 16);
    *at = finite_only<F16>(*at);
  }
}
template <int HD>
__device__ __forceinline__ void put_specials(WaveRows<HD>& w) {
  if (__ballot((w.pos_inf | w.neg_inf) != 0)) {
#pragma unroll
    for (int x = 0; x < HD / 2; ++x) {
      if ((w.pos_inf >> x) & 1) w.o[x >> 4][x & 15] += INFINITY;
      if ((w.neg_inf >> x) & 1) w.o[x >> 4][x & 15] -= INFINITY;
    }
  }
}

template <int HD, bool F16, bool EXTRA>
__global__ __launch_bounds__(256, chunk_wgs_per_cu(HD)) void chunk_attn_kernel(ChunkAttnParams ap) {
  constexpr int kRowB = HD * 2;
  constexpr int kUnitB = 16 * kRowB;             // 16 keys
  constexpr int kStageB = 2 * kChunkKeys * kRowB;  // 64 keys and their values
  constexpr int kWaveB = 2 * 32 * kRowB;         // a wave's own 32 keys and values
  static_assert(4 * kWaveB == 2 * kStageB && 4 * 32 * HD * 4 == 2 * kStageB, "the wide form's two stages hold the narrow form's blocks and its merge buffer");
  __shared__ __attribute__((aligned(16))) unsigned char lds[2 * kStageB + 1024];  // the stages first: LDS-direct loads reach 64 KiB
  float(*sm_m)[32] = reinterpret_cast<float(*)[32]>(lds + 2 * kStageB);
  float(*sm_l)[32] = sm_m + 4;
  const ChunkParams& p = ap.c;
  const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int h = blockIdx.x % p.hkv;
  const int slot = ap.slots - 1 - (int)(blockIdx.x / p.hkv);  // the later rows of a sequence see more keys: they go first
  const int split = blockIdx.y;
  ChunkSeq sq;
  const int b = seq_of_slot(p, slot, sq);
  if (b < 0) return;
  const int rows = sq.n * p.group;   // int: nnz * group is checked on the host
  const int r0 = (slot - first_slot(p, sq.e0, b)) * kChunkRows;
  if (r0 < 0 || r0 >= rows) return;  // below 0: q_indptr does not ascend
  const int nrows = min(rows - r0, kChunkRows);
  const bool narrow = nrows <= 32;   // uniform

  // Tiles of 64 token slots that any row of this workgroup sees: those of the prefix, then from the first row's window to
  // the last row's own token.
  const int off = p.first_page_offset;
  const int pos0 = sq.len - sq.n + r0 / p.group, pos1 = sq.len - sq.n + (r0 + nrows - 1) / p.group;
  const int end = sq.len + off;
  const int n_prefix = (pos1 >= 0 && sq.prefix > 0) ? (sq.prefix + off + kChunkKeys - 1) / kChunkKeys : 0;
  const int seen0 = p.window > 0 ? max(pos0 - p.window + 1, 0) : 0;
  const int t_lo = max((seen0 + off) / kChunkKeys, n_prefix);
  const int t_hi = pos1 >= 0 ? (pos1 + off) / kChunkKeys + 1 : 0;
  const int n_tiles = n_prefix + max(t_hi - t_lo, 0);
  auto tile_at = [&](int it) { return it < n_prefix ? it : it - n_prefix + t_lo; };
  // Spans: a tile with few keys has fewer than the launch provides for, often one, and writes its result itself.
  const int per_span = max(narrow ? ap.span_narrow : ap.span_wide, (n_tiles + ap.num_splits - 1) / ap.num_splits);
  const int spans = max((n_tiles + per_span - 1) / per_span, 1);
  if (split >= spans) return;
  const int it0 = split * per_span, it1 = min(n_tiles, it0 + per_span);

  // Rows: in the narrow form every wave holds all of them.
  const int row = (narrow ? 0 : wave * 32) + (lane & 31);
  WaveRows<HD> w;
  load_rows<HD>(p, sq, h, r0 + row, row < nrows, w);

  // Staging: lane l of load j brings 16 bytes of row (64 / CPR) * j + l / CPR of a unit.
  constexpr int CPR = HD / 8;
  const int row_bytes = p.hkv * kRowB;
  int dma[HD / 32];
#pragma unroll
  for (int j = 0; j < HD / 32; ++j) {
    const int rr = (64 / CPR) * j + lane / CPR;
    dma[j] = rr * row_bytes + (((lane & (CPR - 1)) ^ row_swizzle<HD>(rr)) * 16);
  }
  const int64_t page_bytes = 2ll * p.page_size * row_bytes;
  const char* kvh = reinterpret_cast<const char*>(p.kv) + (int64_t)h * kRowB;
  // Page id of the 16 token slots `unit`; -1 outside the cache.  Ids are fetched a whole batch of blocks ahead, one per lane.
  auto page_of = [&](int unit) -> int {
    const int id = sq.pages[min((unit * 16) >> p.page_shift, sq.n_pages - 1)];
    return (id >= 0 && (int64_t)id < p.num_pages) ? id : -1;
  };
  // Descriptors of a unit's K and V rows; token slots behind the sequence read as zeros, whatever the page holds there.
  auto unit_rsrc = [&](int unit, int id, bool values) {
    const int n = min(max(end - unit * 16, 0), 16);
    const int bytes = (id >= 0 && n > 0) ? (n - 1) * row_bytes + kRowB : 0;
    const int in_page = (unit * 16) & (p.page_size - 1);
    return rsrc_words(kvh + max(id, 0) * page_bytes + (int64_t)(in_page + (values ? p.page_size : 0)) * row_bytes, bytes);
  };

  // LDS-direct loads of the 16 keys (or values) of one unit.  Nontemporal where nobody else reads them.
  auto stage_unit = [&](u32x4 r, const unsigned char* dst, bool stream) {
    const uint32_t at = lds_offset(dst);
#pragma unroll
    for (int j = 0; j < HD / 32; ++j) {
      if (stream) lds_load_16<true>(r, at + j * 1024, dma[j]);
      else lds_load_16<false>(r, at + j * 1024, dma[j]);
    }
  };

  if (narrow) {
    // Blocks of 32 token slots of the tiles it0 .. it1-1, every fourth one for this wave.
    const int n_blocks = (2 * (it1 - it0) - wave + 3) >> 2;
    unsigned char* kbuf = lds + wave * kWaveB;
    unsigned char* vbuf = kbuf + 32 * kRowB;
    auto unit_at = [&](int x) {  // first unit of the wave's block x (the last one's behind the end)
      const int i = wave + 4 * min(x, n_blocks - 1);
      return tile_at(it0 + (i >> 1)) * 4 + (i & 1) * 2;
    };
    auto fetch_ids = [&](int x) { return page_of(unit_at(x + (lane >> 1)) + (lane & 1)); };
    int ids = -1, ids_next = -1, id0 = -1, id1 = -1;
    if (n_blocks > 0) {
      ids = fetch_ids(0);
      if (n_blocks > 31) ids_next = fetch_ids(32);
      id0 = __builtin_amdgcn_readlane(ids, 0);
      id1 = __builtin_amdgcn_readlane(ids, 1);
      const int u = unit_at(0);
      stage_unit(unit_rsrc(u, id0, false), kbuf, true);
      stage_unit(unit_rsrc(u + 1, id1, false), kbuf + kUnitB, true);
      stage_unit(unit_rsrc(u, id0, true), vbuf, true);
      stage_unit(unit_rsrc(u + 1, id1, true), vbuf + kUnitB, true);
    }
    for (int x = 0; x < n_blocks; ++x) {
      const int u = unit_at(x);
      const uint32_t units = (id0 >= 0 ? 1u : 0u) | (id1 >= 0 ? 2u : 0u);
      // the next block (behind the last one: empty descriptors, so that the counts below hold)
      if (((x + 1) & 31) == 0) {
        ids = ids_next;
        if (x + 33 < n_blocks) ids_next = fetch_ids(x + 33);
      }
      int n0 = __builtin_amdgcn_readlane(ids, 2 * ((x + 1) & 31)), n1 = __builtin_amdgcn_readlane(ids, 2 * ((x + 1) & 31) + 1);
      if (x + 1 >= n_blocks) n0 = n1 = -1;
      const int un = unit_at(x + 1);
      const int slot0 = u * 16;
      const bool all = slot0 >= (p.window > 0 ? max(pos1 - p.window + 1, 0) : 0) + off && slot0 + 31 <= pos0 + off;
      const bool masked = !(units == 3u && (all || (slot0 >= off && slot0 + 32 <= sq.prefix + off && pos0 >= 0)));
      __builtin_amdgcn_sched_barrier(0);
      __builtin_amdgcn_s_waitcnt(wait_vm_imm(HD / 16));  // this block's keys are in; its values may be on their way
      __builtin_amdgcn_sched_barrier(0);
      auto after_k = [&]() {
        __builtin_amdgcn_sched_barrier(0);
        __builtin_amdgcn_s_waitcnt(0xc07f);  // the reads of the keys are done (lgkmcnt 0)
        stage_unit(unit_rsrc(un, n0, false), kbuf, true);
        stage_unit(unit_rsrc(un + 1, n1, false), kbuf + kUnitB, true);
        __builtin_amdgcn_sched_barrier(0);
      };
      auto before_v = [&]() {
        __builtin_amdgcn_sched_barrier(0);
        __builtin_amdgcn_s_waitcnt(wait_vm_imm(HD / 16));  // the values are in; the next keys may be on their way
        __builtin_amdgcn_sched_barrier(0);
        if (rows_special<HD, F16, 32>(vbuf)) {
          note_specials<HD, F16>(w, vbuf, 32, slot0, units, off);
          clear_specials<HD, F16>(vbuf, 32);
        }
      };
      attend_block<HD, F16, EXTRA, 1>(p, w, kbuf, vbuf, slot0, masked, units, after_k, before_v);
      __builtin_amdgcn_sched_barrier(0);
      __builtin_amdgcn_s_waitcnt(0xc07f);
      stage_unit(unit_rsrc(un, n0, true), vbuf, true);
      stage_unit(unit_rsrc(un + 1, n1, true), vbuf + kUnitB, true);
      __builtin_amdgcn_sched_barrier(0);
      id0 = n0;
      id1 = n1;
    }
    put_specials<HD>(w);
    __builtin_amdgcn_s_waitcnt(0);
    // Join the waves: every wave leaves its rows' maxima, sums and outputs in LDS.
    w.l += other_half(w.l);
    const float c = EXTRA ? 1.f : p.scale_log2;
    __syncthreads();
    if (lane < 32) {
      sm_m[wave][lane] = w.m == kNegInf ? kNegInf : w.m * c - w.up;
      sm_l[wave][lane] = w.l;
    }
    float* ow = reinterpret_cast<float*>(lds);  // [4 waves][rows][HD]
    if (row < nrows) {
#pragma unroll
      for (int t = 0; t < HD / 32; ++t)
#pragma unroll
        for (int e = 0; e < 16; e += 4)
          *reinterpret_cast<float4*>(ow + ((wave * 32 + row) * HD + t * 32 + acc_row(e, half))) =
              make_float4(w.o[t][e], w.o[t][e + 1], w.o[t][e + 2], w.o[t][e + 3]);
    }
    __syncthreads();
    for (int x = tid; x < nrows * (HD / 4); x += 256) {
      const int r = x / (HD / 4), d = (x - r * (HD / 4)) * 4;
      float mm = kNegInf;
#pragma unroll
      for (int k = 0; k < 4; ++k) mm = fmaxf(mm, sm_m[k][r]);
      const float safe = mm == kNegInf ? 0.f : mm;
      float den = 0.f;
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float f = fast_exp2(sm_m[k][r] - safe);
        const float4 o = *reinterpret_cast<const float4*>(ow + ((k * 32 + r) * HD + d));
        den = fmaf(f, sm_l[k][r], den);
        acc.x = fmaf(f, o.x, acc.x);
        acc.y = fmaf(f, o.y, acc.y);
        acc.z = fmaf(f, o.z, acc.z);
        acc.w = fmaf(f, o.w, acc.w);
      }
      const bool none = mm == kNegInf && den == 0.f;
      const float inv = none ? 0.f : 1.f / den;
      const float lse2 = none ? kNegInf : mm + __log2f(den);
      const int i = (r0 + r) / p.group, g = (r0 + r) - i * p.group;
      const int64_t hq = (int64_t)(sq.e0 + i) * p.hq + h * p.group + g;
      if (d == 0 && split == 0 && ap.num_splits > 1) ap.ws_count[hq] = spans;
      if (spans == 1) {
        uint2 y;
        y.x = pack2<F16>(acc.x * inv, acc.y * inv);
        y.y = pack2<F16>(acc.z * inv, acc.w * inv);
        *reinterpret_cast<uint2*>(ap.out + hq * HD + d) = y;
        if (ap.lse && d == 0) ap.lse[hq] = lse2 * kLn2;
      } else {
        const int64_t at = (int64_t)split * p.nnz * p.hq + hq;
        *reinterpret_cast<float4*>(ap.ws_o + at * HD + d) = make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv);
        if (d == 0) ap.ws_lse[at] = lse2;
      }
    }
    return;
  }

  // ---- more than 32 rows ----
  const bool mine = wave * 32 < nrows;
  const int wpos0 = sq.len - sq.n + (r0 + wave * 32) / p.group;
  const int wpos1 = sq.len - sq.n + (r0 + min(wave * 32 + 31, nrows - 1)) / p.group;
  auto fetch_ids = [&](int it) { return page_of(tile_at(min(it + (lane >> 2), it1 - 1)) * 4 + (lane & 3)); };  // 16 tiles
  int ids = -1, ids_next = -1;
  auto stage_tile = [&](int it, unsigned char* dst, uint32_t& units) {
    const int k = (it - it0) & 15;
    if (k == 0) {
      ids = ids_next;
      if (it + 16 < it1) ids_next = fetch_ids(it + 16);
    }
    units = (uint32_t)(__ballot(ids >= 0) >> (4 * k)) & 15u;
    const int id = __builtin_amdgcn_readlane(ids, 4 * k + wave);
    const int u = tile_at(it) * 4 + wave;
    stage_unit(unit_rsrc(u, id, false), dst + wave * kUnitB, false);
    stage_unit(unit_rsrc(u, id, true), dst + (4 + wave) * kUnitB, false);
  };
  uint32_t units_next = 0;
  if (it0 < it1) {
    ids_next = fetch_ids(it0);
    stage_tile(it0, lds, units_next);
  }
  // No row of [rows at first .. last position] misses a key of the tile.
  auto seen_whole = [&](int slot0, uint32_t units, int first, int last) {
    const bool causal = slot0 >= (p.window > 0 ? max(last - p.window + 1, 0) : 0) + off && slot0 + kChunkKeys - 1 <= first + off;
    return units == 15u && (causal || (slot0 >= off && slot0 + kChunkKeys <= sq.prefix + off && first >= 0));
  };
  for (int it = it0; it < it1; ++it) {
    const int stage = (it - it0) & 1;
    const uint32_t units = units_next;
    unsigned char* kst = lds + stage * kStageB;
    unsigned char* vst = kst + kChunkKeys * kRowB;
    __builtin_amdgcn_s_waitcnt(0);  // this wave's part of the tile is in; behind the barrier, every wave's
    __syncthreads();
    if (it + 1 < it1) stage_tile(it + 1, lds + (1 - stage) * kStageB, units_next);
    const int slot0 = tile_at(it) * kChunkKeys;
    if (!seen_whole(slot0, units, pos0, pos1)) {  // the whole workgroup looks for infinite and NaN values
      const bool any = rows_special<HD, F16, 16>(vst + wave * kUnitB);
      if (lane == 0) sm_m[0][wave] = any ? 1.f : 0.f;
      __syncthreads();
      if (sm_m[0][0] + sm_m[0][1] + sm_m[0][2] + sm_m[0][3] > 0.f) {
        if (mine) note_specials<HD, F16>(w, vst, kChunkKeys, slot0, units, off);
        __syncthreads();
        clear_specials<HD, F16>(vst + wave * kUnitB, 16);
        __syncthreads();
      }
    }
    if (!mine) continue;
    const bool in_prefix = slot0 < sq.prefix + off;
    if (!in_prefix && (slot0 > wpos1 + off || (p.window > 0 && slot0 + kChunkKeys <= wpos0 - p.window + 1 + off))) continue;
    auto nothing = []() {};
    attend_block<HD, F16, EXTRA, 2>(p, w, kst, vst, slot0, !seen_whole(slot0, units, wpos0, wpos1), units, nothing, nothing);
  }
  put_specials<HD>(w);
  if (row < nrows) {
    const float c = EXTRA ? 1.f : p.scale_log2;
    const float l = w.l + other_half(w.l);
    const bool none = w.m == kNegInf && l == 0.f;
    const float inv = none ? 0.f : 1.f / l;
    const float lse2 = none ? kNegInf : w.m * c + (__log2f(l) - w.up);
    const int i = (r0 + row) / p.group, g = (r0 + row) - i * p.group;
    const int64_t hq = (int64_t)(sq.e0 + i) * p.hq + h * p.group + g;
    const int64_t at = (int64_t)split * p.nnz * p.hq + hq;
#pragma unroll
    for (int t = 0; t < HD / 32; ++t)
#pragma unroll
      for (int e = 0; e < 16; e += 4) {
        const int d = t * 32 + acc_row(e, half);
        const floatx4 x = {w.o[t][e] * inv, w.o[t][e + 1] * inv, w.o[t][e + 2] * inv, w.o[t][e + 3] * inv};
        if (spans == 1) {
          uint2 y;
          y.x = pack2<F16>(x[0], x[1]);
          y.y = pack2<F16>(x[2], x[3]);
          *reinterpret_cast<uint2*>(ap.out + hq * HD + d) = y;
        } else {
          *reinterpret_cast<floatx4*>(ap.ws_o + at * HD + d) = x;
        }
      }
    if (half == 0) {
      if (spans > 1) ap.ws_lse[at] = lse2;
      else if (ap.lse) ap.lse[hq] = lse2 * kLn2;
      if (split == 0 && ap.num_splits > 1) ap.ws_count[hq] = spans;
    }
  }
}

// Joins the spans of the keys: HD / 4 lanes per (row, query head), GROUPS of them sharing its spans (few rows have many spans, and
// reading those one after the other is all latency: 16 spans of 32 rows 7.3 us with one group, 3.0 us with eight).
// Rows that belong to no sequence are left alone.
template <int HD, bool F16, int GROUPS>
__global__ __launch_bounds__(256) void merge_chunk_kernel(ChunkAttnParams ap) {
  constexpr int LPR = HD / 4, ROWS = 256 / (LPR * GROUPS);
  __shared__ float sm_m[GROUPS][ROWS], sm_l[GROUPS][ROWS];
  __shared__ __attribute__((aligned(16))) float sm_o[GROUPS][ROWS][HD];
  const int64_t total = (int64_t)ap.c.nnz * ap.c.hq;
  const int d = (threadIdx.x % LPR) * 4, g = threadIdx.x / LPR % GROUPS, r = threadIdx.x / (LPR * GROUPS);
  const int64_t x = (int64_t)blockIdx.x * ROWS + r;
  const int64_t tok = x / ap.c.hq;
  const bool mine = x < total && tok >= ap.c.q_indptr[0] && tok < ap.c.q_indptr[ap.c.batch];
  const int spans = mine ? min(ap.ws_count[x], ap.num_splits) : 0;  // min: a row nobody counted (q_indptr does not ascend)
  float mm = kNegInf, den = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  if (spans > 1) {
#pragma unroll 8
    for (int s = g; s < spans; s += GROUPS) mm = fmaxf(mm, ap.ws_lse[s * total + x]);
    const float safe = mm == kNegInf ? 0.f : mm;
#pragma unroll 8
    for (int s = g; s < spans; s += GROUPS) {
      const float f = fast_exp2(ap.ws_lse[s * total + x] - safe);
      const float4 o = *reinterpret_cast<const float4*>(ap.ws_o + (s * total + x) * HD + d);
      den += f;
      acc.x = fmaf(f, o.x, acc.x);
      acc.y = fmaf(f, o.y, acc.y);
      acc.z = fmaf(f, o.z, acc.z);
      acc.w = fmaf(f, o.w, acc.w);
    }
  }
  if constexpr (GROUPS > 1) {
    if (d == 0) {
      sm_m[g][r] = mm;
      sm_l[g][r] = den;
    }
    *reinterpret_cast<float4*>(&sm_o[g][r][d]) = acc;
    __syncthreads();
    if (g > 0) return;
    mm = kNegInf;
#pragma unroll
    for (int k = 0; k < GROUPS; ++k) mm = fmaxf(mm, sm_m[k][r]);
    const float safe = mm == kNegInf ? 0.f : mm;
    den = 0.f;
    acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int k = 0; k < GROUPS; ++k) {
      const float f = fast_exp2(sm_m[k][r] - safe);
      const float4 o = *reinterpret_cast<const float4*>(&sm_o[k][r][d]);
      den = fmaf(f, sm_l[k][r], den);
      acc.x = fmaf(f, o.x, acc.x);
      acc.y = fmaf(f, o.y, acc.y);
      acc.z = fmaf(f, o.z, acc.z);
      acc.w = fmaf(f, o.w, acc.w);
    }
  }
  if (spans <= 1) return;  // no row, or one whose workgroup wrote the result
  const bool none = mm == kNegInf && den == 0.f;
  const float inv = none ? 0.f : 1.f / den;
  uint2 y;
  y.x = pack2<F16>(acc.x * inv, acc.y * inv);
  y.y = pack2<F16>(acc.z * inv, acc.w * inv);
  *reinterpret_cast<uint2*>(ap.out + x * HD + d) = y;
  if (ap.lse && d == 0) ap.lse[x] = none ? kNegInf : (mm + __log2f(den)) * kLn2;
}

// ---- host side ---------------------------------------------------------------

int check_chunk_args(const char* fn, const void* q, const void* kv_cache, const int32_t* q_indptr, const int32_t* page_indices,
                     const int32_t* page_indptr, const int32_t* last_page_len, int64_t nnz, int batch, int num_q_heads,
                     int num_kv_heads, int head_dim, int page_size, int64_t num_pages, int max_pages_per_seq,
                     int first_page_offset, float sm_scale, float softcap, int window, int max_group) {
  if (!q || !kv_cache || !q_indptr || !page_indices || !page_indptr || !last_page_len)
    return fail(KIN_ERR_NULL_POINTER, "%s: null pointer argument", fn);
  if (int st = check_common_dims(fn, batch, num_q_heads, num_kv_heads, head_dim, page_size, true, max_group)) return st;
  if (int st = check_first_page_offset(fn, first_page_offset, page_size)) return st;
  if (nnz < 0) return fail(KIN_ERR_BAD_SHAPE, "%s: nnz=%lld is negative", fn, (long long)nnz);
  if (nnz * num_q_heads > 0x7fffffffLL / 2) return fail(KIN_ERR_UNSUPPORTED, "%s: nnz*num_q_heads is too large", fn);
  if (num_q_heads > 32768) return fail(KIN_ERR_UNSUPPORTED, "%s: num_q_heads=%d is too many", fn, num_q_heads);
  if (num_pages < 1) return fail(KIN_ERR_BAD_SHAPE, "%s: num_pages=%lld must be >= 1", fn, (long long)num_pages);
  if (max_pages_per_seq < 1)
    return fail(KIN_ERR_BAD_SHAPE, "%s: max_pages_per_seq=%d must be >= 1", fn, max_pages_per_seq);
  if (window < 0) return fail(KIN_ERR_BAD_SHAPE, "%s: window=%d is negative", fn, window);
  if (!(sm_scale >= 0.f) || std::isinf(sm_scale) || !(softcap >= 0.f) || std::isinf(softcap))
    return fail(KIN_ERR_BAD_SHAPE, "%s: sm_scale and softcap must be finite and not negative", fn);
  // what the kernels multiply a raw product with
  const float scale = sm_scale > 0.f ? sm_scale : 1.0f / sqrtf((float)head_dim);
  if (std::isinf((float)((double)scale * 1.4426950408889634)) || (softcap > 0.f && std::isinf(scale / softcap)))
    return fail(KIN_ERR_BAD_SHAPE, "%s: sm_scale=%g with softcap=%g is out of fp32's range", fn, sm_scale, softcap);
  if (!aligned16(q) || !aligned16(kv_cache))
    return fail(KIN_ERR_MISALIGNED, "%s: q and kv_cache must be 16-byte aligned", fn);
  return KIN_OK;
}

void fill_chunk_params(ChunkParams& p, const void* q, const void* kv_cache, const int32_t* q_indptr, const int32_t* page_indices,
                       const int32_t* page_indptr, const int32_t* last_page_len, const float* slopes, const int32_t* prefix_lens,
                       int64_t nnz, int batch, int num_q_heads, int num_kv_heads, int head_dim, int page_size, int64_t num_pages,
                       int first_page_offset, float sm_scale, float softcap, int window) {
  p.q = static_cast<const uint16_t*>(q);
  p.kv = static_cast<const uint16_t*>(kv_cache);
  p.q_indptr = q_indptr;
  p.page_indices = page_indices;
  p.page_indptr = page_indptr;
  p.last_page_len = last_page_len;
  p.slopes = slopes;
  p.prefix_lens = prefix_lens;
  p.num_pages = num_pages;
  p.nnz = (int)nnz;
  p.batch = batch;
  p.hq = num_q_heads;
  p.hkv = num_kv_heads;
  p.group = num_q_heads / num_kv_heads;
  p.page_size = page_size;
  p.page_shift = 4 + page_tile_shift(page_size);
  p.first_page_offset = first_page_offset;
  p.window = window;
  const float scale = sm_scale > 0.f ? sm_scale : 1.0f / sqrtf((float)head_dim);
  p.scale_log2 = (float)((double)scale * 1.4426950408889634);
  p.cap_in = softcap > 0.f ? scale / softcap : 0.f;
  p.cap_log2 = softcap > 0.f ? (float)((double)softcap * 1.4426950408889634) : 0.f;
  double power = (double)scale * 1.4426950408889634;
  p.cap_tiny_top = kTanhTiny;
  for (int i = 0; i < 4; ++i, power *= (double)p.cap_in * p.cap_in) {
    p.cap_tiny[i] = (float)(power * kTanhTinyPoly[i]);
    // An infinite coefficient would make NaN of a score of 0, one that is lost changes the others: the next form then.
    if (!std::isnormal(p.cap_tiny[i])) p.cap_tiny_top = 0.f;
  }
}

// Row tiles of the launch, and the spans into which their keys are cut.
static int64_t chunk_slots(int64_t nnz, int batch, int group) { return nnz * group / kChunkRows + batch; }

// Few rows per sequence on average: mostly decode.
static bool mostly_decode(int64_t nnz, int batch, int group) { return nnz * group <= (int64_t)kChunkRows * batch; }

struct ChunkSpans {
  int splits, narrow, wide;  // most spans of a row tile; tiles of 64 keys in a span
};
// Wide row tiles: enough spans for every workgroup that fits on a CU (bias case of 211 row tiles, heads of 64: 2 / 3 / 4 per CU
// 45.5 / 42.5 / 44.2 us); more would only write more partial results.  Narrow ones (decode)
// leave almost nothing behind, but their sequences' lengths differ: about four times as many spans even them out (60
// sequences of 301..8201 tokens beside four prompts, 8 KV heads of 64: one span 150 us, 4 / 8 / 16 workgroups per CU 134 / 131 / 128).  No span below 4 tiles.
static ChunkSpans chunk_spans(int64_t nnz, int batch, int num_q_heads, int num_kv_heads, int max_pages_per_seq, int page_size,
                              int head_dim, int num_splits) {
  int64_t tiles = ((int64_t)max_pages_per_seq * page_size + kChunkKeys - 1) / kChunkKeys;
  if (tiles > 0x7fffffff) tiles = 0x7fffffff;  // spans are ints
  const int64_t wgs = chunk_slots(nnz, batch, num_q_heads / num_kv_heads) * num_kv_heads;
  auto span_of = [&](int64_t want, int64_t least) {
    if (want > 64 && num_splits == 0) want = 64;
    const int64_t span = (tiles + want - 1) / want;
    return (int)(span > least ? span : least);
  };
  ChunkSpans s;
  if (num_splits > 0) {
    s.narrow = s.wide = span_of(num_splits, 1);
    s.splits = num_splits;
    return s;
  }
  const int64_t places = (int64_t)chunk_wgs_per_cu(head_dim) * kNumCus;
  const int64_t wide = wgs > 0 && places > wgs ? places / wgs : 1;
  const bool decode = mostly_decode(nnz, batch, num_q_heads / num_kv_heads);
  s.wide = span_of(wide, 4);
  s.narrow = decode && wgs > 0 ? span_of((8 * kNumCus + wgs - 1) / wgs, 4) : s.wide;
  s.splits = (int)((tiles + s.narrow - 1) / s.narrow);
  return s;
}

static size_t chunk_workspace(int64_t nnz, int num_q_heads, int head_dim, int splits) {
  return splits <= 1 ? 0 : (size_t)nnz * num_q_heads * ((size_t)splits * (head_dim + 1) + 1) * sizeof(float);
}

template <int HD, bool F16>
static void launch_chunk(const ChunkAttnParams& ap, dim3 grid, bool extra, hipStream_t stream) {
  if (extra) chunk_attn_kernel<HD, F16, true><<<grid, 256, 0, stream>>>(ap);
  else chunk_attn_kernel<HD, F16, false><<<grid, 256, 0, stream>>>(ap);
  if (ap.num_splits > 1) {
    const int64_t rows = (int64_t)ap.c.nnz * ap.c.hq;
    if (rows < 4096) {
      merge_chunk_kernel<HD, F16, 1024 / HD><<<(unsigned)rows, 256, 0, stream>>>(ap);
    } else {
      const int per = 1024 / HD;
      merge_chunk_kernel<HD, F16, 1><<<(unsigned)((rows + per - 1) / per), 256, 0, stream>>>(ap);
    }
  }
}

static int chunk_attention_impl(const char* fn, bool f16, const void* q, const void* kv_cache, const int32_t* q_indptr,
                                const int32_t* page_indices, const int32_t* page_indptr, const int32_t* last_page_len,
                                const float* slopes, const int32_t* prefix_lens, void* out, float* lse, void* workspace,
                                size_t workspace_bytes, int64_t nnz, int batch, int num_q_heads, int num_kv_heads, int head_dim,
                                int page_size, int64_t num_pages, int max_pages_per_seq, int first_page_offset, float sm_scale,
                                float softcap, int window, int num_splits, kin_stream_t stream) {
  if (!out) return fail(KIN_ERR_NULL_POINTER, "%s: null pointer argument", fn);
  if (int st = check_chunk_args(fn, q, kv_cache, q_indptr, page_indices, page_indptr, last_page_len, nnz, batch, num_q_heads,
                                num_kv_heads, head_dim, page_size, num_pages, max_pages_per_seq, first_page_offset, sm_scale,
                                softcap, window, num_q_heads))  // rows are (token, head) pairs: any group
    return st;
  if (num_splits < 0 || num_splits > 1024) return fail(KIN_ERR_BAD_SHAPE, "%s: num_splits=%d must be in [0, 1024]", fn, num_splits);
  if (!aligned16(out)) return fail(KIN_ERR_MISALIGNED, "%s: out must be 16-byte aligned", fn);
  if (batch == 0 || nnz == 0) return KIN_OK;
  ChunkAttnParams ap;
  const int64_t slots = chunk_slots(nnz, batch, num_q_heads / num_kv_heads);
  if (slots * num_kv_heads > max_workgroups(256)) return fail(KIN_ERR_UNSUPPORTED, "%s: too many row tiles", fn);
  const ChunkSpans spans = chunk_spans(nnz, batch, num_q_heads, num_kv_heads, max_pages_per_seq, page_size, head_dim, num_splits);
  ap.num_splits = spans.splits;
  ap.span_narrow = spans.narrow;
  ap.span_wide = spans.wide;
  if (ap.num_splits > 1) {
    if (nnz * num_q_heads > max_workgroups(256) * (1024 / head_dim))  // the join
      return fail(KIN_ERR_UNSUPPORTED, "%s: nnz*num_q_heads is too large for %d splits", fn, ap.num_splits);
    const size_t need = chunk_workspace(nnz, num_q_heads, head_dim, ap.num_splits);
    if (!workspace || workspace_bytes < need)
      return fail(KIN_ERR_WORKSPACE, "%s: %d splits need %zu workspace bytes, got %zu", fn, ap.num_splits, need,
                  workspace ? workspace_bytes : (size_t)0);
    if (!aligned16(workspace)) return fail(KIN_ERR_MISALIGNED, "%s: workspace must be 16-byte aligned", fn);
  }
  fill_chunk_params(ap.c, q, kv_cache, q_indptr, page_indices, page_indptr, last_page_len, slopes, prefix_lens, nnz, batch,
                    num_q_heads, num_kv_heads, head_dim, page_size, num_pages, first_page_offset, sm_scale, softcap, window);
  ap.out = static_cast<uint16_t*>(out);
  ap.lse = lse;
  ap.ws_o = static_cast<float*>(workspace);
  ap.ws_lse = ap.num_splits > 1 ? ap.ws_o + (size_t)ap.num_splits * nnz * num_q_heads * head_dim : nullptr;
  ap.ws_count = ap.num_splits > 1 ? reinterpret_cast<int32_t*>(ap.ws_lse + (size_t)ap.num_splits * nnz * num_q_heads) : nullptr;
  ap.slots = (int)slots;
  const dim3 grid((unsigned)(slots * num_kv_heads), (unsigned)ap.num_splits);
  const bool extra = slopes != nullptr || softcap > 0.f;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (head_dim == kHeadDimSmall) {
    if (f16) launch_chunk<kHeadDimSmall, true>(ap, grid, extra, s);
    else launch_chunk<kHeadDimSmall, false>(ap, grid, extra, s);
  } else {
    if (f16) launch_chunk<kHeadDim, true>(ap, grid, extra, s);
    else launch_chunk<kHeadDim, false>(ap, grid, extra, s);
  }
  return check_hip(hipGetLastError(), "chunk_attn_kernel launch");
}

}  // namespace kin

extern "C" {

size_t kin_chunk_workspace_bytes(int64_t nnz, int batch, int num_q_heads, int num_kv_heads, int max_pages_per_seq,
                                 int page_size, int head_dim, int num_splits) {
  if (nnz <= 0 || batch <= 0 || num_q_heads <= 0 || num_kv_heads <= 0 || num_q_heads % num_kv_heads != 0 || max_pages_per_seq <= 0 ||
      page_size <= 0 || head_dim <= 0)
    return 0;
  return kin::chunk_workspace(nnz, num_q_heads, head_dim,
                              kin::chunk_spans(nnz, batch, num_q_heads, num_kv_heads, max_pages_per_seq, page_size, head_dim, num_splits).splits);
}

int kin_paged_chunk_attention(const kin_bf16_t* q, const kin_bf16_t* kv_cache, const int32_t* q_indptr,
                              const int32_t* page_indices, const int32_t* page_indptr, const int32_t* last_page_len,
                              const float* slopes, const int32_t* prefix_lens, kin_bf16_t* out, float* lse, void* workspace,
                              size_t workspace_bytes, int64_t nnz, int batch, int num_q_heads, int num_kv_heads, int head_dim,
                              int page_size, int64_t num_pages, int max_pages_per_seq, int first_page_offset, float sm_scale,
                              float softcap, int window, int num_splits, kin_stream_t stream) {
  return kin::chunk_attention_impl("kin_paged_chunk_attention", false, q, kv_cache, q_indptr, page_indices, page_indptr,
                                   last_page_len, slopes, prefix_lens, out, lse, workspace, workspace_bytes, nnz, batch,
                                   num_q_heads, num_kv_heads, head_dim, page_size, num_pages, max_pages_per_seq,
                                   first_page_offset, sm_scale, softcap, window, num_splits, stream);
}
int kin_paged_chunk_attention_f16(const kin_f16_t* q, const kin_f16_t* kv_cache, const int32_t* q_indptr,
                                  const int32_t* page_indices, const int32_t* page_indptr, const int32_t* last_page_len,
                                  const float* slopes, const int32_t* prefix_lens, kin_f16_t* out, float* lse, void* workspace,
                                  size_t workspace_bytes, int64_t nnz, int batch, int num_q_heads, int num_kv_heads,
                                  int head_dim, int page_size, int64_t num_pages, int max_pages_per_seq, int first_page_offset,
                                  float sm_scale, float softcap, int window, int num_splits, kin_stream_t stream) {
  return kin::chunk_attention_impl("kin_paged_chunk_attention_f16", true, q, kv_cache, q_indptr, page_indices, page_indptr,
                                   last_page_len, slopes, prefix_lens, out, lse, workspace, workspace_bytes, nnz, batch,
                                   num_q_heads, num_kv_heads, head_dim, page_size, num_pages, max_pages_per_seq,
                                   first_page_offset, sm_scale, softcap, window, num_splits, stream);
}

}  // extern "C"
