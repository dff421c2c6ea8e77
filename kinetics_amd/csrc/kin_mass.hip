// The weight that every cached token received from a chunk of new tokens:
//   scores[b, h, j] += sum over the new rows p and the query heads g of the group that see token j of
//                      exp(s_pgj - lse_pg),
// with the scores s of kin_chunk.h and the log-sum-exp that the attention over the same chunk wrote.
//
// A workgroup owns 128 tokens of one (sequence, KV head), each of four waves 32 of them: their keys are read
// once and stay in registers as the matrix unit's operand, and the rows pass by, 64 at a time, through two
// stages in LDS that all four waves read.  With many rows (RW = 2) there are eight waves, two for the same 32 tokens, and 128 rows to a
// stage: each of the two takes every other 32 rows, and their sums are added at the end.  S = Q K^T on v_mfma_f32_32x32x16 leaves lane l the scores of ONE token (column l % 32) against
// 16 rows, so the sum over rows is a sum over registers: no atomics, one owner per token, and the order of
// the additions never changes.  With many rows the vector unit bounds it, one exponential and seven slots per (row, token) with a
// cap: 2048 rows of 8192 tokens, 32 heads on 8: 230 us, the vector unit 79 % busy.  With single tokens it is the reading of the keys: 256 sequences of
// 1025..8193, 83 us, 3.7 TB/s.  (Rows straight from L2 instead of through LDS: 469 us for the first.)
#include "kin_chunk.h"

namespace kin {

constexpr int kMassKeys = 128;  // tokens of a workgroup
constexpr int kMassMaxGroup = 128;  // so that the short division of its rows is exact

struct MassParams {
  ChunkParams c;
  const float* lse;         // [nnz, hq]
  float* scores;            // [blocks, hkv, stride]
  const int32_t* slot_ids;  // [batch] or null
  int num_blocks, stride;
  int key_tiles;            // workgroups per (sequence, KV head)
};

template <int HD, bool F16, bool EXTRA, int RW>
__global__ __launch_bounds__(256 * RW, 2 * RW) void attention_mass_kernel(MassParams mp) {
  constexpr int kRowB = HD * 2;
  constexpr int kMassRows = 64 * RW;  // rows of a staged tile
  constexpr int kStageB = kMassRows * kRowB;
  constexpr int CPR = HD / 8, kLoads = 64 * CPR / 256;  // LDS-direct loads per wave and stage
  struct Shared {  // the stages first: LDS-direct loads reach 64 KiB
    unsigned char lds[2 * kStageB];
    float lse[2][kMassRows], slope[2][kMassRows];
    int hi[2][kMassRows];
    float sum[RW][kMassKeys];
  };
  __shared__ __attribute__((aligned(16))) Shared sh;
  unsigned char* lds = sh.lds;
  auto& lse_sh = sh.lse;
  auto& slope_sh = sh.slope;
  auto& hi_sh = sh.hi;
  auto& sum_sh = sh.sum;
  const ChunkParams& p = mp.c;
  const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5, col = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int kw = wave & 3, rw = wave >> 2;  // which 32 tokens, and which share of the rows, the wave takes
  const int h = blockIdx.x % p.hkv;
  const int rest = blockIdx.x / p.hkv;
  const int b = rest / mp.key_tiles;
  const int blk = kbar_block_of(mp.slot_ids, mp.num_blocks, b);
  if (blk < 0) return;
  const ChunkSeq sq = chunk_seq(p, b);
  if (sq.n == 0 || sq.len > mp.stride) return;
  const int rows = sq.n * p.group, off = p.first_page_offset, end = sq.len + off;
  const int base = sq.len - sq.n;  // position of the first row
  float* dst = mp.scores + ((int64_t)blk * p.hkv + h) * mp.stride;
  const char* qh = reinterpret_cast<const char*>(p.q) + ((int64_t)sq.e0 * p.hq + h * p.group) * kRowB;
  const int tok_bytes = p.hq * kRowB;

  for (int tile = rest % mp.key_tiles; tile * kMassKeys < end; tile += mp.key_tiles) {
    const int wg_slot0 = tile * kMassKeys;
    const int slot0 = wg_slot0 + kw * 32;  // first token slot of the wave
    const int slot = slot0 + col;
    // this lane's key: chunk 2k + half of its row for step k
    uint4 key[HD / 16];
    int id = -1;
    if (slot < end && slot >= off) id = sq.pages[slot >> p.page_shift];
    const bool ok = id >= 0 && (int64_t)id < p.num_pages;
    const int64_t krow = ((int64_t)(ok ? id : 0) * 2 * p.page_size + (slot & (p.page_size - 1))) * p.hkv + h;
    const uint4* src = reinterpret_cast<const uint4*>(p.kv + krow * HD);
#pragma unroll
    for (int k = 0; k < HD / 16; ++k) key[k] = ok ? src[2 * k + half] : uint4{0, 0, 0, 0};
    const bool all_keys = __ballot(!ok) == 0;

    // rows that can see one of the workgroup's tokens: all of them below the prefix, else from the first token's own position
    // to the end of the last one's window; rows in front of the sequence see nothing
    int i0 = 0, i1 = sq.n;
    if (wg_slot0 >= sq.prefix + off) {
      i0 = max(wg_slot0 - off - base, 0);
      if (p.window > 0) i1 = (int)min((int64_t)sq.n, (int64_t)(wg_slot0 + kMassKeys - 1 - off) + p.window - base);
    }
    i0 = max(i0, -base);
    const int first = i0 * p.group, n_stages = i1 > i0 ? ((i1 - i0) * p.group + kMassRows - 1) / kMassRows : 0;
    const int last = min(i1 * p.group, rows);  // one past the last row to count

    // Rows of a stage as (token, head): x = the head of the stage's first row plus the row, below group + 128, so that
    // x / group is a product and a shift.
    const uint32_t magic = 65536u / p.group + 1;
    auto split = [&](int x, int& q, int& g) {
      q = (int)((uint32_t)x * magic >> 16);
      g = x - q * p.group;
    };
    // Stage `st`: kMassRows rows, swizzled; rows that do not count lie outside the descriptor's 1 GiB and read as zeros.
    auto stage_rows = [&](int st) {
      const int r0 = first + st * kMassRows;
      const int i = r0 / p.group, g0 = r0 - i * p.group;
      const u32x4 rs = rsrc_words(qh + (int64_t)i * tok_bytes, 0x40000000);
      const uint32_t at = lds_offset(lds + (st & 1) * kStageB);
#pragma unroll
      for (int j = 0; j < kLoads; ++j) {
        const int rr = (wave * kLoads + j) * (64 / CPR) + lane / CPR;  // row of the stage
        int di, g;
        split(g0 + rr, di, g);
        const int o = di * tok_bytes + g * kRowB + (((lane & (CPR - 1)) ^ row_swizzle<HD>(rr & 15)) * 16);
        lds_load_16<false>(rs, at + (wave * kLoads + j) * 1024, r0 + rr < last ? o : 0x7fff0000);
      }
    };
    // its rows' log-sum-exp (log2), token slots and slopes: one row per thread of the first waves
    float z = 0.f, sl = 0.f;
    int hi = 0;
    auto fetch_row = [&](int st) {
      const int r0 = first + st * kMassRows, i0s = r0 / p.group;
      int di, g;
      split(r0 - i0s * p.group + tid, di, g);
      const int i = i0s + di;
      const bool valid = r0 + tid < last;
      z = valid ? mp.lse[(int64_t)(sq.e0 + i) * p.hq + h * p.group + g] * kLog2e : INFINITY;
      if (z == kNegInf) z = INFINITY;  // a row that saw nothing gives nothing
      hi = base + i + off;
      if constexpr (EXTRA) sl = (p.slopes && valid) ? p.slopes[h * p.group + g] * kLog2e : 0.f;
    };
    auto put_row = [&](int st) {
      lse_sh[st & 1][tid] = z;
      hi_sh[st & 1][tid] = hi;
      if constexpr (EXTRA) slope_sh[st & 1][tid] = sl;
    };

    float sum = 0.f;
    if (n_stages > 0) {
      stage_rows(0);
      if (tid < kMassRows) {
        fetch_row(0);
        put_row(0);
      }
    }
    for (int st = 0; st < n_stages; ++st) {
      __builtin_amdgcn_s_waitcnt(0);  // this wave's part of the stage is in; behind the barrier, every wave's
      __syncthreads();
      const bool more = st + 1 < n_stages;
      if (more) {
        stage_rows(st + 1);
        if (tid < kMassRows) fetch_row(st + 1);
      }
      const unsigned char* qs = lds + (st & 1) * kStageB;
#pragma unroll
      for (int t2 = 0; t2 < 2; ++t2) {
        const int t = t2 * RW + rw;
        const int r0 = first + st * kMassRows + t * 32;
        const int pos0 = base + r0 / p.group, pos1 = base + min(r0 + 31, last - 1) / p.group;
        if (r0 >= last || slot0 >= end) break;
        if (slot0 >= sq.prefix + off && slot0 - off > pos1) continue;  // behind all of these rows
        floatx16 s;
#pragma unroll
        for (int e = 0; e < 16; ++e) s[e] = 0.f;
        // Behind the last row: that row once more, for its lse of +inf to take out.  (A row of zeros would be NaN against an
        // infinite key; masking the scores instead costs 256 single tokens 83 -> 98 us, this 85.)
        const int rc = min(col, last - 1 - r0);
        const unsigned char* qrow = qs + (t * 32 + rc) * kRowB;
        const int swz = row_swizzle<HD>(rc & 15);
#pragma unroll
        for (int k = 0; k < HD / 16; ++k) {
          const uint4 a = *reinterpret_cast<const uint4*>(qrow + (((2 * k + half) ^ swz) * 16));
          s = mfma_32x32x16<F16>(a, key[k], s);
        }
        const bool seen = all_keys && ((slot0 + 31 - off <= pos0 && (p.window == 0 || pos1 - (slot0 - off) < p.window)) ||
                                       slot0 + 31 < sq.prefix + off);
        const float* zs = lse_sh[st & 1] + t * 32;
        const int* hs = hi_sh[st & 1] + t * 32;
        if constexpr (EXTRA) {
          cap_scores<true>(p, s, [&](int e) { return zs[acc_row(e, half)]; });
          if (p.slopes) {
            const float* ss = slope_sh[st & 1] + t * 32;
#pragma unroll
            for (int e = 0; e < 16; ++e) s[e] = fmaf(-ss[acc_row(e, half)], (float)abs(hs[acc_row(e, half)] - slot), s[e]);
          }
        } else {
#pragma unroll
          for (int e = 0; e < 16; ++e) s[e] = fmaf(s[e], p.scale_log2, -zs[acc_row(e, half)]);
        }
        if (!seen) {
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const int at = hs[acc_row(e, half)];
            const bool on = ok & (((slot <= at) & ((p.window == 0) | (at - slot < p.window))) | (slot < sq.prefix + off));
            s[e] = on ? s[e] : kNegInf;
          }
        }
        float part = 0.f;
#pragma unroll
        for (int e = 0; e < 16; ++e) part += fast_exp2(s[e]);
        sum += part;
      }
      if (more && tid < kMassRows) put_row(st + 1);
    }
    sum += other_half(sum);
    __syncthreads();  // the staging area is free for the next tile of keys
    if constexpr (RW > 1) {
      if (half == 0) sum_sh[rw][kw * 32 + col] = sum;
      __syncthreads();
      if (rw == 0)
        for (int x = 1; x < RW; ++x) sum += sum_sh[x][kw * 32 + col];
    }
    if (rw == 0 && half == 0 && slot >= off && slot < end) dst[slot - off] += sum;
  }
}

template <int HD, bool F16, bool EXTRA>
static void launch_mass(const MassParams& mp, unsigned grid, bool many_rows, hipStream_t s) {
  if (many_rows) attention_mass_kernel<HD, F16, EXTRA, 2><<<grid, 512, 0, s>>>(mp);
  else attention_mass_kernel<HD, F16, EXTRA, 1><<<grid, 256, 0, s>>>(mp);
}
template <int HD, bool F16>
static void launch_mass(const MassParams& mp, unsigned grid, bool extra, bool many_rows, hipStream_t s) {
  if (extra) launch_mass<HD, F16, true>(mp, grid, many_rows, s);
  else launch_mass<HD, F16, false>(mp, grid, many_rows, s);
}

static int attention_mass_impl(const char* fn, bool f16, const void* q, const void* kv_cache, const float* lse, float* scores,
                               const int32_t* q_indptr, const int32_t* page_indices, const int32_t* page_indptr,
                               const int32_t* last_page_len, const float* slopes, const int32_t* prefix_lens, int64_t nnz,
                               int batch, int num_q_heads, int num_kv_heads, int head_dim, int page_size, int64_t num_pages,
                               int max_pages_per_seq, int first_page_offset, float sm_scale, float softcap, int window,
                               int score_blocks, int score_stride, const int32_t* slot_ids, kin_stream_t stream) {
  if (!lse || !scores) return fail(KIN_ERR_NULL_POINTER, "%s: null pointer argument", fn);
  if (int st = check_chunk_args(fn, q, kv_cache, q_indptr, page_indices, page_indptr, last_page_len, nnz, batch, num_q_heads,
                                num_kv_heads, head_dim, page_size, num_pages, max_pages_per_seq, first_page_offset, sm_scale,
                                softcap, window, kMassMaxGroup))
    return st;
  if (score_stride < 1 || score_blocks < 0 || (!slot_ids && score_blocks < batch) || (slot_ids && score_blocks < 1))
    return fail(KIN_ERR_BAD_SHAPE, "%s: scores of %d rows of %d entries for batch=%d", fn, score_blocks, score_stride, batch);
  if (batch == 0 || nnz == 0) return KIN_OK;
  MassParams mp;
  fill_chunk_params(mp.c, q, kv_cache, q_indptr, page_indices, page_indptr, last_page_len, slopes, prefix_lens, nnz, batch,
                    num_q_heads, num_kv_heads, head_dim, page_size, num_pages, first_page_offset, sm_scale, softcap, window);
  mp.lse = lse;
  mp.scores = scores;
  mp.slot_ids = slot_ids;
  mp.num_blocks = score_blocks;
  mp.stride = score_stride;
  const bool extra = slopes != nullptr || softcap > 0.f;
  const bool many_rows = nnz * mp.c.group > 64 * (int64_t)batch;  // on average more than a stage of the small form
  // A workgroup for every tile of the longest page list, or as many as a launch can have: they walk on.
  const int64_t lists = (int64_t)batch * num_kv_heads, most = max_workgroups(many_rows ? 512 : 256) / lists;
  if (most < 1) return fail(KIN_ERR_UNSUPPORTED, "%s: batch*num_kv_heads=%lld is too large", fn, (long long)lists);
  const int64_t tiles = ((int64_t)max_pages_per_seq * page_size + kMassKeys - 1) / kMassKeys;
  mp.key_tiles = (int)(tiles < most ? tiles : most);
  const int64_t grid = lists * mp.key_tiles;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (head_dim == kHeadDimSmall) {
    if (f16) launch_mass<kHeadDimSmall, true>(mp, (unsigned)grid, extra, many_rows, s);
    else launch_mass<kHeadDimSmall, false>(mp, (unsigned)grid, extra, many_rows, s);
  } else {
    if (f16) launch_mass<kHeadDim, true>(mp, (unsigned)grid, extra, many_rows, s);
    else launch_mass<kHeadDim, false>(mp, (unsigned)grid, extra, many_rows, s);
  }
  return check_hip(hipGetLastError(), "attention_mass_kernel launch");
}

}  // namespace kin

extern "C" {

int kin_attention_mass(const kin_bf16_t* q, const kin_bf16_t* kv_cache, const float* lse, float* scores, const int32_t* q_indptr,
                       const int32_t* page_indices, const int32_t* page_indptr, const int32_t* last_page_len,
                       const float* slopes, const int32_t* prefix_lens, int64_t nnz, int batch, int num_q_heads,
                       int num_kv_heads, int head_dim, int page_size, int64_t num_pages, int max_pages_per_seq,
                       int first_page_offset, float sm_scale, float softcap, int window, int score_blocks, int score_stride,
                       const int32_t* slot_ids, kin_stream_t stream) {
  return kin::attention_mass_impl("kin_attention_mass", false, q, kv_cache, lse, scores, q_indptr, page_indices, page_indptr,
                                  last_page_len, slopes, prefix_lens, nnz, batch, num_q_heads, num_kv_heads, head_dim, page_size,
                                  num_pages, max_pages_per_seq, first_page_offset, sm_scale, softcap, window, score_blocks,
                                  score_stride, slot_ids, stream);
}
int kin_attention_mass_f16(const kin_f16_t* q, const kin_f16_t* kv_cache, const float* lse, float* scores,
                           const int32_t* q_indptr, const int32_t* page_indices, const int32_t* page_indptr,
                           const int32_t* last_page_len, const float* slopes, const int32_t* prefix_lens, int64_t nnz, int batch,
                           int num_q_heads, int num_kv_heads, int head_dim, int page_size, int64_t num_pages,
                           int max_pages_per_seq, int first_page_offset, float sm_scale, float softcap, int window,
                           int score_blocks, int score_stride, const int32_t* slot_ids, kin_stream_t stream) {
  return kin::attention_mass_impl("kin_attention_mass_f16", true, q, kv_cache, lse, scores, q_indptr, page_indices, page_indptr,
                                  last_page_len, slopes, prefix_lens, nnz, batch, num_q_heads, num_kv_heads, head_dim, page_size,
                                  num_pages, max_pages_per_seq, first_page_offset, sm_scale, softcap, window, score_blocks,
                                  score_stride, slot_ids, stream);
}

}  // extern "C"
