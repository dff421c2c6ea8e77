// The weight that every cached token received from a chunk of new tokens:
//   scores[b, h, j] += sum over the new rows p and the query heads g of the group that see token j of
//                      exp(s_pgj - lse_pg),
// with the scores s of kin_chunk.h and the log-sum-exp that the attention over the same chunk wrote.
//
// A workgroup owns 128 tokens of one (sequence, KV head), each of its 4 waves 32 of them: their keys are read
// once and stay in registers as the matrix unit's operand, and the rows pass by 32 at a time (they come
// from L2).  S = Q K^T on v_mfma_f32_32x32x16 leaves lane l the scores of ONE token (column l % 32) against
// 16 rows, so the sum over rows is a sum over registers: no atomics, one owner per token, and the order of
// the additions never changes.  One exponential per (row, token): with many rows that is what bounds it.
#include "kin_chunk.h"

namespace kin {

constexpr int kMassKeys = 128;

struct MassParams {
  ChunkParams c;
  const float* lse;         // [nnz, hq]
  float* scores;            // [blocks, hkv, stride]
  const int32_t* slot_ids;  // [batch] or null
  int num_blocks, stride;
  int key_tiles;            // workgroups per (sequence, KV head)
};

template <int HD, bool F16, bool EXTRA>
__global__ __launch_bounds__(256, 2) void attention_mass_kernel(MassParams mp) {
  __shared__ __attribute__((aligned(16))) float sm[4][3][32];
  const ChunkParams& p = mp.c;
  const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5, col = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int h = blockIdx.x % p.hkv;
  const int rest = blockIdx.x / p.hkv;
  const int b = rest / mp.key_tiles;
  const int blk = kbar_block_of(mp.slot_ids, mp.num_blocks, b);
  if (blk < 0) return;
  const ChunkSeq sq = chunk_seq(p, b);
  if (sq.n == 0 || sq.len > mp.stride) return;
  const int rows = sq.n * p.group, off = p.first_page_offset, end = sq.len + off;
  float* lse_sh = sm[wave][0];
  int* hi_sh = reinterpret_cast<int*>(sm[wave][1]);
  float* slope_sh = sm[wave][2];
  float* dst = mp.scores + ((int64_t)blk * p.hkv + h) * mp.stride;

  for (int tile = rest % mp.key_tiles; tile * kMassKeys < end; tile += mp.key_tiles) {
    const int slot0 = tile * kMassKeys + wave * 32;  // first token slot of the wave
    if (slot0 >= end) continue;
    const int slot = slot0 + col;
    // this lane's key: chunk 2k + half of its row for step k
    uint4 key[HD / 16];
    int id = -1;
    if (slot < end && slot >= off) id = sq.pages[slot >> p.page_shift];
    const bool ok = id >= 0 && (int64_t)id < p.num_pages;
    const int64_t row = ((int64_t)(ok ? id : 0) * 2 * p.page_size + (slot & (p.page_size - 1))) * p.hkv + h;
    const uint4* src = reinterpret_cast<const uint4*>(p.kv + row * HD);
#pragma unroll
    for (int k = 0; k < HD / 16; ++k) key[k] = ok ? src[2 * k + half] : uint4{0, 0, 0, 0};

    // rows that can see one of the wave's tokens: all of them below the prefix, else from the first token's own position to
    // the end of the last one's window
    const int base = sq.len - sq.n;
    int i0 = 0, i1 = sq.n;
    if (slot0 >= sq.prefix + off) {
      i0 = max(slot0 - off - base, 0);
      if (p.window > 0) i1 = (int)min((int64_t)sq.n, (int64_t)(slot0 + 31 - off) + p.window - base);
    }
    i0 = max(i0, -base);  // rows in front of the sequence see nothing
    float sum = 0.f;
    for (int r0 = i0 * p.group; r0 < i1 * p.group; r0 += 32) {
      const int r = r0 + col;
      const bool valid = r < rows;
      const int i = valid ? r / p.group : 0, g = valid ? r - i * p.group : 0;
      const int64_t hq = (int64_t)(sq.e0 + i) * p.hq + h * p.group + g;
      const uint4* qs = reinterpret_cast<const uint4*>(p.q + hq * HD);
      floatx16 s;
#pragma unroll
      for (int e = 0; e < 16; ++e) s[e] = 0.f;
      uint4 a[HD / 16];
#pragma unroll
      for (int k = 0; k < HD / 16; ++k) a[k] = valid ? qs[2 * k + half] : uint4{0, 0, 0, 0};
      float z = valid ? mp.lse[hq] * kLog2e : INFINITY;
      if (z == kNegInf) z = INFINITY;  // a row that saw nothing gives nothing
      if (half == 0) {
        lse_sh[col] = z;
        hi_sh[col] = base + i + off;
        if constexpr (EXTRA) slope_sh[col] = (p.slopes && valid) ? p.slopes[h * p.group + g] * kLog2e : 0.f;
      }
#pragma unroll
      for (int k = 0; k < HD / 16; ++k) s = mfma_32x32x16<F16>(a[k], key[k], s);
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int e = 0; e < 16; e += 4) {
        const int rr = acc_row(e, half);
        const float4 z4 = *reinterpret_cast<const float4*>(lse_sh + rr);
        const int4 h4 = *reinterpret_cast<const int4*>(hi_sh + rr);
        const float zz[4] = {z4.x, z4.y, z4.z, z4.w};
        const int hh[4] = {h4.x, h4.y, h4.z, h4.w};
        float sl[4] = {0.f, 0.f, 0.f, 0.f};
        if constexpr (EXTRA) {
          const float4 s4 = *reinterpret_cast<const float4*>(slope_sh + rr);
          sl[0] = s4.x; sl[1] = s4.y; sl[2] = s4.z; sl[3] = s4.w;
        }
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const float y = EXTRA ? chunk_score(p, s[e + x], sl[x], abs(hh[x] - slot)) - zz[x] : fmaf(s[e + x], p.scale_log2, -zz[x]);
          const bool on = ok & (((slot <= hh[x]) & ((p.window == 0) | (hh[x] - slot < p.window))) | (slot < sq.prefix + off));
          sum += on ? fast_exp2(y) : 0.f;
        }
      }
      __builtin_amdgcn_wave_barrier();
    }
    sum += other_half(sum);
    if (half == 0 && slot >= off && slot < end) dst[slot - off] += sum;
  }
}

template <int HD, bool F16>
static void launch_mass(const MassParams& mp, unsigned grid, bool extra, hipStream_t s) {
  if (extra) attention_mass_kernel<HD, F16, true><<<grid, 256, 0, s>>>(mp);
  else attention_mass_kernel<HD, F16, false><<<grid, 256, 0, s>>>(mp);
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
                                softcap, window))
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
  mp.key_tiles = (int)(((int64_t)max_pages_per_seq * page_size + kMassKeys - 1) / kMassKeys);
  const int64_t grid = (int64_t)batch * num_kv_heads * mp.key_tiles;
  if (grid > 0x7fffffffLL) return fail(KIN_ERR_UNSUPPORTED, "%s: batch*num_kv_heads*max_pages_per_seq is too large", fn);
  const bool extra = slopes != nullptr || softcap > 0.f;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (head_dim == kHeadDimSmall) {
    if (f16) launch_mass<kHeadDimSmall, true>(mp, (unsigned)grid, extra, s);
    else launch_mass<kHeadDimSmall, false>(mp, (unsigned)grid, extra, s);
  } else {
    if (f16) launch_mass<kHeadDim, true>(mp, (unsigned)grid, extra, s);
    else launch_mass<kHeadDim, false>(mp, (unsigned)grid, extra, s);
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
