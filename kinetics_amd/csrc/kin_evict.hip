// Eviction from the paged cache by accumulated weight.  A sequence longer than its budget keeps, per KV
// head, its first sink_tokens, its newest local_tokens and, of the rest, the tokens with the largest scores
// (ties: the lowest index).  The rows that stay move up, in their order, to tokens 0 .. budget-1 of the same pages.
//
// Two kernels.  evict_select_kernel, a workgroup per (sequence, KV head): a radix search for the cut score,
// then one ordered pass that writes the list of kept tokens and moves their scores.  evict_move_kernel moves the
// K and V rows along that list, in place: a kept token never moves to a higher place, so a workgroup
// that reads a stretch of the list before it writes it, and takes the stretches in order, overwrites only
// rows that it has read.  K and V, and the parts of a row, move independently and get workgroups of their own.
// 4 sequences of 16384 to 4096 tokens, 8 heads of 128: search 19 us (32 lists, 32 workgroups: loads, an LDS histogram and two
// ordered steps of each, one behind the other), move 38 us (134 MB of rows of 256 bytes in random places, 3.5 TB/s).  96 of about
// 1100 to 1024: 11 and 12 us.  Loads under a condition are written with a clamped index: as branches, each one waited for the
// one before it (search 23 us, move 43).
#include "kin_common.h"

namespace kin {

constexpr int kEvictThreads = 1024;
constexpr int kEvictPer = 8;        // tokens per lane and step of the ordered pass
constexpr int kDigitBits = 13;      // of the radix search: sign, exponent and four bits of the fraction come first, so that mostly
constexpr int kDigits = 1 << kDigitBits;  // few keys share the cut's digit and LDS atomics, which queue up on one address, spread (11 bits: 37 us for equal scores; 24)
constexpr int kDigitsPer = kDigits / kEvictThreads;
constexpr int kMoveThreads = 1024;
constexpr int kMoveRows = 8;        // rows per lane in flight: a stretch is 128 KiB of registers
constexpr int kFewKeys = kEvictThreads / 4;  // so many keys that share the cut's first digits are ranked against one another at once
constexpr int kKeepKeys = 16;       // keys a lane keeps in registers for the search (16384 tokens; the others are read again)

struct EvictParams {
  uint16_t* kv;
  const float* scores;     // [blocks, hkv, stride]
  float* scores_out;       // the same layout; may be scores
  const int32_t* page_indices;
  const int32_t* page_indptr;
  const int32_t* last_page_len;
  const int32_t* slot_ids;
  int32_t* kept;           // [batch, hkv, budget]
  int32_t* new_lens;       // [batch]
  int64_t num_pages;
  int batch, hkv, page_size, page_shift, first_page_offset;
  int num_blocks, stride, budget, sink, local;
};

// A score as an unsigned key of the same order: -0 as +0, NaN above everything.
__device__ __forceinline__ uint32_t score_key(float x) {
  if (x != x) return 0xffffffffu;
  const uint32_t u = __float_as_uint(x + 0.f);
  return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

struct EvictSeq {
  int len, n_pages, blk;
  const int32_t* pages;
};
__device__ __forceinline__ EvictSeq evict_seq(const EvictParams& p, int b) {
  EvictSeq s;
  const int ps = p.page_indptr[b];
  s.n_pages = max(p.page_indptr[b + 1] - ps, 0);
  s.pages = p.page_indices + ps;
  const int last = min(max(p.last_page_len[b], 0), p.page_size);
  s.len = s.n_pages > 0 ? max((s.n_pages - 1) * p.page_size + last - p.first_page_offset, 0) : 0;
  s.blk = kbar_block_of(p.slot_ids, p.num_blocks, b);
  return s;
}

__global__ __launch_bounds__(kEvictThreads) void evict_select_kernel(EvictParams p) {
  __shared__ __attribute__((aligned(16))) uint32_t hist[2][kDigits];  // even and odd lanes count in places of their own
  __shared__ uint32_t pick[2];   // digit that holds the cut, keys above it
  __shared__ uint32_t wave_above[kEvictThreads / 64];
  __shared__ __attribute__((aligned(16))) uint32_t few[kFewKeys];
  __shared__ uint32_t num_few, num_keys;
  __shared__ int2 wave_sum[kEvictThreads / 64];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int b = blockIdx.x / p.hkv, h = blockIdx.x - b * p.hkv;
  const EvictSeq sq = evict_seq(p, b);
  int32_t* kept = p.kept + ((int64_t)b * p.hkv + h) * p.budget;
  const bool known = sq.blk >= 0 && sq.len <= p.stride;
  const int n = sq.len, m = p.budget - p.sink - p.local;
  if (h == 0 && tid == 0) p.new_lens[b] = known ? min(n, p.budget) : n;
  if (!known) {  // a sequence without scores keeps what it has
    for (int i = tid; i < p.budget; i += kEvictThreads) kept[i] = -1;
    return;
  }
  const int64_t at = ((int64_t)sq.blk * p.hkv + h) * p.stride;
  const float* src = p.scores + at;
  float* dst = p.scores_out + at;
  if (n <= p.budget) {
    for (int i = tid; i < p.budget; i += kEvictThreads) kept[i] = i < n ? i : -1;
    if (src != dst)
      for (int i = tid; i < n; i += kEvictThreads) dst[i] = src[i];
    return;
  }
  // The m-th largest key of the tokens sink .. n - local - 1, a digit at a time from the top (13, 13, 6 bits).
  const int c0 = p.sink, c1 = n - p.local;
  uint32_t cut = 0, above = 0;
  if (m > 0) {
    uint32_t key[kKeepKeys];
    const int mine = max((c1 - c0 - tid + kEvictThreads - 1) / kEvictThreads, 0);  // this lane's tokens: c0 + tid + j * 1024
#pragma unroll
    for (int j = 0; j < kKeepKeys; ++j) key[j] = score_key(src[min(c0 + tid + j * kEvictThreads, c1 - 1)]);  // min, not a branch: all loads at once
    auto for_keys = [&](auto f) {
#pragma unroll
      for (int j = 0; j < kKeepKeys; ++j)
        if (j < mine) f(key[j]);
      for (int j0 = kKeepKeys; j0 < mine; j0 += 8) {
        uint32_t k[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) k[j] = score_key(src[min(c0 + tid + (j0 + j) * kEvictThreads, c1 - 1)]);
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (j0 + j < mine) f(k[j]);
      }
    };
    for (int top = 32; top > 0; top -= kDigitBits) {  // bits below `top` are still open
      const int shift = max(top - kDigitBits, 0);
      for (int d = tid * 4; d < 2 * kDigits; d += kEvictThreads * 4) *reinterpret_cast<uint4*>(&hist[0][0] + d) = uint4{0, 0, 0, 0};
      __syncthreads();
      for_keys([&](uint32_t k) {
        if (top == 32 || (k >> top) == (cut >> top)) {
          const uint32_t d = (k >> shift) & ((1u << (top - shift)) - 1);
          const uint64_t here = __ballot(true);
          if (__ballot(d == (uint32_t)__builtin_amdgcn_readfirstlane((int)d)) == here) {  // one digit for all: one of them counts
            if (lane == __builtin_ctzll(here)) atomicAdd(&hist[0][d], (uint32_t)__popcll(here));
          } else {
            atomicAdd(&hist[lane & 1][d], 1u);
          }
        }
      });
      __syncthreads();
      // thread t holds 8 digits, from kDigits - 8t - 1 down: how many keys lie above them?
      const int d0 = kDigits - kDigitsPer * (tid + 1);
      uint32_t h[kDigitsPer], sum = 0;
#pragma unroll
      for (int i = 0; i < kDigitsPer; i += 4) {
        const uint4 x = *reinterpret_cast<const uint4*>(&hist[0][d0 + i]), y = *reinterpret_cast<const uint4*>(&hist[1][d0 + i]);
        h[i] = x.x + y.x;
        h[i + 1] = x.y + y.y;
        h[i + 2] = x.z + y.z;
        h[i + 3] = x.w + y.w;
        sum += h[i] + h[i + 1] + h[i + 2] + h[i + 3];
      }
      const uint32_t incl = wave_inclusive_sum(sum);
      if (lane == 63) wave_above[wave] = incl;
      __syncthreads();
      uint32_t before = above + incl - sum;
#pragma unroll
      for (int w = 0; w < kEvictThreads / 64; ++w) before += w < wave ? wave_above[w] : 0;
      if (before < (uint32_t)m && before + sum >= (uint32_t)m) {  // one thread: the cut is in its digits
#pragma unroll
        for (int i = kDigitsPer - 1; i >= 0; --i) {
          if (before < (uint32_t)m && before + h[i] >= (uint32_t)m) {
            pick[0] = d0 + i;
            pick[1] = before;
            num_keys = h[i];
          }
          before += h[i];
        }
      }
      if (tid == 0) num_few = 0;
      if (tid < kFewKeys) few[tid] = 0;
      __syncthreads();
      cut |= pick[0] << shift;
      above = pick[1];
      if (num_keys > kFewKeys || shift == 0) continue;
      // Few keys share these digits: collect them (in any order) and rank each against the others.
      for_keys([&](uint32_t k) {
        if ((k >> shift) == (cut >> shift)) {
          const uint32_t at = atomicAdd(&num_few, 1u);
          if (at < kFewKeys) few[at] = k;
        }
      });
      __syncthreads();
      // four threads to a key, each against a quarter of the others (zeros behind the last one: no score has key 0)
      const uint32_t total = num_keys, k = few[tid / 4];
      uint32_t over = 0, same = 0;
#pragma unroll 2
      for (uint32_t i = (tid & 3) * 4; i < total; i += 16) {
        const uint4 f = *reinterpret_cast<const uint4*>(few + i);
        over += (f.x > k) + (f.y > k) + (f.z > k) + (f.w > k);
        same += (f.x == k) + (f.y == k) + (f.z == k) + (f.w == k);
      }
      over += __shfl_xor(over, 1);
      same += __shfl_xor(same, 1);
      over += __shfl_xor(over, 2);
      same += __shfl_xor(same, 2);
      if (k != 0 && above + over < (uint32_t)m && above + over + same >= (uint32_t)m) {  // threads with this very key write the same
        pick[0] = k;
        pick[1] = above + over;
      }
      __syncthreads();
      cut = pick[0];
      above = pick[1];
      break;
    }
  }
  const int ties = m - (int)above;  // tokens with the cut score itself that stay, from the lowest index on
  // Ordered pass: a wave owns 64 * kEvictPer tokens of a step; place = tokens kept for good before + ties kept before.
  int sure0 = 0, tie0 = 0;
  for (int base = 0; base < n; base += kEvictThreads * kEvictPer) {
    float x[kEvictPer];
    uint64_t sure[kEvictPer], tie[kEvictPer];
    int ns = 0, nt = 0;
    const int first = base + wave * 64 * kEvictPer + lane;
#pragma unroll
    for (int j = 0; j < kEvictPer; ++j) x[j] = src[min(first + j * 64, n - 1)];
#pragma unroll
    for (int j = 0; j < kEvictPer; ++j) {
      const int i = first + j * 64;
      const uint32_t k = score_key(x[j]);
      const bool mid = i >= c0 && i < c1;
      sure[j] = __ballot(i < n && (!mid || (m > 0 && k > cut)));
      tie[j] = __ballot(mid && m > 0 && k == cut);
      ns += __popcll(sure[j]);
      nt += __popcll(tie[j]);
    }
    if (lane == 0) wave_sum[wave] = make_int2(ns, nt);
    __syncthreads();
    int s = sure0, t = tie0;
#pragma unroll
    for (int w = 0; w < kEvictThreads / 64; ++w) {
      const int2 v = wave_sum[w];
      if (w < wave) {
        s += v.x;
        t += v.y;
      }
      sure0 += v.x;
      tie0 += v.y;
    }
    __syncthreads();  // also: every score of this step is read before any place below it is written
    const uint64_t lower = (1ull << lane) - 1;
#pragma unroll
    for (int j = 0; j < kEvictPer; ++j) {
      const int i = first + j * 64;
      const int sb = s + __popcll(sure[j] & lower), tb = t + __popcll(tie[j] & lower);
      const bool keep = ((sure[j] >> lane) & 1) || (((tie[j] >> lane) & 1) && tb < ties);
      if (keep) {
        const int place = sb + min(tb, ties);
        kept[place] = i;
        dst[place] = x[j];
      }
      s += __popcll(sure[j]);
      t += __popcll(tie[j]);
    }
  }
  __syncthreads();
  for (int i = p.budget + tid; i < n; i += kEvictThreads) dst[i] = 0.f;
}

// A workgroup moves LPR * 16 bytes of every row of one (sequence, KV head, plane); the parts of a row are neighbours on one
// XCD (workgroups go to the 8 XCDs in turn), whose L2 joins their accesses into whole lines.
template <int LPR>
__global__ __launch_bounds__(kMoveThreads) void evict_move_kernel(EvictParams p, int parts, int row_bytes) {
  const int tid = threadIdx.x;
  const int xcd = blockIdx.x % kNumXcds, rest = blockIdx.x / kNumXcds;
  const int part = rest % parts;
  const int64_t list = (int64_t)(rest / parts) * kNumXcds + xcd;  // plane fastest
  if (list >= (int64_t)p.batch * p.hkv * 2) return;
  const int plane = (int)(list & 1);
  const int h = (int)((list >> 1) % p.hkv), b = (int)((list >> 1) / p.hkv);
  const EvictSeq sq = evict_seq(p, b);
  if (sq.blk < 0 || sq.len > p.stride || sq.len <= p.budget) return;
  const int32_t* kept = p.kept + ((int64_t)b * p.hkv + h) * p.budget;
  const int64_t page_bytes = 2ll * p.page_size * row_bytes;
  char* base = reinterpret_cast<char*>(p.kv) + (int64_t)plane * p.page_size * row_bytes + (int64_t)h * (row_bytes / p.hkv) +
               (part * LPR + tid % LPR) * 16;
  // Row of the cache (page * page_size + slot) that holds a token on page `id`; none: the page is outside the cache.
  constexpr uint32_t kNone = 0xffffffffu;
  auto row_of = [&](int token, int id) -> uint32_t {
    const int at = token + p.first_page_offset;
    return id >= 0 && (int64_t)id < p.num_pages ? ((uint32_t)id << p.page_shift) + (at & (p.page_size - 1)) : kNone;
  };
  auto address = [&](uint32_t row) -> char* {
    return base + (int64_t)(row >> p.page_shift) * page_bytes + (int64_t)(row & (p.page_size - 1)) * row_bytes;
  };
  constexpr int kStep = kMoveThreads / LPR;
  uint32_t from[kMoveRows], to[kMoveRows];
  auto find_rows = [&](int first) {
    // all loads of a kind at once, none behind a branch that would wait for it (tokens behind the budget: the last one's)
    int src[kMoveRows], dst[kMoveRows], from_page[kMoveRows], to_page[kMoveRows];
#pragma unroll
    for (int j = 0; j < kMoveRows; ++j) {
      dst[j] = min(first + j * kStep + tid / LPR, p.budget - 1);
      src[j] = kept[dst[j]];
      to_page[j] = sq.pages[(dst[j] + p.first_page_offset) >> p.page_shift];
    }
#pragma unroll
    for (int j = 0; j < kMoveRows; ++j) from_page[j] = sq.pages[(src[j] + p.first_page_offset) >> p.page_shift];
#pragma unroll
    for (int j = 0; j < kMoveRows; ++j) {
      // tokens in front of the first gap stay where they are
      const bool move = src[j] != dst[j] && first + j * kStep + tid / LPR < p.budget;
      from[j] = move ? row_of(src[j], from_page[j]) : kNone;
      to[j] = move ? row_of(dst[j], to_page[j]) : kNone;
    }
  };
  find_rows(p.sink);
  for (int first = p.sink; first < p.budget; first += kStep * kMoveRows) {
    u32x4 v[kMoveRows];
    char* dst[kMoveRows];
#pragma unroll
    for (int j = 0; j < kMoveRows; ++j) {
      const bool move = from[j] != kNone && to[j] != kNone;
      dst[j] = move ? address(to[j]) : nullptr;
      if (move) v[j] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(address(from[j])));
    }
    if (first + kStep * kMoveRows < p.budget) find_rows(first + kStep * kMoveRows);  // of the next stretch, while these rows arrive
    __builtin_amdgcn_s_waitcnt(0);         // every row of the stretch is in registers ...
    __syncthreads();                       // ... in all waves, before any of them is overwritten
#pragma unroll
    for (int j = 0; j < kMoveRows; ++j)
      if (dst[j]) *reinterpret_cast<u32x4*>(dst[j]) = v[j];
  }
}

static int evict_tokens_impl(const char* fn, void* kv_cache, const float* scores, float* scores_out, const int32_t* page_indices,
                             const int32_t* page_indptr, const int32_t* last_page_len, int32_t* kept, int32_t* new_lens,
                             int batch, int num_kv_heads, int head_dim, int page_size, int64_t num_pages, int first_page_offset,
                             int budget, int sink_tokens, int local_tokens, int score_blocks, int score_stride,
                             const int32_t* slot_ids, kin_stream_t stream) {
  if (!kv_cache || !scores || !scores_out || !page_indices || !page_indptr || !last_page_len || !kept || !new_lens)
    return fail(KIN_ERR_NULL_POINTER, "%s: null pointer argument", fn);
  if (int st = check_common_dims(fn, batch, num_kv_heads, num_kv_heads, head_dim, page_size, true)) return st;
  if (int st = check_first_page_offset(fn, first_page_offset, page_size)) return st;
  if (num_pages < 1) return fail(KIN_ERR_BAD_SHAPE, "%s: num_pages=%lld must be >= 1", fn, (long long)num_pages);
  if (sink_tokens < 0 || local_tokens < 0 || budget < 1 || (int64_t)sink_tokens + local_tokens > budget)
    return fail(KIN_ERR_BAD_SHAPE, "%s: budget=%d must be positive and hold sink_tokens=%d and local_tokens=%d", fn, budget,
                sink_tokens, local_tokens);
  if (score_stride < 1 || score_blocks < 0 || (!slot_ids && score_blocks < batch) || (slot_ids && score_blocks < 1))
    return fail(KIN_ERR_BAD_SHAPE, "%s: scores of %d rows of %d entries for batch=%d", fn, score_blocks, score_stride, batch);
  if (!aligned16(kv_cache)) return fail(KIN_ERR_MISALIGNED, "%s: kv_cache must be 16-byte aligned", fn);
  if (num_pages > 0xffffffffLL / page_size - 1)
    return fail(KIN_ERR_UNSUPPORTED, "%s: num_pages=%lld is too many", fn, (long long)num_pages);
  // Bytes of a row per workgroup: whole lines of 128 if that makes a workgroup for every CU, else 64, else 32 (4 x 16384 to
  // 4096 tokens of 8 heads, 128 / 64 / 32 bytes: 70 / 61 / 74 us; 96 of about 1100 to 1024, one head: 25 / 28 / 36 us; one
  // sequence of 32768 to 4096: 72 / 62 / 56 us).
  const int64_t lists = ((int64_t)batch * num_kv_heads * 2 + kNumXcds - 1) / kNumXcds * kNumXcds;
  int part_bytes = 128;
  while (part_bytes > 32 && lists * (head_dim * 2 / part_bytes) < kNumCus) part_bytes /= 2;
  const int parts = head_dim * 2 / part_bytes;
  // both kernels before either is launched
  if (lists * parts > max_workgroups(kMoveThreads) || (int64_t)batch * num_kv_heads > max_workgroups(kEvictThreads))
    return fail(KIN_ERR_UNSUPPORTED, "%s: batch*num_kv_heads is too large", fn);
  if (batch == 0) return KIN_OK;
  EvictParams p;
  p.kv = static_cast<uint16_t*>(kv_cache);
  p.scores = scores;
  p.scores_out = scores_out;
  p.page_indices = page_indices;
  p.page_indptr = page_indptr;
  p.last_page_len = last_page_len;
  p.slot_ids = slot_ids;
  p.kept = kept;
  p.new_lens = new_lens;
  p.num_pages = num_pages;
  p.batch = batch;
  p.hkv = num_kv_heads;
  p.page_size = page_size;
  p.page_shift = 4 + page_tile_shift(page_size);
  p.first_page_offset = first_page_offset;
  p.num_blocks = score_blocks;
  p.stride = score_stride;
  p.budget = budget;
  p.sink = sink_tokens;
  p.local = local_tokens;
  hipStream_t s = static_cast<hipStream_t>(stream);
  evict_select_kernel<<<(unsigned)(batch * num_kv_heads), kEvictThreads, 0, s>>>(p);
  if (int st = check_hip(hipGetLastError(), "evict_select_kernel launch")) return st;
  const unsigned grid = (unsigned)(lists * parts);
  const int row_bytes = num_kv_heads * head_dim * 2;
  if (part_bytes == 128) evict_move_kernel<8><<<grid, kMoveThreads, 0, s>>>(p, parts, row_bytes);
  else if (part_bytes == 64) evict_move_kernel<4><<<grid, kMoveThreads, 0, s>>>(p, parts, row_bytes);
  else evict_move_kernel<2><<<grid, kMoveThreads, 0, s>>>(p, parts, row_bytes);
  return check_hip(hipGetLastError(), "evict_move_kernel launch");
}

}  // namespace kin

extern "C" {

/* Rows are moved as bytes: bfloat16 and float16 caches alike. */
int kin_evict_tokens(void* kv_cache, const float* scores, float* scores_out, const int32_t* page_indices,
                     const int32_t* page_indptr, const int32_t* last_page_len, int32_t* kept, int32_t* new_lens, int batch,
                     int num_kv_heads, int head_dim, int page_size, int64_t num_pages, int first_page_offset, int budget,
                     int sink_tokens, int local_tokens, int score_blocks, int score_stride, const int32_t* slot_ids,
                     kin_stream_t stream) {
  return kin::evict_tokens_impl("kin_evict_tokens", kv_cache, scores, scores_out, page_indices, page_indptr, last_page_len, kept,
                                new_lens, batch, num_kv_heads, head_dim, page_size, num_pages, first_page_offset, budget,
                                sink_tokens, local_tokens, score_blocks, score_stride, slot_ids, stream);
}

}  // extern "C"
