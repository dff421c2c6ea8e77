// What the operators over a chunk of new tokens share (attention of the chunk, and the weight
// every cached token received from it): the ragged batch, which tokens a row sees, and the form
// of the scores.
//
// Sequence b holds L tokens after the append, the last n of them new (n = its rows of q).  Row i
// stands at position p = L - n + i and sees token j when
//     j < prefix[b]   or   ( j <= p  and  (window == 0  or  p - j < window) ).
// Its score is  s = sm_scale * q.k,  capped:  s = cap * tanh(s / cap),  then biased by distance:
// s -= slope[head] * |p - j|.  Everything is kept in units of log2 (scores times log2 e), so that
// a weight is one exp2.
//
// Rows of one KV head are packed as r = i * group + g: the group's query heads share every key
// that is loaded, and a single new token is simply a tile with `group` rows.
#pragma once

#include "kin_attend.h"

namespace kin {

typedef float floatx16 __attribute__((ext_vector_type(16)));
typedef float floatx2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

constexpr float kLog2e = 1.4426950408889634f;

struct ChunkParams {
  const uint16_t* q;              // [nnz, hq, D]
  const uint16_t* kv;
  const int32_t* q_indptr;        // [batch + 1]
  const int32_t* page_indices;
  const int32_t* page_indptr;     // [batch + 1]
  const int32_t* last_page_len;   // [batch]
  const float* slopes;            // [hq] or null
  const int32_t* prefix_lens;     // [batch] or null
  int64_t num_pages;
  int nnz, batch, hq, hkv, group;
  int page_size, page_shift;      // page_size == 1 << page_shift
  int first_page_offset, window;
  float scale_log2;               // sm_scale * log2 e
  float cap_in, cap_log2;         // sm_scale / cap, cap * log2 e (cap_log2 == 0: no cap)
  float cap_tiny[4];              // scale_log2 * kTanhTinyPoly[i] * cap_in^(2i): a small capped score straight from the raw product
  float cap_tiny_top;             // below this part of the cap: kTanhTiny; 0 where cap_tiny leaves fp32's range
};

// One sequence of the batch as the kernels see it; positions are token indices.
struct ChunkSeq {
  int e0, n;        // first row of q, new tokens
  int len;          // tokens after the append
  int prefix;       // tokens every row sees
  int n_pages;
  const int32_t* pages;
};

// From the raw table entries of one sequence.
__device__ __forceinline__ ChunkSeq make_chunk_seq(const ChunkParams& p, int e0, int e1, int ps, int pe, int last, int prefix) {
  ChunkSeq s;
  s.e0 = min(max(e0, 0), p.nnz);
  s.n = min(max(e1, s.e0), p.nnz) - s.e0;
  s.n_pages = max(pe - ps, 0);
  s.pages = p.page_indices + ps;
  last = min(max(last, 0), p.page_size);
  s.len = s.n_pages > 0 ? max((s.n_pages - 1) * p.page_size + last - p.first_page_offset, 0) : 0;
  s.prefix = min(max(prefix, 0), s.len);
  return s;
}
__device__ __forceinline__ ChunkSeq chunk_seq(const ChunkParams& p, int b) {
  return make_chunk_seq(p, p.q_indptr[b], p.q_indptr[b + 1], p.page_indptr[b], p.page_indptr[b + 1], p.last_page_len[b],
                        p.prefix_lens ? p.prefix_lens[b] : 0);
}

// The token slots (tokens shifted by the first page's padding) that one row sees:
// [first, prefix) and [lo, hi].  A row in front of the sequence (more rows than tokens) sees none.
struct RowSpan {
  int lo, hi, prefix;
};
__device__ __forceinline__ RowSpan row_span(const ChunkParams& p, const ChunkSeq& s, int i, bool valid) {
  const int pos = s.len - s.n + i;
  RowSpan r{0, -1, 0};
  if (valid && pos >= 0) {
    r.hi = pos + p.first_page_offset;
    r.lo = (p.window > 0 ? max(pos - p.window + 1, 0) : 0) + p.first_page_offset;
    r.prefix = s.prefix + p.first_page_offset;
  }
  return r;
}
__device__ __forceinline__ bool row_sees(const RowSpan& r, int first, int slot) {
  return ((slot <= r.hi) & (slot >= r.lo)) | ((slot < r.prefix) & (slot >= first));
}

// tanh to about 3 units in the last place: x P(x^2) with the P of least largest relative error, of degree 3 below 1/4 (5.2e-9 by
// its coefficients, 9.3e-8 with the fp32 roundings) and 5 below 3/4 (6.5e-8; 1.6e-7); beyond, 1 - 2 / (exp(2x) + 1), which no longer cancels.
constexpr float kTanhTiny = 0.25f, kTanhSmall = 0.75f;
constexpr double kTanhTinyPoly[4] = {1.0, -0.3333320617675781, 0.13323132693767548, -0.051327724009752274};
__device__ __forceinline__ float tanh_over_x_small(float t) {
  float y = fmaf(t, -0.004716257564723492f, 0.01958290860056877f);
  y = fmaf(t, y, -0.05334443226456642f);
  y = fmaf(t, y, 0.1332540661096573f);
  y = fmaf(t, y, -0.33332958817481995f);
  return fmaf(t, y, 1.0f);
}
__device__ __forceinline__ float tanh_large(float x) {
  const float e = fast_exp2(fabsf(x) * (2.0f * kLog2e));
  return copysignf(1.0f - 2.0f * __builtin_amdgcn_rcpf(e + 1.0f), x);
}

// 16 raw products q.k of a lane as scores in log2 units, capped (without the distance bias), each minus z(e).  With x = score / cap
// the capped score is (score) * (tanh(x) / x).  Scores far below the cap, which is what a cap is for, take the
// short forms: 5 (READY: coefficients made for this scale, in four more scalar registers; the attention kernel has none left and is
// 8 % faster with 7 slots and literals) or 9 instead of about 24 issue slots each, chosen per block.
template <bool READY, typename Minus>
__device__ __forceinline__ void cap_scores(const ChunkParams& p, floatx16& s, Minus z) {
  if (p.cap_log2 == 0.f) {
#pragma unroll
    for (int e = 0; e < 16; ++e) s[e] = fmaf(s[e], p.scale_log2, -z(e));
    return;
  }
  float top = 0.f;
#pragma unroll
  for (int e = 0; e < 16; ++e) top = fmaxf(top, fabsf(s[e]));
  top *= p.cap_in;
  if (!__ballot(!(top < (READY ? p.cap_tiny_top : kTanhTiny)))) {
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      if constexpr (READY) {
        const float t = s[e] * s[e];
        const float y = fmaf(t, fmaf(t, fmaf(t, p.cap_tiny[3], p.cap_tiny[2]), p.cap_tiny[1]), p.cap_tiny[0]);
        s[e] = fmaf(s[e], y, -z(e));
      } else {
        const float x = s[e] * p.cap_in, t = x * x;
        const float y = fmaf(t, fmaf(t, fmaf(t, (float)kTanhTinyPoly[3], (float)kTanhTinyPoly[2]), (float)kTanhTinyPoly[1]), 1.f);
        s[e] = fmaf(s[e] * p.scale_log2, y, -z(e));
      }
    }
  } else if (!__ballot(!(top < kTanhSmall))) {
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const float x = s[e] * p.cap_in;
      s[e] = fmaf(s[e] * p.scale_log2, tanh_over_x_small(x * x), -z(e));
    }
  } else {
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const float x = s[e] * p.cap_in;
      s[e] = (fabsf(x) < kTanhSmall ? s[e] * p.scale_log2 * tanh_over_x_small(x * x) : p.cap_log2 * tanh_large(x)) - z(e);
    }
  }
}

// Row r of a staged tile of head rows holds its 16-byte chunk c at position c ^ row_swizzle(r): 16 rows read at one chunk
// column and 4 rows read at 4 neighbouring ones both cover all LDS banks once.
template <int HD>
__device__ __forceinline__ constexpr int row_swizzle(int row) {
  if (HD == 128) return ((row & 3) << 2) | ((row >> 2) & 3);
  return (((row >> 1) & 1) << 2) | ((row >> 2) & 3);
}

template <bool F16>
__device__ __forceinline__ floatx16 mfma_32x32x16(const uint4& a, const uint4& b, floatx16 c) {
  if constexpr (F16)
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
// Row of a 32x32 accumulator tile that register i of lane half h (lane / 32) holds; its column is lane % 32.
__device__ __forceinline__ constexpr int acc_row(int i, int h) { return 8 * (i >> 2) + 4 * h + (i & 3); }

// Two fp32 to two elements in one dword, round-to-nearest-even.
template <bool F16>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  const floatx2 x = {a, b};
  if constexpr (F16) return __builtin_bit_cast(uint32_t, __builtin_convertvector(x, f16x2));
  else return __builtin_bit_cast(uint32_t, __builtin_convertvector(x, bf16x2));
}

// A buffer descriptor as a plain quad of scalar registers (see make_rsrc).
__device__ __forceinline__ u32x4 rsrc_words(const void* base, int bytes) {
  const uint64_t a = reinterpret_cast<uint64_t>(base);
  return u32x4{(uint32_t)a, (uint32_t)(a >> 32) & 0xffffu, (uint32_t)bytes, 0x00020000u};
}
// 64 lanes x 16 bytes from the buffer straight into 1 KiB of LDS at byte offset lds_off (below 64 KiB); lanes out of the
// buffer's range bring zeros.  Written in assembly because the compiler, which cannot tell the stages of a staging area
// apart, puts a wait for every such load in front of the next LDS read of any stage; the kernels wait where they need to.
// It has no register outputs.  NT: read-once data.
template <bool NT>
__device__ __forceinline__ void lds_load_16(u32x4 rsrc, uint32_t lds_off, int off) {
  if constexpr (NT)
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen nt lds" ::"s"(lds_off), "v"(off), "s"(rsrc) : "memory");
  else
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(lds_off), "v"(off), "s"(rsrc) : "memory");
}
__device__ __forceinline__ uint32_t lds_offset(const void* p) {
  return (uint32_t)reinterpret_cast<uintptr_t>((const __attribute__((address_space(3))) void*)p);
}

// The larger of lane l's and lane l ^ 32's value (no LDS).
__device__ __forceinline__ float max_halves(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
// The value of lane ^ 32.
__device__ __forceinline__ float other_half(float x) { return __shfl_xor(x, 32); }

// Host side: the arguments every chunk operator takes.
int check_chunk_args(const char* fn, const void* q, const void* kv_cache, const int32_t* q_indptr, const int32_t* page_indices,
                     const int32_t* page_indptr, const int32_t* last_page_len, int64_t nnz, int batch, int num_q_heads,
                     int num_kv_heads, int head_dim, int page_size, int64_t num_pages, int max_pages_per_seq,
                     int first_page_offset, float sm_scale, float softcap, int window, int max_group);
void fill_chunk_params(ChunkParams& p, const void* q, const void* kv_cache, const int32_t* q_indptr, const int32_t* page_indices,
                       const int32_t* page_indptr, const int32_t* last_page_len, const float* slopes, const int32_t* prefix_lens,
                       int64_t nnz, int batch, int num_q_heads, int num_kv_heads, int head_dim, int page_size, int64_t num_pages,
                       int first_page_offset, float sm_scale, float softcap, int window);

}  // namespace kin
