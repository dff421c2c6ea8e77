// From the fused projection to q, k and v heads ready for the cache: split, RMSNorm of the q and k heads
// (as kin_qkv_norm_split; optional), and rotary positions with one or several axes (text: one; images and
// video: time, height, width).  Pair i of a head, its elements i and i + D/2, is turned by
//     angle = position[axis[i]] * frequency[i].
// HBM-bound: every row is read once and written once with 16-byte accesses (8191 tokens, 32 + 2 * 8 heads of 128, three axes:
// 35 us, 5.8 TB/s; 4096 tokens of 4 + 2 heads: 6 us).
//
// Positions run to millions, where an fp32 angle has no digits left behind the full turns.  Frequencies are
// therefore turns per position as 64-bit fractions: position times fraction, modulo 2^64, IS the angle of that
// fraction modulo a full turn, exactly, in integer arithmetic; its upper 32 bits go to fp32 as a signed part of a turn
// (2^-26 of a turn off at most, and 2^-32 for the lower bits) and sincospi does the rest.  The D/2 angles of a token are taken once and
// shared by its q and k heads through LDS.
#include "kin_common.h"

namespace kin {

struct RopeParams {
  const u32x4* qkv;
  int64_t row_stride;   // 16-byte units
  const u32x4 *q_weight, *k_weight;  // both null: no norm
  const int32_t* positions;          // [axes, tokens]
  const uint64_t* freq;              // [D / 2] turns per position, as a fraction of 2^64
  const int32_t* axis;               // [D / 2]
  u32x4 *q, *k, *v;
  int tokens, axes, hq, hkv;
  float eps;
};

// 16-bit elements of a 16-byte chunk and back.  Norm and rotation are fp32 in between, with one rounding at the end
// (kin_qkv_norm_split rounds after its norm).
template <bool F16>
__device__ __forceinline__ void unpack8(const u32x4& v, float (&x)[8]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = elem_lo<F16>(w[i]);
    x[2 * i + 1] = elem_hi<F16>(w[i]);
  }
}
template <bool F16>
__device__ __forceinline__ u32x4 pack8(const float (&x)[8]) {
  u32x4 v;
  v.x = f32_to_elem<F16>(x[0]) | (f32_to_elem<F16>(x[1]) << 16);
  v.y = f32_to_elem<F16>(x[2]) | (f32_to_elem<F16>(x[3]) << 16);
  v.z = f32_to_elem<F16>(x[4]) | (f32_to_elem<F16>(x[5]) << 16);
  v.w = f32_to_elem<F16>(x[6]) | (f32_to_elem<F16>(x[7]) << 16);
  return v;
}

// LPR lanes per head row of D = LPR * 8 elements.  A workgroup of 256 threads owns TOK tokens; the 256 / TOK threads of
// a token take its head rows 256 / TOK / LPR at a time.  Lane l of a row holds the elements 8l .. 8l + 7; their partners
// are lane l ^ (LPR / 2)'s, and both turn by the pairs 8 * (l % (LPR / 2)) ...
template <bool F16, int LPR, int TOK, bool NORM>
__global__ __launch_bounds__(256) void qkv_norm_rope_kernel(RopeParams p) {
  constexpr int D = LPR * 8, PAIRS = D / 2, TPT = 256 / TOK, RPT = TPT / LPR;
  __shared__ __attribute__((aligned(16))) float2 cs[TOK][PAIRS];
  const int tid = threadIdx.x;
  const int t0 = blockIdx.x * TOK;
  for (int x = tid; x < TOK * PAIRS; x += 256) {
    const int t = t0 + x / PAIRS, i = x % PAIRS;
    float c = 1.f, s = 0.f;
    const int ax = p.axis[i];
    if (t < p.tokens && (unsigned)ax < (unsigned)p.axes) {
      const int64_t pos = p.positions[(int64_t)ax * p.tokens + t];
      const uint64_t turn = (uint64_t)pos * p.freq[i];
      sincospif((float)(int32_t)(turn >> 32) * 0x1p-31f, &s, &c);
    }
    cs[x / PAIRS][i] = make_float2(c, s);
  }
  __syncthreads();
  const int sub = tid / TPT, in = tid % TPT;
  const int t = t0 + sub;
  if (t >= p.tokens) return;
  const int l = in % LPR, row0 = in / LPR;
  const bool upper = l >= LPR / 2;
  float c[8], s[8];
  uint32_t turned[8];  // the partner's bits, or none where a pair is not turned: 0 times an infinity would be NaN
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float2 z = cs[sub][8 * (l & (LPR / 2 - 1)) + i];
    c[i] = z.x;
    s[i] = upper ? z.y : -z.y;  // lower half: lo c - hi s; upper half: hi c + lo s
    turned[i] = z.y == 0.f ? 0u : ~0u;
  }
  float wq[8], wk[8];
  if constexpr (NORM) {
    unpack8<F16>(p.q_weight[l], wq);
    unpack8<F16>(p.k_weight[l], wk);
  }
  const u32x4* src = p.qkv + (int64_t)t * p.row_stride + l;
  const int heads = p.hq + 2 * p.hkv;
  for (int j = row0; j < heads; j += RPT) {
    u32x4 raw = __builtin_nontemporal_load(src + (int64_t)j * LPR);
    if (j >= p.hq + p.hkv) {
      p.v[((int64_t)t * p.hkv + (j - p.hq - p.hkv)) * LPR + l] = raw;
      continue;
    }
    const bool is_q = j < p.hq;
    float x[8];
    unpack8<F16>(raw, x);
    if constexpr (NORM) {
      float ss = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) ss = fmaf(x[i], x[i], ss);
      const float r = rsqrtf(row_sum<LPR>(ss) * (1.0f / D) + p.eps);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = x[i] * r * (is_q ? wq[i] : wk[i]);
    }
    float y[8];
#pragma unroll
    for (int i = 0; i < 8; ++i)
      y[i] = fmaf(x[i], c[i], __uint_as_float(__float_as_uint(__shfl_xor(x[i], LPR / 2)) & turned[i]) * s[i]);
    u32x4* dst = is_q ? p.q + ((int64_t)t * p.hq + j) * LPR : p.k + ((int64_t)t * p.hkv + (j - p.hq)) * LPR;
    dst[l] = pack8<F16>(y);
  }
}

// Few heads: four tokens a workgroup, so that its threads have rows to take.
static int tokens_per_workgroup(int hq, int hkv, int lanes_per_row) { return ((int64_t)hq + 2 * (int64_t)hkv) * lanes_per_row <= 128 ? 4 : 1; }
template <bool F16, int LPR, bool NORM>
static void launch_rope(const RopeParams& p, hipStream_t s) {
  if (tokens_per_workgroup(p.hq, p.hkv, LPR) == 4) qkv_norm_rope_kernel<F16, LPR, 4, NORM><<<(unsigned)((p.tokens + 3) / 4), 256, 0, s>>>(p);
  else qkv_norm_rope_kernel<F16, LPR, 1, NORM><<<(unsigned)p.tokens, 256, 0, s>>>(p);
}

static int qkv_norm_rope_impl(const char* fn, bool f16, const void* qkv, int64_t qkv_row_stride, const void* q_weight,
                              const void* k_weight, float eps, const int32_t* positions, int num_axes, const int64_t* freq,
                              const int32_t* axis, void* q, void* k, void* v, int tokens, int num_q_heads, int num_kv_heads,
                              int head_dim, kin_stream_t stream) {
  if (!qkv || !positions || !freq || !axis || !q || !k || !v) return fail(KIN_ERR_NULL_POINTER, "%s: null pointer argument", fn);
  if (!q_weight != !k_weight) return fail(KIN_ERR_NULL_POINTER, "%s: q_weight and k_weight are both given or both NULL", fn);
  if (tokens < 0 || num_q_heads < 1 || num_kv_heads < 1 || num_axes < 1)
    return fail(KIN_ERR_BAD_SHAPE, "%s: tokens=%d num_q_heads=%d num_kv_heads=%d num_axes=%d", fn, tokens, num_q_heads,
                num_kv_heads, num_axes);
  if (!supported_head_dim(head_dim))
    return fail(KIN_ERR_UNSUPPORTED, "%s: head_dim=%d, only %d and %d are built", fn, head_dim, kHeadDimSmall, kHeadDim);
  const int64_t width = ((int64_t)num_q_heads + 2 * (int64_t)num_kv_heads) * head_dim;
  if (width > 0x7fffffffLL) return fail(KIN_ERR_UNSUPPORTED, "%s: too many heads", fn);
  if (tokens > max_workgroups(256) * tokens_per_workgroup(num_q_heads, num_kv_heads, head_dim / 8))
    return fail(KIN_ERR_UNSUPPORTED, "%s: tokens=%d are too many for a call", fn, tokens);
  if (qkv_row_stride < width || qkv_row_stride % 8 != 0)
    return fail(KIN_ERR_BAD_SHAPE, "%s: qkv_row_stride=%lld must be a multiple of 8 and at least the row width %lld", fn,
                (long long)qkv_row_stride, (long long)width);
  if (!aligned16(qkv) || !aligned16(q_weight) || !aligned16(k_weight) || !aligned16(q) || !aligned16(k) || !aligned16(v))
    return fail(KIN_ERR_MISALIGNED, "%s: pointers must be 16-byte aligned", fn);
  if (!(eps >= 0.f)) return fail(KIN_ERR_BAD_SHAPE, "%s: eps must be non-negative", fn);
  if (tokens == 0) return KIN_OK;
  RopeParams p;
  p.qkv = static_cast<const u32x4*>(qkv);
  p.row_stride = qkv_row_stride / 8;
  p.q_weight = static_cast<const u32x4*>(q_weight);
  p.k_weight = static_cast<const u32x4*>(k_weight);
  p.positions = positions;
  p.freq = reinterpret_cast<const uint64_t*>(freq);
  p.axis = axis;
  p.q = static_cast<u32x4*>(q);
  p.k = static_cast<u32x4*>(k);
  p.v = static_cast<u32x4*>(v);
  p.tokens = tokens;
  p.axes = num_axes;
  p.hq = num_q_heads;
  p.hkv = num_kv_heads;
  p.eps = eps;
  hipStream_t s = static_cast<hipStream_t>(stream);
#define KIN_ROPE_LAUNCH(LPR)                          \
  do {                                                \
    if (f16) {                                        \
      if (q_weight) launch_rope<true, LPR, true>(p, s);   \
      else launch_rope<true, LPR, false>(p, s);       \
    } else {                                          \
      if (q_weight) launch_rope<false, LPR, true>(p, s);  \
      else launch_rope<false, LPR, false>(p, s);      \
    }                                                 \
  } while (0)
  if (head_dim == kHeadDimSmall) KIN_ROPE_LAUNCH(8);
  else KIN_ROPE_LAUNCH(16);
#undef KIN_ROPE_LAUNCH
  return check_hip(hipGetLastError(), "qkv_norm_rope_kernel launch");
}

}  // namespace kin

extern "C" {

int kin_qkv_norm_rope_split(const void* qkv, int64_t qkv_row_stride, const void* q_weight, const void* k_weight, float eps,
                            const int32_t* positions, int num_axes, const int64_t* freq, const int32_t* axis, void* q, void* k,
                            void* v, int tokens, int num_q_heads, int num_kv_heads, int head_dim, kin_stream_t stream) {
  return kin::qkv_norm_rope_impl("kin_qkv_norm_rope_split", false, qkv, qkv_row_stride, q_weight, k_weight, eps, positions,
                                 num_axes, freq, axis, q, k, v, tokens, num_q_heads, num_kv_heads, head_dim, stream);
}
int kin_qkv_norm_rope_split_f16(const void* qkv, int64_t qkv_row_stride, const void* q_weight, const void* k_weight, float eps,
                                const int32_t* positions, int num_axes, const int64_t* freq, const int32_t* axis, void* q,
                                void* k, void* v, int tokens, int num_q_heads, int num_kv_heads, int head_dim,
                                kin_stream_t stream) {
  return kin::qkv_norm_rope_impl("kin_qkv_norm_rope_split_f16", true, qkv, qkv_row_stride, q_weight, k_weight, eps, positions,
                                 num_axes, freq, axis, q, k, v, tokens, num_q_heads, num_kv_heads, head_dim, stream);
}

}  // extern "C"
