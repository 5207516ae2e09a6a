// Attention of one query row at any head width up to 512, shared by the paged
// and the packed kernels for the shapes their matrix-core kernels do not take.
#pragma once
#include "common.h"

#define RXW8_ATTN_ANY_MAX_D 512

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kMinusInf = -__builtin_huge_valf();

// The running softmax of one wave: maximum and sum of weights (log2 units),
// lane l the accumulators of dims l, l + 64, ...
struct AnyState {
  float m = kMinusInf, l = 0.f;
  float acc[RXW8_ATTN_ANY_MAX_D / 64] = {};
};

__device__ __forceinline__ float any_load(const void *p, int64_t i, bool f32) {
  return f32 ? ((const float *)p)[i] : bf16_bits_to_f32(((const uint16_t *)p)[i]);
}

__device__ __forceinline__ float wave_max64(float v) {
  for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o));
  return v;
}

// v as a sum of bf16 parts, high bits first: two leave |v| 2^-16 at most (the second is
// rounded), three are v exactly (8 bits of its 24 each). A part is cut, not rounded, and
// is one step less where that would leave nothing: every part of a v that is not 0 has
// its sign and is not 0, so that a product with an infinite factor is the infinity that
// v's own would be.
__device__ __forceinline__ uint32_t cut_weight(float v) {  // v >= 0: f32 bits, low half zero
  return __builtin_elementwise_sub_sat(__float_as_uint(v), 1u) & 0xffff0000u;
}
__device__ __forceinline__ uint32_t cut_bf16(float v) {
  return cut_weight(fabsf(v)) | (__float_as_uint(v) & 0x80000000u);
}
// Parts of two values (Weights: not below 0), packed in pairs: N = 2 or 3
template <bool Weights = false, int N>
__device__ __forceinline__ void split_bf16x2(float a, float b, uint32_t (&part)[N]) {
#pragma unroll
  for (int n = 0; n + 1 < N; ++n) {
    const uint32_t x = Weights ? cut_weight(a) : cut_bf16(a), y = Weights ? cut_weight(b) : cut_bf16(b);
    part[n] = (x >> 16) | y;
    a -= __uint_as_float(x), b -= __uint_as_float(y);
  }
  part[N - 1] = pack_bf16x2(a, b);
}

// One wave over keys first, first + 1, .. in chunks of 64 (lane = key), the next
// chunk `step` chunks on: s_j = c q.k_j (c = scale log2 e), online softmax,
// acc += p v. row(j) is the element offset of key j's row (K and V alike), or
// negative where the key is not seen; a key whose weight is zero adds nothing,
// whatever its value holds. q: D floats in LDS.
template <typename Row>
__device__ void any_walk(AnyState &st, const float *q, const void *k, const void *v, bool kv_f32,
                         int d, int64_t first, int64_t end, int step, float c, Row row) {
  const int lane = threadIdx.x & 63;
  for (int64_t j0 = first; j0 < end; j0 += (int64_t)64 * step) {
    const int64_t j = j0 + lane;
    const int64_t off = j < end ? row(j) : -1;
    float s = kMinusInf;
    if (off >= 0) {
      float dot = 0.f;
      for (int i = 0; i < d; ++i) dot = fmaf(q[i], any_load(k, off + i, kv_f32), dot);
      s = dot * c;
    }
    // (fmaxf passes over a NaN; its weight below is NaN all the same)
    const float m_new = fmaxf(st.m, wave_max64(s));
    const float ref = m_new == kMinusInf ? 0.f : m_new;
    const float f = exp2f(st.m - ref), p = off >= 0 ? exp2f(s - ref) : 0.f;
    st.m = m_new;
    st.l = st.l * f + wave_sum64(p);
#pragma unroll
    for (int i = 0; i < RXW8_ATTN_ANY_MAX_D / 64; ++i) st.acc[i] *= f;
    const int n = (int)(end - j0 < 64 ? end - j0 : 64);
    for (int t = 0; t < n; ++t) {
      const float pt = __shfl(p, t);
      if (pt == 0.f) continue;
      const int64_t ot = __shfl(off, t);
#pragma unroll
      for (int i = 0; i < RXW8_ATTN_ANY_MAX_D / 64; ++i)
        if (lane + 64 * i < d) st.acc[i] = fmaf(pt, any_load(v, ot + lane + 64 * i, kv_f32), st.acc[i]);
    }
  }
}

// out[i] = acc / l; a row that saw no key (or only weights of zero) is 0
__device__ __forceinline__ void any_store(const AnyState &st, void *out, int64_t at, int d, bool f32) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int i = 0; i < RXW8_ATTN_ANY_MAX_D / 64; ++i)
    if (lane + 64 * i < d) {
      const float y = st.l == 0.f ? 0.f : st.acc[i] / st.l;
      if (f32)
        ((float *)out)[at + lane + 64 * i] = y;
      else
        ((uint16_t *)out)[at + lane + 64 * i] = f32_to_bf16_bits(y);
    }
}

// The sequence that packed row t belongs to, by offsets [nseq + 1]: the largest b
// with offsets[b] <= t, or -1 before the first; t may lie behind its end. A wave
// looks at 64 offsets at a time: two round trips up to 4096 sequences.
__device__ __forceinline__ int any_sequence(const int32_t *offsets, int nseq, int64_t t) {
  const int lane = threadIdx.x & 63;
  int lo = 0, n = nseq;  // the answer is lo - 1 + (how many of offsets[lo .. lo + n) are <= t)
  while (n > 64) {
    const int step = (n + 63) / 64, i = lo + lane * step;
    const unsigned long long le = __ballot(lane * step < n && offsets[i < nseq ? i : nseq] <= t);
    const int c = __popcll(le);  // (offsets do not decrease: the lanes of `le` are the first ones)
    if (c == 0) return lo - 1;
    const int skip = (c - 1) * step;
    lo += skip;
    n = n - skip < step ? n - skip : step;
  }
  const int i = lo + lane;
  return lo - 1 + __popcll(__ballot(lane < n && offsets[i < nseq ? i : nseq] <= t));
}
