// What stands between the output layer and sampling: penalties for words that a row's
// history holds, biases for single words, and masks of the words that a grammar allows.
// Per row, z the logit of a word in f32, seen and n whether and how often its history
// holds the word (n without the first `prompts` tokens):
//   z = z > 0 ? z / repetition : z repetition   if seen
//   z = z - frequency n - presence              if n > 0
//   z = z + bias                                the last of the row's entries for the word
//   z = -inf                                    if the row's mask lacks the word
#include "attn_any.h"

struct LogitsArgs {
  const void *logits;            // [B, V] f32 | bf16
  void *out;                     // [B, V] f32 | bf16 (may be `logits`)
  const int32_t *tokens;         // [T], or null
  const int32_t *offsets;        // [B + 1]
  const int32_t *prompts;        // [B], or null: 0
  const float *repetition, *frequency, *presence;  // [B], or null
  const int32_t *bias_words;     // [E], or null
  const float *bias;             // [E]
  const int32_t *bias_offsets;   // [B + 1]
  const uint32_t *mask;          // [R, (V + 31) / 32], or null
  const int32_t *mask_rows;      // [B], or null: row b
  int64_t T, E, R, V;
  int in_f32, out_f32;
  int chunk, chunks;             // words of a workgroup; workgroups of a row
};

// A workgroup takes `chunk` words of a row. It counts those of the row's history that
// fall on them in LDS (bit 31: seen in the prompt; the rest: n; additions of whole numbers,
// whose order changes nothing) and finds the last bias entry of each, then goes over the
// words once.
constexpr int kLogitsThreads = 256;

struct LogitsRow {
  int64_t b, w0, e0;        // row, its workgroup's first word, its first bias entry
  int n;                    // words
  float r, f, p;
  const uint32_t *mask;
  uint32_t *counts, *entries;
};

__device__ __forceinline__ LogitsRow logits_row(const LogitsArgs &a, uint32_t *lds) {
  LogitsRow x;
  x.b = blockIdx.x / a.chunks, x.w0 = (int64_t)(blockIdx.x - x.b * a.chunks) * a.chunk;
  x.n = (int)min((int64_t)a.chunk, a.V - x.w0);
  x.counts = lds, x.entries = lds + (a.tokens ? a.chunk : 0);
  x.r = a.repetition ? a.repetition[x.b] : 1.f;
  x.f = a.frequency ? a.frequency[x.b] : 0.f;
  x.p = a.presence ? a.presence[x.b] : 0.f;
  const int64_t m = a.mask ? a.mask_rows ? a.mask_rows[x.b] : x.b : -1;
  x.mask = m >= 0 && m < a.R ? a.mask + m * ((a.V + 31) / 32) : nullptr;
  return x;
}

// Counts and entries of the workgroup's words
__device__ __forceinline__ void logits_count(const LogitsArgs &a, LogitsRow &x) {
  typedef uint32_t u32x4a __attribute__((ext_vector_type(4)));
  const int64_t b = x.b, w0 = x.w0;
  const int total = a.chunk * ((a.tokens != nullptr) + (a.bias != nullptr));  // (multiples of 4)
  for (int i = 4 * threadIdx.x; i < total; i += 4 * kLogitsThreads) *(u32x4a *)(x.counts + i) = u32x4a{0, 0, 0, 0};
  __syncthreads();
  auto bounded = [](int64_t i, int64_t most) { return i < 0 ? 0 : i < most ? i : most; };
  if (a.tokens) {
    const int64_t t0 = bounded(a.offsets[b], a.T), t1 = bounded(a.offsets[b + 1], a.T);
    const int64_t mine = t0 + (a.prompts ? max(a.prompts[b], 0) : 0);
    constexpr int U = 8;  // loads under way
    for (int64_t t = t0 + threadIdx.x; t < t1; t += U * kLogitsThreads) {
      int w[U];
#pragma unroll
      for (int u = 0; u < U; ++u) w[u] = t + u * kLogitsThreads < t1 ? a.tokens[t + u * kLogitsThreads] : -1;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int64_t at = (int64_t)w[u] - w0;
        if (at < 0 || at >= x.n) continue;
        if (t + u * kLogitsThreads < mine) atomicOr(x.counts + at, 0x80000000u);
        else atomicAdd(x.counts + at, 1u);
      }
    }
  }
  x.e0 = a.bias ? bounded(a.bias_offsets[b], a.E) : 0;
  const int64_t e1 = a.bias ? bounded(a.bias_offsets[b + 1], a.E) : 0;
  for (int64_t e = x.e0 + threadIdx.x; e < e1; e += kLogitsThreads) {
    const int64_t at = (int64_t)a.bias_words[e] - w0;
    if (at >= 0 && at < x.n) atomicMax(x.entries + at, (uint32_t)(e - x.e0 + 1));
  }
  __syncthreads();
}

// One word's logit: c its count, e its bias entry, allowed by the mask
__device__ __forceinline__ float logits_word(const LogitsArgs &a, const LogitsRow &x, float z, uint32_t c, uint32_t e, bool allowed) {
  if (c) {
    if (x.r > 0.f) z = z > 0.f ? z / x.r : z * x.r;
    if (const uint32_t m = c & 0x7fffffffu) z -= x.f * (float)m + x.p;
  }
  if (e) z += a.bias[x.e0 + e - 1];
  return allowed ? z : kMinusInf;
}

// Rows of any length and alignment: a word a thread
extern "C" __global__ void __launch_bounds__(kLogitsThreads) rxw8_logits_any(LogitsArgs a) {
  extern __shared__ __attribute__((aligned(16))) uint32_t lds[];  // counts [chunk], entries [chunk]
  LogitsRow x = logits_row(a, lds);
  logits_count(a, x);
  for (int i = threadIdx.x; i < x.n; i += kLogitsThreads) {
    const int64_t w = x.w0 + i, at = x.b * a.V + w;
    const float z = logits_word(a, x, any_load(a.logits, at, a.in_f32), a.tokens ? x.counts[i] : 0, a.bias ? x.entries[i] : 0,
                                !x.mask || x.mask[w >> 5] >> (w & 31) & 1);
    if (a.out_f32) ((float *)a.out)[at] = z;
    else ((uint16_t *)a.out)[at] = f32_to_bf16_bits(z);
  }
}

// Rows of whole 8 words at 16-byte boundaries: 8 words a thread, I times, whose logits and
// mask bits are on their way while the history is counted
template <typename S, typename P, int I>
__device__ __forceinline__ void logits_adjust(const LogitsArgs &a, uint32_t *lds) {
  constexpr int NS = sizeof(S) / 2;  // 16-byte words of 8 logits
  LogitsRow x = logits_row(a, lds);
  u32x4 in[I][NS];
  uint32_t bits[I];
  const u32x4 *const from = (const u32x4 *)((const S *)a.logits + x.b * a.V + x.w0);
#pragma unroll
  for (int i = 0; i < I; ++i) {
    const int p = threadIdx.x + i * kLogitsThreads;  // of the workgroup's pieces of 8 words
    bits[i] = 0xff;
    if (8 * p < x.n) {
#pragma unroll
      for (int k = 0; k < NS; ++k) in[i][k] = from[p * NS + k];
      if (x.mask) bits[i] = ((const uint8_t *)x.mask)[(x.w0 >> 3) + p];
    }
  }
  logits_count(a, x);
#pragma unroll
  for (int i = 0; i < I; ++i) {
    const int p = threadIdx.x + i * kLogitsThreads;
    if (8 * p >= x.n) return;
    u32x4 c[2] = {}, e[2] = {};
    if (a.tokens) c[0] = *(const u32x4 *)(x.counts + 8 * p), c[1] = *(const u32x4 *)(x.counts + 8 * p + 4);
    if (a.bias) e[0] = *(const u32x4 *)(x.entries + 8 * p), e[1] = *(const u32x4 *)(x.entries + 8 * p + 4);
    float z[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const uint32_t w = in[i][k / (8 / NS)][NS == 2 ? k & 3 : k >> 1];
      z[k] = __uint_as_float(NS == 2 ? w : k & 1 ? w & 0xffff0000u : w << 16);
      z[k] = logits_word(a, x, z[k], c[k >> 2][k & 3], e[k >> 2][k & 3], bits[i] >> k & 1);
    }
    u32x4 *const to = (u32x4 *)((P *)a.out + x.b * a.V + x.w0) + p * (sizeof(P) / 2);
    if constexpr (sizeof(P) == 4) {
#pragma unroll
      for (int k = 0; k < 2; ++k)
        to[k] = u32x4{__float_as_uint(z[4 * k]), __float_as_uint(z[4 * k + 1]), __float_as_uint(z[4 * k + 2]), __float_as_uint(z[4 * k + 3])};
    } else {
      to[0] = u32x4{pack_bf16x2(z[0], z[1]), pack_bf16x2(z[2], z[3]), pack_bf16x2(z[4], z[5]), pack_bf16x2(z[6], z[7])};
    }
  }
}
#define RXW8_LOGITS(I)                                                                              \
  extern "C" __global__ void __launch_bounds__(kLogitsThreads) rxw8_logits_adjust##I(LogitsArgs a) { \
    extern __shared__ __attribute__((aligned(16))) uint32_t lds[];                                  \
    if (a.in_f32 && a.out_f32) logits_adjust<float, float, I>(a, lds);                              \
    else if (a.in_f32) logits_adjust<float, uint16_t, I>(a, lds);                                   \
    else if (a.out_f32) logits_adjust<uint16_t, float, I>(a, lds);                                  \
    else logits_adjust<uint16_t, uint16_t, I>(a, lds);                                              \
  }
RXW8_LOGITS(1)
RXW8_LOGITS(2)
RXW8_LOGITS(4)
