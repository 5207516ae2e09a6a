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
  int given;                     // bits kOffsets ..: what there is (else a readable word stands there)
};

// A workgroup takes `chunk` words of a row. It counts those of the row's history that
// fall on them in LDS (bit 31: seen in the prompt; the rest: n; additions of whole numbers,
// whose order changes nothing) and finds the last bias entry of each, then goes over the
// words once. Under a full memory system every load that waits for another one costs
// microseconds, so there are two rounds of them: the row's settings beside the logits, then the
// mask's bits, the first tokens and the biases together. 64 rows of 248320 f32 logits with
// histories of 1 to 8000, up to 300 biases and masks: 31.1 us, 4.1 TB/s (33.7 with a wait for
// each setting, 46 with the other loads one after another too; 25 with no setting at all, a
// copy). Chunks of 1024, 2048, 4096 and 8192 words, 8 a thread: 39.8, 32.4, 31.1 and 31.9 us,
// and 16 rows of 151936 bf16 logits 7.2, 6.1, 6.2 and 7.0 (every workgroup of a row goes over
// its history). Two, 4 and 8 tokens a thread at once, before that: 34.2, 33.4 and 33.6, and 7.2,
// 6.9 and 7.7 us. One row of 151936 and 800 tokens: 5 us, the two rounds and the launch. What a history
// costs grows with the workgroups of its row: 64 rows of 248320 with 800, 8000, 32000 and 128000 tokens each 22, 29,
// 52 and 153 us; one of 151936 4, 5, 9 and 26.
enum { kOffsets, kPrompts, kRepetition, kFrequency, kPresence, kBiases, kRows };
constexpr int kThreads = 512, kTokens = 4, kValues = 512;  // tokens of a thread under way; biases kept in LDS

struct LogitsRow {
  int64_t b, w0;                        // row, first word
  uint32_t t0, t1, mine, e0, e1;        // its tokens, and those behind the prompt; its bias entries
  uint32_t n;                           // words of the workgroup
  float r, f, p;
  const uint32_t *mask;
  uint32_t *counts, *entries;
  float *values;
  int tokens[kTokens], word;            // the thread's first ones
  float value;

  __device__ __forceinline__ LogitsRow(const LogitsArgs &a, uint32_t *lds) {
    b = blockIdx.x / a.chunks, w0 = (int64_t)(blockIdx.x - b * a.chunks) * a.chunk;
    n = (uint32_t)min((int64_t)a.chunk, a.V - w0);
    counts = lds, entries = lds + (a.tokens ? a.chunk : 0), values = (float *)(entries + a.chunk);
    // (scalar loads: the launch writes none of it, and the address is the wave's. No branches between them, one
    // wait for all; T, E and R are 0 where there is none)
    auto load = [&](int bit, auto *p, int i) {
      const uint32_t at = (uint32_t)(b + i) * 4 & (uint32_t)__builtin_amdgcn_sbfe(a.given, bit, 1);
      return *(const __attribute__((address_space(4))) uint32_t *)((uintptr_t)p + at);
    };
    auto or_zero = [&](int bit, uint32_t v) { return v & (uint32_t)__builtin_amdgcn_sbfe(a.given, bit, 1); };
    uint32_t from = load(kOffsets, a.offsets, 0), to = load(kOffsets, a.offsets, 1), own = load(kPrompts, a.prompts, 0),
             first = load(kBiases, a.bias_offsets, 0), end = load(kBiases, a.bias_offsets, 1), row = load(kRows, a.mask_rows, 0),
             factor = load(kRepetition, a.repetition, 0), each = load(kFrequency, a.frequency, 0), once = load(kPresence, a.presence, 0);
    asm volatile("" : "+s"(from), "+s"(to), "+s"(own), "+s"(first), "+s"(end), "+s"(row), "+s"(factor), "+s"(each), "+s"(once));
    auto bounded = [](uint32_t i, int64_t most) { return min((uint32_t)max((int)i, 0), (uint32_t)most); };
    t0 = bounded(from, a.T), t1 = bounded(to, a.T), e0 = bounded(first, a.E), e1 = bounded(end, a.E);
    mine = t0 + (uint32_t)max((int)or_zero(kPrompts, own), 0);
    r = a.given >> kRepetition & 1 ? __uint_as_float(factor) : 1.f;
    f = __uint_as_float(or_zero(kFrequency, each)), p = __uint_as_float(or_zero(kPresence, once));
    const int64_t m = a.given >> kRows & 1 ? (int)row : b;
    mask = m >= 0 && m < a.R ? a.mask + m * ((a.V + 31) / 32) : nullptr;
  }
  __device__ __forceinline__ void load_tokens(const LogitsArgs &a, uint32_t t) {
#pragma unroll
    for (int u = 0; u < kTokens; ++u) {
      const uint32_t i = t + u * kThreads;
      const int token = a.tokens[min(i, (uint32_t)a.T - 1)];  // (no branch between the loads)
      tokens[u] = i < t1 ? token : -1;
    }
  }
  __device__ __forceinline__ void load(const LogitsArgs &a) {
    if (a.tokens) load_tokens(a, t0 + threadIdx.x);
    if (!a.bias) return;
    const uint32_t e = min(e0 + threadIdx.x, (uint32_t)a.E - 1);
    word = a.bias_words[e], value = a.bias[e];
  }
  // Counts and entries of the workgroup's words
  __device__ __forceinline__ void count(const LogitsArgs &a) {
    const int total = a.chunk * ((a.tokens != nullptr) + (a.bias != nullptr));  // (a multiple of 4)
    for (int i = 4 * threadIdx.x; i < total; i += 4 * kThreads) *(u32x4 *)(counts + i) = u32x4{0, 0, 0, 0};
    __syncthreads();
    for (uint32_t t = t0 + threadIdx.x; t < t1; t += kTokens * kThreads) {
      if (t >= t0 + kTokens * kThreads) load_tokens(a, t);
#pragma unroll
      for (int u = 0; u < kTokens; ++u) {
        const uint32_t at = (uint32_t)tokens[u] - (uint32_t)w0;  // (words before the first wrap past n)
        if (at >= n) continue;
        if (t + u * kThreads < mine) atomicOr(counts + at, 0x80000000u);
        else atomicAdd(counts + at, 1u);
      }
    }
    for (uint32_t e = e0 + threadIdx.x; e < e1; e += kThreads) {
      const bool first = e < e0 + kThreads;
      const uint32_t at = (uint32_t)(first ? word : a.bias_words[e]) - (uint32_t)w0;
      if (at >= n) continue;
      atomicMax(entries + at, e - e0 + 1);
      if (e - e0 < kValues) values[e - e0] = first ? value : a.bias[e];
    }
    __syncthreads();
  }
  // One word's logit: c its count, e its bias entry, allowed by the mask
  __device__ __forceinline__ float adjust(const LogitsArgs &a, float z, uint32_t c, uint32_t e, bool allowed) const {
    if (c) {
      if (r > 0.f) z = z > 0.f ? z / r : z * r;
      if (const uint32_t m = c & 0x7fffffffu) z -= f * (float)m + p;
    }
    if (e) z += e <= kValues ? values[e - 1] : a.bias[e0 + e - 1];
    return allowed ? z : kMinusInf;
  }
};

// Rows of any length and alignment: a word a thread at a time
extern "C" __global__ void __launch_bounds__(kThreads) rxw8_logits_any(LogitsArgs a) {
  extern __shared__ __attribute__((aligned(16))) uint32_t lds[];  // counts [chunk], entries [chunk], values
  LogitsRow x(a, lds);
  x.load(a);
  x.count(a);
  for (uint32_t i = threadIdx.x; i < x.n; i += kThreads) {
    const int64_t w = x.w0 + i, at = x.b * a.V + w;
    const float z = x.adjust(a, any_load(a.logits, at, a.in_f32), a.tokens ? x.counts[i] : 0, a.bias ? x.entries[i] : 0,
                             !x.mask || x.mask[w >> 5] >> (w & 31) & 1);
    if (a.out_f32) ((float *)a.out)[at] = z;
    else ((uint16_t *)a.out)[at] = f32_to_bf16_bits(z);
  }
}

// Rows of whole 8 words at 16-byte boundaries: 8 words a thread (chunk = 8 threads)
template <typename S, typename P>
__device__ __forceinline__ void logits_adjust(const LogitsArgs &a, uint32_t *lds) {
  constexpr int NS = sizeof(S) / 2;  // 16-byte words of 8 logits
  const int64_t b = blockIdx.x / a.chunks, w = (int64_t)(blockIdx.x - b * a.chunks) * a.chunk + 8 * threadIdx.x, at = b * a.V + w;
  const bool mine = w < a.V;
  u32x4 in[NS];
  uint32_t bits = 0xff;
  if (mine) {
#pragma unroll
    for (int k = 0; k < NS; ++k) in[k] = ((const u32x4 *)((const S *)a.logits + at))[k];
  }
  LogitsRow x(a, lds);
  if (mine && x.mask) bits = ((const uint8_t *)x.mask)[w >> 3];
  u32x4 c[2] = {}, e[2] = {};
  if (a.tokens || a.bias) {
    x.load(a);
    x.count(a);
    if (a.tokens) c[0] = *(const u32x4 *)(x.counts + 8 * threadIdx.x), c[1] = *(const u32x4 *)(x.counts + 8 * threadIdx.x + 4);
    if (a.bias) e[0] = *(const u32x4 *)(x.entries + 8 * threadIdx.x), e[1] = *(const u32x4 *)(x.entries + 8 * threadIdx.x + 4);
  }
  if (!mine) return;
  float z[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const uint32_t w = in[k / (8 / NS)][NS == 2 ? k & 3 : k >> 1];
    z[k] = __uint_as_float(NS == 2 ? w : k & 1 ? w & 0xffff0000u : w << 16);
    z[k] = x.adjust(a, z[k], c[k >> 2][k & 3], e[k >> 2][k & 3], bits >> k & 1);
  }
  u32x4 *const to = (u32x4 *)((P *)a.out + at);
  if constexpr (sizeof(P) == 4) {
#pragma unroll
    for (int k = 0; k < 2; ++k)
      to[k] = u32x4{__float_as_uint(z[4 * k]), __float_as_uint(z[4 * k + 1]), __float_as_uint(z[4 * k + 2]), __float_as_uint(z[4 * k + 3])};
  } else {
    to[0] = u32x4{pack_bf16x2(z[0], z[1]), pack_bf16x2(z[2], z[3]), pack_bf16x2(z[4], z[5]), pack_bf16x2(z[6], z[7])};
  }
}
extern "C" __global__ void __launch_bounds__(kThreads) rxw8_logits_adjust(LogitsArgs a) {
  extern __shared__ __attribute__((aligned(16))) uint32_t lds[];
  if (a.in_f32 && a.out_f32) logits_adjust<float, float>(a, lds);
  else if (a.in_f32) logits_adjust<float, uint16_t>(a, lds);
  else if (a.out_f32) logits_adjust<uint16_t, float>(a, lds);
  else logits_adjust<uint16_t, uint16_t>(a, lds);
}
