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
constexpr int kLogitsThreads = 512;

extern "C" __global__ void __launch_bounds__(kLogitsThreads) rxw8_logits_adjust(LogitsArgs a) {
  extern __shared__ uint32_t lds[];  // counts [chunk], entries [chunk]
  const int64_t b = blockIdx.x / a.chunks, w0 = (int64_t)(blockIdx.x - b * a.chunks) * a.chunk;
  const int n = (int)min((int64_t)a.chunk, a.V - w0);
  uint32_t *const counts = lds, *const entries = lds + (a.tokens ? a.chunk : 0);
  for (int i = threadIdx.x; i < n; i += kLogitsThreads) {
    if (a.tokens) counts[i] = 0;
    if (a.bias) entries[i] = 0;
  }
  __syncthreads();
  auto bounded = [](int64_t x, int64_t most) { return x < 0 ? 0 : x < most ? x : most; };
  if (a.tokens) {
    const int64_t t0 = bounded(a.offsets[b], a.T), t1 = bounded(a.offsets[b + 1], a.T);
    const int64_t mine = t0 + (a.prompts ? max(a.prompts[b], 0) : 0);
    for (int64_t t = t0 + threadIdx.x; t < t1; t += kLogitsThreads) {
      const int64_t w = (int64_t)a.tokens[t] - w0;
      if (w < 0 || w >= n) continue;
      if (t < mine) atomicOr(counts + w, 0x80000000u);
      else atomicAdd(counts + w, 1u);
    }
  }
  const int64_t e0 = a.bias ? bounded(a.bias_offsets[b], a.E) : 0, e1 = a.bias ? bounded(a.bias_offsets[b + 1], a.E) : 0;
  for (int64_t e = e0 + threadIdx.x; e < e1; e += kLogitsThreads) {
    const int64_t w = (int64_t)a.bias_words[e] - w0;
    if (w >= 0 && w < n) atomicMax(entries + w, (uint32_t)(e - e0 + 1));
  }
  __syncthreads();
  const float r = a.repetition ? a.repetition[b] : 1.f, f = a.frequency ? a.frequency[b] : 0.f, p = a.presence ? a.presence[b] : 0.f;
  const int64_t mr = a.mask ? a.mask_rows ? a.mask_rows[b] : b : -1;
  const uint32_t *const mask = mr >= 0 && mr < a.R ? a.mask + mr * ((a.V + 31) / 32) : nullptr;
  for (int i = threadIdx.x; i < n; i += kLogitsThreads) {
    const int64_t w = w0 + i;
    float z = any_load(a.logits, b * a.V + w, a.in_f32);
    if (const uint32_t c = a.tokens ? counts[i] : 0) {
      if (r > 0.f) z = z > 0.f ? z / r : z * r;
      if (const uint32_t m = c & 0x7fffffffu) z -= f * (float)m + p;
    }
    if (a.bias)
      if (const uint32_t e = entries[i]) z += a.bias[e0 + e - 1];
    if (mask && !(mask[w >> 5] >> (w & 31) & 1)) z = kMinusInf;
    if (a.out_f32) ((float *)a.out)[b * a.V + w] = z;
    else ((uint16_t *)a.out)[b * a.V + w] = f32_to_bf16_bits(z);
  }
}
