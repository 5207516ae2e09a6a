// The next token of each row of logits, from given random numbers.
//
// A row's words in order of (logit descending, index ascending); of these the first
// top_k; with weights w = exp((l - max) / T) the shortest prefix whose mass is at
// least top_p times the mass of the first top_k; of that the words with w >= min_p;
// the first word always. The token is the first whose running mass exceeds u times
// the mass of what is left. Every filter leaves a prefix of the order, so what the
// filters leave is known by its mass alone: the least of the prefixes' masses.
//
// Masses are whole numbers, round(w 2^s) in 64 bits with V 2^s < 2^62, w in f64:
// their sums do not depend on the order of the additions (atomics included), and a
// sum over V words is off by at most V / 2 units of 2^-s (2^-45 of the largest
// weight each at V = 2^18). Equal logits have equal masses, so within a run of
// ties a mass says how many of them it takes, and the lowest indices come first.
#include "common.h"

struct SampleArgs {
  const void *logits;          // [B, V] f32 | bf16
  const float *uniform;        // [B]
  const float *temperature;    // [B] or null (1)
  const int32_t *top_k;        // [B] or null (off)
  const float *top_p, *min_p;  // [B] or null (off)
  int32_t *out;                // [B]
  int64_t V;
  int shift;                   // s
  int bf16;
};

typedef unsigned long long u64;

// Ascending keys for ascending values, -0 and +0 alike
__device__ __forceinline__ uint32_t sample_key(float v) {
  const uint32_t b = __float_as_uint(v + 0.f);
  return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float sample_value(uint32_t key) {
  return __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key);
}

struct Found {
  u64 mass, count;
  uint32_t key, ties;
};

// One workgroup per row. Radix descent over the keys, 8 bits a pass: a pass counts
// the words and masses of 256 bins among those that share the bits found so far.
extern "C" __global__ void __launch_bounds__(1024) rxw8_sample_any(SampleArgs a) {
  __shared__ unsigned cnt[256];
  __shared__ u64 mass[256];
  __shared__ u64 red[16];
  __shared__ Found found;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t row = blockIdx.x, base = row * a.V;
  auto value = [&](int64_t i) {
    return a.bf16 ? bf16_bits_to_f32(((const uint16_t *)a.logits)[base + i]) : ((const float *)a.logits)[base + i];
  };
  // the first maximum, a NaN above every number: (key, lowest index) packed for a maximum
  u64 best = 0;
  for (int64_t i = tid; i < a.V; i += 1024) {
    const float v = value(i);
    const u64 c = ((u64)(v != v ? 0xffffffffu : sample_key(v)) << 32) | (0xffffffffu - (uint32_t)i);
    best = c > best ? c : best;
  }
  for (int o = 32; o > 0; o >>= 1) {
    const u64 c = __shfl_xor(best, o);
    best = c > best ? c : best;
  }
  if (lane == 0) red[wave] = best;
  __syncthreads();
  for (int w = 0; w < 16; ++w) best = red[w] > best ? red[w] : best;
  const uint32_t top = (uint32_t)(best >> 32);
  const float vmax = sample_value(top);
  const float T = a.temperature ? a.temperature[row] : 1.f;
  if (!(T > 0.f) || top == 0xffffffffu || !(fabsf(vmax) < __builtin_huge_valf())) {
    if (tid == 0) a.out[row] = (int32_t)(0xffffffffu - (uint32_t)best);
    return;
  }
  const double inv = 1.0 / (double)T, unit = (double)(1ull << a.shift);
  auto weight = [&](float v) { return v == -__builtin_huge_valf() ? 0.0 : exp(((double)v - (double)vmax) * inv); };
  auto units = [&](float v) { return (u64)(weight(v) * unit + 0.5); };

  // The word at which the running count reaches `count` (if above 0), else the running
  // mass m satisfies m >= want (m > want where `over`), which some word does: its key,
  // how many words have it, and the count and mass of the words of larger keys.
  auto descend = [&](u64 count, bool over, double want) {
    Found f{};
    for (int shift = 24; shift >= 0; shift -= 8) {
      for (int i = tid; i < 256; i += 1024) cnt[i] = 0, mass[i] = 0;
      __syncthreads();
      for (int64_t i = tid; i < a.V; i += 1024) {
        const float v = value(i);
        const uint32_t k = sample_key(v);
        if (shift < 24 && (k >> (shift + 8)) != f.key) continue;
        atomicAdd(&cnt[(k >> shift) & 255], 1u);
        atomicAdd(&mass[(k >> shift) & 255], units(v));
      }
      __syncthreads();
      if (tid == 0) {
        int bin = 255;
        for (; bin > 0; --bin) {
          const u64 m = f.mass + mass[bin], c = f.count + cnt[bin];
          if (cnt[bin] && (count ? c >= count : over ? (double)m > want : (double)m >= want)) break;
          f.mass = m, f.count = c;
        }
        f.key = (f.key << 8) | (uint32_t)bin;
        f.ties = cnt[bin];
        found = f;
      }
      __syncthreads();
      f = found;
      __syncthreads();
    }
    return f;
  };
  auto sum_units = [&](auto keep) {
    u64 s = 0;
    for (int64_t i = tid; i < a.V; i += 1024) {
      const float v = value(i);
      if (keep(v)) s += units(v);
    }
    for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o);
    __syncthreads();
    if (lane == 0) red[wave] = s;
    __syncthreads();
    s = 0;
    for (int w = 0; w < 16; ++w) s += red[w];
    return s;
  };

  u64 kept = sum_units([](float) { return true; });
  const int64_t k = a.top_k ? a.top_k[row] : 0;
  if (k > 0 && k < a.V) {
    const Found f = descend((u64)k, false, 0.0);
    kept = f.mass + ((u64)k - f.count) * units(sample_value(f.key));
  }
  const float p = a.top_p ? a.top_p[row] : 1.f;
  const float mp = a.min_p ? a.min_p[row] : 0.f;
  const double all = (double)kept;
  if (p < 1.f) {
    const double want = (double)p * all;
    const Found f = descend(0, false, want);
    const u64 one = units(sample_value(f.key));
    const double n = ceil((want - (double)f.mass) / (double)one);  // (want lies in these ties: one > 0)
    const u64 m = f.mass + (n > 1.0 ? (u64)n : 1) * one;
    kept = m < kept ? m : kept;
  }
  if (mp > 0.f) {
    const u64 m = sum_units([&](float v) { return weight(v) >= (double)mp; });
    kept = m < kept ? m : kept;
  }
  if (kept < (1ull << a.shift)) kept = 1ull << a.shift;  // the first word stays
  const float r = a.uniform[row], u = r > 0.f ? fminf(r, 0x1.fffffep-1f) : 0.f;
  const double want = (double)u * (double)kept;
  const Found f = descend(0, true, want);
  u64 nth = (u64)((want - (double)f.mass) / (double)units(sample_value(f.key)));
  if (nth >= f.ties) nth = f.ties - 1;
  // the nth (from 0) of the words with this key, by index
  u64 seen = 0;
  for (int64_t i0 = 0; seen <= nth; i0 += 1024) {
    __syncthreads();
    const bool hit = i0 + tid < a.V && sample_key(value(i0 + tid)) == f.key;
    const unsigned long long bal = __ballot(hit);
    if (lane == 0) red[wave] = __popcll(bal);
    __syncthreads();
    u64 before = seen + __popcll(bal & ((1ull << lane) - 1));
    for (int w = 0; w < 16; ++w) {
      if (w < wave) before += red[w];
      seen += red[w];
    }
    if (hit && before == nth) a.out[row] = (int32_t)(i0 + tid);
  }
}
