// The next token of each row of logits, from given random numbers.
//
// A row's words in order of (logit descending, index ascending); of these the first
// top_k; with weights w = exp((l - max) / T) the shortest prefix whose mass is at
// least top_p times the mass of the first top_k; of that the words with w >= min_p;
// the first word always. The token is the first whose running mass exceeds u times
// the mass of what is left. Every filter leaves a prefix of the order, so what the
// filters leave is known by its mass alone: the least of the prefixes' masses.
//
// Masses are whole numbers, round(w 2^s) in 64 bits with V 2^s <= 2^62, w in f64:
// their sums do not depend on the order of the additions (atomics included), and a
// sum over V words is off by at most V / 2 units of 2^-s (2^-45 of the largest
// weight each at V = 2^18). Words lighter than half a unit weigh nothing and can
// neither be drawn nor move a sum; they are passed over. Equal logits have equal
// masses, so within a run of ties a mass says how many of them it takes, and the
// lowest indices come first.
//
// Nothing is sorted. With z = (max - l) log2(e) / T the words go into bins of z, so
// the bins are in the words' order; the running counts and masses of the bins tell the
// bins that the borders of top_k, top_p and min_p and the token can lie in; and only the
// words of those bins, one row's some dozens to hundreds, are looked at one by one. Words
// that top_k cannot reach are passed over from the start (SampleExtremes::floor); where
// it is small, the others come as a list and the row is read twice.
// Three launches where workgroups share a row (the maxima; the bins, which the last
// workgroup of a row to arrive joins, or the list, from which it draws; the words, where
// there is no list), one where each has its own. What bounds a batch is reading the
// logits, once from memory and once or twice more from the caches; a row without a list
// takes an exponential in f64 and an LDS atomic or two for each word besides. 64 rows of
// 248320 f32 words: 46 to 49 us with top_k 200 (1.3 TB/s of logits read once; by themselves 17 us
// the maxima, 30 the list and what follows, 4 the last launch, which finds nothing to do), 76 to 92
// without a filter, 99 to 109 with top_p alone. A single row of 151936 is bound by the length of
// the chain: 26 us, of it 9, 17 and 4 by themselves.
#include <stddef.h>

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
  // S workgroups share a row, `chunk` words each (1 and V: one has it alone): extremes
  // [B][S], arrivals [B] and listed words [B] (zero between launches), and bins [B][S] of
  // 12 KiB; the row's joined bins take the place of the first's, its Borders and words that
  // of the others'
  int S;
  int64_t chunk;
  struct SampleExtremes *extremes;
  int *arrivals;
  int *listed;
  char *bins;
};

typedef unsigned long long u64;

namespace {

constexpr int kThreads = 1024, kBins = 1024, kList = 8192, kPairwise = 512;

// Ascending keys for ascending values, -0 and +0 alike; above them all a NaN
__device__ __forceinline__ uint32_t sample_key(float v) {
  const uint32_t b = __float_as_uint(v + 0.f);
  return v != v ? 0xffffffffu : b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float sample_value(uint32_t key) {
  return __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key);
}
// A word, the larger the earlier in the order
__device__ __forceinline__ u64 sample_word(uint32_t key, uint32_t index) { return (u64)key << 32 | (0xffffffffu - index); }

// f(value, index) for the words lo <= index < hi of a row, by the workgroup's threads, 16
// bytes a load but for the ends. (One load at a time: 16 waves to a CU are 16 KiB under way; two or
// four at a time took 3 to 8% longer for 64 rows of 248320, all loads of a step then being waited for.)
template <typename F>
__device__ void each_word(const void *row, bool bf16, int64_t lo, int64_t hi, F f) {
  const int tid = threadIdx.x, es = bf16 ? 2 : 4, W = 16 / es;
  const char *const p = (const char *)row;
  auto one = [&](int64_t i) {
    f(bf16 ? bf16_bits_to_f32(((const uint16_t *)row)[i]) : ((const float *)row)[i], (uint32_t)i);
  };
  const int64_t head = min(hi, lo + (int64_t)((16 - ((uintptr_t)(p + lo * es) & 15)) & 15) / es);
  const int64_t body = head + (hi - head) / W * W;
  if (lo + tid < head) one(lo + tid);
  for (int64_t i = head + (int64_t)W * tid; i < body; i += (int64_t)W * kThreads) {
    const u32x4 x = *(const u32x4 *)(p + i * es);
    if (bf16) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        f(__uint_as_float(x[e] << 16), (uint32_t)i + 2 * e);
        f(__uint_as_float(x[e] & 0xffff0000u), (uint32_t)i + 2 * e + 1);
      }
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) f(__uint_as_float(x[e]), (uint32_t)i + e);
    }
  }
  if (body + tid < hi) one(body + tid);
}

__device__ __forceinline__ u64 max_u64(u64 a, u64 b) { return a > b ? a : b; }

}  // namespace

// The first maximum of some words (a NaN above every number), their least value that is
// not -inf, and a key that at least top_k words of the row reach once all its parts' are
// joined by their minimum (0: no such key)
struct SampleExtremes {
  u64 top;
  float least;
  uint32_t floor;
};

namespace {

struct Found {
  u64 mass, count;  // of the words before those with `key`
  uint32_t key, ties;
};

struct SampleShared {
  u64 mass[kBins];      // (mass and count: 12 KiB in one piece)
  uint32_t count[kBins];
  u64 list[kList];      // words of the bins looked at
  u64 unit[kPairwise];  // their masses and bins, where they are few
  uint16_t bin[kPairwise];
  uint8_t marked[kBins];
  double exp2_table[64];
  u64 wave_mass[16];
  uint32_t wave_count[16];
  SampleExtremes wave_ext[16];
  Found found;
  u64 result;
  int n, flag, at[2];
};

struct Row {
  const void *words;
  bool bf16;
  int64_t V;
  float top;         // the maximum
  double inv;        // log2(e) / T
  double span;       // the largest z of the words in bins
  double per_bin;    // bins per unit of z
  double unit;       // 2^s
  double far;        // z from which on words weigh nothing
  float floor;       // words below it are not asked for: they come after top_k, or min_p, alone

  __device__ double z(float v) const { return ((double)top - (double)v) * inv; }
  // (zv at most span, else what this gives means nothing and indexes nothing: the nearest whole
  // number, in the low bits of a sum with 1.5 2^52)
  __device__ int bin(double zv) const {
    return min((int)(uint32_t)__builtin_bit_cast(u64, fma(zv, per_bin, 0x1.8p52)), kBins - 1);
  }
};

// 2^(-i / 64), i < 64, bit by bit
__device__ __forceinline__ void fill_table(SampleShared &sh) {
  const int tid = threadIdx.x;
  if (tid < 64) {
    double t = 1.0;
    if (tid & 1) t *= 0x1.fa7c1819e90d8p-1;
    if (tid & 2) t *= 0x1.f50765b6e4540p-1;
    if (tid & 4) t *= 0x1.ea4afa2a490dap-1;
    if (tid & 8) t *= 0x1.d5818dcfba487p-1;
    if (tid & 16) t *= 0x1.ae89f995ad3adp-1;
    if (tid & 32) t *= 0x1.6a09e667f3bcdp-1;
    sh.exp2_table[tid] = t;
  }
}

// The mass of z, 0 <= z < 54: round(2^(s - z)). z = n / 64 + r with |r| <= 1 / 128 (the addition
// rounds to 64ths and leaves n in its low bits), 2^(-n / 64) from a table of 64 and the
// exponent, 2^-r from the series of exp(-r ln 2) to the fifth power, the next term of which is
// below 2^-54; and the sum with 2^52 holds the whole number in its low bits. (Another z: no
// matter what, but nothing is read out of range.)
__device__ __forceinline__ double exp2_minus(const SampleShared &sh, double z) {
  const double t = z + 0x1.8p46;
  const int n = (int)(uint32_t)__builtin_bit_cast(u64, t);
  const double x = (z - (t - 0x1.8p46)) * -0.69314718055994530942;
  double p = fma(x, 1.0 / 120.0, 1.0 / 24.0);
  p = fma(x, p, 1.0 / 6.0);
  p = fma(x, p, 0.5);
  p = fma(x, p, 1.0);
  p = fma(x, p, 1.0);
  return __builtin_bit_cast(double, __builtin_bit_cast(u64, p * sh.exp2_table[n & 63]) - ((u64)(n >> 6) << 52));
}
__device__ __forceinline__ u64 units_of(const Row &r, double w) {
  return __builtin_bit_cast(u64, fma(w, r.unit, 0x1p52)) & 0xfffffffffffffull;
}
// Whether min_p = m > 0 leaves a word of weight w at z. (m = 1 leaves the first's ties alone, though w
// rounds to 1 from z = 2^-53 down; the m below it is 1 - 2^-24.)
__device__ __forceinline__ bool min_p_leaves(double m, double z, double w) { return m < 1.0 ? w >= m : m == 1.0 && z == 0.0; }
// The mass of a word (0 from r.far on)
__device__ __forceinline__ u64 units_at(const SampleShared &sh, const Row &r, float v) {
  const double z = r.z(v);
  return z < r.far ? units_of(r, exp2_minus(sh, z)) : 0;
}

// Extremes over the workgroup, in every thread
__device__ SampleExtremes join_extremes(SampleShared &sh, SampleExtremes e) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (int o = 32; o > 0; o >>= 1) {
    e.top = max_u64(e.top, __shfl_xor(e.top, o));
    e.least = fminf(e.least, __shfl_xor(e.least, o));
    e.floor = min(e.floor, __shfl_xor(e.floor, o));
  }
  __syncthreads();
  if (lane == 0) sh.wave_ext[wave] = e;
  __syncthreads();
  for (int w = 0; w < kThreads / 64; ++w) {
    e.top = max_u64(e.top, sh.wave_ext[w].top);
    e.least = fminf(e.least, sh.wave_ext[w].least);
    e.floor = min(e.floor, sh.wave_ext[w].floor);
  }
  return e;
}
// ... of the words lo <= index < hi of a row. The floor: of the threads' maxima (not -inf) the
// top_k / S-th from above or one a little below it, found in a histogram over their range.
// (As many words reach it and not many more: each thread has its words from all over the row.)
__device__ SampleExtremes extremes_of(SampleShared &sh, const SampleArgs &a, int64_t row, const void *words, int64_t lo, int64_t hi) {
  const int tid = threadIdx.x;
  uint32_t key = 0, index = 0xffffffffu;
  float least = __builtin_huge_valf();
  each_word(words, a.bf16, lo, hi, [&](float v, uint32_t i) {  // (a thread's words come in order)
    const uint32_t k = sample_key(v);
    const bool better = k > key;
    key = better ? k : key, index = better ? i : index;
    least = fminf(least, v > -__builtin_huge_valf() ? v : __builtin_huge_valf());
  });
  const uint32_t none = sample_key(-__builtin_huge_valf());
  const bool has = key > none && key != 0xffffffffu;
  SampleExtremes e = join_extremes(sh, SampleExtremes{sample_word(key, index), least, has ? key : 0xffffffffu});
  const int64_t k = a.top_k ? a.top_k[row] : 0, wanted = (k + a.S - 1) / a.S;
  const float from = sample_value(e.floor), to = sample_value((uint32_t)(e.top >> 32));
  e.floor = 0;
  if (k <= 0 || k >= a.V || wanted > kThreads / 2 || !(to < __builtin_huge_valf()) || !(from <= to)) return e;
  const float per = to - from, scale = per > 0.f ? (float)(kBins - 1) / per : 0.f;
  const int bin = has ? min((int)((sample_value(key) - from) * scale), kBins - 1) : -1;
  sh.count[tid] = 0;
  if (tid == 0) sh.at[0] = -1, sh.at[1] = -1;
  __syncthreads();
  if (has) atomicAdd(&sh.count[bin], 1u);
  __syncthreads();
  if (tid < 64) {  // 16 bins a lane, from the last down
    const uint32_t *const mine = sh.count + kBins - 16 * (tid + 1);
    uint32_t sum = 0;
    for (int i = 0; i < 16; ++i) sum += mine[i];
    uint32_t all = sum;
    for (int o = 1; o < 64; o <<= 1) {
      const uint32_t x = __shfl_up(all, o);
      if (tid >= o) all += x;
    }
    uint32_t before = all - sum;
    if (before < wanted && all >= wanted) {
      int i = 15;
      while ((before += mine[i]) < wanted) --i;
      sh.at[0] = kBins - 16 * (tid + 1) + i;
    }
  }
  __syncthreads();
  const int border = sh.at[0];
  if (border >= 0) {  // (below 0: not as many threads have words)
    uint32_t floor = bin >= border ? key : 0xffffffffu;
    for (int o = 32; o > 0; o >>= 1) floor = min(floor, __shfl_xor(floor, o));
    if ((tid & 63) == 0) atomicMin((uint32_t *)&sh.at[1], floor);
    __syncthreads();
    e.floor = (uint32_t)sh.at[1];
  }
  return e;
}

// Radix descent, 8 bits a pass, over the words that each(f) hands to f(here, key, units), whole
// waves at a time: the key at which the running count reaches `count` (if above 0), else the
// running mass m satisfies m >= want (m > want where `over`), as some key's does; counts and
// masses begin with `before`'s.
template <typename Each>
__device__ Found descend(SampleShared &sh, Each each, Found before, u64 count, bool over, double want) {
  const int tid = threadIdx.x;
  Found f = before;
  f.key = 0;
  for (int shift = 24; shift >= 0; shift -= 8) {
    __syncthreads();
    if (tid < 256) sh.count[tid] = 0, sh.mass[tid] = 0;
    __syncthreads();
    each([&](bool word, uint32_t k, u64 u) {
      const bool here = word && (shift == 24 || (k >> (shift + 8)) == f.key);
      const u64 all = __ballot(here);
      if (!all) return;
      // words of one digit, as ties are, in one addition: 64 of them to one address take turns
      const uint32_t digit = (k >> shift) & 255;
      const int lead = __builtin_ctzll(all);
      const bool same = here && digit == (uint32_t)__builtin_amdgcn_readlane((int)digit, lead);
      const int together = __popcll(__ballot(same));
      if (together > 8) {
        u64 sum = same ? u : 0;
        for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o);
        if ((tid & 63) == lead) {
          atomicAdd(&sh.count[digit], (uint32_t)together);
          atomicAdd(&sh.mass[digit], sum);
        }
      }
      if (here && !(same && together > 8)) {
        atomicAdd(&sh.count[digit], 1u);
        atomicAdd(&sh.mass[digit], u);
      }
    });
    __syncthreads();
    if (tid < 64) {  // the bins from the last down, four to a lane
      uint32_t cnt[4];
      u64 m[4], own_m = 0, own_c = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        cnt[j] = sh.count[255 - 4 * tid - j], m[j] = sh.mass[255 - 4 * tid - j];
        own_m += m[j], own_c += cnt[j];
      }
      u64 all_m = own_m, all_c = own_c;
      for (int o = 1; o < 64; o <<= 1) {
        const u64 x = __shfl_up(all_m, o), y = __shfl_up(all_c, o);
        if (tid >= o) all_m += x, all_c += y;
      }
      Found g{f.mass + all_m - own_m, f.count + all_c - own_c, 0, 0};
      bool hit = false;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (!hit) {
          const int b = 255 - 4 * tid - j;
          const u64 mass = g.mass + m[j], n = g.count + cnt[j];
          hit = b == 0 || (cnt[j] && (count ? n >= count : over ? (double)mass > want : (double)mass >= want));
          if (hit)
            g.key = (f.key << 8) | (uint32_t)b, g.ties = cnt[j];
          else
            g.mass = mass, g.count = n;
        }
      if (tid == __builtin_ctzll(__ballot(hit))) sh.found = g;  // (the last lane's is one at least)
    }
    __syncthreads();
    f = sh.found;
  }
  __syncthreads();
  return f;
}

struct Settings {
  float u, p, m;
  int64_t k;
};

// The mass of a prefix that ends within ties: `before` and as many of them as reach `want`
__device__ u64 mass_reaching(const Found &f, u64 one, double want) {
  const double n = one ? ceil((want - (double)f.mass) / (double)one) : 1.0;
  return f.mass + (n > 1.0 ? min((u64)n, (u64)f.ties) : 1) * one;
}
// Which of the ties (from 0) the running mass passes `want` at
__device__ u64 tie_passing(const Found &f, u64 one, double want) {
  const u64 n = one && want > (double)f.mass ? (u64)((want - (double)f.mass) / (double)one) : 0;
  return n < f.ties ? n : f.ties - 1;
}

// The token by descents over all words of the row (where a bin holds more of them than the list:
// long runs of ties): 1.7 ms for 151936 equal logits, as every descent reads the row four times
__device__ int32_t draw_from_row(SampleShared &sh, const Row &r, const Settings &s) {
  auto each_of_row = [&](auto f) {  // f(here, value, index), four loads at a time
    for (int64_t i0 = threadIdx.x; i0 - threadIdx.x < r.V; i0 += 4 * kThreads) {
      float v[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int64_t i = min(i0 + e * kThreads, r.V - 1);
        v[e] = r.bf16 ? bf16_bits_to_f32(((const uint16_t *)r.words)[i]) : ((const float *)r.words)[i];
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) f(i0 + e * kThreads < r.V, v[e], (uint32_t)(i0 + e * kThreads));
    }
  };
  auto word = [&](auto f) { each_of_row([&](bool here, float v, uint32_t) { f(here, sample_key(v), units_at(sh, r, v)); }); };
  auto sum = [&](double min_p) {  // of the words that min_p leaves (0: all)
    u64 m = 0;
    each_word(r.words, r.bf16, 0, r.V, [&](float v, uint32_t) {
      const double z = r.z(v), w = z < r.far ? exp2_minus(sh, z) : 0.0;
      if (!(min_p > 0.0) || min_p_leaves(min_p, z, w)) m += units_of(r, w);
    });
    for (int o = 32; o > 0; o >>= 1) m += __shfl_xor(m, o);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sh.wave_mass[threadIdx.x >> 6] = m;
    __syncthreads();
    m = 0;
    for (int w = 0; w < kThreads / 64; ++w) m += sh.wave_mass[w];
    return m;
  };
  const Found none{};
  u64 kept = sum(0.0);
  if (s.k > 0 && s.k < r.V) {
    const Found f = descend(sh, word, none, (u64)s.k, false, 0.0);
    kept = f.mass + ((u64)s.k - f.count) * units_at(sh, r, sample_value(f.key));
  }
  const double all = (double)kept;
  if (s.p < 1.f) {
    const Found f = descend(sh, word, none, 0, false, (double)s.p * all);
    kept = min(kept, mass_reaching(f, units_at(sh, r, sample_value(f.key)), (double)s.p * all));
  }
  if (s.m > 0.f) kept = min(kept, sum((double)s.m));
  kept = max_u64(kept, (u64)r.unit);
  const double want = (double)s.u * (double)kept;
  const Found f = descend(sh, word, none, 0, true, want);
  const u64 nth = tie_passing(f, units_at(sh, r, sample_value(f.key)), want);
  const Found at = descend(sh, [&](auto g) {
    each_of_row([&](bool here, float v, uint32_t i) { g(here && sample_key(v) == f.key, 0xffffffffu - i, 0); });
  }, none, nth + 1, false, 0.0);
  return (int32_t)(0xffffffffu - at.key);
}

// The bins that a row's borders and token can lie in
struct Borders {
  u64 total;          // the row's mass
  float least, most;  // what the values of these bins lie between
  int kb, mb;         // the bins of top_k's border, and of min_p's, give or take one (-1: none)
  int pb0, pb1;       // ... of top_p's (pb0 > pb1: none)
  int db0, db1;       // ... of the token
  int done;           // the token is out already
};

// ... from the counts and masses of the row's bins, which become running ones (in sh)
__device__ Borders borders_of(SampleShared &sh, const Row &r, const Settings &s) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  // ---- running masses and counts before each bin, in place: a bin a thread
  const u64 mine = sh.mass[tid];
  const uint32_t mine_c = sh.count[tid];
  u64 m = mine;
  uint32_t c = mine_c;
  for (int o = 1; o < 64; o <<= 1) {
    const u64 x = __shfl_up(m, o);
    const uint32_t y = __shfl_up(c, o);
    if (lane >= o) m += x, c += y;
  }
  if (lane == 63) sh.wave_mass[wave] = m, sh.wave_count[wave] = c;
  __syncthreads();
  u64 total = 0;
  uint32_t counted = 0;
  for (int w = 0; w < kThreads / 64; ++w) {
    if (w < wave) m += sh.wave_mass[w], c += sh.wave_count[w];
    total += sh.wave_mass[w], counted += sh.wave_count[w];
  }
  const double end = (double)m;  // of this thread's bin
  m -= mine, c -= mine_c;
  const double begin = (double)m;
  sh.mass[tid] = m, sh.count[tid] = c;
  auto mass_end = [&](int b) { return b + 1 < kBins ? sh.mass[b + 1] : total; };
  // The bins in which masses want[0] and want[1] are reached (`over`: passed): the thread whose bin it is says so
  auto bins_of = [&](bool over, double want0, double want1, int &b0, int &b1) {
    if (tid < 2) sh.at[tid] = over ? kBins - 1 : 0;
    __syncthreads();
    if (over ? begin <= want0 && end > want0 : begin < want0 && end >= want0) sh.at[0] = tid;
    if (over ? begin <= want1 && end > want1 : begin < want1 && end >= want1) sh.at[1] = tid;
    __syncthreads();
    b0 = sh.at[0], b1 = sh.at[1];
    __syncthreads();
  };
  // ---- the bins in which borders and token can lie (uniform over the workgroup)
  u64 kept_lo = total, kept_hi = total;  // bounds of what is left
  int kb = -1, pb0 = 1, pb1 = 0, mb = -1, db0, db1;
  __syncthreads();
  if (s.k > 0 && s.k < counted) {
    if (c < s.k && c + mine_c >= s.k) sh.at[0] = tid;
    __syncthreads();
    kb = sh.at[0];
    __syncthreads();
    kept_lo = sh.mass[kb], kept_hi = mass_end(kb);
  }
  if (s.p < 1.f) {
    bins_of(false, (double)s.p * (double)kept_lo, (double)s.p * (double)kept_hi, pb0, pb1);
    kept_lo = min(kept_lo, sh.mass[pb0]);
    kept_hi = min(kept_hi, mass_end(pb1));
  }
  if (s.m > 0.f) {
    // (min_p's border may lie far behind the last word: bins are as fine as the row's span is short)
    mb = s.m >= 1.f ? 0 : r.bin(fmin(-log2((double)s.m), r.span));
    kept_lo = min(kept_lo, sh.mass[max(mb - 1, 0)]);
    kept_hi = min(kept_hi, mass_end(min(mb + 1, kBins - 1)));
  }
  const u64 first = (u64)r.unit;  // the first word stays
  kept_lo = max_u64(kept_lo, first), kept_hi = max_u64(kept_hi, first);
  bins_of(true, (double)s.u * (double)kept_lo, (double)s.u * (double)kept_hi, db0, db1);
  // ... and the values these bins lie between, a bin and two steps wider
  int b_lo = min(db0, kBins - 1), b_hi = db1;
  if (kb >= 0) b_lo = min(b_lo, kb), b_hi = max(b_hi, kb);
  if (pb0 <= pb1) b_lo = min(b_lo, pb0), b_hi = max(b_hi, pb1);
  if (mb >= 0) b_lo = min(b_lo, mb - 1), b_hi = max(b_hi, mb + 1);
  auto key_at = [&](int b) { return sample_key((float)((double)r.top - (double)b / (r.per_bin * r.inv))); };
  const float v_lo = sample_value(max(key_at(b_hi + 1) - 2, sample_key(-__builtin_huge_valf())));
  const float v_hi = b_lo <= 1 ? r.top : sample_value(min(key_at(b_lo - 1) + 2, sample_key(r.top)));
  return Borders{total, b_hi + 1 < kBins ? fmaxf(v_lo, r.floor) : r.floor, v_hi, kb, mb, pb0, pb1, db0, db1, 0};
}

__device__ __forceinline__ bool looked_at(const Borders &b, int bin) {
  return bin == b.kb || (bin >= b.pb0 && bin <= b.pb1) || (b.mb >= 0 && abs(bin - b.mb) <= 1) ||
         (bin >= b.db0 && bin <= b.db1);
}
__device__ __forceinline__ void list_word(SampleShared &sh, u64 word) {
  const int at = atomicAdd(&sh.n, 1);
  if (at < kList) sh.list[at] = word;
}
// The words lo <= index < hi in these bins, the first kList of them in sh.list; sh.n of them
__device__ void words_of(SampleShared &sh, const Row &r, const Borders &b, int64_t lo, int64_t hi) {
  const int tid = threadIdx.x;
  __syncthreads();
  sh.marked[tid] = looked_at(b, tid);
  if (tid == 0) sh.n = 0;
  __syncthreads();
  each_word(r.words, r.bf16, lo, hi, [&](float v, uint32_t i) {
    if (!(v >= b.least && v <= b.most)) return;
    const double z = r.z(v);
    if (z < r.far && sh.marked[r.bin(z)]) list_word(sh, sample_word(sample_key(v), i));
  });
  __syncthreads();
}
// ... not below the row's floor
__device__ void words_from_floor(SampleShared &sh, const Row &r, int64_t lo, int64_t hi) {
  __syncthreads();
  if (threadIdx.x == 0) sh.n = 0;
  __syncthreads();
  each_word(r.words, r.bf16, lo, hi, [&](float v, uint32_t i) {
    if (v >= r.floor) list_word(sh, sample_word(sample_key(v), i));
  });
  __syncthreads();
}

// The token, from these words and the running masses and counts (in sh)
__device__ int32_t draw(SampleShared &sh, const Row &r, const Settings &s, const Borders &borders) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const u64 total = borders.total, first = (u64)r.unit;
  const int kb = borders.kb, mb = borders.mb, pb0 = borders.pb0, pb1 = borders.pb1, db0 = borders.db0, db1 = borders.db1;
  const int n = sh.n;
  if (n > kList) return draw_from_row(sh, r, s);

  u64 kept = total;
  if (n <= kPairwise) {
    // of each word those before it in its bin, by as many threads as there are. (A thread each,
    // for up to 1024 words: 123 us for 4 rows of 248320 bf16 words cut in a crowd of ties, 58 so.)
    u64 *const ahead = sh.list + kPairwise;
    uint32_t *const ranks = (uint32_t *)(sh.list + 2 * kPairwise);
    int wide = 64;
    while (wide < n) wide <<= 1;
    u64 word = 0, one = 0, before = 0;
    uint32_t rank = 0;
    double z = 0.0, w = 0.0;
    int b = -1;
    if (tid < n) {
      word = sh.list[tid];
      z = r.z(sample_value((uint32_t)(word >> 32)));
      b = r.bin(z), w = exp2_minus(sh, z), one = units_of(r, w);
      sh.bin[tid] = (uint16_t)b, sh.unit[tid] = one;
      ahead[tid] = sh.mass[b], ranks[tid] = sh.count[b];
    }
    __syncthreads();
    if (const int at = tid & (wide - 1); at < n) {
      const u64 its = sh.list[at];
      const int its_bin = sh.bin[at];
      u64 sum = 0;
      uint32_t some = 0;
      for (int j = tid / wide; j < n; j += kThreads / wide)
        if (sh.list[j] > its && sh.bin[j] == its_bin) sum += sh.unit[j], ++some;
      if (some) {
        atomicAdd(&ahead[at], sum);
        atomicAdd(&ranks[at], some);
      }
    }
    __syncthreads();
    if (tid < n) before = ahead[tid], rank = ranks[tid];
    auto ask = [&](bool here, u64 answer) {  // from the one thread that has it
      if (here) sh.result = answer;
      __syncthreads();
      const u64 a = sh.result;
      __syncthreads();
      return a;
    };
    const u64 end_of = before + one;
    if (kb >= 0) kept = ask(tid < n && b == kb && rank + 1 == s.k, end_of);
    if (s.p < 1.f) {
      const double want = (double)s.p * (double)kept;
      if (tid == 0) sh.result = first;  // (want not above 0: the first word)
      __syncthreads();
      const u64 at = ask(tid < n && (double)before < want && (double)end_of >= want, end_of);
      kept = min(kept, at);
    }
    if (mb >= 0) {
      u64 sum = tid < n && abs(b - mb) <= 1 && min_p_leaves((double)s.m, z, w) ? one : 0;
      for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o);
      if (lane == 0) sh.wave_mass[wave] = sum;
      __syncthreads();
      sum = sh.mass[max(mb - 1, 0)];
      for (int x = 0; x < kThreads / 64; ++x) sum += sh.wave_mass[x];
      kept = min(kept, sum);
    }
    kept = max_u64(kept, first);
    const double want = (double)s.u * (double)kept;
    return (int32_t)ask(tid < n && (double)before <= want && (double)end_of > want, 0xffffffffu - (uint32_t)word);
  }

  // many words: descents over the list, bin by bin (sh.mass and sh.count are the descents' own:
  // what begins before a bin is read first)
  auto begin_of = [&](int b) { return Found{sh.mass[b], sh.count[b], 0, 0}; };
  const Found kf = begin_of(max(kb, 0)), mf = begin_of(max(mb - 1, 0));
  // (running masses at the ends of the bins from pb0 and db0 on, at most kPairwise of them)
  __syncthreads();
  const int np = s.p < 1.f ? pb1 - pb0 + 1 : 0, nd = db1 - db0 + 1;
  if (np + nd + 2 > kPairwise) return draw_from_row(sh, r, s);
  for (int i = tid; i < np + nd; i += kThreads) sh.unit[i] = sh.mass[i < np ? pb0 + i : db0 + i - np];
  __syncthreads();
  auto each_of_list = [&](auto f) {  // f(here, word)
    for (int i0 = 0; i0 < n; i0 += kThreads) f(i0 + tid < n, i0 + tid < n ? sh.list[i0 + tid] : 0);
  };
  auto in_bin = [&](int bin) {
    return [&, bin](auto f) {
      each_of_list([&](bool here, u64 word) {
        const uint32_t k = (uint32_t)(word >> 32);
        const double z = r.z(sample_value(k));
        f(here && r.bin(z) == bin, k, units_of(r, exp2_minus(sh, z)));
      });
    };
  };
  auto last_before = [&](int at, int count, bool over, double want) {  // the bin the mass `want` lies in
    int i = 0;
    while (i + 1 < count && (over ? (double)sh.unit[at + i + 1] <= want : (double)sh.unit[at + i + 1] < want)) ++i;
    return i;
  };
  if (kb >= 0) {
    const Found f = descend(sh, in_bin(kb), kf, (u64)s.k, false, 0.0);
    kept = f.mass + ((u64)s.k - f.count) * units_at(sh, r, sample_value(f.key));
  }
  if (s.p < 1.f) {
    const double want = (double)s.p * (double)kept;
    const int i = last_before(0, np, false, want);
    const Found f = descend(sh, in_bin(pb0 + i), Found{sh.unit[i], 0, 0, 0}, 0, false, want);
    kept = min(kept, want > 0.0 ? mass_reaching(f, units_at(sh, r, sample_value(f.key)), want) : first);
  }
  if (mb >= 0) {
    u64 sum = 0;
    for (int i = tid; i < n; i += kThreads) {
      const double z = r.z(sample_value((uint32_t)(sh.list[i] >> 32))), w = exp2_minus(sh, z);
      if (abs(r.bin(z) - mb) <= 1 && min_p_leaves((double)s.m, z, w)) sum += units_of(r, w);
    }
    for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o);
    __syncthreads();
    if (lane == 0) sh.wave_mass[wave] = sum;
    __syncthreads();
    sum = mf.mass;
    for (int x = 0; x < kThreads / 64; ++x) sum += sh.wave_mass[x];
    kept = min(kept, sum);
  }
  kept = max_u64(kept, first);
  const double want = (double)s.u * (double)kept;
  const int i = last_before(np, nd, true, want);
  const Found f = descend(sh, in_bin(db0 + i), Found{sh.unit[np + i], 0, 0, 0}, 0, true, want);
  const u64 nth = tie_passing(f, units_at(sh, r, sample_value(f.key)), want);
  const Found at = descend(sh, [&](auto g) {
    each_of_list([&](bool here, u64 word) { g(here && (uint32_t)(word >> 32) == f.key, (uint32_t)word, 0); });
  }, Found{}, nth + 1, false, 0.0);
  return (int32_t)(0xffffffffu - at.key);
}

constexpr int kBinWords = 12 * 1024 / 8;  // masses, then counts two to a word, none above 2^24
static_assert(sizeof SampleShared::mass + sizeof SampleShared::count == 8 * kBinWords &&
                  offsetof(SampleShared, count) == sizeof SampleShared::mass && sizeof(Borders) <= 64,
              "mass and count in one piece");

__device__ const void *words_at(const SampleArgs &a, int64_t row) { return (const char *)a.logits + row * a.V * (a.bf16 ? 2 : 4); }
__device__ u64 *bins_at(const SampleArgs &a, int64_t row, int part) { return (u64 *)a.bins + (row * a.S + part) * kBinWords; }
__device__ Borders *borders_at(const SampleArgs &a, int64_t row) { return (Borders *)bins_at(a, row, 1); }
__device__ u64 *list_at(const SampleArgs &a, int64_t row) { return bins_at(a, row, 1) + 8; }
__device__ int list_size(const SampleArgs &a) { return min((a.S - 1) * kBinWords - 8, kList); }

__device__ SampleExtremes row_extremes(const SampleArgs &a, int64_t row) {
  SampleExtremes e = a.extremes[row * a.S + min((int)(threadIdx.x & 63), a.S - 1)];
  for (int o = 32; o > 0; o >>= 1) {
    e.top = max_u64(e.top, __shfl_xor(e.top, o));
    e.least = fminf(e.least, __shfl_xor(e.least, o));
    e.floor = min(e.floor, __shfl_xor(e.floor, o));
  }
  return e;
}

// False where the token is the first maximum: no temperature, a NaN, or an infinite maximum
// (uniform over the row)
__device__ bool set_row(const SampleArgs &a, int64_t row, const SampleExtremes &e, Row &r, Settings &s) {
  r.words = words_at(a, row), r.bf16 = a.bf16, r.V = a.V;
  const uint32_t top = (uint32_t)(e.top >> 32);
  const float T = a.temperature ? a.temperature[row] : 1.f;
  r.top = sample_value(top);
  if (!(T > 0.f) || top == 0xffffffffu || !(fabsf(r.top) < __builtin_huge_valf())) return false;
  r.inv = 1.44269504088896340736 / (double)T;
  r.unit = (double)(1ull << a.shift);
  r.far = (double)a.shift + 1.0;
  const float u = a.uniform[row];
  s.u = u > 0.f ? fminf(u, 0x1.fffffep-1f) : 0.f;
  s.k = a.top_k ? a.top_k[row] : 0;
  s.p = a.top_p ? a.top_p[row] : 1.f;
  s.m = a.min_p ? a.min_p[row] : 0.f;
  if (s.k >= a.V) s.k = 0;
  const float lowest = -__builtin_huge_valf();
  r.floor = e.floor > sample_key(lowest) ? sample_value(e.floor) : lowest;
  if (s.m > 0.f && !(s.p < 1.f)) {  // (min_p leaves nothing below two steps under this)
    const double z = fmin(fmax(-log2((double)s.m), 0.0) + 0x1p-20, r.far);
    r.floor = fmaxf(r.floor, sample_value(max(sample_key((float)((double)r.top - z / r.inv)) - 2, sample_key(lowest))));
  }
  // bins over what weighs something, and no further than the row goes
  r.span = fmin(r.z(fmaxf(e.least, r.floor)), r.far);
  r.per_bin = r.span > 0.0 ? (double)(kBins - 1) / r.span : 0.0;
  return true;
}
// Whether this workgroup is the row's last to arrive; what all have stored past the dies' caches
// (agent scope) before is then there to read, and the counter is back at zero
__device__ bool last_of_row(const SampleArgs &a, SampleShared &sh, int64_t row) {
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (threadIdx.x == 0) {
    sh.flag = __hip_atomic_fetch_add(a.arrivals + row, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == a.S - 1;
    if (sh.flag) __hip_atomic_store(a.arrivals + row, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __syncthreads();
  return sh.flag;
}

// The words that a row's workgroups have each in its sh.list, sh.n of them, in the last one's:
// whether this is it. (sh.n above kList: they are not there, the row's list being too small.)
__device__ bool list_of_row(const SampleArgs &a, SampleShared &sh, int64_t row) {
  const int tid = threadIdx.x, n = sh.n, most = list_size(a);
  u64 *const list = list_at(a, row);
  if (tid == 0) sh.flag = __hip_atomic_fetch_add(a.listed + row, n, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  __syncthreads();
  const int at = sh.flag;
  for (int i = tid; i < n && at + i < most; i += kThreads)
    __hip_atomic_store(list + at + i, sh.list[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  if (!last_of_row(a, sh, row)) return false;
  if (tid == 0) {
    const int all = __hip_atomic_load(a.listed + row, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    sh.n = all <= most ? all : kList + 1;
    __hip_atomic_store(a.listed + row, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __syncthreads();
  if (sh.n <= kList)
    for (int i = tid; i < sh.n; i += kThreads)
      sh.list[i] = __hip_atomic_load(list + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  __syncthreads();
  return true;
}

}  // namespace

static_assert(sizeof(SampleShared) <= 92 << 10 && sizeof(SampleExtremes) == 16, "what the host lays out");

extern "C" __global__ void __launch_bounds__(kThreads) rxw8_sample_extremes(SampleArgs a) {
  extern __shared__ __attribute__((aligned(16))) char lds[];
  SampleShared &sh = *(SampleShared *)lds;
  const int64_t row = blockIdx.x / a.S, part = blockIdx.x - row * a.S, lo = part * a.chunk;
  const SampleExtremes e = extremes_of(sh, a, row, words_at(a, row), lo, min(lo + a.chunk, a.V));
  if (threadIdx.x == 0) a.extremes[blockIdx.x] = e;
}

extern "C" __global__ void __launch_bounds__(kThreads) rxw8_sample_draw(SampleArgs a) {
  extern __shared__ __attribute__((aligned(16))) char lds[];
  SampleShared &sh = *(SampleShared *)lds;
  const int tid = threadIdx.x;
  const int64_t row = blockIdx.x / a.S, part = blockIdx.x - row * a.S;
  Row r;
  SampleExtremes e;
  if (a.S == 1) {
    e = extremes_of(sh, a, row, words_at(a, row), 0, a.V);
  } else {
    e = row_extremes(a, row);
  }
  Settings s;
  if (!set_row(a, row, e, r, s)) {
    if (part == 0 && tid == 0) a.out[row] = (int32_t)(0xffffffffu - (uint32_t)e.top);
    return;
  }
  static_assert(kBins == kThreads, "a bin a thread");
  sh.mass[tid] = 0, sh.count[tid] = 0;
  fill_table(sh);
  __syncthreads();
  const int64_t lo = part * a.chunk, hi = min(lo + a.chunk, a.V);
  // (the arithmetic for every word, wanted or not: branches around it, which keep the words'
  // chains from running side by side, took 40 us longer for 64 rows of 248320 without top_k)
  auto weigh = [&](float v) {
    const double z = r.z(v);
    const int b = r.bin(z);
    const u64 units = units_of(r, exp2_minus(sh, z));
    if (v >= r.floor && z < r.far) {
      atomicAdd(&sh.mass[b], units);
      if (s.k > 0) atomicAdd(&sh.count[b], 1u);
    }
  };
  const bool listed_path = s.k > 0 && 2 * s.k + 64 <= (a.S > 1 ? list_size(a) : kList) && e.floor > sample_key(-__builtin_huge_valf());
  bool listed = false;  // (too many for the list: this workgroup takes the row's bins alone)
  if (listed_path) {
    // top_k leaves few words that it can reach, as a rule not twice as many: these go into a
    // list, and from there into the bins
    words_from_floor(sh, r, lo, hi);
    if (a.S > 1 && !list_of_row(a, sh, row)) return;
    listed = sh.n <= kList;
    if (listed)
      for (int i = tid; i < sh.n; i += kThreads) weigh(sample_value((uint32_t)(sh.list[i] >> 32)));
    else
      each_word(r.words, r.bf16, 0, a.V, [&](float v, uint32_t) { weigh(v); });
    __syncthreads();
  } else {
    each_word(r.words, r.bf16, lo, hi, [&](float v, uint32_t) { weigh(v); });
    __syncthreads();
  }
  if (a.S > 1 && !listed_path) {
    // the row's last workgroup joins the bins of all
    u64 *const here = sh.mass;
    const int used = s.k > 0 ? kBinWords : kBins;
    for (int i = tid; i < used; i += kThreads)
      __hip_atomic_store(bins_at(a, row, part) + i, here[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    if (!last_of_row(a, sh, row)) return;
    for (int i = tid; i < used; i += kThreads) {
      u64 x[8], sum = 0;
#pragma unroll
      for (int p = 0; p < 8; ++p)
        x[p] = p < a.S ? __hip_atomic_load(bins_at(a, row, p) + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : 0;
#pragma unroll
      for (int p = 0; p < 8; ++p) sum += x[p];
      here[i] = sum;
    }
    __syncthreads();
  }
  Borders b = borders_of(sh, r, s);
  if (listed) {
    // of the list the words in the bins looked at
    u64 word[kList / kThreads];
#pragma unroll
    for (int j = 0; j < kList / kThreads; ++j) {
      const int i = j * kThreads + tid;
      word[j] = i < sh.n ? sh.list[i] : 0;  // (no word is 0)
    }
    __syncthreads();
    if (tid == 0) sh.n = 0;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kList / kThreads; ++j) {
      const double z = r.z(sample_value((uint32_t)(word[j] >> 32)));
      if (word[j] && z < r.far && looked_at(b, r.bin(z))) list_word(sh, word[j]);
    }
    __syncthreads();
    b.done = 1;
  }
  if (a.S > 1) {
    if (!b.done)
      for (int i = tid; i < kBinWords; i += kThreads) bins_at(a, row, 0)[i] = sh.mass[i];
    if (tid == 0) *borders_at(a, row) = b;
    if (!b.done) return;
  }
  if (!b.done) words_of(sh, r, b, 0, a.V);
  const int32_t token = draw(sh, r, s, b);
  if (tid == 0) a.out[row] = token;
}

// The words of a shared row that are looked at, and its token
extern "C" __global__ void __launch_bounds__(kThreads) rxw8_sample_words(SampleArgs a) {
  extern __shared__ __attribute__((aligned(16))) char lds[];
  SampleShared &sh = *(SampleShared *)lds;
  const int tid = threadIdx.x;
  const int64_t row = blockIdx.x / a.S, part = blockIdx.x - row * a.S;
  const Borders b = *borders_at(a, row);
  if (b.done) return;  // (where the token is the first maximum, whatever this is: set_row says so)
  const SampleExtremes e = row_extremes(a, row);
  Row r;
  Settings s;
  if (!set_row(a, row, e, r, s)) return;
  fill_table(sh);
  const int64_t lo = part * a.chunk;
  words_of(sh, r, b, lo, min(lo + a.chunk, a.V));
  if (!list_of_row(a, sh, row)) return;
  if (sh.n > kList) words_of(sh, r, b, 0, a.V);  // more than the list takes: all of them by this one
  for (int i = tid; i < kBinWords; i += kThreads) sh.mass[i] = bins_at(a, row, 0)[i];
  __syncthreads();
  const int32_t token = draw(sh, r, s, b);
  if (tid == 0) a.out[row] = token;
}
