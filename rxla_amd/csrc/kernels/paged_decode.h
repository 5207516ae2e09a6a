// The matrix-core kernels over paged caches.
#pragma once
#include <type_traits>

#include "paged.h"

// ---- head widths 64, 128, 256, pages of whole 16-row pieces: matrix cores --------
//
// What bounds it is the cache: 2 D keys' bytes read once, for G = Hq / Hkv query
// heads together (they are the columns of the products, up to 16; more heads take
// further workgroups). So the work is dealt by bytes: the keys of a kv head, all
// sequences one after another, are a run of tiles of KT keys; each of its `units`
// workgroups (one fills a CU, by LDS) takes an equal piece of the run and each wave
// of it an equal piece of that, whatever the sequences' lengths. A wave that meets
// a sequence's end goes on with the next one. (8 sequences of 512 to 8192 keys, 32 / 8 heads
// of 128, bf16: 24.5 us, 3.9 TB/s; 96 of 1 to 1500, 16 / 8 heads: 59.6 us, 3.5 TB/s.)
//
// A wave copies its tiles by LDS DMA into memory of its own, K and V a tile each, and
// the next K goes out when the products with this one are done, the next V likewise:
// the loop has no barrier and holds no registers for loads, and a CU has some 64 KiB on
// their way. (Twice that, with two tiles of each: 32.2 us against 30.7 for 8 sequences
// of 4096 keys, 32 / 8 heads; what is more in flight than the memory takes only waits
// longer, and the waves end further apart.) Rows keep their order in LDS, their 16-byte
// chunks XOR-swizzled by row. Per 16 keys and 16 heads:
//   S^T = K q^T    A = K rows, B = q: 16x16x32 bf16 (an f32 q as its three bf16 parts:
//                  exact products), 16x16x4 f32;
//   softmax        lane = head, its four lanes share the keys; O is rescaled only
//                  where the running maximum moves;
//   O^T += V^T P^T A = V by transposing reads (bf16), B = P straight from the score
//                  registers, as its three bf16 parts for an f32 output, as two (2^-16
//                  of P, behind an output rounded to 2^-8) for a bf16 one (16x16x16);
//                  f32 caches take f32 products, the dims in the order of 16-byte pieces.
// V rows that a tile's last key or a missing page leaves unseen are cleared in LDS
// (their weights are zero, what they hold may be NaN); K's scores there are -inf.
//
// 8-bit rows come as codes, half the bytes, and their scales beside them by 4-byte copies: a
// tile's K and V scales are under way with its K rows. What bounds them is the arithmetic
// (a vector instruction takes four cycles of its SIMD), so everything there is in f16, which
// has 8-bit numbers for two instructions a pair: a byte pair spread by a permute is a pair of
// subnormals u 2^-24, and one packed fma gives (u - 128) 2^-9, exactly. Scores and weights
// take the scales outside the products:
//   q      times the power of two that brings its row's largest magnitude to 2^14: one part
//          for bf16 (exact to 2^-39 of the largest), two for f32 (2^-22);
//   p s_v  are held between 2^-24 and 2^15 by a power of two of the row's: p = exp2(s - ref), ref a
//          score that need not be the largest, and the products take p up s_v. Where a tile's largest of
//          them passes 2^15 or its sum of p 2^10, ref becomes the largest score and `up` what
//          brings the largest product to 2^10. No maximum is taken otherwise, of lanes or
//          tiles. (One reference for both loses the sum where s_v are far apart: rows of 0
//          and of 1e26 have products 2^126 from each other and weigh the same.) One f16 part
//          behind bf16 q and output (2^-11 of a weight, the output's rounding
//          is 2^-8 of it; two parts take the batch of 8 from 19.1 to 19.6 us), two else; what is
//          below 2^-24 / 2^10 of the largest weight so far rounds to multiples of that.
// V needs no transposing reads: a lane takes D / 16 dims of its own of each of its keys, one
// read a key, and converts byte n of four keys into the operand of product n; 32 keys at a
// time (16x16x32). What is not seen is masked at the scores and the weights: codes are
// numbers whatever they hold. (The two batches above over 8-bit pages: 19.1 us, 2.6 TB/s, and, with
// f32 queries, 32.6, 3.3; some 8 us of each go by before the first product and after the last.)
namespace {

typedef short s16x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ float max4(float v) {  // over the four lanes of a column
  uint2 p = pair_xor16(v);
  v = fmaxf(__uint_as_float(p.x), __uint_as_float(p.y));
  p = pair_xor32(v);
  return fmaxf(__uint_as_float(p.x), __uint_as_float(p.y));
}
__device__ __forceinline__ float sum4(float v) { return sum_xor32(sum_xor16(v)); }

// Invariant device memory at a wave-uniform address (scalar loads)
__device__ __forceinline__ int uniform_load(const int32_t *p, int64_t i) {
  return ((const __attribute__((address_space(4))) int32_t *)(uintptr_t)p)[i];
}

template <int N>
__device__ __forceinline__ void wait_vm() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
__device__ __forceinline__ void wait_lds() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

// n things dealt to m takers in order: taker i starts at start(i)
struct Deal {
  int base, rem;
  __device__ Deal(int n, int m) : base(n / m), rem(n % m) {}
  __device__ int start(int i) const { return i * base + min(i, rem); }
  __device__ int taker(int x) const {  // (x < n)
    const int big = rem * (base + 1);
    return x < big ? x / (base + 1) : rem + (x - big) / base;
  }
};

constexpr int kPagedWaves = 8;

enum { kBf16, kF32, kCodes };  // what pages hold
// What q and the output are, for the parts that bf16 products take: as the arguments say;
// both bf16; or anything, in the three parts of f32 (beside f32 pages all are one)
enum { kAny, kLow, kHigh };

template <int D, int KIND>
constexpr int paged_keys() {
  return KIND == kCodes ? (D == 64 ? 64 : 32) : D * (KIND == kF32 ? 4 : 2) < 256 ? 32 : 16;
}
template <int D, int KIND, int KEYS = paged_keys<D, KIND>()>
struct PagedTile {
  static constexpr bool F32 = KIND == kF32, CODES = KIND == kCodes;
  static constexpr int ES = F32 ? 4 : CODES ? 1 : 2, ROW = D * ES, CH = ROW / 16;
  static constexpr int KT = KEYS;                // keys of a tile
  static constexpr int SUB = KT / 16, HALF = KT * ROW, N = HALF / 1024, RPI = 1024 / ROW;
  static constexpr int NS = CODES ? KT / 32 : 0;  // copies of 64 scales: the tile's K's, its V's
  static constexpr int NK = N + NS;               // copies that K's products wait for
  static constexpr int RING = 2 * HALF + 256 * NS;  // a wave's K and V, scales behind them
  static constexpr int REC = D + 4;               // floats of a record: acc [D], max, sum
  static __device__ __forceinline__ int kx(int row) { return row & (CH < 16 ? CH - 1 : 15); }
  static __device__ __forceinline__ int vx(int row) { return KIND != kBf16 ? 0 : 2 * (row & (CH < 16 ? 3 : 7)); }
};

// (max, sum, acc) records joined in order: NB of them, number k0 + k with
// get(k, min(k0 + k, count - 1), m, l, o); those from `count` on do not count. o is two
// of a head's dims. Over codes acc is divided by its sum already (NORMAL): acc by itself has a
// power of two beside it that would have to be joined too.
struct Joined {
  float M = kMinusInf, L = 0.f;
  float2 O = float2{0.f, 0.f};
};
__device__ __forceinline__ float record_weight(float m, float l, float M) {
  return m == kMinusInf ? (l == 0.f ? 0.f : 1.f) : __builtin_amdgcn_exp2f(m - M);  // (l NaN: scores were)
}
template <int NB, bool NORMAL, typename Get>
__device__ __forceinline__ void join(Joined &j, int k0, int count, Get get) {
  float m[NB], l[NB], M = j.M;
  float2 o[NB];
#pragma unroll
  for (int k = 0; k < NB; ++k) get(k, min(k0 + k, count - 1), m[k], l[k], o[k]);
#pragma unroll
  for (int k = 0; k < NB; ++k) {
    if (k0 + k >= count) m[k] = kMinusInf, l[k] = 0.f, o[k] = float2{0.f, 0.f};
    M = fmaxf(M, m[k]);
  }
  const float f0 = record_weight(j.M, j.L, M);
  if constexpr (NORMAL) {
    j.M = M, j.L *= f0;
    float L = j.L;
#pragma unroll
    for (int k = 0; k < NB; ++k) l[k] *= record_weight(m[k], l[k], M), L += l[k];
    const float inv = L == 0.f ? 0.f : 1.0f / L;
    j.O.x *= j.L * inv, j.O.y *= j.L * inv;
#pragma unroll
    for (int k = 0; k < NB; ++k) {
      j.O.x += l[k] * inv * o[k].x;
      j.O.y += l[k] * inv * o[k].y;
    }
    j.L = L;
    return;
  }
  j.M = M, j.L *= f0, j.O.x *= f0, j.O.y *= f0;
#pragma unroll
  for (int k = 0; k < NB; ++k) {
    const float f = record_weight(m[k], l[k], M);
    j.L += f * l[k];
    j.O.x += f * o[k].x;
    j.O.y += f * o[k].y;
  }
}
// Two floats of a record, written through to where every workgroup sees them
__device__ __forceinline__ void store_pair(float *p, float x, float y) {
  const unsigned long long v = (unsigned long long)__float_as_uint(y) << 32 | __float_as_uint(x);
  __hip_atomic_store((unsigned long long *)p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
// A wave-uniform address, in scalar registers
__device__ __forceinline__ const void *uniform(const void *p) {
  const uint64_t x = (uint64_t)(uintptr_t)p;
  return (const void *)(uintptr_t)((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(x >> 32)) << 32 |
                                   (uint32_t)__builtin_amdgcn_readfirstlane((int)x));
}
// dma16 (common.h) of what others wrote so: past this die's caches
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void dma16_coherent(const void *base, uint32_t voff, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %1\n\tglobal_load_lds_dwordx4 %0, %2 sc1"
               :: "v"(voff), "s"(lds), "s"(base) : "memory", "m0");
}
#pragma clang diagnostic pop

// Inclusive sum over the 64 lanes
__device__ __forceinline__ int scan64(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);  // row_shr:1
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);  // row_bcast:15
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);  // row_bcast:31
  return v;
}

// f(0), f(1), .., f(N - 1) with constants for arguments
template <int N, int I = 0, typename F>
__device__ __forceinline__ void unrolled(F f) {
  if constexpr (I < N) {
    f(std::integral_constant<int, I>{});
    unrolled<N, I + 1>(f);
  }
}
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
// Codes as f16 pairs of (u - 128) 2^-9: byte i of x and byte j of y
template <int I, int J>
__device__ __forceinline__ uint32_t codes_f16(uint32_t x, uint32_t y) {
  const f16x2 u = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(y, x, 0x0c000c00u | (4 + J) << 16 | I));
  const f16x2 up = {(_Float16)32768.f, (_Float16)32768.f}, less = {(_Float16)-0.25f, (_Float16)-0.25f};
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(u, up, less));
}
constexpr float kCodeUnit = 0x1p9f;
// The largest power that p (up to 2^10) is taken times ahead of s_v: finite in f32, and enough for every
// scale from 2^-106 on (the append's begin at 2^-47)
constexpr float kMostUp = 116.f;
// Two f32 as an f16 pair, round to nearest even, and what that leaves
__device__ __forceinline__ uint32_t pack_f16x2(float a, float b) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2_t){a, b}, f16x2));
}
__device__ __forceinline__ uint32_t rest_f16x2(float a, float b, uint32_t part) {
  const f16x2 h = __builtin_bit_cast(f16x2, part);
  return pack_f16x2(a - (float)h[0], b - (float)h[1]);
}
__device__ __forceinline__ f32x4 mfma_f16(u32x4 a, u32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

struct Piece {  // of a sequence, that one wave or workgroup went over
  int b, first, n;  // sequence; its first tile in the head's run; its tiles
};

// dma16's 4-byte form, an address a lane: lane l copies to LDS bytes [lds + 4 l, +4)
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void dma4(const void *from, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %1\n\tglobal_load_lds_dword %0, off" :: "v"(from), "s"(lds) : "memory", "m0");
}
#pragma clang diagnostic pop

}  // namespace

// (the functions below hold the wave's registers: they have to be part of the kernel)
#define RXW8_INLINE __attribute__((always_inline))

// What a wave holds for CT x 16 query rows (columns of the products) of one kv head: q, O
// and the softmax, and the steps over a tile in its memory `mem` (K, V, scales).
template <int D, int KIND, int CT, int PREC, int KEYS = paged_keys<D, KIND>()>
struct PagedWave {
  using T = PagedTile<D, KIND, KEYS>;
  static constexpr bool F32 = T::F32, CODES = T::CODES;
  static constexpr int NQ = F32 ? D / 16 : D / 32;  // 16-byte pieces of a row's q per lane
  // (not where two tries at the weights and q's three parts want more registers than there are:
  // 41 sequences of 87 keys behind 7, 64 / 8 heads of 256, f32 queries: 71 us with it, 50 without)
  static constexpr bool LAZY = KIND == kBf16 && PREC != kAny && !(D == 256 && PREC == kHigh);
  // an f32 q's further parts: two over bf16 rows, one over codes
  static constexpr int NL = F32 || PREC == kLow ? 1 : NQ, NE = CODES ? 1 : NL;
  typedef const __attribute__((address_space(3))) char *Lds;

  struct Tile {
    int t, seen, holes;             // its number, keys in it; bit s: its 16-key piece s has no page
  };

  const PagedDecodeArgs &a;
  const int lane, col, g4, h;
  // the walk over a page table: its entries and positions, the next tile, the entry and the
  // 16-key piece within its page that it begins at, its pieces' pages (on their way while
  // the tile before is worked on); of the tile last begun, bytes from the pool's start
  const int32_t *table;
  int entries, len, t, e, r, page[T::SUB];
  int64_t off[T::SUB];
  const uint32_t mem;               // LDS address of the wave's K, V and scales
  u32x4 q[CT][NQ], ql[CT][NL], qe[CT][NE];
  f32x4 o[CT][D / 16], s[CT][T::SUB];
  f32x4 vs[CODES ? T::SUB : 1];     // V's scales
  float m[CT], l[CT];               // (codes: m is the reference)
  float up[CODES ? CT : 1];         // codes: what weights are multiplied by in the products, a power of two
  float unit[CODES ? CT : 1];       // codes: what a product of q and codes counts in a score, but for s_k

  __device__ RXW8_INLINE PagedWave(const PagedDecodeArgs &a, int h, char *mem)
      : a(a), lane(threadIdx.x & 63), col(lane & 15), g4(lane >> 4), h(h), mem(lds_addr(mem)) {}

  // Walks on at tile t0 of the `n` positions that `pages` [m] has the pages of
  __device__ RXW8_INLINE void begin(const int32_t *pages, int m, int n, int t0) {
    const unsigned sub = (unsigned)(t0 * T::SUB), ps16 = (unsigned)a.ps >> 4;
    table = pages, entries = m, len = n, t = t0;
    e = (int)(sub / ps16), r = (int)(sub - e * ps16);
    look();
  }
  __device__ RXW8_INLINE void look() {
    int e1 = e, r1 = r;
#pragma unroll
    for (int u = 0; u < T::SUB; ++u) {
      page[u] = uniform_load(table, min(e1, entries - 1));
      if (++r1 == a.ps >> 4) r1 = 0, ++e1;
    }
  }
  // The next tile
  __device__ RXW8_INLINE Tile tile() {
    Tile x;
    x.t = t, x.holes = 0;
    x.seen = min(len - t * T::KT, T::KT);
#pragma unroll
    for (int u = 0; u < T::SUB; ++u) {
      if (16 * u >= x.seen) {
        off[u] = off[0];
        continue;
      }
      int id = page[u];
      if (id < 0 || id >= a.P) id = 0, x.holes |= 1 << u;
      off[u] = (((int64_t)id * a.Hkv + h) * a.ps + 16 * r) * T::ROW;
      if (++r == a.ps >> 4) r = 0, ++e;
    }
    ++t;
    look();
    return x;
  }
  __device__ RXW8_INLINE void copy(const void *pool, int half) const {
    const uint32_t dst = mem + half * T::HALF;
    const int lrow = lane / T::CH, lch = lane % T::CH;
#pragma unroll
    for (int i = 0; i < T::N; ++i) {
      const int row = i * T::RPI + lrow, sx = half ? T::vx(row) : T::kx(row);
      int from = row & 15;
      // (V's codes: keys j, 4 + j, 8 + j, 12 + j beside one another, which a read takes)
      if (CODES && half) from = 4 * (from & 3) + (from >> 2);
      dma16((const char *)pool + off[i * T::RPI / 16], (uint32_t)from * T::ROW + ((lch ^ sx) << 4), dst + 1024 * i);
    }
  }
  // The copies of the tile last begun
  __device__ RXW8_INLINE void copy_k() const {
    copy(a.kp, 0);
    if constexpr (CODES) {
#pragma unroll
      for (int i = 0; i < T::NS; ++i) {
        const int at = 64 * i + lane, key = at & (T::KT - 1);  // K's KT scales, then V's
        int64_t from = off[0];
#pragma unroll
        for (int u = 1; u < T::SUB; ++u) from = key >> 4 == u ? off[u] : from;
        dma4((const char *)(at < T::KT ? a.ks : a.vs) + from / T::ROW * 4 + 4 * (key & 15), mem + 2 * T::HALF + 256 * i);
      }
    }
  }
  __device__ RXW8_INLINE void copy_v() const { copy(a.vp, 1); }

  __device__ RXW8_INLINE bool q_parts() const { return PREC == kAny ? a.q_f32 : PREC == kHigh; }
  __device__ RXW8_INLINE bool p_parts() const { return PREC == kAny ? a.out_f32 : PREC == kHigh; }
  __device__ RXW8_INLINE void load_q_f16(int c, int64_t qo) {
    float x[NQ][8];
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < NQ; ++i) {
      const int64_t at = qo + 64 * (i >> 1) + 16 * g4 + 8 * (i & 1);
      if (PREC != kLow && a.q_f32) {
        const f32x4 r[2] = {*(const f32x4 *)((const float *)a.q + at), *(const f32x4 *)((const float *)a.q + at + 4)};
#pragma unroll
        for (int k = 0; k < 8; ++k) x[i][k] = r[k >> 2][k & 3];
      } else {
        const u32x4 r = *(const u32x4 *)((const uint16_t *)a.q + at);
#pragma unroll
        for (int k = 0; k < 8; ++k) x[i][k] = __uint_as_float(k & 1 ? r[k >> 1] & 0xffff0000u : r[k >> 1] << 16);
      }
    }
#pragma unroll
    for (int i = 0; i < NQ; ++i)
#pragma unroll
      for (int k = 0; k < 8; ++k) top = max(top, __float_as_uint(x[i][k]) & 0x7fffffffu);
    uint2 two = pair_xor16(__uint_as_float(top));
    two = pair_xor32(__uint_as_float(max(two.x, two.y)));
    // 2^14 / 2^e, e the exponent of the largest (2^126 at most: its inverse is no subnormal)
    const int scale = min(127 + 14 + 127 - (int)(max(two.x, two.y) >> 23), 253);
    const float up = __uint_as_float((uint32_t)scale << 23);
    unit[c] = a.c * (kCodeUnit * __uint_as_float((uint32_t)(254 - scale) << 23));  // (a.c may be near f32's end)
#pragma unroll
    for (int i = 0; i < NQ; ++i)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float y = x[i][2 * k] * up, z = x[i][2 * k + 1] * up;
        q[c][i][k] = pack_f16x2(y, z);
        if constexpr (PREC != kLow) ql[c][NL > 1 ? i : 0][k] = rest_f16x2(y, z, q[c][i][k]);
      }
  }
  // q of the lane's row of column tile c, at element qo
  __device__ RXW8_INLINE void load_q(int c, int64_t qo) {
    if constexpr (CODES) load_q_f16(c, qo);
#pragma unroll
    for (int i = 0; i < NQ; ++i) {
      if constexpr (CODES) break;
      if constexpr (F32) {
        const int64_t at4 = qo + 16 * i + 4 * g4;
        if (a.q_f32) {
          q[c][i] = *(const u32x4 *)((const float *)a.q + at4);
        } else {
          const uint2 r = *(const uint2 *)((const uint16_t *)a.q + at4);
          q[c][i] = u32x4{r.x << 16, r.x & 0xffff0000u, r.y << 16, r.y & 0xffff0000u};
        }
      } else {
        if (PREC == kHigh && D == 256 && i == NQ / 2) __builtin_amdgcn_sched_barrier(0);  // (registers for half of q at a time)
        const int64_t at8 = qo + 32 * i + 8 * g4;
        if (PREC != kLow && a.q_f32) {
          const f32x4 r[2] = {*(const f32x4 *)((const float *)a.q + at8), *(const f32x4 *)((const float *)a.q + at8 + 4)};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            uint32_t x[3];
            split_bf16x2(r[e >> 1][2 * (e & 1)], r[e >> 1][2 * (e & 1) + 1], x);
            q[c][i][e] = x[0], ql[c][NL > 1 ? i : 0][e] = x[1], qe[c][NE > 1 ? i : 0][e] = x[2];
          }
        } else {
          q[c][i] = *(const u32x4 *)((const uint16_t *)a.q + at8);
          if constexpr (PREC == kHigh) ql[c][NL > 1 ? i : 0] = qe[c][NE > 1 ? i : 0] = u32x4{0, 0, 0, 0};
        }
      }
    }
    m[c] = kMinusInf;
    l[c] = 0.f;
    if constexpr (CODES) up[c] = 1.f;
#pragma unroll
    for (int i = 0; i < D / 16; ++i) o[c][i] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  // Waits here for q: a wait for it later would be a wait for the copies ahead
  __device__ RXW8_INLINE void wait_q() {
#pragma unroll
    for (int c = 0; c < CT; ++c)
#pragma unroll
      for (int n = 0; n < NQ; ++n) asm volatile("" : "+v"(q[c][n]));
  }

  // S^T = K q^T of the tile whose K is there, for the first `ct` column tiles
  __device__ RXW8_INLINE void scores(int ct) {
    const uint32_t kf = mem + col * T::ROW;
    constexpr int NA = F32 ? 4 : CT > 1 ? 1 : 2;  // sums in turn: no product waits for the one before
#pragma unroll
    for (int u = 0; u < T::SUB; ++u) {
      f32x4 acc[CT][NA];
#pragma unroll
      for (int c = 0; c < CT; ++c)
#pragma unroll
        for (int n = 0; n < NA; ++n) acc[c][n] = f32x4{0.f, 0.f, 0.f, 0.f};
      auto add = [&](int n, u32x4 f) RXW8_INLINE {
#pragma unroll
        for (int c = 0; c < CT; ++c) {
          if (c && c >= ct) break;
          if constexpr (CODES) {
            acc[c][n & (NA - 1)] = mfma_f16(f, q[c][n], acc[c][n & (NA - 1)]);
            if constexpr (PREC != kLow) acc[c][~n & (NA - 1)] = mfma_f16(f, ql[c][NL > 1 ? n : 0], acc[c][~n & (NA - 1)]);
            continue;
          }
          acc[c][n & (NA - 1)] = mfma16x16x32(as_bf16x8(f), as_bf16x8(q[c][n]), acc[c][n & (NA - 1)]);
          if (q_parts()) {
            acc[c][~n & (NA - 1)] = mfma16x16x32(as_bf16x8(f), as_bf16x8(ql[c][NL > 1 ? n : 0]), acc[c][~n & (NA - 1)]);
            acc[c][n & (NA - 1)] = mfma16x16x32(as_bf16x8(f), as_bf16x8(qe[c][NE > 1 ? n : 0]), acc[c][n & (NA - 1)]);
          }
        }
      };
#pragma unroll
      for (int n = 0; n < (CODES ? NQ / 2 : NQ); ++n) {
        const u32x4 f = *(const __attribute__((address_space(3))) u32x4 *)(uintptr_t)(
            kf + u * 16 * T::ROW + (((4 * n + g4) ^ T::kx(col)) << 4));
        if constexpr (F32) {
#pragma unroll
          for (int c = 0; c < CT; ++c) {
            if (c && c >= ct) break;
#pragma unroll
            for (int e = 0; e < 4; ++e)
              acc[c][e] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(f[e]), __uint_as_float(q[c][n][e]), acc[c][e], 0, 0, 0);
          }
        } else if constexpr (CODES) {
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const uint32_t x = f[2 * k], y = f[2 * k + 1];
            add(2 * n + k, u32x4{codes_f16<0, 1>(x, x), codes_f16<2, 3>(x, x), codes_f16<0, 1>(y, y), codes_f16<2, 3>(y, y)});
          }
        } else {
          add(n, f);
        }
      }
      f32x4 scale = f32x4{a.c, a.c, a.c, a.c};
      if constexpr (CODES) {
        const uint32_t at = mem + 2 * T::HALF + 4 * (16 * u + 4 * g4);
        scale = *(const __attribute__((address_space(3))) f32x4 *)(uintptr_t)at;
        vs[u] = *(const __attribute__((address_space(3))) f32x4 *)(uintptr_t)(at + 4 * T::KT);
      }
#pragma unroll
      for (int c = 0; c < CT; ++c) {
        s[c][u] = acc[c][0];
        if constexpr (NA > 1) s[c][u] += acc[c][1];
        if constexpr (F32) s[c][u] += acc[c][2] + acc[c][3];
        s[c][u] *= CODES ? scale * unit[CODES ? c : 0] : scale;
      }
    }
  }

  // Scores into weights; O is rescaled only where a running maximum moves
  __device__ RXW8_INLINE void softmax(const Tile &x, bool part, int ct) {
#pragma unroll
    for (int c = 0; c < CT; ++c) {
      if (c && c >= ct) break;
      if constexpr (CODES) {
        softmax_codes(c, x, part);
        continue;
      }
      if constexpr (LAZY) {
        softmax_lazy(c, x, part);
        continue;
      }
      float mt = kMinusInf;
#pragma unroll
      for (int u = 0; u < T::SUB; ++u)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          if (part && (16 * u + 4 * g4 + r >= x.seen || (x.holes >> u & 1))) s[c][u][r] = kMinusInf;
          mt = fmaxf(mt, s[c][u][r]);
        }
      mt = max4(mt);
      if (__ballot(mt > m[c])) {
        const float mn = fmaxf(m[c], mt), ref = mn == kMinusInf ? 0.f : mn, f = exp2f(m[c] - ref);
        m[c] = mn;
        l[c] *= f;
#pragma unroll
        for (int n = 0; n < D / 16; ++n) o[c][n] *= f;
      }
      const float ref = m[c] == kMinusInf ? 0.f : m[c];
#pragma unroll
      for (int u = 0; u < T::SUB; ++u)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float p = __builtin_amdgcn_exp2f(s[c][u][r] - ref);
          l[c] += p;
          s[c][u][r] = p;
        }
    }
  }

  // The reference up to 8 above the largest score, so that weights are at most 1 (as large values need: acc
  // is theirs times the weights) and it need not move with every new maximum
  __device__ RXW8_INLINE void softmax_lazy(int c, const Tile &x, bool part) {
    f32x4 w[T::SUB];
    float sum, top;
    if (part) {
#pragma unroll
      for (int u = 0; u < T::SUB; ++u)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (16 * u + 4 * g4 + r >= x.seen || (x.holes >> u & 1)) s[c][u][r] = kMinusInf;
    }
    auto weigh = [&]() RXW8_INLINE {
      const float ref = m[c] == kMinusInf ? 0.f : m[c];
      sum = top = 0.f;
#pragma unroll
      for (int u = 0; u < T::SUB; ++u)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          w[u][r] = __builtin_amdgcn_exp2f(s[c][u][r] - ref);
          sum += w[u][r];
          top = fmaxf(top, w[u][r]);
        }
    };
    weigh();
    if (__ballot(top > 1.f || m[c] == kMinusInf)) {
      float highest = kMinusInf;
#pragma unroll
      for (int u = 0; u < T::SUB; ++u)
#pragma unroll
        for (int r = 0; r < 4; ++r) highest = fmaxf(highest, s[c][u][r]);
      const float to = fmaxf(m[c], max4(highest) + 8.f);
      const float f = to == kMinusInf ? 1.f : exp2f(m[c] - to);
      m[c] = to;
      l[c] *= f;
#pragma unroll
      for (int n = 0; n < D / 16; ++n) o[c][n] *= f;
      weigh();
    }
    l[c] += sum;
#pragma unroll
    for (int u = 0; u < T::SUB; ++u) s[c][u] = w[u];
  }

  // The power of up[c]
  __device__ RXW8_INLINE float up_of(int c) const { return (float)((int)(__float_as_uint(up[CODES ? c : 0]) >> 23) - 127); }
  __device__ RXW8_INLINE void softmax_codes(int c, const Tile &x, bool part) {
    f32x4 w[T::SUB];
    float sum, top;
    if (part) {
#pragma unroll
      for (int u = 0; u < T::SUB; ++u)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (16 * u + 4 * g4 + r >= x.seen || (x.holes >> u & 1)) s[c][u][r] = kMinusInf, vs[u][r] = 0.f;
    }
    auto weigh = [&]() RXW8_INLINE {
      const float ref = m[c] == kMinusInf ? 0.f : m[c];
      sum = top = 0.f;
#pragma unroll
      for (int u = 0; u < T::SUB; ++u)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float p = __builtin_amdgcn_exp2f(s[c][u][r] - ref);
          sum += p;
          w[u][r] = p * up[c] * vs[u][r];
          top = fmaxf(top, fabsf(w[u][r]));
        }
    };
    bool move = __ballot(m[c] == kMinusInf);
    if (CT > 1 || !move) {  // (not before the first reference, where registers allow that)
      weigh();
      move = __ballot(top > 0x1p15f || sum > 0x1p10f || m[c] == kMinusInf);
    }
    if (move) {
      float highest = kMinusInf, largest = kMinusInf;
#pragma unroll
      for (int u = 0; u < T::SUB; ++u)
#pragma unroll
        for (int r = 0; r < 4; ++r) highest = fmaxf(highest, s[c][u][r]);
      const float to = fmaxf(m[c], max4(highest)), ref = to == kMinusInf ? 0.f : to;
#pragma unroll
      for (int u = 0; u < T::SUB; ++u)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          largest = fmaxf(largest, s[c][u][r] - ref + fminf(__builtin_amdgcn_logf(fabsf(vs[u][r])), 128.f));
      // (no product so far grows: m / up does not fall; the first fminf passes over a NaN)
      const float was = up_of(c), moved = to - m[c];
      const float power = fminf(fminf(floorf(was + moved), 10.f - floorf(max4(largest))), kMostUp);
      const float f = to == kMinusInf ? 1.f : exp2f(-moved), g = to == kMinusInf ? 1.f : exp2f(power - was - moved);
      m[c] = to;
      up[c] = __uint_as_float((uint32_t)((int)power + 127) << 23);
      l[c] *= f;
#pragma unroll
      for (int n = 0; n < D / 16; ++n) o[c][n] *= g;
      weigh();
    }
    l[c] += sum;
#pragma unroll
    for (int u = 0; u < T::SUB; ++u) s[c][u] = w[u];
  }

  // V rows that are not seen, cleared
  __device__ RXW8_INLINE void clear_v(const Tile &x) const {
    const int lrow = lane / T::CH;
#pragma unroll
    for (int n = 0; n < T::N; ++n) {
      const int row = n * T::RPI + lrow;
      if (row >= x.seen || (x.holes >> (row >> 4) & 1))
        *(__attribute__((address_space(3))) u32x4 *)(uintptr_t)(mem + T::HALF + 1024 * n + 16 * lane) = u32x4{0, 0, 0, 0};
    }
    wait_lds();
  }

  // O^T += V^T P^T of the tile whose V is there
  __device__ RXW8_INLINE void values(int ct) {
    const uint32_t v0 = mem + T::HALF;
    if constexpr (F32) {
      const uint32_t vf = v0 + 4 * g4 * T::ROW + 16 * col;
#pragma unroll
      for (int u = 0; u < T::SUB; ++u)
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int n = 0; n < D / 64; ++n) {
            const u32x4 f = *(const __attribute__((address_space(3))) u32x4 *)(uintptr_t)(vf + u * 16 * T::ROW + r * T::ROW + 256 * n);
#pragma unroll
            for (int c = 0; c < CT; ++c) {
              if (c && c >= ct) break;
#pragma unroll
              for (int e = 0; e < 4; ++e)
                o[c][4 * n + e] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(f[e]), s[c][u][r], o[c][4 * n + e], 0, 0, 0);
            }
          }
      return;
    }
    if constexpr (CODES) {
      values_codes(ct, v0);
      return;
    }
    // weights in parts: three behind an f32 output, two behind a bf16 one
    struct Parts {
      uint2 k0, k1, k2;
    };
    auto parts = [&](f32x4 w) RXW8_INLINE {
      if (p_parts()) {
        uint32_t x[3], y[3];
        split_bf16x2<true>(w[0], w[1], x);
        split_bf16x2<true>(w[2], w[3], y);
        return Parts{uint2{x[0], y[0]}, uint2{x[1], y[1]}, uint2{x[2], y[2]}};
      }
      uint32_t x[2], y[2];
      split_bf16x2<true>(w[0], w[1], x);
      split_bf16x2<true>(w[2], w[3], y);
      return Parts{uint2{x[0], y[0]}, uint2{x[1], y[1]}, uint2{0, 0}};
    };
    const int tr_j = col >> 2, tr_q = col & 3;
    const uint32_t vf = v0 + (4 * g4 + tr_j) * T::ROW + 8 * (tr_q & 1);
    auto read = [&](int u, int n) RXW8_INLINE {
      return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4 *)(uintptr_t)(
          vf + u * 16 * T::ROW + (((2 * n + (tr_q >> 1)) ^ T::vx(4 * g4 + tr_j)) << 4)));
    };
    if constexpr (PREC != kAny && T::SUB % 2 == 0) {  // 32 keys at a time
#pragma unroll
      for (int u = 0; u < T::SUB; u += 2) {
        Parts p[CT][2];
#pragma unroll
        for (int c = 0; c < CT; ++c) {
          if (c && c >= ct) break;
          p[c][0] = parts(s[c][u]);
          p[c][1] = parts(s[c][u + 1]);
        }
#pragma unroll
        for (int n = 0; n < D / 16; ++n) {
          const uint2 lo = __builtin_bit_cast(uint2, read(u, n)), hi = __builtin_bit_cast(uint2, read(u + 1, n));
          const u32x4 f = {lo.x, lo.y, hi.x, hi.y};
#pragma unroll
          for (int c = 0; c < CT; ++c) {
            if (c && c >= ct) break;
            auto add = [&](uint2 x, uint2 y) RXW8_INLINE { o[c][n] = mfma16x16x32(as_bf16x8(f), as_bf16x8(u32x4{x.x, x.y, y.x, y.y}), o[c][n]); };
            add(p[c][0].k0, p[c][1].k0);
            add(p[c][0].k1, p[c][1].k1);
            if (p_parts()) add(p[c][0].k2, p[c][1].k2);
          }
        }
      }
      return;
    }
#pragma unroll
    for (int u = 0; u < T::SUB; ++u) {
      Parts p[CT];
#pragma unroll
      for (int c = 0; c < CT; ++c) {
        if (c && c >= ct) break;
        p[c] = parts(s[c][u]);
      }
#pragma unroll
      for (int n = 0; n < D / 16; ++n) {
        const s16x4 f = read(u, n);
#pragma unroll
        for (int c = 0; c < CT; ++c) {
          if (c && c >= ct) break;
          auto add = [&](uint2 x) RXW8_INLINE {
            o[c][n] = __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(f, __builtin_bit_cast(s16x4, x), o[c][n], 0, 0, 0);
          };
          add(p[c].k0);
          add(p[c].k1);
          if (p_parts()) add(p[c].k2);
        }
      }
    }
  }

  __device__ RXW8_INLINE void values_codes(int ct, uint32_t v0) {
    constexpr int W = D / 64;  // dwords of a lane's dims of a key
#pragma unroll
    for (int u = 0; u < T::SUB; u += 2) {
      uint32_t w[2][4][W];
#pragma unroll
      for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t at = v0 + ((u + k) * 16 + 4 * j + g4) * T::ROW + 4 * W * col;
          if constexpr (W == 1) {
            w[k][j][0] = *(const __attribute__((address_space(3))) uint32_t *)(uintptr_t)at;
          } else if constexpr (W == 2) {
            typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
            const u32x2 x = *(const __attribute__((address_space(3))) u32x2 *)(uintptr_t)at;
            w[k][j][0] = x[0], w[k][j][1] = x[1];
          } else {
            const u32x4 x = *(const __attribute__((address_space(3))) u32x4 *)(uintptr_t)at;
#pragma unroll
            for (int i = 0; i < 4; ++i) w[k][j][i] = x[i];
          }
        }
      u32x4 p[CT], rest[PREC == kLow ? 1 : CT];
#pragma unroll
      for (int c = 0; c < CT; ++c) {
        if (c && c >= ct) break;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float x = s[c][u + (i >> 1)][2 * (i & 1)], y = s[c][u + (i >> 1)][2 * (i & 1) + 1];
          p[c][i] = pack_f16x2(x, y);
          if constexpr (PREC != kLow) rest[c][i] = rest_f16x2(x, y, p[c][i]);
        }
      }
      auto dim = [&](auto n) RXW8_INLINE {  // byte n % 4 of dword n / 4 of eight keys
        constexpr int N = decltype(n)::value, I = N & 3, i = N >> 2;
        const u32x4 f = {codes_f16<I, I>(w[0][0][i], w[0][1][i]), codes_f16<I, I>(w[0][2][i], w[0][3][i]),
                         codes_f16<I, I>(w[1][0][i], w[1][1][i]), codes_f16<I, I>(w[1][2][i], w[1][3][i])};
#pragma unroll
        for (int c = 0; c < CT; ++c) {
          if (c && c >= ct) break;
          o[c][N] = mfma_f16(f, p[c], o[c][N]);
          if constexpr (PREC != kLow) o[c][N] = mfma_f16(f, rest[PREC == kLow ? 0 : c], o[c][N]);
        }
      };
      unrolled<D / 16>(dim);
    }
  }

  // Four of the lane's row of O and the first of their dims: i < D / 16.
  // (o[i][r] is of dim 16 i + 4 g4 + r (bf16), 64 (i / 4) + 16 g4 + 4 r + i % 4 (f32),
  // D / 16 (4 g4 + r) + i (codes))
  __device__ RXW8_INLINE f32x4 quad(int c, int i) const {
    if (KIND == kBf16) return o[c][i];
    f32x4 y;
#pragma unroll
    for (int r = 0; r < 4; ++r) y[r] = o[c][(i & ~3) + r][i & 3];
    return y;
  }
  __device__ RXW8_INLINE int quad_dim(int i) const {
    return KIND == kBf16 ? 16 * i + 4 * g4 : F32 ? 64 * (i >> 2) + 16 * g4 + 4 * (i & 3) : D / 16 * (4 * g4 + (i & 3)) + 4 * (i >> 2);
  }
  // What quads are to be multiplied by for an output (sum: of all lanes)
  __device__ RXW8_INLINE float inverse(int c, float sum) const {
    if (sum == 0.f) return 0.f;
    const float inv = 1.0f / sum;
    if constexpr (CODES) return inv * (kCodeUnit * __uint_as_float((254u << 23) - __float_as_uint(up[c])));
    return inv;
  }
  // The lane's row of column tile c as a record
  __device__ RXW8_INLINE void record(int c, float *rec) const {
    const float sum = sum4(l[c]);
#pragma unroll
    for (int i = 0; i < D / 16; ++i) *(f32x4 *)(rec + quad_dim(i)) = CODES ? quad(c, i) * inverse(c, sum) : quad(c, i);
    if (g4 == 0) rec[D] = m[c], rec[D + 1] = sum;
  }
};

// Workgroup `unit` of `units` for head `hk` (a kv head and 16 of its query heads).
// RECORDS: instead of output rows, records (row b Hq + hq: acc, max, sum) into `rows`,
// of the sequences that have keys.
struct PagedPlaceOf {
  int hk, unit, units;
  float *rows;
};
__device__ __forceinline__ PagedPlaceOf paged_place_of(const PagedDecodeArgs &a) {
  const int heads = a.Hkv * ((a.Hq / a.Hkv + 15) / 16);
  return PagedPlaceOf{(int)(blockIdx.x % heads), (int)(blockIdx.x / heads), a.units, nullptr};
}

template <int D, int KIND, bool RECORDS = false, int PREC = kAny>
__device__ RXW8_INLINE void paged_decode(const PagedDecodeArgs &a, PagedPlaceOf place) {
  using T = PagedTile<D, KIND>;
  using Wave = PagedWave<D, KIND, 1, PREC>;
  constexpr bool NORMAL = KIND == kCodes;  // (as join)
  extern __shared__ __attribute__((aligned(16))) char lds[];
  __shared__ Piece piece[kPagedWaves][2];
  __shared__ int last_one[2];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int nw = a.waves, col = lane & 15;
  const int G = a.Hq / a.Hkv, HT = (G + 15) / 16, heads = a.Hkv * HT, gcap = min(G, 16);
  const int hk = place.hk, unit = place.unit, h = hk / HT, ht = hk - h * HT;
  const int gt = min(16, G - 16 * ht), hq0 = h * G + 16 * ht;
  const int most = a.M * a.ps;
  // (unsigned: a length may be near 2^31)
  auto tiles_of = [&](int len) { return (int)(((unsigned)min(max(len, 0), most) + T::KT - 1) / T::KT); };

  // the head's run: total tiles, and (up to 64 sequences) where each begins
  int total = 0, incl = 0, mine = 0;
  auto scan = [&](int b0) {  // of 64 sequences: lane's tiles and their inclusive sum
    mine = b0 + lane < a.B ? tiles_of(a.lens[b0 + lane]) : 0;
    incl = scan64(mine);
    return __builtin_amdgcn_readlane(incl, 63);
  };
  for (int b0 = 0; b0 < a.B; b0 += 64) total += scan(b0);
  const int units = min(place.units, (total + nw - 1) / nw);
  const Deal deal(total, max(units, 1));
  const int u0 = unit < units ? deal.start(unit) : 0, u1 = unit < units ? deal.start(unit + 1) : 0;
  const Deal waves(u1 - u0, nw);
  int at = u0 + waves.start(wave), left = u0 + waves.start(wave + 1) - at;  // (wave < nw)
  piece[wave][0].b = piece[wave][1].b = -1;

  // a wave's memory: its tiles, over them its last record when they are done, and its
  // first record behind both
  const int rec_bytes = gcap * T::REC * 4, first_at = max(T::RING, rec_bytes);
  char *const mem = lds + wave * (first_at + rec_bytes);
  float *const first_rec = (float *)(mem + first_at), *const last_rec = (float *)mem;
  if (wave < nw && left > 0) {
    // ---- the sequence of the wave's first tile
    int b, t;
    {
      int run = 0, b0 = 0;
      if (a.B > 64)
        for (int n; run + (n = scan(b0)) <= at; b0 += 64) run += n;
      const int k = __popcll(__ballot(run + incl <= at));  // (sequences without tiles are passed over)
      b = b0 + k;
      t = at - (run + __builtin_amdgcn_readlane(incl, k) - __builtin_amdgcn_readlane(mine, k));
    }
    b = __builtin_amdgcn_readfirstlane(b);
    t = __builtin_amdgcn_readfirstlane(t);
    left = __builtin_amdgcn_readfirstlane(left);
    at = __builtin_amdgcn_readfirstlane(at);

    // ---- tiles ahead: what the copies need
    struct Ahead {
      int b, t, len, n;
    } ah;
    ah.b = b, ah.t = t;
    ah.len = min(max(uniform_load(a.lens, b), 0), most);
    ah.n = tiles_of(ah.len);
    struct Tile : Wave::Tile {
      int b, n;
    };
    Wave w(a, h, mem);
    w.begin(a.table + (int64_t)b * a.M, a.M, ah.len, t);
    auto next = [&](bool more) {  // the tile that `ah` stands at; `more`: another one follows
      Tile x;
      (typename Wave::Tile &)x = w.tile();
      x.b = ah.b, x.n = ah.n;
      if (more && ++ah.t == ah.n) {
        do {
          ++ah.b;
          ah.len = min(max(uniform_load(a.lens, ah.b), 0), most);
        } while (ah.len == 0);
        ah.n = tiles_of(ah.len);
        ah.t = 0;
        w.begin(a.table + (int64_t)ah.b * a.M, a.M, ah.len, 0);
      }
      return x;
    };

    Tile cur;  // that the copies out are of
    auto start = [&](int seq) { w.load_q(0, ((int64_t)seq * a.Hq + hq0 + min(col, gt - 1)) * D); };
    auto finish = [&](int seq, int first, int n, bool whole, float *rec, Piece *p) {
      if (whole) {
        const int64_t row = (int64_t)seq * a.Hq + hq0 + col;
        const float sum = sum4(w.l[0]);  // (by all lanes)
        if constexpr (RECORDS) {
          if (col < gt) {
            const float inv = w.inverse(0, sum);
            float *const to = place.rows + row * T::REC;
#pragma unroll
            for (int i = 0; i < D / 16; ++i) *(f32x4 *)(to + w.quad_dim(i)) = NORMAL ? w.quad(0, i) * inv : w.quad(0, i);
            if (w.g4 == 0) *(float2 *)(to + D) = float2{w.m[0], sum};
          }
        } else {
          if (col < gt) {
            const float inv = w.inverse(0, sum);
#pragma unroll
            for (int i = 0; i < D / 16; ++i) {
              const f32x4 y = w.quad(0, i) * inv;
              const int64_t d = row * D + w.quad_dim(i);
              if (a.out_f32)
                *(f32x4 *)((float *)a.out + d) = y;
              else
                *(uint2 *)((uint16_t *)a.out + d) = uint2{pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3])};
            }
          }
        }
        return;
      }
      const float sum = sum4(w.l[0]);
      if (col < gt) {
        const float inv = w.inverse(0, sum);
        float *const to = rec + col * T::REC;
#pragma unroll
        for (int i = 0; i < D / 16; ++i) *(f32x4 *)(to + w.quad_dim(i)) = NORMAL ? w.quad(0, i) * inv : w.quad(0, i);
        if (w.g4 == 0) to[D] = w.m[0], to[D + 1] = sum;
      }
      if (lane == 0) *p = Piece{seq, first, n};
    };

    if constexpr (PREC == kAny) {
      // (q is on its way while the first pages are looked up, and in before the copies
      // go out)
      start(b);
      cur = next(left > 1);
      w.wait_q();
      w.copy_k();
      w.copy_v();
    } else {  // (the wait for q is one for the first tile as well: it is needed next)
      cur = next(left > 1);
      w.copy_k();
      w.copy_v();
      start(b);
      w.wait_q();
    }

    int begun = cur.t;  // the tile at which this wave began the sequence
    for (;;) {
      wait_vm<T::N>();  // (copies complete in order: all but this tile's V)
      w.scores(1);
      wait_lds();
      const Tile done = cur;
      if (left > 1) {
        cur = next(left > 2);
        w.copy_k();
      }
      const bool part = done.seen < T::KT || done.holes;
      w.softmax(done, part, 1);
      if (left > 1) wait_vm<T::NK>();
      else wait_vm<0>();
      if (part && KIND != kCodes) w.clear_v(done);
      w.values(1);
      wait_lds();
      if (left > 1) w.copy_v();
      // ---- the sequence's end, or the wave's
      const bool ends = done.t == done.n - 1;
      if (ends || left == 1) {
        const bool whole = ends && begun == 0;
        finish(done.b, at - done.t, done.n, whole, left > 1 ? first_rec : last_rec, &piece[wave][left > 1 ? 0 : 1]);
      }
      ++at;
      if (--left == 0) break;
      if (ends) {
        start(cur.b);
        w.wait_q();
        begun = 0;
      }
    }
  }

  // ---- rows of sequences without keys
  for (int b = unit * kPagedWaves + wave; !RECORDS && b < a.B; b += place.units * kPagedWaves)
    if (tiles_of(uniform_load(a.lens, b)) == 0)
      for (int i = lane; i < gt * D; i += 64) {
        const int64_t to = ((int64_t)b * a.Hq + hq0) * D + i;
        if (a.out_f32) ((float *)a.out)[to] = 0.f;
        else ((uint16_t *)a.out)[to] = 0;
      }
  if (unit >= units) return;

  // ---- the waves' pieces, in order: lane 2 w + k has wave w's k-th
  __syncthreads();
  Piece mine_p;
  mine_p.b = -1, mine_p.first = mine_p.n = 0;
  if (lane < 2 * nw) mine_p = piece[lane >> 1][lane & 1];
  const int64_t rec_size = (gcap * T::REC + 255) & ~255;  // of a record in device memory: whole KiB
  constexpr int DP = D / 2;  // a thread joins two dims of a head
  auto write = [&](int b, int i, const Joined &j) {
    if constexpr (RECORDS) {
      const int r = i / DP, d = 2 * (i - r * DP);
      float *const rec = place.rows + ((int64_t)b * a.Hq + hq0 + r) * T::REC;
      *(float2 *)(rec + d) = j.O;
      if (d == 0) *(float2 *)(rec + D) = float2{j.M, j.L};
      return;
    }
    const int64_t to = ((int64_t)b * a.Hq + hq0) * D + 2 * i;
    const float inv = NORMAL ? 1.f : j.L == 0.f ? 0.f : 1.0f / j.L;
    if (a.out_f32) *(float2 *)((float *)a.out + to) = float2{j.O.x * inv, j.O.y * inv};
    else *(uint32_t *)((uint16_t *)a.out + to) = pack_bf16x2(j.O.x * inv, j.O.y * inv);
  };
  // sequences that other workgroups have keys of: from before, and onwards
  Piece out0, out1;
  out0.b = out1.b = -1;
  for (uint32_t left_p = (uint32_t)__ballot(mine_p.b >= 0); left_p;) {
    const int e = __builtin_ctz(left_p);
    Piece p;
    p.b = __builtin_amdgcn_readlane(mine_p.b, e);
    p.first = __builtin_amdgcn_readlane(mine_p.first, e);
    p.n = __builtin_amdgcn_readlane(mine_p.n, e);
    const uint32_t same = (uint32_t)__ballot(mine_p.b == p.b) & left_p;
    left_p &= ~same;
    const bool onwards = p.first >= u0, whole = onwards && p.first + p.n <= u1;
    if (!whole) (onwards ? out1 : out0) = p;
    float *const to = a.part + (((int64_t)onwards * heads + hk) * place.units + unit) * rec_size;
    for (int i = threadIdx.x; i < gt * DP; i += blockDim.x) {
      const int r = i / DP, d = 2 * (i - r * DP);
      Joined j;
      uint32_t bits = same;
      int x = e;
      auto get = [&](int, int, float &m, float &l, float2 &o) {
        if (bits) x = __builtin_ctz(bits), bits &= bits - 1;
        const float *const rec = (const float *)(lds + (x >> 1) * (first_at + rec_bytes) + ((x & 1) ? 0 : first_at)) + r * T::REC;
        const float2 ml = *(const float2 *)(rec + D);
        m = ml.x, l = ml.y, o = *(const float2 *)(rec + d);
      };
      const int n = __builtin_popcount(same);
#pragma unroll 1
      for (int k0 = 0; k0 < n; k0 += 4) join<4, NORMAL>(j, k0, n, get);
      if (whole) {
        write(p.b, i, j);
      } else {
        float *const tr = to + r * T::REC;
        store_pair(tr + d, j.O.x, j.O.y);
        if (d == 0) store_pair(tr + D, j.M, j.L);
      }
    }
  }
  if (out0.b < 0 && out1.b < 0) return;
  wait_vm<0>();  // this wave's record stores are done
  __syncthreads();
  int from[2], count[2];
  for (int w = 0; w < 2; ++w) {
    const Piece p = w ? out1 : out0;
    from[w] = p.b < 0 ? 0 : deal.taker(p.first);
    count[w] = p.b < 0 ? 0 : deal.taker(p.first + p.n - 1) - from[w] + 1;
    if (p.b >= 0 && threadIdx.x == 64 * w)
      last_one[w] = __hip_atomic_fetch_add(a.counters + (int64_t)hk * place.units + from[w], 1, __ATOMIC_RELAXED,
                                           __HIP_MEMORY_SCOPE_AGENT) == count[w] - 1;
  }
  __syncthreads();
#pragma unroll 1
  for (int w = 0; w < 2; ++w) {
    const Piece p = w ? out1 : out0;
    if (p.b < 0 || !last_one[w]) continue;
    // The records: the first workgroup's among those that go onwards, the others' among
    // those that come from before, one after another, brought into LDS as many at a time
    // as fit. (This runs once a workgroup, and what it costs beside the round trip is the
    // fetching of instructions that no cache holds yet: joining 19 records of 4 KiB took
    // 9 us with the loop over them unrolled.)
    const int pieces = (int)(rec_size >> 8), fit = T::RING * nw / (1024 * pieces), pairs = gt * DP;
    const int64_t on = ((int64_t)heads + hk) * place.units + from[w], past = (int64_t)hk * place.units + from[w];
#pragma unroll 1
    for (int i0 = 0; i0 < pairs; i0 += blockDim.x) {
      const int i = min(i0 + (int)threadIdx.x, pairs - 1), r = i / DP, d = 2 * (i - r * DP);
      Joined j;
#pragma unroll 1
      for (int c0 = 0; c0 < count[w]; c0 += fit) {
        const int n = min(fit, count[w] - c0);
        if (i0 == 0 || count[w] > fit) {
          __syncthreads();  // (what LDS holds has been read)
#pragma unroll 1
          for (int y = wave; y < n * pieces; y += kPagedWaves) {
            const int c = y / pieces;
            dma16_coherent(uniform(a.part + (c0 + c == 0 ? on : past + c0 + c) * rec_size + 256 * (y - c * pieces)), 16 * lane,
                           lds_addr(lds) + 1024 * y);
          }
          wait_vm<0>();
          __syncthreads();
        }
#pragma unroll 1
        for (int k0 = 0; k0 < n; k0 += 4)
          join<4, NORMAL>(j, k0, n, [&](int, int c, float &m, float &l, float2 &o) {
            const float *const rec = (const float *)lds + c * rec_size + r * T::REC;
            const float2 ml = *(const float2 *)(rec + D);
            m = ml.x, l = ml.y, o = *(const float2 *)(rec + d);
          });
      }
      if (i0 + (int)threadIdx.x < pairs) write(p.b, i, j);
    }
    if (threadIdx.x == 0)
      __hip_atomic_store(a.counters + (int64_t)hk * place.units + from[w], 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
}
