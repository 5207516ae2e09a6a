// Attention of one new token per sequence where sequences share a prefix: those of
// groups[n] .. groups[n + 1] - 1 see the first prefix_lens[n] positions of the page table
// prefixes[n], and behind them the first lens[b] positions of their own table.
#include "paged_decode.h"

struct SharedArgs {
  PagedDecodeArgs d;          // the sequences' own keys (d.units: workgroups a head, of both kinds)
  const int32_t *prefixes;    // [N, MP]
  const int32_t *prefix_lens; // [N]
  const int32_t *groups;      // [N + 1]
  int N, MP;
  int b0;                     // the first of this launch's d.B sequences
  int kind;                   // 0 bf16, 1 f32, 2 u8 pages
  // the matrix-core kernels: records of the rows' own keys and of whole prefixes [d.B d.Hq],
  // of parts of prefixes [2, Hkv, units], and how the workgroups were dealt
  float *own, *whole, *parts;
  int *plan;
  int columns, keys;          // of a block; of a prefix's tile
};

// Any head width up to 512, any page size: one workgroup of 4 waves per (sequence, query
// head) over its prefix and its own keys, the waves' chunks of 64 keys in turn
extern "C" __global__ void __launch_bounds__(256) rxw8_shared_any(SharedArgs a) {
  __shared__ float q[RXW8_ATTN_ANY_MAX_D], part[4][RXW8_ATTN_ANY_MAX_D], mw[4], lw[4];
  const int wave = threadIdx.x >> 6;
  const PagedDecodeArgs &d = a.d;
  const int b = blockIdx.x / d.Hq, hq = blockIdx.x - b * d.Hq, h = hq / (d.Hq / d.Hkv);
  const int64_t at = (int64_t)blockIdx.x * d.D;
  for (int i = threadIdx.x; i < d.D; i += 256) q[i] = any_load(d.q, at + i, d.q_f32);
  __syncthreads();
  AnyState st;
  auto walk = [&](const int32_t *table, int64_t n, int m) {
    const int64_t most = (int64_t)m * d.ps;
    auto row = [&](int64_t j) -> int64_t {
      const int64_t page = table[j / d.ps];
      return page < 0 || page >= d.P ? -1 : ((page * d.Hkv + h) * d.ps + j % d.ps) * d.D;
    };
    n = n < most ? n : most;
    if (a.kind == 2)
      any_walk(st, q, AnyCodes{(const uint8_t *)d.kp, (const uint8_t *)d.vp, d.ks, d.vs, d.D}, d.D, 64 * wave, n, 4, d.c, row);
    else
      any_walk(st, q, AnyPlain{d.kp, d.vp, a.kind == 1}, d.D, 64 * wave, n, 4, d.c, row);
  };
  const int g = any_sequence(a.groups, a.N, b);
  if (g >= 0 && b < a.groups[g + 1]) walk(a.prefixes + (int64_t)g * a.MP, a.prefix_lens[g], a.MP);
  walk(d.table + (int64_t)b * d.M, d.lens[b], d.M);
  AnyState all;
  if (!any_join(all, st, part, mw, lw)) return;
  any_store(all, d.out, at, d.D, d.out_f32);
}

// ---- head widths 64, 128, 256, pages of whole 16-row pieces: matrix cores --------
//
// The G query heads of a kv head of all of a prefix's sequences are rows of one product:
// B_n G of them, in blocks of CT x 16 columns that a wave holds in registers. A workgroup walks
// a piece of a prefix for one block, its waves equal pieces of that with a ring of their own each
// (paged_decode.h), so a block's keys are read once by one workgroup, and by the blocks of
// a head out of its die's cache (the workgroups of a head are 8 or more apart, on one die
// where there are 8 heads).
//
// The launch has both kinds of work: of a head's `units` workgroups some walk prefixes, the
// others the sequences' own keys (paged_decode). A prefix's blocks are cut into equal pieces, in
// number by its share of all prefixes' tiles (plan_of), and a workgroup has one, or a few whole:
// what a piece costs beside its tiles (q's way and the first tile's, the joins) is some tiles'
// time, and pieces dealt by tiles alone, across the borders of blocks, made many workgroups
// pay it twice (48 sequences behind 8192 positions in 8 bits, 32 / 4 heads of 128: 37.6 us, 34.0
// so; 20 behind 4 prefixes of 6391, 32 / 8 heads, f32: 31.4, 25.6; 64 behind 6000, bf16,
// 32 / 8 heads: 48.2, 47.0). Both kinds leave records (acc, max, sum) of their rows; a second
// launch joins those of a row in order: the pieces of its prefix, its own. (These and the other
// comparisons here are of when a choice was made. All together now: 48 behind 8192 in 8 bits 35.1 us, 64 behind
// 6000 47.5, 96 behind 3 prefixes of 700 to 4000, f32 queries, 40.7.)
namespace {

// What a tile of a prefix costs of one of own keys, and a piece and a sequence of own keys of a
// tile, beside their tiles. (3 prefixes of 700 to 4000 before 96 sequences of up to 300, f32, 16 / 8 heads
// of 128: 41.1 us; with 4 for a sequence 50.6, own keys left to too few. 166 of up to 78 behind 1 to 4
// positions, 8 heads: 23.0; with 8 for a piece 22.9, with 8 and 16 for a sequence 26.3.)
constexpr float kPrefixTile = 2.f, kPrefixBlock = 24.f, kOwnSequence = 8.f;

// Column tiles of a block: as many as the registers hold (all of one tile: 64 sequences behind
// 6000 positions, bf16, heads of 128, 60.3 us against 47.0; 48 behind 8192 in 8 bits 37.2, 34.0)
template <int D, int KIND, int PREC>
constexpr int block_tiles() {
  return D == 256 ? 1 : D == 128 ? (PREC == kHigh ? 1 : 2) : PREC == kHigh || KIND == kCodes ? 2 : 4;
}

// Keys of a prefix's tile: as many as registers and the rings of 8 waves have room for, so
// that a wave has more to do while the next ones come (16 of bf16 and 32 of 8 bits: the same
// 60.7 us against 47.0 and 36.2, 34.0; f32 queries behind 3 prefixes 51.5, 41.2)
template <int D, int KIND>
constexpr int prefix_keys() {
  return KIND == kCodes ? (D == 256 ? 32 : 64) : KIND == kF32 || D == 256 ? 16 : 32;
}

// Group n's sequences within this launch's (relative to b0), blocks and tiles
struct Group {
  int g0, rows, blocks, len, tiles;
};
__device__ __forceinline__ Group group_of(const SharedArgs &a, int g_from, int g_to, int len) {
  Group x;
  const int end = a.b0 + a.d.B, most = a.MP * a.d.ps;
  x.g0 = min(max(g_from, a.b0), end) - a.b0;
  x.rows = max(min(max(g_to, a.b0), end) - a.b0 - x.g0, 0) * (a.d.Hq / a.d.Hkv);
  x.blocks = (x.rows + a.columns - 1) >> __builtin_ctz(a.columns);  // (powers of two, both)
  x.len = min(max(len, 0), most);
  x.tiles = (int)(((unsigned)x.len + a.keys - 1) >> __builtin_ctz(a.keys));
  return x;
}

// Pieces of a prefix of `tiles`, `rate` of them to a tile: one at least, and a tile for every wave.
// (fmaf: the walk and the join's launch, which read each other's records, round alike)
__device__ __forceinline__ int pieces_of(int tiles, float rate) {
  return min(max((int)fmaf((float)tiles, rate, 0.5f), 1), (int)(((unsigned)tiles + kPagedWaves - 1) / kPagedWaves));
}
// Groups in lanes: those from n0 on
__device__ __forceinline__ Group groups_from(const SharedArgs &a, int n0) {
  const int lane = threadIdx.x & 63, i = min(n0 + lane, a.N - 1);
  Group x = group_of(a, a.groups[i], a.groups[i + 1], a.prefix_lens[i]);
  if (n0 + lane >= a.N) x.rows = x.blocks = 0;
  return x;
}
struct Pieces {
  int each, count, incl, parts, part_incl;  // of a block, of all; the sums; those that leave parts
  __device__ __forceinline__ Pieces(const Group &x, float rate) {
    each = pieces_of(x.tiles, rate);
    count = x.blocks * each;
    parts = each > 1 ? count : 0;
    incl = scan64(count), part_incl = scan64(parts);
  }
};
__device__ __forceinline__ int max64(int v) {  // over the 64 lanes, of numbers from 0 on
  v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false));
  v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false));
  v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false));
  v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false));
  v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false));
  v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false));
  return __builtin_amdgcn_readlane(v, 63);
}
// Workgroups of a kv head (its HT heads of columns together) for its prefixes, and the pieces'
// rate: those by which the longer of two takes least, the longest piece (times the pieces of a
// workgroup) and a workgroup's share of the own keys, in tiles. Tried are rates around the one
// that makes both the same, each with a workgroup to a piece and with as many as that one has.
// By a whole wave.
struct Plan {
  int takers;
  float rate;
};
__device__ __forceinline__ Plan plan_of(const SharedArgs &a, const Group &first, float own, int HT) {
  constexpr int kRates = 4;
  const float factor[kRates] = {0.7f, 0.85f, 1.f, 1.2f};
  int tiles = 0, blocks = 0, finest = 0;
  for (int n0 = 0; n0 < a.N; n0 += 64) {
    const Group x = n0 ? groups_from(a, n0) : first;
    finest += __builtin_amdgcn_readlane(scan64(x.blocks * pieces_of(x.tiles, 1.f)), 63);
    tiles += __builtin_amdgcn_readlane(scan64(x.blocks * x.tiles), 63);
    blocks += __builtin_amdgcn_readlane(scan64(x.tiles ? x.blocks : 0), 63);
  }
  if (tiles <= 0) return Plan{0, 0.f};
  const int most = (own == 0.f ? a.d.units : max(a.d.units - 1, 1)) * HT;
  const float cost = kPrefixTile * ((float)tiles + kPrefixBlock * (float)blocks) / HT;
  const int even = min(max((int)rintf(a.d.units * HT * cost / (cost + own)), 1), most);
  if (finest <= even) return Plan{finest, 1.f};
  const float rate = (float)even / (float)tiles;
  int items[kRates] = {0, 0, 0, 0}, longest[kRates] = {0, 0, 0, 0};
  for (int n0 = 0; n0 < a.N; n0 += 64) {
    const Group x = n0 ? groups_from(a, n0) : first;
#pragma unroll
    for (int j = 0; j < kRates; ++j) {
      const int each = pieces_of(x.tiles, factor[j] * rate);
      const int len = x.blocks && each ? (int)ceilf((float)x.tiles * __builtin_amdgcn_rcpf((float)each)) : 0;
      items[j] += __builtin_amdgcn_readlane(scan64(x.blocks * each), 63);
      longest[j] = max(longest[j], max64(len));
    }
  }
  Plan best{1, 0.f};
  float least = INFINITY;
#pragma unroll
  for (int j = 0; j < kRates; ++j)
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int takers = max(min(k ? even : items[j], most), 1), up = (takers + HT - 1) / HT;
      const float walk = kPrefixTile * ((float)longest[j] + kPrefixBlock) * ceilf((float)items[j] * __builtin_amdgcn_rcpf((float)takers) - 0.01f);
      const float rest = own * __builtin_amdgcn_rcpf((float)max(a.d.units - up, 1)), t = fmaxf(walk, rest);
      if (t < least) least = t, best = Plan{takers, factor[j] * rate};
    }
  best.takers = __builtin_amdgcn_readfirstlane(best.takers);
  best.rate = __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(best.rate)));
  return best;
}
// The place of a part's record of kv head h: at most 2 d.units HT of them by plan_of
__device__ __forceinline__ float *part_of(const SharedArgs &a, int HT, int h, int at) {
  const int most = 2 * a.d.units * HT;
  return a.parts + ((int64_t)h * most + min(max(at, 0), most - 1)) * ((int64_t)a.columns * (a.d.D + 4));
}

}  // namespace

// Workgroup `unit` of plan.takers for the prefixes of kv head h
template <int D, int KIND, int PREC>
__device__ RXW8_INLINE void prefix_walk(const SharedArgs &a, int h, int unit, int HT, const Plan &plan, const Group &in_lanes) {
  using T = PagedTile<D, KIND, prefix_keys<D, KIND>()>;
  constexpr int CT = block_tiles<D, KIND, PREC>(), CB = 16 * CT;
  using Wave = PagedWave<D, KIND, CT, PREC, T::KT>;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int nw = a.d.waves, G = a.d.Hq / a.d.Hkv;
  int n0 = 0, before = 0, parts = 0;  // 64 groups, and what those before have
  Wave w(a.d, h, lds + wave * T::RING);
  for (int item = unit;; item += plan.takers) {
    // ---- the group, block and piece of the item
    Group x;
    int n, at, pieces, part_at;
    for (;; n0 += 64) {
      if (n0 >= a.N) return;
      const Group g = n0 || D == 256 || KIND == kF32 ? groups_from(a, n0) : in_lanes;  // (no registers to keep them in)
      const Pieces p(g, plan.rate);
      const int total = __builtin_amdgcn_readlane(p.incl, 63);
      if (item - before >= total) {
        before += total, parts += __builtin_amdgcn_readlane(p.part_incl, 63);
        continue;
      }
      const int k = __popcll(__ballot(p.incl <= item - before));
      auto of = [&](int v) RXW8_INLINE { return __builtin_amdgcn_readlane(v, k); };
      n = n0 + k, at = item - before - of(p.incl - p.count), pieces = of(p.each);
      part_at = parts + of(p.part_incl - p.parts) + at;
      x.g0 = of(g.g0), x.rows = of(g.rows), x.len = of(g.len), x.tiles = of(g.tiles);
      break;
    }
    const int block = __builtin_amdgcn_readfirstlane(at / pieces);
    const Deal deal(x.tiles, pieces);
    const int t0 = __builtin_amdgcn_readfirstlane(deal.start(at - block * pieces));
    const int piece = __builtin_amdgcn_readfirstlane(deal.start(at - block * pieces + 1)) - t0;
    if (item != unit) __syncthreads();  // (the records have been read: the rings may be written)
    const int cols = min(CB, x.rows - block * CB), ct = (cols + 15) / 16;
    const Deal waves(piece, nw);
    const int first = t0 + waves.start(wave);
    int left = wave < nw ? t0 + waves.start(wave + 1) - first : 0;
    if (left > 0) {
      w.begin(a.prefixes + (int64_t)n * a.MP, a.MP, x.len, first);
      typename Wave::Tile cur = w.tile();
      w.copy_k();
      w.copy_v();
#pragma unroll
      for (int c = 0; c < CT; ++c) {
        const int i = min(block * CB + 16 * c + w.col, x.rows - 1), r = i / G;
        w.load_q(c, ((int64_t)(x.g0 + r) * a.d.Hq + h * G + (i - r * G)) * D);
      }
      w.wait_q();  // (and for the first tile)
      for (;;) {
        wait_vm<T::N>();
        w.scores(ct);
        wait_lds();
        const typename Wave::Tile done = cur;
        if (left > 1) {
          cur = w.tile();
          w.copy_k();
        }
        const bool part = done.seen < T::KT || done.holes;
        w.softmax(done, part, ct);
        if (left > 1) wait_vm<T::NK>();
        else wait_vm<0>();
        if (part && KIND != kCodes) w.clear_v(done);
        w.values(ct);
        wait_lds();
        if (left > 1) w.copy_v();
        if (--left == 0) break;
      }
    }
    // ---- the waves' records joined, 16 columns at a time
    const int count = min(nw, piece);
    const bool all = pieces == 1;
    float *const part = part_of(a, HT, h, part_at);
#pragma unroll
    for (int c = 0; c < CT; ++c) {
      if (c >= ct) break;
      __syncthreads();
      if (wave < count) w.record(c, (float *)lds + (wave * 16 + w.col) * T::REC);
      __syncthreads();
      for (int i = threadIdx.x; i < 16 * (D / 4); i += blockDim.x) {  // (four dims of a row)
        const int r = i / (D / 4), d = 4 * (i - r * (D / 4)), at = 16 * c + r;
        if (at >= cols) break;
        const float *const rec = (const float *)lds + r * T::REC;
        float2 ml[kPagedWaves];
        float M = kMinusInf, L = 0.f;
        f32x4 O = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < kPagedWaves; ++k) {
          ml[k] = k < count ? *(const float2 *)(rec + k * 16 * T::REC + D) : float2{kMinusInf, 0.f};
          M = fmaxf(M, ml[k].x);
        }
#pragma unroll
        for (int k = 0; k < kPagedWaves; ++k)
          if (k < count) {
            ml[k].x = record_weight(ml[k].x, ml[k].y, M);
            L += ml[k].x * ml[k].y;
          }
        const float inv = L == 0.f ? 0.f : 1.0f / L;
#pragma unroll
        for (int k = 0; k < kPagedWaves; ++k)  // (over codes as join's records)
          if (k < count) O += (KIND == kCodes ? ml[k].x * ml[k].y * inv : ml[k].x) * *(const f32x4 *)(rec + k * 16 * T::REC + d);
        float *to = part + at * T::REC;
        if (all) {
          const int row = block * CB + at, seq = row / G;
          to = a.whole + ((int64_t)(x.g0 + seq) * a.d.Hq + h * G + (row - seq * G)) * T::REC;
        }
        *(f32x4 *)(to + d) = O;
        if (d == 0) *(float2 *)(to + D) = float2{M, L};
      }
    }
  }
}

template <int D, int KIND, int PREC>
__device__ RXW8_INLINE void shared_walk(const SharedArgs &a) {
  using T = PagedTile<D, KIND>;
  const int lane = threadIdx.x & 63, G = a.d.Hq / a.d.Hkv, HT = (G + 15) / 16, heads = a.d.Hkv * HT;
  const int hk = blockIdx.x % heads, unit = blockIdx.x / heads, units = a.d.units, most = a.d.M * a.d.ps;
  const Group first = groups_from(a, 0);
  int own = 0, some = 0;  // tiles, and sequences that have any
  for (int b0 = 0; b0 < a.d.B; b0 += 64) {
    const int len = b0 + lane < a.d.B ? a.d.lens[b0 + lane] : 0;
    const int tiles = (int)(((unsigned)min(max(len, 0), most) + T::KT - 1) / T::KT);
    own += __builtin_amdgcn_readlane(scan64(tiles), 63);
    some += __popcll(__ballot(tiles > 0));
  }
  // a head's workgroups for its prefixes, and for the sequences' own keys
  const Plan plan = plan_of(a, first, (float)own + kOwnSequence * (float)some, HT);
  const int up = (plan.takers + HT - 1) / HT, uo = own == 0 ? 0 : max(units - up, 1);
  if (blockIdx.x == 0 && threadIdx.x == 0) a.plan[0] = __float_as_int(plan.rate);
  if (unit < up && unit * HT + hk % HT < plan.takers) prefix_walk<D, KIND, PREC>(a, hk / HT, unit * HT + hk % HT, HT, plan, first);
  if (unit >= units - uo) {
    if (unit < up) __syncthreads();  // (one workgroup to a head does both)
    paged_decode<D, KIND, true, PREC>(a.d, PagedPlaceOf{hk, unit - (units - uo), uo, a.own});
  }
}

#define RXW8_SHARED(D, NAME, KIND, PREC)                                                           \
  extern "C" __global__ void __launch_bounds__(64 * kPagedWaves) rxw8_shared_##NAME##_d##D(SharedArgs a) { \
    shared_walk<D, KIND, PREC>(a);                                                                 \
  }
#define RXW8_SHARED_D(D)                   \
  RXW8_SHARED(D, bf16, kBf16, kLow)        \
  RXW8_SHARED(D, bf16_high, kBf16, kHigh)  \
  RXW8_SHARED(D, q8, kCodes, kLow)         \
  RXW8_SHARED(D, q8_high, kCodes, kHigh)   \
  RXW8_SHARED(D, f32, kF32, kAny)
RXW8_SHARED_D(64)
RXW8_SHARED_D(128)
RXW8_SHARED_D(256)

// The records of a row joined: a wave a row. Up to 64 groups, all that a row has to know is
// loaded at once, its records next: the two round trips bound it (4 to 5 us for 2048 rows).
extern "C" __global__ void __launch_bounds__(256) rxw8_shared_join(SharedArgs a) {
  const int lane = threadIdx.x & 63, D = a.d.D, REC = D + 4, G = a.d.Hq / a.d.Hkv, HT = (G + 15) / 16;
  const unsigned at32 = blockIdx.x * 4 + (threadIdx.x >> 6);  // (fewer than 2^24 rows)
  if (at32 >= (unsigned)(a.d.B * a.d.Hq)) return;  // whole waves only; no barriers below
  const int i0 = min(lane, a.N - 1), from = a.groups[i0], to = a.groups[i0 + 1], of = a.prefix_lens[i0];
  const float rate = __int_as_float(a.plan[0]);
  const int b = (int)(at32 / (unsigned)a.d.Hq), hq = (int)at32 - b * a.d.Hq, h = (int)((unsigned)hq / (unsigned)G);
  const int len = a.d.lens[b];
  const int64_t row = at32;
  const float *first = nullptr;  // of the prefix
  int prefix = 0, parts = 0;
  for (int n0 = 0; n0 < a.N; n0 += 64) {
    Group g = n0 ? groups_from(a, n0) : group_of(a, from, to, of);
    if (n0 + lane >= a.N) g.rows = g.blocks = 0;
    const Pieces p(g, rate);
    const unsigned long long in = __ballot(g.g0 <= b && g.rows > (b - g.g0) * G);
    if (in) {
      const int k = __builtin_ctzll(in);
      const int i = (b - __builtin_amdgcn_readlane(g.g0, k)) * G + (hq - h * G), block = i >> __builtin_ctz(a.columns), col = i & (a.columns - 1);
      prefix = __builtin_amdgcn_readlane(p.each, k);
      const int at = parts + __builtin_amdgcn_readlane(p.part_incl - p.parts, k) + block * prefix;
      first = prefix == 1 ? a.whole + row * REC : part_of(a, HT, h, at) + col * REC;
      break;
    }
    parts += __builtin_amdgcn_readlane(p.part_incl, 63);
  }
  const int count = prefix + (len > 0 && a.d.M > 0);
  auto out = [&](auto normal) {
    constexpr bool NORMAL = decltype(normal)::value;  // (as join)
    for (int d = 2 * lane; d < D; d += 128) {
      Joined j;
#pragma unroll 1
      for (int k0 = 0; k0 < count; k0 += 8)
        join<8, NORMAL>(j, k0, count, [&](int, int k, float &m, float &l, float2 &o) {
          const float *const rec = k >= prefix ? a.own + row * REC : first + (int64_t)k * a.columns * REC;
          const float2 ml = *(const float2 *)(rec + D);
          m = ml.x, l = ml.y, o = *(const float2 *)(rec + d);
        });
      const float inv = NORMAL ? 1.f : j.L == 0.f ? 0.f : 1.0f / j.L;
      if (a.d.out_f32) *(float2 *)((float *)a.d.out + row * D + d) = float2{j.O.x * inv, j.O.y * inv};
      else *(uint32_t *)((uint16_t *)a.d.out + row * D + d) = pack_bf16x2(j.O.x * inv, j.O.y * inv);
    }
  };
  if (a.kind == 2) out(std::true_type{});
  else out(std::false_type{});
}
