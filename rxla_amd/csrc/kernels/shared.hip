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
// B_n G of them, in blocks of CT x 16 columns that a wave holds in registers. A workgroup walks a piece of a prefix for one block, its waves
// equal pieces of that with a ring of their own each (paged_decode.h), so a block's keys
// are read once by one workgroup, and by the blocks of a head out of its die's cache (the
// workgroups of a head are 8 or more apart, on one die where there are 8 heads).
//
// The launch has both kinds of work: of a head's `units` workgroups some walk prefixes,
// the others the sequences' own keys (paged_decode), in proportion to the tiles that each
// kind has, a prefix's counting kPrefixTile. Both leave records (acc, max, sum) of their
// rows; a second launch joins those of a row in order: the parts of its prefix, its own.
// How the prefixes' tiles were dealt follows from the same numbers there.
namespace {

constexpr float kPrefixTile = 1.4f, kPrefixCodes = 2.f, kPrefixBlock = 4.f;

// Column tiles of a block: as many as leave no register spilled
template <int D, int KIND, int PREC>
constexpr int block_tiles() {
  return D == 256 ? 1 : D == 128 ? (PREC == kHigh ? 1 : 2) : PREC == kHigh || KIND == kCodes ? 2 : 4;
}

// Keys of a prefix's tile: as many as registers and the rings of 8 waves have room for, so
// that a wave has more to do while the next ones come
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
  x.blocks = (x.rows + a.columns - 1) / a.columns;
  x.len = min(max(len, 0), most);
  x.tiles = (int)(((unsigned)x.len + a.keys - 1) / a.keys);
  return x;
}

// Tiles and blocks of a head's run. By a whole wave.
struct Run {
  int tiles, blocks;
};
__device__ __forceinline__ Run run_of(const SharedArgs &a) {
  const int lane = threadIdx.x & 63;
  int tiles = 0, blocks = 0;
  for (int n0 = 0; n0 < a.N; n0 += 64) {
    const int i = min(n0 + lane, a.N - 1);
    const Group x = group_of(a, a.groups[i], a.groups[i + 1], a.prefix_lens[i]);
    const bool in = n0 + lane < a.N && x.tiles > 0;
    tiles += __builtin_amdgcn_readlane(scan64(in ? x.blocks * x.tiles : 0), 63);
    blocks += __builtin_amdgcn_readlane(scan64(in ? x.blocks : 0), 63);
  }
  return Run{tiles, blocks};
}

}  // namespace

// Workgroup `unit` of `units` for the prefixes of kv head h, whose run has `total` tiles
template <int D, int KIND, int PREC>
__device__ RXW8_INLINE void prefix_walk(const SharedArgs &a, int h, int unit, int units, int used, int total) {
  using T = PagedTile<D, KIND, prefix_keys<D, KIND>()>;
  constexpr int CT = block_tiles<D, KIND, PREC>(), CB = 16 * CT;
  using Wave = PagedWave<D, KIND, CT, PREC, T::KT>;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int nw = a.d.waves, G = a.d.Hq / a.d.Hkv;
  if (unit >= used) return;
  const Deal deal(total, used);
  int u0 = __builtin_amdgcn_readfirstlane(deal.start(unit));
  const int u1 = __builtin_amdgcn_readfirstlane(deal.start(unit + 1));

  // the group, block and tile of the run's tile u0
  auto uniform_group = [&](int n) RXW8_INLINE {
    return group_of(a, uniform_load(a.groups, n), uniform_load(a.groups, n + 1), uniform_load(a.prefix_lens, n));
  };
  int n = 0, before = 0;
  Group x = uniform_group(0);
  while (before + x.blocks * x.tiles <= u0) before += x.blocks * x.tiles, x = uniform_group(++n);
  int block = (u0 - before) / x.tiles, t0 = (u0 - before) - block * x.tiles;

  Wave w(a.d, h, lds + wave * T::RING);
  for (;;) {
    const int piece = min(u1 - u0, x.tiles - t0);
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
    const bool all = piece == x.tiles;
    float *const part = a.parts + (((int64_t)(t0 == 0) * a.d.Hkv + h) * units + unit) * (CB * T::REC);
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
            const float f = record_weight(ml[k].x, ml[k].y, M);
            L += f * ml[k].y;
            O += f * *(const f32x4 *)(rec + k * 16 * T::REC + d);
          }
        float *to = part + at * T::REC;
        if (all) {
          const int row = block * CB + at, seq = row / G;
          to = a.whole + ((int64_t)(x.g0 + seq) * a.d.Hq + h * G + (row - seq * G)) * T::REC;
        }
        *(f32x4 *)(to + d) = O;
        if (d == 0) *(float2 *)(to + D) = float2{M, L};
      }
    }
    u0 += piece;
    if (u0 >= u1) return;
    __syncthreads();  // (the records have been read: the rings may be written)
    t0 = 0;
    if (++block == x.blocks) {
      block = 0;
      do x = uniform_group(++n);
      while (x.blocks * x.tiles == 0);
    }
  }
}

template <int D, int KIND, int PREC>
__device__ RXW8_INLINE void shared_walk(const SharedArgs &a) {
  using T = PagedTile<D, KIND>;
  const int lane = threadIdx.x & 63, G = a.d.Hq / a.d.Hkv, HT = (G + 15) / 16, heads = a.d.Hkv * HT;
  const int hk = blockIdx.x % heads, unit = blockIdx.x / heads, units = a.d.units, most = a.d.M * a.d.ps;
  const Run run = run_of(a);
  int own = 0;
  for (int b0 = 0; b0 < a.d.B; b0 += 64) {
    const int len = b0 + lane < a.d.B ? a.d.lens[b0 + lane] : 0;
    own += __builtin_amdgcn_readlane(scan64((int)(((unsigned)min(max(len, 0), most) + T::KT - 1) / T::KT)), 63);
  }
  // a head's workgroups for its prefixes, and for the sequences' own keys
  const float cost = (KIND == kCodes ? kPrefixCodes : kPrefixTile) * ((float)run.tiles + kPrefixBlock * (float)run.blocks) / HT;
  int up = __builtin_amdgcn_readfirstlane((int)rintf(units * cost / fmaxf(cost + (float)own, 1.f)));
  up = run.tiles == 0 ? 0 : own == 0 ? units : min(max(up, 1), max(units - 1, 1));
  const int uo = own == 0 ? 0 : max(units - up, 1);
  // one to every wave's tile, or to every block of fewer
  const int used = min(up * HT, max((run.tiles + a.d.waves - 1) / a.d.waves, run.blocks));
  if (blockIdx.x == 0 && threadIdx.x == 0) a.plan[0] = up * HT, a.plan[1] = used;
  if (unit < up) prefix_walk<D, KIND, PREC>(a, hk / HT, unit * HT + hk % HT, up * HT, used, run.tiles);
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
// loaded at once, its records next: the two round trips are what bounds it.
extern "C" __global__ void __launch_bounds__(256) rxw8_shared_join(SharedArgs a) {
  const int lane = threadIdx.x & 63, D = a.d.D, REC = D + 4, G = a.d.Hq / a.d.Hkv;
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= (int64_t)a.d.B * a.d.Hq) return;  // whole waves only; no barriers below
  const int b = (int)(row / a.d.Hq), hq = (int)(row - (int64_t)b * a.d.Hq), h = hq / G;
  const int units = a.plan[0], used = a.plan[1], len = a.d.lens[b];
  Group x;
  int start = 0, total = 0;
  x.tiles = x.rows = 0;
  for (int n0 = 0; n0 < a.N; n0 += 64) {
    const int i = min(n0 + lane, a.N - 1);
    const Group g = group_of(a, a.groups[i], a.groups[i + 1], a.prefix_lens[i]);
    const int mine = n0 + lane < a.N ? g.blocks * g.tiles : 0, incl = scan64(mine);
    // (the row's group, the last that begins at it or before and has rows: offsets do not decrease)
    const unsigned long long in = __ballot(n0 + lane < a.N && g.g0 <= b && g.g0 + g.rows / G > b);
    if (in) {
      const int k = __builtin_ctzll(in);
      x.g0 = __builtin_amdgcn_readlane(g.g0, k), x.rows = __builtin_amdgcn_readlane(g.rows, k);
      x.tiles = __builtin_amdgcn_readlane(g.tiles, k);
      start = total + __builtin_amdgcn_readlane(incl, k) - __builtin_amdgcn_readlane(mine, k);
    }
    total += __builtin_amdgcn_readlane(incl, 63);
  }
  const float *first_rec = nullptr, *others = nullptr;  // of the prefix
  int prefix = 0;
  if (x.rows && x.tiles) {
    const int i = (b - x.g0) * G + (hq - h * G), block = i / a.columns, col = i - block * a.columns;
    start += block * x.tiles;
    const Deal deal(total, used);
    const int first = deal.taker(start);
    prefix = deal.taker(start + x.tiles - 1) - first + 1;
    const int64_t size = (int64_t)a.columns * REC;
    first_rec = prefix == 1 ? a.whole + row * REC : a.parts + (((int64_t)a.d.Hkv + h) * units + first) * size + col * REC;
    others = a.parts + ((int64_t)h * units + first) * size + col * REC;
  }
  const int count = prefix + (len > 0 && a.d.M > 0);
  for (int d = 2 * lane; d < D; d += 128) {
    Joined j;
#pragma unroll 1
    for (int k0 = 0; k0 < count; k0 += 8)
      join<8>(j, k0, count, [&](int, int k, float &m, float &l, float2 &o) {
        const float *const rec = k >= prefix ? a.own + row * REC : k == 0 ? first_rec : others + (int64_t)k * a.columns * REC;
        const float2 ml = *(const float2 *)(rec + D);
        m = ml.x, l = ml.y, o = *(const float2 *)(rec + d);
      });
    const float inv = j.L == 0.f ? 0.f : 1.0f / j.L;
    if (a.d.out_f32) *(float2 *)((float *)a.d.out + row * D + d) = float2{j.O.x * inv, j.O.y * inv};
    else *(uint32_t *)((uint16_t *)a.d.out + row * D + d) = pack_bf16x2(j.O.x * inv, j.O.y * inv);
  }
}
