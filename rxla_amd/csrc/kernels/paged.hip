// The paged key/value cache: the append that fills its pages and the attention of
// one new token per sequence that reads them. Pages are [P, Hkv, ps, D] (a kv
// head's ps rows of a page in one piece); table [B, M] I32 gives sequence b the
// page of its positions ps i .. ps i + ps - 1 in entry i, anything outside [0, P)
// where it has none. An entry is checked before its page is touched.
#include "attn_any.h"

struct PagedAppendArgs {
  const void *k, *v;         // [T, Hkv, D] f32 | bf16
  void *kp, *vp;             // [P, Hkv, ps, D] f32 | bf16
  const int32_t *table;      // [B, M]
  const int32_t *starts;     // [B] position of a sequence's first new row
  const int32_t *offsets;    // [B + 1] packed rows of the sequences, or null: row b of sequence b
  int64_t T, P;
  int B, M, Hkv, D, ps;
  int k_f32, p_f32;
};

// Row i of sequence b goes to position starts[b] + i. One wave per (row, kv head);
// rows outside every sequence and positions without a page are passed over. An f32
// row is rounded once (RNE) on its way into bf16 pages, a bf16 row widened exactly.
extern "C" __global__ void __launch_bounds__(256) rxw8_paged_append(PagedAppendArgs a) {
  const int lane = threadIdx.x & 63;
  const int64_t unit = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (unit >= a.T * a.Hkv) return;
  const int64_t t = unit / a.Hkv;
  const int h = (int)(unit - t * a.Hkv);
  int64_t b = t, i = 0;
  if (a.offsets) {
    b = any_sequence(a.offsets, a.B, t);
    if (b < 0 || t >= a.offsets[b + 1]) return;
    i = t - a.offsets[b];
  }
  const int64_t pos = a.starts[b] + i;
  if (pos < 0 || pos >= (int64_t)a.M * a.ps) return;
  const int64_t page = a.table[b * a.M + pos / a.ps];
  if (page < 0 || page >= a.P) return;
  const int64_t src = unit * a.D, dst = ((page * a.Hkv + h) * a.ps + pos % a.ps) * a.D;
  for (int e = lane; e < a.D; e += 64) {
    const float x = any_load(a.k, src + e, a.k_f32), y = any_load(a.v, src + e, a.k_f32);
    if (a.p_f32) {
      ((float *)a.kp)[dst + e] = x;
      ((float *)a.vp)[dst + e] = y;
    } else {
      ((uint16_t *)a.kp)[dst + e] = f32_to_bf16_bits(x);
      ((uint16_t *)a.vp)[dst + e] = f32_to_bf16_bits(y);
    }
  }
}

struct PagedDecodeArgs {
  const void *q;          // [B, Hq, D] f32 | bf16
  const void *kp, *vp;    // [P, Hkv, ps, D] f32 | bf16
  const int32_t *table;   // [B, M]
  const int32_t *lens;    // [B]
  void *out;              // [B, Hq, D] f32 | bf16
  int64_t P;
  int B, M, Hq, Hkv, D, ps;
  float c;                // scale log2 e
  int q_f32, p_f32, out_f32;
  // the matrix-core kernels: `units` workgroups for each kv head and 16 of its
  // query heads; counters [Hkv HT units], zero between launches, and partials
  // [Hkv HT units][2][min(G, 16)][D + 4]
  int units;
  int *counters;
  float *part;
};

__device__ __forceinline__ int64_t paged_len(const PagedDecodeArgs &a, int b) {
  const int64_t n = a.lens[b], most = (int64_t)a.M * a.ps;
  return n < 0 ? 0 : n > most ? most : n;
}

// Any head width up to 512, any page size: one workgroup of 4 waves per (sequence,
// query head), the waves' chunks of 64 keys in turn, merged in LDS.
extern "C" __global__ void __launch_bounds__(256) rxw8_paged_decode_any(PagedDecodeArgs a) {
  __shared__ float q[RXW8_ATTN_ANY_MAX_D], part[4][RXW8_ATTN_ANY_MAX_D], mw[4], lw[4];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int b = blockIdx.x / a.Hq, hq = blockIdx.x - b * a.Hq, h = hq / (a.Hq / a.Hkv);
  const int64_t at = (int64_t)blockIdx.x * a.D;
  for (int i = threadIdx.x; i < a.D; i += 256) q[i] = any_load(a.q, at + i, a.q_f32);
  __syncthreads();
  AnyState st;
  any_walk(st, q, a.kp, a.vp, a.p_f32, a.D, 64 * wave, paged_len(a, b), 4, a.c, [&](int64_t j) -> int64_t {
    const int64_t page = a.table[(int64_t)b * a.M + j / a.ps];
    return page < 0 || page >= a.P ? -1 : ((page * a.Hkv + h) * a.ps + j % a.ps) * a.D;
  });
  if (lane == 0) mw[wave] = st.m, lw[wave] = st.l;
#pragma unroll
  for (int i = 0; i < RXW8_ATTN_ANY_MAX_D / 64; ++i) part[wave][lane + 64 * i] = st.acc[i];
  __syncthreads();
  if (wave) return;
  float m = kMinusInf;
  for (int w = 0; w < 4; ++w) m = fmaxf(m, mw[w]);
  AnyState all;
  for (int w = 0; w < 4; ++w) {
    const float f = mw[w] == kMinusInf ? (lw[w] != lw[w] ? lw[w] : 0.f) : exp2f(mw[w] - m);
    all.l += f * lw[w];
#pragma unroll
    for (int i = 0; i < RXW8_ATTN_ANY_MAX_D / 64; ++i) all.acc[i] += f * part[w][lane + 64 * i];
  }
  any_store(all, a.out, at, a.D, a.out_f32);
}

// ---- head widths 64, 128, 256, pages of whole 16-row pieces: matrix cores --------
//
// What bounds it is the cache: 2 D keys' bytes read once, for G = Hq / Hkv query
// heads together (they are the columns of the products, up to 16; more heads take
// further workgroups). So the work is dealt by bytes: the keys of a kv head, all
// sequences one after another, are a run of tiles of KT keys; each of its `units`
// workgroups (one fills a CU, by LDS) takes an equal piece of the run and each wave
// of it an equal piece of that, whatever the sequences' lengths. A wave that meets
// a sequence's end goes on with the next one.
//
// A wave copies its tiles by LDS DMA into a ring of its own, two tiles deep (the
// next tile's 8 to 32 KiB in flight while one is worked on), so the loop has no
// barrier and holds no registers for loads. Rows keep their order in LDS, their
// 16-byte chunks XOR-swizzled by row. Per 16 keys and 16 heads:
//   S^T = K q^T    A = K rows, B = q: 16x16x32 bf16 (an f32 q as high and low
//                  parts: exact products of what two bf16 hold), 16x16x4 f32;
//   softmax        lane = head, its four lanes share the keys; O is rescaled only
//                  where the running maximum moves;
//   O^T += V^T P^T A = V by transposing reads (bf16), B = P straight from the score
//                  registers as high and low parts (16x16x16); f32 caches take the
//                  f32 products and the dims in the order of 16-byte pieces.
// V rows that a tile's last key or a missing page leaves unseen are cleared in LDS
// (their weights are zero, what they hold may be NaN); K's scores there are -inf.
//
// A sequence inside one wave's piece is written at once. Pieces of a sequence are
// joined in the order of its keys: the waves' in LDS, then, if it passes a
// workgroup's piece, by the last of its workgroups to arrive, over (max, sum, acc)
// records in device memory (at most two a workgroup). Stores and loads of those are
// device-coherent around an arrival counter; the last one sets it back to zero.
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

template <int D, bool F32>
struct PagedTile {
  static constexpr int ES = F32 ? 4 : 2, ROW = D * ES, CH = ROW / 16;
  static constexpr int KT = ROW < 256 ? 32 : 16;  // keys of a tile
  static constexpr int SUB = KT / 16, HALF = KT * ROW, N = HALF / 1024, RPI = 1024 / ROW;
  static constexpr int RING = 4 * HALF;           // two tiles of K and V
  static constexpr int REC = D + 4;               // floats of a record: acc [D], max, sum
  static __device__ __forceinline__ int kx(int row) { return row & (CH < 16 ? CH - 1 : 15); }
  static __device__ __forceinline__ int vx(int row) { return F32 ? 0 : 2 * (row & (CH < 16 ? 3 : 7)); }
};

struct Piece {  // of a sequence, that one wave or workgroup went over
  int b, first, n;  // sequence; its first tile in the head's run; its tiles
};

}  // namespace

template <int D, bool F32>
__device__ void paged_decode(const PagedDecodeArgs &a) {
  using T = PagedTile<D, F32>;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  __shared__ Piece piece[kPagedWaves][2];
  __shared__ int last_one[2];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int nw = blockDim.x >> 6, col = lane & 15, g4 = lane >> 4;
  const int G = a.Hq / a.Hkv, HT = (G + 15) / 16, heads = a.Hkv * HT, gcap = min(G, 16);
  const int hk = blockIdx.x % heads, unit = blockIdx.x / heads, h = hk / HT, ht = hk - h * HT;
  const int gt = min(16, G - 16 * ht), hq0 = h * G + 16 * ht;
  const int most = a.M * a.ps;
  auto tiles_of = [&](int len) { return (min(max(len, 0), most) + T::KT - 1) / T::KT; };

  // the head's run: total tiles, and (up to 64 sequences) where each begins
  int total = 0, incl = 0, mine = 0;
  auto scan = [&](int b0) {  // of 64 sequences: lane's tiles and their inclusive sum
    mine = b0 + lane < a.B ? tiles_of(a.lens[b0 + lane]) : 0;
    incl = mine;
    for (int o = 1; o < 64; o <<= 1) {
      const int y = __shfl_up(incl, o);
      if (lane >= o) incl += y;
    }
    return __builtin_amdgcn_readlane(incl, 63);
  };
  for (int b0 = 0; b0 < a.B; b0 += 64) total += scan(b0);
  const int units = min(a.units, (total + nw - 1) / nw);
  const Deal deal(total, max(units, 1));
  const int u0 = unit < units ? deal.start(unit) : 0, u1 = unit < units ? deal.start(unit + 1) : 0;
  const Deal waves(u1 - u0, nw);
  int at = u0 + waves.start(wave), left = u0 + waves.start(wave + 1) - at;
  piece[wave][0].b = piece[wave][1].b = -1;

  char *const mem = lds + wave * (T::RING + gcap * T::REC * 4);
  float *const first_rec = (float *)(mem + T::RING), *const last_rec = (float *)mem;
  if (left > 0) {
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
    struct Tile {
      int b, t, n, seen, holes;       // keys in it; bit s: its 16-key piece s has no page
      int64_t off[T::SUB];            // bytes from the pool's start
    };
    const int ps16 = a.ps >> 4;
    auto next = [&](bool more) {  // the tile that `ah` stands at; `more`: another one follows
      Tile x;
      x.b = ah.b, x.t = ah.t, x.n = ah.n, x.holes = 0;
      x.seen = min(ah.len - ah.t * T::KT, T::KT);
#pragma unroll
      for (int s = 0; s < T::SUB; ++s) {
        const unsigned sub = (unsigned)(ah.t * T::SUB + (16 * s < x.seen ? s : 0));
        const unsigned e = sub / (unsigned)ps16;
        int page = uniform_load(a.table, (int64_t)ah.b * a.M + e);
        if (page < 0 || page >= a.P) page = 0, x.holes |= 1 << s;
        x.off[s] = (((int64_t)page * a.Hkv + h) * a.ps + 16 * (int)(sub - e * ps16)) * T::ROW;
      }
      if (more && ++ah.t == ah.n) {
        do {
          ++ah.b;
          ah.len = min(max(uniform_load(a.lens, ah.b), 0), most);
        } while (ah.len == 0);
        ah.n = tiles_of(ah.len);
        ah.t = 0;
      }
      return x;
    };
    const int lrow = lane / T::CH, lch = lane % T::CH;
    auto copy = [&](const void *pool, const Tile &x, int slot, int half) {
      const uint32_t dst = lds_addr(mem) + (2 * slot + half) * T::HALF;
#pragma unroll
      for (int i = 0; i < T::N; ++i) {
        const int row = i * T::RPI + lrow, sx = half ? T::vx(row) : T::kx(row);
        dma16((const char *)pool + x.off[i * T::RPI / 16], (uint32_t)(row & 15) * T::ROW + ((lch ^ sx) << 4),
              dst + 1024 * i);
      }
    };

    Tile cur, nx;  // the tile at hand, the one after it
    // ---- q, O and the softmax of the sequence at hand
    constexpr int NQ = F32 ? D / 16 : D / 32;  // 16-byte pieces of a head's q per lane
    u32x4 q[NQ], ql[F32 ? 1 : NQ];
    f32x4 o[D / 16];
    float m = kMinusInf, l = 0.f;
    auto start = [&](int seq) {
      const int64_t qo = ((int64_t)seq * a.Hq + hq0 + min(col, gt - 1)) * D;
#pragma unroll
      for (int i = 0; i < NQ; ++i) {
        if constexpr (F32) {
          const int64_t at4 = qo + 16 * i + 4 * g4;
          if (a.q_f32) {
            q[i] = *(const u32x4 *)((const float *)a.q + at4);
          } else {
            const uint2 r = *(const uint2 *)((const uint16_t *)a.q + at4);
            q[i] = u32x4{r.x << 16, r.x & 0xffff0000u, r.y << 16, r.y & 0xffff0000u};
          }
        } else {
          const int64_t at8 = qo + 32 * i + 8 * g4;
          if (a.q_f32) {
            const f32x4 r[2] = {*(const f32x4 *)((const float *)a.q + at8), *(const f32x4 *)((const float *)a.q + at8 + 4)};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              uint32_t hi, lo;
              split_bf16x2(r[e >> 1][2 * (e & 1)], r[e >> 1][2 * (e & 1) + 1], hi, lo);
              q[i][e] = hi, ql[i][e] = lo;
            }
          } else {
            q[i] = *(const u32x4 *)((const uint16_t *)a.q + at8);
          }
        }
      }
      m = kMinusInf;
      l = 0.f;
#pragma unroll
      for (int i = 0; i < D / 16; ++i) o[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    };
    // dims of o[i]: bf16 16 i + 4 g4 + r; f32 64 (i / 4) + 16 g4 + 4 r + i % 4
    auto finish = [&](int seq, int first, bool whole, float *rec, Piece *p) {
      const float sum = sum4(l);
      if (whole) {
        if (col < gt) {
          const float inv = sum == 0.f ? 0.f : 1.0f / sum;
          const int64_t to = ((int64_t)seq * a.Hq + hq0 + col) * D;
#pragma unroll
          for (int i = 0; i < D / 16; ++i) {
            f32x4 y;
#pragma unroll
            for (int r = 0; r < 4; ++r) y[r] = (F32 ? o[(i & ~3) + r][i & 3] : o[i][r]) * inv;
            const int64_t d = to + (F32 ? 64 * (i >> 2) + 16 * g4 + 4 * (i & 3) : 16 * i + 4 * g4);
            if (a.out_f32)
              *(f32x4 *)((float *)a.out + d) = y;
            else
              *(uint2 *)((uint16_t *)a.out + d) = uint2{pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3])};
          }
        }
        return;
      }
      if (col < gt) {
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
          f32x4 y;
#pragma unroll
          for (int r = 0; r < 4; ++r) y[r] = F32 ? o[(i & ~3) + r][i & 3] : o[i][r];
          *(f32x4 *)(rec + col * T::REC + (F32 ? 64 * (i >> 2) + 16 * g4 + 4 * (i & 3) : 16 * i + 4 * g4)) = y;
        }
        if (g4 == 0) rec[col * T::REC + D] = m, rec[col * T::REC + D + 1] = sum;
      }
      if (lane == 0) *p = Piece{seq, first, cur.n};
    };

    // (q is on its way while the first pages are looked up, and in before the copies
    // go out: a wait for it later would be a wait for them)
    start(b);
    cur = next(left > 1);
#pragma unroll
    for (int i = 0; i < NQ; ++i) asm volatile("" : "+v"(q[i]));
    copy(a.kp, cur, 0, 0);
    copy(a.vp, cur, 0, 1);
    if (left > 1) {
      nx = next(left > 2);
      copy(a.kp, nx, 1, 0);
      copy(a.vp, nx, 1, 1);
    }

    // LDS byte addresses of the fragments in tile 0 (the swizzles are XORs below)
    const uint32_t kf = lds_addr(mem) + col * T::ROW;
    const int tr_j = col >> 2, tr_q = col & 3;
    const uint32_t vf = lds_addr(mem) + T::HALF + (F32 ? 4 * g4 * T::ROW + 16 * col : (4 * g4 + tr_j) * T::ROW + 8 * (tr_q & 1));
    int begun = cur.t;  // the tile at which this wave began the sequence
    for (int i = 0;; ++i) {
      const int slot = i & 1;
      if (left > 1) wait_vm<3 * T::N>();
      else wait_vm<T::N>();
      f32x4 s[T::SUB];
      const uint32_t ka = kf + slot * 2 * T::HALF;
#pragma unroll
      for (int u = 0; u < T::SUB; ++u) {
        s[u] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
          const u32x4 f = *(const __attribute__((address_space(3))) u32x4 *)(uintptr_t)(
              ka + u * 16 * T::ROW + (((4 * n + g4) ^ T::kx(col)) << 4));
          if constexpr (F32) {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              s[u] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(f[e]), __uint_as_float(q[n][e]), s[u], 0, 0, 0);
          } else {
            s[u] = mfma16x16x32(as_bf16x8(f), as_bf16x8(q[n]), s[u]);
            if (a.q_f32) s[u] = mfma16x16x32(as_bf16x8(f), as_bf16x8(ql[n]), s[u]);
          }
        }
      }
      wait_lds();
      const Tile done = cur;
      Tile nn;
      if (left > 2) {
        nn = next(left > 3);
        copy(a.kp, nn, slot, 0);
      }
      // ---- softmax
      const bool part = done.seen < T::KT || done.holes;
      float mt = kMinusInf;
#pragma unroll
      for (int u = 0; u < T::SUB; ++u)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          s[u][r] *= a.c;
          if (part && (16 * u + 4 * g4 + r >= done.seen || (done.holes >> u & 1))) s[u][r] = kMinusInf;
          mt = fmaxf(mt, s[u][r]);
        }
      mt = max4(mt);
      if (__ballot(mt > m)) {
        const float mn = fmaxf(m, mt), ref = mn == kMinusInf ? 0.f : mn, f = exp2f(m - ref);
        m = mn;
        l *= f;
#pragma unroll
        for (int n = 0; n < D / 16; ++n) o[n] *= f;
      }
      const float ref = m == kMinusInf ? 0.f : m;
#pragma unroll
      for (int u = 0; u < T::SUB; ++u)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          s[u][r] = __builtin_amdgcn_exp2f(s[u][r] - ref);
          l += s[u][r];
        }
      // ---- O^T += V^T P^T
      if (left > 2) wait_vm<3 * T::N>();
      else if (left > 1) wait_vm<2 * T::N>();
      else wait_vm<0>();
      if (part) {
#pragma unroll
        for (int n = 0; n < T::N; ++n) {
          const int row = n * T::RPI + lrow;
          if (row >= done.seen || (done.holes >> (row >> 4) & 1))
            *(__attribute__((address_space(3))) u32x4 *)(uintptr_t)(lds_addr(mem) + (2 * slot + 1) * T::HALF + 1024 * n + 16 * lane) = u32x4{0, 0, 0, 0};
        }
        wait_lds();
      }
      const uint32_t va = vf + slot * 2 * T::HALF;
#pragma unroll
      for (int u = 0; u < T::SUB; ++u) {
        if constexpr (F32) {
#pragma unroll
          for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int n = 0; n < D / 64; ++n) {
              const u32x4 f = *(const __attribute__((address_space(3))) u32x4 *)(uintptr_t)(va + r * T::ROW + 256 * n);
#pragma unroll
              for (int e = 0; e < 4; ++e)
                o[4 * n + e] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(f[e]), s[u][r], o[4 * n + e], 0, 0, 0);
            }
        } else {
          uint2 hi, lo;
          split_bf16x2(s[u][0], s[u][1], hi.x, lo.x);
          split_bf16x2(s[u][2], s[u][3], hi.y, lo.y);
#pragma unroll
          for (int n = 0; n < D / 16; ++n) {
            const s16x4 f = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4 *)(uintptr_t)(
                va + u * 16 * T::ROW + (((2 * n + (tr_q >> 1)) ^ T::vx(4 * g4 + tr_j)) << 4)));
            o[n] = __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(f, __builtin_bit_cast(s16x4, hi), o[n], 0, 0, 0);
            o[n] = __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(f, __builtin_bit_cast(s16x4, lo), o[n], 0, 0, 0);
          }
        }
      }
      wait_lds();
      if (left > 2) copy(a.vp, nn, slot, 1);
      // ---- the sequence's end, or the wave's
      const bool ends = done.t == done.n - 1;
      if (ends || left == 1) {
        const bool whole = ends && begun == 0;
        finish(done.b, at - done.t, whole, left > 1 ? first_rec : last_rec, &piece[wave][left > 1 ? 0 : 1]);
      }
      ++at;
      if (--left == 0) break;
      cur = nx;
      nx = nn;
      if (ends) {
        start(cur.b);
        begun = 0;
      }
    }
  }

  // ---- rows of sequences without keys
  for (int b = unit * nw + wave; b < a.B; b += a.units * nw)
    if (tiles_of(uniform_load(a.lens, b)) == 0)
      for (int i = lane; i < gt * D; i += 64) {
        const int64_t to = ((int64_t)b * a.Hq + hq0) * D + i;
        if (a.out_f32) ((float *)a.out)[to] = 0.f;
        else ((uint16_t *)a.out)[to] = 0;
      }
  if (unit >= units) return;

  // ---- the waves' pieces, in order; a sequence's are next to each other
  __syncthreads();
  auto write = [&](int b, int i, float y) {
    const int64_t to = ((int64_t)b * a.Hq + hq0) * D + i;
    if (a.out_f32) ((float *)a.out)[to] = y;
    else ((uint16_t *)a.out)[to] = f32_to_bf16_bits(y);
  };
  const int64_t rec_size = (int64_t)gcap * T::REC;
  Piece out[2];  // sequences that other workgroups have keys of: from before, and onwards
  out[0].b = out[1].b = -1;
  for (int e = 0; e < 2 * nw;) {
    const Piece p = piece[e >> 1][e & 1];
    if (p.b < 0) {
      ++e;
      continue;
    }
    int e1 = e + 1;
    while (e1 < 2 * nw && (piece[e1 >> 1][e1 & 1].b < 0 || piece[e1 >> 1][e1 & 1].b == p.b)) ++e1;
    const bool whole = p.first >= u0 && p.first + p.n <= u1;
    const int which = p.first >= u0;
    float *to = a.part + (((int64_t)hk * a.units + unit) * 2 + which) * rec_size;
    if (!whole) out[which] = p;
    for (int i = threadIdx.x; i < gt * D; i += blockDim.x) {
      const int r = i / D, d = i - r * D;
      auto rec = [&](int x) {
        return (const float *)(lds + (x >> 1) * (T::RING + gcap * T::REC * 4) + ((x & 1) ? 0 : T::RING)) + r * T::REC;
      };
      float M = kMinusInf, L = 0.f, O = 0.f;
      for (int x = e; x < e1; ++x)
        if (piece[x >> 1][x & 1].b >= 0) M = fmaxf(M, rec(x)[D]);
      for (int x = e; x < e1; ++x)
        if (piece[x >> 1][x & 1].b >= 0) {
          const float *const rx = rec(x);
          const float f = rx[D] == kMinusInf ? (rx[D + 1] == 0.f ? 0.f : 1.f) : exp2f(rx[D] - M);
          L += f * rx[D + 1];
          O += f * rx[d];
        }
      if (whole) {
        write(p.b, i, L == 0.f ? 0.f : O / L);
      } else {
        float *const tr = to + r * T::REC;
        __hip_atomic_store(tr + d, O, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        if (d == 0) {
          __hip_atomic_store(tr + D, M, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
          __hip_atomic_store(tr + D + 1, L, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
      }
    }
    e = e1;
  }
  if (out[0].b < 0 && out[1].b < 0) return;
  wait_vm<0>();  // this wave's record stores are done
  __syncthreads();
  int from[2], count[2];
  for (int w = 0; w < 2; ++w) {
    if (out[w].b < 0) continue;
    from[w] = deal.taker(out[w].first);
    count[w] = deal.taker(out[w].first + out[w].n - 1) - from[w] + 1;
    if (threadIdx.x == 0)
      last_one[w] = __hip_atomic_fetch_add(a.counters + (int64_t)hk * a.units + from[w], 1, __ATOMIC_RELAXED,
                                           __HIP_MEMORY_SCOPE_AGENT) == count[w] - 1;
  }
  __syncthreads();
  for (int w = 0; w < 2; ++w) {
    if (out[w].b < 0 || !last_one[w]) continue;
    // records of workgroups from .. from + count - 1: the first's is its second one
    const float *const base = a.part + ((int64_t)hk * a.units + from[w]) * 2 * rec_size;
    auto rec = [&](int c) { return base + (2 * c + (c == 0)) * rec_size; };
    float *const ml = (float *)lds;  // [count][gt][2]
    for (int i = threadIdx.x; i < count[w] * gt; i += blockDim.x) {
      const float *const p = rec(i / gt) + (i % gt) * T::REC + D;
      ml[2 * i] = __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      ml[2 * i + 1] = __hip_atomic_load(p + 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < gt * D; i += blockDim.x) {
      const int r = i / D, d = i - r * D;
      float M = kMinusInf, L = 0.f, O = 0.f;
      for (int c = 0; c < count[w]; ++c) M = fmaxf(M, ml[2 * (c * gt + r)]);
      for (int c0 = 0; c0 < count[w]; c0 += 8) {
        float x[8];
#pragma unroll
        for (int c = 0; c < 8; ++c)
          x[c] = c0 + c < count[w] ? __hip_atomic_load(rec(c0 + c) + r * T::REC + d, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : 0.f;
#pragma unroll
        for (int c = 0; c < 8; ++c)
          if (c0 + c < count[w]) {
            const float mc = ml[2 * ((c0 + c) * gt + r)], lc = ml[2 * ((c0 + c) * gt + r) + 1];
            const float f = mc == kMinusInf ? (lc == 0.f ? 0.f : 1.f) : exp2f(mc - M);
            L += f * lc;
            O += f * x[c];
          }
      }
      write(out[w].b, i, L == 0.f ? 0.f : O / L);
    }
    if (threadIdx.x == 0)
      __hip_atomic_store(a.counters + (int64_t)hk * a.units + from[w], 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
  }
}

#define RXW8_PAGED_DECODE(D, NAME, F)                                                        \
  extern "C" __global__ void __launch_bounds__(64 * kPagedWaves) rxw8_paged_decode_##NAME##_d##D(PagedDecodeArgs a) { \
    paged_decode<D, F>(a);                                                                   \
  }
RXW8_PAGED_DECODE(64, bf16, false)
RXW8_PAGED_DECODE(128, bf16, false)
RXW8_PAGED_DECODE(256, bf16, false)
RXW8_PAGED_DECODE(64, f32, true)
RXW8_PAGED_DECODE(128, f32, true)
RXW8_PAGED_DECODE(256, f32, true)
