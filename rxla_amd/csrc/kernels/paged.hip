// The paged key/value cache: the append that fills its pages and the attention of
// one new token per sequence that reads them.
#include <type_traits>

#include "paged.h"

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

// Any width and alignment: a wave for each (row, kv head), an element a lane (9000 bf16 rows of 8
// heads of 100: 30 us, 1.9 TB/s).
extern "C" __global__ void __launch_bounds__(256) rxw8_paged_append_any(PagedAppendArgs a) {
  const int lane = threadIdx.x & 63;
  const int64_t unit = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (unit >= a.T * a.Hkv) return;
  const int64_t t = unit / a.Hkv;
  const int h = (int)(unit - t * a.Hkv);
  const PagedPlace to = paged_place(a, t);
  if (to.page < 0) return;
  const int64_t src = unit * a.D, dst = ((to.page * a.Hkv + h) * a.ps + to.at) * a.D;
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

// Widths of whole 8 elements at 16-byte boundaries: a wave for each row and `kAppend` x 64
// of its pieces of 8 elements, all heads' in a row, with K's and V's pieces under way before
// the wave looks for its sequence and page. An f32 row is rounded once (RNE) on its way into
// bf16 pages, a bf16 row widened exactly. Bound by memory for prompts (9000 bf16 rows of 8
// heads of 128: 12.7 to 13.8 us, 5.3 to 5.8 TB/s read and written, the cache's part included; f32
// rows into f32 pages 33 us, 4.4 TB/s), by the launch
// and the chain of dependent loads (offsets, start, table) for a step's single rows (3.8 us).
constexpr int kAppend = 2;

template <typename S, typename P>
__device__ __forceinline__ void paged_append(const PagedAppendArgs &a) {
  constexpr int NS = sizeof(S) / 2, NP = sizeof(P) / 2;  // 16-byte words of 8 elements
  const int lane = threadIdx.x & 63, per_head = a.D / 8, pieces = a.Hkv * per_head;
  const int parts = (pieces + 64 * kAppend - 1) / (64 * kAppend);
  const int64_t unit = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6), t = unit / parts;
  const int p0 = (int)(unit - t * parts) * 64 * kAppend + lane;
  if (t >= a.T) return;
  u32x4 k[kAppend][NS], v[kAppend][NS];
#pragma unroll
  for (int n = 0; n < kAppend; ++n)
    if (p0 + 64 * n < pieces) {
      const int64_t at = (t * pieces + p0 + 64 * n) * NS;
#pragma unroll
      for (int i = 0; i < NS; ++i) k[n][i] = ((const u32x4 *)a.k)[at + i], v[n][i] = ((const u32x4 *)a.v)[at + i];
    }
  const PagedPlace to = paged_place(a, t);
  if (to.page < 0) return;
  auto put = [&](void *pages, int64_t at, const u32x4 *x) {
    u32x4 y[NP];
    if constexpr (NS == NP) {
#pragma unroll
      for (int i = 0; i < NP; ++i) y[i] = x[i];
    } else if constexpr (NS == 2) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        y[0][i] = pack_bf16x2(__uint_as_float(x[i / 2][2 * i % 4]), __uint_as_float(x[i / 2][2 * i % 4 + 1]));
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) y[i / 2][2 * i % 4] = x[0][i] << 16, y[i / 2][2 * i % 4 + 1] = x[0][i] & 0xffff0000u;
    }
#pragma unroll
    for (int i = 0; i < NP; ++i) ((u32x4 *)pages)[at + i] = y[i];
  };
#pragma unroll
  for (int n = 0; n < kAppend; ++n) {
    const int p = p0 + 64 * n;
    if (p < pieces) {
      const int h = p / per_head;
      const int64_t at = (((to.page * a.Hkv + h) * a.ps + to.at) * per_head + (p - h * per_head)) * NP;
      put(a.kp, at, k[n]);
      put(a.vp, at, v[n]);
    }
  }
}
extern "C" __global__ void __launch_bounds__(256) rxw8_paged_append(PagedAppendArgs a) {
  if (a.k_f32 && a.p_f32)
    paged_append<float, float>(a);
  else if (a.k_f32)
    paged_append<float, uint16_t>(a);
  else if (a.p_f32)
    paged_append<uint16_t, float>(a);
  else
    paged_append<uint16_t, uint16_t>(a);
}

// Any head width up to 512, any page size: one workgroup of 4 waves per (sequence,
// query head), the waves' chunks of 64 keys in turn, merged in LDS. Bound by its reads of a key a
// lane, element by element (8 sequences of 512 to 8192 keys, 32 / 8 heads: 1.9 ms at a width of 96).
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
  AnyState all;
  if (!any_join(all, st, part, mw, lw)) return;
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
// a sequence's end goes on with the next one. (8 sequences of 512 to 8192 keys, 32 / 8 heads of 128, bf16:
// 24.5 us, 3.9 TB/s; 96 of 1 to 1500: 59.6 us, 3.5 TB/s.)
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
// A sequence inside one wave's piece is written at once. Pieces of a sequence are
// joined in the order of its keys: the waves' in LDS, then, if it passes a
// workgroup's piece, by the last of its workgroups to arrive, over (max, sum, acc)
// records in device memory (at most two a workgroup). Those are stored and copied
// past the dies' own caches, around an arrival counter that the last one sets back to
// zero.
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
  static constexpr int RING = 2 * HALF;           // a wave's K and V
  static constexpr int REC = D + 4;               // floats of a record: acc [D], max, sum
  static __device__ __forceinline__ int kx(int row) { return row & (CH < 16 ? CH - 1 : 15); }
  static __device__ __forceinline__ int vx(int row) { return F32 ? 0 : 2 * (row & (CH < 16 ? 3 : 7)); }
};

// (max, sum, acc) records joined in order: NB of them, number k0 + k with
// get(k, min(k0 + k, count - 1), m, l, o); those from `count` on do not count. o is two
// of a head's dims.
struct Joined {
  float M = kMinusInf, L = 0.f;
  float2 O = float2{0.f, 0.f};
};
__device__ __forceinline__ float record_weight(float m, float l, float M) {
  return m == kMinusInf ? (l == 0.f ? 0.f : 1.f) : __builtin_amdgcn_exp2f(m - M);  // (l NaN: scores were)
}
template <int NB, typename Get>
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
  const int nw = a.waves, col = lane & 15, g4 = lane >> 4;
  const int G = a.Hq / a.Hkv, HT = (G + 15) / 16, heads = a.Hkv * HT, gcap = min(G, 16);
  const int hk = blockIdx.x % heads, unit = blockIdx.x / heads, h = hk / HT, ht = hk - h * HT;
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
  const int units = min(a.units, (total + nw - 1) / nw);
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
    auto copy = [&](const void *pool, const Tile &x, int half) {
      const uint32_t dst = lds_addr(mem) + half * T::HALF;
#pragma unroll
      for (int i = 0; i < T::N; ++i) {
        const int row = i * T::RPI + lrow, sx = half ? T::vx(row) : T::kx(row);
        dma16((const char *)pool + x.off[i * T::RPI / 16], (uint32_t)(row & 15) * T::ROW + ((lch ^ sx) << 4),
              dst + 1024 * i);
      }
    };

    Tile cur;  // that the copies out are of
    // ---- q, O and the softmax of the sequence at hand
    constexpr int NQ = F32 ? D / 16 : D / 32;  // 16-byte pieces of a head's q per lane
    u32x4 q[NQ], ql[F32 ? 1 : NQ], qe[F32 ? 1 : NQ];  // (f32 q over bf16 caches: three parts)
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
              uint32_t x[3];
              split_bf16x2(r[e >> 1][2 * (e & 1)], r[e >> 1][2 * (e & 1) + 1], x);
              q[i][e] = x[0], ql[i][e] = x[1], qe[i][e] = x[2];
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
    auto finish = [&](int seq, int first, int n, bool whole, float *rec, Piece *p) {
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
      if (lane == 0) *p = Piece{seq, first, n};
    };

    // (q is on its way while the first pages are looked up, and in before the copies
    // go out: a wait for it later would be a wait for them)
    start(b);
    cur = next(left > 1);
#pragma unroll
    for (int i = 0; i < NQ; ++i) asm volatile("" : "+v"(q[i]));
    copy(a.kp, cur, 0);
    copy(a.vp, cur, 1);

    // LDS byte addresses of the fragments in tile 0 (the swizzles are XORs below)
    const uint32_t kf = lds_addr(mem) + col * T::ROW;
    const int tr_j = col >> 2, tr_q = col & 3;
    const uint32_t vf = lds_addr(mem) + T::HALF + (F32 ? 4 * g4 * T::ROW + 16 * col : (4 * g4 + tr_j) * T::ROW + 8 * (tr_q & 1));
    int begun = cur.t;  // the tile at which this wave began the sequence
    for (;;) {
      wait_vm<T::N>();  // (copies complete in order: all but this tile's V)
      f32x4 s[T::SUB];
#pragma unroll
      for (int u = 0; u < T::SUB; ++u) {
        constexpr int NA = F32 ? 4 : 2;  // sums in turn: no product waits for the one before
        f32x4 acc[NA];
#pragma unroll
        for (int n = 0; n < NA; ++n) acc[n] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
          const u32x4 f = *(const __attribute__((address_space(3))) u32x4 *)(uintptr_t)(
              kf + u * 16 * T::ROW + (((4 * n + g4) ^ T::kx(col)) << 4));
          if constexpr (F32) {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              acc[e] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(f[e]), __uint_as_float(q[n][e]), acc[e], 0, 0, 0);
          } else {
            acc[n & 1] = mfma16x16x32(as_bf16x8(f), as_bf16x8(q[n]), acc[n & 1]);
            if (a.q_f32) {
              acc[~n & 1] = mfma16x16x32(as_bf16x8(f), as_bf16x8(ql[n]), acc[~n & 1]);
              acc[n & 1] = mfma16x16x32(as_bf16x8(f), as_bf16x8(qe[n]), acc[n & 1]);
            }
          }
        }
        s[u] = acc[0] + acc[1];
        if constexpr (F32) s[u] += acc[2] + acc[3];
      }
      wait_lds();
      const Tile done = cur;
      if (left > 1) {
        cur = next(left > 2);
        copy(a.kp, cur, 0);
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
      if (left > 1) wait_vm<T::N>();
      else wait_vm<0>();
      if (part) {
#pragma unroll
        for (int n = 0; n < T::N; ++n) {
          const int row = n * T::RPI + lrow;
          if (row >= done.seen || (done.holes >> (row >> 4) & 1))
            *(__attribute__((address_space(3))) u32x4 *)(uintptr_t)(lds_addr(mem) + T::HALF + 1024 * n + 16 * lane) = u32x4{0, 0, 0, 0};
        }
        wait_lds();
      }
#pragma unroll
      for (int u = 0; u < T::SUB; ++u) {
        if constexpr (F32) {
#pragma unroll
          for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int n = 0; n < D / 64; ++n) {
              const u32x4 f = *(const __attribute__((address_space(3))) u32x4 *)(uintptr_t)(vf + r * T::ROW + 256 * n);
#pragma unroll
              for (int e = 0; e < 4; ++e)
                o[4 * n + e] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(f[e]), s[u][r], o[4 * n + e], 0, 0, 0);
            }
        } else {
          uint32_t p01[3], p23[3];
          if (a.out_f32) {
            split_bf16x2<true>(s[u][0], s[u][1], p01);
            split_bf16x2<true>(s[u][2], s[u][3], p23);
          } else {
            uint32_t x[2], y[2];
            split_bf16x2<true>(s[u][0], s[u][1], x);
            split_bf16x2<true>(s[u][2], s[u][3], y);
            p01[0] = x[0], p01[1] = x[1], p23[0] = y[0], p23[1] = y[1];
          }
#pragma unroll
          for (int n = 0; n < D / 16; ++n) {
            const s16x4 f = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4 *)(uintptr_t)(
                vf + u * 16 * T::ROW + (((2 * n + (tr_q >> 1)) ^ T::vx(4 * g4 + tr_j)) << 4)));
            auto add = [&](int k) {
              o[n] = __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(f, __builtin_bit_cast(s16x4, (uint2{p01[k], p23[k]})), o[n], 0, 0, 0);
            };
            add(0);
            add(1);
            if (a.out_f32) add(2);
          }
        }
      }
      wait_lds();
      if (left > 1) copy(a.vp, cur, 1);
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
        // (waited for here, with the copies ahead of it: a wait at the loop's top
        // would drain the ring at every tile)
#pragma unroll
        for (int n = 0; n < NQ; ++n) asm volatile("" : "+v"(q[n]));
        begun = 0;
      }
    }
  }

  // ---- rows of sequences without keys
  for (int b = unit * kPagedWaves + wave; b < a.B; b += a.units * kPagedWaves)
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
    const int64_t to = ((int64_t)b * a.Hq + hq0) * D + 2 * i;
    const float inv = j.L == 0.f ? 0.f : 1.0f / j.L;
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
    float *const to = a.part + (((int64_t)onwards * heads + hk) * a.units + unit) * rec_size;
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
      for (int k0 = 0; k0 < n; k0 += 4) join<4>(j, k0, n, get);
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
      last_one[w] = __hip_atomic_fetch_add(a.counters + (int64_t)hk * a.units + from[w], 1, __ATOMIC_RELAXED,
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
    const int64_t on = ((int64_t)heads + hk) * a.units + from[w], past = (int64_t)hk * a.units + from[w];
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
            dma16_coherent(a.part + (c0 + c == 0 ? on : past + c0 + c) * rec_size + 256 * (y - c * pieces), 16 * lane,
                           lds_addr(lds) + 1024 * y);
          }
          wait_vm<0>();
          __syncthreads();
        }
#pragma unroll 1
        for (int k0 = 0; k0 < n; k0 += 4)
          join<4>(j, k0, n, [&](int, int c, float &m, float &l, float2 &o) {
            const float *const rec = (const float *)lds + c * rec_size + r * T::REC;
            const float2 ml = *(const float2 *)(rec + D);
            m = ml.x, l = ml.y, o = *(const float2 *)(rec + d);
          });
      }
      if (i0 + (int)threadIdx.x < pairs) write(p.b, i, j);
    }
    if (threadIdx.x == 0)
      __hip_atomic_store(a.counters + (int64_t)hk * a.units + from[w], 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
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
