// Causal attention of packed prompts: sequence b owns rows offsets[b] ..
// offsets[b + 1] - 1 of q [T, Hq, D] and of k, v [T, Hkv, D], and row t of it sees
// rows offsets[b] .. t. Offsets are read on the device and clamped into [0, T].
#include <type_traits>

#include "attn_any.h"

struct PackedArgs {
  const void *q;               // [T, Hq, D] f32 | bf16
  const uint16_t *k, *v;       // [T, Hkv, D] bf16
  const int32_t *offsets;      // [B + 1]
  void *out;                   // [T, Hq, D] f32 | bf16
  int64_t T;
  int B, Hq, Hkv, D;
  float c;                     // scale log2 e
  int q_f32, out_f32;
  int fill;                    // rows outside every sequence: zeros (else left as they are)
  int heads;                   // query heads of a workgroup (1, 2 or 4; divides Hq / Hkv)
};

// Any head width up to 512: one wave per (row, query head).
extern "C" __global__ void __launch_bounds__(256) rxw8_packed_prefill_any(PackedArgs a) {
  __shared__ float qs[4][RXW8_ATTN_ANY_MAX_D];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t unit = (int64_t)blockIdx.x * 4 + wave;
  if (unit >= a.T * a.Hq) return;  // whole waves only; no barriers below
  const int64_t t = unit / a.Hq;
  const int hq = (int)(unit - t * a.Hq), h = hq / (a.Hq / a.Hkv);
  const int b = any_sequence(a.offsets, a.B, t);
  const int64_t start = b < 0 ? 0 : a.offsets[b] < 0 ? 0 : a.offsets[b];
  AnyState st;
  if (b < 0 || t >= a.offsets[b + 1]) {
    if (a.fill) any_store(st, a.out, unit * a.D, a.D, a.out_f32);
    return;
  }
  for (int i = lane; i < a.D; i += 64) qs[wave][i] = any_load(a.q, unit * a.D + i, a.q_f32);
  __builtin_amdgcn_wave_barrier();
  any_walk(st, qs[wave], a.k, a.v, false, a.D, start, t + 1, 1, a.c,
           [&](int64_t j) { return (j * a.Hkv + h) * a.D; });
  any_store(st, a.out, unit * a.D, a.D, a.out_f32);
}

// Rows outside every sequence of a new output
extern "C" __global__ void __launch_bounds__(256) rxw8_packed_fill(PackedArgs a) {
  const int64_t first = min((int64_t)max(a.offsets[0], 0), a.T), end = min((int64_t)max(a.offsets[a.B], 0), a.T);
  const int64_t row = (int64_t)a.Hq * a.D, n = a.T * row;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
    const int64_t at = i < first * row ? i : end * row + (i - first * row);
    if (at >= n) return;
    if (a.out_f32) ((float *)a.out)[at] = 0.f;
    else ((uint16_t *)a.out)[at] = 0;
  }
}

// ---- head widths 64, 128, 256 on the matrix cores ------------------------------------
//
// A workgroup of 4 waves, one to a SIMD, takes 4 x 32 QT rows: HW query heads of one kv
// head times 4 / HW groups of 32 QT rows of one sequence. It walks the sequence's keys
// in steps of 32, whose K and V rows it copies by LDS DMA into rings of 4 (row-major,
// 16-byte chunks XOR-swizzled by row), two to three steps ahead, a barrier a step.
// Per wave and step, on 32x32x16 bf16 products:
//   S^T = K q^T     lane (l % 32) = row, keys 8 (r / 4) + 4 (l / 32) + r % 4 in register r;
//   p = exp2(c s - m), m the row's reference;
//   O^T += V^T P^T  P straight from the score registers, V^T by transposing LDS reads
//                   in the same order of keys.
// In a step the products are those of S one step ahead and of O one step behind, so
// none of them waits for the softmax between: every LDS read is followed by its
// products, and these by a share of the softmax, in that order (a barrier to the
// scheduler keeps it). bf16 q and outputs of 128 run QT = 1 with two workgroups to a CU,
// whose prologues and stores pass under the other's products: 12 prompts of 64 to 2000 rows, 32 / 8
// heads, take 114 us so and 126 with QT = 2 on a CU alone, though there the LDS reads take half
// the time of the products (one fragment of K or V serves 32 QT rows); of 5000 and 7000 rows, 64 /
// 8 heads, 1137 (1.07 PFLOP/s) and 1166. At 64 QT = 2 leaves registers for two workgroups all the
// same (78 us for 4 of 2048 rows, 82 with QT = 1 and four). At 256 O alone is 128 registers: QT = 1
// and one workgroup. f32 ones split q and P in their three bf16 parts (exact products, f32 sums)
// and run QT = 1, from 128 on a CU alone (two spill: 480 us for 4 of 2048 rows, 32 / 8 heads of
// 128, 382 so: 0.36 PFLOP/s, each product counted once). Behind a bf16 output the weights are one
// bf16 part, rounded by 2^-8 at most, as the output itself is, their sum taken before that: a second
// part would add half of all products again. The outputs of the two sets of prompts above are 2.0e-3
// and 2.1e-3 of their norm off the 64-bit ones, 1.6e-3 where the output alone is rounded.
//
// m is the maximum of the row's first 32 keys (0 where these are at -inf) and does not move:
// weights may grow past 1 as far as f32 and bf16 go (2^127), and O / l is the same. Rows whose l
// or O leaves that range, whose l shows that weights were lost below it, or that meet values that
// are no numbers (a key that a row does not see has weight 0, and 0 times an infinity is none),
// are done again, key by key, by the wave alone: right, but slow (the 12 prompts above with an
// infinite value in the 41st row of one, which all its rows after that see: 2.2 ms).
// (the lambdas below hold the wave's registers: they have to be part of the kernel)
#define RXW8_INLINE __attribute__((always_inline))

namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ f32x16 mfma32(u32x4 a, u32x4 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(as_bf16x8(a), as_bf16x8(b), c, 0, 0, 0);
}
__device__ __forceinline__ float max_xor32(float v) {
  const uint2 p = pair_xor32(v);
  return fmaxf(__uint_as_float(p.x), __uint_as_float(p.y));
}
// Sum over the 64 lanes, in every lane
__device__ __forceinline__ int sum64(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);  // row_shr 1, 2, 4, 8
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);  // row_bcast 15, 31
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);
  return __builtin_amdgcn_readlane(v, 63);
}

// f(0), f(1), .., f(N - 1) with constants for arguments
template <int N, int I = 0, typename F>
__device__ __forceinline__ void unrolled(F f) {
  if constexpr (I < N) {
    f(std::integral_constant<int, I>{});
    unrolled<N, I + 1>(f);
  }
}

constexpr int kStep = 32;  // keys
// The fragments' LDS addresses are formed by XOR within a row: dynamic LDS begins at a multiple of
// the longest, whatever static LDS comes before it
constexpr int kLdsAlign = 512;
// A row's least sum of weights: with 2^20 keys, weights down to 2^-24 of the largest and the
// third bf16 parts of these (2^-16 below) are normal numbers
constexpr float kLeastSum = 0x1p-60f;

// The row tile of the given rank, those that see the most keys first: its index in its
// sequence, whose first row and length these are (-1: there are not that many)
__device__ __forceinline__ int row_tile(const PackedArgs &a, int ROWS, int rank, int64_t &first, int &len) {
  const int lane = threadIdx.x & 63;
  auto bounds = [&](int b, int64_t &s) {
    s = min((int64_t)max(a.offsets[b], 0), a.T);
    const int64_t e = min((int64_t)max(a.offsets[b + 1], 0), a.T);
    return (int)max(e - s, (int64_t)0);
  };
  for (int b0 = 0; b0 < a.B; b0 += 64) {
    int64_t s = 0;
    const int n = b0 + lane < a.B ? bounds(b0 + lane, s) : 0, tiles = (n + ROWS - 1) / ROWS;
    const int all = sum64(tiles);
    if (rank >= all) {  // (of another 64 sequences)
      rank -= all;
      continue;
    }
    // tiles of index x and above, over the sequences: more than rank for x = lo, not for hi
    int lo = 0, hi = (int)min((a.T + ROWS - 1) / ROWS, (int64_t)all), above = 0;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1, c = sum64(max(tiles - mid, 0));
      if (c > rank) lo = mid;
      else hi = mid;
    }
    above = sum64(max(tiles - lo - 1, 0));
    const unsigned long long have = __ballot(tiles > lo);
    const bool me = tiles > lo && __popcll(have & ((1ull << lane) - 1)) == rank - above;
    const int src = __builtin_ctzll(__ballot(me));
    len = __builtin_amdgcn_readlane(n, src);
    first = (uint32_t)__builtin_amdgcn_readlane((int)s, src);  // (T is below 2^31)
    return lo;
  }
  return -1;
}

}  // namespace

// Rows row, row + step, .. below end of a sequence again, key by key, where some did not
// come out as numbers
__device__ __forceinline__ void rows_again(const PackedArgs &a, int D, float *qs, int64_t first, int row, int end, int step, int hq) {
  const int lane = threadIdx.x & 63, kvh = hq / (a.Hq / a.Hkv);
  __builtin_amdgcn_wave_barrier();
#pragma unroll 1
  for (; row < end; row += step) {
    const int64_t at = ((first + row) * a.Hq + hq) * D;
    for (int i = lane; i < D; i += 64) qs[i] = any_load(a.q, at + i, a.q_f32);
    __builtin_amdgcn_wave_barrier();
    AnyState st;
    any_walk(st, qs, a.k, a.v, false, D, first, first + row + 1, 1, a.c,
             [&](int64_t j) { return (j * a.Hkv + kvh) * D; });
    any_store(st, a.out, at, D, a.out_f32);
  }
}

// PQ, P: bf16 parts of q and of the weights (1 or 3). QL: the third parts of q stay in LDS,
// where the registers do not hold them (D = 256: O takes 128, two parts of q as many), and
// the rings have three places: V is then copied a step later.
template <int D, int QT, int PQ, int P, bool QL = PQ == 3 && D == 256>
__device__ void packed_prefill(const PackedArgs &a) {
  extern __shared__ __attribute__((aligned(kLdsAlign))) uint16_t lds[];  // [RING][32][D] K, the same V; q's third parts
  constexpr int ROWB = 2 * D, CH = D / 8, TILE = kStep * ROWB, NI = TILE / 4096;  // copies of a wave per tile
  static_assert(ROWB <= kLdsAlign, "rows begin at multiples of their size");
  constexpr int RING = QL ? 3 : 4, QR = QL ? PQ - 1 : PQ;                         // parts of q in registers
  constexpr int NK = D / 16, ND = D / 32, WR = 32 * QT;                            // WR: rows of a wave
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 31, hf = lane >> 5;
  const int G = a.Hq / a.Hkv, HW = a.heads, RG = 4 / HW, ROWS = WR * RG, HP = G / HW, per = a.Hkv * HP;
  const int kvh = blockIdx.x % a.Hkv, hp = blockIdx.x / a.Hkv % HP;
  const int rank = blockIdx.x / per;

  int64_t first = 0;
  int len = 0;
  const int tile = row_tile(a, ROWS, rank, first, len);
  if (tile < 0) return;

  const int head = wave % HW, r0 = tile * ROWS + wave / HW * WR;  // the wave's first row
  const int hq = kvh * G + hp * HW + head;
  const int last_row = min(tile * ROWS + ROWS, len);              // past the workgroup's rows
  const int steps = (last_row + kStep - 1) / kStep;
  const int full = r0 / kStep;                                     // steps without a mask
  const int mine = r0 < len ? (min(r0 + WR, len) + kStep - 1) / kStep : 0;

  // ---- copies: instruction i of a wave takes rows RPI (4 i + wave) .. of a step's 32
  constexpr int RPI = 1024 / ROWB;
  auto kx = [](int row) { return row & (CH < 16 ? CH - 1 : 15); };
  auto vx = [](int row) { return 2 * (row & (CH < 16 ? 3 : 7)); };
  const uint32_t stride = (uint32_t)a.Hkv * ROWB;
  const char *const kbase = (const char *)a.k + (first * a.Hkv + kvh) * ROWB;
  const char *const vbase = (const char *)a.v + (first * a.Hkv + kvh) * ROWB;
  auto place = [](int step) RXW8_INLINE { return RING == 4 ? step & 3 : (int)((unsigned)step % RING); };
  auto copy = [&](const char *base, int step, bool is_v) RXW8_INLINE {
    const uint32_t dst = lds_addr(lds) + ((is_v ? RING : 0) + place(step)) * TILE;
    const char *const from = base + (int64_t)step * kStep * stride;
    const int most = len - 1 - step * kStep;  // (rows past the sequence repeat its last)
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int row = RPI * (4 * i + wave) + lane / CH, x = is_v ? vx(row) : kx(row);
      dma16(from, (uint32_t)min(row, most) * stride + (((lane % CH) ^ x) << 4), dst + 1024 * (4 * i + wave));
    }
  };
  copy(kbase, 0, false);
  if (QL && steps > 1) copy(kbase, 1, false);
  copy(vbase, 0, true);
  if (!QL && steps > 1) {
    copy(kbase, 1, false);
    copy(vbase, 1, true);
  }
  if (steps > 2) copy(kbase, 2, false);

  // ---- q
  u32x4 q[QT][NK][QR];
  u32x4 *const q_low = (u32x4 *)((char *)lds + 2 * RING * TILE) + wave * NK * 64 + lane;  // [NK][64] (QL)
  constexpr int NL = QL ? 8 : NK;  // fragments asked for at a time
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    const int64_t at = ((first + min(r0 + 32 * t + col, len - 1)) * a.Hq + hq) * D + 8 * hf;
    unrolled<NK / NL>([&](auto g) RXW8_INLINE {
#pragma unroll
      for (int n = g * NL; n < (g + 1) * NL; ++n) {
        if constexpr (PQ == 3) {
          const f32x4 x = *(const f32x4 *)((const float *)a.q + at + 16 * n), y = *(const f32x4 *)((const float *)a.q + at + 16 * n + 4);
          u32x4 low;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            uint32_t part[3];
            split_bf16x2(e < 2 ? x[2 * e] : y[2 * e - 4], e < 2 ? x[2 * e + 1] : y[2 * e - 3], part);
#pragma unroll
            for (int p = 0; p < QR; ++p) q[t][n][p][e] = part[p];
            low[e] = part[2];
          }
          if constexpr (QL) q_low[64 * n] = low;
        } else {
          q[t][n][0] = *(const u32x4 *)((const uint16_t *)a.q + at + 16 * n);
        }
      }
      if constexpr (QL) {
#pragma unroll
        for (int n = g * NL; n < (g + 1) * NL; ++n)
#pragma unroll
          for (int p = 0; p < QR; ++p) asm volatile("" : "+v"(q[t][n][p]));  // (here: one group's rows at a time)
      }
    });
  }
  // ---- state
  f32x16 o[QT][ND], sa[QT], sb[QT];
  u32x4 pa[QT][2][P], pb[QT][2][P];
  float m[QT], l[QT];
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    m[t] = 0.f, l[t] = 0.f;
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int r = 0; r < 16; ++r) o[t][d][r] = 0.f;
  }
  const float c = a.c;
  int h = 0;
  // Before step h every wave's copies of K up to h + 1 and V up to h (QL: h - 1) are in; the
  // slots of K h - 1 (QL: h) and V h - 2 are free.
  auto begin = [&](bool k = true) RXW8_INLINE {
    __builtin_amdgcn_sched_barrier(0);
    if (h + 2 < steps) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(2 * NI) : "memory");
    else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    if (h + (QL ? 1 : 2) < steps) copy(vbase, h + (QL ? 1 : 2), true);
    if (k && h + 3 < steps) copy(kbase, h + 3, false);
    __builtin_amdgcn_sched_barrier(0);
  };
  auto third = [&]() RXW8_INLINE {  // K of step 3, into the place of step 0's, which every wave has read
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    if (steps > 3) copy(kbase, 3, false);
    __builtin_amdgcn_sched_barrier(0);
  };
  // LDS byte addresses of the fragments: one XOR from a lane's base in the step's slot
  // (chunk 2 n + hf of K row col; chunks 4 d + .. of V rows 4 hf + j, 8 rows apart two reads)
  const uint32_t k0 = lds_addr(lds) + col * ROWB + ((hf ^ kx(col)) << 4);
  const int tr_j = (lane & 15) >> 2, tr_q = lane & 3;
  const uint32_t v0 = lds_addr(lds) + RING * TILE + (4 * hf + tr_j) * ROWB + 8 * (tr_q & 1) +
                      (((2 * ((lane >> 4) & 1) + (tr_q >> 1)) ^ vx(4 * hf + tr_j)) << 4);
  auto slot = [&](uint32_t base, int step) RXW8_INLINE {
    uint32_t at = base + place(step) * TILE;
    asm("" : "+v"(at));  // (the XORs stay where they are used, not in registers)
    return at;
  };
  auto k_frag = [&](uint32_t base, int n) RXW8_INLINE {
    return *(const __attribute__((address_space(3))) u32x4 *)(uintptr_t)(base ^ (n << 5));
  };
  auto v_frag = [&](uint32_t base, int n) RXW8_INLINE {
    u32x4 f;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4 *)(uintptr_t)(
          (base ^ (n % ND << 6)) + (16 * (n / ND) + 8 * e) * ROWB));
      const uint2 u = __builtin_bit_cast(uint2, x);
      f[2 * e] = u.x, f[2 * e + 1] = u.y;
    }
    return f;
  };
  // The products of a fragment, after(i) behind the i-th (QT PQ of K's n-th, QT P of V's)
  auto qk = [&](f32x16 (&s)[QT], auto n, u32x4 f, u32x4 low, auto after) RXW8_INLINE {
    unrolled<QT * PQ>([&](auto i) RXW8_INLINE {
      constexpr int t = i % QT, x = i / QT;
      if constexpr (n == 0 && x == 0) {
        f32x16 zero;
#pragma unroll
        for (int r = 0; r < 16; ++r) zero[r] = 0.f;
        s[t] = mfma32(f, q[t][n][x], zero);
      } else {
        s[t] = mfma32(f, QL && x == PQ - 1 ? low : q[t][n][x < QR ? x : 0], s[t]);
      }
      after(i);
    });
  };
  auto pv = [&](u32x4 (&p)[QT][2][P], auto n, u32x4 f, auto after) RXW8_INLINE {
    unrolled<QT * P>([&](auto i) RXW8_INLINE {
      constexpr int t = i % QT, x = i / QT, ks = n / ND, d = n % ND;
      o[t][d] = mfma32(f, p[t][ks][x], o[t][d]);
      after(i);
    });
  };
  const auto nothing = [](auto) {};
  // keys that the rows do not see
  auto mask = [&](f32x16 (&s)[QT]) RXW8_INLINE {
    const int rel = r0 + col - h * kStep - 4 * hf;  // a row of tile 0's last key, counted from the lane's first
#pragma unroll
    for (int t = 0; t < QT; ++t)
#pragma unroll
      for (int r = 0; r < 16; ++r)
        if (8 * (r >> 2) + (r & 3) > rel + 32 * t) s[t][r] = kMinusInf;
  };
  // The softmax of a step in shares, some behind each product: two weights at a time, each
  // of which waits for nothing that the one before it has just asked for. Pair g of a
  // lane's 8 QT: exponentials, sum and bf16 parts.
  constexpr int ITEMS = P == 1 ? 2 : 5;  // of a pair
  float w0 = 0.f, w1 = 0.f, was0 = 0.f, was1 = 0.f;
  uint32_t part = 0;
  auto item = [&](f32x16 (&s)[QT], u32x4 (&p)[QT][2][P], auto i) RXW8_INLINE {
    constexpr int g = i / ITEMS, k = i % ITEMS, t = g >> 3, r = 2 * (g & 7), ks = r >> 3, at = (r >> 1) & 3;
    // (formed here: the compiler would sink the exponentials to their use, a step later)
    auto weigh = [&](int e) RXW8_INLINE {
      float w = __builtin_amdgcn_exp2f(fmaf(s[t][r + e], c, -m[t]));
      asm volatile("" : "+v"(w));
      return w;
    };
    auto keep = [&](int tt, int kk, int aa, int x, uint32_t v) RXW8_INLINE {
      asm volatile("" : "+v"(v));
      p[tt][kk][x][aa] = v;
    };
    if constexpr (P == 1) {
      constexpr int gp = g - 1, tp = gp >> 3, rp = 2 * (gp & 7);  // the pair before
      if constexpr (k == 0) {
        was0 = w0, was1 = w1;
        w0 = weigh(0);
        if constexpr (g > 0) l[tp] += was0;
      } else {
        w1 = weigh(1);
        if constexpr (g > 0) {
          l[tp] += was1;
          asm volatile("" : "+v"(l[tp]));
          keep(tp, rp >> 3, (rp >> 1) & 3, 0, pack_bf16x2(was0, was1));
        }
      }
    } else {
      if constexpr (k == 0) w0 = weigh(0);
      if constexpr (k == 1) w1 = weigh(1);
      if constexpr (k == 2 || k == 3) {
        if constexpr (k == 2) {
          l[t] += w0 + w1;
          asm volatile("" : "+v"(l[t]));
        }
        const uint32_t x = cut_weight(w0), y = cut_weight(w1);
        keep(t, ks, at, k - 2, (x >> 16) | y);
        w0 -= __uint_as_float(x), w1 -= __uint_as_float(y);
      }
      if constexpr (k == 4) keep(t, ks, at, 2 % P, pack_bf16x2(w0, w1));
    }
  };
  auto last_item = [&](u32x4 (&p)[QT][2][P]) RXW8_INLINE {
    if constexpr (P == 1) {
      l[QT - 1] += w0 + w1;
      uint32_t v = pack_bf16x2(w0, w1);
      asm volatile("" : "+v"(v), "+v"(l[QT - 1]));
      p[QT - 1][1][0][3] = v;
    }
  };
  // Step h of the pipeline: S of step h + 1 into sn (with_qk), O of step h - 1 from p
  // (with_pv), and between them the weights of step h, from s to pn
  constexpr int AHEAD = D == 256 && P == 3 ? 2 : 4;  // fragments asked for ahead, by registers
  auto body = [&](auto with_pv, auto with_qk, f32x16 (&s)[QT], f32x16 (&sn)[QT], u32x4 (&p)[QT][2][P], u32x4 (&pn)[QT][2][P]) RXW8_INLINE {
    constexpr bool PV = decltype(with_pv)::value, QK = decltype(with_qk)::value;
    // fragments, products and shares of the softmax
    constexpr int NF = (QK ? NK : 0) + (PV ? 2 * ND : 0), NM = QT * ((QK ? PQ * NK : 0) + (PV ? P * 2 * ND : 0)), NE = 8 * QT * ITEMS;
    static_assert(NK == 2 * ND, "K and V take turns");
    const uint32_t ks = slot(k0, h + 1), vs = slot(v0, h - 1);
    u32x4 fr[AHEAD + 1], lows[QL ? AHEAD + 1 : 1];
    auto read = [&](auto n) RXW8_INLINE {
      constexpr bool k = QK && (!PV || n % 2 == 0);
      constexpr int at = QK && PV ? n / 2 : n;
      fr[n % (AHEAD + 1)] = k ? k_frag(ks, at) : v_frag(vs, at);
      if constexpr (QL && k) lows[n % (AHEAD + 1)] = q_low[64 * at];
    };
    unrolled<AHEAD>(read);
    unrolled<NF>([&](auto n) RXW8_INLINE {
      constexpr bool k = QK && (!PV || n % 2 == 0);
      constexpr std::integral_constant<int, QK && PV ? n / 2 : n> at{};
      constexpr int before = QT * (QK && PV ? (n + 1) / 2 * PQ + n / 2 * P : QK ? n * PQ : n * P);  // products
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (n + AHEAD < NF) read(std::integral_constant<int, n + AHEAD>{});
      const u32x4 f = fr[n % (AHEAD + 1)];
      auto share = [&](auto i) RXW8_INLINE {
        constexpr int e0 = (before + i) * NE / NM, e1 = (before + i + 1) * NE / NM;
        unrolled<e1 - e0>([&](auto e) RXW8_INLINE { item(s, pn, std::integral_constant<int, e0 + e>{}); });
        __builtin_amdgcn_sched_barrier(0);
      };
      if constexpr (k) qk(sn, at, f, lows[QL ? n % (AHEAD + 1) : 0], share);
      else pv(p, at, f, share);
    });
    last_item(pn);
    __builtin_amdgcn_sched_barrier(0);
  };
  auto finish = [&](u32x4 (&p)[QT][2][P]) RXW8_INLINE {  // O of the last step
    begin();
    const uint32_t vs = slot(v0, h - 1);
    unrolled<2 * ND>([&](auto n) RXW8_INLINE { pv(p, n, v_frag(vs, n), nothing); });
    ++h;
  };

  // Every wave goes through steps + 1 barriers (QL: one more behind the first). (The loop holds two steps, for the two
  // sets of registers, and nothing else: with the mask's or the end's branches in it the
  // allocator moves O about.)
  constexpr std::true_type yes{};
  constexpr std::false_type no{};
  if (mine > 0) {
    begin(!QL);
    const uint32_t ks = slot(k0, 0);
    unrolled<NK>([&](auto n) RXW8_INLINE { qk(sa, n, k_frag(ks, n), QL ? q_low[64 * n] : u32x4{}, nothing); });
    if constexpr (QL) third();
    if (full == 0) mask(sa);
#pragma unroll
    for (int t = 0; t < QT; ++t) {  // the reference: step 0's maximum
      float mx = kMinusInf;
#pragma unroll
      for (int r = 0; r < 16; ++r) mx = fmaxf(mx, sa[t][r]);
      mx = max_xor32(mx) * c;
      m[t] = mx == kMinusInf ? 0.f : mx;
    }
    body(no, yes, sa, sb, pb, pa);
    for (h = 1; h + 1 < full;) {
      begin();
      body(yes, yes, sb, sa, pa, pb);
      ++h;
      begin();
      body(yes, yes, sa, sb, pb, pa);
      ++h;
    }
    // S of step h in sb, P of the one before in pa
    bool swapped = false;  // (sa and pb instead)
    if (h < full) {
      begin();
      body(yes, yes, sb, sa, pa, pb);
      ++h;
      if constexpr (QT == 2) {  // (here always, where full > 0: it is even)
        begin();
        mask(sa);
        body(yes, yes, sa, sb, pb, pa);
        ++h;
      } else {
        begin();
        mask(sa);
        body(yes, no, sa, sb, pb, pa);
        ++h;
        finish(pa);
        swapped = true;
      }
    }
    if (!swapped) {
      if (h < mine) {
        begin();
        mask(sb);
        body(yes, no, sb, sa, pa, pb);
        ++h;
        finish(pb);
      } else {
        finish(pa);
      }
    }
  }
  if (QL && h == 0) {
    begin(false);
    third();
    ++h;
  }
  for (; h <= steps; ++h) begin();
  __syncthreads();  // (the rings are read)
  if (mine == 0) return;

  // ---- rows out, turned in LDS: 16 bytes of one row a lane
  auto store = [&](auto f32_out) RXW8_INLINE {
    constexpr bool F = decltype(f32_out)::value;
    constexpr int OB = D * (F ? 4 : 2), OC = OB / 16, RPS = 1024 / OB;  // bytes and pieces of a row, rows a store
    const uint32_t mem = lds_addr(lds) + wave * WR * OB;
    auto ox = [](int row) { return row & (OC < 16 ? OC - 1 : 15); };
    float odd = 0.f;  // 0 times a number is 0
#pragma unroll
    for (int t = 0; t < QT; ++t) {
      const float sum = sum_xor32(l[t]), inv = sum == 0.f ? 0.f : 1.0f / sum;
      odd = sum < kLeastSum ? 1.f : fmaf(sum, 0.f, odd);
      const uint32_t row = mem + (32 * t + col) * OB;
#pragma unroll
      for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          f32x4 y;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            y[e] = o[t][d][4 * x + e];
            odd = fmaf(y[e], 0.f, odd);
            y[e] *= inv;
          }
          if constexpr (F)
            *(__attribute__((address_space(3))) f32x4 *)(uintptr_t)(row + (((8 * d + 2 * x + hf) ^ ox(col)) << 4)) = y;
          else
            *(__attribute__((address_space(3))) u32x2 *)(uintptr_t)(row + (((4 * d + x) ^ ox(col)) << 4) + 8 * hf) =
                u32x2{pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3])};
        }
    }
    if (__ballot(odd != 0.f)) return false;
    const int piece = lane % OC;
#pragma unroll 4
    for (int i = 0; i < WR / RPS; ++i) {
      const int row = i * RPS + lane / OC;
      const u32x4 y = *(const __attribute__((address_space(3))) u32x4 *)(uintptr_t)(mem + row * OB + ((piece ^ ox(row)) << 4));
      if (r0 + row < len) *(u32x4 *)((char *)a.out + ((first + r0 + row) * a.Hq + hq) * OB + 16 * piece) = y;
    }
    return true;
  };
  if (P == 3 && a.out_f32 ? store(yes) : store(no)) return;

  // (q in this wave's own rows' place: the others may still be turning theirs)
  float *const qs = (float *)((char *)lds + wave * WR * D * (P == 3 && a.out_f32 ? 4 : 2));
  rows_again(a, D, qs, first, r0, min(r0 + WR, len), 1, hq);
}

#define RXW8_PACKED_PREFILL(D, QT, PQ, P, W, NAME)                                                   \
  extern "C" __global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(W, W)))       \
      rxw8_packed_prefill_##NAME##_d##D(PackedArgs a) {                                              \
    packed_prefill<D, QT, PQ, P>(a);                                                                 \
  }
// q and output bf16; q bf16, output f32; q f32
RXW8_PACKED_PREFILL(64, 2, 1, 1, 2, bf16)
RXW8_PACKED_PREFILL(128, 1, 1, 1, 2, bf16)
RXW8_PACKED_PREFILL(256, 1, 1, 1, 1, bf16)
RXW8_PACKED_PREFILL(64, 1, 1, 3, 2, bf16_f32)
RXW8_PACKED_PREFILL(128, 1, 1, 3, 1, bf16_f32)
RXW8_PACKED_PREFILL(256, 1, 1, 3, 1, bf16_f32)
RXW8_PACKED_PREFILL(64, 1, 3, 3, 2, f32)
RXW8_PACKED_PREFILL(128, 1, 3, 3, 1, f32)
RXW8_PACKED_PREFILL(256, 1, 3, 3, 1, f32)

// ---- few rows: the waves share the keys -----------------------------------------------
//
// Where the tiles above would leave CUs idle, a workgroup takes 32 rows of one query head
// and each of its 4 waves every fourth step of 32 keys: up to 8 times as many workgroups,
// each a quarter as long (a half of that again in rows). A wave goes alone, without a
// barrier: its K and V tiles in LDS are its own, one each, copied by LDS DMA as soon as the
// products with the one before are done; S, its softmax with a running maximum, and O
// follow one another. At the end the four (m, l, O) are joined in LDS, in the order of the
// waves. (16 heads of 128 over 8, one prompt of 500 rows: 10.5 us, 13.7 on the tiles above; of
// 1000: 16.2 and 21.9.) Rows that do not come out as numbers are done again as above, and so are
// those whose weights were lost (c s is rounded for the maximum and not for the weights, from
// 2^31 on by more than their exponents hold). QL: the third parts of an f32 q stay in LDS, where
// the registers do not hold them (at D = 256 O takes 128, two parts of q as many).
template <int D, int PQ, int P, bool QL = PQ == 3 && D == 256>
__device__ void packed_quarters(const PackedArgs &a) {
  extern __shared__ __attribute__((aligned(kLdsAlign))) uint16_t lds[];  // [4][K, V of 32 rows], then [4][32] (m, l), a flag, q's third parts
  constexpr int ROWB = 2 * D, CH = D / 8, TILE = kStep * ROWB, NI = TILE / 1024, NK = D / 16, ND = D / 32;
  static_assert(ROWB <= kLdsAlign, "rows begin at multiples of their size");
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 31, hf = lane >> 5;
  const int hq = blockIdx.x % a.Hq, kvh = hq / (a.Hq / a.Hkv);
  int64_t first = 0;
  int len = 0;
  const int tile = row_tile(a, 32, blockIdx.x / a.Hq, first, len);
  if (tile < 0) return;
  const int r0 = tile * 32, steps = tile + 1;  // (the last one holds the tile's diagonal)

  const uint32_t own = lds_addr(lds) + wave * 2 * TILE;
  float2 *const ml = (float2 *)((char *)lds + 8 * TILE);
  int &again = *(int *)(ml + 128);
  u32x4 *const q_low = (u32x4 *)((char *)lds + 8 * TILE + 2048) + lane;  // [NK][64]
  constexpr int QR = QL ? PQ - 1 : PQ;                                    // parts in registers
  if (threadIdx.x == 0) again = 0;
  auto kx = [](int row) { return row & (CH < 16 ? CH - 1 : 15); };
  auto vx = [](int row) { return 2 * (row & (CH < 16 ? 3 : 7)); };
  const uint32_t stride = (uint32_t)a.Hkv * ROWB;
  const char *const kbase = (const char *)a.k + (first * a.Hkv + kvh) * ROWB;
  const char *const vbase = (const char *)a.v + (first * a.Hkv + kvh) * ROWB;
  auto copy = [&](const char *base, int step, bool is_v) RXW8_INLINE {
    const char *const from = base + (int64_t)step * kStep * stride;
    const int most = len - 1 - step * kStep;  // (rows past the sequence repeat its last)
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int row = 1024 / ROWB * i + lane / CH, x = is_v ? vx(row) : kx(row);
      dma16(from, (uint32_t)min(row, most) * stride + (((lane % CH) ^ x) << 4), __builtin_amdgcn_readfirstlane(own + is_v * TILE + 1024 * i));
    }
  };
  if (wave < steps) {
    copy(kbase, wave, false);
    copy(vbase, wave, true);
  }

  // ---- q
  u32x4 q[NK][QR];
  const int64_t q_at = ((first + min(r0 + col, len - 1)) * a.Hq + hq) * D + 8 * hf;
  constexpr int NL = 8;  // fragments asked for at a time
  unrolled<NK / (NK < NL ? NK : NL)>([&](auto g) RXW8_INLINE {
    constexpr int n0 = g * NL, N = NK < NL ? NK : NL;
    if constexpr (PQ == 3) {
      f32x4 x[N][2];
#pragma unroll
      for (int n = 0; n < N; ++n)
#pragma unroll
        for (int i = 0; i < 2; ++i) x[n][i] = *(const f32x4 *)((const float *)a.q + q_at + 16 * (n0 + n) + 4 * i);
#pragma unroll
      for (int n = 0; n < N; ++n) {
        u32x4 low;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          uint32_t part[3];
          split_bf16x2(x[n][e / 2][2 * e % 4], x[n][e / 2][2 * e % 4 + 1], part);
#pragma unroll
          for (int p = 0; p < QR; ++p) q[n0 + n][p][e] = part[p];
          low[e] = part[2];
        }
        if constexpr (QL) q_low[64 * (n0 + n)] = low;  // (the same from each wave)
      }
    } else {
#pragma unroll
      for (int n = 0; n < N; ++n) q[n0 + n][0] = *(const u32x4 *)((const uint16_t *)a.q + q_at + 16 * (n0 + n));
    }
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
      for (int p = 0; p < QR; ++p) asm volatile("" : "+v"(q[n0 + n][p]));  // (here, before the loop)
  });
  if constexpr (QL) asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
  f32x16 o[ND];
#pragma unroll
  for (int d = 0; d < ND; ++d)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[d][r] = 0.f;
  float m = kMinusInf, l = 0.f;
  const uint32_t k0 = own + col * ROWB + ((hf ^ kx(col)) << 4);
  const int tr_j = (lane & 15) >> 2, tr_q = lane & 3;
  const uint32_t v0 = own + TILE + (4 * hf + tr_j) * ROWB + 8 * (tr_q & 1) +
                      (((2 * ((lane >> 4) & 1) + (tr_q >> 1)) ^ vx(4 * hf + tr_j)) << 4);
#pragma unroll 1
  for (int h = wave; h < steps; h += 4) {
    const bool more = h + 4 < steps;
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(NI) : "memory");  // K is in (V, behind it, may not be)
    f32x16 s;
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = 0.f;
#pragma unroll
    for (int n = 0; n < NK; ++n) {
      const u32x4 f = *(const __attribute__((address_space(3))) u32x4 *)(uintptr_t)(k0 ^ (n << 5));
#pragma unroll
      for (int p = 0; p < QR; ++p) s = mfma32(f, q[n][p], s);
      if constexpr (QL) s = mfma32(f, q_low[64 * n], s);
    }
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    if (more) copy(kbase, h + 4, false);
    if (h == tile) {
#pragma unroll
      for (int r = 0; r < 16; ++r)
        if (8 * (r >> 2) + (r & 3) + 4 * hf > col) s[r] = kMinusInf;
    }
    // ---- softmax
    float mx = kMinusInf;
#pragma unroll
    for (int r = 0; r < 16; ++r) mx = fmaxf(mx, s[r]);
    mx = fmaxf(m, max_xor32(mx) * a.c);
    const float ref = mx == kMinusInf ? 0.f : mx;
    if (__ballot(mx != m)) {
      const float f = __builtin_amdgcn_exp2f(m - ref);
      m = mx, l *= f;
#pragma unroll
      for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[d][r] *= f;
    }
    u32x4 w[2][P];
#pragma unroll
    for (int g = 0; g < 8; ++g) {
      const int r = 2 * g;
      const float x = __builtin_amdgcn_exp2f(fmaf(s[r], a.c, -ref)), y = __builtin_amdgcn_exp2f(fmaf(s[r + 1], a.c, -ref));
      l += x + y;
      if constexpr (P == 3) {
        uint32_t part[3];
        split_bf16x2<true>(x, y, part);
#pragma unroll
        for (int p = 0; p < P; ++p) w[r >> 3][p][(r >> 1) & 3] = part[p];
      } else {
        w[r >> 3][0][(r >> 1) & 3] = pack_bf16x2(x, y);
      }
    }
    if (more) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(NI) : "memory");  // V is in
    else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
#pragma unroll
    for (int n = 0; n < 2 * ND; ++n) {
      u32x4 f;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4 *)(uintptr_t)(
            (v0 ^ (n % ND << 6)) + (16 * (n / ND) + 8 * e) * ROWB));
        const uint2 u = __builtin_bit_cast(uint2, x);
        f[2 * e] = u.x, f[2 * e + 1] = u.y;
      }
#pragma unroll
      for (int p = 0; p < P; ++p) o[n % ND] = mfma32(f, w[n / ND][p], o[n % ND]);
    }
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    if (more) copy(vbase, h + 4, true);
  }

  // ---- the waves' (m, l, O), in their own tiles' place: row by row, pieces of 4 swizzled
  auto ox = [](int row) { return row & 15; };
  if (wave < steps) {
    l = sum_xor32(l);
    if (hf == 0) ml[32 * wave + col] = float2{m, l};
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int x = 0; x < 4; ++x)
        *(__attribute__((address_space(3))) f32x4 *)(uintptr_t)(own + col * 4 * D + (((8 * d + 2 * x + hf) ^ ox(col)) << 4)) =
            f32x4{o[d][4 * x], o[d][4 * x + 1], o[d][4 * x + 2], o[d][4 * x + 3]};
  }
  __syncthreads();
  const int waves = min(steps, 4);
  constexpr int OC = D / 4;  // pieces of a row
  float odd = 0.f;
#pragma unroll 1
  for (int i = wave * 64; i < 32 * OC; i += 256) {
    const int row = (i + lane) / OC, piece = (i + lane) % OC;
    float M = kMinusInf, L = 0.f;
    for (int j = 0; j < waves; ++j) M = fmaxf(M, ml[32 * j + row].x);
    const float ref = M == kMinusInf ? 0.f : M;
    f32x4 y{0.f, 0.f, 0.f, 0.f};
    for (int j = 0; j < waves; ++j) {
      const float2 x = ml[32 * j + row];
      const float f = __builtin_amdgcn_exp2f(x.x - ref);
      const f32x4 z = *(const __attribute__((address_space(3))) f32x4 *)(uintptr_t)(
          lds_addr(lds) + j * 2 * TILE + row * 4 * D + ((piece ^ ox(row)) << 4));
      L = fmaf(f, x.y, L);
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] = fmaf(f, z[e], y[e]);
    }
    const float inv = L == 0.f ? 0.f : 1.0f / L;
    odd = L < kLeastSum ? 1.f : fmaf(L, 0.f, odd);
#pragma unroll
    for (int e = 0; e < 4; ++e) odd = fmaf(y[e], 0.f, odd), y[e] *= inv;
    if (r0 + row < len) {
      const int64_t to = ((first + r0 + row) * a.Hq + hq) * D + 4 * piece;
      if (P == 3 && a.out_f32) *(f32x4 *)((float *)a.out + to) = y;
      else *(u32x2 *)((uint16_t *)a.out + to) = u32x2{pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3])};
    }
  }
  if (odd != 0.f) again = 1;
  __syncthreads();
  if (!again) return;
  float *const qs = (float *)((char *)lds + wave * 4 * D);
  rows_again(a, D, qs, first, r0 + wave, min(r0 + 32, len), 4, hq);
}

#define RXW8_PACKED_QUARTERS(D, PQ, P, W, NAME)                                                      \
  extern "C" __global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(W, W)))       \
      rxw8_packed_quarters_##NAME##_d##D(PackedArgs a) {                                             \
    packed_quarters<D, PQ, P>(a);                                                                    \
  }
RXW8_PACKED_QUARTERS(64, 1, 1, 2, bf16)
RXW8_PACKED_QUARTERS(128, 1, 1, 2, bf16)
RXW8_PACKED_QUARTERS(256, 1, 1, 1, bf16)
RXW8_PACKED_QUARTERS(64, 1, 3, 2, bf16_f32)
RXW8_PACKED_QUARTERS(128, 1, 3, 2, bf16_f32)
RXW8_PACKED_QUARTERS(256, 1, 3, 1, bf16_f32)
RXW8_PACKED_QUARTERS(64, 3, 3, 2, f32)
RXW8_PACKED_QUARTERS(128, 3, 3, 2, f32)
RXW8_PACKED_QUARTERS(256, 3, 3, 1, f32)
