// The paged cache in 8 bits: a row x [D] of a kv head is held as codes (int8 + 128) and
// one f32 scale,
//   s = max(amax |x|, 1e-12) / 127,  code = clamp(rne(x / s), -127, 127) + 128,
// and stands for (code - 128) s: at most s / 2 off (1/254 of the row's largest), and the
// same codes as rxw8_quantize_w8 with groups of D. A row that holds a NaN or an infinity
// has the scale NaN and the codes 128: all of it stands for NaN. Here are the append that
// writes such rows, the reading back of pages of any type, and the attention of one new
// token per sequence over 8-bit pages.
#include "paged_decode.h"

struct PagedQ8Args {
  const void *k, *v;         // [T, Hkv, D] f32 | bf16
  uint8_t *kp, *vp;          // [P, Hkv, ps, D]
  float *ks, *vs;            // [P, Hkv, ps]
  const int32_t *table;      // [B, M]
  const int32_t *starts;     // [B]
  const int32_t *offsets;    // [B + 1], or null: row b of sequence b
  int64_t T, P;
  int B, M, Hkv, D, ps;
  int k_f32;
};

// The scale of a row from its largest magnitude (NaN: the row holds a NaN or an infinity)
__device__ __forceinline__ float q8_scale(float amax) { return (amax >= 1e-12f ? amax : amax != amax ? amax : 1e-12f) / 127.0f; }
__device__ __forceinline__ uint32_t q8_code(float x, float s) {
  return s != s ? 128u : (uint32_t)(fminf(fmaxf(rintf(x / s), -127.0f), 127.0f) + 128.0f);
}
// |x| for a maximum by bits: NaN for what is no finite number, above every other
__device__ __forceinline__ uint32_t q8_size(float x) {
  const uint32_t u = __float_as_uint(x) & 0x7fffffffu;
  return u >= 0x7f800000u ? 0x7fc00000u : u;
}

// Any width and alignment: a wave for each (row, kv head), an element a lane
extern "C" __global__ void __launch_bounds__(256) rxw8_q8_append_any(PagedQ8Args a) {
  const int lane = threadIdx.x & 63;
  const int64_t unit = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (unit >= a.T * a.Hkv) return;  // whole waves only; no barriers below
  const int64_t t = unit / a.Hkv;
  const int h = (int)(unit - t * a.Hkv);
  const PagedPlace to = paged_place(a, t);
  if (to.page < 0) return;
  const int64_t src = unit * a.D, row = (to.page * a.Hkv + h) * a.ps + to.at;
#pragma unroll
  for (int kv = 0; kv < 2; ++kv) {
    const void *x = kv ? a.v : a.k;
    uint8_t *codes = (kv ? a.vp : a.kp) + row * a.D;
    uint32_t top = 0;
    for (int e = lane; e < a.D; e += 64) top = max(top, q8_size(any_load(x, src + e, a.k_f32)));
    for (int o = 32; o > 0; o >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, o));
    const float s = q8_scale(__uint_as_float(top));
    for (int e = lane; e < a.D; e += 64) codes[e] = (uint8_t)q8_code(any_load(x, src + e, a.k_f32), s);
    if (lane == 0) (kv ? a.vs : a.ks)[row] = s;
  }
}

// Head widths of 64, 128, 256 and 512 at 16-byte boundaries: a wave for each row and
// `kRows` x 64 of its pieces of 8 elements, D / 8 lanes to a head, K's and V's pieces
// under way before the wave looks for its sequence and page. Its arithmetic is what takes
// the time unless it is few instructions an element, so
//  - the largest magnitude is one of bit patterns (of two bf16 at once): above every number
//    there stand the infinities and NaN;
//  - s = amax / 127 is q + (amax - 127 q) / 127 of q = amax (1 / 127), rounded once: the
//    correctly rounded quotient (Markstein's step; no amax in range differs);
//  - x / s likewise, from the rounded 1 / s, so that no code is ever divided for (products
//    with 1 / s alone, and divisions where they come near the middle between two codes: 22.8
//    us for the 9000 rows below, bf16 rows have many such). Adding 1.5 2^23 + 128 rounds the
//    quotient: the code is the sum's lowest byte.
// 9000 bf16 rows of 8 heads of 128: 17.4 us, 3.2 TB/s; 96 f32 rows, one a sequence: 4.2 us.
constexpr int kRows = 2;

// The largest over a head's lanes (8, 16, 32 or 64 of them, beside one another)
__device__ __forceinline__ uint32_t head_max(uint32_t v, int lanes) {
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xb1, 0xf, 0xf, false));   // quad_perm: ^ 1
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x4e, 0xf, 0xf, false));   // ^ 2
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x141, 0xf, 0xf, false));  // row_half_mirror
  if (lanes > 8) v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x140, 0xf, 0xf, false));  // row_mirror
  if (lanes > 16) {
    const uint2 p = pair_xor16(__uint_as_float(v));
    v = max(p.x, p.y);
  }
  if (lanes > 32) {
    const uint2 p = pair_xor32(__uint_as_float(v));
    v = max(p.x, p.y);
  }
  return v;
}

template <typename S>
__device__ __forceinline__ void q8_append(const PagedQ8Args &a) {
  constexpr int NS = sizeof(S) / 2;  // 16-byte words of 8 elements
  const int lane = threadIdx.x & 63, per_head = a.D / 8, pieces = a.Hkv * per_head, log2 = __builtin_ctz(per_head);
  const int64_t t = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int p0 = blockIdx.y * 64 * kRows + lane;
  if (t >= a.T) return;  // whole waves only; no barriers below
  u32x4 x[kRows][2][NS];
#pragma unroll
  for (int n = 0; n < kRows; ++n)
    if (p0 + 64 * n < pieces) {
      const int64_t at = (t * pieces + p0 + 64 * n) * NS;
#pragma unroll
      for (int i = 0; i < NS; ++i) x[n][0][i] = ((const u32x4 *)a.k)[at + i], x[n][1][i] = ((const u32x4 *)a.v)[at + i];
    }
  const PagedPlace to = paged_place(a, t);
  if (to.page < 0) return;
#pragma unroll
  for (int n = 0; n < kRows; ++n) {
    const int p = p0 + 64 * n;
    const bool mine = p < pieces;  // (whole heads: the lanes of one are all in or all out)
    const int h = p >> log2;
    const int64_t row = (to.page * a.Hkv + h) * a.ps + to.at;
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
      float v[8];
      uint32_t top = 0;
      if constexpr (NS == 2) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          v[i] = __uint_as_float(x[n][kv][i >> 2][i & 3]);
          top = max(top, x[n][kv][i >> 2][i & 3] & 0x7fffffffu);
        }
      } else {
        typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
        u16x2 two = {0, 0};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t w = x[n][kv][0][i];
          v[2 * i] = __uint_as_float(w << 16), v[2 * i + 1] = __uint_as_float(w & 0xffff0000u);
          two = __builtin_elementwise_max(two, __builtin_bit_cast(u16x2, w & 0x7fff7fffu));
        }
        top = (uint32_t)max(two[0], two[1]) << 16;
      }
      top = head_max(top, per_head);
      const float amax = fmaxf(__uint_as_float(top), 1e-12f);
      const float part = 1.0f / 127.0f, q = amax * part;
      float s = fmaf(fmaf(-127.0f, q, amax), part, q);
      const float inv = 1.0f / s;
      uint32_t y[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float q = v[i] * inv, quotient = fmaf(fmaf(-s, q, v[i]), inv, q);
        y[i] = __float_as_uint(quotient + (12582912.f + 128.f));
      }
      uint32_t code[2];
#pragma unroll
      for (int i = 0; i < 2; ++i)
        code[i] = __builtin_amdgcn_perm(y[4 * i + 1], y[4 * i], 0x0c0c0400) | __builtin_amdgcn_perm(y[4 * i + 3], y[4 * i + 2], 0x04000c0c);
      if (top >= 0x7f800000u) {
        s = __builtin_nanf("");
        code[0] = code[1] = 0x80808080u;
      }
      if (mine) {
        *(uint2 *)((kv ? a.vp : a.kp) + row * a.D + 8 * (p - h * per_head)) = uint2{code[0], code[1]};
        if (p == h * per_head) (kv ? a.vs : a.ks)[row] = s;
      }
    }
  }
}
extern "C" __global__ void __launch_bounds__(256) rxw8_q8_append(PagedQ8Args a) {
  if (a.k_f32) q8_append<float>(a);
  else q8_append<uint16_t>(a);
}

struct PagedReadArgs {
  const void *kp, *vp;       // [P, Hkv, ps, D] bf16 | f32 | u8
  const float *ks, *vs;      // [P, Hkv, ps] (u8)
  void *k, *v;               // [T, Hkv, D] f32 | bf16
  const int32_t *table;      // [B, M]
  const int32_t *starts;     // [B]
  const int32_t *offsets;    // [B + 1], or null: row b of sequence b
  int64_t T, P;
  int B, M, Hkv, D, ps;
  int kind;                  // 0 bf16, 1 f32, 2 u8 pages
  int k_f32;
};

// Any width and alignment: a wave for each (row, kv head), an element a lane
extern "C" __global__ void __launch_bounds__(256) rxw8_q8_read_any(PagedReadArgs a) {
  const int lane = threadIdx.x & 63;
  const int64_t unit = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (unit >= a.T * a.Hkv) return;
  const int64_t t = unit / a.Hkv;
  const int h = (int)(unit - t * a.Hkv);
  const PagedPlace of = paged_place(a, t);
  if (of.at < 0) return;
  const int64_t dst = unit * a.D, row = (of.page * a.Hkv + h) * a.ps + of.at;
#pragma unroll
  for (int kv = 0; kv < 2; ++kv) {
    const void *pages = kv ? a.vp : a.kp;
    void *to = kv ? a.v : a.k;
    const float s = of.page >= 0 && a.kind == 2 ? (kv ? a.vs : a.ks)[row] : 1.f;
    for (int e = lane; e < a.D; e += 64) {
      float y = 0.f;
      if (of.page >= 0)
        y = a.kind == 2 ? ((float)((const uint8_t *)pages)[row * a.D + e] - 128.f) * s : any_load(pages, row * a.D + e, a.kind);
      if (a.k_f32) ((float *)to)[dst + e] = y;
      else ((uint16_t *)to)[dst + e] = f32_to_bf16_bits(y);
    }
  }
}

// Widths of whole 8 elements at 16-byte boundaries: a wave for each row and `kRows` x 64
// of its pieces of 8 elements, bound by HBM: 13800 positions of 8 heads of 128 in 8 bits to bf16
// rows 18.5 us, 4.6 TB/s (pieces of 64 for a wave, one round of loads each: 20.3)
template <int KIND, typename S>
__device__ __forceinline__ void paged_read(const PagedReadArgs &a) {
  constexpr int NP = KIND == 1 ? 2 : 1, NS = sizeof(S) / 2;  // 16-byte words of 8 elements (codes: half a one)
  const int lane = threadIdx.x & 63, per_head = a.D / 8, pieces = a.Hkv * per_head;
  const int64_t t = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int p0 = blockIdx.y * 64 * kRows + lane;
  if (t >= a.T) return;
  const PagedPlace of = paged_place(a, t);
  if (of.at < 0) return;
  u32x4 x[kRows][2][NP];
  float s[kRows][2];
#pragma unroll
  for (int n = 0; n < kRows; ++n) {
    const int p = p0 + 64 * n, h = p / per_head;
    const int64_t row = (of.page * a.Hkv + h) * a.ps + of.at, at = row * per_head + (p - h * per_head);
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
      const void *pages = kv ? a.vp : a.kp;
      s[n][kv] = 0.f;
#pragma unroll
      for (int i = 0; i < NP; ++i) x[n][kv][i] = KIND == 2 ? u32x4{0x80808080u, 0x80808080u, 0, 0} : u32x4{0, 0, 0, 0};
      if (p >= pieces || of.page < 0) continue;
      if constexpr (KIND == 2) {
        const uint2 c = ((const uint2 *)pages)[at];
        x[n][kv][0][0] = c.x, x[n][kv][0][1] = c.y;
        s[n][kv] = (kv ? a.vs : a.ks)[row];
      } else {
#pragma unroll
        for (int i = 0; i < NP; ++i) x[n][kv][i] = ((const u32x4 *)pages)[at * NP + i];
      }
    }
  }
#pragma unroll
  for (int n = 0; n < kRows; ++n) {
    const int p = p0 + 64 * n;
    if (p >= pieces) return;
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
      float v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if constexpr (KIND == 2) v[i] = ((float)(x[n][kv][0][i >> 2] >> 8 * (i & 3) & 0xffu) - 128.f) * s[n][kv];
        else if constexpr (KIND == 1) v[i] = __uint_as_float(x[n][kv][i >> 2][i & 3]);
        else v[i] = __uint_as_float(i & 1 ? x[n][kv][0][i >> 1] & 0xffff0000u : x[n][kv][0][i >> 1] << 16);
      }
      u32x4 *const to = (u32x4 *)(kv ? a.v : a.k) + (t * pieces + p) * NS;
      if constexpr (NS == 2) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
          to[i] = u32x4{__float_as_uint(v[4 * i]), __float_as_uint(v[4 * i + 1]), __float_as_uint(v[4 * i + 2]), __float_as_uint(v[4 * i + 3])};
      } else {
        to[0] = u32x4{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7])};
      }
    }
  }
}
extern "C" __global__ void __launch_bounds__(256) rxw8_q8_read(PagedReadArgs a) {
  if (a.k_f32) {
    if (a.kind == 2) paged_read<2, float>(a);
    else if (a.kind == 1) paged_read<1, float>(a);
    else paged_read<0, float>(a);
  } else {
    if (a.kind == 2) paged_read<2, uint16_t>(a);
    else if (a.kind == 1) paged_read<1, uint16_t>(a);
    else paged_read<0, uint16_t>(a);
  }
}

// Any head width up to 512, any page size: one workgroup of 4 waves per (sequence, query
// head), the waves' chunks of 64 keys in turn, merged in LDS
extern "C" __global__ void __launch_bounds__(256) rxw8_q8_decode_any(PagedDecodeArgs a) {
  __shared__ float q[RXW8_ATTN_ANY_MAX_D], part[4][RXW8_ATTN_ANY_MAX_D], mw[4], lw[4];
  const int wave = threadIdx.x >> 6;
  const int b = blockIdx.x / a.Hq, hq = blockIdx.x - b * a.Hq, h = hq / (a.Hq / a.Hkv);
  const int64_t at = (int64_t)blockIdx.x * a.D;
  for (int i = threadIdx.x; i < a.D; i += 256) q[i] = any_load(a.q, at + i, a.q_f32);
  __syncthreads();
  AnyState st;
  any_walk(st, q, AnyCodes{(const uint8_t *)a.kp, (const uint8_t *)a.vp, a.ks, a.vs, a.D}, a.D, 64 * wave, paged_len(a, b), 4, a.c,
           [&](int64_t j) -> int64_t {
             const int64_t page = a.table[(int64_t)b * a.M + j / a.ps];
             return page < 0 || page >= a.P ? -1 : ((page * a.Hkv + h) * a.ps + j % a.ps) * a.D;
           });
  AnyState all;
  if (!any_join(all, st, part, mw, lw)) return;
  any_store(all, a.out, at, a.D, a.out_f32);
}

#define RXW8_Q8_DECODE(D, NAME, PREC)                                                          \
  extern "C" __global__ void __launch_bounds__(64 * kPagedWaves) rxw8_q8_decode##NAME##_d##D(PagedDecodeArgs a) { \
    paged_decode<D, kCodes, false, PREC>(a, paged_place_of(a));                                \
  }
RXW8_Q8_DECODE(64, , kLow)
RXW8_Q8_DECODE(128, , kLow)
RXW8_Q8_DECODE(256, , kLow)
RXW8_Q8_DECODE(64, _high, kHigh)
RXW8_Q8_DECODE(128, _high, kHigh)
RXW8_Q8_DECODE(256, _high, kHigh)
