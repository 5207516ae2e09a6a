// The paged key/value cache: the append that fills its pages and the attention of
// one new token per sequence that reads them.
#include "paged_decode.h"

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

#define RXW8_PAGED_DECODE(D, NAME, F)                                                        \
  extern "C" __global__ void __launch_bounds__(64 * kPagedWaves) rxw8_paged_decode_##NAME##_d##D(PagedDecodeArgs a) { \
    paged_decode<D, F>(a, paged_place_of(a));                                                \
  }
RXW8_PAGED_DECODE(64, bf16, kBf16)
RXW8_PAGED_DECODE(128, bf16, kBf16)
RXW8_PAGED_DECODE(256, bf16, kBf16)
RXW8_PAGED_DECODE(64, f32, kF32)
RXW8_PAGED_DECODE(128, f32, kF32)
RXW8_PAGED_DECODE(256, f32, kF32)
