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
