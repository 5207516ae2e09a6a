// The page tables: where a sequence's positions are, for the kernels that write, read
// back and attend over paged caches. Pages are [P, Hkv, ps, D] (a kv head's ps rows of a
// page in one piece); table [B, M] I32 gives sequence b the page of its positions ps i ..
// ps i + ps - 1 in entry i, anything outside [0, P) where it has none. An entry is
// checked before its page is touched.
#pragma once
#include "attn_any.h"

// Row t of k and v: the page and the place in it (page below 0: none) of the position
// starts[b] + i, for row i of sequence b; rows outside every sequence (place below 0)
// and positions without a page have none. By a whole wave, t uniform.
struct PagedPlace {
  int64_t page;
  int at;
};
// (As any_sequence, the starts beside the offsets: what the row's position needs is in the
// lanes when its sequence is known, and the page table is the next thing that is waited for.)
template <typename Args>
__device__ __forceinline__ PagedPlace paged_place(const Args &a, int64_t t) {
  int64_t b = t, pos;
  if (a.offsets) {
    const int lane = threadIdx.x & 63;
    int lo = 0, n = a.B;
    while (n > 64) {
      const int step = (n + 63) / 64, i = lo + lane * step;
      const unsigned long long le = __ballot(lane * step < n && a.offsets[i < a.B ? i : a.B] <= t);
      const int c = __popcll(le);
      if (c == 0) return PagedPlace{-1, -1};
      const int skip = (c - 1) * step;
      lo += skip;
      n = n - skip < step ? n - skip : step;
    }
    const int i = lo + lane < a.B ? lo + lane : a.B;
    const int first = a.offsets[i], start = i < a.B ? a.starts[i] : 0;
    const int c = __popcll(__ballot(lane < n && first <= t));
    if (c == 0) return PagedPlace{-1, -1};
    b = lo + c - 1;
    const int64_t end = c < 64 ? __builtin_amdgcn_readlane(first, c) : a.offsets[b + 1];
    if (t >= end) return PagedPlace{-1, -1};
    pos = (int64_t)__builtin_amdgcn_readlane(start, c - 1) + (t - __builtin_amdgcn_readlane(first, c - 1));
  } else {
    pos = a.starts[b];
  }
  if (pos < 0 || pos >= (int64_t)a.M * a.ps) return PagedPlace{-1, 0};
  const int slot = (int)((uint32_t)pos / (uint32_t)a.ps);  // (positions of a table are 31 bits)
  const int64_t page = a.table[b * a.M + slot];
  return PagedPlace{page < a.P ? page : -1, (int)pos - slot * a.ps};
}

struct PagedDecodeArgs {
  const void *q;          // [B, Hq, D] f32 | bf16
  const void *kp, *vp;    // [P, Hkv, ps, D] f32 | bf16 | u8
  const int32_t *table;   // [B, M]
  const int32_t *lens;    // [B]
  void *out;              // [B, Hq, D] f32 | bf16
  int64_t P;
  int B, M, Hq, Hkv, D, ps;
  float c;                // scale log2 e
  int q_f32, p_f32, out_f32;
  // the matrix-core kernels: `units` workgroups for each kv head and 16 of its
  // query heads; counters [Hkv HT units], zero between launches, and two
  // records of min(G, 16) (D + 4) floats each, padded to whole KiB
  int units, waves;       // waves that walk keys (a workgroup has 8; the others help to join)
  int *counters;
  float *part;
  const float *ks, *vs;   // [P, Hkv, ps]: the scales of 8-bit rows
};

__device__ __forceinline__ int64_t paged_len(const PagedDecodeArgs &a, int b) {
  const int64_t n = a.lens[b], most = (int64_t)a.M * a.ps;
  return n < 0 ? 0 : n > most ? most : n;
}

// Rows of 8-bit pages: an element is (code - 128) s, s the row's scale
struct AnyCodes {
  const uint8_t *k, *v;
  const float *ks, *vs;
  int d;
  __device__ __forceinline__ float key(int64_t off, int i) const { return (float)k[off + i] - 128.f; }
  __device__ __forceinline__ float value(int64_t off, int i) const { return (float)v[off + i] - 128.f; }
  __device__ __forceinline__ float key_scale(int64_t off) const { return ks[off / d]; }
  __device__ __forceinline__ float value_scale(int64_t off) const { return vs[off / d]; }
};
