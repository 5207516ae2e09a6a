// Attention of one new token per sequence where sequences share a prefix: those of
// groups[n] .. groups[n + 1] - 1 see the first prefix_lens[n] positions of the page table
// prefixes[n], and behind them the first lens[b] positions of their own table.
#include "paged.h"

struct SharedArgs {
  const void *q;              // [B, Hq, D] f32 | bf16
  const void *kp, *vp;        // [P, Hkv, ps, D] bf16 | f32 | u8
  const float *ks, *vs;       // [P, Hkv, ps] (u8)
  const int32_t *prefixes;    // [N, MP]
  const int32_t *prefix_lens; // [N]
  const int32_t *groups;      // [N + 1]
  const int32_t *table;       // [B, M]
  const int32_t *lens;        // [B]
  void *out;                  // [B, Hq, D] f32 | bf16
  int64_t P;
  int B, N, MP, M, Hq, Hkv, D, ps;
  float c;                    // scale log2 e
  int q_f32, kind, out_f32;   // kind: 0 bf16, 1 f32, 2 u8 pages
};

// Any head width up to 512, any page size: one workgroup of 4 waves per (sequence, query
// head) over its prefix and its own keys, the waves' chunks of 64 keys in turn
extern "C" __global__ void __launch_bounds__(256) rxw8_shared_any(SharedArgs a) {
  __shared__ float q[RXW8_ATTN_ANY_MAX_D], part[4][RXW8_ATTN_ANY_MAX_D], mw[4], lw[4];
  const int wave = threadIdx.x >> 6;
  const int b = blockIdx.x / a.Hq, hq = blockIdx.x - b * a.Hq, h = hq / (a.Hq / a.Hkv);
  const int64_t at = (int64_t)blockIdx.x * a.D;
  for (int i = threadIdx.x; i < a.D; i += 256) q[i] = any_load(a.q, at + i, a.q_f32);
  __syncthreads();
  AnyState st;
  auto walk = [&](const int32_t *table, int64_t n, int m) {
    const int64_t most = (int64_t)m * a.ps;
    auto row = [&](int64_t j) -> int64_t {
      const int64_t page = table[j / a.ps];
      return page < 0 || page >= a.P ? -1 : ((page * a.Hkv + h) * a.ps + j % a.ps) * a.D;
    };
    n = n < most ? n : most;
    if (a.kind == 2)
      any_walk(st, q, AnyCodes{(const uint8_t *)a.kp, (const uint8_t *)a.vp, a.ks, a.vs, a.D}, a.D, 64 * wave, n, 4, a.c, row);
    else
      any_walk(st, q, AnyPlain{a.kp, a.vp, a.kind == 1}, a.D, 64 * wave, n, 4, a.c, row);
  };
  const int g = any_sequence(a.groups, a.N, b);
  if (g >= 0 && b < a.groups[g + 1]) walk(a.prefixes + (int64_t)g * a.MP, a.prefix_lens[g], a.MP);
  walk(a.table + (int64_t)b * a.M, a.lens[b], a.M);
  AnyState all;
  if (!any_join(all, st, part, mw, lw)) return;
  any_store(all, a.out, at, a.D, a.out_f32);
}
