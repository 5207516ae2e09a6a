// Causal attention of packed prompts: sequence b owns rows offsets[b] ..
// offsets[b + 1] - 1 of q [T, Hq, D] and of k, v [T, Hkv, D], and row t of it sees
// rows offsets[b] .. t. Offsets are read on the device and clamped into [0, T].
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
