// The serving operators: the paged key/value cache (append, decode attention),
// causal attention of packed prompts, and sampling of the next token.
#include <algorithm>
#include <cmath>
#include <cstdint>
#include <cstdio>

#include "internal.h"

namespace rxw8 {

// (the kernels' argument structs: kernels/paged.hip, packed.hip, sample.hip)
struct PagedAppendArgs {
  const void *k, *v;
  void *kp, *vp;
  const int32_t *table, *starts, *offsets;
  int64_t T, P;
  int B, M, Hkv, D, ps;
  int k_f32, p_f32;
};
struct PagedDecodeArgs {
  const void *q, *kp, *vp;
  const int32_t *table, *lens;
  void *out;
  int64_t P;
  int B, M, Hq, Hkv, D, ps;
  float c;
  int q_f32, p_f32, out_f32;
  int units, waves;
  int *counters;
  float *part;
};
struct PackedArgs {
  const void *q;
  const uint16_t *k, *v;
  const int32_t *offsets;
  void *out;
  int64_t T;
  int B, Hq, Hkv, D;
  float c;
  int q_f32, out_f32;
  int fill;
  int heads;
};
struct SampleArgs {
  const void *logits;
  const float *uniform, *temperature;
  const int32_t *top_k;
  const float *top_p, *min_p;
  int32_t *out;
  int64_t V;
  int shift;
  int bf16;
  int S;
  int64_t chunk;
  char *extremes;
  int *arrivals, *listed;
  char *bins;
};
constexpr int64_t kSampleExtremes = 16, kSampleBins = 12 << 10;  // bytes of a workgroup's records
constexpr size_t kSampleLds = 92 << 10;                          // SampleShared

static bool is_f(int dt) { return dt == RXW8_F32 || dt == RXW8_BF16; }
static bool is_vec(const Buffer *b, int dtype, int64_t n) {
  return b->dtype == dtype && b->rank == 1 && b->dims[0] == n;
}
static bool same_shape(const Buffer *a, const Buffer *b) {
  bool same = a->dtype == b->dtype && a->rank == b->rank;
  for (int i = 0; same && i < a->rank; ++i) same = a->dims[i] == b->dims[i];
  return same;
}
// Workgroups of `threads` that one launch takes: 2^32 - 1 threads
constexpr int64_t grid_max(int threads) { return (((int64_t)1 << 32) - 1) / threads; }
constexpr int64_t kAnyMaxD = 512;  // RXW8_ATTN_ANY_MAX_D

// Whether the buffers (NULL ones aside) are the runtime's, and none of the first `written`
// shares memory with another
static int check_buffers(const char *what, const Runtime *rt, std::initializer_list<const Buffer *> bufs, int written) {
  for (const Buffer *b : bufs)
    if (b && b->rt != rt) return fail(RXW8_INVALID_ARGUMENT, "%s: buffers of another runtime", what);
  int i = 0;
  for (const Buffer *w : bufs) {
    if (i++ == written) break;
    int j = 0;
    for (const Buffer *b : bufs)
      if (j++ != i - 1 && w && b && w->bytes && b->bytes && (char *)w->ptr < (char *)b->ptr + b->bytes &&
          (char *)b->ptr < (char *)w->ptr + w->bytes)
        return fail(RXW8_INVALID_ARGUMENT, "%s: what is written must not share memory with another argument", what);
  }
  return RXW8_OK;
}

// Pages [P, Hkv, ps, D] F32|BF16 and the table I32 [B, M]
static int check_pages(const char *what, const Buffer *kp, const Buffer *vp, const Buffer *table) {
  if (kp->rank != 4 || !is_f(kp->dtype) || !same_shape(kp, vp))
    return fail(RXW8_INVALID_ARGUMENT, "%s: pages must be two F32/BF16 [P,Hkv,ps,D] of one shape and type", what);
  if (kp->dims[1] <= 0 || kp->dims[2] <= 0 || kp->dims[3] <= 0)
    return fail(RXW8_INVALID_ARGUMENT, "%s: pages %s need positive heads, rows and width", what, dims_str(kp).c_str());
  if (table->dtype != RXW8_I32 || table->rank != 2)
    return fail(RXW8_INVALID_ARGUMENT, "%s: the page table must be I32 [B,M]", what);
  for (int i = 1; i < 4; ++i)
    if (kp->dims[i] > INT32_MAX) return fail(RXW8_UNIMPLEMENTED, "%s: pages %s", what, dims_str(kp).c_str());
  // positions are I32
  if (table->dims[0] > INT32_MAX || (table->dims[1] > 0 && kp->dims[2] > INT32_MAX / table->dims[1]))
    return fail(RXW8_UNIMPLEMENTED, "%s: %lld pages of %lld positions exceed 32-bit positions", what,
                (long long)table->dims[1], (long long)kp->dims[2]);
  return RXW8_OK;
}

constexpr float kScaleLog2e = 1.4426950408889634f;
static float softmax_scale(float scale, int64_t D) {
  // (above 0 for every scale, so that -inf times it stays -inf)
  return (scale <= 0.f ? 1.0f / std::sqrt((float)D) : scale) * kScaleLog2e;
}
static int check_scale(float scale) {
  if (!std::isfinite(scale)) return fail(RXW8_INVALID_ARGUMENT, "attention scale must be finite");
  if (scale > 0.f && !std::isfinite(scale * kScaleLog2e))
    return fail(RXW8_INVALID_ARGUMENT, "attention scale %g times log2(e) must be finite", (double)scale);
  return RXW8_OK;
}

static int check_paged_decode(const Buffer *q, const Buffer *kp, const Buffer *vp, const Buffer *table,
                              const Buffer *lens, float scale) {
  if (!q || !kp || !vp || !table || !lens) return fail(RXW8_INVALID_ARGUMENT, "paged GQA decode: NULL buffer");
  if (int rc = check_pages("paged GQA decode", kp, vp, table)) return rc;
  if (q->rank != 3 || !is_f(q->dtype))
    return fail(RXW8_INVALID_ARGUMENT, "paged GQA decode requires F32/BF16 q [B,Hq,D]");
  const int64_t B = q->dims[0], Hq = q->dims[1], D = q->dims[2];
  if (table->dims[0] != B || D != kp->dims[3])
    return fail(RXW8_INVALID_ARGUMENT, "paged GQA decode: q, page table and pages differ in batch or head width");
  if (Hq <= 0 || Hq % kp->dims[1] != 0)
    return fail(RXW8_INVALID_ARGUMENT, "GQA requires equal batch prefixes and divisible positive head counts");
  if (!is_vec(lens, RXW8_I32, B)) return fail(RXW8_INVALID_ARGUMENT, "paged GQA decode: lens must be I32 [B]");
  if (int rc = check_scale(scale)) return rc;
  if (D > kAnyMaxD) return fail(RXW8_UNIMPLEMENTED, "paged GQA decode: head dim %lld > 512", (long long)D);
  if (Hq > INT32_MAX || B > grid_max(256) / Hq)
    return fail(RXW8_UNIMPLEMENTED, "paged GQA decode: %lld x %lld rows exceed the kernel's grid", (long long)B,
                (long long)Hq);
  return RXW8_OK;
}

static int check_packed(const Buffer *q, const Buffer *k, const Buffer *v, const Buffer *offsets, float scale) {
  if (!q || !k || !v || !offsets) return fail(RXW8_INVALID_ARGUMENT, "packed GQA prefill: NULL buffer");
  if (q->rank != 3 || k->rank != 3 || !is_f(q->dtype) || k->dtype != RXW8_BF16 || !same_shape(k, v))
    return fail(RXW8_INVALID_ARGUMENT, "packed GQA prefill requires F32/BF16 q [T,Hq,D] and BF16 k, v [T,Hkv,D]");
  const int64_t T = q->dims[0], Hq = q->dims[1], D = q->dims[2];
  if (k->dims[0] != T || k->dims[2] != D || D <= 0)
    return fail(RXW8_INVALID_ARGUMENT, "packed GQA prefill: q and k, v differ in rows or head width");
  if (Hq <= 0 || k->dims[1] <= 0 || Hq % k->dims[1] != 0)
    return fail(RXW8_INVALID_ARGUMENT, "GQA requires equal batch prefixes and divisible positive head counts");
  if (offsets->dtype != RXW8_I32 || offsets->rank != 1 || offsets->dims[0] < 1)
    return fail(RXW8_INVALID_ARGUMENT, "packed GQA prefill: offsets must be I32 [sequences + 1]");
  if (int rc = check_scale(scale)) return rc;
  if (D > kAnyMaxD) return fail(RXW8_UNIMPLEMENTED, "packed GQA prefill: head dim %lld > 512", (long long)D);
  if (T > INT32_MAX || Hq > INT32_MAX || T > 4 * grid_max(256) / Hq || offsets->dims[0] > INT32_MAX)
    return fail(RXW8_UNIMPLEMENTED, "packed GQA prefill: %lld x %lld rows exceed the kernel's grid", (long long)T,
                (long long)Hq);
  return RXW8_OK;
}

// The matrix-core kernels take head widths 64, 128 and 256, pages of whole 16-row
// pieces, 16-byte aligned operands and tile counts within 32 bits; else the plain
// kernel. As many waves walk keys, up to 8, as tiles and records of the group's heads
// fit in LDS. `units` workgroups for each kv head (and 16 query heads): the number that
// leaves the fewest CUs idle in the last round.
static int paged_decode_launch(Runtime *rt, PagedDecodeArgs a) {
  const int64_t G = a.Hq / a.Hkv, heads = a.Hkv * ((G + 15) / 16), gcap = G < 16 ? G : 16;
  const int es = a.p_f32 ? 4 : 2, row = a.D * es, tile = row < 256 ? 32 : 16;
  if ((a.D != 64 && a.D != 128 && a.D != 256) || a.ps % 16 || a.P == 0 || heads > 4096 ||
      ((uintptr_t)a.q | (uintptr_t)a.kp | (uintptr_t)a.vp | (uintptr_t)a.out) % 16 ||
      (int64_t)a.B * (((int64_t)a.M * a.ps + tile - 1) / tile) >= ((int64_t)1 << 30))
    return launch(rt, "rxw8_paged_decode_any", dim3((unsigned)a.B * (unsigned)a.Hq), dim3(256), a);
  const size_t record = (size_t)gcap * (size_t)(a.D + 4) * sizeof(float), wave = std::max((size_t)(2 * tile * row), record) + record;
  a.waves = (int)std::min<size_t>(8, (rt->lds_max - 1024) / wave);
  const int64_t most = std::max<int64_t>(1, std::min<int64_t>({256, (int64_t)(RXW8_NOALLOC_COUNTER_BYTES / sizeof(int)) / heads,
                                                               (int64_t)(RXW8_NOALLOC_PARTIAL_BYTES / (2 * ((record + 1023) & ~(size_t)1023))) / heads}));
  a.units = 1;
  for (int64_t u = 2; u <= most; ++u) {  // rounds of workgroups per unit of work
    const int64_t r0 = (heads * a.units + rt->cus - 1) / rt->cus, r1 = (heads * u + rt->cus - 1) / rt->cus;
    if (r1 * a.units < r0 * u) a.units = (int)u;
  }
  char *block = rt->f32_attn[stream_capturing(rt) ? 1 : 0];
  a.counters = (int *)block;
  a.part = (float *)(block + RXW8_NOALLOC_COUNTER_BYTES);
  char kname[40];
  std::snprintf(kname, sizeof kname, "rxw8_paged_decode_%s_d%d", a.p_f32 ? "f32" : "bf16", a.D);
  return launch(rt, kname, dim3((unsigned)(heads * a.units)), dim3(512), a, wave * (size_t)a.waves);
}

static int packed_launch(Runtime *rt, const Buffer *q, const Buffer *k, const Buffer *v, const Buffer *offsets,
                         float scale, const Buffer *out, bool fill) {
  const int64_t T = q->dims[0], Hq = q->dims[1], D = q->dims[2];
  if (T == 0) return RXW8_OK;
  const int64_t B = offsets->dims[0] - 1, Hkv = k->dims[1], G = Hq / Hkv;
  PackedArgs a{q->ptr, (const uint16_t *)k->ptr, (const uint16_t *)v->ptr, (const int32_t *)offsets->ptr, out->ptr, T,
               (int)B, (int)Hq, (int)Hkv, (int)D, softmax_scale(scale, D), q->dtype == RXW8_F32,
               out->dtype == RXW8_F32, fill, G % 4 == 0 ? 4 : G % 2 == 0 ? 2 : 1};
  // Row tiles of a workgroup: 4 waves of 32 or 64 rows (kernels/packed.hip) over its
  // heads; at most one more than T's for each sequence
  const bool f32 = a.q_f32 || a.out_f32;
  const int64_t rows = (f32 || D > 64 ? 32 : 64) * (4 / a.heads);
  const int64_t grid = ((T + rows - 1) / rows + B) * (Hq / a.heads);
  if ((D != 64 && D != 128 && D != 256) || Hkv * D * 2 * 32 >= ((int64_t)1 << 31) || grid > grid_max(256) ||
      ((uintptr_t)a.q | (uintptr_t)a.k | (uintptr_t)a.v | (uintptr_t)a.out) % 16)
    return launch(rt, "rxw8_packed_prefill_any", dim3((unsigned)((T * Hq + 3) / 4)), dim3(256), a);
  if (fill) {
    int rc = launch(rt, "rxw8_packed_fill", dim3((unsigned)std::min<int64_t>((T * Hq * D + 255) / 256, 2048)), dim3(256), a);
    if (rc) return rc;
  }
  // Few rows: the kernel whose waves share a row's keys, 32 rows of one head to a workgroup, two
  // of them on a CU (one at D = 256). It needs no more rounds of workgroups than pay for steps
  // done a quarter at a time, by the sequences' mean length: 3/4 and one more for each 512 rows,
  // at most 2; or, for bf16 rows of 128 (whose tiles run two workgroups to a CU) and of 256, 2/5 and
  // one more for each 800, at most 1.05. In us, the tiles above and that one. 16 heads of 128, bf16: 8 x 100
  // rows 8.1, 8.6; 1 x 300 10.6, 9.4; 4 x 300 11.4, 16.6; 1 x 1000 21.9, 16.2; 2 x 1000 23.7, 27.8;
  // f32: 1 x 2000 78.3, 69.5; 4 x 500 27.9, 32.5. 16 of 256, f32: 1 x 1000 68.3, 59.9;
  // 1 x 1100 73.7, 78.3; 3 x 100 18.1, 16.7; 4 x 150 21.6, 29.3; bf16: 1 x 500 21.8, 19.1;
  // 1 x 850 31.4, 35.2. 32 of 64, bf16: 1 x 1000 23.1, 17.3; 1 x 2000 40.5, 43.2.
  const int64_t quarters = ((T + 31) / 32 + B) * Hq;
  const double likely = (T / 32.0 + B / 2.0) * (double)Hq, mean = (double)T / std::max<int64_t>(B, 1);
  const double rounds = !f32 && D > 64 ? std::min(0.4 + mean / 800, 1.05) : std::min(0.75 + mean / 512, 2.0);
  const bool few = likely <= rounds * (D == 256 ? 1 : 2) * rt->cus && quarters <= grid_max(256);
  const size_t tiles = (size_t)(2 * 4 * 32 * 2) * (size_t)D;  // K and V of 128 keys
  char kname[48];
  std::snprintf(kname, sizeof kname, "rxw8_packed_%s_%s_d%d", few ? "quarters" : "prefill",
                a.q_f32 ? "f32" : a.out_f32 ? "bf16_f32" : "bf16", (int)D);
  if (few)  // and the records' maxima and sums, and the third parts of an f32 q of 256
    return launch(rt, kname, dim3((unsigned)quarters), dim3(256), a, tiles + (2 << 10) + (a.q_f32 && D == 256 ? 16 << 10 : 0));
  return launch(rt, kname, dim3((unsigned)grid), dim3(256), a, a.q_f32 && D == 256 ? (size_t)160 << 10 : tiles);
}

}  // namespace rxw8

using namespace rxw8;

extern "C" {

int rxw8_paged_kv_append(rxw8_runtime *rt, rxw8_buffer *k_pages, rxw8_buffer *v_pages, rxw8_buffer *k,
                         rxw8_buffer *v, rxw8_buffer *table, rxw8_buffer *starts, rxw8_buffer *offsets) {
  if (!rt || !k_pages || !v_pages || !k || !v || !table || !starts)
    return fail(RXW8_INVALID_ARGUMENT, "paged KV append: NULL argument");
  if (int rc = check_pages("paged KV append", k_pages, v_pages, table)) return rc;
  if (k_pages == v_pages) return fail(RXW8_INVALID_ARGUMENT, "K and V pages must be distinct buffers");
  if (k->rank != 3 || !is_f(k->dtype) || !same_shape(k, v) || k->dims[1] != k_pages->dims[1] ||
      k->dims[2] != k_pages->dims[3])
    return fail(RXW8_INVALID_ARGUMENT, "paged KV append requires F32/BF16 k, v [T,Hkv,D] of the pages' heads and width");
  const int64_t T = k->dims[0], B = table->dims[0];
  if (!is_vec(starts, RXW8_I32, B)) return fail(RXW8_INVALID_ARGUMENT, "paged KV append: starts must be I32 [B]");
  if (offsets ? !is_vec(offsets, RXW8_I32, B + 1) : T != B)
    return fail(RXW8_INVALID_ARGUMENT, "paged KV append: offsets must be I32 [B+1] (without them k, v hold one row a sequence)");
  // a wave takes 128 pieces of 8 elements of a row, or a row of one head
  const int64_t parts = (k->dims[1] * k->dims[2] / 8 + 127) / 128;
  if (T > 4 * grid_max(256) / std::max(k->dims[1], parts))
    return fail(RXW8_UNIMPLEMENTED, "paged KV append: %lld rows exceed the kernel's grid", (long long)T);
  if (int rc = check_buffers("paged KV append", rt, {k_pages, v_pages, k, v, table, starts, offsets}, 2)) return rc;
  if (T == 0) return RXW8_OK;
  std::lock_guard<std::recursive_mutex> g(rt->mu);
  PagedAppendArgs a{k->ptr, v->ptr, k_pages->ptr, v_pages->ptr, (const int32_t *)table->ptr,
                    (const int32_t *)starts->ptr, offsets ? (const int32_t *)offsets->ptr : nullptr, T,
                    k_pages->dims[0], (int)B, (int)table->dims[1], (int)k->dims[1], (int)k->dims[2],
                    (int)k_pages->dims[2], k->dtype == RXW8_F32, k_pages->dtype == RXW8_F32};
  if (a.D % 8 || ((uintptr_t)a.k | (uintptr_t)a.v | (uintptr_t)a.kp | (uintptr_t)a.vp) & 15)
    return launch(rt, "rxw8_paged_append_any", dim3((unsigned)((T * a.Hkv + 3) / 4)), dim3(256), a);
  return launch(rt, "rxw8_paged_append", dim3((unsigned)((T * parts + 3) / 4)), dim3(256), a);
}

int rxw8_gqa_decode_paged_into(rxw8_runtime *rt, rxw8_buffer *q, rxw8_buffer *k_pages, rxw8_buffer *v_pages,
                               rxw8_buffer *table, rxw8_buffer *lens, float scale, rxw8_buffer *out) {
  if (!rt || !out) return fail(RXW8_INVALID_ARGUMENT, "NULL argument");
  if (int rc = check_paged_decode(q, k_pages, v_pages, table, lens, scale)) return rc;
  bool ok = is_f(out->dtype) && out->rank == 3;
  for (int i = 0; ok && i < 3; ++i) ok = out->dims[i] == q->dims[i];
  if (!ok) return fail(RXW8_INVALID_ARGUMENT, "paged GQA decode output: shape or dtype mismatch");
  if (int rc = check_buffers("paged GQA decode", rt, {out, q, k_pages, v_pages, table, lens}, 1)) return rc;
  const int64_t B = q->dims[0], Hq = q->dims[1], D = q->dims[2];
  if (B == 0) return RXW8_OK;
  std::lock_guard<std::recursive_mutex> g(rt->mu);
  PagedDecodeArgs a{q->ptr, k_pages->ptr, v_pages->ptr, (const int32_t *)table->ptr, (const int32_t *)lens->ptr,
                    out->ptr, k_pages->dims[0], (int)B, (int)table->dims[1], (int)Hq, (int)k_pages->dims[1], (int)D,
                    (int)k_pages->dims[2], softmax_scale(scale, D), q->dtype == RXW8_F32,
                    k_pages->dtype == RXW8_F32, out->dtype == RXW8_F32, 0, 0, nullptr, nullptr};
  return paged_decode_launch(rt, a);
}

int rxw8_gqa_decode_paged(rxw8_runtime *rt, rxw8_buffer *q, rxw8_buffer *k_pages, rxw8_buffer *v_pages,
                          rxw8_buffer *table, rxw8_buffer *lens, float scale, int out_dtype, rxw8_buffer **out) {
  if (!rt || !out) return fail(RXW8_INVALID_ARGUMENT, "NULL argument");
  if (int rc = check_paged_decode(q, k_pages, v_pages, table, lens, scale)) return rc;
  if (!is_f(out_dtype)) return fail(RXW8_INVALID_ARGUMENT, "GQA: out dtype must be F32 or BF16");
  if (int rc = check_buffers("paged GQA decode", rt, {q, k_pages, v_pages, table, lens}, 0)) return rc;
  std::lock_guard<std::recursive_mutex> g(rt->mu);
  Buffer *o = nullptr;
  int rc = new_buffer(rt, out_dtype, q->dims, 3, false, &o);
  if (rc) return rc;
  rc = rxw8_gqa_decode_paged_into(rt, q, k_pages, v_pages, table, lens, scale, static_cast<rxw8_buffer *>(o));
  if (rc) {
    rxw8_buffer_release(static_cast<rxw8_buffer *>(o));
    return rc;
  }
  *out = static_cast<rxw8_buffer *>(o);
  return RXW8_OK;
}

int rxw8_gqa_prefill_packed_into(rxw8_runtime *rt, rxw8_buffer *q, rxw8_buffer *k, rxw8_buffer *v,
                                 rxw8_buffer *offsets, float scale, rxw8_buffer *out) {
  if (!rt || !out) return fail(RXW8_INVALID_ARGUMENT, "NULL argument");
  if (int rc = check_packed(q, k, v, offsets, scale)) return rc;
  bool ok = is_f(out->dtype) && out->rank == 3;
  for (int i = 0; ok && i < 3; ++i) ok = out->dims[i] == q->dims[i];
  if (!ok) return fail(RXW8_INVALID_ARGUMENT, "packed GQA prefill output: shape or dtype mismatch");
  if (int rc = check_buffers("packed GQA prefill", rt, {out, q, k, v, offsets}, 1)) return rc;
  std::lock_guard<std::recursive_mutex> g(rt->mu);
  return packed_launch(rt, q, k, v, offsets, scale, out, false);
}

int rxw8_gqa_prefill_packed(rxw8_runtime *rt, rxw8_buffer *q, rxw8_buffer *k, rxw8_buffer *v, rxw8_buffer *offsets,
                            float scale, int out_dtype, rxw8_buffer **out) {
  if (!rt || !out) return fail(RXW8_INVALID_ARGUMENT, "NULL argument");
  if (int rc = check_packed(q, k, v, offsets, scale)) return rc;
  if (!is_f(out_dtype)) return fail(RXW8_INVALID_ARGUMENT, "GQA prefill: out dtype must be F32 or BF16");
  if (int rc = check_buffers("packed GQA prefill", rt, {q, k, v, offsets}, 0)) return rc;
  std::lock_guard<std::recursive_mutex> g(rt->mu);
  Buffer *o = nullptr;
  int rc = new_buffer(rt, out_dtype, q->dims, 3, false, &o);
  if (rc) return rc;
  rc = packed_launch(rt, q, k, v, offsets, scale, o, true);
  if (rc) {
    rxw8_buffer_release(static_cast<rxw8_buffer *>(o));
    return rc;
  }
  *out = static_cast<rxw8_buffer *>(o);
  return RXW8_OK;
}

static int check_sample(const Buffer *logits, const Buffer *uniform, const Buffer *temperature, const Buffer *top_k,
                        const Buffer *top_p, const Buffer *min_p) {
  if (!logits || !uniform) return fail(RXW8_INVALID_ARGUMENT, "sample: NULL buffer");
  if (logits->rank != 2 || !is_f(logits->dtype) || logits->dims[1] <= 0)
    return fail(RXW8_INVALID_ARGUMENT, "sample requires F32/BF16 logits [B,V] with V > 0");
  const int64_t B = logits->dims[0], V = logits->dims[1];
  if (!is_vec(uniform, RXW8_F32, B)) return fail(RXW8_INVALID_ARGUMENT, "sample: uniform must be F32 [B]");
  if ((temperature && !is_vec(temperature, RXW8_F32, B)) || (top_k && !is_vec(top_k, RXW8_I32, B)) ||
      (top_p && !is_vec(top_p, RXW8_F32, B)) || (min_p && !is_vec(min_p, RXW8_F32, B)))
    return fail(RXW8_INVALID_ARGUMENT, "sample: temperature, top_p and min_p must be F32 [B], top_k I32 [B]");
  if (V > ((int64_t)1 << 24)) return fail(RXW8_UNIMPLEMENTED, "sample: %lld words > 2^24", (long long)V);
  if (B > grid_max(1024)) return fail(RXW8_UNIMPLEMENTED, "sample: %lld rows exceed the kernel's grid", (long long)B);
  return RXW8_OK;
}

int rxw8_sample_into(rxw8_runtime *rt, rxw8_buffer *logits, rxw8_buffer *uniform, rxw8_buffer *temperature,
                     rxw8_buffer *top_k, rxw8_buffer *top_p, rxw8_buffer *min_p, rxw8_buffer *out) {
  if (!rt || !out) return fail(RXW8_INVALID_ARGUMENT, "NULL argument");
  if (int rc = check_sample(logits, uniform, temperature, top_k, top_p, min_p)) return rc;
  const int64_t B = logits->dims[0], V = logits->dims[1];
  if (!is_vec(out, RXW8_I32, B)) return fail(RXW8_INVALID_ARGUMENT, "sample output must be I32 [B]");
  if (int rc = check_buffers("sample", rt, {out, logits, uniform, temperature, top_k, top_p, min_p}, 1)) return rc;
  if (B == 0) return RXW8_OK;
  int bits = 0;  // ceil(log2 V)
  while (((int64_t)1 << bits) < V) ++bits;
  std::lock_guard<std::recursive_mutex> g(rt->mu);
  SampleArgs a{logits->ptr, (const float *)uniform->ptr, temperature ? (const float *)temperature->ptr : nullptr,
               top_k ? (const int32_t *)top_k->ptr : nullptr, top_p ? (const float *)top_p->ptr : nullptr,
               min_p ? (const float *)min_p->ptr : nullptr, (int32_t *)out->ptr, V, 62 - bits > 51 ? 51 : 62 - bits,
               logits->dtype == RXW8_BF16, 1, V, nullptr, nullptr, nullptr, nullptr};
  // Workgroups to a row: as many as leave one to a CU, but no more than 8, whose bins one joins;
  // or one, where sharing spares it fewer than 48 Ki words, the price of two more launches. Of 16
  // rows, one against 8 to a row, no top_k: 27 and 33 us at 32000 words, 42 and 34 at 64000, 57 and
  // 36 at 100000; of 100 rows, one against 2: 30 and 38, 48 and 48, 69 and 58 us.
  a.S = (int)std::max<int64_t>(1, std::min<int64_t>(8, rt->cus / B));
  if (V - V / a.S < 48 << 10) a.S = 1;
  a.chunk = (V + a.S - 1) / a.S;
  if (a.S > 1) {
    char *block = rt->f32_attn[stream_capturing(rt) ? 1 : 0];
    a.arrivals = (int *)block;
    a.listed = a.arrivals + B;
    a.extremes = block + RXW8_NOALLOC_COUNTER_BYTES;
    a.bins = a.extremes + (64 << 10);
    if (a.S * B * kSampleExtremes > (64 << 10) || a.S * B * kSampleBins > (int64_t)RXW8_NOALLOC_PARTIAL_BYTES - (64 << 10))
      a.S = 1, a.chunk = V;
  }
  if (a.S > 1) {
    int rc = launch(rt, "rxw8_sample_extremes", dim3((unsigned)(B * a.S)), dim3(1024), a, kSampleLds);
    if (rc) return rc;
  }
  int rc = launch(rt, "rxw8_sample_draw", dim3((unsigned)(B * a.S)), dim3(1024), a, kSampleLds);
  if (rc || a.S == 1) return rc;
  return launch(rt, "rxw8_sample_words", dim3((unsigned)(B * a.S)), dim3(1024), a, kSampleLds);
}

int rxw8_sample(rxw8_runtime *rt, rxw8_buffer *logits, rxw8_buffer *uniform, rxw8_buffer *temperature,
                rxw8_buffer *top_k, rxw8_buffer *top_p, rxw8_buffer *min_p, rxw8_buffer **out) {
  if (!rt || !out) return fail(RXW8_INVALID_ARGUMENT, "NULL argument");
  if (int rc = check_sample(logits, uniform, temperature, top_k, top_p, min_p)) return rc;
  if (int rc = check_buffers("sample", rt, {logits, uniform, temperature, top_k, top_p, min_p}, 0)) return rc;
  std::lock_guard<std::recursive_mutex> g(rt->mu);
  Buffer *o = nullptr;
  int rc = new_buffer(rt, RXW8_I32, logits->dims, 1, false, &o);
  if (rc) return rc;
  rc = rxw8_sample_into(rt, logits, uniform, temperature, top_k, top_p, min_p, static_cast<rxw8_buffer *>(o));
  if (rc) {
    rxw8_buffer_release(static_cast<rxw8_buffer *>(o));
    return rc;
  }
  *out = static_cast<rxw8_buffer *>(o);
  return RXW8_OK;
}

}  // extern "C"
