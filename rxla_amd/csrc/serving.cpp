// The serving operators: the paged key/value cache (append, reading back, decode
// attention, over a shared prefix too; in 8 bits too), causal attention of packed
// prompts, the logits' adjustments and sampling of the next token.
#include <algorithm>
#include <cmath>
#include <cstdint>
#include <cstdio>

#include "internal.h"

namespace rxw8 {

// (the kernels' argument structs: kernels/paged.h, paged.hip, paged_q8.hip, shared.hip,
// packed.hip, logits.hip, sample.hip)
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
  const float *ks, *vs;
};
struct PagedQ8Args {
  const void *k, *v;
  uint8_t *kp, *vp;
  float *ks, *vs;
  const int32_t *table, *starts, *offsets;
  int64_t T, P;
  int B, M, Hkv, D, ps;
  int k_f32;
};
struct PagedReadArgs {
  const void *kp, *vp;
  const float *ks, *vs;
  void *k, *v;
  const int32_t *table, *starts, *offsets;
  int64_t T, P;
  int B, M, Hkv, D, ps;
  int kind;
  int k_f32;
};
struct SharedArgs {
  PagedDecodeArgs d;
  const int32_t *prefixes, *prefix_lens, *groups;
  int N, MP;
  int b0;
  int kind;
  float *own, *whole, *parts;
  int *plan;
  int columns, keys;
};
struct LogitsArgs {
  const void *logits;
  void *out;
  const int32_t *tokens, *offsets, *prompts;
  const float *repetition, *frequency, *presence;
  const int32_t *bias_words;
  const float *bias;
  const int32_t *bias_offsets;
  const uint32_t *mask;
  const int32_t *mask_rows;
  int64_t T, E, R, V;
  int in_f32, out_f32;
  int chunk, chunks;
  int given;
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
constexpr int64_t kLogitsChunk = 4096;   // words of a workgroup, 8 a thread
constexpr size_t kLogitsValues = 512;    // biases that it keeps in LDS
static int page_kind(const Buffer *pages) { return pages->dtype == RXW8_U8 ? 2 : pages->dtype == RXW8_F32 ? 1 : 0; }

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

// A page table I32 [B, M] over pages of `ps` positions
static int check_table(const char *what, const Buffer *table, int64_t ps) {
  if (table->dtype != RXW8_I32 || table->rank != 2)
    return fail(RXW8_INVALID_ARGUMENT, "%s: the page table must be I32 [B,M]", what);
  // positions are I32
  if (table->dims[0] > INT32_MAX || (table->dims[1] > 0 && ps > INT32_MAX / table->dims[1]))
    return fail(RXW8_UNIMPLEMENTED, "%s: %lld pages of %lld positions exceed 32-bit positions", what,
                (long long)table->dims[1], (long long)ps);
  return RXW8_OK;
}

// Pages [P, Hkv, ps, D] F32|BF16, or U8 with scales F32 [P, Hkv, ps], and the table I32 [B, M]
static int check_pages(const char *what, const Buffer *kp, const Buffer *vp, const Buffer *table,
                       const Buffer *ks = nullptr, const Buffer *vs = nullptr) {
  const bool codes = ks || vs;
  if (kp->rank != 4 || !(codes ? kp->dtype == RXW8_U8 : is_f(kp->dtype)) || !same_shape(kp, vp))
    return fail(RXW8_INVALID_ARGUMENT, "%s: pages must be two %s [P,Hkv,ps,D] of one shape and type", what,
                codes ? "U8" : "F32/BF16");
  if (kp->dims[1] <= 0 || kp->dims[2] <= 0 || kp->dims[3] <= 0)
    return fail(RXW8_INVALID_ARGUMENT, "%s: pages %s need positive heads, rows and width", what, dims_str(kp).c_str());
  if (codes) {
    bool ok = ks && vs && ks->dtype == RXW8_F32 && ks->rank == 3 && same_shape(ks, vs);
    for (int i = 0; ok && i < 3; ++i) ok = ks->dims[i] == kp->dims[i];
    if (!ok) return fail(RXW8_INVALID_ARGUMENT, "%s: 8-bit pages need two F32 [P,Hkv,ps] of scales", what);
  }
  for (int i = 1; i < 4; ++i)
    if (kp->dims[i] > INT32_MAX) return fail(RXW8_UNIMPLEMENTED, "%s: pages %s", what, dims_str(kp).c_str());
  return check_table(what, table, kp->dims[2]);
}

// Waves of a row [Hkv, D]: 128 pieces of 8 elements each
static int64_t row_parts(const Buffer *k) { return (k->dims[1] * k->dims[2] / 8 + 127) / 128; }

// Rows k, v F32|BF16 [T, Hkv, D] of the pages' heads and width, their sequences' first
// positions I32 [B] and the rows of each I32 [B + 1] (NULL: one each). A wave takes a part
// of a row, or a row of one head.
static int check_rows(const char *what, const Buffer *kp, const Buffer *k, const Buffer *v, const Buffer *table,
                      const Buffer *starts, const Buffer *offsets) {
  if (k->rank != 3 || !is_f(k->dtype) || !same_shape(k, v) || k->dims[1] != kp->dims[1] || k->dims[2] != kp->dims[3])
    return fail(RXW8_INVALID_ARGUMENT, "%s requires F32/BF16 k, v [T,Hkv,D] of the pages' heads and width", what);
  const int64_t T = k->dims[0], B = table->dims[0];
  if (!is_vec(starts, RXW8_I32, B)) return fail(RXW8_INVALID_ARGUMENT, "%s: starts must be I32 [B]", what);
  if (offsets ? !is_vec(offsets, RXW8_I32, B + 1) : T != B)
    return fail(RXW8_INVALID_ARGUMENT, "%s: offsets must be I32 [B+1] (without them k, v hold one row a sequence)", what);
  if (T > 4 * grid_max(256) / std::max(k->dims[1], row_parts(k)))
    return fail(RXW8_UNIMPLEMENTED, "%s: %lld rows exceed the kernel's grid", what, (long long)T);
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

static int check_decode(const char *what, const Buffer *q, const Buffer *kp, const Buffer *table, const Buffer *lens,
                        float scale) {
  if (q->rank != 3 || !is_f(q->dtype)) return fail(RXW8_INVALID_ARGUMENT, "%s requires F32/BF16 q [B,Hq,D]", what);
  const int64_t B = q->dims[0], Hq = q->dims[1], D = q->dims[2];
  if (table->dims[0] != B || D != kp->dims[3])
    return fail(RXW8_INVALID_ARGUMENT, "%s: q, page table and pages differ in batch or head width", what);
  if (Hq <= 0 || Hq % kp->dims[1] != 0)
    return fail(RXW8_INVALID_ARGUMENT, "GQA requires equal batch prefixes and divisible positive head counts");
  if (!is_vec(lens, RXW8_I32, B)) return fail(RXW8_INVALID_ARGUMENT, "%s: lens must be I32 [B]", what);
  if (int rc = check_scale(scale)) return rc;
  if (D > kAnyMaxD) return fail(RXW8_UNIMPLEMENTED, "%s: head dim %lld > 512", what, (long long)D);
  if (Hq > INT32_MAX || B > grid_max(256) / Hq)
    return fail(RXW8_UNIMPLEMENTED, "%s: %lld x %lld rows exceed the kernel's grid", what, (long long)B, (long long)Hq);
  return RXW8_OK;
}
static int check_paged_decode(const Buffer *q, const Buffer *kp, const Buffer *vp, const Buffer *table,
                              const Buffer *lens, float scale) {
  if (!q || !kp || !vp || !table || !lens) return fail(RXW8_INVALID_ARGUMENT, "paged GQA decode: NULL buffer");
  if (int rc = check_pages("paged GQA decode", kp, vp, table)) return rc;
  return check_decode("paged GQA decode", q, kp, table, lens, scale);
}
static int check_paged_decode_q8(const Buffer *q, const Buffer *kp, const Buffer *vp, const Buffer *ks, const Buffer *vs,
                                 const Buffer *table, const Buffer *lens, float scale) {
  const char *what = "8-bit paged GQA decode";
  if (!q || !kp || !vp || !ks || !vs || !table || !lens) return fail(RXW8_INVALID_ARGUMENT, "%s: NULL buffer", what);
  if (int rc = check_pages(what, kp, vp, table, ks, vs)) return rc;
  return check_decode(what, q, kp, table, lens, scale);
}
static int check_shared(const Buffer *q, const Buffer *kp, const Buffer *vp, const Buffer *ks, const Buffer *vs,
                        const Buffer *prefixes, const Buffer *prefix_lens, const Buffer *groups, const Buffer *table,
                        const Buffer *lens, float scale) {
  const char *what = "GQA decode over shared prefixes";
  if (!q || !kp || !vp || !prefixes || !prefix_lens || !groups || !table || !lens)
    return fail(RXW8_INVALID_ARGUMENT, "%s: NULL buffer", what);
  if (int rc = check_pages(what, kp, vp, table, ks, vs)) return rc;
  if (int rc = check_table(what, prefixes, kp->dims[2])) return rc;
  const int64_t N = prefixes->dims[0];
  if (!is_vec(prefix_lens, RXW8_I32, N) || !is_vec(groups, RXW8_I32, N + 1))
    return fail(RXW8_INVALID_ARGUMENT, "%s: prefix_lens must be I32 [N] and groups I32 [N+1] for prefixes I32 [N,M]", what);
  return check_decode(what, q, kp, table, lens, scale);
}
static bool is_output(const Buffer *out, const Buffer *q) {  // F32|BF16 of q's shape
  bool ok = is_f(out->dtype) && out->rank == q->rank;
  for (int i = 0; ok && i < q->rank; ++i) ok = out->dims[i] == q->dims[i];
  return ok;
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

// PagedTile (kernels/paged_decode.h): a tile's keys, and the bytes of a wave's K, V and scales
struct PagedTiles {
  int keys, ring;
  PagedTiles(int kind, int64_t D) {  // kind: page_kind
    const int row = (int)D * (kind == 2 ? 1 : kind == 1 ? 4 : 2);
    keys = kind == 2 ? (D == 64 ? 64 : 32) : row < 256 ? 32 : 16;
    ring = 2 * keys * row + (kind == 2 ? 8 * keys : 0);
  }
};

// The matrix-core kernels take head widths 64, 128 and 256, pages of whole 16-row
// pieces, 16-byte aligned operands and tile counts within 32 bits; else the plain
// kernel. As many waves walk keys, up to 8, as tiles and records of the group's heads
// fit in LDS. `units` workgroups for each kv head (and 16 query heads): the number that
// leaves the fewest CUs idle in the last round.
static int paged_decode_launch(Runtime *rt, PagedDecodeArgs a) {
  const int64_t G = a.Hq / a.Hkv, heads = a.Hkv * ((G + 15) / 16), gcap = G < 16 ? G : 16;
  const PagedTiles t(a.ks ? 2 : a.p_f32, a.D);
  if ((a.D != 64 && a.D != 128 && a.D != 256) || a.ps % 16 || a.P == 0 || heads > 4096 ||
      ((uintptr_t)a.q | (uintptr_t)a.kp | (uintptr_t)a.vp | (uintptr_t)a.out) % 16 ||
      (int64_t)a.B * (((int64_t)a.M * a.ps + t.keys - 1) / t.keys) >= ((int64_t)1 << 30))
    return launch(rt, a.ks ? "rxw8_q8_decode_any" : "rxw8_paged_decode_any", dim3((unsigned)a.B * (unsigned)a.Hq), dim3(256), a);
  const size_t record = (size_t)gcap * (size_t)(a.D + 4) * sizeof(float), wave = std::max((size_t)t.ring, record) + record;
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
  if (a.ks) std::snprintf(kname, sizeof kname, "rxw8_q8_decode%s_d%d", a.q_f32 || a.out_f32 ? "_high" : "", a.D);
  else std::snprintf(kname, sizeof kname, "rxw8_paged_decode_%s_d%d", a.p_f32 ? "f32" : "bf16", a.D);
  return launch(rt, kname, dim3((unsigned)(heads * a.units)), dim3(512), a, wave * (size_t)a.waves);
}

// The matrix-core kernels on paged decode's terms. Records of parts take at most 12 MiB of the
// runtime's block (all of it where a single one is larger), those of rows the rest: a
// batch with more rows than fit goes in several launches of the two.
static int shared_launch(Runtime *rt, SharedArgs a) {
  PagedDecodeArgs &d = a.d;
  const int64_t G = d.Hq / d.Hkv, HT = (G + 15) / 16, heads = d.Hkv * HT, rec = (int64_t)(d.D + 4) * sizeof(float);
  const PagedTiles t(a.kind, d.D);
  // block_tiles (kernels/shared.hip)
  const bool high = (d.q_f32 || d.out_f32) && a.kind != 1;
  const int ct = d.D == 256 ? 1 : d.D == 128 ? (high ? 1 : 2) : high || a.kind == 2 ? 2 : 4;
  // prefix_keys (kernels/shared.hip)
  a.keys = a.kind == 2 ? (d.D == 256 ? 32 : 64) : a.kind == 1 || d.D == 256 ? 16 : 32;
  a.columns = 16 * ct;
  const int row = d.D * (a.kind == 2 ? 1 : a.kind == 1 ? 4 : 2), ring = 2 * a.keys * row + (a.kind == 2 ? 8 * a.keys : 0);
  auto tiles = [&](int64_t m) { return (m * d.ps + std::min(t.keys, a.keys) - 1) / std::min(t.keys, a.keys); };
  const int64_t blocks = (int64_t)d.B * G / a.columns + a.N;
  bool any = (d.D != 64 && d.D != 128 && d.D != 256) || d.ps % 16 || d.P == 0 || heads > 4096 || a.N == 0 || a.MP == 0 ||
             ((uintptr_t)d.q | (uintptr_t)d.kp | (uintptr_t)d.vp | (uintptr_t)d.out) % 16 ||
             tiles(d.M) >= ((int64_t)1 << 30) / d.B || tiles(a.MP) >= ((int64_t)1 << 30) / blocks;
  const size_t record = (size_t)std::min<int64_t>(G, 16) * (size_t)rec;
  // LDS of a wave: its own keys' ring and two records, or a prefix's ring and, over that, 16 of a block's records
  const size_t wave = std::max(std::max((size_t)t.ring, record) + record, (size_t)std::max<int64_t>(ring, 16 * rec));
  d.waves = (int)std::min<size_t>(8, (rt->lds_max - 1024) / wave);
  const int64_t block = (int64_t)RXW8_NOALLOC_PARTIAL_BYTES - 1024;
  auto round = [](int64_t x) { return (x + 1023) & ~(int64_t)1023; };
  const int64_t own_part = round((int64_t)record), prefix_part = a.columns * rec;
  auto parts = [&](int64_t units) { return round(2 * heads * units * own_part) + round(2 * heads * units * prefix_part); };
  d.units = 1;
  for (int64_t u = 2; u <= std::min<int64_t>(256, (int64_t)(RXW8_NOALLOC_COUNTER_BYTES / sizeof(int)) / heads) && parts(u) <= 12 << 20; ++u) {
    const int64_t r0 = (heads * d.units + rt->cus - 1) / rt->cus, r1 = (heads * u + rt->cus - 1) / rt->cus;
    if (r1 * d.units < r0 * u) d.units = (int)u;
  }
  const int64_t most = (block - parts(d.units)) / (2 * rec * d.Hq);
  if (any || most < 1) return launch(rt, "rxw8_shared_any", dim3((unsigned)d.B * (unsigned)d.Hq), dim3(256), a);
  const int64_t launches = (d.B + most - 1) / most, each = (d.B + launches - 1) / launches;
  char *const at = rt->f32_attn[stream_capturing(rt) ? 1 : 0], *const recs = at + RXW8_NOALLOC_COUNTER_BYTES + 1024;
  d.counters = (int *)at;
  a.plan = (int *)(at + RXW8_NOALLOC_COUNTER_BYTES);
  d.part = (float *)recs;
  a.parts = (float *)(recs + round(2 * heads * d.units * own_part));
  a.own = (float *)(recs + parts(d.units));
  a.whole = a.own + each * d.Hq * (d.D + 4);
  char kname[40];
  std::snprintf(kname, sizeof kname, "rxw8_shared_%s%s_d%d", a.kind == 2 ? "q8" : a.kind == 1 ? "f32" : "bf16", high ? "_high" : "", d.D);
  const int64_t B = d.B, q_size = d.q_f32 ? 4 : 2, out_size = d.out_f32 ? 4 : 2;
  for (int64_t b0 = 0; b0 < B; b0 += each) {
    SharedArgs c = a;
    c.b0 = (int)b0;
    c.d.B = (int)std::min(each, B - b0);
    c.d.q = (const char *)d.q + b0 * d.Hq * d.D * q_size;
    c.d.out = (char *)d.out + b0 * d.Hq * d.D * out_size;
    c.d.table = d.table + b0 * d.M;
    c.d.lens = d.lens + b0;
    if (int rc = launch(rt, kname, dim3((unsigned)(heads * d.units)), dim3(512), c, wave * (size_t)d.waves)) return rc;
    if (int rc = launch(rt, "rxw8_shared_join", dim3((unsigned)(((int64_t)c.d.B * d.Hq + 3) / 4)), dim3(256), c)) return rc;
  }
  return RXW8_OK;
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
  if (int rc = check_rows("paged KV append", k_pages, k, v, table, starts, offsets)) return rc;
  const int64_t T = k->dims[0], B = table->dims[0], parts = row_parts(k);
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
                    k_pages->dtype == RXW8_F32, out->dtype == RXW8_F32, 0, 0, nullptr, nullptr, nullptr, nullptr};
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

int rxw8_paged_kv_append_q8(rxw8_runtime *rt, rxw8_buffer *k_pages, rxw8_buffer *v_pages, rxw8_buffer *k_scales,
                            rxw8_buffer *v_scales, rxw8_buffer *k, rxw8_buffer *v, rxw8_buffer *table,
                            rxw8_buffer *starts, rxw8_buffer *offsets) {
  const char *what = "8-bit paged KV append";
  if (!rt || !k_pages || !v_pages || !k_scales || !v_scales || !k || !v || !table || !starts)
    return fail(RXW8_INVALID_ARGUMENT, "%s: NULL argument", what);
  if (int rc = check_pages(what, k_pages, v_pages, table, k_scales, v_scales)) return rc;
  if (k_pages == v_pages || k_scales == v_scales)
    return fail(RXW8_INVALID_ARGUMENT, "K and V pages and scales must be distinct buffers");
  if (int rc = check_rows(what, k_pages, k, v, table, starts, offsets)) return rc;
  if (int rc = check_buffers(what, rt, {k_pages, v_pages, k_scales, v_scales, k, v, table, starts, offsets}, 4)) return rc;
  const int64_t T = k->dims[0];
  if (T == 0) return RXW8_OK;
  std::lock_guard<std::recursive_mutex> g(rt->mu);
  PagedQ8Args a{k->ptr, v->ptr, (uint8_t *)k_pages->ptr, (uint8_t *)v_pages->ptr, (float *)k_scales->ptr,
                (float *)v_scales->ptr, (const int32_t *)table->ptr, (const int32_t *)starts->ptr,
                offsets ? (const int32_t *)offsets->ptr : nullptr, T, k_pages->dims[0], (int)table->dims[0],
                (int)table->dims[1], (int)k->dims[1], (int)k->dims[2], (int)k_pages->dims[2], k->dtype == RXW8_F32};
  if ((a.D != 64 && a.D != 128 && a.D != 256 && a.D != 512) || row_parts(k) > 65535 ||
      ((uintptr_t)a.k | (uintptr_t)a.v | (uintptr_t)a.kp | (uintptr_t)a.vp) & 15)
    return launch(rt, "rxw8_q8_append_any", dim3((unsigned)((T * a.Hkv + 3) / 4)), dim3(256), a);
  return launch(rt, "rxw8_q8_append", dim3((unsigned)((T + 3) / 4), (unsigned)row_parts(k)), dim3(256), a);
}

int rxw8_paged_kv_read(rxw8_runtime *rt, rxw8_buffer *k_pages, rxw8_buffer *v_pages, rxw8_buffer *k_scales,
                       rxw8_buffer *v_scales, rxw8_buffer *table, rxw8_buffer *starts, rxw8_buffer *offsets,
                       rxw8_buffer *k, rxw8_buffer *v) {
  const char *what = "paged KV read";
  if (!rt || !k_pages || !v_pages || !k || !v || !table || !starts)
    return fail(RXW8_INVALID_ARGUMENT, "%s: NULL argument", what);
  if (int rc = check_pages(what, k_pages, v_pages, table, k_scales, v_scales)) return rc;
  if (k == v) return fail(RXW8_INVALID_ARGUMENT, "%s: k and v must be distinct buffers", what);
  if (int rc = check_rows(what, k_pages, k, v, table, starts, offsets)) return rc;
  if (int rc = check_buffers(what, rt, {k, v, k_pages, v_pages, k_scales, v_scales, table, starts, offsets}, 2)) return rc;
  const int64_t T = k->dims[0];
  if (T == 0) return RXW8_OK;
  std::lock_guard<std::recursive_mutex> g(rt->mu);
  PagedReadArgs a{k_pages->ptr, v_pages->ptr, k_scales ? (const float *)k_scales->ptr : nullptr,
                  v_scales ? (const float *)v_scales->ptr : nullptr, k->ptr, v->ptr, (const int32_t *)table->ptr,
                  (const int32_t *)starts->ptr, offsets ? (const int32_t *)offsets->ptr : nullptr, T,
                  k_pages->dims[0], (int)table->dims[0], (int)table->dims[1], (int)k->dims[1], (int)k->dims[2],
                  (int)k_pages->dims[2], page_kind(k_pages), k->dtype == RXW8_F32};
  if (a.D % 8 || row_parts(k) > 65535 || ((uintptr_t)a.k | (uintptr_t)a.v | (uintptr_t)a.kp | (uintptr_t)a.vp) & 15)
    return launch(rt, "rxw8_q8_read_any", dim3((unsigned)((T * a.Hkv + 3) / 4)), dim3(256), a);
  return launch(rt, "rxw8_q8_read", dim3((unsigned)((T + 3) / 4), (unsigned)row_parts(k)), dim3(256), a);
}

int rxw8_gqa_decode_paged_q8_into(rxw8_runtime *rt, rxw8_buffer *q, rxw8_buffer *k_pages, rxw8_buffer *v_pages,
                                  rxw8_buffer *k_scales, rxw8_buffer *v_scales, rxw8_buffer *table, rxw8_buffer *lens,
                                  float scale, rxw8_buffer *out) {
  const char *what = "8-bit paged GQA decode";
  if (!rt || !out) return fail(RXW8_INVALID_ARGUMENT, "NULL argument");
  if (int rc = check_paged_decode_q8(q, k_pages, v_pages, k_scales, v_scales, table, lens, scale)) return rc;
  if (!is_output(out, q)) return fail(RXW8_INVALID_ARGUMENT, "%s output: shape or dtype mismatch", what);
  if (int rc = check_buffers(what, rt, {out, q, k_pages, v_pages, k_scales, v_scales, table, lens}, 1)) return rc;
  const int64_t B = q->dims[0], Hq = q->dims[1], D = q->dims[2];
  if (B == 0) return RXW8_OK;
  std::lock_guard<std::recursive_mutex> g(rt->mu);
  PagedDecodeArgs a{q->ptr, k_pages->ptr, v_pages->ptr, (const int32_t *)table->ptr, (const int32_t *)lens->ptr,
                    out->ptr, k_pages->dims[0], (int)B, (int)table->dims[1], (int)Hq, (int)k_pages->dims[1], (int)D,
                    (int)k_pages->dims[2], softmax_scale(scale, D), q->dtype == RXW8_F32, 0, out->dtype == RXW8_F32,
                    0, 0, nullptr, nullptr, (const float *)k_scales->ptr, (const float *)v_scales->ptr};
  return paged_decode_launch(rt, a);
}

int rxw8_gqa_decode_paged_q8(rxw8_runtime *rt, rxw8_buffer *q, rxw8_buffer *k_pages, rxw8_buffer *v_pages,
                             rxw8_buffer *k_scales, rxw8_buffer *v_scales, rxw8_buffer *table, rxw8_buffer *lens,
                             float scale, int out_dtype, rxw8_buffer **out) {
  if (!rt || !out) return fail(RXW8_INVALID_ARGUMENT, "NULL argument");
  if (int rc = check_paged_decode_q8(q, k_pages, v_pages, k_scales, v_scales, table, lens, scale)) return rc;
  if (!is_f(out_dtype)) return fail(RXW8_INVALID_ARGUMENT, "GQA: out dtype must be F32 or BF16");
  if (int rc = check_buffers("8-bit paged GQA decode", rt, {q, k_pages, v_pages, k_scales, v_scales, table, lens}, 0)) return rc;
  std::lock_guard<std::recursive_mutex> g(rt->mu);
  Buffer *o = nullptr;
  int rc = new_buffer(rt, out_dtype, q->dims, 3, false, &o);
  if (rc) return rc;
  rc = rxw8_gqa_decode_paged_q8_into(rt, q, k_pages, v_pages, k_scales, v_scales, table, lens, scale,
                                     static_cast<rxw8_buffer *>(o));
  if (rc) {
    rxw8_buffer_release(static_cast<rxw8_buffer *>(o));
    return rc;
  }
  *out = static_cast<rxw8_buffer *>(o);
  return RXW8_OK;
}

int rxw8_gqa_decode_shared_into(rxw8_runtime *rt, rxw8_buffer *q, rxw8_buffer *k_pages, rxw8_buffer *v_pages,
                                rxw8_buffer *k_scales, rxw8_buffer *v_scales, rxw8_buffer *prefixes,
                                rxw8_buffer *prefix_lens, rxw8_buffer *groups, rxw8_buffer *table, rxw8_buffer *lens,
                                float scale, rxw8_buffer *out) {
  const char *what = "GQA decode over shared prefixes";
  if (!rt || !out) return fail(RXW8_INVALID_ARGUMENT, "NULL argument");
  if (int rc = check_shared(q, k_pages, v_pages, k_scales, v_scales, prefixes, prefix_lens, groups, table, lens, scale)) return rc;
  if (!is_output(out, q)) return fail(RXW8_INVALID_ARGUMENT, "%s output: shape or dtype mismatch", what);
  if (int rc = check_buffers(what, rt, {out, q, k_pages, v_pages, k_scales, v_scales, prefixes, prefix_lens, groups, table, lens}, 1))
    return rc;
  const int64_t B = q->dims[0], Hq = q->dims[1], D = q->dims[2];
  if (B == 0) return RXW8_OK;
  std::lock_guard<std::recursive_mutex> g(rt->mu);
  PagedDecodeArgs d{q->ptr, k_pages->ptr, v_pages->ptr, (const int32_t *)table->ptr, (const int32_t *)lens->ptr,
                    out->ptr, k_pages->dims[0], (int)B, (int)table->dims[1], (int)Hq, (int)k_pages->dims[1], (int)D,
                    (int)k_pages->dims[2], softmax_scale(scale, D), q->dtype == RXW8_F32, k_pages->dtype == RXW8_F32,
                    out->dtype == RXW8_F32, 0, 0, nullptr, nullptr, k_scales ? (const float *)k_scales->ptr : nullptr,
                    v_scales ? (const float *)v_scales->ptr : nullptr};
  return shared_launch(rt, SharedArgs{d, (const int32_t *)prefixes->ptr, (const int32_t *)prefix_lens->ptr,
                                      (const int32_t *)groups->ptr, (int)prefixes->dims[0], (int)prefixes->dims[1], 0,
                                      page_kind(k_pages), nullptr, nullptr, nullptr, nullptr, 0, 0});
}

int rxw8_gqa_decode_shared(rxw8_runtime *rt, rxw8_buffer *q, rxw8_buffer *k_pages, rxw8_buffer *v_pages,
                           rxw8_buffer *k_scales, rxw8_buffer *v_scales, rxw8_buffer *prefixes,
                           rxw8_buffer *prefix_lens, rxw8_buffer *groups, rxw8_buffer *table, rxw8_buffer *lens,
                           float scale, int out_dtype, rxw8_buffer **out) {
  if (!rt || !out) return fail(RXW8_INVALID_ARGUMENT, "NULL argument");
  if (int rc = check_shared(q, k_pages, v_pages, k_scales, v_scales, prefixes, prefix_lens, groups, table, lens, scale)) return rc;
  if (!is_f(out_dtype)) return fail(RXW8_INVALID_ARGUMENT, "GQA: out dtype must be F32 or BF16");
  if (int rc = check_buffers("GQA decode over shared prefixes", rt,
                             {q, k_pages, v_pages, k_scales, v_scales, prefixes, prefix_lens, groups, table, lens}, 0))
    return rc;
  std::lock_guard<std::recursive_mutex> g(rt->mu);
  Buffer *o = nullptr;
  int rc = new_buffer(rt, out_dtype, q->dims, 3, false, &o);
  if (rc) return rc;
  rc = rxw8_gqa_decode_shared_into(rt, q, k_pages, v_pages, k_scales, v_scales, prefixes, prefix_lens, groups, table,
                                   lens, scale, static_cast<rxw8_buffer *>(o));
  if (rc) {
    rxw8_buffer_release(static_cast<rxw8_buffer *>(o));
    return rc;
  }
  *out = static_cast<rxw8_buffer *>(o);
  return RXW8_OK;
}

static int check_logits(const rxw8_logits_options *o, const Buffer *logits) {
  const char *what = "logits adjustment";
  if (!logits || !o) return fail(RXW8_INVALID_ARGUMENT, "%s: NULL argument", what);
  if (logits->rank != 2 || !is_f(logits->dtype) || logits->dims[1] <= 0)
    return fail(RXW8_INVALID_ARGUMENT, "%s requires F32/BF16 logits [B,V] with V > 0", what);
  const int64_t B = logits->dims[0], V = logits->dims[1];
  if (!o->tokens != !o->offsets || (!o->tokens && (o->prompts || o->repetition || o->frequency || o->presence)))
    return fail(RXW8_INVALID_ARGUMENT, "%s: prompts and penalties need tokens and their offsets", what);
  if (o->tokens && (o->tokens->dtype != RXW8_I32 || o->tokens->rank != 1 || !is_vec(o->offsets, RXW8_I32, B + 1) ||
                    (o->prompts && !is_vec(o->prompts, RXW8_I32, B))))
    return fail(RXW8_INVALID_ARGUMENT, "%s: tokens must be I32 [T], offsets I32 [B+1], prompts I32 [B]", what);
  for (const rxw8_buffer *x : {o->repetition, o->frequency, o->presence})
    if (x && !is_vec(x, RXW8_F32, B))
      return fail(RXW8_INVALID_ARGUMENT, "%s: repetition, frequency and presence must be F32 [B]", what);
  if (!o->bias != !o->bias_words || !o->bias != !o->bias_offsets)
    return fail(RXW8_INVALID_ARGUMENT, "%s: biases need bias_words, bias and bias_offsets", what);
  if (o->bias && (o->bias->rank != 1 || !is_vec(o->bias, RXW8_F32, o->bias->dims[0]) ||
                  !is_vec(o->bias_words, RXW8_I32, o->bias->dims[0]) || !is_vec(o->bias_offsets, RXW8_I32, B + 1)))
    return fail(RXW8_INVALID_ARGUMENT, "%s: bias_words must be I32 [E], bias F32 [E], bias_offsets I32 [B+1]", what);
  if (o->mask_rows && !o->mask) return fail(RXW8_INVALID_ARGUMENT, "%s: mask_rows need a mask", what);
  if (o->mask && (o->mask->dtype != RXW8_I32 || o->mask->rank != 2 || o->mask->dims[1] != (V + 31) / 32 ||
                  (o->mask_rows ? !is_vec(o->mask_rows, RXW8_I32, B) : o->mask->dims[0] != B)))
    return fail(RXW8_INVALID_ARGUMENT, "%s: mask must be I32 [R,(V+31)/32] and mask_rows I32 [B] (without them R = B)", what);
  if (V > ((int64_t)1 << 24)) return fail(RXW8_UNIMPLEMENTED, "%s: %lld words > 2^24", what, (long long)V);
  for (const rxw8_buffer *x : {o->tokens, o->bias})
    if (x && x->dims[0] > INT32_MAX)
      return fail(RXW8_UNIMPLEMENTED, "%s: %lld entries exceed 32-bit offsets", what, (long long)x->dims[0]);
  if (B > grid_max(kLogitsChunk / 8) / ((V + kLogitsChunk - 1) / kLogitsChunk))
    return fail(RXW8_UNIMPLEMENTED, "%s: %lld rows exceed the kernel's grid", what, (long long)B);
  return RXW8_OK;
}

int rxw8_adjust_logits_into(rxw8_runtime *rt, rxw8_buffer *logits, const rxw8_logits_options *o, rxw8_buffer *out) {
  const char *what = "logits adjustment";
  if (!rt || !out) return fail(RXW8_INVALID_ARGUMENT, "NULL argument");
  if (int rc = check_logits(o, logits)) return rc;
  if (!is_output(out, logits)) return fail(RXW8_INVALID_ARGUMENT, "%s output: shape or dtype mismatch", what);
  // (in place: each logit is read by the thread that writes it)
  const bool in_place = out->ptr == logits->ptr && out->dtype == logits->dtype && out->rt == logits->rt;
  if (int rc = check_buffers(what, rt, {out, in_place ? nullptr : logits, o->tokens, o->offsets, o->prompts, o->repetition,
                                        o->frequency, o->presence, o->bias_words, o->bias, o->bias_offsets, o->mask, o->mask_rows}, 1))
    return rc;
  const int64_t B = logits->dims[0], V = logits->dims[1];
  if (B == 0) return RXW8_OK;
  std::lock_guard<std::recursive_mutex> g(rt->mu);
  // what a row loads of each setting that is off: a word of the runtime's own
  const void *const none = rt->f32_attn[0];
  int given = 0, bit = 0;
  auto setting = [&](const rxw8_buffer *b) {
    given |= (b != nullptr) << bit++;
    return b ? b->ptr : none;
  };
  LogitsArgs a{};
  a.logits = logits->ptr, a.out = out->ptr;
  a.offsets = (const int32_t *)setting(o->offsets), a.prompts = (const int32_t *)setting(o->prompts);
  a.repetition = (const float *)setting(o->repetition), a.frequency = (const float *)setting(o->frequency);
  a.presence = (const float *)setting(o->presence), a.bias_offsets = (const int32_t *)setting(o->bias_offsets);
  a.mask_rows = (const int32_t *)setting(o->mask_rows);
  a.T = o->tokens ? o->tokens->dims[0] : 0, a.E = o->bias ? o->bias->dims[0] : 0, a.R = o->mask ? o->mask->dims[0] : 0, a.V = V;
  if (a.T) a.tokens = (const int32_t *)o->tokens->ptr;
  if (a.E) a.bias_words = (const int32_t *)o->bias_words->ptr, a.bias = (const float *)o->bias->ptr;
  if (a.R) a.mask = (const uint32_t *)o->mask->ptr;
  a.in_f32 = logits->dtype == RXW8_F32, a.out_f32 = out->dtype == RXW8_F32, a.given = given;
  a.chunk = (int)kLogitsChunk, a.chunks = (int)((V + kLogitsChunk - 1) / kLogitsChunk);
  const bool pieces = V % 8 == 0 && !(((uintptr_t)a.logits | (uintptr_t)a.out) & 15);
  return launch(rt, pieces ? "rxw8_logits_adjust" : "rxw8_logits_any", dim3((unsigned)(B * a.chunks)), dim3(kLogitsChunk / 8), a,
                sizeof(int) * (size_t)a.chunk * ((a.tokens != nullptr) + (a.bias != nullptr)) + (a.bias ? kLogitsValues * sizeof(float) : 0));
}

int rxw8_adjust_logits(rxw8_runtime *rt, rxw8_buffer *logits, const rxw8_logits_options *o, int out_dtype,
                       rxw8_buffer **out) {
  if (!rt || !out) return fail(RXW8_INVALID_ARGUMENT, "NULL argument");
  if (int rc = check_logits(o, logits)) return rc;
  if (!is_f(out_dtype)) return fail(RXW8_INVALID_ARGUMENT, "logits adjustment: out dtype must be F32 or BF16");
  if (int rc = check_buffers("logits adjustment", rt, {logits, o->tokens, o->offsets, o->prompts, o->repetition, o->frequency, o->presence,
                                                       o->bias_words, o->bias, o->bias_offsets, o->mask, o->mask_rows}, 0))
    return rc;
  std::lock_guard<std::recursive_mutex> g(rt->mu);
  Buffer *y = nullptr;
  int rc = new_buffer(rt, out_dtype, logits->dims, 2, false, &y);
  if (rc) return rc;
  rc = rxw8_adjust_logits_into(rt, logits, o, static_cast<rxw8_buffer *>(y));
  if (rc) {
    rxw8_buffer_release(static_cast<rxw8_buffer *>(y));
    return rc;
  }
  *out = static_cast<rxw8_buffer *>(y);
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
