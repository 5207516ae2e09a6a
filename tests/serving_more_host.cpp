// The host code of the operators over 8-bit pages and shared prefixes and of the logits'
// adjustments, without a GPU: a launch is noted with its arguments instead of run.
#include "../rxla_amd/csrc/serving.cpp"

#include <cstdarg>
#include <cstring>
#include <type_traits>

namespace {
struct Noted {
  char kernel[64];
  unsigned grid, threads, lds, rows;
  rxw8::SharedArgs shared;
  rxw8::PagedDecodeArgs decode;
  rxw8::LogitsArgs logits;
};
Noted noted[4096];
int count, capturing;
char message[512];
}  // namespace

namespace rxw8 {
int fail(int code, const char *fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  std::vsnprintf(message, sizeof message, fmt, ap);
  va_end(ap);
  return code;
}
int hip_fail(hipError_t, const char *) { return RXW8_INTERNAL; }
std::string dims_str(const Buffer *) { return "(dims)"; }
bool stream_capturing(const Runtime *) { return capturing; }
hipFunction_t Runtime::fn(const char *name) { return (hipFunction_t)strdup(name); }
int new_buffer(Runtime *rt, int dtype, const int64_t *dims, int rank, bool zero, Buffer **out) {
  if (zero) return fail(RXW8_INTERNAL, "a cleared buffer");  // (a memset, which no capture may record)
  auto *b = new rxw8_buffer;
  b->rt = rt, b->dtype = dtype, b->rank = rank, b->ptr = (void *)((uintptr_t)1 << 50);
  std::copy(dims, dims + rank, b->dims);
  *out = b;
  return RXW8_OK;
}
}  // namespace rxw8

extern "C" {
int rxw8_buffer_release(rxw8_buffer *b) {
  delete b;
  return RXW8_OK;
}
hipError_t hipModuleLaunchKernel(hipFunction_t f, unsigned gx, unsigned gy, unsigned, unsigned bx, unsigned, unsigned,
                                 unsigned lds, hipStream_t, void **params, void **) {
  Noted &n = noted[count++ % 4096];
  std::snprintf(n.kernel, sizeof n.kernel, "%s", (const char *)f);
  std::free((void *)f);
  n.grid = gx, n.rows = gy, n.threads = bx, n.lds = lds;
  auto take = [&](const char *prefix, auto &to) {
    if (!std::strncmp(n.kernel, prefix, std::strlen(prefix))) to = *(std::remove_reference_t<decltype(to)> *)params[0];
  };
  take("rxw8_shared_", n.shared);
  take("rxw8_q8_decode", n.decode);
  take("rxw8_logits_", n.logits);
  return hipSuccess;
}

rxw8_runtime *host_runtime(int cus, size_t lds) {
  auto *rt = new rxw8_runtime;
  rt->cus = cus, rt->lds_max = lds;
  rt->f32_attn[0] = (char *)((uintptr_t)1 << 40), rt->f32_attn[1] = (char *)((uintptr_t)2 << 40);
  return rt;
}
rxw8_buffer *host_buffer(rxw8_runtime *rt, int dtype, int rank, const int64_t *dims, uintptr_t at, int64_t bytes) {
  auto *b = new rxw8_buffer;
  b->rt = rt, b->dtype = dtype, b->rank = rank, b->ptr = (void *)at, b->bytes = (size_t)bytes;
  std::copy(dims, dims + rank, b->dims);
  return b;
}
void host_capturing(int on) { capturing = on; }
const char *host_message() { return message; }
int host_launches(int clear) {
  const int n = count;
  if (clear) count = 0, message[0] = 0;
  return n;
}
const char *host_launch(int i, unsigned *grid, unsigned *threads, unsigned *lds) {
  *grid = noted[i].grid * noted[i].rows, *threads = noted[i].threads, *lds = noted[i].lds;
  return noted[i].kernel;
}
// launch i: first sequence, sequences, units, waves, columns and keys of a prefix's block; the addresses of
// the counters, the plan, the sequences' parts, the prefixes', the records of own rows and of whole
// prefixes; those of q, out, table and lens
void host_shared(int i, int64_t *out) {
  const rxw8::SharedArgs &a = noted[i].shared;
  const int64_t x[] = {a.b0, a.d.B, a.d.units, a.d.waves, a.columns, a.keys, (int64_t)a.d.counters, (int64_t)a.plan,
                       (int64_t)a.d.part, (int64_t)a.parts, (int64_t)a.own, (int64_t)a.whole, (int64_t)a.d.q,
                       (int64_t)a.d.out, (int64_t)a.d.table, (int64_t)a.d.lens};
  std::copy(x, x + 16, out);
}
void host_decode(int i, int64_t *out) {
  const rxw8::PagedDecodeArgs &a = noted[i].decode;
  out[0] = a.units, out[1] = a.waves, out[2] = (int64_t)a.counters, out[3] = (int64_t)a.part;
}
void host_logits(int i, int64_t *out) {
  const rxw8::LogitsArgs &a = noted[i].logits;
  out[0] = a.chunk, out[1] = a.chunks;
}
}
