// The serving operators' host code (argument checks and launch plans) without a GPU: a launch
// is noted instead of run.
#include "../rxla_amd/csrc/serving.cpp"

#include <cstdarg>
#include <cstring>

namespace {
struct Noted {
  char kernel[64];
  unsigned grid, threads, lds;
};
Noted noted[8];
int count, capturing;
char message[512];
rxw8::PagedDecodeArgs decode_args;
rxw8::SampleArgs sample_args;
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
hipError_t hipModuleLaunchKernel(hipFunction_t f, unsigned gx, unsigned, unsigned, unsigned bx, unsigned, unsigned,
                                 unsigned lds, hipStream_t, void **params, void **) {
  Noted &n = noted[count++ % 8];
  std::snprintf(n.kernel, sizeof n.kernel, "%s", (const char *)f);
  std::free((void *)f);
  n.grid = gx, n.threads = bx, n.lds = lds;
  if (!std::strncmp(n.kernel, "rxw8_paged_decode", 17)) decode_args = *(rxw8::PagedDecodeArgs *)params[0];
  if (!std::strncmp(n.kernel, "rxw8_sample", 11)) sample_args = *(rxw8::SampleArgs *)params[0];
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
  *grid = noted[i].grid, *threads = noted[i].threads, *lds = noted[i].lds;
  return noted[i].kernel;
}
// units, waves, address of the counters, of the partials
void host_decode(int64_t *out) {
  out[0] = decode_args.units, out[1] = decode_args.waves;
  out[2] = (int64_t)decode_args.counters, out[3] = (int64_t)decode_args.part;
}
// S, chunk, shift, and the addresses of extremes, arrivals, listed and bins
void host_sample(int64_t *out) {
  out[0] = sample_args.S, out[1] = sample_args.chunk, out[2] = sample_args.shift;
  out[3] = (int64_t)sample_args.extremes, out[4] = (int64_t)sample_args.arrivals;
  out[5] = (int64_t)sample_args.listed, out[6] = (int64_t)sample_args.bins;
}
}
