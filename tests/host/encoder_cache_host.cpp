// encoder_cache_host.cpp -- the encoder's kept prompts on the host: api_encoder.hip and
// api_prompts.hip as built for the library over stand-ins for the device (memory of the host's) and
// for the kernels (kv8_append notes the table and lengths it is given).  Allocations of the host's
// and strided copies fail when told to.  Loaded by test_encoder_cache_host.py.
#include "../../ex-nihilo_amd/csrc/api_host.h"
#include <cstdlib>
#include <new>

static std::string g_err;
static exn_ctx g_ctx;
static long g_fail_new = -1;    // allocations until one fails
static int g_fail_copy = -1;    // strided copies until one fails
static std::vector<int32_t> g_table, g_lens;

void* operator new(size_t n) {
  if (g_fail_new >= 0 && g_fail_new-- == 0) throw std::bad_alloc();
  void* p = malloc(n ? n : 1);
  if (!p) throw std::bad_alloc();
  return p;
}
void operator delete(void* p) noexcept { free(p); }
void operator delete(void* p, size_t) noexcept { free(p); }

namespace exn {
void set_error(const char* fmt, ...) {
  static char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof buf, fmt, ap);
  va_end(ap);
  const long f = g_fail_new;
  g_fail_new = -1;
  g_err = buf;
  g_fail_new = f;
}
hipError_t kv8_append(hipStream_t, const Kv8& c, const SeqTile*, int n, int, const uint16_t*, int64_t, const uint16_t*, int64_t) {
  const long f = g_fail_new;
  g_fail_new = -1;
  g_table.assign(c.table, c.table + (size_t)n * c.cols);
  g_lens.assign(c.lens, c.lens + n);
  g_fail_new = f;
  return hipSuccess;
}
hipError_t kv8_read(hipStream_t, const Kv8&, const SeqTile*, int, int, uint16_t*, int64_t, uint16_t*, int64_t) { return hipSuccess; }
hipError_t kv8_advance(hipStream_t, const Kv8&, const SeqTile*, int) { return hipSuccess; }
int64_t kv8_attend_part(int64_t, const int64_t*, int, int, int, int, int) { return 12; }
hipError_t kv8_attend(hipStream_t, const Kv8&, const SeqTile* const*, const int64_t*, int64_t, int, int, const uint16_t*,
                      int64_t, float, uint16_t*, int, int64_t, float*, int64_t) {
  return hipSuccess;
}
hipError_t attend_packed(hipStream_t, const SeqTile* const*, const int64_t*, int, int, int, int, const uint16_t*, int64_t,
                         const uint16_t*, int64_t, const uint16_t*, int64_t, float, uint16_t*, int, int64_t) {
  return hipSuccess;
}
hipError_t enc_qkv_rows(hipStream_t, uint16_t*, const float*, int, int64_t, const float*, const float*, const float*) { return hipSuccess; }
hipError_t enc_embed(hipStream_t, const int32_t*, int, int64_t, const int8_t*, const uint16_t*, const float*, int, float*) { return hipSuccess; }
hipError_t synth_normal(hipStream_t, uint64_t, int64_t n, float, float, int, float* out) {
  memset(out, 0, (size_t)n * 4);
  return hipSuccess;
}
hipError_t synth_q8(hipStream_t, uint64_t, int64_t, int64_t, int64_t, const int32_t*, int8_t*, uint16_t*) { return hipSuccess; }
hipError_t rms_norm(hipStream_t, int, int, float, const float*, const float*, void*, int) { return hipSuccess; }
hipError_t split_sum_rms(hipStream_t, int, int64_t, int64_t, const float*, const EpiArgs&, float, const float*, uint16_t*) { return hipSuccess; }
hipError_t gate_add(hipStream_t, int64_t, int, int, int, int, float*, const float*, const float*) { return hipSuccess; }
hipError_t qkv_prep(hipStream_t, const uint16_t*, int64_t, const float*, const float*, const float*, uint16_t*, uint16_t*,
                    uint16_t*, int64_t, int64_t, int64_t, int) {
  return hipSuccess;
}
hipError_t qkv_prep_part(hipStream_t, const float*, int, int64_t, const float*, const float*, const float*, uint16_t*,
                         uint16_t*, uint16_t*, int64_t, int64_t, int64_t, int) {
  return hipSuccess;
}
hipError_t attend(hipStream_t, const uint16_t*, const uint16_t*, const uint16_t*, void*, int, int, int, int, int64_t, int,
                  int, float, int, int64_t) {
  return hipSuccess;
}
hipError_t gemm_split_rows(hipStream_t, const uint16_t*, int64_t, const WOp&, int64_t, int64_t, int64_t, Epi, const EpiArgs&,
                           float*, int64_t, int, int* ns) {
  if (ns) *ns = 0;
  return hipSuccess;
}
}  // namespace exn

hipError_t gemm_any(hipStream_t, const exn_w*, const uint16_t*, int64_t, int64_t, Epi, const EpiArgs&) { return hipSuccess; }
int w_resident(exn_w*, bool) { return EXN_OK; }
int upload_q8_blocks(exn_ctx*, const void*, int64_t, int64_t, const int32_t*, int8_t*, uint16_t*) { return EXN_OK; }
int retile(exn_w*) { return EXN_OK; }
uint64_t gen_key(uint64_t s, uint64_t t) { return s + t; }
WOp wop_n(const exn_w*, int64_t) { return WOp{}; }
int w_new(exn_ctx* c, int, int64_t rows, int64_t cols, exn_w** out) {
  *out = new exn_w();
  (*out)->ctx = c;
  (*out)->rows = rows;
  (*out)->cols = cols;
  return EXN_OK;
}
int use(exn_ctx* c) {
  if (!c) FAIL(EXN_EINVAL, "null context");
  return EXN_OK;
}
int dev_alloc(void** p, size_t n) {
  *p = malloc(n ? n : 1);
  return *p ? EXN_OK : EXN_ENOMEM;
}
void dev_free(void* p) { free(p); }
int ctx_tmp(exn_ctx* c, size_t n, void** out) {
  if (c->tmp_bytes < n) {
    free(c->tmp);
    c->tmp = malloc(n);
    c->tmp_bytes = n;
  }
  *out = c->tmp;
  return EXN_OK;
}

extern "C" {
int exn_weight_free(exn_w* w) {
  delete w;
  return EXN_OK;
}
hipError_t hipMemcpy(void* dst, const void* src, size_t n, hipMemcpyKind) {
  memcpy(dst, src, n);
  return hipSuccess;
}
hipError_t hipMemcpyAsync(void* dst, const void* src, size_t n, hipMemcpyKind, hipStream_t) {
  memcpy(dst, src, n);
  return hipSuccess;
}
hipError_t hipMemcpy2DAsync(void* dst, size_t dp, const void* src, size_t sp, size_t w, size_t h, hipMemcpyKind, hipStream_t) {
  if (g_fail_copy >= 0 && g_fail_copy-- == 0) return hipErrorUnknown;
  for (size_t i = 0; i < h; ++i) memcpy((char*)dst + i * dp, (const char*)src + i * sp, w);
  return hipSuccess;
}
hipError_t hipMemsetAsync(void*, int, size_t, hipStream_t) { return hipSuccess; }
hipError_t hipStreamSynchronize(hipStream_t) { return hipSuccess; }
hipError_t hipSetDevice(int) { return hipSuccess; }
hipError_t hipStreamIsCapturing(hipStream_t, hipStreamCaptureStatus* s) {
  *s = hipStreamCaptureStatusNone;
  return hipSuccess;
}
const char* hipGetErrorString(hipError_t) { return "a planted failure"; }

exn_ctx* eh_ctx() { return &g_ctx; }
const char* eh_error() { return g_err.c_str(); }
// the allocation after N others fails; whether the last one planted did
void eh_fail_new(long n) { g_fail_new = n; }
int eh_failed() { return g_fail_new < 0; }
void eh_fail_copy(int n) { g_fail_copy = n; }
// what the last append was given: the table and the lengths before the step
int eh_table(int32_t* out, int cap) {
  for (size_t i = 0; i < g_table.size() && (int)i < cap; ++i) out[i] = g_table[i];
  return (int)g_table.size();
}
}
