// prompts_host.cpp -- the prompt side's attention on the host: api_prompts.hip as built for the
// library over stand-ins for the device (memory of the host's, kernels that note their call), and
// the cache's rules (places, pages, scales, codes) that the kernels share with the host.  Loaded by
// test_prompts_host.py.
#include "../../ex-nihilo_amd/csrc/api_host.h"
#include <cstdlib>

static std::string g_err, g_log;
static exn_ctx g_ctx;
static int g_capturing = 0;
static std::vector<SeqTile> g_tiles;

namespace exn {
void set_error(const char* fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof buf, fmt, ap);
  va_end(ap);
  g_err = buf;
}
static hipError_t note(const char* what) {
  g_log += what;
  g_log += ' ';
  return hipSuccess;
}
hipError_t attend_packed(hipStream_t, const SeqTile* const* tiles, const int64_t* n, int, int, int, int, const uint16_t*,
                         int64_t, const uint16_t*, int64_t, const uint16_t*, int64_t, float, uint16_t*, int, int64_t) {
  g_tiles.clear();
  for (int z = 0; z < SEQ_TTS; ++z) {
    g_tiles.push_back(SeqTile{-1, SEQ_TT0 << z, 0, 0});
    g_tiles.insert(g_tiles.end(), tiles[z], tiles[z] + n[z]);
  }
  return note("packed");
}
hipError_t kv8_append(hipStream_t, const Kv8&, const SeqTile*, int, int, const uint16_t*, int64_t, const uint16_t*, int64_t) {
  return note("append");
}
hipError_t kv8_read(hipStream_t, const Kv8&, const SeqTile*, int, int, uint16_t*, int64_t, uint16_t*, int64_t) {
  return note("read");
}
hipError_t kv8_advance(hipStream_t, const Kv8&, const SeqTile*, int) { return note("advance"); }
int64_t kv8_attend_part(int64_t, const int64_t*, int, int, int, int, int) { return 12; }
hipError_t kv8_attend(hipStream_t, const Kv8&, const SeqTile* const*, const int64_t*, int64_t, int, int,
                      const uint16_t*, int64_t, float, uint16_t*, int, int64_t, float*, int64_t) {
  return note("attend");
}
}  // namespace exn

int use(exn_ctx* c) {
  if (!c) FAIL(EXN_EINVAL, "null context");
  return EXN_OK;
}
int dev_alloc(void** p, size_t n) {
  *p = malloc(n ? n : 1);
  return *p ? EXN_OK : EXN_ENOMEM;
}
void dev_free(void* p) { free(p); }

extern "C" {
hipError_t hipMemcpyAsync(void* dst, const void* src, size_t n, hipMemcpyKind, hipStream_t) {
  memcpy(dst, src, n);
  return hipSuccess;
}
hipError_t hipStreamSynchronize(hipStream_t) { return hipSuccess; }
hipError_t hipSetDevice(int) { return hipSuccess; }
hipError_t hipStreamIsCapturing(hipStream_t, hipStreamCaptureStatus* s) {
  *s = g_capturing ? hipStreamCaptureStatusActive : hipStreamCaptureStatusNone;
  return hipSuccess;
}
const char* hipGetErrorString(hipError_t) { return "an error"; }

exn_ctx* ph_ctx() { return &g_ctx; }
void ph_device(int d) { g_ctx.device = d; }
void ph_capturing(int on) { g_capturing = on; }
const char* ph_error() { return g_err.c_str(); }
// the kernels called since the last time
const char* ph_log() {
  static std::string l;
  l.swap(g_log);
  g_log.clear();
  return l.c_str();
}
// the plan that the last attend_packed got: (row0, len, t0, seq) each, a list begun by (-1, tokens a tile, 0, 0)
int ph_tiles(int32_t* out, int cap) {
  const int n = (int)g_tiles.size();
  memcpy(out, g_tiles.data(), sizeof(SeqTile) * (size_t)(n < cap ? n : cap));
  return n;
}

// a sequence's place and page by the kernels' rules
void ph_place(const int32_t* table, int32_t* lens, int cols, int64_t pages, int seq, int n, int block, int* base, int* total,
              int64_t* page) {
  Kv8 c{};
  c.table = table;
  c.lens = lens;
  c.cols = cols;
  c.pages = pages;
  *base = kv8_base(c, seq);
  *total = kv8_total(c, *base, n);
  *page = kv8_page(c, seq, block);
}
// a block's scale and codes by the kernels' rules
float ph_block(const float* x, int n, int8_t* codes) {
  uint32_t top = 0;
  for (int i = 0; i < n; ++i) {
    uint32_t u;
    memcpy(&u, x + i, 4);
    u &= 0x7FFFFFFFu;
    if (u > top) top = u;
  }
  const float d = kv8_scale(top);
  for (int i = 0; i < n; ++i) codes[i] = kv8_code(x[i], d);
  return d;
}
}
