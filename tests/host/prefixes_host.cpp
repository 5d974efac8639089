// prefixes_host.cpp -- plans of prefixes and rotaries on the host: api_prefixes.hip and api_rope.hip (with
// api_prompts.hip's plans) as built for the library over stand-ins for the device: memory of the host's,
// kernels that note their call and keep what they were given.  Loaded by test_prefixes_host.py.
#include "../../ex-nihilo_amd/csrc/api_host.h"
#include <cstdlib>

static std::string g_err, g_log;
static exn_ctx g_ctx;
static int g_capturing = 0, g_no_memory = 0;
static Kv8Shared g_shared;
static RopeArgs g_rope;

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
hipError_t attend_packed(hipStream_t, const SeqTile* const*, const int64_t*, int, int, int, int, const uint16_t*, int64_t,
                         const uint16_t*, int64_t, const uint16_t*, int64_t, float, uint16_t*, int, int64_t) {
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
int64_t kv8_shared_part(int64_t, int, const Kv8Shared&, int, int, int, int, const int64_t*) { return 34; }
hipError_t kv8_attend_shared(hipStream_t, const Kv8&, const SeqTile* const*, const int64_t*, int64_t, int,
                             const Kv8Shared& sh, int, const uint16_t*, int64_t, float, uint16_t*, int, int64_t, float*,
                             int64_t) {
  g_shared = sh;
  return note("shared");
}
hipError_t rope_rows(hipStream_t, const RopeArgs& a, int, int, int, int64_t, int) {
  g_rope = a;
  return note("rope");
}
}  // namespace exn

int use(exn_ctx* c) {
  if (!c) FAIL(EXN_EINVAL, "null context");
  return EXN_OK;
}
int dev_alloc(void** p, size_t n) {
  *p = g_no_memory ? nullptr : malloc(n ? n : 1);
  if (!*p) FAIL(EXN_ENOMEM, "no memory");
  return EXN_OK;
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
void ph_no_memory(int on) { g_no_memory = on; }
const char* ph_error() { return g_err.c_str(); }
const char* ph_log() {
  static std::string l;
  l.swap(g_log);
  g_log.clear();
  return l.c_str();
}
// what the last attend_shared got: {rows, most, blocks}; the SEQS sequences' {first, blocks, row, 0}; the rows' {row,
// sequence}; then each list's tiles with their blocks after (-1, tokens a tile, 0, 0, 0)
int ph_shared(int32_t* out, int seqs) {
  int32_t* o = out;
  for (int64_t v : {g_shared.rows, (int64_t)g_shared.most, (int64_t)g_shared.blocks}) *o++ = (int32_t)v;
  memcpy(o, g_shared.of, 16 * (size_t)seqs);
  o += 4 * seqs;
  memcpy(o, g_shared.entry, 8 * (size_t)g_shared.rows);
  o += 2 * g_shared.rows;
  for (int z = 0; z < SEQ_TTS; ++z)
    for (int64_t i = -1; i < g_shared.ntiles[z]; ++i, o += 5) {
      const SeqTile t = i < 0 ? SeqTile{-1, SEQ_TT0 << z, 0, 0} : g_shared.tiles[z][i];
      memcpy(o, &t, sizeof t);
      o[4] = i < 0 ? 0 : g_shared.tile_blocks[z][i];
    }
  return (int)(o - out);
}
// the turns and axes of the last rope_rows
int ph_rope(uint64_t* turns, int32_t* axis) {
  memcpy(turns, g_rope.turns, 8 * (size_t)g_rope.pairs);
  memcpy(axis, g_rope.axis, 4 * (size_t)g_rope.pairs);
  return g_rope.pairs;
}
}
