// encoder_fork_host.cpp -- encoder_cache_host.cpp's stand-ins with strided copies that are made when
// the host waits for the stream, as a device makes them, or then fail; and a stream that captures when
// told to.  Loaded by test_encoder_cache_fork_host.py.
#include "../../ex-nihilo_amd/csrc/api_host.h"

#define hipMemcpy2DAsync copy_2d_at_once
#define hipStreamSynchronize wait_for_nothing
#define hipStreamIsCapturing never_capturing
#include "encoder_cache_host.cpp"
#undef hipMemcpy2DAsync
#undef hipStreamSynchronize
#undef hipStreamIsCapturing

namespace {
struct Copy {
  void* dst;
  size_t dp;
  const void* src;
  size_t sp, w, h;
};
std::vector<Copy> g_queue;
int g_fail_wait = 0, g_capturing = 0;
}  // namespace

extern "C" {
hipError_t hipMemcpy2DAsync(void* dst, size_t dp, const void* src, size_t sp, size_t w, size_t h, hipMemcpyKind, hipStream_t) {
  g_queue.push_back(Copy{dst, dp, src, sp, w, h});
  return hipSuccess;
}
hipError_t hipStreamSynchronize(hipStream_t) {
  std::vector<Copy> q;
  q.swap(g_queue);
  if (g_fail_wait) return hipErrorUnknown;
  for (const Copy& c : q) copy_2d_at_once(c.dst, c.dp, c.src, c.sp, c.w, c.h, hipMemcpyDeviceToDevice, nullptr);
  return hipSuccess;
}
hipError_t hipStreamIsCapturing(hipStream_t, hipStreamCaptureStatus* s) {
  *s = g_capturing ? hipStreamCaptureStatusActive : hipStreamCaptureStatusNone;
  return hipSuccess;
}
int ef_queued() { return (int)g_queue.size(); }
void ef_fail_wait(int on) { g_fail_wait = on; }
void ef_capturing(int on) { g_capturing = on; }
}
