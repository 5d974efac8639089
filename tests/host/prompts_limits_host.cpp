// prompts_limits_host.cpp -- the prompt side's launches (packed.hip and kv8.hip as built for the library)
// asked for sizes that no grid holds: the status before anything is launched.  Without a device a launch
// that is tried returns another one.  Loaded by test_prompts_limits_host.py.
#include "../../ex-nihilo_amd/csrc/exn_common.h"
using namespace exn;

extern "C" {
// sequences of one new token, N of them: 0 where the launch is refused for its size
int pl_packed(int n, int heads, int kv_heads, int head_dim) {
  const SeqTile* tiles[SEQ_TTS] = {};
  const int64_t ntiles[SEQ_TTS] = {n, n, n, n, n};
  const int64_t w = (int64_t)heads * head_dim;
  return attend_packed(nullptr, tiles, ntiles, 0, heads, kv_heads, head_dim, nullptr, w, nullptr, w, nullptr, w, 1.f, nullptr, 0,
                       w) != hipErrorInvalidConfiguration;
}
static Kv8 cache(int kv_heads, int cols) {
  Kv8 c{};
  c.kv_heads = kv_heads;
  c.head_dim = 64;
  c.cols = cols;
  c.pages = 1;
  return c;
}
int pl_append(int n, int kv_heads) {
  return kv8_append(nullptr, cache(kv_heads, 1), nullptr, n, 1, nullptr, 64 * kv_heads, nullptr, 64 * kv_heads) !=
         hipErrorInvalidConfiguration;
}
int pl_read(int n, int kv_heads) {
  return kv8_read(nullptr, cache(kv_heads, 1), nullptr, n, 1, nullptr, 64 * kv_heads, nullptr, 64 * kv_heads) !=
         hipErrorInvalidConfiguration;
}
int pl_attend(int n, int longest, int heads, int kv_heads, int cols) {
  const SeqTile* tiles[SEQ_TTS] = {};
  int64_t ntiles[SEQ_TTS];
  for (int z = 0; z < SEQ_TTS; ++z) ntiles[z] = (int64_t)n * ((longest + (SEQ_TT0 << z) - 1) / (SEQ_TT0 << z));
  return kv8_attend(nullptr, cache(kv_heads, cols), tiles, ntiles, (int64_t)n * longest, longest, heads, nullptr, heads * 64, 1.f,
                    nullptr, 0, heads * 64, nullptr, 0) != hipErrorInvalidConfiguration;
}
}
