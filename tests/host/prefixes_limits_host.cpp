// prefixes_limits_host.cpp -- attend_shared's launches (kv8.hip as built for the library) asked for sizes that no
// grid holds: the status before anything is launched.  Without a device a launch that is tried returns another one.
// Loaded by test_prefixes_limits_host.py.
#include "../../ex-nihilo_amd/csrc/exn_common.h"
using namespace exn;

static Kv8Shared shared(int n, int blocks) {
  Kv8Shared sh{};
  for (int z = 0; z < SEQ_TTS; ++z) sh.ntiles[z] = (n + (SEQ_TT0 << z) - 1) / (SEQ_TT0 << z);
  sh.rows = sh.most = sh.seqs = n;
  sh.blocks = sh.fewest = blocks;
  sh.saved = (int64_t)(n - 1) * blocks;
  return sh;
}

extern "C" {
// N sequences of one new token after BLOCKS blocks: 0 where the launch is refused for its size
int ps_shared(int n, int heads, int kv_heads, int blocks) {
  const SeqTile* tiles[SEQ_TTS] = {};
  const int64_t ntiles[SEQ_TTS] = {n, n, n, n, n};
  Kv8 c{};
  c.kv_heads = kv_heads;
  c.head_dim = 64;
  c.cols = blocks + 2;
  c.pages = 1;
  return kv8_attend_shared(nullptr, c, tiles, ntiles, n, 1, shared(n, blocks), heads, nullptr, heads * 64, 1.f, nullptr, 0,
                           heads * 64, nullptr, INT64_MAX) != hipErrorInvalidConfiguration;
}
// the floats of scratch that such a call has a use for, and kv8_attend's
int64_t ps_part(int n, int longest, int heads, int kv_heads, int hd, int blocks, int cols, int64_t* alone) {
  int64_t ntiles[SEQ_TTS];
  for (int z = 0; z < SEQ_TTS; ++z) ntiles[z] = (int64_t)n * ((longest + (SEQ_TT0 << z) - 1) / (SEQ_TT0 << z));
  Kv8Shared sh = shared(n, blocks);
  sh.rows = sh.most = n * longest;
  for (int z = 0; z < SEQ_TTS; ++z) sh.ntiles[z] = (sh.rows + (SEQ_TT0 << z) - 1) / (SEQ_TT0 << z);
  *alone = kv8_attend_part((int64_t)n * longest, ntiles, longest, heads, kv_heads, hd, cols);
  return kv8_shared_part((int64_t)n * longest, longest, sh, heads, kv_heads, hd, cols, ntiles);
}
}
