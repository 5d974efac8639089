// api_prefixes.hip -- the C ABI of attention over the 8-bit cache for sequences that begin alike: the
// plan of their prefixes, and the call.
#include "api_prompts.h"

#include <new>

int exn_prefixes_create(exn_ctx* ctx, const exn_seqs* s, const int32_t* of, const int32_t* blocks, int prefixes,
                        exn_prefixes** out) {
  if (!out) FAIL(EXN_EINVAL, "null output");
  *out = nullptr;
  TRY(check_seqs(ctx, s));
  TRY(use(ctx));
  if (!of || prefixes < 0 || prefixes > s->seqs || (prefixes > 0 && !blocks))
    FAIL(EXN_EINVAL, "prefixes: %d of them for %d sequences", prefixes, s->seqs);
  for (int i = 0; i < s->seqs; ++i)
    if (of[i] < -1 || of[i] >= prefixes) FAIL(EXN_EINVAL, "prefixes: sequence %d has prefix %d of %d", i, of[i], prefixes);
  for (int i = 0; i < prefixes; ++i)
    if (blocks[i] < 0 || blocks[i] > (1 << 20)) FAIL(EXN_EINVAL, "prefixes: prefix %d of %d blocks", i, blocks[i]);
  hipStreamCaptureStatus cap = hipStreamCaptureStatusNone;
  HIPCHK(hipStreamIsCapturing(ctx->stream, &cap));
  if (cap != hipStreamCaptureStatusNone) FAIL(EXN_ESTATE, "prefixes: a plan is made before a capture, not in it");
  exn_prefixes* p = nullptr;
  try {
    p = new exn_prefixes();
    p->device = ctx->device;
    p->plan = s->id;
    // a prefix is shared where two sequences of it have rows
    std::vector<int64_t> rows((size_t)prefixes, 0);
    std::vector<int> seqs((size_t)prefixes, 0), first((size_t)prefixes, -1);
    for (int i = 0; i < s->seqs; ++i)
      if (of[i] >= 0 && s->lens[(size_t)i] > 0) {
        const size_t g = (size_t)of[i];
        rows[g] += s->lens[(size_t)i];
        if (seqs[g]++ == 0) first[g] = i;
      }
    auto shared = [&](int g) { return g >= 0 && seqs[(size_t)g] > 1 && blocks[g] > 0; };
    Kv8Shared& sh = p->sh;
    std::vector<int32_t> at((size_t)prefixes, 0), words;
    for (int g = 0; g < prefixes; ++g)
      if (shared(g)) {
        at[(size_t)g] = (int32_t)sh.rows;
        sh.rows += rows[(size_t)g];
        sh.most = std::max(sh.most, (int)rows[(size_t)g]);
        sh.seqs = std::max(sh.seqs, seqs[(size_t)g]);
        sh.blocks = std::max(sh.blocks, blocks[g]);
        sh.saved += (int64_t)(seqs[(size_t)g] - 1) * blocks[g];
      }
    sh.fewest = sh.blocks;
    for (int i = 0; i < s->seqs; ++i)
      if (s->lens[(size_t)i] > 0) sh.fewest = std::min(sh.fewest, shared(of[i]) ? blocks[of[i]] : 0);
    // each list's tiles; then their blocks; of each sequence; the rows
    std::vector<SeqTile> tiles;
    size_t lists[SEQ_TTS];
    for (int z = 0; z < SEQ_TTS; ++z) {
      lists[z] = tiles.size();
      const int tt = SEQ_TT0 << z;
      for (int g = 0; g < prefixes; ++g)
        for (int64_t t0 = 0; shared(g) && t0 < rows[(size_t)g]; t0 += tt) {
          tiles.push_back(SeqTile{at[(size_t)g], (int32_t)rows[(size_t)g], (int32_t)t0, first[(size_t)g]});
          words.push_back(blocks[g]);
        }
      sh.ntiles[z] = (int64_t)(tiles.size() - lists[z]);
    }
    words.resize((words.size() + 3) / 4 * 4);   // of each sequence: 16 bytes
    const size_t of0 = words.size(), entry0 = of0 + 4 * (size_t)s->seqs;
    words.resize(entry0 + 2 * (size_t)sh.rows);
    for (int i = 0, r = 0; i < s->seqs; r += s->lens[(size_t)i++]) {
      int32_t* mine = &words[of0 + 4 * (size_t)i];
      mine[0] = -1;
      if (!shared(of[i])) continue;
      int32_t& e = at[(size_t)of[i]];
      mine[0] = first[(size_t)of[i]];
      mine[1] = blocks[of[i]];
      mine[2] = e;
      for (int k = 0; k < s->lens[(size_t)i]; ++k, ++e) {
        words[entry0 + 2 * (size_t)e] = r + k;
        words[entry0 + 2 * (size_t)e + 1] = i;
      }
    }
    const size_t tb = tiles.size() * sizeof(SeqTile), wb = words.size() * sizeof(int32_t);
    int r = dev_alloc(&p->mem, tb + wb);
    if (r == EXN_OK) {
      hipError_t e = hipSuccess;
      if (tb) e = hipMemcpyAsync(p->mem, tiles.data(), tb, hipMemcpyHostToDevice, ctx->stream);
      if (e == hipSuccess) e = hipMemcpyAsync((char*)p->mem + tb, words.data(), wb, hipMemcpyHostToDevice, ctx->stream);
      if (e == hipSuccess) e = hipStreamSynchronize(ctx->stream);
      if (e != hipSuccess) {
        exn::set_error("prefixes: upload: %s", hipGetErrorString(e));
        r = EXN_EHIP;
      }
    }
    if (r != EXN_OK) {
      dev_free(p->mem);
      delete p;
      return r;
    }
    const int32_t* w = (const int32_t*)((const char*)p->mem + tb);
    for (int z = 0; z < SEQ_TTS; ++z) {
      sh.tiles[z] = (const SeqTile*)p->mem + lists[z];
      sh.tile_blocks[z] = w + lists[z];
    }
    sh.of = w + of0;
    sh.entry = w + entry0;
  } catch (const std::bad_alloc&) {
    delete p;
    FAIL(EXN_ENOMEM, "prefixes: host memory");
  }
  *out = p;
  return EXN_OK;
}

int exn_prefixes_free(exn_prefixes* p) {
  if (!p) return EXN_OK;
  HIPCHK(hipSetDevice(p->device));
  dev_free(p->mem);   // waits for the device
  delete p;
  return EXN_OK;
}

namespace {

int check_prefixes(const exn_seqs* s, const exn_prefixes* p) {
  if (!s) FAIL(EXN_EINVAL, "null sequences");
  if (!p) FAIL(EXN_EINVAL, "null prefixes");
  if (p->plan != s->id) FAIL(EXN_EINVAL, "prefixes of another plan of sequences");
  return EXN_OK;
}

}  // namespace

int exn_attend_shared_part(const exn_seqs* s, const exn_prefixes* p, int heads, int kv_heads, int head_dim, int cols,
                           int64_t* floats) {
  if (!floats) FAIL(EXN_EINVAL, "attend_shared_part: null pointer");
  TRY(check_prefixes(s, p));
  TRY(check_heads(EXN_DT_F16, EXN_DT_F16, heads, kv_heads, head_dim));
  if (cols < 1 || cols > (1 << 20)) FAIL(EXN_EINVAL, "attend_shared_part: %d columns", cols);
  *floats = s->rows == 0 ? 0 : kv8_shared_part(s->rows, s->longest, p->sh, heads, kv_heads, head_dim, cols, s->ntiles);
  return EXN_OK;
}

int exn_attend_shared(exn_ctx* ctx, const exn_kv8* c, const exn_seqs* s, const exn_prefixes* p, int heads, const void* q,
                      int64_t ldq, float scale, void* out, int odt, int64_t ldo, float* part, int64_t part_cap) {
  TRY(check_kv8(c, s));
  TRY(check_prefixes(s, p));
  TRY(check_heads(c->dt, odt, heads, c->kv_heads, c->head_dim));
  TRY(check_rows("attend_shared q", q, ldq, (int64_t)heads * c->head_dim));
  TRY(check_rows("attend_shared out", out, ldo, (int64_t)heads * c->head_dim));
  if (part_cap < 0 || (part_cap > 0 && (!part || (uintptr_t)part % 16)))
    FAIL(EXN_EINVAL, "attend_shared: %lld floats of scratch at %p", (long long)part_cap, (const void*)part);
  TRY(check_seqs(ctx, s));
  TRY(use(ctx));
  return launched("attend_shared",
                  kv8_attend_shared(ctx->stream, kv8_of(c), s->tiles, s->ntiles, s->rows, s->longest, p->sh,
                                    heads, (const uint16_t*)q, ldq, scale, (uint16_t*)out, odt == EXN_DT_BF16, ldo, part,
                                    part_cap));
}
