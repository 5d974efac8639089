// api_prompts.hip -- the C ABI of the prompt side's attention: plans of packed sequences, causal
// attention over them, and the cache held in 8 bits.
#include "api_host.h"

#include <new>
#include <numeric>

constexpr int kSeqsMax = 1 << 16;
constexpr int64_t kSeqRowsMax = 1 << 22;
constexpr int kNewMax = 1 << 21;   // new tokens of a sequence: its blocks are a grid's second axis

int exn_seqs_create(exn_ctx* ctx, const int32_t* lens, int seqs, exn_seqs** out) {
  if (!out) FAIL(EXN_EINVAL, "null output");
  *out = nullptr;
  TRY(use(ctx));
  if (seqs < 1 || seqs > kSeqsMax || !lens) FAIL(EXN_EINVAL, "sequences: %d of them (1 to %d)", seqs, kSeqsMax);
  int64_t rows = 0;
  for (int i = 0; i < seqs; ++i) {
    if (lens[i] < 0) FAIL(EXN_EINVAL, "sequences: length %d is %d", i, lens[i]);
    rows += lens[i];
    if (rows > kSeqRowsMax) FAIL(EXN_EINVAL, "sequences: more than %lld rows", (long long)kSeqRowsMax);
  }
  hipStreamCaptureStatus cap = hipStreamCaptureStatusNone;
  HIPCHK(hipStreamIsCapturing(ctx->stream, &cap));
  if (cap != hipStreamCaptureStatusNone) FAIL(EXN_ESTATE, "sequences: a plan is made before a capture, not in it");
  exn_seqs* s = nullptr;
  try {
    s = new exn_seqs();
    s->device = ctx->device;
    s->seqs = seqs;
    s->rows = rows;
    s->lens.assign(lens, lens + seqs);
    std::vector<int32_t> row0((size_t)seqs), order((size_t)seqs);
    for (int i = 0, r = 0; i < seqs; r += lens[i++]) row0[(size_t)i] = r;
    std::iota(order.begin(), order.end(), 0);
    std::stable_sort(order.begin(), order.end(), [&](int a, int b) { return lens[a] > lens[b]; });
    s->longest = lens[order[0]];
    std::vector<SeqTile> all;
    size_t at[SEQ_TTS];
    for (int z = 0; z < SEQ_TTS; ++z) {
      const int tt = SEQ_TT0 << z;
      at[z] = all.size();
      for (int t0 = (s->longest - 1) / tt * tt; t0 >= 0 && s->longest > 0; t0 -= tt)
        for (int i : order) {
          if (lens[i] <= t0) break;
          all.push_back(SeqTile{row0[(size_t)i], lens[i], t0, i});
        }
      s->ntiles[z] = (int64_t)(all.size() - at[z]);
    }
    const size_t whole = all.size();
    for (int i = 0; i < seqs; ++i) all.push_back(SeqTile{row0[(size_t)i], lens[i], 0, i});
    const size_t bytes = all.size() * sizeof(SeqTile);
    int r = dev_alloc(&s->mem, bytes);
    if (r == EXN_OK) {
      // on the context's stream, whose work reads it (the null stream would not be ordered with it)
      hipError_t e = hipMemcpyAsync(s->mem, all.data(), bytes, hipMemcpyHostToDevice, ctx->stream);
      if (e == hipSuccess) e = hipStreamSynchronize(ctx->stream);
      if (e != hipSuccess) {
        exn::set_error("sequences: upload: %s", hipGetErrorString(e));
        r = EXN_EHIP;
      }
    }
    if (r != EXN_OK) {
      dev_free(s->mem);
      delete s;
      return r;
    }
    for (int z = 0; z < SEQ_TTS; ++z) s->tiles[z] = (const SeqTile*)s->mem + at[z];
    s->whole = (const SeqTile*)s->mem + whole;
  } catch (const std::bad_alloc&) {
    delete s;
    FAIL(EXN_ENOMEM, "sequences: host memory");
  }
  *out = s;
  return EXN_OK;
}

int exn_seqs_info(const exn_seqs* s, int* seqs, int64_t* rows, int* longest) {
  if (!s) FAIL(EXN_EINVAL, "null sequences");
  if (seqs) *seqs = s->seqs;
  if (rows) *rows = s->rows;
  if (longest) *longest = s->longest;
  return EXN_OK;
}

int exn_seqs_free(exn_seqs* s) {
  if (!s) return EXN_OK;
  HIPCHK(hipSetDevice(s->device));
  dev_free(s->mem);   // waits for the device
  delete s;
  return EXN_OK;
}

namespace {

bool half_type(int dt) { return dt == EXN_DT_F16 || dt == EXN_DT_BF16; }

// heads and types that the attention kernels take
int check_heads(int dt, int odt, int heads, int kv_heads, int head_dim) {
  if (!half_type(dt) || !half_type(odt)) FAIL(EXN_EINVAL, "attention dtypes %d, %d (EXN_DT_F16 or EXN_DT_BF16)", dt, odt);
  if (kv_heads < 1 || kv_heads > 1024 || heads < kv_heads || heads > 1024 || heads % kv_heads)
    FAIL(EXN_EINVAL, "attention: %d heads over %d key/value heads (a multiple, at most 1024)", heads, kv_heads);
  if (head_dim != 64 && head_dim != 128) FAIL(EXN_EINVAL, "attention: heads of %d (64 or 128)", head_dim);
  return EXN_OK;
}

// rows of WIDTH 16-bit values LD apart: 16-byte loads
int check_rows(const char* what, const void* p, int64_t ld, int64_t width) {
  if (!p) FAIL(EXN_EINVAL, "%s: null pointer", what);
  if (ld < width || ld % 8 || ld > (1 << 24) || (uintptr_t)p % 16)
    FAIL(EXN_EINVAL, "%s: rows of %lld, %lld apart, at %p (a stride of 8 values' multiples, 16-byte aligned)", what,
         (long long)width, (long long)ld, p);
  return EXN_OK;
}

int check_seqs(const exn_ctx* ctx, const exn_seqs* s) {
  if (!ctx) FAIL(EXN_EINVAL, "null context");
  if (!s) FAIL(EXN_EINVAL, "null sequences");
  if (s->device != ctx->device) FAIL(EXN_EINVAL, "sequences planned on device %d, the context's is %d", s->device, ctx->device);
  return EXN_OK;
}

int check_kv8(const exn_kv8* c, const exn_seqs* s) {
  if (!c) FAIL(EXN_EINVAL, "null cache");
  TRY(check_heads(c->dt, c->dt, c->kv_heads, c->kv_heads, c->head_dim));
  if (c->pages < 1 || c->pages > INT32_MAX || c->cols < 1 || c->cols > (1 << 20))
    FAIL(EXN_EINVAL, "cache: %lld pages, %d columns", (long long)c->pages, c->cols);
  if (!s) FAIL(EXN_EINVAL, "null sequences");
  if (c->seqs != s->seqs) FAIL(EXN_EINVAL, "cache of %d sequences, a plan of %d", c->seqs, s->seqs);
  if (!c->k || !c->v || !c->scales || !c->tk || !c->tv || !c->table || !c->lens) FAIL(EXN_EINVAL, "cache: null pointer");
  for (const void* p : {(const void*)c->k, (const void*)c->v, (const void*)c->tk, (const void*)c->tv})
    if ((uintptr_t)p % 16) FAIL(EXN_EINVAL, "cache: codes and tails are 16-byte aligned");
  if ((uintptr_t)c->scales % 8 || (uintptr_t)c->table % 4 || (uintptr_t)c->lens % 4)
    FAIL(EXN_EINVAL, "cache: scales are 8-byte, table and lens 4-byte aligned");
  return EXN_OK;
}

// what a launch returned: the sizes it has no grid for are the caller's
int launched(const char* what, hipError_t e) {
  if (e == hipErrorInvalidConfiguration)
    FAIL(EXN_EINVAL, "%s: more than 2^24 - 1 workgroups (fewer sequences or key/value heads)", what);
  if (e != hipSuccess) FAIL(e == hipErrorOutOfMemory ? EXN_ENOMEM : EXN_EHIP, "%s: %s", what, hipGetErrorString(e));
  return EXN_OK;
}

Kv8 kv8_of(const exn_kv8* c) {
  Kv8 k;
  k.bf16 = c->dt == EXN_DT_BF16;
  k.kv_heads = c->kv_heads;
  k.head_dim = c->head_dim;
  k.cols = c->cols;
  k.pages = c->pages;
  k.k = c->k;
  k.v = c->v;
  k.scales = c->scales;
  k.tk = (uint16_t*)c->tk;
  k.tv = (uint16_t*)c->tv;
  k.table = c->table;
  k.lens = c->lens;
  return k;
}

}  // namespace

int exn_attend_packed(exn_ctx* ctx, const exn_seqs* s, int dt, int heads, int kv_heads, int head_dim, const void* q,
                      int64_t ldq, const void* k, int64_t ldk, const void* v, int64_t ldv, float scale, void* out,
                      int odt, int64_t ldo) {
  TRY(check_heads(dt, odt, heads, kv_heads, head_dim));
  TRY(check_rows("attend_packed q", q, ldq, (int64_t)heads * head_dim));
  TRY(check_rows("attend_packed k", k, ldk, (int64_t)kv_heads * head_dim));
  TRY(check_rows("attend_packed v", v, ldv, (int64_t)kv_heads * head_dim));
  TRY(check_rows("attend_packed out", out, ldo, (int64_t)heads * head_dim));
  TRY(check_seqs(ctx, s));
  TRY(use(ctx));
  return launched("attend_packed",
                  attend_packed(ctx->stream, s->tiles, s->ntiles, dt == EXN_DT_BF16, heads, kv_heads, head_dim,
                                (const uint16_t*)q, ldq, (const uint16_t*)k, ldk, (const uint16_t*)v, ldv, scale,
                                (uint16_t*)out, odt == EXN_DT_BF16, ldo));
}

int exn_kv8_append(exn_ctx* ctx, const exn_kv8* c, const exn_seqs* s, const void* k, int64_t ldk, const void* v,
                   int64_t ldv) {
  TRY(check_kv8(c, s));
  TRY(check_rows("kv8_append k", k, ldk, (int64_t)c->kv_heads * c->head_dim));
  TRY(check_rows("kv8_append v", v, ldv, (int64_t)c->kv_heads * c->head_dim));
  if (s->longest > kNewMax) FAIL(EXN_EINVAL, "kv8_append: %d new tokens of a sequence (at most %d)", s->longest, kNewMax);
  TRY(check_seqs(ctx, s));
  TRY(use(ctx));
  return launched("kv8_append", kv8_append(ctx->stream, kv8_of(c), s->whole, s->seqs, s->longest, (const uint16_t*)k,
                                           ldk, (const uint16_t*)v, ldv));
}

int exn_kv8_read(exn_ctx* ctx, const exn_kv8* c, const exn_seqs* s, void* k, int64_t ldk, void* v, int64_t ldv) {
  TRY(check_kv8(c, s));
  TRY(check_rows("kv8_read k", k, ldk, (int64_t)c->kv_heads * c->head_dim));
  TRY(check_rows("kv8_read v", v, ldv, (int64_t)c->kv_heads * c->head_dim));
  if (s->longest > kNewMax) FAIL(EXN_EINVAL, "kv8_read: %d new tokens of a sequence (at most %d)", s->longest, kNewMax);
  TRY(check_seqs(ctx, s));
  TRY(use(ctx));
  return launched("kv8_read", kv8_read(ctx->stream, kv8_of(c), s->whole, s->seqs, s->longest, (uint16_t*)k, ldk,
                                       (uint16_t*)v, ldv));
}

int exn_kv8_advance(exn_ctx* ctx, const exn_kv8* c, const exn_seqs* s) {
  TRY(check_kv8(c, s));
  TRY(check_seqs(ctx, s));
  TRY(use(ctx));
  HIPCHK(kv8_advance(ctx->stream, kv8_of(c), s->whole, s->seqs));
  return EXN_OK;
}

int exn_kv8_attend_part(const exn_seqs* s, int heads, int kv_heads, int head_dim, int cols, int64_t* floats) {
  if (!s || !floats) FAIL(EXN_EINVAL, "kv8_attend_part: null pointer");
  TRY(check_heads(EXN_DT_F16, EXN_DT_F16, heads, kv_heads, head_dim));
  if (cols < 1 || cols > (1 << 20)) FAIL(EXN_EINVAL, "kv8_attend_part: %d columns", cols);
  *floats = kv8_attend_part(s->rows, s->ntiles, s->longest, heads, kv_heads, head_dim, cols);
  return EXN_OK;
}

int exn_kv8_attend(exn_ctx* ctx, const exn_kv8* c, const exn_seqs* s, int heads, const void* q, int64_t ldq,
                   float scale, void* out, int odt, int64_t ldo, float* part, int64_t part_cap) {
  TRY(check_kv8(c, s));
  TRY(check_heads(c->dt, odt, heads, c->kv_heads, c->head_dim));
  TRY(check_rows("kv8_attend q", q, ldq, (int64_t)heads * c->head_dim));
  TRY(check_rows("kv8_attend out", out, ldo, (int64_t)heads * c->head_dim));
  if (part_cap < 0 || (part_cap > 0 && (!part || (uintptr_t)part % 16)))
    FAIL(EXN_EINVAL, "kv8_attend: %lld floats of scratch at %p", (long long)part_cap, (const void*)part);
  TRY(check_seqs(ctx, s));
  TRY(use(ctx));
  return launched("kv8_attend",
                  kv8_attend(ctx->stream, kv8_of(c), s->tiles, s->ntiles, s->rows, s->longest, heads, (const uint16_t*)q,
                             ldq, scale, (uint16_t*)out, odt == EXN_DT_BF16, ldo, part, part_cap));
}
