// api_rope.hip -- the C ABI of rotary positions: frequencies, rotaries, and rows normed and turned by them.
#include "api_prompts.h"

#include <new>

constexpr double kPi = 3.14159265358979323846;

int exn_rope_freqs(int dims, double base, int scaling, double factor, double kept, double low, double high, double* freq) {
  if (!freq) FAIL(EXN_EINVAL, "rope_freqs: null pointer");
  if (dims < 2 || dims % 2 || dims > 256) FAIL(EXN_EINVAL, "rope_freqs: %d dims (even, 2 to 256)", dims);
  if (!(base > 0) || !std::isfinite(base)) FAIL(EXN_EINVAL, "rope_freqs: base %g", base);
  if (scaling < EXN_ROPE_PLAIN || scaling > EXN_ROPE_INDEX) FAIL(EXN_EINVAL, "rope_freqs: scaling %d", scaling);
  if (scaling != EXN_ROPE_PLAIN && (!(factor > 0) || !std::isfinite(factor)))
    FAIL(EXN_EINVAL, "rope_freqs: factor %g", factor);
  if (scaling == EXN_ROPE_BASE && dims < 4) FAIL(EXN_EINVAL, "rope_freqs: a stretched base of %d dims (4 at least)", dims);
  const bool blend = scaling == EXN_ROPE_TURNS || scaling == EXN_ROPE_INDEX;
  if (blend && (!(kept > 0) || !std::isfinite(kept) || !std::isfinite(low) || !std::isfinite(high) || !(high > low)))
    FAIL(EXN_EINVAL, "rope_freqs: %g tokens, %g to %g turns", kept, low, high);
  if (scaling == EXN_ROPE_INDEX && (!(low > 0) || !(base > 1)))
    FAIL(EXN_EINVAL, "rope_freqs: %g turns, base %g (turns over 0, a base over 1)", low, base);
  if (scaling == EXN_ROPE_BASE) base *= std::pow(factor, (double)dims / (dims - 2));
  double first = 0, last = 0;
  if (scaling == EXN_ROPE_INDEX) {
    auto at = [&](double turns) { return dims * std::log(kept / (2 * kPi * turns)) / (2 * std::log(base)); };
    first = std::min(std::max(std::floor(at(high)), 0.0), dims - 1.0);
    last = std::min(std::max(std::ceil(at(low)), 0.0), dims - 1.0);
    if (last == first) last += 1e-3;   // a step
  }
  for (int j = 0; j < dims / 2; ++j) {
    const double f = std::pow(base, -2.0 * j / dims);
    double r = scaling == EXN_ROPE_LINEAR ? 0.0 : 1.0;
    if (scaling == EXN_ROPE_TURNS) r = std::min(1.0, std::max(0.0, (kept * f / (2 * kPi) - low) / (high - low)));
    if (scaling == EXN_ROPE_INDEX) r = 1.0 - std::min(1.0, std::max(0.0, (j - first) / (last - first)));
    freq[j] = r == 1.0 ? f : r * f + (1 - r) * f / factor;
  }
  return EXN_OK;
}

int exn_rope_create(exn_ctx* ctx, const double* freq, int pairs, int layout, const int32_t* axis, int axes, float amp,
                    exn_rope** out) {
  if (!out) FAIL(EXN_EINVAL, "null output");
  *out = nullptr;
  TRY(use(ctx));
  if (!freq || pairs < 1 || pairs > 128) FAIL(EXN_EINVAL, "rotary: %d pairs (1 to 128)", pairs);
  if (layout != EXN_ROPE_HALF && layout != EXN_ROPE_PAIRS) FAIL(EXN_EINVAL, "rotary: layout %d", layout);
  if (axes < 1 || axes > 8) FAIL(EXN_EINVAL, "rotary: %d axes (1 to 8)", axes);
  if (!std::isfinite(amp)) FAIL(EXN_EINVAL, "rotary: amplitude %g", (double)amp);
  for (int j = 0; j < pairs; ++j) {
    if (!(std::fabs(freq[j]) <= 1024)) FAIL(EXN_EINVAL, "rotary: frequency %d is %g", j, freq[j]);
    if (axis && (axis[j] < 0 || axis[j] >= axes)) FAIL(EXN_EINVAL, "rotary: pair %d on axis %d of %d", j, axis[j], axes);
  }
  hipStreamCaptureStatus cap = hipStreamCaptureStatusNone;
  HIPCHK(hipStreamIsCapturing(ctx->stream, &cap));
  if (cap != hipStreamCaptureStatusNone) FAIL(EXN_ESTATE, "rotary: made before a capture, not in it");
  // the turns, 64-bit fractions, then the axes
  uint64_t words[128 + 64] = {};
  for (int j = 0; j < pairs; ++j) {
    long double t = freq[j] / 6.283185307179586476925286766559L;
    t = std::ldexp(t - std::floor(t), 64);
    words[j] = t >= 18446744073709551615.0L ? 0 : (uint64_t)std::round(t);
    const int32_t a = axis ? axis[j] : 0;
    memcpy((char*)(words + 128) + 4 * j, &a, 4);
  }
  exn_rope* r = new (std::nothrow) exn_rope();
  if (!r) FAIL(EXN_ENOMEM, "rotary: host memory");
  r->device = ctx->device;
  r->pairs = pairs;
  r->layout = layout;
  r->axes = axes;
  r->amp = amp;
  int rc = dev_alloc(&r->mem, sizeof(words));
  if (rc == EXN_OK) {
    hipError_t e = hipMemcpyAsync(r->mem, words, sizeof(words), hipMemcpyHostToDevice, ctx->stream);
    if (e == hipSuccess) e = hipStreamSynchronize(ctx->stream);
    if (e != hipSuccess) {
      exn::set_error("rotary: upload: %s", hipGetErrorString(e));
      rc = EXN_EHIP;
    }
  }
  if (rc != EXN_OK) {
    dev_free(r->mem);
    delete r;
    return rc;
  }
  *out = r;
  return EXN_OK;
}

int exn_rope_free(exn_rope* r) {
  if (!r) return EXN_OK;
  HIPCHK(hipSetDevice(r->device));
  dev_free(r->mem);   // waits for the device
  delete r;
  return EXN_OK;
}

namespace {

bool any_type(int dt) { return dt == EXN_DT_F32 || dt == EXN_DT_BF16 || dt == EXN_DT_F16; }

// one of the two sides' rows in and out, and their norm's weights
int check_side(const char* what, const void* x, int64_t ldx, const float* w, const void* y, int64_t ldy, int64_t width,
               bool same) {
  TRY(check_rows(what, x, ldx, width));
  TRY(check_rows(what, y, ldy, width));
  if ((uintptr_t)w % 16) FAIL(EXN_EINVAL, "%s: norm weights at %p (16-byte aligned)", what, (const void*)w);
  if (x == y && !same) FAIL(EXN_EINVAL, "%s: in place with another type or stride", what);
  return EXN_OK;
}

}  // namespace

int exn_rope_rows(exn_ctx* ctx, const exn_rope* r, const exn_seqs* s, const int32_t* pos, const int32_t* lens,
                  int head_dim, int dt, int odt, float eps, int heads, const void* q, int64_t ldq, const float* wq,
                  void* qo, int64_t ldqo, int kv_heads, const void* k, int64_t ldk, const float* wk, void* ko,
                  int64_t ldko) {
  TRY(check_seqs(ctx, s));
  if (!r) FAIL(EXN_EINVAL, "rope_rows: null rotary");
  if (r->device != ctx->device) FAIL(EXN_EINVAL, "rotary made on device %d, the context's is %d", r->device, ctx->device);
  if (!any_type(dt) || !any_type(odt)) FAIL(EXN_EINVAL, "rope_rows: dtypes %d, %d", dt, odt);
  if (head_dim < 8 || head_dim % 8 || head_dim > 256) FAIL(EXN_EINVAL, "rope_rows: heads of %d (a multiple of 8, at most 256)", head_dim);
  if (2 * r->pairs > head_dim) FAIL(EXN_EINVAL, "rope_rows: %d pairs in heads of %d", r->pairs, head_dim);
  if (heads < 1 || heads > 1024 || kv_heads < 0 || kv_heads > 1024) FAIL(EXN_EINVAL, "rope_rows: %d and %d heads", heads, kv_heads);
  if (!(eps >= 0) || !std::isfinite(eps)) FAIL(EXN_EINVAL, "rope_rows: eps %g", (double)eps);
  if (pos && lens) FAIL(EXN_EINVAL, "rope_rows: positions and lengths (one of them)");
  if (!pos && r->axes != 1) FAIL(EXN_EINVAL, "rope_rows: a rotary of %d axes takes positions", r->axes);
  if ((uintptr_t)pos % 4 || (uintptr_t)lens % 4) FAIL(EXN_EINVAL, "rope_rows: positions and lengths are 4-byte aligned");
  TRY(check_side("rope_rows q", q, ldq, wq, qo, ldqo, (int64_t)heads * head_dim, dt == odt && ldq == ldqo));
  if (kv_heads) TRY(check_side("rope_rows k", k, ldk, wk, ko, ldko, (int64_t)kv_heads * head_dim, dt == odt && ldk == ldko));
  TRY(use(ctx));
  RopeArgs a = {};
  a.tiles = s->tiles[0];
  a.turns = (const uint64_t*)r->mem;
  a.axis = (const int32_t*)(a.turns + 128);
  a.pos = pos;
  a.lens = lens;
  a.pairs = r->pairs;
  a.axes = r->axes;
  a.hd = head_dim;
  a.amp = r->amp;
  a.eps = eps;
  a.t[0] = RopeSide{q, ldq, wq, qo, ldqo, heads};
  if (kv_heads) a.t[1] = RopeSide{k, ldk, wk, ko, ldko, kv_heads};
  return launched("rope_rows", rope_rows(ctx->stream, a, dt, odt, r->layout == EXN_ROPE_HALF, s->ntiles[0], s->longest));
}
