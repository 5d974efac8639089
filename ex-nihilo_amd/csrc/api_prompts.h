// api_prompts.h -- what the prompt side's entry points (api_prompts.hip, api_prefixes.hip) check
// alike: heads, types, rows, plans and the 8-bit cache.
#pragma once

#include "api_host.h"

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
