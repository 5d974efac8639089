// encoder.hip -- the prompt encoder's own kernels (Qwen3-VL-8B's text model, read for its
// last block's states: src/encoder.lisp:143-183).  Its products, norms, q/k norm with the
// rotary, causal attention and SwiGLU run on the DiT's kernels (gemm.hip, attn.hip,
// eltwise.hip): the text model has the DiT block's widths (4096, 32 heads of 128, FFN 12288).
#include "exn_common.h"

namespace exn {

// one workgroup a token: row ids[t] of the token embedding, from Q8_0 codes and scales
// (fp32(d) x q, exact) or from fp32 rows; an id outside 0 .. vocab-1 gives a row of zeros (the
// host entry point rejects such ids before they get here)
__global__ void __launch_bounds__(256)
k_enc_embed(const int32_t* __restrict__ ids, int64_t vocab, const int8_t* __restrict__ qs,
            const uint16_t* __restrict__ d, const float* __restrict__ f32, int width, float* __restrict__ out) {
  const int t = blockIdx.x;
  const int64_t id = ids[t];
  float* o = out + (int64_t)t * width;
  const bool live = id >= 0 && id < vocab;
  for (int c = 4 * threadIdx.x; c < width; c += 1024) {
    if (!live) {
      *(f32x4*)(o + c) = f32x4{0.f, 0.f, 0.f, 0.f};
    } else if (f32) {
      *(f32x4*)(o + c) = *(const f32x4*)(f32 + id * width + c);
    } else {
      const float sc = f16_to_f32(d[(id * width + c) / 32]);
      const uint32_t q = *(const uint32_t*)(qs + id * width + c);
      f32x4 v;
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = sc * (float)(int8_t)(q >> (8 * e));
      *(f32x4*)(o + c) = v;
    }
  }
}

hipError_t enc_embed(hipStream_t s, const int32_t* ids, int n, int64_t vocab, const int8_t* qs, const uint16_t* d,
                     const float* f32, int width, float* out) {
  if (n <= 0) return hipSuccess;
  if (width % 32) return hipErrorInvalidValue;
  hipLaunchKernelGGL(k_enc_embed, dim3(n), dim3(256), 0, s, ids, vocab, qs, d, f32, width, out);
  return hipGetLastError();
}

// A packed pass's q | k | v rows as the attention over them takes them: q and k of each head RMS-normed
// (weights WQ, WK, eps 1e-6) and turned by CS, v as it is, all fp16 in rows of 6144 (32 query heads, 8 for
// k and 8 for v).  From the product's fp16 rows in place (S 0), or from a split product's S partial sums,
// which make the same fp16 rows first.  16 lanes a head, 8 dims each; bytes are what it costs.
template <int S>
__global__ void __launch_bounds__(256)
k_enc_qkv_rows(uint16_t* __restrict__ qkv, const float* __restrict__ part, int64_t n, const float* __restrict__ wq,
               const float* __restrict__ wk, const float* __restrict__ cs) {
  constexpr int HEADS = S ? 48 : 40;   // v stays where it is when it is there already
  const int64_t i = (int64_t)blockIdx.x * 16 + threadIdx.x / 16;
  if (i >= n * HEADS) return;   // whole groups of 16 lanes
  const int64_t t = i / HEADS;
  const int h = (int)(i % HEADS), d8 = threadIdx.x % 16 * 8;
  uint16_t* row = qkv + t * 6144 + h * 128 + d8;
  u32x4 u;
  if constexpr (S == 0) {
    u = *(const u32x4*)row;
  } else {
    const float* p = part + t * 6144 + h * 128 + d8;
    f32x4 a = *(const f32x4*)p, b = *(const f32x4*)(p + 4);
#pragma unroll
    for (int z = 1; z < S; ++z) {
      a += *(const f32x4*)(p + (int64_t)z * n * 6144);
      b += *(const f32x4*)(p + (int64_t)z * n * 6144 + 4);
    }
    u = u32x4{pack_f16x2(a[0], a[1]), pack_f16x2(a[2], a[3]), pack_f16x2(b[0], b[1]), pack_f16x2(b[2], b[3])};
  }
  if (h < 40) {
    const float* w = (h < 32 ? wq : wk) + d8;
    float a[8], ss = 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      a[2 * e] = f16_lo(u[e]);
      a[2 * e + 1] = f16_hi(u[e]);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) ss += a[e] * a[e];
    const float inv = rsqrtf(row16_sum(ss) * (1.f / 128.f) + 1e-6f);
    const float* c = cs + t * 128 + d8;   // cos, sin of pairs d8 / 2 ..
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float x = a[2 * e] * inv * w[2 * e], y = a[2 * e + 1] * inv * w[2 * e + 1];
      u[e] = pack_f16x2(x * c[2 * e] - y * c[2 * e + 1], x * c[2 * e + 1] + y * c[2 * e]);
    }
  }
  *(u32x4*)row = u;
}

hipError_t enc_qkv_rows(hipStream_t s, uint16_t* qkv, const float* part, int S, int64_t n, const float* wq,
                        const float* wk, const float* cs) {
  if (n <= 0) return hipSuccess;
  const dim3 grid((unsigned)((n * (S ? 48 : 40) + 15) / 16));
  auto go = [&](auto kern) { hipLaunchKernelGGL(kern, grid, dim3(256), 0, s, qkv, part, n, wq, wk, cs); };
  switch (S) {
    case 0: go(k_enc_qkv_rows<0>); break;
    case 1: go(k_enc_qkv_rows<1>); break;
    case 2: go(k_enc_qkv_rows<2>); break;
    case 3: go(k_enc_qkv_rows<3>); break;
    case 4: go(k_enc_qkv_rows<4>); break;
    case 5: go(k_enc_qkv_rows<5>); break;
    case 6: go(k_enc_qkv_rows<6>); break;
    case 7: go(k_enc_qkv_rows<7>); break;
    case 8: go(k_enc_qkv_rows<8>); break;
    default: return hipErrorInvalidValue;
  }
  return hipGetLastError();
}

}  // namespace exn
