// packed.hip -- causal attention over whole prompts of different lengths, packed one after the
// other: for query row i of a sequence and head h (of g query heads to a key/value head)
//   o[i, h] = sum_{j <= i} p_j v[j, h / g] / sum_{j <= i} p_j,  p_j = 2^(scale log2(e) q[i, h].k[j, h / g] - m).
#include "exn_common.h"

namespace exn {

template <int BF>
__device__ __forceinline__ float load16(const uint16_t* p) {
  return BF ? bf16_to_f32(*p) : f16_to_f32(*p);
}
__device__ __forceinline__ uint16_t store16(float v, int bf) {
  return bf ? __builtin_bit_cast(uint16_t, (__bf16)v) : __builtin_bit_cast(uint16_t, (_Float16)v);
}

// one wave a query row and head: 64 keys at a time, a score a lane, then a dim (two at HD 128) a lane
template <int BF, int HD>
__global__ void __launch_bounds__(64)
k_attend_packed(const SeqTile* __restrict__ tiles, int tt, int group, const uint16_t* __restrict__ q, int64_t ldq,
                const uint16_t* __restrict__ k, int64_t ldk, const uint16_t* __restrict__ v, int64_t ldv, float scale,
                uint16_t* __restrict__ out, int obf, int64_t ldo) {
  __shared__ float qs[HD], ps[64];
  const SeqTile t = tiles[blockIdx.x];
  const int lane = threadIdx.x, h = blockIdx.y, i = t.t0 + blockIdx.z;
  if (i >= t.len) return;
  const uint16_t* qr = q + (int64_t)(t.row0 + i) * ldq + h * HD;
  for (int d = lane; d < HD; d += 64) qs[d] = load16<BF>(qr + d) * scale;
  __syncthreads();
  const uint16_t* kb = k + (int64_t)t.row0 * ldk + h / group * HD;
  const uint16_t* vb = v + (int64_t)t.row0 * ldv + h / group * HD;
  float m = -INFINITY, l = 0.f, o[HD / 64] = {};
  for (int j0 = 0; j0 <= i; j0 += 64) {
    const int j = j0 + lane;
    float s = -INFINITY;
    if (j <= i) {
      s = 0.f;
      for (int d = 0; d < HD; ++d) s += qs[d] * load16<BF>(kb + (int64_t)j * ldk + d);
    }
    const float mn = fmaxf(m, wave_max(s)), mu = mn == -INFINITY ? 0.f : mn;
    const float a = exp2f(m - mu), p = exp2f(s - mu);
    l = l * a + wave_sum(p);
    m = mn;
    __syncthreads();
    ps[lane] = p;
    __syncthreads();
    for (int e = 0; e < HD / 64; ++e) {
      float acc = o[e] * a;
      for (int c = 0; c < 64 && j0 + c <= i; ++c) acc += ps[c] * load16<BF>(vb + (int64_t)(j0 + c) * ldv + e * 64 + lane);
      o[e] = acc;
    }
  }
  for (int e = 0; e < HD / 64; ++e)
    out[(int64_t)(t.row0 + i) * ldo + h * HD + e * 64 + lane] = store16(l > 0.f || l != l ? o[e] / l : 0.f, obf);
}

hipError_t attend_packed(hipStream_t s, const SeqTile* const* tiles, const int64_t* ntiles, int bf16, int heads,
                         int kv_heads, int head_dim, const uint16_t* q, int64_t ldq, const uint16_t* k, int64_t ldk,
                         const uint16_t* v, int64_t ldv, float scale, uint16_t* out, int obf, int64_t ldo) {
  if (ntiles[0] == 0) return hipSuccess;
  const dim3 grid((unsigned)ntiles[0], heads, SEQ_TT0);
  const float sc = scale * 1.4426950408889634f;
  auto go = [&](auto kern) {
    hipLaunchKernelGGL(kern, grid, dim3(64), 0, s, tiles[0], SEQ_TT0, heads / kv_heads, q, ldq, k, ldk, v, ldv, sc, out,
                       obf, ldo);
  };
  if (bf16)
    head_dim == 128 ? go(k_attend_packed<1, 128>) : go(k_attend_packed<1, 64>);
  else
    head_dim == 128 ? go(k_attend_packed<0, 128>) : go(k_attend_packed<0, 64>);
  return hipGetLastError();
}

}  // namespace exn
