// kv8.hip -- keys and values kept in 8 bits, a scale for each block of 64 tokens and key/value
// head, and the attention over them.  A block of rows x is held as codes rint(x / d) and
//   d = max |x| / 127, rounded up to 12 significant bits:
// (c + 1/2) d then has at most 20 bits and x at most 11, so that x / d is either exactly between
// two codes or at least 2^-20 (relative) away from there: every correctly rounded quotient gives
// the same code, no |code| is over 127, and code x d (19 bits) is exact in fp32.  A block that is
// not full stays in its 16 bits (the tail) until its 64th token: no value is rounded twice, and
// tokens appended one by one give the cache that all at once give.  A block with an infinity or a
// NaN has the scale NaN: what is read of it is NaN.
#include "exn_common.h"

namespace exn {

__device__ __forceinline__ float ld16(const uint16_t* p, int bf) { return bf ? bf16_to_f32(*p) : f16_to_f32(*p); }
__device__ __forceinline__ uint16_t st16(float v, int bf) {
  return bf ? __builtin_bit_cast(uint16_t, (__bf16)v) : __builtin_bit_cast(uint16_t, (_Float16)v);
}

// One workgroup a (sequence, key/value head, block the step can touch, keys or values).  Block 0's
// also writes the tail, after it has read the old one: the one slot serves the block that fills and
// the block begun after it.
__global__ void __launch_bounds__(256)
k_kv8_append(Kv8 c, const SeqTile* __restrict__ seqs, const uint16_t* __restrict__ k, int64_t ldk,
             const uint16_t* __restrict__ v, int64_t ldv) {
  __shared__ uint32_t tops[4];
  const SeqTile t = seqs[blockIdx.x / c.kv_heads];
  const int h = blockIdx.x % c.kv_heads, isv = blockIdx.z, hd = c.head_dim, tid = threadIdx.x;
  const int base = kv8_base(c, t.seq), total = kv8_total(c, base, t.len);
  const int first = base / 64, b = first + blockIdx.y;
  if (t.len == 0 || total <= base) return;
  const int64_t ld = isv ? ldv : ldk;
  const uint16_t* x = (isv ? v : k) + (int64_t)t.row0 * ld + h * hd;
  uint16_t* tail = (isv ? c.tv : c.tk) + ((int64_t)t.seq * c.kv_heads + h) * 64 * hd;
  if ((b + 1) * 64 <= total) {   // the block is full now
    auto at = [&](int e) {
      const int pos = b * 64 + e / hd;
      return ld16(pos < base ? tail + e : x + (pos - base) * ld + e % hd, c.bf16);
    };
    uint32_t top = 0;
    for (int e = tid; e < 64 * hd; e += 256) top = max(top, __float_as_uint(at(e)) & 0x7FFFFFFFu);
    for (int o = 32; o > 0; o >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, o, 64));
    if (tid % 64 == 0) tops[tid / 64] = top;
    __syncthreads();
    const float d = kv8_scale(max(max(tops[0], tops[1]), max(tops[2], tops[3])));
    const int64_t page = kv8_page(c, t.seq, b);
    if (page >= 0) {
      int8_t* dst = (isv ? c.v : c.k) + (page * c.kv_heads + h) * 64 * hd;
      for (int e = tid; e < 64 * hd; e += 256) dst[isv ? e % hd * 64 + e / hd : e] = kv8_code(at(e), d);
      if (tid == 0) c.scales[(page * c.kv_heads + h) * 2 + isv] = d;
    }
  }
  if (blockIdx.y == 0 && total % 64) {
    __syncthreads();   // the old tail has been read
    const int from = max(base, total / 64 * 64);
    for (int e = tid; e < (total - from) * hd; e += 256) {
      const int pos = from + e / hd;
      tail[pos % 64 * hd + e % hd] = x[(pos - base) * ld + e % hd];
    }
  }
}

hipError_t kv8_append(hipStream_t s, const Kv8& c, const SeqTile* seqs, int n, int longest, const uint16_t* k,
                      int64_t ldk, const uint16_t* v, int64_t ldv) {
  if (n == 0 || longest == 0) return hipSuccess;
  const dim3 grid(n * c.kv_heads, (62 + longest) / 64 + 1, 2);
  hipLaunchKernelGGL(k_kv8_append, grid, dim3(256), 0, s, c, seqs, k, ldk, v, ldv);
  return hipGetLastError();
}

// the step's rows as the cache holds them, 16 bits (code x d rounded once); a place past the
// table, or on a page that is none, reads zeros
__global__ void __launch_bounds__(256)
k_kv8_read(Kv8 c, const SeqTile* __restrict__ tiles, int tt, uint16_t* __restrict__ k, int64_t ldk,
           uint16_t* __restrict__ v, int64_t ldv) {
  const SeqTile t = tiles[blockIdx.x];
  const int h = blockIdx.y, isv = blockIdx.z, hd = c.head_dim;
  const int base = kv8_base(c, t.seq), total = kv8_total(c, base, t.len);
  for (int e = threadIdx.x; e < min(tt, t.len - t.t0) * hd; e += 256) {
    const int i = t.t0 + e / hd, d = e % hd, pos = base + i;
    uint16_t y = 0;
    if (pos < total / 64 * 64) {
      const int64_t page = kv8_page(c, t.seq, pos / 64);
      if (page >= 0) {
        const int64_t ph = page * c.kv_heads + h;
        const int8_t q = (isv ? c.v + ph * 64 * hd + d * 64 + pos % 64 : c.k + ph * 64 * hd + pos % 64 * hd + d)[0];
        y = st16((float)q * c.scales[ph * 2 + isv], c.bf16);
      }
    } else if (pos < total) {
      y = (isv ? c.tv : c.tk)[(((int64_t)t.seq * c.kv_heads + h) * 64 + pos % 64) * hd + d];
    }
    (isv ? v : k)[(int64_t)(t.row0 + i) * (isv ? ldv : ldk) + h * hd + d] = y;
  }
}

hipError_t kv8_read(hipStream_t s, const Kv8& c, const SeqTile* tiles, int64_t n, int tt, uint16_t* k, int64_t ldk,
                    uint16_t* v, int64_t ldv) {
  if (n == 0) return hipSuccess;
  hipLaunchKernelGGL(k_kv8_read, dim3((unsigned)n, c.kv_heads, 2), dim3(256), 0, s, c, tiles, tt, k, ldk, v, ldv);
  return hipGetLastError();
}

__global__ void k_kv8_advance(Kv8 c, const SeqTile* __restrict__ seqs, int n) {
  const int i = blockIdx.x * blockDim.x + threadIdx.x;
  if (i < n) c.lens[seqs[i].seq] = kv8_total(c, kv8_base(c, seqs[i].seq), seqs[i].len);
}

hipError_t kv8_advance(hipStream_t s, const Kv8& c, const SeqTile* seqs, int n) {
  if (n == 0) return hipSuccess;
  hipLaunchKernelGGL(k_kv8_advance, dim3((n + 255) / 256), dim3(256), 0, s, c, seqs, n);
  return hipGetLastError();
}

// one wave a query row and head: 64 keys at a time, a score a lane, then a dim (two at 128) a lane
template <int HD>
__global__ void __launch_bounds__(64)
k_kv8_attend(Kv8 c, const SeqTile* __restrict__ tiles, int group, const uint16_t* __restrict__ q, int64_t ldq,
             float scale, uint16_t* __restrict__ out, int obf, int64_t ldo) {
  __shared__ float qs[HD], ps[64];
  const SeqTile t = tiles[blockIdx.x];
  const int lane = threadIdx.x, h = blockIdx.y, kvh = h / group, i = t.t0 + blockIdx.z;
  if (i >= t.len) return;
  const int base = kv8_base(c, t.seq), total = kv8_total(c, base, t.len), lim = min(base + i + 1, total);
  for (int d = lane; d < HD; d += 64) qs[d] = ld16(q + (int64_t)(t.row0 + i) * ldq + h * HD + d, c.bf16) * scale;
  __syncthreads();
  float m = -INFINITY, l = 0.f, o[HD / 64] = {};
  for (int j0 = 0; j0 < lim; j0 += 64) {
    const bool full = j0 + 64 <= total;
    const int64_t page = full ? kv8_page(c, t.seq, j0 / 64) : 0;
    if (page < 0) continue;
    const int64_t ph = page * c.kv_heads + kvh, th = ((int64_t)t.seq * c.kv_heads + kvh) * 64 * HD;
    const float kd = full ? c.scales[ph * 2] : 1.f, vd = full ? c.scales[ph * 2 + 1] : 1.f;
    float s = -INFINITY;
    if (j0 + lane < lim) {
      s = 0.f;
      for (int d = 0; d < HD; ++d)
        s += qs[d] * (full ? (float)c.k[ph * 64 * HD + lane * HD + d] : ld16(c.tk + th + lane * HD + d, c.bf16));
      s *= kd;
    }
    const float mn = fmaxf(m, wave_max(s)), mu = mn == -INFINITY ? 0.f : mn;
    const float a = exp2f(m - mu), p = exp2f(s - mu);
    l = l * a + wave_sum(p);
    m = mn;
    __syncthreads();
    ps[lane] = p;
    __syncthreads();
    for (int e = 0; e < HD / 64; ++e) {
      const int d = e * 64 + lane;
      float acc = 0.f;
      for (int j = 0; j < 64 && j0 + j < lim; ++j)
        acc += ps[j] * (full ? (float)c.v[ph * 64 * HD + d * 64 + j] : ld16(c.tv + th + j * HD + d, c.bf16));
      o[e] = o[e] * a + acc * vd;
    }
  }
  for (int e = 0; e < HD / 64; ++e)
    out[(int64_t)(t.row0 + i) * ldo + h * HD + e * 64 + lane] = st16(l > 0.f || l != l ? o[e] / l : 0.f, obf);
}

int64_t kv8_attend_part(int64_t rows, int seqs, int longest, int heads, int kv_heads, int head_dim, int cols) { return 0; }

hipError_t kv8_attend(hipStream_t s, const Kv8& c, const SeqTile* const* tiles, const int64_t* ntiles, int64_t rows,
                      int seqs, int longest, int heads, const uint16_t* q, int64_t ldq, float scale, uint16_t* out,
                      int obf, int64_t ldo, float* part, int64_t part_cap) {
  if (ntiles[0] == 0) return hipSuccess;
  const dim3 grid((unsigned)ntiles[0], heads, SEQ_TT0);
  const float sc = scale * 1.4426950408889634f;
  if (c.head_dim == 128)
    hipLaunchKernelGGL(k_kv8_attend<128>, grid, dim3(64), 0, s, c, tiles[0], heads / c.kv_heads, q, ldq, sc, out, obf, ldo);
  else
    hipLaunchKernelGGL(k_kv8_attend<64>, grid, dim3(64), 0, s, c, tiles[0], heads / c.kv_heads, q, ldq, sc, out, obf, ldo);
  return hipGetLastError();
}

}  // namespace exn
