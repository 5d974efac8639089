// rope.hip -- rows of heads as an attention takes them: each head RMS-normed (or not), its first 2 P dims
// turned by its position, in one pass:
//   x <- w x / sqrt(mean(x^2) + eps);   (x, y) <- amp (x cos a - y sin a, x sin a + y cos a),  a = f_j p
// for pair j (dims 2j, 2j + 1, or j, j + P) and the row's position p on the pair's axis.
//
// An angle is p f_j / 2 pi turns, of which only what is past the whole turns counts: f_j / 2 pi is held as a
// 64-bit fraction of a turn, and p times it, modulo 2^64, is that fraction to 2^-64 p, for positions of
// either sign and any size.  An fp32 product p f_j would be 2^-24 p f_j radians off: 0.008 at 131071.
#include "exn_common.h"

#include <type_traits>

namespace exn {

// cos and sin of PH 2^-64 turns: the nearest quarter turn, and series in what is left, at most pi / 4
// (their first left-out terms are under 2^-29 and 2^-31)
__device__ __forceinline__ f32x2 turned(uint64_t ph) {
  const uint64_t a = ph + (1ull << 61);
  const int quarter = (int)(a >> 62);
  const float x = (float)((int64_t)(a & ((1ull << 62) - 1)) - (1ll << 61)) * 3.4061215800998545e-19f;   // 2 pi 2^-64
  const float z = x * x;
  const float s = __builtin_fmaf(__builtin_fmaf(__builtin_fmaf(__builtin_fmaf(z, 1.f / 362880, -1.f / 5040), z, 1.f / 120), z, -1.f / 6), z * x, x);
  const float c = __builtin_fmaf(
      __builtin_fmaf(__builtin_fmaf(__builtin_fmaf(__builtin_fmaf(z, -1.f / 3628800, 1.f / 40320), z, -1.f / 720), z, 1.f / 24), z, -0.5f), z, 1.f);
  const float u = quarter & 1 ? -s : c, v = quarter & 1 ? c : s;
  return quarter & 2 ? f32x2{-u, -v} : f32x2{u, v};
}

// eight consecutive values of a type (EXN_DT_F32 0, EXN_DT_BF16 1, EXN_DT_F16 2)
template <int T>
struct Eight {
  u32x4 w[T == 0 ? 2 : 1];
};
template <int T>
__device__ __forceinline__ void eight_load(Eight<T>& r, const void* p, int64_t at) {
  const char* b = (const char*)p + at * (T == 0 ? 4 : 2);
  r.w[0] = *(const u32x4*)b;
  if constexpr (T == 0) r.w[1] = *(const u32x4*)(b + 16);
}
template <int T>
__device__ __forceinline__ void eight_get(const Eight<T>& r, float* f) {
#pragma unroll
  for (int e = 0; e < 8; ++e)
    f[e] = T == 0 ? __uint_as_float(r.w[e / 4 % (T == 0 ? 2 : 1)][e % 4])
           : T == 1 ? (e & 1 ? bf16_hi(r.w[0][e / 2]) : bf16_lo(r.w[0][e / 2]))
                    : (e & 1 ? f16_hi(r.w[0][e / 2]) : f16_lo(r.w[0][e / 2]));
}
template <int T>
__device__ __forceinline__ void eight_store(void* p, int64_t at, const float* f) {
  char* b = (char*)p + at * (T == 0 ? 4 : 2);
  if constexpr (T == 0) {
    *(f32x4*)b = f32x4{f[0], f[1], f[2], f[3]};
    *(f32x4*)(b + 16) = f32x4{f[4], f[5], f[6], f[7]};
  } else {
    u32x4 w;
#pragma unroll
    for (int e = 0; e < 4; ++e) w[e] = T == 1 ? pack_bf16x2(f[2 * e], f[2 * e + 1]) : pack_f16x2(f[2 * e], f[2 * e + 1]);
    *(u32x4*)b = w;
  }
}

// the sum of v over a head's G lanes, in each of them
template <int G>
__device__ __forceinline__ float head_sum(float v) {
  v += dpp_f<0xB1>(v);
  v += dpp_f<0x4E>(v);
  v += dpp_f<0x141>(v);
  if constexpr (G >= 16) v += dpp_f<0x140>(v);
  if constexpr (G >= 32) {
    float a = v, b = v;
    xswap16(a, b);
    v = a + b;
  }
  return v;
}

// u / n for u n under 2^32, M = 2^32 / n rounded up
__device__ __forceinline__ int over(int u, uint64_t m) { return (int)((uint64_t)(uint32_t)u * m >> 32); }

enum { PAIRED = 0, HALVES = 1, HALVES_ANY = 2 };   // pairs (2j, 2j + 1); (j, j + P), P a multiple of 8; any P

// One workgroup a tile of at most 8 tokens (and a share of their heads, blockIdx.y): the tile's cosines and
// sines into LDS once for all heads, then G lanes a head, 8 dims each, as many heads at a time as 256 threads
// hold, the next ones' loads ahead of the work.  Bytes are what it costs: each value is read and written once.
// 2 documents of 8192 tokens (40 heads of 128, bf16) 73.6 us, 4.6 TB/s of what a copy's 5.2 allow; 4 x 1100..1180 from
// fp32 to fp16 32.1 us, 4.4 TB/s; one token of 4 sequences 3.8 us, a launch.  Two units ahead, or 4096 workgroups for 2048
// of a short call (a tile's angles made once in each), took longer: 16 x 21..257 12.6 us, so 9.7.
template <int XT, int YT, int G, int WAY>
__global__ void __launch_bounds__(256)
k_rope_rows(RopeArgs A) {
  constexpr int SLOTS = 256 / G;
  __shared__ f32x2 cs[8][128];
  __shared__ float buf[WAY == HALVES_ANY ? 256 : 1][8];   // a lane's normed values
  const SeqTile T = A.tiles[blockIdx.x];
  const int tid = threadIdx.x, l = tid % G, slot = tid / G;
  const int live = min(8, T.len - T.t0);
  const int64_t row0 = (int64_t)T.row0 + T.t0;
  const int H = A.t[0].heads + A.t[1].heads, units = live * H;
  const bool has = 8 * l < A.hd;
  float wq[8], wk[8];
  if (has && A.t[0].w) {
    *(f32x4*)wq = *(const f32x4*)(A.t[0].w + 8 * l);
    *(f32x4*)(wq + 4) = *(const f32x4*)(A.t[0].w + 8 * l + 4);
  }
  if (has && A.t[1].w) {
    *(f32x4*)wk = *(const f32x4*)(A.t[1].w + 8 * l);
    *(f32x4*)(wk + 4) = *(const f32x4*)(A.t[1].w + 8 * l + 4);
  }
  // unit u: row u / H of the tile, head u % H of q's and k's
  const int step = SLOTS * gridDim.y;
  Eight<XT> x;
  auto load = [&](int u) __attribute__((always_inline)) {
    if (u >= units || !has) return;
    const int i = over(u, A.magic), h = u - i * H;
    const RopeSide& t = A.t[h >= A.t[0].heads];
    eight_load<XT>(x, t.x, (row0 + i) * t.ldx + (int64_t)(h >= A.t[0].heads ? h - A.t[0].heads : h) * A.hd + 8 * l);
  };
  int u = blockIdx.y * SLOTS + slot;
  load(u);
  for (int z = tid; z < live * A.pairs; z += 256) {
    const int i = over(z, A.pair_magic), j = z - i * A.pairs;
    const int64_t p = A.pos ? A.pos[(row0 + i) * A.axes + A.axis[j]] : (int64_t)(A.lens ? A.lens[T.seq] : 0) + T.t0 + i;
    cs[i][j] = turned((uint64_t)p * A.turns[j]) * A.amp;
  }
  __syncthreads();
  const int P = A.pairs;
  for (int base = blockIdx.y * SLOTS; base < units; base += step, u += step) {
    const int at = min(u, units - 1), i = over(at, A.magic), h = at - i * H, side = h >= A.t[0].heads;
    const RopeSide& t = A.t[side];
    float f[8] = {};
    if (has) eight_get<XT>(x, f);
    load(u + step);
    if (t.w) {
      float ss = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) ss += f[e] * f[e];
      ss = head_sum<G>(ss);
      float eps = A.eps;
      // squares past fp32's range, or under it with nothing else in the root: of values 2^96 times as small or large
      const float by = ss >= 0x1p120f ? 0x1p-96f : ss < 0x1p-100f && eps < 0x1p-100f ? 0x1p96f : 1.f;
      if (__ballot(by != 1.f)) {
        ss = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          f[e] *= by;
          ss += f[e] * f[e];
        }
        ss = head_sum<G>(ss);
        eps = eps * by * by;
      }
      const float inv = rsqrtf(ss * A.per + eps);
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] = f[e] * inv * (side ? wk[e] : wq[e]);   // weights of any size: the head first
    }
    float y[8];
    if constexpr (WAY == PAIRED) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const f32x2 r = cs[i][min(4 * l + e, 127)];
        const bool turn = 4 * l + e < P;
        y[2 * e] = turn ? f[2 * e] * r[0] - f[2 * e + 1] * r[1] : f[2 * e];
        y[2 * e + 1] = turn ? f[2 * e] * r[1] + f[2 * e + 1] * r[0] : f[2 * e + 1];
      }
    } else if constexpr (WAY == HALVES) {
      const int lh = P / 8;
      const bool second = l >= lh, turn = l < 2 * lh;
      const int from = (tid & 63) + (!turn ? 0 : second ? -lh : lh), j0 = turn ? 8 * (second ? l - lh : l) : 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float o = __shfl(f[e], from, 64);
        const f32x2 r = cs[i][j0 + e];
        const float v = f[e] * r[0] + (second ? o : -o) * r[1];
        y[e] = turn ? v : f[e];
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; e += 4) *(f32x4*)&buf[tid][e] = f32x4{f[e], f[e + 1], f[e + 2], f[e + 3]};
      asm volatile("" ::: "memory");   // a head's lanes are one wave's, whose LDS accesses keep their order
      const float* head = &buf[tid - l][0];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int d = 8 * l + e;
        const bool second = d >= P, turn = d < 2 * P;
        const float o = head[!turn ? d : second ? d - P : d + P];
        const f32x2 r = cs[i][!turn ? 0 : second ? d - P : d];
        y[e] = turn ? f[e] * r[0] + (second ? o : -o) * r[1] : f[e];
      }
      asm volatile("" ::: "memory");
    }
    if (u < units && has)
      eight_store<YT>(t.y, (row0 + i) * t.ldy + (int64_t)(side ? h - A.t[0].heads : h) * A.hd + 8 * l, y);
  }
}

hipError_t rope_rows(hipStream_t s, const RopeArgs& args, int xt, int yt, int halves, int64_t ntiles, int longest) {
  if (ntiles == 0) return hipSuccess;
  RopeArgs a = args;
  const int H = a.t[0].heads + a.t[1].heads, g = a.hd <= 64 ? 8 : a.hd <= 128 ? 16 : 32, slots = 256 / g;
  a.magic = ((1ull << 32) + H - 1) / H;
  a.pair_magic = ((1ull << 32) + a.pairs - 1) / a.pairs;
  a.per = 1.f / a.hd;
  const int passes = ((longest < 8 ? longest : 8) * H + slots - 1) / slots;
  int64_t y = 2048 / ntiles;   // workgroups that share a tile's heads
  y = y < 1 ? 1 : y > passes ? passes : y;
  const dim3 grid((unsigned)ntiles, (unsigned)y);
  const int way = !halves ? PAIRED : a.pairs % 8 ? HALVES_ANY : HALVES;
  auto go = [&](auto kern) { hipLaunchKernelGGL(kern, grid, dim3(256), 0, s, a); };
  typedef std::integral_constant<int, 0> I0;
  typedef std::integral_constant<int, 1> I1;
  typedef std::integral_constant<int, 2> I2;
  typedef std::integral_constant<int, 8> G8;
  typedef std::integral_constant<int, 16> G16;
  typedef std::integral_constant<int, 32> G32;
  auto ways = [&](auto x, auto y, auto gg) {
    constexpr int X = decltype(x)::value, Y = decltype(y)::value, G = decltype(gg)::value;
    way == PAIRED ? go(k_rope_rows<X, Y, G, PAIRED>) : way == HALVES ? go(k_rope_rows<X, Y, G, HALVES>)
                                                                     : go(k_rope_rows<X, Y, G, HALVES_ANY>);
  };
  auto lanes = [&](auto x, auto y) { g == 8 ? ways(x, y, G8()) : g == 16 ? ways(x, y, G16()) : ways(x, y, G32()); };
  auto outs = [&](auto x) { yt == 0 ? lanes(x, I0()) : yt == 1 ? lanes(x, I1()) : lanes(x, I2()); };
  xt == 0 ? outs(I0()) : xt == 1 ? outs(I1()) : outs(I2());
  return hipGetLastError();
}

}  // namespace exn
