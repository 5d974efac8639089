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

#include <algorithm>
#include <cmath>
#include <type_traits>

namespace exn {

__device__ __forceinline__ float ld16(const uint16_t* p, int bf) { return bf ? bf16_to_f32(*p) : f16_to_f32(*p); }
// HD / 16 consecutive 16-bit values
template <int HD>
struct Piece {
  uint32_t w[HD / 32];
};
template <int HD>
__device__ __forceinline__ Piece<HD> load_piece(const uint16_t* p) {
  if constexpr (HD == 128) {
    const u32x4 x = *(const u32x4*)p;
    return Piece<HD>{{x[0], x[1], x[2], x[3]}};
  } else {
    const u32x2 x = *(const u32x2*)p;
    return Piece<HD>{{x[0], x[1]}};
  }
}
template <int HD>
__device__ __forceinline__ void store_piece(uint16_t* p, const Piece<HD>& x) {
  if constexpr (HD == 128)
    *(u32x4*)p = u32x4{x.w[0], x.w[1], x.w[2], x.w[3]};
  else
    *(u32x2*)p = u32x2{x.w[0], x.w[1]};
}
template <int BF>
__device__ __forceinline__ float half_of(uint32_t w, int e) {
  return BF ? (e & 1 ? bf16_hi(w) : bf16_lo(w)) : (e & 1 ? f16_hi(w) : f16_lo(w));
}
// kv8_code of four values, a byte each; R = 1 / d to an ulp, d of at least 2^-100.  One correction makes
// a quotient that is exactly between two codes exact, and any other is further from there than it is
// off; adding 1.5 x 2^23 rounds it to the nearest even whole number, in the low bits.
__device__ __forceinline__ uint32_t kv8_codes4(const float* x, float d, float r) {
  uint32_t u[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float q = x[e] * r;
    u[e] = __float_as_uint(__builtin_fmaf(__builtin_fmaf(-q, d, x[e]), r, q) + 12582912.f);
  }
  const uint32_t a = __builtin_amdgcn_perm(u[1], u[0], 0x0C0C0400u), b = __builtin_amdgcn_perm(u[3], u[2], 0x0C0C0400u);
  return __builtin_amdgcn_perm(b, a, 0x05040100u);
}

// One workgroup a (sequence and key/value head, block the step can touch, keys or values): bytes are
// what it costs.  A thread has 4 tokens x HD / 16 dims of a block in registers, from the tail or the
// new rows, between the block's largest |x| and its codes; values leave through LDS, where four
// tokens' codes of a dim are a dword.  Block 0's workgroup also writes the tail, after it has read the
// old one: the one slot serves the block that fills and the block begun after it.  With the read below,
// 8 x 1100 tokens (8 heads of 128, bf16) 22.1 us, 4.9 TB/s of what a copy's 5.1 allow; 64 x 1 token
// 10 us, two launches' time.
template <int BF, int HD>
__global__ void __launch_bounds__(256)
k_kv8_append(Kv8 c, const SeqTile* __restrict__ seqs, const uint16_t* __restrict__ k, int64_t ldk,
             const uint16_t* __restrict__ v, int64_t ldv) {
  constexpr int E = HD / 16, LD = 17;   // dims a thread; dwords a dim's row in LDS
  __shared__ uint32_t tops[4], cols[HD * LD];
  const SeqTile t = seqs[blockIdx.x / c.kv_heads];
  const int h = blockIdx.x % c.kv_heads, isv = blockIdx.z, tid = threadIdx.x;
  const int base = kv8_base(c, t.seq), total = kv8_total(c, base, t.len);
  const int first = base / 64, b = first + blockIdx.y;
  if (t.len == 0 || total <= base) return;
  const int64_t ld = isv ? ldv : ldk;
  const uint16_t* x = (isv ? v : k) + (int64_t)t.row0 * ld + h * HD;
  uint16_t* tail = (isv ? c.tv : c.tk) + ((int64_t)t.seq * c.kv_heads + h) * 64 * HD;
  const int d0 = (tid & 15) * E, quad = tid >> 4;
  if ((b + 1) * 64 <= total) {   // the block is full now
    const int64_t page = kv8_page(c, t.seq, b);
    Piece<HD> r[4];
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int pos = b * 64 + 4 * quad + i;
      r[i] = load_piece<HD>(pos < base ? tail + pos % 64 * HD + d0 : x + (int64_t)(pos - base) * ld + d0);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int e = 0; e < E; ++e) top = max(top, __float_as_uint(half_of<BF>(r[i].w[e / 2], e)) & 0x7FFFFFFFu);
    for (int o = 32; o > 0; o >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, o, 64));
    if (tid % 64 == 0) tops[tid / 64] = top;
    __syncthreads();
    const float d = kv8_scale(max(max(tops[0], tops[1]), max(tops[2], tops[3])));
    if (page >= 0) {
      int8_t* dst = (isv ? c.v : c.k) + (page * c.kv_heads + h) * 64 * HD;
      uint32_t code[4][E / 4];
      const bool plain = d >= 0x1p-100f;   // else zeros, values next to nothing, or not finite ones
      const float rd = __builtin_amdgcn_rcpf(d);
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e4 = 0; e4 < E / 4; ++e4) {
          float y[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) y[e] = half_of<BF>(r[i].w[2 * e4 + e / 2], e);
          code[i][e4] = kv8_codes4(y, d, rd);
        }
      if (!plain) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int e4 = 0; e4 < E / 4; ++e4) {
            uint32_t w = 0;
#pragma unroll
            for (int e = 0; e < 4; ++e)
              w |= (uint32_t)(uint8_t)kv8_code(half_of<BF>(r[i].w[2 * e4 + e / 2], e), d) << (8 * e);
            code[i][e4] = w;
          }
      }
      if (isv) {
#pragma unroll
        for (int e = 0; e < E; ++e) {
          uint32_t w = 0;
#pragma unroll
          for (int i = 0; i < 4; ++i) w |= (code[i][e / 4] >> (8 * (e % 4)) & 0xFFu) << (8 * i);
          cols[(d0 + e) * LD + quad] = w;
        }
        __syncthreads();
        for (int i = tid; i < HD * 4; i += 256) {
          const uint32_t* p = cols + i / 4 * LD + i % 4 * 4;
          *(u32x4*)(dst + i * 16) = u32x4{p[0], p[1], p[2], p[3]};
        }
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          int8_t* p = dst + (4 * quad + i) * HD + d0;
          if constexpr (HD == 128)
            *(u32x2*)p = u32x2{code[i][0], code[i][1]};
          else
            *(uint32_t*)p = code[i][0];
        }
      }
      if (tid == 0) c.scales[(page * c.kv_heads + h) * 2 + isv] = d;
    }
  }
  if (blockIdx.y == 0 && total % 64) {
    __syncthreads();   // the old tail has been read
    const int from = max(base, total / 64 * 64);
    for (int pos = from + quad; pos < total; pos += 16)
      store_piece<HD>(tail + pos % 64 * HD + d0, load_piece<HD>(x + (int64_t)(pos - base) * ld + d0));
  }
}

hipError_t kv8_append(hipStream_t s, const Kv8& c, const SeqTile* seqs, int n, int longest, const uint16_t* k,
                      int64_t ldk, const uint16_t* v, int64_t ldv) {
  if (n == 0 || longest == 0) return hipSuccess;
  if ((int64_t)n * c.kv_heads > WG256_MAX) return hipErrorInvalidConfiguration;
  const dim3 grid(n * c.kv_heads, (62 + longest) / 64 + 1, 2);
  auto go = [&](auto kern) { hipLaunchKernelGGL(kern, grid, dim3(256), 0, s, c, seqs, k, ldk, v, ldv); };
  if (c.head_dim == 128)
    c.bf16 ? go(k_kv8_append<1, 128>) : go(k_kv8_append<0, 128>);
  else
    c.bf16 ? go(k_kv8_append<1, 64>) : go(k_kv8_append<0, 64>);
  return hipGetLastError();
}

// The step's rows as the cache holds them, 16 bits (code x d rounded once): workgroups and threads as
// in the append; a place past the table, or on a page that is none, reads zeros
template <int HD>
__global__ void __launch_bounds__(256)
k_kv8_read(Kv8 c, const SeqTile* __restrict__ seqs, uint16_t* __restrict__ k, int64_t ldk, uint16_t* __restrict__ v,
           int64_t ldv) {
  constexpr int E = HD / 16, LD = 17;
  __shared__ uint32_t cols[HD * LD];
  const SeqTile t = seqs[blockIdx.x / c.kv_heads];
  const int h = blockIdx.x % c.kv_heads, isv = blockIdx.z, tid = threadIdx.x;
  const int base = kv8_base(c, t.seq), total = kv8_total(c, base, t.len);
  const int b = base / 64 + blockIdx.y, end = base + t.len;   // the last places may be past the table
  if (t.len == 0 || b * 64 >= end) return;
  const int64_t ld = isv ? ldv : ldk;
  uint16_t* y = (isv ? v : k) + (int64_t)t.row0 * ld + h * HD;
  const int d0 = (tid & 15) * E, quad = tid >> 4;
  Piece<HD> r[4] = {};
  if ((b + 1) * 64 <= total) {
    const int64_t page = kv8_page(c, t.seq, b);
    if (page >= 0) {
      const int64_t ph = page * c.kv_heads + h;
      const float d = c.scales[ph * 2 + isv];
      const int8_t* src = (isv ? c.v : c.k) + ph * 64 * HD;
      uint32_t code[4][E / 4] = {};
      if (isv) {
        for (int i = tid; i < HD * 4; i += 256) {
          const u32x4 w = *(const u32x4*)(src + i * 16);
          uint32_t* p = cols + i / 4 * LD + i % 4 * 4;
          p[0] = w[0];
          p[1] = w[1];
          p[2] = w[2];
          p[3] = w[3];
        }
        __syncthreads();
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const uint32_t w = cols[(d0 + e) * LD + quad];
#pragma unroll
          for (int i = 0; i < 4; ++i) code[i][e / 4] |= (w >> (8 * i) & 0xFFu) << (8 * (e % 4));
        }
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int8_t* p = src + (4 * quad + i) * HD + d0;
          if constexpr (HD == 128) {
            const u32x2 w = *(const u32x2*)p;
            code[i][0] = w[0];
            code[i][1] = w[1];
          } else {
            code[i][0] = *(const uint32_t*)p;
          }
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < E; e += 2) {
          const float a = d * (float)(int8_t)(code[i][e / 4] >> (8 * (e % 4)));
          const float z = d * (float)(int8_t)(code[i][e / 4] >> (8 * (e % 4) + 8));
          r[i].w[e / 2] = c.bf16 ? pack_bf16x2(a, z) : pack_f16x2_in(a, z);
        }
    }
  } else {
    const uint16_t* tail = (isv ? c.tv : c.tk) + ((int64_t)t.seq * c.kv_heads + h) * 64 * HD;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (b * 64 + 4 * quad + i < total) r[i] = load_piece<HD>(tail + (4 * quad + i) * HD + d0);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int pos = b * 64 + 4 * quad + i;
    if (pos >= base && pos < end) store_piece<HD>(y + (int64_t)(pos - base) * ld + d0, r[i]);
  }
}

hipError_t kv8_read(hipStream_t s, const Kv8& c, const SeqTile* seqs, int n, int longest, uint16_t* k, int64_t ldk,
                    uint16_t* v, int64_t ldv) {
  if (n == 0 || longest == 0) return hipSuccess;
  if ((int64_t)n * c.kv_heads > WG256_MAX) return hipErrorInvalidConfiguration;
  const dim3 grid(n * c.kv_heads, (62 + longest) / 64 + 1, 2);
  if (c.head_dim == 128)
    hipLaunchKernelGGL(k_kv8_read<128>, grid, dim3(256), 0, s, c, seqs, k, ldk, v, ldv);
  else
    hipLaunchKernelGGL(k_kv8_read<64>, grid, dim3(256), 0, s, c, seqs, k, ldk, v, ldv);
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

// --- attention over the cache --------------------------------------------------------------------

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) void lds_void;
typedef short s16x8 __attribute__((ext_vector_type(8)));

// four int8 codes as fp16: each byte, its sign bit flipped, under 0x64 is 1024 + 128 + code; as
// bf16: the upper halves of the fp32 values (a code has 7 bits)
__device__ __forceinline__ u32x2 codes_f16(uint32_t w) {
  const uint32_t x = w ^ 0x80808080u;
  const f16x2 off = {(_Float16)-1152.f, (_Float16)-1152.f};
  const f16x2 a = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, x, 0x04010400u)) + off;
  const f16x2 b = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, x, 0x04030402u)) + off;
  return u32x2{__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b)};
}
__device__ __forceinline__ u32x2 codes_bf16(uint32_t w) {
  asm("" : "+v"(w));   // taken apart here: not byte by byte where it was loaded, in four registers
  float f[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) f[e] = (float)(int8_t)(w >> (8 * e));
  return u32x2{__builtin_amdgcn_perm(__float_as_uint(f[1]), __float_as_uint(f[0]), 0x07060302u),
               __builtin_amdgcn_perm(__float_as_uint(f[3]), __float_as_uint(f[2]), 0x07060302u)};
}
template <int BF>
__device__ __forceinline__ s16x8 codes8(uint32_t a, uint32_t b) {
  const u32x2 x = BF ? codes_bf16(a) : codes_f16(a), y = BF ? codes_bf16(b) : codes_f16(b);
  return __builtin_bit_cast(s16x8, u32x4{x[0], x[1], y[0], y[1]});
}
template <int BF>
__device__ __forceinline__ f32x4 mfma16(s16x8 a, s16x8 b, f32x4 c) {
  if constexpr (BF)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ float max_groups(float v) {   // over lanes l, l ^ 16, l ^ 32, l ^ 48
  float a = v, b = v;
  xswap16(a, b);
  a = b = fmaxf(a, b);
  xswap32(a, b);
  return fmaxf(a, b);
}
__device__ __forceinline__ float sum_groups(float v) {
  float a = v, b = v;
  xswap16(a, b);
  a = b = a + b;
  xswap32(a, b);
  return a + b;
}

// results of a cache of type BF (bf16's may well be past fp16's range)
__device__ __forceinline__ uint32_t pack_out(float a, float b, int bf, int obf) {
  return obf ? pack_bf16x2(a, b) : bf ? pack_f16x2(a, b) : pack_f16x2_in(a, b);
}

struct Kv8Args {
  Kv8 c;
  const SeqTile* tiles;
  int ntiles;
  const uint16_t* q;
  uint16_t* out;
  int64_t ldq, ldo;
  float scale;            // times log2(e)
  int heads, group;
  int tt, hh, chunks;     // tokens and heads a workgroup; workgroups a key/value head's group
  uint32_t magic;         // ceil(65536 / hh)
  int obf;
  // k_kv8_few: workgroups that share the sequences' blocks evenly, 0: one a sequence.
  // k_kv8_chunk: splits of each tile's blocks
  int splits;
  int least;              // blocks a workgroup takes at least, where they are shared or split
  // the sums, then their reference and weight: k_kv8_few: [workgroup and head][2][16 RT rows][dim],
  // [..][2][16 RT rows][2], and [tile and head][2], the first and last workgroup that had a part of it;
  // k_kv8_chunk: [split][row][head][dim], [split][row][head][2]
  float* part;
  int64_t rows;
  // the passes of attend_shared: pairs {row, sequence} of each prefix's rows, each tile's prefix's blocks, {first
  // sequence of its prefix or -1, blocks, first of its rows in ENTRY} of each sequence (Kv8Shared); the sums'
  // references and weights [split][row][head][2] beside part's [split][row][head][dim]; rows times heads of
  // them; the prefix pass's splits; for the join, of each of a sequence's tiles: its splits, all with the
  // prefix's, and the first of its rows there
  const int32_t *entry, *blocks;
  const int32x4* of;
  float* ml;
  int64_t n;
  int psplits, pleast;
  int32x4* notes;
};
enum { ALONE = 0, PREFIX = 1, OWN = 2 };   // all of a sequence's keys; a prefix's, for all its rows; a sequence's others

// the blocks of a tile's NB that split I of S takes: [*lo, *hi); the number of splits with any
__device__ __forceinline__ int kv8_split(int nb, int S, int least, int i, int* lo, int* hi) {
  const int per = max(least, (nb + S - 1) / S);
  *lo = min(nb, i * per);
  *hi = min(nb, (i + 1) * per);
  return (nb + per - 1) / per;
}

// Which blocks a prefix's pass takes of a sequence: of each of the pass's splits, from its first block on, those full
// before the step whose pages the sequence's table names as that of FIRST, the prefix's first sequence, does, up to
// the first that is another.  Found out on the device in every call, by a split's workgroups for its own blocks and by
// the sequence's for all of them.
struct Kv8Own {
  int first, nb, per;   // blocks below NB may be the pass's, in splits of PER
  const int* ends;      // where they part: of each split (64 at most), the first block that is not the pass's
};
// page P of block B, or -1 where it is taken
__device__ __forceinline__ int kv8_untaken(const Kv8Own& w, int b, int p) {
  return b < w.nb && b < w.ends[min(b, w.nb - 1) / w.per] ? -1 : p;
}
__device__ __forceinline__ Kv8Own kv8_own(const Kv8Args& A, const int32x4& of, int base) {
  if (of[0] < 0) return Kv8Own{0, 0, 1, nullptr};
  const int all = min(of[1], A.c.cols);
  return Kv8Own{of[0], min(all, base / 64), max(A.pleast, (all + A.psplits - 1) / A.psplits), nullptr};
}
// the first block of a sequence that is not taken (a wave finds it out)
__device__ __forceinline__ int kv8_own_from(const Kv8& c, int seq, const Kv8Own& w) {
  const int32_t *mine = c.table + (int64_t)seq * c.cols, *its = c.table + (int64_t)w.first * c.cols;
  int run = w.nb;
#pragma unroll 8
  for (int i = threadIdx.x & 63; i < w.nb; i += 64) run = min(run, mine[i] != its[i] ? i : run);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) run = min(run, __shfl_xor(run, o, 64));
  return __builtin_amdgcn_readfirstlane(run);
}
// the ends of a sequence whose table parts at block RUN, a split a lane, 64 blocks' entries at a time.  Found once and
// looked up: a walk back to the split's first block for each look-up costs the square of a long split (8 x 1 after 131008
// with scratch for one, a table that parts half-way: 1495 us, so 1095)
__device__ __forceinline__ void kv8_parted(const Kv8& c, int seq, Kv8Own& w, int run, int* ends) {
  const int32_t *mine = c.table + (int64_t)seq * c.cols, *its = c.table + (int64_t)w.first * c.cols;
  const int lane = threadIdx.x & 63, b0 = lane * w.per, b1 = b0 + w.per;
  int end = b1;
#pragma unroll 4
  for (int at = run & ~63; at < w.nb; at += 64) {
    const int i = min(at + lane, w.nb - 1), from = max(b0 - at, 0), to = min(b1 - at, 64);
    uint64_t differ = __ballot(mine[i] != its[i]);
    if (from < to) {
      differ = differ >> from << from & ~0ull >> (64 - to);
      if (differ) end = min(end, at + __builtin_ctzll(differ));
    }
  }
  ends[lane] = end;
  asm volatile("" ::: "memory");   // read by this wave alone, whose LDS accesses keep their order
  w.ends = ends;
}
// split I of a sequence's own blocks, FROM .. NB - 1 (taken ones among them are left out one by one): [*lo, *hi); the
// splits with any
__device__ __forceinline__ int kv8_own_split(const Kv8Args& A, int from, int nb, int i, int* lo, int* hi) {
  const int n = kv8_split(max(0, nb - from), A.splits, A.least, i, lo, hi);
  *lo += from;
  *hi += from;
  return n;
}
// for the join: tile TILE's own splits, and where its rows are in the prefixes' pass
__device__ __forceinline__ void kv8_note(const Kv8Args& A, const int32x4& of, int tile, int t0, int own) {
  int a, b;
  const int theirs = of[0] < 0 ? 0 : kv8_split(min(of[1], A.c.cols), A.psplits, A.pleast, 0, &a, &b);
  A.notes[tile] = int32x4{own, own + theirs, of[2] + t0, 0};
}
// For the N rows of a prefix's tile: where the blocks [B0, B1) that each sees end.  RUN is of the first row of each
// sequence in each 64 rows, which HEAD names.
template <int N>
struct PrefixRows {
  int seq[N], head[N], run[N];
};
// what a body keeps of that in LDS: nothing but in a prefix's pass
template <int MODE, int N>
struct RowsLds {
  __device__ __forceinline__ PrefixRows<N>* rows() { return nullptr; }
};
template <int N>
struct RowsLds<PREFIX, N> {
  PrefixRows<N> pfx;
  __device__ __forceinline__ PrefixRows<N>* rows() { return &pfx; }
};
template <int N>
struct RowsLds<OWN, N> {
  int ends[4][64];   // each wave's Kv8Own's
  __device__ __forceinline__ PrefixRows<N>* rows() { return nullptr; }
};
__device__ __forceinline__ void lds_barrier() {   // with loads from memory in flight
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0xC07F);   // lgkmcnt(0)
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}
// in two steps, the first blocks' loads asked for between them
template <int N>
__device__ __forceinline__ void prefix_rows(const Kv8Args& A, const SeqTile& T, int n, int b1, PrefixRows<N>& R) {
  const Kv8& c = A.c;
  const int tid = threadIdx.x, lane = tid & 63;
  if (tid < n) {
    const int seq = A.entry[2 * ((int64_t)T.row0 + T.t0 + tid) + 1], before = __shfl_up(seq, 1, 64);
    const uint64_t heads = __ballot(lane == 0 || seq != before);
    R.seq[tid] = seq;
    R.head[tid] = tid - lane + 63 - __builtin_clzll(heads & (~0ull >> (63 - lane)));
    R.run[tid] = min(b1, kv8_base(c, seq) / 64);
  }
}
template <int N>
__device__ __forceinline__ void prefix_ends(const Kv8Args& A, const SeqTile& T, int n, int b0, int b1, PrefixRows<N>& R) {
  const Kv8& c = A.c;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  lds_barrier();
  const int32_t* its = c.table + (int64_t)T.seq * c.cols;
  for (int t = 4 * wave; t < n; t += 16) {   // four rows at a time
    int at[4], end[4];
    const int32_t* mine[4];
    bool old = t % 64 > 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      at[j] = min(t + j, n - 1);
      end[j] = b1;
      mine[j] = c.table + (int64_t)R.seq[at[j]] * c.cols;
      old = old && R.head[at[j]] < t;
    }
    if (old) continue;
#pragma unroll 2
    for (int i = b0 + lane; i < b1; i += 64) {
      const int x = its[i];
#pragma unroll
      for (int j = 0; j < 4; ++j) end[j] = min(end[j], mine[j][i] != x ? i : b1);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (end[j] < b1) atomicMin(&R.run[at[j]], end[j]);
  }
  lds_barrier();
}

// a sequence's blocks after its new tokens
__device__ __forceinline__ int kv8_blocks(const Kv8& c, const SeqTile& t) {
  return (kv8_total(c, kv8_base(c, t.seq), t.len) + 63) >> 6;
}
// How k_kv8_few's workgroups share the blocks of all tiles, one after the other (a wave finds it out).
// SHARE consecutive ones each; or, where there is a workgroup for every tile and the longest is at most
// 16 blocks over an even share, a tile each: then nothing is left to be joined (64 x 1000..2000 tokens
// 42.1 us, shared 46.3; 4 x 1000..2000 12.9 shared, 23.8 a tile each).
struct Kv8Share {
  int all, share;   // share 0: a tile each
  int own;          // the blocks of the lane's tile of the first 64
};
__device__ __forceinline__ Kv8Share kv8_share(const Kv8Args& A) {
  const int lane = threadIdx.x & 63;
  int own = 0;
  if (lane < A.ntiles) own = kv8_blocks(A.c, A.tiles[lane]);
  int all = own, most = own;
#pragma unroll 4
  for (int t = lane + 64; t < A.ntiles; t += 64) {
    const int nb = kv8_blocks(A.c, A.tiles[t]);
    all += nb;
    most = max(most, nb);
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    all += __shfl_xor(all, o, 64);
    most = max(most, __shfl_xor(most, o, 64));
  }
  const bool each = A.ntiles <= A.splits && most <= all / A.splits + 16;
  return Kv8Share{__builtin_amdgcn_readfirstlane(all),
                  each ? 0 : __builtin_amdgcn_readfirstlane(max(A.least, (all + A.splits - 1) / A.splits)),
                  own};
}

// A.part's last piece
__device__ __forceinline__ uint32_t* kv8_parts(const Kv8Args& A, int per, int rt, int hd) {
  return (uint32_t*)(A.part + (int64_t)A.splits * per * 32 * rt * (hd + 2));
}

// Weights are 2^(score - reference), the reference at most MAX_SLACK under the row's largest score, and
// fp16 for codes of either type.  fp16 has none under 2^-24, which the many small ones beside one that
// takes nearly all would be: they are held 2^LIFT higher (up to 2^15), and what is lost is under 2^-32
// of a row's largest.  A key of no value with 0.999 of the weight before 8,100 others, fp16 rows: 2.3e-4
// off (relative L2), which is their rounding, and unlifted 1.4e-2 (k_kv8_chunk).  Sums of weights are kept
// as high, sums of weights and values are not (a block's scale takes the 2^-LIFT, exactly: it has 12
// significant bits or is a multiple of 2^-137).
#define MAX_SLACK 8.f
#define LIFT 7.f
#define LIFT2 128.f   // 2^LIFT

// --- few rows ------------------------------------------------------------------------------------
//
// The cache's bytes are the cost.  A key/value head's blocks of all sequences, one after the other, are
// shared evenly by the workgroups of that head, however long each sequence is: the loop reads at the
// memory's rate, and what a workgroup takes to begin (four loads that wait for each other, microseconds
// next to that many reads) and to end is paid once.  A workgroup whose share ends within a sequence
// leaves its sums to k_kv8_join_few.  Waves take a sequence's blocks in turn, each with sums of its own,
// which meet in LDS.  RT row tiles of 16 (rows: tokens times a group's heads).  Codes go from memory to
// the matrix operands in registers: a lane's 16 bytes of K are its own dims of a key, of V its own keys
// of a dim, so nothing is turned; eight waves a workgroup, or codes read through the caches, took longer.
//
// With the join (8 heads of 128, groups of 4): 64 x 1 token over 700..8191, bf16, 81.1 us and 1 over
// 131071, fp16, 52.5 us, 5.0 and 5.1 TB/s, a copy's rate; 4 over 270..333 9.3 us, which is latency.
//
// Grid: workgroups x kv_heads x chunks, the heads fastest.
// LDS at a multiple of 1024 bytes; in ALONE no more than the tail and the sums
template <int HD, int MODE>
struct FewSums {
  alignas(16) uint8_t tbuf[2][MODE == PREFIX ? 16 : 64 * HD * 2];   // the tail's K and V
  float obuf[4][16][HD + 4];
  float mbuf[4][16], lbuf[4][16], pbuf[MODE == PREFIX ? 1 : 64][17];
};
template <int HD, int RT, int MODE>
struct FewLds : FewSums<HD, MODE>, RowsLds<MODE, 16 * RT> {};
template <int BF, int HD, int RT, int MODE>
__device__ __forceinline__ void few_rows(const Kv8Args& A, FewLds<HD, RT, MODE>& lds, const int bx, const int by) {
  constexpr int WV = 4;                       // waves
  constexpr int NS = HD / 32, ND = HD / 16;   // k-steps of a score; 16-dim tiles of O
  constexpr int KL = HD / 64;                 // 16-byte loads a lane, key tile and block of K
  constexpr int ROWB = HD * 2, CH = HD / 8;
  auto &obuf = lds.obuf;
  auto &tbuf = lds.tbuf;
  auto &mbuf = lds.mbuf, &lbuf = lds.lbuf;
  auto &pbuf = lds.pbuf;
  PrefixRows<16 * RT>* const pfx = lds.rows();
  const Kv8& c = A.c;
  const int per = c.kv_heads * A.chunks;
  const int w = bx / per, hc = bx % per, kvh = hc % c.kv_heads, chunk = hc / c.kv_heads;
  const int tid = threadIdx.x, lane = tid & 63, col = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int heads = min(A.hh, A.group - chunk * A.hh);
  // key of row r of key tile t: 16 (r / 4) + 4 t + r % 4, so that a lane's scores of the four tiles
  // are 16 consecutive keys, the ones whose V codes it loads as 16 bytes
  const int key0 = 16 * (col >> 2) + (col & 3);

  // this workgroup's share: blocks [from, to) of the run of all tiles' blocks; tile I's begin at AT
  int i = w, at = 0, from = 0, to = 0x7FFFFFFF;
  const Kv8Share sh = MODE == ALONE && A.splits ? kv8_share(A) : Kv8Share{0, 0, 0};
  if (i >= A.ntiles && sh.share == 0) return;
  if (sh.share) {
    from = w * sh.share;
    to = min(sh.all, from + sh.share);
    if (from >= to) return;
    i = 0;
    for (int t0 = 0; t0 < A.ntiles; t0 += 64) {   // the tile in which FROM lies
      int nb = sh.own;
      if (t0 > 0) nb = t0 + lane < A.ntiles ? kv8_blocks(c, A.tiles[t0 + lane]) : 0;
      int upto = nb;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const int x = __shfl_up(upto, o, 64);
        upto += lane >= o ? x : 0;
      }
      const uint64_t past = __ballot(at + upto > from);
      if (past) {
        const int l = __builtin_ctzll(past);
        i = t0 + l;
        at += __builtin_amdgcn_readlane(upto, l) - __builtin_amdgcn_readlane(nb, l);
        break;
      }
      at += __builtin_amdgcn_readlane(upto, 63);
    }
  }

  // a tile's part of the share; of a prefix, a split of its blocks; of a sequence's own, a split of those
  struct Seg {
    SeqTile T;
    int base, total, nfull, nb, lo, hi, its;
    int ahead;   // OWN: a lane's first page
  };
  Kv8Own own;   // OWN: what the sequence's prefix takes
  auto page_at = [&](const Seg& s, int it) __attribute__((always_inline)) {
    const int b = s.lo + wave + WV * (it + lane);
    int p = b < min(s.hi, s.nfull) ? (int)kv8_page(c, s.T.seq, b) : -1;
    if (MODE == OWN && s.lo < own.nb) p = kv8_untaken(own, b, p);
    return p;
  };
  auto segment = [&](int i, int at) __attribute__((always_inline)) {
    Seg s;
    s.T = A.tiles[i];
    int32x4 of;
    if constexpr (MODE == OWN) of = A.of[s.T.seq];
    if constexpr (MODE == PREFIX) {
      s.base = s.total = min(A.blocks[i], c.cols) * 64;
    } else {
      s.base = kv8_base(c, s.T.seq);
      s.total = kv8_total(c, s.base, s.T.len);
    }
    s.nfull = s.total / 64;
    s.nb = (s.total + 63) / 64;
    if constexpr (MODE == ALONE) {
      s.lo = max(0, from - at);
      s.hi = min(s.nb, to - at);
    } else if constexpr (MODE == PREFIX) {
      kv8_split(s.nb, A.splits, A.least, by, &s.lo, &s.hi);
    } else {
      // its first pages are asked for as if all that may be taken were, while that is found out
      own = kv8_own(A, of, s.base);
      int n = kv8_own_split(A, own.nb, s.nb, by, &s.lo, &s.hi);
      const int b = s.lo + wave + WV * lane;
      s.ahead = b < min(s.hi, s.nfull) ? (int)kv8_page(c, s.T.seq, b) : -1;
      const int run = kv8_own_from(c, s.T.seq, own);
      if (run != own.nb) {
        kv8_parted(c, s.T.seq, own, run, lds.ends[wave]);
        n = kv8_own_split(A, run, s.nb, by, &s.lo, &s.hi);
        s.ahead = page_at(s, 0);
      }
      if (by == 0 && hc == 0 && tid == 0) kv8_note(A, of, i, s.T.t0, n);
    }
    s.its = (min(s.hi, s.nfull) - s.lo - wave + WV - 1) / WV;   // full blocks lo + wave + WV it of this wave
    return s;
  };
  int pages = 0;
  float kds = 0.f, vds = 0.f;
  // 64 of the wave's blocks' pages and scales, a lane each
  auto look = [&](const Seg& s, int it) __attribute__((always_inline)) {
    pages = MODE == OWN && it == 0 ? s.ahead : page_at(s, it);
    const int64_t p = max(pages, 0);
    const f32x2 d = *(const f32x2*)(c.scales + (p * c.kv_heads + kvh) * 2);
    kds = d[0];
    vds = d[1] * (1.f / LIFT2);
  };
  u32x4 kr[4][KL], vr[ND];
  // the codes are read once: past the caches
  auto load_k = [&](int page) __attribute__((always_inline)) {
    const int8_t* p = c.k + ((int64_t)max(page, 0) * c.kv_heads + kvh) * 64 * HD;
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int e = 0; e < KL; ++e)
        kr[t][e] = __builtin_nontemporal_load((const u32x4*)(p + (key0 + 4 * t) * HD + 16 * g + 64 * e));
  };
  auto load_v = [&](int page) __attribute__((always_inline)) {
    const int8_t* p = c.v + ((int64_t)max(page, 0) * c.kv_heads + kvh) * 64 * HD;
#pragma unroll
    for (int d = 0; d < ND; ++d) vr[d] = __builtin_nontemporal_load((const u32x4*)(p + (16 * d + col) * 64 + 16 * g));
  };
  auto has_tail = [&](const Seg& s) { return s.nfull < s.hi && s.nfull >= s.lo && (s.nfull - s.lo) % WV == wave; };
  // the first loads of a tile's part: its first block's codes, and its tail into LDS (the wave that
  // takes it): 16-byte chunk x of row r at x ^ (r % 16) (HD 64: x ^ (r / 2 % 8)) for K, at
  // x ^ 4 (r % 4) (HD 64: x ^ 4 (r / 2 % 2)) for V
  auto begin = [&](const Seg& s) __attribute__((always_inline)) {
    if (s.its > 0) {
      look(s, 0);
      load_k(__builtin_amdgcn_readlane(pages, 0));
      load_v(__builtin_amdgcn_readlane(pages, 0));
    }
    if (MODE != PREFIX && has_tail(s)) {
      const int64_t th = ((int64_t)s.T.seq * c.kv_heads + kvh) * 64 * HD;
#pragma unroll 1
      for (int e = 0; e < CH; ++e) {
        const int r = (64 / CH) * e + lane / CH, x = lane % CH;
        const int kx = x ^ (HD == 128 ? r & 15 : (r >> 1) & 7), vx = x ^ (HD == 128 ? 4 * (r & 3) : 4 * ((r >> 1) & 1));
        __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(c.tk + th + r * HD + 8 * kx),
                                         (lds_void*)(tbuf[0] + e * 1024), 16, 0, 0);
        __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(c.tv + th + r * HD + 8 * vx),
                                         (lds_void*)(tbuf[1] + e * 1024), 16, 0, 0);
      }
    }
  };

  Seg S = segment(i, at);
  if (MODE != ALONE && S.lo >= S.hi) return;
  if constexpr (MODE == PREFIX) prefix_rows(A, S.T, S.T.len, S.hi, *pfx);
  begin(S);
  if constexpr (MODE == PREFIX) prefix_ends(A, S.T, S.T.len, S.lo, S.hi, *pfx);
  for (;;) {
    const SeqTile T = S.T;
    const int live = T.len;
    int lim[RT], base = S.base;
    s16x8 qf[RT][NS];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      const int r = rt * 16 + col, tok = min((int)(r * A.magic >> 16), live - 1);
      const int head = min(r - (int)(r * A.magic >> 16) * A.hh, heads - 1);
      lim[rt] = MODE == PREFIX ? pfx->run[pfx->head[tok]] * 64 - 1 : min(S.base + tok, S.total - 1);
      if constexpr (MODE == PREFIX) {   // BASE: what every row sees all keys before
        int least = lim[rt] + 1;
#pragma unroll
        for (int o = 1; o < 16; o <<= 1) least = min(least, __shfl_xor(least, o, 64));
        base = min(base, __builtin_amdgcn_readfirstlane(least));
      }
      // dims of k-step s: 16 g + 8 (s % 2) + 64 (s / 2) .., as the 16 bytes of codes a lane loads
      const uint16_t* qr = A.q + (int64_t)(MODE == PREFIX ? A.entry[2 * ((int64_t)T.row0 + tok)] : T.row0 + tok) * A.ldq + (int64_t)(kvh * A.group + chunk * A.hh + head) * HD + 16 * g;
#pragma unroll
      for (int s = 0; s < NS; ++s) qf[rt][s] = *(const s16x8*)(qr + 8 * (s % 2) + 64 * (s / 2));
    }
    f32x4 o[RT][ND];
    float mrun[RT], lrun[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
#pragma unroll
      for (int d = 0; d < ND; ++d) o[rt][d] = f32x4{};
      mrun[rt] = -INFINITY;
      lrun[rt] = 0.f;
    }
    float s[RT][16];   // scores of keys 16 g + e of the block in hand
    uint32_t pk[RT][8], pl[RT][BF ? 8 : 1];   // weights; the tail's, in bf16, as two parts

    // from scores (log2 units, hidden ones -inf) to weights: the rows' references, sums and pk
    auto weights = [&](auto bf_c) __attribute__((always_inline)) {
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        float mx = s[rt][0];
#pragma unroll
        for (int e = 1; e < 16; ++e) mx = fmaxf(mx, s[rt][e]);
        mx = max_groups(mx);
        // a first reference (any above -inf), or one that has fallen behind
        if (__ballot(mx > mrun[rt] + (MAX_SLACK + LIFT))) {
          const float mn = mx > mrun[rt] + (MAX_SLACK + LIFT) ? mx - LIFT : mrun[rt];
          const float a = mn == mrun[rt] ? 1.f : __builtin_amdgcn_exp2f(mrun[rt] - mn);
          mrun[rt] = mn;
          lrun[rt] *= a;
#pragma unroll
          for (int d = 0; d < ND; ++d) o[rt][d] *= a;
        }
        constexpr bool WB = decltype(bf_c)::value;
        const float ref = mrun[rt] == -INFINITY ? 0.f : mrun[rt];
#pragma unroll
        for (int e = 0; e < 16; e += 2) {
          const float p0 = __builtin_amdgcn_exp2f(s[rt][e] - ref), p1 = __builtin_amdgcn_exp2f(s[rt][e + 1] - ref);
          pk[rt][e / 2] = WB ? pack_bf16x2(p0, p1) : pack_f16x2(p0, p1);
          if constexpr (WB)
            pl[rt][e / 2] = pack_bf16x2(p0 - bf16_lo(pk[rt][e / 2]), p1 - bf16_hi(pk[rt][e / 2]));
          lrun[rt] += p0;
          lrun[rt] += p1;
        }
      }
    };
    auto pfrag = [&](int rt, int u) {
      return __builtin_bit_cast(s16x8, u32x4{pk[rt][4 * u], pk[rt][4 * u + 1], pk[rt][4 * u + 2], pk[rt][4 * u + 3]});
    };

    // MORE: another block follows (true, false), or the lambda is to find out
    auto block = [&](auto more_c, int it) __attribute__((always_inline)) {
      const bool more = decltype(more_c)::value == 2 ? it + 1 < S.its : decltype(more_c)::value;
      const int page = __builtin_amdgcn_readlane(pages, it & 63);
      const float kd = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, kds), it & 63)) * A.scale;
      const float vd = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, vds), it & 63));
      if ((it & 63) == 63 && more) look(S, it + 1);
      const int next = more ? __builtin_amdgcn_readlane(pages, (it + 1) & 63) : 0;
      const int k0 = (S.lo + wave + WV * it) * 64;
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        f32x4 a[RT];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) a[rt] = f32x4{};
#pragma unroll
        for (int ks = 0; ks < NS; ++ks) {
          const u32x4 x = kr[t][ks / 2];
          const s16x8 kf = codes8<BF>(x[2 * (ks % 2)], x[2 * (ks % 2) + 1]);
#pragma unroll
          for (int rt = 0; rt < RT; ++rt) a[rt] = mfma16<BF>(kf, qf[rt][ks], a[rt]);
        }
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[rt][4 * t + e] = a[rt][e] * kd;
        if (RT == 1 || MODE == ALONE) __builtin_amdgcn_sched_barrier(0);
      }
      if (more) load_k(next);
      float vdl[RT];   // a row that sees nothing of the block takes nothing of its scale, which may be NaN
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        vdl[rt] = page >= 0 && k0 <= lim[rt] ? vd : 0.f;
        if (page < 0 || k0 + (MODE == PREFIX ? 64 : 63) > base) {
#pragma unroll
          for (int e = 0; e < 16; ++e)
            if (page < 0 || k0 + 16 * g + e > lim[rt]) s[rt][e] = -INFINITY;
        }
      }
      weights(std::integral_constant<int, 0>());
#pragma unroll
      for (int d = 0; d < ND; ++d) {
        const s16x8 v0 = codes8<0>(vr[d][0], vr[d][1]), v1 = codes8<0>(vr[d][2], vr[d][3]);
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
          const f32x4 a = mfma16<0>(v1, pfrag(rt, 1), mfma16<0>(v0, pfrag(rt, 0), f32x4{}));
#pragma unroll
          for (int e = 0; e < 4; ++e) o[rt][d][e] = __builtin_fmaf(a[e], vdl[rt], o[rt][d][e]);
        }
        if ((RT == 1 || MODE == ALONE) && d % 2) __builtin_amdgcn_sched_barrier(0);
      }
      if (more) load_v(next);
    };
    if constexpr (MODE == ALONE) {
      for (int it = 0; it < S.its; ++it) block(std::integral_constant<int, 2>(), it);
    } else {
      // the last one apart: where loads always follow, the wait for a block's K leaves its V's in flight
      for (int it = 0; it + 1 < S.its; ++it) block(std::integral_constant<int, 1>(), it);
      if (S.its > 0) block(std::integral_constant<int, 0>(), S.its - 1);
    }

    // the tail, in 16 bits, by the wave whose turn it is
    if (MODE != PREFIX && has_tail(S)) {
      const int left = S.total - S.nfull * 64, t0 = S.nfull * 64;
      int l = lane;
      asm volatile("" : "+v"(l));   // its addresses are made here, not kept through the loop above
      const int col = l & 15, g = l >> 4, key0 = 16 * (col >> 2) + (col & 3);
      asm volatile("" ::: "memory");
      __builtin_amdgcn_s_waitcnt(0x0F70);   // vmcnt(0): its rows are in LDS
      asm volatile("" ::: "memory");
      // V's rows past the last token may hold anything: zeros
      for (int e = left * CH + lane; e < 64 * CH; e += 64) *(u32x4*)(tbuf[1] + e * 16) = u32x4{};
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        f32x4 a[RT];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) a[rt] = f32x4{};
#pragma unroll
        for (int ks = 0; ks < NS; ++ks) {
          const int r = key0 + 4 * t, x = 2 * g + ks % 2 + 8 * (ks / 2);
          const s16x8 kf = *(const s16x8*)(tbuf[0] + r * ROWB + ((x ^ (HD == 128 ? r & 15 : (r >> 1) & 7)) << 4));
#pragma unroll
          for (int rt = 0; rt < RT; ++rt) a[rt] = mfma16<BF>(kf, qf[rt][ks], a[rt]);
        }
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            s[rt][4 * t + e] = t0 + 16 * g + 4 * t + e > lim[rt] ? -INFINITY : a[rt][e] * A.scale;
        __builtin_amdgcn_sched_barrier(0);
      }
      weights(std::integral_constant<int, BF>());
      asm volatile("" ::: "memory");
      __builtin_amdgcn_s_waitcnt(0xC07F);   // lgkmcnt(0): the zeros are in LDS
      asm volatile("" ::: "memory");
      typedef __attribute__((address_space(3))) s16x4 lds_s4;
      // lane l of 16 addresses key l / 4's dims 4 (l % 4) .. and gets dim l of the 4 keys
      auto v4 = [&](int key, int d) {
        const int r = key + (col >> 2), x = 2 * d + ((col & 3) >> 1);
        return __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (lds_s4*)(tbuf[1] + r * ROWB + ((x ^ (HD == 128 ? 4 * (r & 3) : 4 * ((r >> 1) & 1))) << 4) + 8 * (col & 1)));
      };
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        f32x4 a[ND];
        uint32_t bad = 0;
#pragma unroll
        for (int d = 0; d < ND; ++d) {
          s16x8 v[2];
#pragma unroll
          for (int u = 0; u < 2; ++u)
            v[u] = __builtin_shufflevector(v4(16 * g + 8 * u, d), v4(16 * g + 8 * u + 4, d), 0, 1, 2, 3, 4, 5, 6, 7);
          a[d] = mfma16<BF>(v[1], pfrag(rt, 1), mfma16<BF>(v[0], pfrag(rt, 0), f32x4{}));
          if constexpr (BF) {
#pragma unroll
            for (int u = 0; u < 2; ++u)
              a[d] = mfma16<BF>(v[u], __builtin_bit_cast(s16x8, u32x4{pl[rt][4 * u], pl[rt][4 * u + 1], pl[rt][4 * u + 2], pl[rt][4 * u + 3]}), a[d]);
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) bad |= (__float_as_uint(a[d][e]) & 0x7F800000u) == 0x7F800000u;
          __builtin_amdgcn_sched_barrier(0);
        }
        float down = 1.f / LIFT2;
        if (__ballot(bad)) {
          // an infinity or a NaN among the values, or a sum past fp32's largest: again, each row over the
          // keys it sees only, with weights that are not lifted
          down = 1.f;
#pragma unroll
          for (int e = 0; e < 16; ++e)
            pbuf[16 * g + e][col] = __builtin_amdgcn_exp2f(s[rt][e] - (mrun[rt] == -INFINITY ? 0.f : mrun[rt])) * (1.f / LIFT2);
          asm volatile("" ::: "memory");
          __builtin_amdgcn_s_waitcnt(0xC07F);
          asm volatile("" ::: "memory");
#pragma unroll
          for (int d = 0; d < ND; ++d) a[d] = f32x4{};
#pragma unroll 1
          for (int j = 0; j < left && t0 + j <= lim[rt]; ++j) {
            const float p = pbuf[j][col];
            const int z = HD == 128 ? 4 * (j & 3) : 4 * ((j >> 1) & 1);
#pragma unroll
            for (int d = 0; d < ND; ++d)
#pragma unroll
              for (int e = 0; e < 4; ++e)
                a[d][e] += p * ld16((const uint16_t*)(tbuf[1] + j * ROWB + (((2 * d + (g >> 1)) ^ z) << 4)) + 4 * (g & 1) + e, BF);
          }
        }
#pragma unroll
        for (int d = 0; d < ND; ++d) o[rt][d] += a[d] * down;
      }
    }

    int mt = tid;
    asm volatile("" : "+v"(mt));   // as above
    // the next tile's first loads, then this one's sums meet: 16 threads a row, all waves' sums of it
    const bool whole = MODE == ALONE && S.lo == 0 && S.hi == S.nb, more = sh.share && at + S.nb < to;
    const int nb = S.nb, lo = S.lo;
    if constexpr (MODE == ALONE) {
      if (A.splits && lo == 0 && tid == 0)
        *(u32x2*)(kv8_parts(A, per, RT, HD) + 2 * ((int64_t)i * per + hc)) =
            u32x2{(uint32_t)w, (uint32_t)(sh.share ? (at + nb - 1) / sh.share : w)};
    }
    if (more) {
      at += nb;
      ++i;
      S = segment(i, at);
      __syncthreads();   // the tail in LDS is done with
      begin(S);
    }
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      __syncthreads();
#pragma unroll
      for (int d = 0; d < ND; ++d) *(f32x4*)&obuf[wave][col][16 * d + 4 * g] = o[rt][d];
      const float l = sum_groups(lrun[rt]) * (1.f / LIFT2);
      if (g == 0) {
        mbuf[wave][col] = mrun[rt] + LIFT;
        lbuf[wave][col] = l;
      }
      __syncthreads();
      const int rr = mt >> 4, r = rt * 16 + rr, tok = (int)(r * A.magic >> 16), head = r - tok * A.hh;
      if (tok >= live || head >= heads) continue;
      float m = mbuf[0][rr];
#pragma unroll
      for (int k = 1; k < WV; ++k) m = fmaxf(m, mbuf[k][rr]);
      float wt[WV], sum = 0.f;
#pragma unroll
      for (int k = 0; k < WV; ++k) {
        wt[k] = mbuf[k][rr] == -INFINITY ? 0.f : mbuf[k][rr] == m ? 1.f : __builtin_amdgcn_exp2f(mbuf[k][rr] - m);
        sum += mbuf[k][rr] == -INFINITY ? lbuf[k][rr] : wt[k] * lbuf[k][rr];   // no reference: 0, or NaN
      }
      const float inv = !whole ? 1.f : sum == 0.f ? 0.f : 1.f / sum;
      constexpr int E = HD / 16;   // dims a thread
      const int d0 = (mt & 15) * E;
      float y[E];
#pragma unroll
      for (int e = 0; e < E; ++e) {
        y[e] = 0.f;
#pragma unroll
        for (int k = 0; k < WV; ++k)
          if (wt[k] > 0.f) y[e] = __builtin_fmaf(wt[k], obuf[k][rr][d0 + e], y[e]);
        y[e] *= inv;
      }
      if constexpr (MODE != ALONE) {
        const int64_t slot = by * A.n + (int64_t)(T.row0 + tok) * A.heads + kvh * A.group + chunk * A.hh + head;
#pragma unroll
        for (int e = 0; e < E; e += 4) *(f32x4*)(A.part + slot * HD + d0 + e) = f32x4{y[e], y[e + 1], y[e + 2], y[e + 3]};
        if ((mt & 15) == 0) *(f32x2*)(A.ml + slot * 2) = f32x2{m, sum};
      } else if (!whole) {   // the share's own first part (0) or the one begun in it (1)
        const int64_t slot = ((int64_t)bx * 2 + (lo == 0)) * 16 * RT + r;
#pragma unroll
        for (int e = 0; e < E; e += 4) *(f32x4*)(A.part + slot * HD + d0 + e) = f32x4{y[e], y[e + 1], y[e + 2], y[e + 3]};
        if ((mt & 15) == 0) *(f32x2*)(A.part + (int64_t)A.splits * per * 32 * RT * HD + slot * 2) = f32x2{m, sum};
      } else {
        uint32_t x[E / 2];
        if (A.obf) {
#pragma unroll
          for (int e = 0; e < E; e += 2) x[e / 2] = pack_bf16x2(y[e], y[e + 1]);
        } else {
#pragma unroll
          for (int e = 0; e < E; e += 2) x[e / 2] = pack_out(y[e], y[e + 1], BF, 0);
        }
        uint16_t* po = A.out + (int64_t)(T.row0 + tok) * A.ldo + (int64_t)(kvh * A.group + chunk * A.hh + head) * HD + d0;
        if constexpr (E == 8)
          *(u32x4*)po = u32x4{x[0], x[1], x[2], x[3]};
        else
          *(u32x2*)po = u32x2{x[0], x[1]};
      }
    }
    if (!more) return;
  }
}

template <int BF, int HD, int RT>
__global__ void __launch_bounds__(256, RT == 1 ? 2 : 1)
k_kv8_few(Kv8Args A) {
  __shared__ __align__(1024) FewLds<HD, RT, ALONE> lds;
  few_rows<BF, HD, RT, ALONE>(A, lds, blockIdx.x, 0);
}

// The sums of k_kv8_few's workgroups of each tile that more than one had a part of, in a fixed order:
// HD / 4 threads take a row's dims in each of SH shares of them, 1024 / HD / SH rows a workgroup
// (blockIdx.y: which).
template <int HD, int RT, int SH>
__global__ void __launch_bounds__(256)
k_kv8_join_few(Kv8Args A) {
  constexpr int TH = HD / 4, RW = 256 / TH / SH;   // threads a share; rows
  __shared__ __align__(16) float ys[256 / TH][HD];
  __shared__ float ss[256 / TH], ms[256 / TH];
  const int per = A.c.kv_heads * A.chunks;
  const int i = blockIdx.x / per, hc = blockIdx.x % per, kvh = hc % A.c.kv_heads, chunk = hc / A.c.kv_heads;
  const u32x2 parts = *(const u32x2*)(kv8_parts(A, per, RT, HD) + 2 * (int64_t)blockIdx.x);
  const SeqTile T = A.tiles[i];
  const int w0 = (int)parts[0], w1 = (int)parts[1];
  if (w0 == w1) return;
  const int tid = threadIdx.x, g = tid / TH, sh = g % SH, d = tid % TH * 4;
  const int r = min((int)blockIdx.y * RW + g / SH, 16 * RT - 1), tok = (int)(r * A.magic >> 16), head = r - tok * A.hh;
  const float* ml = A.part + (int64_t)A.splits * per * 32 * RT * HD;
  auto slot = [&](int w) { return (((int64_t)w * per + hc) * 2 + (w == w0)) * 16 * RT + r; };
  float m = -INFINITY;
  for (int w = w0 + sh; w <= w1; w += SH) m = fmaxf(m, ml[slot(w) * 2]);
  if (d == 0) ms[g] = m;
  __syncthreads();
#pragma unroll
  for (int k = 0; k < SH; ++k) m = fmaxf(m, ms[g - sh + k]);
  float sum = 0.f;
  f32x4 y = {};
#pragma unroll 4
  for (int w = w0 + sh; w <= w1; w += SH) {
    const f32x2 p = *(const f32x2*)(ml + slot(w) * 2);
    const f32x4 x = *(const f32x4*)(A.part + slot(w) * HD + d);
    const float f = p[0] == -INFINITY ? 0.f : p[0] == m ? 1.f : __builtin_amdgcn_exp2f(p[0] - m);
    sum += p[0] == -INFINITY ? p[1] : f * p[1];   // no reference: 0, or NaN
    if (f > 0.f) y += f * x;
  }
  *(f32x4*)&ys[g][d] = y;
  if (d == 0) ss[g] = sum;
  __syncthreads();
  if (sh || (int)blockIdx.y * RW + g / SH > r || tok >= T.len || head >= min(A.hh, A.group - chunk * A.hh)) return;
#pragma unroll
  for (int k = 1; k < SH; ++k) {
    y += *(const f32x4*)&ys[g + k][d];
    sum += ss[g + k];
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  uint16_t* po = A.out + (int64_t)(T.row0 + tok) * A.ldo + (int64_t)(kvh * A.group + chunk * A.hh + head) * HD + d;
  *(u32x2*)po = u32x2{pack_out(y[0] * inv, y[1] * inv, A.c.bf16, A.obf), pack_out(y[2] * inv, y[3] * inv, A.c.bf16, A.obf)};
}

// --- many rows: 128 a workgroup -------------------------------------------------------------------
//
// packed.hip's arrangement (32 rows a wave, S^T = K Q^T, O^T += V^T P^T, the S product of the next
// block interleaved with this one's exp2), with each block's codes made 16 bits on the way into LDS: a
// wave converts a quarter of a block for all four, 96 VALU instructions of about 300 a block, and the
// next codes are asked for a block ahead.  Codes are whole numbers: K's scale goes into the scores'
// factor, and a block's products of weights (fp16) and V codes meet the sums under V's scale.  (The scale
// in the weights' exponent saves those multiply-adds, but then a value 2^17 times the others, seen or
// not, takes the others' weights below fp16's least.)  Two workgroups a CU hide a part of the conversion only: 4 x 512 tokens
// over 2500..4001 (2 heads of 64, groups of 8, bf16) 63.0 us, 390 TFLOP/s; 1 x 76 over 1100 (8 heads of
// 128) 17.6 us, of which a third is its start (tile, length, page, scale and codes wait for each other),
// a third the join.
template <int BF>
__device__ __forceinline__ f32x16 mfma32(s16x8 a, s16x8 b, f32x16 c) {
  if constexpr (BF)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}

// One row by a whole wave, blocks [lo, hi), nothing that it does not see multiplied: for rows whose
// sums came out not finite (a hidden value of the tail that is not, times a weight of zero)
template <int BF, int HD, int MODE>
__device__ void kv8_row(const Kv8& c, int seq, const Kv8Own& own, int kvh, int lo, int hi, int total, int lim, const uint16_t* q,
                        float scale, float* m_, float* l_, float* o) {
  const int lane = threadIdx.x & 63;
  float m = -INFINITY, l = 0.f;
  for (int e = 0; e < HD / 64; ++e) o[e] = 0.f;
#pragma unroll 1
  for (int b = lo; b < hi && b * 64 <= lim; ++b) {
    const bool full = b * 64 + 64 <= total;
    int64_t page = full ? kv8_page(c, seq, b) : 0;
    if (MODE == OWN && b < own.nb) page = kv8_untaken(own, b, (int)page);
    if (page < 0) continue;
    const int64_t ph = (page * c.kv_heads + kvh), th = ((int64_t)seq * c.kv_heads + kvh) * 64 * HD;
    const float kd = full ? c.scales[ph * 2] : 1.f, vd = full ? c.scales[ph * 2 + 1] : 1.f;
    float s = -INFINITY;
    if (b * 64 + lane <= lim) {
      s = 0.f;
#pragma unroll 1
      for (int d = 0; d < HD; ++d)
        s += ld16(q + d, BF) * (full ? (float)c.k[ph * 64 * HD + lane * HD + d] : ld16(c.tk + th + lane * HD + d, BF));
      s *= scale * kd;
    }
    const float mn = fmaxf(m, wave_max(s)), mu = mn == -INFINITY ? 0.f : mn;
    const float a = exp2f(m - mu), p = exp2f(s - mu);
    l = l * a + wave_sum(p);
    m = mn;
    for (int e = 0; e < HD / 64; ++e) o[e] *= a;
#pragma unroll 1
    for (int j = 0; j < 64 && b * 64 + j <= lim; ++j) {
      const float pj = __shfl(p, j, 64);
      for (int e = 0; e < HD / 64; ++e) {
        const int d = e * 64 + lane;
        o[e] += pj * (full ? (float)c.v[ph * 64 * HD + d * 64 + j] * vd : ld16(c.tv + th + j * HD + d, BF));
      }
    }
  }
  *m_ = m;
  *l_ = l;
}

template <int HD>
struct ChunkStages {
  // K stage s at s STAGE: rows of keys, 16-byte chunk c at c ^ (key % 16) (HD 64: c ^ (key / 2 % 8)).
  // V^T stage s at (2 + s) STAGE: rows of dims of 128 bytes, chunk c at c ^ (dim / 2 % 8); a row's
  // keys in vt_pos's order, the one in which a lane's weights lie.  The tail's V is as in memory, rows
  // of keys, chunk c at c ^ 4 (key % 4) (HD 64: c ^ 4 (key / 2 % 2)), and is turned when it is read.
  alignas(16) uint8_t smem[4 * 64 * HD * 2];
};
template <int HD, int MODE>
struct ChunkLds : ChunkStages<HD>, RowsLds<MODE, 128> {};   // at a multiple of 1024 bytes
template <int BF, int HD, int MODE, int KG>
__device__ __forceinline__ void chunk_rows(const Kv8Args& A, ChunkLds<HD, MODE>& lds, const int bx, const int by) {
  constexpr int ROWB = HD * 2, STAGE = 64 * ROWB;   // bytes of a key's row; of a block's K or V^T
  constexpr int NS = HD / 16, ND = HD / 32;
  // a wave's halves of a block of keys: both, or, in tiles of 64 rows, one (waves 2 and 3 take the second's)
  constexpr int NH = 2 / KG, NU = 2 * NH;
  constexpr int CI = HD / 64;                       // 16-byte loads of codes a thread and block
  uint8_t* const smem = lds.smem;
  PrefixRows<128>* const pfx = lds.rows();
  const Kv8& c = A.c;
  const int per = c.kv_heads * A.chunks;
  const SeqTile T = A.tiles[bx / per];
  const int hc = bx % per, kvh = hc % c.kv_heads, chunk = hc / c.kv_heads;
  const int tid = threadIdx.x, lane = tid & 63, hi = lane >> 5, lo = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int base = MODE == PREFIX ? min(A.blocks[bx / per], c.cols) * 64 : kv8_base(c, T.seq);
  const int total = MODE == PREFIX ? base : kv8_total(c, base, T.len), nfull = total / 64;
  const int live = min(A.tt, T.len - T.t0), heads = min(A.hh, A.group - chunk * A.hh);
  int b0, b1, active;   // the blocks taken here; the splits
  Kv8Own own{};         // OWN: what the sequence's prefix takes
  if constexpr (MODE == PREFIX) {
    active = kv8_split(nfull, A.splits, A.least, by, &b0, &b1);
  } else if constexpr (MODE == OWN) {
    const int32x4 of = A.of[T.seq];
    own = kv8_own(A, of, base);
    const int run = kv8_own_from(c, T.seq, own);
    if (run != own.nb) kv8_parted(c, T.seq, own, run, lds.ends[wave]);
    active = kv8_own_split(A, run, (min(base + T.t0 + live, total) + 63) / 64, by, &b0, &b1);
    if (by == 0 && hc == 0 && tid == 0) kv8_note(A, of, bx / per, T.t0, active);
  } else {
    active = max(1, kv8_split((min(base + T.t0 + live, total) + 63) / 64, A.splits, A.least, by, &b0, &b1));
  }
  if (by >= active) return;
  const int rw = wave % (4 / KG), kg = wave / (4 / KG);
  const int row = rw * 32 + lo, tok = (int)(row * A.magic >> 16), head = row - tok * A.hh;
  const bool mine = tok < live && head < heads;
  const int ctok = min(tok, live - 1), chead = kvh * A.group + chunk * A.hh + min(head, heads - 1);
  // waves without a row do their part of each block's way into LDS only
  const bool idle = MODE != ALONE && (int)(rw * 32 * A.magic >> 16) >= live;
  int lim, minlim;
  s16x8 qf[NS];   // Q^T as the B operand: this lane's row, dims 16s + 8 hi ..
  auto rows_here = [&]() __attribute__((always_inline)) {
    const int64_t qrow = MODE == PREFIX ? A.entry[2 * ((int64_t)T.row0 + T.t0 + ctok)] : T.row0 + T.t0 + ctok;
    const uint16_t* qr = A.q + qrow * A.ldq + (int64_t)chead * HD;
#pragma unroll
    for (int s = 0; s < NS; ++s) qf[s] = *(const s16x8*)(qr + 16 * s + 8 * hi);
    if constexpr (MODE == PREFIX) {
      prefix_ends(A, T, live, b0, b1, *pfx);
      lim = minlim = pfx->run[pfx->head[ctok]] * 64 - 1;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) minlim = min(minlim, __shfl_xor(minlim, o, 64));
      minlim = __builtin_amdgcn_readfirstlane(minlim);
    } else {
      lim = min(base + T.t0 + ctok, total - 1);
      minlim = min(base + T.t0 + min((int)(rw * 32 * A.magic >> 16), live - 1), total - 1);
    }
  };
  if constexpr (MODE != PREFIX) rows_here();

  // 64 blocks' pages and scales from block B on, a lane each
  int pages = 0;
  float kds = 1.f, vds = 1.f;
  auto look = [&](int b) __attribute__((always_inline)) {
    int64_t p = b + lane < min(b1, nfull) ? kv8_page(c, T.seq, b + lane) : -1;
    if (MODE == OWN && b < own.nb) p = kv8_untaken(own, b + lane, (int)p);
    pages = (int)p;
    p = p < 0 ? 0 : p;
    const f32x2 d = *(const f32x2*)(c.scales + (p * c.kv_heads + kvh) * 2);
    kds = b + lane < nfull ? d[0] : 1.f;
    vds = b + lane < nfull ? d[1] : 1.f;
  };
  // a block's page and scales: the looked-up 64 are replaced once its last is asked for by FETCH, three
  // blocks ahead of its use, so each block's facts ride along
  struct Facts {
    int page;
    float kd, vd;
  };
  auto facts = [&](int b) __attribute__((always_inline)) {
    const int i = (b - b0) & 63;
    if (i == 0) look(b);
    return Facts{__builtin_amdgcn_readlane(pages, i), __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, kds), i)),
                 __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, vds), i))};
  };
  struct Codes {
    u32x4 w[CI];
  };
  auto fetch = [&](const int8_t* all, int page) __attribute__((always_inline)) {
    const int8_t* p = all + ((int64_t)max(page, 0) * c.kv_heads + kvh) * 64 * HD;
    Codes x;
#pragma unroll
    for (int i = 0; i < CI; ++i) x.w[i] = *(const u32x4*)(p + (tid + 256 * i) * 16);
    return x;
  };
  const int64_t th = ((int64_t)T.seq * c.kv_heads + kvh) * 64 * HD;
  // the tail's 64 rows by DMA; those past its last token hold anything
  auto tail = [&](const uint16_t* all, uint8_t* p, auto swizzle) __attribute__((always_inline)) {
#pragma unroll 1
    for (int e = wave; e < 64 * ROWB / 1024; e += 4) {
      const int r = e * (1024 / ROWB) + lane / (HD / 8), x = lane % (HD / 8) ^ swizzle(r);
      __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(all + th + r * HD + 8 * x),
                                       (lds_void*)(p + e * 1024), 16, 0, 0);
    }
  };
  // block B's K, the codes X or the tail's rows, into a stage
  auto fill_k = [&](int b, int st, const Codes& x) __attribute__((always_inline)) {
    uint8_t* p = smem + st * STAGE;
    if (b < nfull) {
#pragma unroll
      for (int i = 0; i < CI; ++i) {
        const int ci = tid + 256 * i, key = ci / (HD / 16), c2 = ci % (HD / 16) * 2;
        const int z = HD == 128 ? key & 15 : (key >> 1) & 7;
        *(s16x8*)(p + key * ROWB + ((c2 ^ z) << 4)) = codes8<BF>(x.w[i][0], x.w[i][1]);
        *(s16x8*)(p + key * ROWB + (((c2 + 1) ^ z) << 4)) = codes8<BF>(x.w[i][2], x.w[i][3]);
      }
    } else {
      tail(c.tk, p, [&](int r) { return HD == 128 ? r & 15 : (r >> 1) & 7; });
    }
  };
  auto fill_v = [&](int b, int st, const Codes& x) __attribute__((always_inline)) {
    uint8_t* p = smem + (2 + st) * STAGE;
    if (b < nfull) {
#pragma unroll
      for (int i = 0; i < CI; ++i) {
        const int ci = tid + 256 * i, dim = ci >> 2, c2 = 2 * (ci & 3), z = (dim >> 1) & 7;
        *(s16x8*)(p + dim * 128 + ((c2 ^ z) << 4)) = codes8<0>(x.w[i][0], x.w[i][2]);
        *(s16x8*)(p + dim * 128 + (((c2 + 1) ^ z) << 4)) = codes8<0>(x.w[i][1], x.w[i][3]);
      }
    } else {
      tail(c.tv, p, [&](int r) { return HD == 128 ? 4 * (r & 3) : 4 * ((r >> 1) & 1); });
    }
  };
  int kofs[NS], vofs[NU];   // K row lo (of the wave's half), chunk 2s + hi; V^T row lo, chunk 2u + hi
#pragma unroll
  for (int s = 0; s < NS; ++s) kofs[s] = (32 * kg + lo) * ROWB + (((2 * s + hi) ^ (HD == 128 ? lo & 15 : (lo >> 1) & 7)) << 4);
#pragma unroll
  for (int u = 0; u < NU; ++u) vofs[u] = 2 * STAGE + lo * 128 + (((2 * (u + 2 * kg) + hi) ^ ((lo >> 1) & 7)) << 4);
  auto kfrag = [&](int i) { return *(const s16x8*)(smem + kofs[i / NH] + (i % NH) * 32 * ROWB); };
  auto vfrag = [&](auto tail_c, int u, int d) __attribute__((always_inline)) {
    if constexpr (decltype(tail_c)::value) {
      typedef __attribute__((address_space(3))) s16x4 lds_s4;
      const int r = 4 * hi + ((lane & 15) >> 2), x = 4 * d + 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
      uint8_t* p = smem + ((vofs[0] & ~(STAGE - 1)) + (16 * (u + 2 * kg) + r) * ROWB +
                           ((x ^ (HD == 128 ? 4 * (r & 3) : 4 * ((r >> 1) & 1))) << 4) + 8 * (lane & 1));
      return __builtin_shufflevector(__builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)p),
                                     __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(p + 8 * ROWB)), 0, 1, 2, 3, 4, 5, 6, 7);
    } else {
      return *(const s16x8*)(smem + vofs[u] + d * 32 * 128);
    }
  };

  f32x16 o[ND], sc[NH];
  float mrun = 0.f, lrun = 0.f;
  bool set = false;          // the row has a reference
#pragma unroll
  for (int d = 0; d < ND; ++d) o[d] = f32x16{};
  auto barrier = [&](bool dma) __attribute__((always_inline)) {   // DMA: with the tail's rows asked for before it
    asm volatile("" ::: "memory");
    if (dma) __builtin_amdgcn_s_waitcnt(0x0070);   // vmcnt(0) lgkmcnt(0)
    __builtin_amdgcn_s_waitcnt(0xC07F);            // lgkmcnt(0)
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };

  // Block B of facts F: its softmax, the S product of block b+1 interleaved with its exp2, O^T += V^T P^T
  auto step = [&](auto last_c, auto tail_c, int b, const Facts& F) __attribute__((always_inline)) {
    constexpr bool LAST = decltype(last_c)::value, TAIL = decltype(tail_c)::value;
    constexpr int WB = TAIL && BF;   // weights: fp16, or with values in bf16 two bf16 parts
    constexpr float UP = WB ? 0.f : LIFT;
    const int k0 = b * 64;
    const float factor = F.kd * A.scale;
    const bool gone = F.page < 0 && b < nfull;
#pragma unroll
    for (int h = 0; h < NH; ++h)
#pragma unroll
      for (int r = 0; r < 16; ++r) sc[h][r] = __builtin_fmaf(sc[h][r], factor, UP - mrun);
    if (gone || k0 + 63 > minlim) {
#pragma unroll
      for (int h = 0; h < NH; ++h)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int key = k0 + 32 * (h + kg) + 8 * (r >> 2) + 4 * hi + (r & 3);
          if (gone || key > lim) sc[h][r] = -INFINITY;
        }
    }
    float m4[2 * NH];
#pragma unroll
    for (int q = 0; q < 2 * NH; ++q) {
      const int h = q / 2, r0 = (q % 2) * 8;
      float m = max3(sc[h][r0], sc[h][r0 + 1], sc[h][r0 + 2]);
      m = max3(m, sc[h][r0 + 3], sc[h][r0 + 4]);
      m = max3(m, sc[h][r0 + 5], sc[h][r0 + 6]);
      m4[q] = fmaxf(m, sc[h][r0 + 7]);
    }
    float ma = fmaxf(m4[0], m4[1]);
    if constexpr (NH == 2) ma = fmaxf(ma, fmaxf(m4[2], m4[3]));
    float mb = ma;
    xswap32(ma, mb);
    const float mx = fmaxf(ma, mb);
    const bool move = set ? mx > MAX_SLACK + UP : mx > -INFINITY;
    if (__ballot(move)) {
      const float shift = move ? mx - UP : 0.f;
      const float alpha = set ? __builtin_amdgcn_exp2f(-shift) : 1.f;   // without a reference the sums are 0, or NaN
      lrun *= alpha;
#pragma unroll
      for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[d][r] *= alpha;
      mrun += shift;
#pragma unroll
      for (int h = 0; h < NH; ++h)
#pragma unroll
        for (int r = 0; r < 16; ++r) sc[h][r] -= shift;
      set = set || move;
    }
    constexpr int KD = 3, NI = NH * NS, PS = 8 / NS;
    f32x16 sn[NH];
    uint32_t pk[8 * NH], pl[WB ? 8 * NH : 1];
    float ls[2] = {lrun, 0.f};
    s16x8 kq[KD], vq[KD];
    if constexpr (!LAST) {
#pragma unroll
      for (int h = 0; h < NH; ++h) sn[h] = f32x16{};
#pragma unroll
      for (int i = 0; i < KD; ++i) kq[i] = kfrag(i);
    }
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      if constexpr (!LAST) {
        s16x8 kn = {};
        if (i + KD < NI) kn = kfrag(i + KD);
        sn[i % NH] = mfma32<BF>(kq[0], qf[i / NH], sn[i % NH]);
#pragma unroll
        for (int d = 0; d + 1 < KD; ++d) kq[d] = kq[d + 1];
        kq[KD - 1] = kn;
      }
      if (i >= NI - KD) vq[i - (NI - KD)] = vfrag(tail_c, (i - (NI - KD)) % NU, (i - (NI - KD)) / NU);
#pragma unroll
      for (int z = 0; z < PS; ++z) {
        const int pi = PS * i + z, h = pi / 8, r = 2 * (pi % 8);
        const float p0 = __builtin_amdgcn_exp2f(sc[h][r]), p1 = __builtin_amdgcn_exp2f(sc[h][r + 1]);
        pk[pi] = WB ? pack_bf16x2(p0, p1) : pack_f16x2(p0, p1);
        if constexpr (WB) pl[pi] = pack_bf16x2(p0 - bf16_lo(pk[pi]), p1 - bf16_hi(pk[pi]));
        ls[0] += WB ? p0 * LIFT2 : p0;
        ls[1] += WB ? p1 * LIFT2 : p1;
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    lrun = ls[0] + ls[1];
    // a block's products of codes, then its scale; a row that sees nothing of it takes nothing of the scale,
    // which may be NaN
    const float vd = gone || k0 > lim ? 0.f : (TAIL ? 1.f : F.vd) * (1.f / LIFT2);
    f32x16 t[2];
#pragma unroll
    for (int j = 0; j < NU * ND; ++j) {
      s16x8 vn = {};
      if (j + KD < NU * ND) vn = vfrag(tail_c, (j + KD) % NU, (j + KD) / NU);
      const int u = j % NU, d = j / NU;
      const s16x8 pb = __builtin_bit_cast(s16x8, u32x4{pk[4 * u], pk[4 * u + 1], pk[4 * u + 2], pk[4 * u + 3]});
      if constexpr (WB) {
        o[d] = mfma32<1>(vq[0], pb, o[d]);
        o[d] = mfma32<1>(vq[0], __builtin_bit_cast(s16x8, u32x4{pl[4 * u], pl[4 * u + 1], pl[4 * u + 2], pl[4 * u + 3]}), o[d]);
      } else {
        t[d % 2] = mfma32<0>(vq[0], pb, u == 0 ? f32x16{} : t[d % 2]);
        if (d > 0) {
#pragma unroll
          for (int r = 16 / NU * u; r < 16 / NU * (u + 1); ++r) o[d - 1][r] = __builtin_fmaf(t[(d - 1) % 2][r], vd, o[d - 1][r]);
        }
      }
#pragma unroll
      for (int d = 0; d + 1 < KD; ++d) vq[d] = vq[d + 1];
      vq[KD - 1] = vn;
      __builtin_amdgcn_sched_barrier(0);
    }
    if constexpr (!WB) {
#pragma unroll
      for (int r = 0; r < 16; ++r) o[ND - 1][r] = __builtin_fmaf(t[(ND - 1) % 2][r], vd, o[ND - 1][r]);
    }
    if constexpr (!LAST) {
#pragma unroll
      for (int h = 0; h < NH; ++h) sc[h] = sn[h];
    }
    asm volatile("" : "+v"(lrun));
  };

  // block b's K is filled two steps ahead of its softmax, its V one; codes are asked for one step
  // before they are filled
  if constexpr (MODE == PREFIX) prefix_rows(A, T, live, b1, *pfx);
  Facts F0 = facts(b0), F1 = F0, F2 = F0;
  Codes kc = fetch(c.k, F0.page), vc = fetch(c.v, F0.page), kn = kc;
  if (b0 + 1 < b1) {
    F1 = facts(b0 + 1);
    kn = fetch(c.k, F1.page);
  }
  if constexpr (MODE == PREFIX) rows_here();   // while the first codes are on their way
  fill_k(b0, 0, kc);
  barrier(b0 == nfull);
#pragma unroll
  for (int h = 0; h < NH; ++h) sc[h] = f32x16{};
  if (!idle) {
#pragma unroll
    for (int i = 0; i < NH * NS; ++i) {
      sc[i % NH] = mfma32<BF>(kfrag(i), qf[i / NH], sc[i % NH]);
      if (i % 4 == 3) __builtin_amdgcn_sched_barrier(0);
    }
  }
  fill_v(b0, 0, vc);
  if (b0 + 1 < b1) {
    vc = fetch(c.v, F1.page);
    if (b0 + 2 < b1) {
      F2 = facts(b0 + 2);
      kc = fetch(c.k, F2.page);
    }
    fill_k(b0 + 1, 1, kn);
  }
#pragma unroll
  for (int s = 0; s < NS; ++s) kofs[s] ^= STAGE;
  int b = b0;
  for (; b + 1 < b1; ++b) {
    // K of block b+1 and V of block b are filled; K of b and V of b-1 are done with
    barrier(b + 1 == nfull);
    fill_v(b + 1, (b + 1 - b0) & 1, vc);
    if (b + 2 < b1) {
      fill_k(b + 2, (b - b0) & 1, kc);
      vc = fetch(c.v, F2.page);
    }
    Facts F3 = F2;
    if (b + 3 < b1) {
      F3 = facts(b + 3);
      kc = fetch(c.k, F3.page);
    }
    if (!idle) step(std::integral_constant<bool, false>(), std::integral_constant<bool, false>(), b, F0);
    F0 = F1;
    F1 = F2;
    F2 = F3;
#pragma unroll
    for (int s = 0; s < NS; ++s) kofs[s] ^= STAGE;
#pragma unroll
    for (int u = 0; u < NU; ++u) vofs[u] ^= STAGE;
  }
  barrier(b == nfull);
  if (MODE == PREFIX || b < nfull) {
    if (!idle) step(std::integral_constant<bool, true>(), std::integral_constant<bool, false>(), b, F0);
  } else {
    uint8_t* p = smem + (2 + ((b - b0) & 1)) * STAGE;   // V's rows past the last token: zeros
    for (int e = (total - b * 64) * (HD / 8) + tid; e < 64 * HD / 8; e += 256) *(u32x4*)(p + e * 16) = u32x4{};
    barrier(false);
    if (!idle) step(std::integral_constant<bool, true>(), std::integral_constant<bool, true>(), b, F0);
  }
  if constexpr (KG == 2) {   // the second half's sums to the first's wave
    constexpr int N = 16 * ND + 2;
    float* buf = (float*)smem + rw * N * 64 + lane;
    barrier(false);   // all reads of the blocks are done
    if (kg && !idle) {
#pragma unroll
      for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) buf[(16 * d + r) * 64] = o[d][r];
      buf[16 * ND * 64] = set ? mrun : -INFINITY;
      buf[(16 * ND + 1) * 64] = lrun;
    }
    barrier(false);
    if (kg || idle) return;
    const float m = buf[16 * ND * 64], l = buf[(16 * ND + 1) * 64];
    if (m == -INFINITY) {
      lrun += l;   // 0, or NaN
    } else {
      const float mn = set ? fmaxf(mrun, m) : m;
      const float a = set ? __builtin_amdgcn_exp2f(mrun - mn) : 1.f, w = __builtin_amdgcn_exp2f(m - mn);
      lrun = lrun * a + l * w;
#pragma unroll
      for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[d][r] = __builtin_fmaf(w, buf[(16 * d + r) * 64], o[d][r] * a);
      mrun = mn;
      set = true;
    }
  }
  if (idle) return;

  float la = lrun, lb = lrun;
  xswap32(la, lb);
  const bool parts = MODE != ALONE || active > 1;
  const float sum = (la + lb) * (1.f / LIFT2), mul = parts ? 1.f : sum == 0.f ? 0.f : 1.f / sum;
  float zero[4] = {sum * 0.f};
  const int64_t rowhead = (int64_t)(T.row0 + T.t0 + tok) * A.heads + chead, n = MODE == ALONE ? A.rows * A.heads : A.n;
  float* ml = MODE == ALONE ? A.part + A.splits * n * HD : A.ml;
  auto leave = [&](auto obf) __attribute__((always_inline)) {
    uint16_t* po = A.out + (int64_t)(T.row0 + T.t0 + tok) * A.ldo + (int64_t)chead * HD + 4 * hi;
    float* pp = A.part + ((int64_t)by * n + rowhead) * HD + 4 * hi;
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int r4 = 0; r4 < 4; ++r4) {
        float y[4];
#pragma unroll
        for (int z = 0; z < 4; ++z) {
          zero[z] = __builtin_fmaf(o[d][4 * r4 + z], 0.f, zero[z]);
          y[z] = o[d][4 * r4 + z] * mul;
        }
        if (!mine) continue;
        if constexpr (decltype(obf)::value == 2)
          *(f32x4*)(pp + 32 * d + 8 * r4) = f32x4{y[0], y[1], y[2], y[3]};
        else if constexpr (decltype(obf)::value == 1)
          *(u32x2*)(po + 32 * d + 8 * r4) = u32x2{pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3])};
        else
          *(u32x2*)(po + 32 * d + 8 * r4) = u32x2{pack_out(y[0], y[1], BF, 0), pack_out(y[2], y[3], BF, 0)};
      }
  };
  if (parts) {
    leave(std::integral_constant<int, 2>());
    if (mine && hi == 0) *(f32x2*)(ml + ((int64_t)by * n + rowhead) * 2) = f32x2{set ? mrun : -INFINITY, sum};
  } else if (A.obf) {
    leave(std::integral_constant<int, 1>());
  } else {
    leave(std::integral_constant<int, 0>());
  }
  const uint64_t redo = __ballot(!(zero[0] + zero[1] + zero[2] + zero[3] == 0.f) && mine);
#pragma unroll 1
  for (uint32_t rows = (uint32_t)(redo | redo >> 32); rows; rows &= rows - 1) {
    const int r = rw * 32 + __builtin_ctz(rows), rt = (int)(r * A.magic >> 16);
    const int64_t rh = kvh * A.group + chunk * A.hh + r - rt * A.hh, at = T.row0 + T.t0 + rt;
    float m, l, y[HD / 64];
    const int64_t qrow = MODE == PREFIX ? A.entry[2 * at] : at;
    const int sees = MODE == PREFIX ? pfx->run[pfx->head[rt]] * 64 - 1 : min(base + T.t0 + rt, total - 1);
    kv8_row<BF, HD, MODE>(c, T.seq, own, kvh, b0, b1, total, sees, A.q + qrow * A.ldq + rh * HD, A.scale, &m, &l, y);
    const int64_t slot = (int64_t)by * n + at * A.heads + rh;
    for (int z = 0; z < HD / 64; ++z) {
      const float w = parts ? y[z] : l == 0.f ? 0.f : y[z] / l;
      if (parts)
        A.part[slot * HD + z * 64 + lane] = w;
      else
        A.out[at * A.ldo + rh * HD + z * 64 + lane] = (uint16_t)pack_out(w, 0.f, BF, A.obf);
    }
    if (parts && lane == 0) *(f32x2*)(ml + slot * 2) = f32x2{m, l};
  }
}

template <int BF, int HD>
__global__ void __launch_bounds__(256, 2)
k_kv8_chunk(Kv8Args A) {
  __shared__ __align__(1024) ChunkLds<HD, ALONE> lds;
  chunk_rows<BF, HD, ALONE, 1>(A, lds, blockIdx.x, blockIdx.y);
}

// The splits' sums of each row and head, in a fixed order: HD / 4 threads take one's dims in each of SH
// shares of the splits (all 256 threads of a workgroup for few rows and many splits, SH 1 for many rows),
// then the shares are summed.  Rows whose keys were not split are done.
template <int HD, int SH>
__global__ void __launch_bounds__(256)
k_kv8_join(Kv8Args A) {
  constexpr int TH = HD / 4, RW = 256 / TH / SH;   // threads a row and share; rows a workgroup
  __shared__ __align__(16) float ys[256 / TH][HD];
  __shared__ float ss[256 / TH], ms[256 / TH];
  const Kv8& c = A.c;
  const SeqTile T = A.tiles[blockIdx.x];
  const int base = kv8_base(c, T.seq), total = kv8_total(c, base, T.len);
  const int live = min(A.tt, T.len - T.t0);
  int lo, hi;
  const int active = kv8_split((min(base + T.t0 + live, total) + 63) / 64, A.splits, A.least, 0, &lo, &hi);
  if (active < 2 || (int)blockIdx.y * RW >= live * A.heads) return;
  const int tid = threadIdx.x, sh = tid / TH % SH, r = tid / TH / SH, d = tid % TH * 4;
  const int i = min((int)blockIdx.y * RW + r, live * A.heads - 1);
  const int64_t rowhead = (int64_t)(T.row0 + T.t0) * A.heads + i, n = A.rows * A.heads;
  const float* ml = A.part + A.splits * n * HD + rowhead * 2;
  float m = -INFINITY;
  for (int z = sh; z < active; z += SH) m = fmaxf(m, ml[z * n * 2]);
  if constexpr (SH > 1) {
    if (d == 0) ms[tid / TH] = m;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < SH; ++k) m = fmaxf(m, ms[r * SH + k]);
  }
  float sum = 0.f;
  f32x4 y = {};
#pragma unroll 4
  for (int z = sh; z < active; z += SH) {
    const f32x2 p = *(const f32x2*)(ml + z * n * 2);
    const f32x4 x = *(const f32x4*)(A.part + (z * n + rowhead) * HD + d);
    const float w = p[0] == -INFINITY ? 0.f : p[0] == m ? 1.f : __builtin_amdgcn_exp2f(p[0] - m);
    sum += p[0] == -INFINITY ? p[1] : w * p[1];   // no reference: 0, or NaN
    if (w > 0.f) y += w * x;
  }
  if constexpr (SH > 1) {
    *(f32x4*)&ys[tid / TH][d] = y;
    if (d == 0) ss[tid / TH] = sum;
    __syncthreads();
    if (sh) return;
#pragma unroll
    for (int k = 1; k < SH; ++k) {
      y += *(const f32x4*)&ys[r * SH + k][d];
      sum += ss[r * SH + k];
    }
  }
  if ((int)blockIdx.y * RW + r >= live * A.heads) return;
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  uint16_t* po = A.out + (rowhead / A.heads) * A.ldo + (rowhead % A.heads) * HD + d;
  *(u32x2*)po = u32x2{pack_out(y[0] * inv, y[1] * inv, A.c.bf16, A.obf), pack_out(y[2] * inv, y[3] * inv, A.c.bf16, A.obf)};
}

namespace {

struct Kv8Way {
  int rt;                  // row tiles of 16 a workgroup (1 or 2), or 0: k_kv8_chunk's 128 rows
  int z, hh, chunks;       // the tiles' list; heads a workgroup, workgroups a group
  int splits, least;
  int64_t floats;          // of scratch that the splits take
};
// Splits go as far as the caller's scratch.  Times below are of 8 key/value heads of 128 and groups of 4,
// fp16, in us a call by the host's clock over 40 calls (short ones come out up to 3 above the kernels' own
// figures), unless said; the other side of each rule was built and timed with it.
// The lengths are on the device, so the rules go by COLS: the tables timed are as wide as their longest
// sequence, and one that is wider may pay for splits that its sequences have no use for (4 x 1 over
// 270..333 in a table of 25 blocks 12.2, of 6 9.5).  So do sequences of one new token beside one of
// many, which decides for all of a plan (64 x 1 over 700..8191, bf16: 79, with one of 76 among them 239).
Kv8Way kv8_way(int64_t rows, int longest, int heads, int kv_heads, int head_dim, int cols, const int64_t* ntiles,
               int64_t part_cap) {
  Kv8Way w;
  const int group = heads / kv_heads;
  w.hh = group < 16 ? group : 16;
  w.z = 0;
  w.splits = 0;
  w.floats = 0;
  // Few rows: k_kv8_few, which reads codes into registers (64 x 1 token over 700..8191, bf16: 81, with
  // k_kv8_chunk 220).  Two row tiles are one workgroup a CU, whose start and end short tables do not make
  // up for: 17 to 32 rows take k_kv8_chunk up to 32 columns (1 x 8 tokens over 1100 14.0, with k_kv8_few
  // 15.3; 64 x 8 over 700..2000 69, 74) and k_kv8_few past them (16 x 8 over 4000 45, 54; 64 x 8 over
  // 700..8191, bf16, 119, 221).
  if (longest * w.hh <= (cols > 32 ? 32 : 16)) {
    w.rt = longest * w.hh <= 16 ? 1 : 2;
    while ((SEQ_TT0 << w.z) < longest) ++w.z;
    w.chunks = (group + w.hh - 1) / w.hh;
    const int per = kv_heads * w.chunks;
    // as many workgroups as the chip holds at once (64 x 1 over 700..8191, bf16: half of them 89, twice 89,
    // these 81; 1 x 1 over 131071: 53.1, 56.3, 52.4)
    const int slots = 256 * (w.rt == 1 ? (head_dim == 64 ? 4 : 2) : (head_dim == 64 ? 2 : 1));
    int64_t s = slots / per > 0 ? slots / per : 1;
    const int64_t each = (int64_t)per * 32 * w.rt * (head_dim + 2), parts = 2 * ntiles[w.z] * per;
    if (s * each + parts > part_cap) s = (part_cap - parts) / each;
    w.least = 2;   // 4 x 1 over 1100..4000: 14.2, with 4 blocks 16.1, with 16 20.2
    // Tables of up to 16 blocks a workgroup a sequence: the sharing's own steps and the join cost more
    // than it evens out (4 x 1 over 270..333 9.6, shared 11.9; 64 x 1 over 600..1000 25.4, 27.6; past it, 4
    // x 1 over 1100..4000 shared 14.2, else 29.2).  Many sequences nearly even themselves out (300 x 1 over
    // 300..4000 173, shared 167): past 4 tiles a place nothing is shared.
    if (cols > 16 && s > 1 && ntiles[w.z] * per <= 4 * slots && ntiles[w.z] * cols <= INT32_MAX) {
      w.splits = (int)s;
      w.floats = s * each + parts;
    }
    return w;
  }
  w.rt = 0;
  w.hh = group < 8 ? group : 8;   // as attend_packed
  while (w.z + 1 < SEQ_TTS && (SEQ_TT0 << (w.z + 1)) * w.hh <= 128) ++w.z;
  w.least = 2;   // 1 x 76 over 1100 21.0, with 1 block 26.6, with 4 20.9
  w.chunks = (group + w.hh - 1) / w.hh;
  const int64_t groups = ntiles[w.z] * w.chunks * kv_heads, most = (cols + w.least - 1) / w.least;
  const int64_t each = rows * heads * (head_dim + 2);
  // two workgroups a CU: 4 x 512 over 2500..4001 (2 heads of 64, groups of 8, bf16) 63, with 256 in all
  // 79, with 1024 70; 1 x 64 over 16000 41.5, 43.6, 53.1
  int64_t s = groups > 0 ? 512 / groups : 1;
  if (s > most) s = most;
  if (each > 0 && s * each > part_cap) s = part_cap / each;
  w.splits = s < 1 ? 1 : (int)s;
  w.floats = w.splits > 1 ? w.splits * each : 0;
  return w;
}

}  // namespace

int64_t kv8_attend_part(int64_t rows, const int64_t* ntiles, int longest, int heads, int kv_heads, int head_dim, int cols) {
  return rows == 0 ? 0 : kv8_way(rows, longest, heads, kv_heads, head_dim, cols, ntiles, INT64_MAX).floats;
}

hipError_t kv8_attend(hipStream_t s, const Kv8& c, const SeqTile* const* tiles, const int64_t* ntiles, int64_t rows,
                      int longest, int heads, const uint16_t* q, int64_t ldq, float scale, uint16_t* out, int obf,
                      int64_t ldo, float* part, int64_t part_cap) {
  if (ntiles[0] == 0) return hipSuccess;
  const Kv8Way w = kv8_way(rows, longest, heads, c.kv_heads, c.head_dim, c.cols, ntiles, part_cap);
  Kv8Args a;
  a.c = c;
  a.tiles = tiles[w.z];
  a.ntiles = (int)ntiles[w.z];
  a.q = q;
  a.out = out;
  a.ldq = ldq;
  a.ldo = ldo;
  a.scale = scale * 1.4426950408889634f;
  a.heads = heads;
  a.group = heads / c.kv_heads;
  a.tt = SEQ_TT0 << w.z;
  a.hh = w.hh;
  a.chunks = w.chunks;
  a.magic = (65536 + w.hh - 1) / w.hh;
  a.obf = obf;
  a.splits = w.splits;
  a.least = w.least;
  a.part = part;
  a.rows = rows;
  const int64_t groups = (w.rt && w.splits ? w.splits : ntiles[w.z]) * w.chunks * c.kv_heads;
  const int64_t joins = ntiles[w.z] * w.chunks * c.kv_heads;
  if (groups > WG256_MAX || (w.splits > 1 && joins > WG256_MAX)) return hipErrorInvalidConfiguration;
  const dim3 grid((unsigned)groups, w.rt ? 1 : w.splits);
  auto go = [&](auto kern) { hipLaunchKernelGGL(kern, grid, dim3(256), 0, s, a); };
  auto rts = [&](auto bf, auto hd) {
    constexpr int BF = decltype(bf)::value, HD = decltype(hd)::value;
    if (w.rt == 0) return go(k_kv8_chunk<BF, HD>);
    w.rt == 2 ? go(k_kv8_few<BF, HD, 2>) : go(k_kv8_few<BF, HD, 1>);
  };
  typedef std::integral_constant<int, 0> I0;
  typedef std::integral_constant<int, 1> I1;
  typedef std::integral_constant<int, 64> I64;
  typedef std::integral_constant<int, 128> I128;
  if (c.head_dim == 128)
    c.bf16 ? rts(I1(), I128()) : rts(I0(), I128());
  else
    c.bf16 ? rts(I1(), I64()) : rts(I0(), I64());
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || w.splits < 2) return e;
  if (w.rt) {
    // a row a workgroup where a tile has many parts (1 x 1 over 131071 52.4, else 56.9), or two shares
    // and four rows (64-wide: eight)
    const bool few = ntiles[w.z] * 8 <= w.splits;
    const int rw = few ? 1 : 512 / c.head_dim;
    const dim3 jg((unsigned)joins, (longest * w.hh + rw - 1) / rw);
    auto join = [&](auto kern) { hipLaunchKernelGGL(kern, jg, dim3(256), 0, s, a); };
    auto jrt = [&](auto rt) {
      constexpr int RT = decltype(rt)::value;
      if (c.head_dim == 128)
        few ? join(k_kv8_join_few<128, RT, 8>) : join(k_kv8_join_few<128, RT, 2>);
      else
        few ? join(k_kv8_join_few<64, RT, 16>) : join(k_kv8_join_few<64, RT, 2>);
    };
    w.rt == 1 ? jrt(std::integral_constant<int, 1>()) : jrt(std::integral_constant<int, 2>());
    return hipGetLastError();
  }
  const int th = c.head_dim / 4, most = (a.tt < longest ? a.tt : longest) * heads;   // a tile's rows and heads
  // The splits in as many shares as leave a row a workgroup, in half as many, or in one: 1 x 64 over 16000
  // (32 splits) 41.5, 45.5, 50.2; 1 x 76 over 1100 (9) 21.6, 20.9, 21.4; 4 x 512 over 2500..4001 (64-wide, 2
  // splits) 99, -, 63
  const int rw = w.splits > 16 ? 1 : w.splits > 4 ? 2 : 256 / th;
  const dim3 jg((unsigned)ntiles[w.z], (most + rw - 1) / rw);
  auto join = [&](auto kern) { hipLaunchKernelGGL(kern, jg, dim3(256), 0, s, a); };
  if (c.head_dim == 128)
    rw == 1 ? join(k_kv8_join<128, 8>) : rw == 2 ? join(k_kv8_join<128, 4>) : join(k_kv8_join<128, 1>);
  else
    rw == 1 ? join(k_kv8_join<64, 16>) : rw == 2 ? join(k_kv8_join<64, 8>) : join(k_kv8_join<64, 1>);
  return hipGetLastError();
}

// --- attention of sequences that begin alike --------------------------------------------------------
//
// A prefix's blocks are read once for the rows of all its sequences (PREFIX: its rows are one tile's, or
// several's, whatever sequence each is of), each sequence's other blocks as ever (OWN); both leave sums
// relative to a reference of their own, which meet here:
//   m = max m_i, l = sum l_i 2^(m_i - m), o = sum o_i 2^(m_i - m) / l.
// Which blocks those are is found out on the device (Kv8Own): the plan of prefixes is a hint, and what comes
// out is kv8_attend's answer whatever the tables hold.
//
// 64 x 1 token, 60..2000 of their own after 8192 (8 heads of 128, groups of 4, bf16): 48.8 us, kv8_attend 134;
// its bytes would take 18.7: the prefix's products and the own blocks take turns on the CUs, whose places (two
// workgroups each) one launch's 128 prefix workgroups and 512 others fill unevenly.  8 x 1 after 131008, fp16:
// 61 us (kernel 56, 4.9 TB/s; join 7), kv8_attend 288.  16 x 1 after 1088: 15.7 us, 19.2: five loads that wait for
// each other, two blocks, the sums out and in again.  32 x 9 tokens, 12..200 of their own after 8192: 76 us, 164.

// Both passes in one launch: PW workgroups of the prefixes', which take their rows as WAY says (0, 3: chunk_rows, tiles
// of 64 and 128 rows; 1, 2: few_rows with as many row tiles), then the sequences' own by few_rows; WAY 4: tiles of 128 rows
// and of 64
template <int HD, int WAY>
struct PrefixLds : FewLds<HD, WAY, PREFIX> {};
template <int HD>
struct PrefixLds<HD, 0> : ChunkLds<HD, PREFIX> {};
template <int HD>
struct PrefixLds<HD, 3> : ChunkLds<HD, PREFIX> {};
template <int HD>
struct PrefixLds<HD, 4> : ChunkLds<HD, PREFIX> {};
template <int HD, int WAY>
struct OwnLds : FewLds<HD, 1, OWN> {};
template <int HD>
struct OwnLds<HD, 4> : ChunkLds<HD, OWN> {};
template <int BF, int HD, int WAY>
__global__ void __launch_bounds__(256, 2)
k_kv8_shared(Kv8Args P, Kv8Args O, uint32_t pw, uint32_t pgroups, uint32_t ogroups) {
  __shared__ __align__(1024) union Lds {
    PrefixLds<HD, WAY> p;
    OwnLds<HD, WAY> o;
  } lds;
  if (blockIdx.x >= pw) {
    const uint32_t i = blockIdx.x - pw;
    if constexpr (WAY == 4)
      chunk_rows<BF, HD, OWN, 2>(O, lds.o, i % ogroups, i / ogroups);
    else
      few_rows<BF, HD, 1, OWN>(O, lds.o, i % ogroups, i / ogroups);
  } else if constexpr (WAY == 0 || WAY > 2) {
    chunk_rows<BF, HD, PREFIX, WAY == 0 ? 2 : 1>(P, lds.p, blockIdx.x % pgroups, blockIdx.x / pgroups);
  } else {
    few_rows<BF, HD, WAY, PREFIX>(P, lds.p, blockIdx.x % pgroups, blockIdx.x / pgroups);
  }
}

struct Kv8Meet {
  Kv8Args own;
  const float *part, *ml;   // the prefixes' sums
  int64_t n;
};
// The sums of a sequence's own splits and of its prefix's of each row and head, in a fixed order, one pass over them: HD / 4
// threads take one's dims in each of SH shares of the splits, then the shares are summed
template <int HD, int SH>
__global__ void __launch_bounds__(256)
k_kv8_meet(Kv8Meet M) {
  constexpr int TH = HD / 4, RW = 256 / TH / SH;   // threads a row and share; rows a workgroup
  __shared__ __align__(16) float ys[256 / TH][HD];
  __shared__ float ss[256 / TH], ms[256 / TH];
  const Kv8Args& A = M.own;
  const Kv8& c = A.c;
  const SeqTile T = A.tiles[blockIdx.x];
  const int32x4 note = A.notes[blockIdx.x];
  const int live = min(A.tt, T.len - T.t0);
  if ((int)blockIdx.y * RW >= live * A.heads) return;
  const int owns = note[0], all = note[1];
  const int tid = threadIdx.x, sh = tid / TH % SH, r = tid / TH / SH, d = tid % TH * 4;
  const int i = min((int)blockIdx.y * RW + r, live * A.heads - 1);
  const int64_t mine = (int64_t)(T.row0 + T.t0) * A.heads + i, theirs = (int64_t)note[2] * A.heads + i;
  auto slot = [&](int z) { return z < owns ? z * A.n + mine : (z - owns) * M.n + theirs; };
  // a share's sums as they come, under the largest reference so far
  float m = -INFINITY, sum = 0.f;
  f32x4 y = {};
#pragma unroll 4
  for (int z = sh; z < all; z += SH) {
    const int64_t at = slot(z);
    const f32x2 ml = *(const f32x2*)((z < owns ? A.ml : M.ml) + at * 2);
    const f32x4 x = *(const f32x4*)((z < owns ? A.part : M.part) + at * HD + d);
    if (ml[0] == -INFINITY) {   // no reference: a weight of 0, or NaN
      sum += ml[1];
      continue;
    }
    const float mn = fmaxf(m, ml[0]);
    const float a = m == mn ? 1.f : __builtin_amdgcn_exp2f(m - mn), w = ml[0] == mn ? 1.f : __builtin_amdgcn_exp2f(ml[0] - mn);
    sum = sum * a + w * ml[1];
    y *= a;
    if (w > 0.f) y += w * x;
    m = mn;
  }
  if constexpr (SH > 1) {
    if (d == 0) ms[tid / TH] = m;
    __syncthreads();
    float top = m;
#pragma unroll
    for (int k = 0; k < SH; ++k) top = fmaxf(top, ms[r * SH + k]);
    if (m != top) {
      const float a = m == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - top);
      sum *= a;
      y *= a;
    }
  }
  if constexpr (SH > 1) {
    *(f32x4*)&ys[tid / TH][d] = y;
    if (d == 0) ss[tid / TH] = sum;
    __syncthreads();
    if (sh) return;
#pragma unroll
    for (int k = 1; k < SH; ++k) {
      y += *(const f32x4*)&ys[r * SH + k][d];
      sum += ss[r * SH + k];
    }
  }
  if ((int)blockIdx.y * RW + r >= live * A.heads) return;
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  uint16_t* po = A.out + (mine / A.heads) * A.ldo + (mine % A.heads) * HD + d;
  *(u32x2*)po = u32x2{pack_out(y[0] * inv, y[1] * inv, c.bf16, A.obf), pack_out(y[2] * inv, y[3] * inv, c.bf16, A.obf)};
}

namespace {

// one of attend_shared's passes: how its rows are taken (k_kv8_shared's WAY), and into how many splits their blocks
struct PassWay {
  int way, z, hh, chunks, splits, least;
  int64_t groups;   // workgroups a split
};
// HH heads a workgroup, in tiles that hold TOKENS (or in the largest)
PassWay pass_rows(int way, int hh, int tokens, int group, int kv_heads, const int64_t* ntiles) {
  PassWay w{way, 0, hh, (group + hh - 1) / hh, 1, 1, 0};
  while ((SEQ_TT0 << w.z) < tokens && w.z + 1 < SEQ_TTS) ++w.z;
  w.groups = ntiles[w.z] * w.chunks * kv_heads;
  return w;
}
// As many splits as SLOTS workgroups are, none of less than LEAST blocks; at most 64, whose sums the join reads (2
// x 1 after 32768, 16 heads over 1: 25.5, at most 128 32.9, 16 27.9; 4 x 1: 28.0, 30.7, 49.0)
void pass_splits(PassWay& w, double slots, int blocks, int least) {
  w.least = least;
  const int64_t s = w.groups > 0 ? (int64_t)(slots / w.groups) : 1, pays = (blocks + least - 1) / least;
  w.splits = (int)std::max<int64_t>(1, std::min<int64_t>(std::min(s, pays), 64));
}
struct SharedWay {
  bool pays;
  PassWay pre, own;
  int64_t pre_each, own_each, notes, floats;   // floats of a split of either, of the notes, in all
};
// Microseconds of a call of kv8_attend whose sequences have BLOCKS blocks in all of their prefixes, and of one in the two
// passes W: lines through the times of 3029 calls, taken on either side (1 to 32 key/value heads of 64 and 128, groups of 1 to
// 16, 2 to 256 sequences of 12..200 tokens of their own and 1 to 160 new ones, prefixes of 4 to 2000 blocks, bf16), those of
// MANY rows a head and sequence (past 64) by themselves; root mean square 15% off, of many rows 6%.  What they are to get
// right is which is the smaller.  By them and the rule in shared_way 14 of the 1726 calls of up to 64 rows run the slower side
// at a loss of more than 3%, 3.8 us at most (by counts of saved blocks alone 105, 16 us at most), and 63 of the 1303 of more,
// 9 us at most (158, 32 us); of 350 others, drawn at random, also of long sequences of their own, 34, by sharing 10 of them,
// 8.3 us at most.
double alone_us(int64_t rows, int longest, int64_t blocks, int heads, int kv_heads, int head_dim, int cols,
                const int64_t* ntiles, bool many) {
  const Kv8Way a = kv8_way(rows, longest, heads, kv_heads, head_dim, cols, ntiles, INT64_MAX);
  const int64_t per = (int64_t)kv_heads * a.chunks, tiles = (longest + (SEQ_TT0 << a.z) - 1) / (SEQ_TT0 << a.z);
  // those that one of 512 places takes, of a key/value head of 128; a split's sums, in and out again
  const double steps = (double)blocks * tiles * per * head_dim / 128 / 512, sums = (double)rows * heads * head_dim / 128e3;
  const double joined = a.splits > 1 ? sums * a.splits : 0;
  if (many) return 12.3 + (head_dim == 64 ? 3.24 : 2.42) * steps + 0.283 * joined + 0.37 * sums;
  if (a.rt == 0) return 13.8 + 2.95 * steps + 0.195 * joined;
  if (a.rt == 1) return (cols > 16 ? 15.9 : 8) + 1.36 * steps;   // one launch up to 16 columns
  // two row tiles: workgroups of whole sequences where there are as many places (32 x 8 after 2048 35, 16 x 8 32, 64 x 8 82)
  return (ntiles[a.z] * per == 256 * (head_dim == 64 ? 2 : 1) ? 14 : 22.5) + 1.21 * steps;
}
double shared_us(const SharedWay& w, int64_t rows, int heads, int head_dim, int blocks, bool many) {
  // a workgroup's blocks one after the other; the splits with any
  const int way = w.pre.way, chain = std::max(w.pre.least, (blocks + w.pre.splits - 1) / w.pre.splits);
  const int S = (blocks + chain - 1) / chain;
  const double sums = (double)rows * heads * head_dim / 128e3, own = w.own.groups / 512.;
  if (many) {   // a prefix's workgroups past the places run in turns, and past half of them share the CUs
    const double turns = (double)w.pre.groups * w.pre.splits / 512;
    return 8.7 + (head_dim == 64 ? 1.18 : 1.75) * chain * (std::max(1., std::ceil(turns)) + 0.59 * std::max(0., turns - 0.5)) +
           0.44 * sums * S + 0.07 * S + 6.7 * own;
  }
  const double step = (way == 4 ? 1.79 : way == 0 || way == 3 ? 1.82 : 0.37) * (head_dim == 64 ? 0.4 : 1);
  return (way == 4 ? 14.25 + 0.3 * sums : 10 + 1.56 * sums) + step * chain + (way == 4 ? 0.21 : 0.225) * sums * S +
         0.05 * S + 0.065 * std::max(0, S - 32) + 1.5 * own;
}
// The rules' times are as kv8_way's, of one new token a sequence in bf16 with 12 to 200 of its own, unless said.
SharedWay shared_way(int64_t rows, int longest, const Kv8Shared& sh, int heads, int kv_heads, int head_dim, int cols,
                     const int64_t* ntiles) {
  SharedWay w{};
  const int group = heads / kv_heads, h16 = group < 16 ? group : 16, h8 = group < 8 ? group : 8;
  const int blocks = sh.blocks < cols ? sh.blocks : cols, own = cols > sh.fewest ? cols - sh.fewest : 1;
  const int64_t saved = std::min(sh.saved, sh.rows * cols);   // a hint may say more than tables hold
  const bool few = longest * h16 <= 16;
  auto tokens = [&](int rows) {   // that tiles of ROWS rows hold
    int n = SEQ_TT0;
    while (2 * n * h8 <= rows && n < (SEQ_TT0 << (SEQ_TTS - 1))) n *= 2;
    return n;
  };
  const int64_t held = tokens(128), room = (longest + held - 1) / held * held;   // tokens of a sequence's tiles of 128 rows
  // Shared where enough blocks need not be read again, counted as of 8 key/value heads where there are more, and
  // where the estimates above are for it.  Enough: of prefixes past 16 blocks (up to there
  // kv8_attend is one launch, 64 x 1 after 640 19.5, shared 24.8, which 100 MB make up for: 64 x 1 after 1024, 32 heads, 529
  // MB, 98.9, 41.9; 16 x 1 after 512, 63 MB, 19.4, 22.4) so many (8 x 1 after 1088, 119: 17.2, 14.4; 4 after 2048, 96: 13.9,
  // 15.4; 2 after 8192, 128: 18.3, 20.8, after 32768, 512: 33.0, 26.3); of sequences of 17 rows a key/value head and more 384
  // (4 x 8 after 4096, 192: 28.8, 25.6, 4 x 16: 30.8, 31.9; 4 x 16 after 8192, 384: 38.9, 36.3; 32 x 9 after 8192, 3968: 164,
  // 76); of more than 64 where kv8_attend's tiles of 128 would be a good part empty, which is what a prefix's are not (20 of
  // 32 tokens and less: 16 x 40 after 8192, 1920: 175, 126; 8 x 40 after 4096, 448: 61.8, 63.1; 16 x 24 after 4096, 960: 62.2,
  // 65.5; 32 x 32 after 4096 107, 116).
  const int64_t least = few ? (sh.seqs < 4 ? 384 : 112) : longest * h8 <= 64 ? 384 : 8ll * longest <= 5 * room ? 896 : INT64_MAX;
  const bool enough = blocks > 16 ? saved * std::max(kv_heads, 8) / 8 >= least
                                  : few && saved * kv_heads * head_dim >= 100000000 / 128;
  if (sh.rows == 0 || !enough) return w;
  w.own = few ? pass_rows(1, h16, longest, group, kv_heads, ntiles) : pass_rows(0, h8, tokens(64), group, kv_heads, ntiles);
  // A sequence's own blocks are split as far as there are places for the workgroups, by all the table's: any may come to be
  // its own, where its table parts from its prefix (4 x 1 after 32768, 2 heads of 64, one parted at its first: 26 us, split
  // by the blocks past the shortest prefix 165; 8 x 1 after 131008: 187, 504)
  pass_splits(w.own, 256 * (head_dim == 64 ? 4 : 2), cols, 8);
  if (few && (int64_t)sh.most * h16 <= 32) {
    // The bytes are the cost: few_rows.  17 to 32 rows are two row tiles of a workgroup (8 x 1 after 131008 58.7), or
    // in shorter prefixes workgroups of half the heads, whose blocks' second reading the L2 has (8 x 1 after 8192
    // 17.2, two row tiles 20.1; after 32768 30.3, 27.9)
    const bool half = sh.most * h16 > 16 && sh.most <= 16 && blocks < 400;
    w.pre = pass_rows(sh.most * h16 <= 16 || half ? 1 : 2, half ? 16 / sh.most : h16, sh.most, group, kv_heads, sh.ntiles);
    // one workgroup a CU, the other place is the sequences' (8 x 1 after 131008: 58.7, 192 in all 67.6, 320 74.3)
    pass_splits(w.pre, 256, blocks, 4);
  } else {
    // The products are: chunk_rows, tiles of 128 rows, up to 64 rows of 64 (a wave half of a block's keys: 16 x 1 after
    // 131008 105, with half of the waves idle 121)
    const int way = !few ? 4 : (int64_t)sh.most * h8 <= 64 ? 0 : 3;
    w.pre = pass_rows(way, h8, tokens(way ? 128 : 64), group, kv_heads, sh.ntiles);
    // The share of the CUs, a workgroup each, that this pass is of both, where each would take so long with all of them:
    // 1.5 us a block of a tile, a quarter of the own blocks that there may be at 5 TB/s (64 x 1 after 8192, 60..2000 of
    // their own: 128 workgroups 48.4, 64 69.5, 256 53.1, 512 62.9; 12..200: 128 44, 256 33.5); two each for long ones (64
    // x 1 after 65536: 106, one each 125)
    const double units = w.pre.groups * (double)blocks;
    const double a = units * 1.5 / 256, b = w.own.groups * (double)own / 4 * (head_dim * 128) / 5e6;
    pass_splits(w.pre, std::min(512., a / (a + b) * (units >= 16 * 512 ? 512 : 256) + w.pre.groups - 1), blocks, 2);
  }
  const bool many = longest * h8 > 64;
  w.pays = shared_us(w, rows, heads, head_dim, blocks, many) <
           alone_us(rows, longest, saved + blocks, heads, kv_heads, head_dim, cols, ntiles, many);
  if (!w.pays) return w;
  w.pre_each = sh.rows * heads * (head_dim + 2);
  w.own_each = rows * heads * (head_dim + 2);
  w.notes = 4 * ntiles[w.own.z];
  w.floats = w.pre.splits * w.pre_each + w.own.splits * w.own_each + w.notes;
  return w;
}

}  // namespace

int64_t kv8_shared_part(int64_t rows, int longest, const Kv8Shared& sh, int heads, int kv_heads, int head_dim,
                        int cols, const int64_t* ntiles) {
  const SharedWay w = shared_way(rows, longest, sh, heads, kv_heads, head_dim, cols, ntiles);
  return w.pays ? w.floats : kv8_attend_part(rows, ntiles, longest, heads, kv_heads, head_dim, cols);
}

hipError_t kv8_attend_shared(hipStream_t s, const Kv8& c, const SeqTile* const* tiles, const int64_t* ntiles,
                             int64_t rows, int longest, const Kv8Shared& sh, int heads, const uint16_t* q,
                             int64_t ldq, float scale, uint16_t* out, int obf, int64_t ldo, float* part, int64_t part_cap) {
  if (ntiles[0] == 0) return hipSuccess;
  SharedWay w = shared_way(rows, longest, sh, heads, c.kv_heads, c.head_dim, c.cols, ntiles);
  if (!w.pays || part_cap < w.notes + w.pre_each + w.own_each ||
      w.pre.groups * w.pre.splits + w.own.groups * w.own.splits > WG256_MAX)
    return kv8_attend(s, c, tiles, ntiles, rows, longest, heads, q, ldq, scale, out, obf, ldo, part, part_cap);
  if (w.floats > part_cap) {   // fewer splits, the prefixes' first to keep theirs
    const int64_t spare = part_cap - w.notes - w.pre_each - w.own_each, p = 1 + spare / w.pre_each;
    if (p < w.pre.splits) w.pre.splits = (int)p;
    const int64_t o = 1 + (spare - (w.pre.splits - 1) * w.pre_each) / w.own_each;
    if (o < w.own.splits) w.own.splits = (int)o;
  }
  Kv8Args a;
  a.c = c;
  a.q = q;
  a.out = out;
  a.ldq = ldq;
  a.ldo = ldo;
  a.scale = scale * 1.4426950408889634f;
  a.heads = heads;
  a.group = heads / c.kv_heads;
  a.obf = obf;
  a.rows = rows;
  a.entry = sh.entry;
  a.blocks = sh.tile_blocks[w.pre.z];
  a.of = (const int32x4*)sh.of;
  Kv8Args b = a;   // a: the prefixes' pass, b: the sequences' own
  a.tiles = sh.tiles[w.pre.z];
  a.ntiles = (int)sh.ntiles[w.pre.z];
  a.n = sh.rows * heads;
  b.tiles = tiles[w.own.z];
  b.ntiles = (int)ntiles[w.own.z];
  b.n = rows * heads;
  auto fill = [&](Kv8Args& x, const PassWay& p) {
    x.tt = SEQ_TT0 << p.z;
    x.hh = p.hh;
    x.chunks = p.chunks;
    x.magic = (65536 + p.hh - 1) / p.hh;
    x.splits = p.splits;
    x.least = p.least;
  };
  fill(a, w.pre);
  fill(b, w.own);
  a.part = part;
  b.part = a.part + a.splits * a.n * c.head_dim;
  b.notes = (int32x4*)(b.part + b.splits * b.n * c.head_dim);
  a.ml = (float*)(b.notes + b.ntiles);
  b.ml = a.ml + a.splits * a.n * 2;
  a.notes = nullptr;
  b.psplits = a.splits;
  b.pleast = a.least;
  const int64_t pw = w.pre.groups * a.splits;
  typedef std::integral_constant<int, 0> I0;
  typedef std::integral_constant<int, 1> I1;
  typedef std::integral_constant<int, 64> I64;
  typedef std::integral_constant<int, 128> I128;
  auto go = [&](auto kern) {
    hipLaunchKernelGGL(kern, dim3((unsigned)(pw + w.own.groups * b.splits)), dim3(256), 0, s, a, b, (uint32_t)pw,
                       (uint32_t)w.pre.groups, (uint32_t)w.own.groups);
  };
  auto ways = [&](auto bf, auto hd) {
    constexpr int BF = decltype(bf)::value, HD = decltype(hd)::value;
    w.pre.way == 0   ? go(k_kv8_shared<BF, HD, 0>)
    : w.pre.way == 1 ? go(k_kv8_shared<BF, HD, 1>)
    : w.pre.way == 2 ? go(k_kv8_shared<BF, HD, 2>)
    : w.pre.way == 3 ? go(k_kv8_shared<BF, HD, 3>)
                     : go(k_kv8_shared<BF, HD, 4>);
  };
  if (c.head_dim == 128)
    c.bf16 ? ways(I1(), I128()) : ways(I0(), I128());
  else
    c.bf16 ? ways(I1(), I64()) : ways(I0(), I64());
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  Kv8Meet m;
  m.own = b;
  m.part = a.part;
  m.ml = a.ml;
  m.n = a.n;
  const int th = c.head_dim / 4, most = (b.tt < longest ? b.tt : longest) * heads;   // a tile's rows and heads
  const int rw = a.splits + b.splits > 16 ? 1 : a.splits + b.splits > 4 ? 2 : 256 / th;
  const dim3 jg((unsigned)ntiles[w.own.z], (most + rw - 1) / rw);
  auto join = [&](auto kern) { hipLaunchKernelGGL(kern, jg, dim3(256), 0, s, m); };
  if (c.head_dim == 128)
    rw == 1 ? join(k_kv8_meet<128, 8>) : rw == 2 ? join(k_kv8_meet<128, 4>) : join(k_kv8_meet<128, 1>);
  else
    rw == 1 ? join(k_kv8_meet<64, 16>) : rw == 2 ? join(k_kv8_meet<64, 8>) : join(k_kv8_meet<64, 1>);
  return hipGetLastError();
}

}  // namespace exn
