// packed.hip -- causal attention over whole prompts of different lengths, packed one after the
// other, on gfx950's MFMA: for query i of a sequence and head h (g query heads a key/value head)
//   o[i, h] = sum_{j <= i} p_j v[j, h / g] / sum_{j <= i} p_j,  p_j = 2^(scale log2(e) q[i, h].k[j, h / g] - m)
// in one pass over the keys with m a running reference (the row's running max, which it may lag by
// MAX_SLACK; sums and rescales in fp32, p rounded to the inputs' 16 bits for the second product: half
// a step of a weight, as much as the output's own rounding).  fp16 has no weight under 2^-24, which many
// small ones beside one that takes nearly all would be, so m lies F16_LIFT under the reference: weights reach
// 2^(F16_LIFT + MAX_SLACK) of fp16's 2^16, and what is lost is under 2^-32 of a row's largest (a key of no
// value with 0.999 of the weight before 5,000 others, fp16 rows: 2.1e-4 off, unlifted 3.8e-2).
//
// A workgroup takes TT tokens of one sequence times the HH query heads of one key/value head: 128
// rows, 32 a wave, row r being token r / HH and head r % HH.  The heads of a group so share every
// key and value tile, and at 4 heads a group a tile spans 32 tokens: its last key tile wastes at most
// 63 keys a row, where 128 tokens would waste 190.
//
// The products are taken transposed (attn.hip's arrangement): S^T = K Q^T leaves a query in a lane's
// column, whose p are then the B operand of O^T += V^T P^T as they are.  V lies in LDS as in memory,
// [key][dim]; gfx950's transposing LDS read hands each lane four keys of its dim.
//
// Matrix instructions bound it for long prompts: 2 x 8192 tokens (32 heads of 128, 8 of keys and values,
// bf16) 1,005 us, 1,090 TFLOP/s where a large library product reaches 1,210 (matrix units busy 57% of the
// cycles at a clock that power holds at 1.6 to 1.9 GHz).  Two waves of a SIMD alternate between products
// and exp2; 64 rows a wave took 1.21 ms, eight waves in two fixed phases 1.06 ms.  Short ones are bound
// by the start and end of a workgroup: 4 x 1100..1180 58 us (735 TFLOP/s), 16 x 21..257 11.4 us, 1 x 24
// 6.9 us; 24 x 5..4001 (16 heads of 64, 2 of keys and values) 89.5 us (830 TFLOP/s).
#include "exn_common.h"

#include <type_traits>

namespace exn {

#define PK 64            // keys a tile
#define MAX_SLACK 8.f    // log2 units the running max may lag the true max by
#define F16_LIFT 7.f     // log2 units that fp16 weights are held higher

typedef __attribute__((address_space(3))) void lds_void;
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));

template <int BF>
__device__ __forceinline__ float ld16(const uint16_t* p) {
  return BF ? bf16_to_f32(*p) : f16_to_f32(*p);
}
__device__ __forceinline__ uint32_t pack16(float a, float b, int bf) { return bf ? pack_bf16x2(a, b) : pack_f16x2(a, b); }
// results of inputs of type BF (bf16's may well be past fp16's range)
template <int BF>
__device__ __forceinline__ uint32_t pack_out(float a, float b, int obf) {
  return obf ? pack_bf16x2(a, b) : BF ? pack_f16x2(a, b) : pack_f16x2_in(a, b);
}

template <int BF>
__device__ __forceinline__ f32x16 mfma32(s16x8 a, s16x8 b, f32x16 c) {
  if constexpr (BF)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// max of three that have come out of VALU instructions (a plain fmaxf first quiets each operand)
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}
__device__ __forceinline__ float pmax32(float v) {   // with lane ^ 32
  float a = v, b = v;
  xswap32(a, b);
  return fmaxf(a, b);
}
__device__ __forceinline__ float psum32(float v) {
  float a = v, b = v;
  xswap32(a, b);
  return a + b;
}

// One row by a whole wave, keys 0 .. LIM: nothing that the row does not see is multiplied.  For
// rows whose sums came out not finite: a hidden value in a row's own tile, an infinity or a NaN, times
// its weight of zero is a NaN in the matrix units.
template <int BF, int HD>
__device__ void packed_row(const uint16_t* __restrict__ q, const uint16_t* __restrict__ k, int64_t ldk,
                           const uint16_t* __restrict__ v, int64_t ldv, int lim, float scale, uint16_t* __restrict__ out,
                           int obf) {
  const int lane = threadIdx.x & 63;
  float m = -INFINITY, l = 0.f, o[HD / 64] = {};
  for (int j0 = 0; j0 <= lim; j0 += 64) {
    const int j = j0 + lane;
    float s = -INFINITY;
    if (j <= lim) {
      s = 0.f;
      for (int d = 0; d < HD; ++d) s += ld16<BF>(q + d) * ld16<BF>(k + (int64_t)j * ldk + d);
      s *= scale;
    }
    const float mn = fmaxf(m, wave_max(s)), mu = mn == -INFINITY ? 0.f : mn;
    const float a = exp2f(m - mu), p = exp2f(s - mu);
    l = l * a + wave_sum(p);
    m = mn;
    for (int c = 0; c < 64 && j0 + c <= lim; ++c) {
      const float pc = __shfl(p, c, 64);
      for (int e = 0; e < HD / 64; ++e)
        o[e] = (c == 0 ? o[e] * a : o[e]) + pc * ld16<BF>(v + (int64_t)(j0 + c) * ldv + e * 64 + lane);
    }
  }
  for (int e = 0; e < HD / 64; ++e) out[e * 64 + lane] = (uint16_t)pack_out<BF>(o[e] / l, 0.f, obf);
}

struct PackedArgs {
  const SeqTile* tiles;
  const uint16_t *q, *k, *v;
  uint16_t* out;
  int64_t ldq, ldk, ldv, ldo;
  float scale;             // times log2(e)
  int kv_heads, group;
  int tt, hh, chunks;      // tokens and heads a workgroup; workgroups a key/value head's group
  uint32_t magic;          // ceil(65536 / hh): r / hh = r magic >> 16 for r < 256
  int obf;
};

// grid: tiles x chunks x kv_heads, the heads fastest; block 256.  LO: weights as two bf16 parts, where
// bf16 inputs give fp16 rows: one part's half step, 2^-9, would be eight of the output's (4 x 1100..1180
// tokens 75 us where bf16 rows take 58; 2.2e-4 from the exact values, in one part 1.2e-3).
template <int BF, int HD, int LO>
__global__ void __launch_bounds__(256, HD == 64 ? 3 : 2)
k_attend_packed(PackedArgs A) {
  constexpr int ROWB = HD * 2, STAGE = PK * ROWB;   // bytes of a key's row; of a tile
  constexpr int CH = HD / 8;                        // 16-byte chunks a row
  constexpr int RI = 1024 / ROWB;                   // rows a DMA instruction moves
  constexpr int DI = PK / RI / 4;                   // DMA instructions a wave and tile
  constexpr int NS = HD / 16;                       // k-steps of the S product
  constexpr int ND = HD / 32;                       // 32-dim blocks of O
  constexpr float LIFT = BF ? 0.f : F16_LIFT;
  // K stage s at s STAGE, V stage s at (2 + s) STAGE, in two rings one tile apart: step t reads K of
  // tile t+1 and V of tile t.  K rows: 16-byte chunk c at c ^ (row % 16) (HD 64: c ^ (row / 2 % 8)),
  // so that 32 rows' same chunk meets every bank once; V rows: c ^ 4 (row % 4) (HD 64: c ^ 4 (row / 2
  // % 2)), so that the transposing read's 4 rows of 64 bytes do.
  __shared__ __align__(1024) uint8_t smem[5 * STAGE];
  const int per = A.kv_heads * A.chunks;
  const SeqTile T = A.tiles[blockIdx.x / per];
  const int hc = blockIdx.x % per, kvh = hc % A.kv_heads, chunk = hc / A.kv_heads;
  const int tid = threadIdx.x, lane = tid & 63, hi = lane >> 5, lo = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int live = min(A.tt, T.len - T.t0);                       // tokens here
  const int heads = min(A.hh, A.group - chunk * A.hh);
  const int row = wave * 32 + lo, tok = (int)(row * A.magic >> 16), head = row - tok * A.hh;
  const bool mine = tok < live && head < heads;
  const int lim = T.t0 + min(tok, live - 1);

  const int tiles = (T.t0 + live - 1) / PK + 1;
  const int minlim = T.t0 + (int)(wave * 32 * A.magic >> 16);     // the wave's first token

  const uint16_t* kbase = A.k + (int64_t)T.row0 * A.ldk + kvh * HD;
  const uint16_t* vbase = A.v + (int64_t)T.row0 * A.ldv + kvh * HD;
  // DMA i of wave w: rows (4i + w) RI .. + RI - 1 of a tile.  A tile's resource ends with the
  // sequence's last row, so that rows past it read zeros, whatever follows.
  uint32_t koff[DI], voff[DI];
#pragma unroll
  for (int i = 0; i < DI; ++i) {
    const int r = (4 * i + wave) * RI + lane / CH, c = lane % CH;
    const int kc = HD == 128 ? c ^ (r & 15) : c ^ ((r >> 1) & 7), vc = HD == 128 ? c ^ (4 * (r & 3)) : c ^ (4 * ((r >> 1) & 1));
    koff[i] = (r * (uint32_t)A.ldk + 8 * kc) * 2u;
    voff[i] = (r * (uint32_t)A.ldv + 8 * vc) * 2u;
  }
  auto dma = [&](const uint16_t* base, int64_t ld, const uint32_t* off, int t, uint8_t* dst) {
    const int64_t ext = ((int64_t)(T.len - t * PK - 1) * ld + HD) * 2;
    const uint32_t records = ext >> 32 ? 0xFFFFFFFFu : (uint32_t)ext;   // a tile's offsets are under 2^31
    __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc((void*)(base + (int64_t)t * PK * ld), 0, (int)records,
                                                                 0x00020000);
#pragma unroll
    for (int i = 0; i < DI; ++i)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_void*)(dst + (4 * i + wave) * 1024), 16, off[i], 0, 0, 0);
  };
  auto dma_k = [&](int t) { dma(kbase, A.ldk, koff, t, smem + (t & 1) * STAGE); };
  auto dma_v = [&](int t) { dma(vbase, A.ldv, voff, t, smem + (2 + (t & 1)) * STAGE); };

  dma_k(0);

  // The wave's rows of Q by DMA too, into V's stage 1 and the stage after it, which nobody needs yet:
  // whole rows of memory at a time, where reading the operand's 16-byte pieces of 32 rows a load keeps
  // the address unit busy several times as long.
  uint8_t* qmem = smem + 3 * STAGE + wave * 32 * ROWB;
#pragma unroll
  for (int i = 0; i < 32 / RI; ++i) {
    const int r = i * RI + lane / CH, gr = wave * 32 + r, rt = (int)(gr * A.magic >> 16);
    const int c = lane % CH ^ (HD == 128 ? r & 15 : (r >> 1) & 7);
    const uint16_t* qr = A.q + (int64_t)(T.row0 + T.t0 + min(rt, live - 1)) * A.ldq +
                         (int64_t)(kvh * A.group + chunk * A.hh + min(gr - rt * A.hh, heads - 1)) * HD + 8 * c;
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)qr, (lds_void*)(qmem + i * 1024), 16, 0, 0);
  }
  dma_v(0);
  if (tiles > 1) dma_k(1);
  // per-lane LDS offsets: K row 32b + lo, chunk 2s + hi; V key 16u + 8e + 4 hi + i / 4 (i the lane of
  // its 16), dims 32d + 16 (lane / 16 % 2) + 4 (i % 4) ..: u, e and b are immediates, the
  // stage is toggled (one body for both keeps the accumulators in one place)
  int kofs[NS], vofs[ND];
#pragma unroll
  for (int s = 0; s < NS; ++s)
    kofs[s] = lo * ROWB + (((2 * s + hi) ^ (HD == 128 ? lo & 15 : (lo >> 1) & 7)) << 4);
  {
    const int r = (lane & 15) >> 2;
#pragma unroll
    for (int d = 0; d < ND; ++d) {
      const int c = 4 * d + 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
      vofs[d] = 2 * STAGE + (4 * hi + r) * ROWB + ((c ^ (HD == 128 ? 4 * r : 4 * (r >> 1))) << 4) + 8 * (lane & 1);
    }
  }
  // S product i = 2s + b: K fragment of 32-key block b, k-step s; O product j = ND u + d: V^T
  // fragment of dims 32d .., keys 16u ..
  auto kfrag = [&](int i) { return *(const s16x8*)(smem + kofs[i / 2] + (i % 2) * 32 * ROWB); };
  auto vfrag = [&](int j) {
    typedef __attribute__((address_space(3))) s16x4 lds_s4;
    uint8_t* p = smem + vofs[j % ND] + (j / ND) * 16 * ROWB;
    const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)p);
    const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(p + 8 * ROWB));
    return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
  };

  s16x8 qf[NS];   // Q^T as the B operand: this lane's row, dims 16s + 8 hi ..
  f32x16 o[ND];
#pragma unroll
  for (int d = 0; d < ND; ++d) o[d] = f32x16{};
  float mrun = 0.f, lrun = 0.f;
  f32x16 sc[2];   // q.k of the tile in hand: two 32-key blocks x this wave's 32 rows

  // Step t: the softmax of tile t, the S product of tile t+1 interleaved with tile t's exp2, then
  // O^T += V^T P^T of tile t.
  auto step = [&](auto last_c, int t) __attribute__((always_inline)) {
    constexpr bool LAST = decltype(last_c)::value;
    // K of tile t+1 and V of tile t have landed for every wave, and every wave is done with K of
    // tile t and V of tile t-1
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt((0x7 << 4) | (0x0 << 8));   // vmcnt(0) lgkmcnt(0)
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    if constexpr (!LAST) {
      if (t + 2 < tiles) dma_k(t + 2);
      dma_v(t + 1);
    }
    const int k0 = t * PK;
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int r = 0; r < 16; ++r) sc[b][r] = __builtin_fmaf(sc[b][r], A.scale, LIFT - mrun);
    if (k0 + PK - 1 > minlim) {   // some key of this tile is hidden from some row
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int key = k0 + 32 * b + 8 * (r >> 2) + 4 * hi + (r & 3);
          if (key > lim) sc[b][r] = -INFINITY;
        }
    }
    float m4[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const int b = c / 2, r0 = (c % 2) * 8;
      float m = max3(sc[b][r0], sc[b][r0 + 1], sc[b][r0 + 2]);
      m = max3(m, sc[b][r0 + 3], sc[b][r0 + 4]);
      m = max3(m, sc[b][r0 + 5], sc[b][r0 + 6]);
      m4[c] = fmaxf(m, sc[b][r0 + 7]);
    }
    const float mx = pmax32(max3(max3(m4[0], m4[1], m4[2]), m4[3], m4[3]));
    // the first tile always sets the reference (its key 0 is visible to every row)
    const bool move = t == 0 || mx > MAX_SLACK + LIFT;
    if (__ballot(move)) {
      const float shift = move ? mx - LIFT : 0.f;
      if (t > 0) {
        const float alpha = __builtin_amdgcn_exp2f(-shift);
        lrun *= alpha;
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
          for (int r = 0; r < 16; ++r) o[d][r] *= alpha;
      }
      mrun += shift;
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int r = 0; r < 16; ++r) sc[b][r] -= shift;
    }

    // Fragment reads run KD MFMAs ahead of their use; the first KD V^T fragments go out in the last
    // slots of the S product.  A slot of the S product takes its share of the tile's 16 pairs of p.
    constexpr int KD = 3, NI = 2 * NS, PS = 16 / NI;
    f32x16 sn[2];
    uint32_t pk[16], pl[LO ? 16 : 1];   // pair i: keys of S element (i / 8, 2 (i % 8)) and the next
    s16x8 kq[KD], vq[KD];
    if constexpr (!LAST) {
      sn[0] = f32x16{};
      sn[1] = f32x16{};
#pragma unroll
      for (int i = 0; i < KD; ++i) kq[i] = kfrag(i);
    }
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      if constexpr (!LAST) {
        s16x8 kn = {};
        if (i + KD < NI) kn = kfrag(i + KD);
        sn[i % 2] = mfma32<BF>(kq[0], qf[i / 2], sn[i % 2]);
#pragma unroll
        for (int d = 0; d + 1 < KD; ++d) kq[d] = kq[d + 1];
        kq[KD - 1] = kn;
      }
      if (i >= NI - KD) vq[i - (NI - KD)] = vfrag(i - (NI - KD));
#pragma unroll
      for (int e = 0; e < PS; ++e) {
        const int pi = PS * i + e, b = pi / 8, r = 2 * (pi % 8);
        const float p0 = __builtin_amdgcn_exp2f(sc[b][r]), p1 = __builtin_amdgcn_exp2f(sc[b][r + 1]);
        pk[pi] = pack16(p0, p1, BF);
        if constexpr (LO) pl[pi] = pack_bf16x2(p0 - bf16_lo(pk[pi]), p1 - bf16_hi(pk[pi]));
        lrun += p0;
        lrun += p1;
      }
      __builtin_amdgcn_sched_barrier(0);
    }

    // O^T += V^T P^T over 4 steps of 16 keys (step u: block u / 2, rows 8 (u % 2) ..)
#pragma unroll
    for (int j = 0; j < 4 * ND; ++j) {
      s16x8 vn = {};
      if (j + KD < 4 * ND) vn = vfrag(j + KD);
      const int u = j / ND;
      const s16x8 pb = __builtin_bit_cast(s16x8, u32x4{pk[4 * u], pk[4 * u + 1], pk[4 * u + 2], pk[4 * u + 3]});
      o[j % ND] = mfma32<BF>(vq[0], pb, o[j % ND]);
      if constexpr (LO)
        o[j % ND] = mfma32<BF>(vq[0], __builtin_bit_cast(s16x8, u32x4{pl[4 * u], pl[4 * u + 1], pl[4 * u + 2], pl[4 * u + 3]}),
                               o[j % ND]);
#pragma unroll
      for (int d = 0; d + 1 < KD; ++d) vq[d] = vq[d + 1];
      vq[KD - 1] = vn;
      __builtin_amdgcn_sched_barrier(0);
    }
    if constexpr (!LAST) {
      sc[0] = sn[0];
      sc[1] = sn[1];
    }
    asm volatile("" : "+v"(lrun));
  };

  // S of tile 0 once its K has landed: V 0 and K 1, asked for after it (and after Q), still move
  asm volatile("" ::: "memory");
  if (tiles > 1)
    __builtin_amdgcn_s_waitcnt(0xF70 | 2 * DI);
  else
    __builtin_amdgcn_s_waitcnt(0xF70 | DI);
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
#pragma unroll
  for (int s = 0; s < NS; ++s) qf[s] = *(const s16x8*)(qmem + kofs[s]);
  sc[0] = f32x16{};
  sc[1] = f32x16{};
#pragma unroll
  for (int i = 0; i < 2 * NS; ++i) {
    sc[i % 2] = mfma32<BF>(kfrag(i), qf[i / 2], sc[i % 2]);
    if (i % 4 == 3) __builtin_amdgcn_sched_barrier(0);
  }

#pragma unroll
  for (int s = 0; s < NS; ++s) kofs[s] ^= STAGE;
  int t = 0;
  for (; t + 1 < tiles; ++t) {
    step(std::integral_constant<bool, false>(), t);
#pragma unroll
    for (int s = 0; s < NS; ++s) kofs[s] ^= STAGE;
#pragma unroll
    for (int d = 0; d < ND; ++d) vofs[d] ^= STAGE;
  }
  step(std::integral_constant<bool, true>(), t);

  // the wave's rows through its share of K's stages, which nobody reads in the last step, so that 16
  // bytes a lane leave in whole rows: HD / 8 lanes a row
  const float inv = 1.f / psum32(lrun);
  float zero[4] = {lrun * 0.f};   // not zero where a sum is not finite
  uint8_t* mem = smem + wave * 32 * ROWB;
  auto leave = [&](auto obf) __attribute__((always_inline)) {
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int r4 = 0; r4 < 4; ++r4) {
        const int c = 4 * d + r4;
#pragma unroll
        for (int e = 0; e < 4; ++e) zero[e] = __builtin_fmaf(o[d][4 * r4 + e], 0.f, zero[e]);
        *(u32x2*)(mem + lo * ROWB + ((c ^ (HD == 128 ? lo & 15 : (lo >> 1) & 7)) << 4) + 8 * hi) =
            u32x2{pack_out<BF>(o[d][4 * r4] * inv, o[d][4 * r4 + 1] * inv, decltype(obf)::value),
                  pack_out<BF>(o[d][4 * r4 + 2] * inv, o[d][4 * r4 + 3] * inv, decltype(obf)::value)};
      }
  };
  if (A.obf)
    leave(std::integral_constant<int, 1>());
  else
    leave(std::integral_constant<int, 0>());
#pragma unroll
  for (int i = 0; i < 32 / RI; ++i) {
    const int r = i * RI + lane / CH, c = lane % CH, gr = wave * 32 + r, rt = (int)(gr * A.magic >> 16), rh = gr - rt * A.hh;
    const u32x4 x = *(const u32x4*)(mem + r * ROWB + ((c ^ (HD == 128 ? r & 15 : (r >> 1) & 7)) << 4));
    if (rt < live && rh < heads)
      *(u32x4*)(A.out + (int64_t)(T.row0 + T.t0 + rt) * A.ldo + (int64_t)(kvh * A.group + chunk * A.hh + rh) * HD + 8 * c) = x;
  }
  const bool bad = !(zero[0] + zero[1] + zero[2] + zero[3] == 0.f);
  uint64_t redo = __ballot(bad && mine);
  for (uint32_t rows = (uint32_t)(redo | redo >> 32); rows; rows &= rows - 1) {
    const int r = wave * 32 + __builtin_ctz(rows), rt = (int)(r * A.magic >> 16);
    const int64_t rh = kvh * A.group + chunk * A.hh + r - rt * A.hh, at = T.row0 + T.t0 + rt;
    packed_row<BF, HD>(A.q + at * A.ldq + rh * HD, kbase, A.ldk, vbase, A.ldv, T.t0 + rt, A.scale,
                       A.out + at * A.ldo + rh * HD, A.obf);
  }
}

hipError_t attend_packed(hipStream_t s, const SeqTile* const* tiles, const int64_t* ntiles, int bf16, int heads,
                         int kv_heads, int head_dim, const uint16_t* q, int64_t ldq, const uint16_t* k, int64_t ldk,
                         const uint16_t* v, int64_t ldv, float scale, uint16_t* out, int obf, int64_t ldo) {
  if (ntiles[0] == 0) return hipSuccess;
  PackedArgs a;
  a.q = q;
  a.k = k;
  a.v = v;
  a.out = out;
  a.ldq = ldq;
  a.ldk = ldk;
  a.ldv = ldv;
  a.ldo = ldo;
  a.scale = scale * 1.4426950408889634f;
  a.kv_heads = kv_heads;
  a.group = heads / kv_heads;
  // up to 8 heads of a group share a tile: with groups of 4, 16 x 21..257 tokens 11.9 us, 2 at a time 13.2,
  // alone 15.0, and 4 x 1100..1180 60.8, 62.6, 66.0; with groups of 8 (64-wide), 24 x 5..4001 90, 4 at a
  // time 94, alone 98
  a.hh = a.group < 8 ? a.group : 8;
  a.chunks = (a.group + a.hh - 1) / a.hh;
  a.magic = (65536 + a.hh - 1) / a.hh;
  int z = 0;
  while (z + 1 < SEQ_TTS && (SEQ_TT0 << (z + 1)) * a.hh <= 128) ++z;
  a.tt = SEQ_TT0 << z;
  a.tiles = tiles[z];
  a.obf = obf;
  const int64_t groups = ntiles[z] * a.chunks * kv_heads;
  if (groups > WG256_MAX) return hipErrorInvalidConfiguration;
  auto go = [&](auto kern) { hipLaunchKernelGGL(kern, dim3((unsigned)groups), dim3(256), 0, s, a); };
  if (bf16 && obf)
    head_dim == 128 ? go(k_attend_packed<1, 128, 0>) : go(k_attend_packed<1, 64, 0>);
  else if (bf16)
    head_dim == 128 ? go(k_attend_packed<1, 128, 1>) : go(k_attend_packed<1, 64, 1>);
  else
    head_dim == 128 ? go(k_attend_packed<0, 128, 0>) : go(k_attend_packed<0, 64, 0>);
  return hipGetLastError();
}

}  // namespace exn
