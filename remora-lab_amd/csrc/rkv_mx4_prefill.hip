// rkv_mx4_prefill.hip -- chunked prefill attention over 4-bit pages (rkv_mx4.h)
// for gfx950: the units, causal ranges and combine of rkv_prefill.hip with a
// kernel of its own.
//
// A workgroup of 4 waves takes a block of 128 query rows of one (entry, kv
// head), wave w rows 32w .. 32w+31 as two column groups of 16, and walks the
// block's tiles of 32 tokens.
//   QK: bf16 16x16x32 on K codes widened with their scales, exact.  Each wave
//     loads the tile's K codes (the CU's L1 serves four of them) and widens
//     them itself.
//   PV: f16 16x16x32 on V codes times their scales, exact in f16 too, and held
//     times 2^6: 2^-17 to 6 * 2^13 (the product of a subnormal f16 keeps the
//     bits that its unnormalised exponent leaves: without the 2^6 V of 3e-7
//     came out 1.3e-5 off).  One product of the weights cut to f16 for bf16
//     rows (11 bits: 1.4e-4 of a row beside the 1.7e-3 of its own rounding),
//     two for f32 rows (22 bits).  V costs a conversion and a multiplication a
//     pair, so each wave widens a quarter of the next tile's into LDS, in two
//     buffers, one barrier a tile.
// Bound by issue: besides a 16-cycle matrix instruction a SIMD issues about two
// others, from either of its two waves, and each further one costs 4.6 cycles.
// A wave's tile takes 96 matrix instructions for f32 rows (64 for bf16) and 237
// others at head_dim 256, counted; widening V in every wave took 357 (804 us
// for the first case below).  The queries' first half stays in registers and the second
// in LDS: both in LDS leave no room for two workgroups a CU, both in registers
// spill.
// Measured (2 kv heads of 256, 8 query heads each): eight chunks of 512 rows
// after 8192 tokens 694 us with f32 rows (817 TFLOP/s), 552 with bf16 rows
// (1028); six chunks of 173..567 rows, 6 query heads on 4, after 422..2954
// tokens 150 (691).
// Not faster: 64 rows a wave, one wave a SIMD (979).
#include <algorithm>
#include <type_traits>

#include "rkv_mx4_attn.h"

namespace rkv {
namespace {

constexpr int kMx4PrefillWaves = 4;

#if defined(__HIP_DEVICE_COMPILE__)
typedef uint8_t __attribute__((address_space(3))) lds_u8;

// A wave's 32 rows of the block, and its part of the widening: D/64 of the
// tile's D/16 V operands.
template <int D, bool kTwo>
struct Mx4Block : Mx4Rows<D, 2, kTwo> {
  using Rows = Mx4Rows<D, 2, kTwo>;
  using Rows::acc, Rows::rlim, Rows::lane, Rows::li, Rows::lg;
  static constexpr int H = D / 128, NB = D / 32, kOwn = D / 64;
  static constexpr int kOwnBlocks = kOwn / 2;

  v8b q0[2][4];                                    // half 0 of the query operand
  const __attribute__((address_space(3))) v8b *q1; // half 1, [group][step][lane], the wave's own
  __attribute__((address_space(3))) v8h *vs;       // [2 tiles][D/16][lane] widened V
  lds_u8 *nan;                                     // [2 tiles][group of 8 tokens][NB] NaN blocks, a bit a token
  v4i kc[2 * H];                                   // K codes of (j, h) and their scales
  uint32_t ks;
  uint32_t vc[kOwn];                               // the wave's V codes of the next tile,
  uint32_t vb[2 * kOwnBlocks];                     // and their scales
  int wave;
  int32_t whole, end;                              // positions attended by all, and by any, of the block's rows

  __device__ __forceinline__ void load_k(const uint8_t *k) {
#pragma unroll
    for (int i = 0; i < 2 * H; ++i) kc[i] = load16_nt(k + 1024 * i + 16 * lane);
    if constexpr (H == 2) ks = *reinterpret_cast<const uint32_t *>(k + 16 * D + 4 * lane);
    else ks = *reinterpret_cast<const uint16_t *>(k + 16 * D + 2 * lane);
  }
  __device__ __forceinline__ void load_v(const uint8_t *v) {
    const uint8_t *s = v + 16 * D + 8 * (NB * lg + kOwnBlocks * wave);
    if constexpr (D == 256) {
      const v4i c = *reinterpret_cast<const v4i *>(v + 1024 * wave + 16 * lane), x = *reinterpret_cast<const v4i *>(s);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        vc[i] = (uint32_t)c[i];
        vb[i] = (uint32_t)x[i];
      }
    } else {
      const v2u c = *reinterpret_cast<const v2u *>(v + 1024 * (wave / 2) + 16 * lane + 8 * (wave & 1)),
                x = *reinterpret_cast<const v2u *>(s);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        vc[i] = c[i];
        vb[i] = x[i];
      }
    }
  }

  // The wave's part of the tile at tok to LDS.  In a tile that some rows
  // attend in part, NaN blocks go in as zeros beside their bits (a weight of 0
  // times NaN is NaN), and tokens behind the block's as zeros.
  __device__ __forceinline__ void widen(int buf, int32_t tok) {
    const bool masked = tok + kTile > whole;
#pragma unroll
    for (int bb = 0; bb < kOwnBlocks; ++bb) {
      const int b = kOwnBlocks * wave + bb;
      uint32_t s0 = vb[2 * bb], s1 = vb[2 * bb + 1];
      if (masked) {
        s0 &= mx4_keep(end - tok - 8 * lg);
        s1 &= mx4_keep(end - tok - 8 * lg - 4);
        const uint32_t n0 = mx4_nans(s0), n1 = mx4_nans(s1);
        s0 &= ~((n0 >> 7) * 0xffu);
        s1 &= ~((n1 >> 7) * 0xffu);
        auto bits = [](uint32_t n) { return (n >> 7 & 1u) | (n >> 14 & 2u) | (n >> 21 & 4u) | (n >> 28 & 8u); };
        if (li == 0)
          nan[(4 * buf + lg) * NB + b] = (uint8_t)(bits(n0) | bits(n1) << 4);
      }
      const v8h m = mx4_v_scales(s0, s1);
#pragma unroll
      for (int odd = 0; odd < 2; ++odd)
        vs[((D / 16) * buf + 2 * b + odd) * 64 + lane] = mx4_widen_v(vc[2 * bb + odd], 0x1p-2f) * m;  // V times 2^6
    }
  }

  // The tile at tok, K in registers and V in buffer buf; the next one's K at
  // `next` (NULL: none) and the V of the one after it at `after`.
  template <bool kMasked>
  __device__ __forceinline__ void compute(int buf, int32_t tok, const uint8_t *next, const uint8_t *after) {
    // the tile's V is whole, and nobody reads the one before it
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
    v4f sc[2][2];
#pragma unroll
    for (int g = 0; g < 2; ++g) sc[g][0] = sc[g][1] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int h = 0; h < H; ++h)
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        v8b b[2];
#pragma unroll
        for (int g = 0; g < 2; ++g) b[g] = h == 0 ? q0[g][u] : q1[(4 * g + u) * 64 + lane];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const float scale = __builtin_bit_cast(float, (ks >> (8 * (j * H + h)) & 0xffu) << 23);
          const v8b a = mx4_widen_k((uint32_t)kc[j * H + h][u], scale);
#pragma unroll
          for (int g = 0; g < 2; ++g) sc[g][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b[g], sc[g][j], 0, 0, 0);
        }
      }
    if (next != nullptr) {
      load_k(next);
      widen(buf ^ 1, tok + kTile);
      if (after != nullptr) load_v(after);
    }
    v8h w[2][Rows::kTerms];
    Rows::template weights<kMasked>(sc, tok, w);
    if constexpr (kMasked) add_nan(buf, tok);
    // each step's V operands are on their way during the step before
    v8h a[2][2];
    auto load = [&](int s) {
#pragma unroll
      for (int i = 0; i < 2; ++i) a[s & 1][i] = vs[((D / 16) * buf + 2 * s + i) * 64 + lane];
    };
    load(0);
#pragma unroll
    for (int s = 0; s < NB; ++s) {
      if (s + 1 < NB) load(s + 1);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int k = 0; k < Rows::kTerms; ++k)
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int g = 0; g < 2; ++g)
            acc[g][2 * s + i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a[s & 1][i], w[g][k], acc[g][2 * s + i], 0, 0, 0);
    }
  }

  // Rows that attend a NaN V block of a masked tile get NaN in its dims.
  __device__ __forceinline__ void add_nan(int buf, int32_t tok) {
    const lds_u8 *mine = nan + (4 * buf + lg) * NB;
    uint32_t any = 0;
#pragma unroll
    for (int b = 0; b < NB; b += 4) any |= *reinterpret_cast<const __attribute__((address_space(3))) uint32_t *>(mine + b);
    if (__ballot(any != 0) == 0) return;
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      const uint32_t n = mine[b];
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        const int32_t live = min(max(rlim[g] - tok - 8 * lg, 0), 8);
        int hit = (n & ((1u << live) - 1u)) != 0u;
        hit |= __shfl_xor(hit, 16);
        hit |= __shfl_xor(hit, 32);
        const float add = hit ? __builtin_nanf("") : 0.0f;
        acc[g][2 * b] += add;
        acc[g][2 * b + 1] += add;
      }
    }
  }
};
#endif  // __HIP_DEVICE_COMPILE__

// Three waves a SIMD at head_dim 128, for 20 bytes of scratch a lane (eight
// chunks of 1344 rows of 24 heads after 3000 tokens 648 us, with two 796).
template <int D, bool kTwo>
__global__ __launch_bounds__(64 * kMx4PrefillWaves, D == 128 ? 3 : 2) void mx4_prefill_kernel(PrefillLaunch pf) {
#if defined(__HIP_DEVICE_COMPILE__)
  using Pre = Mx4Block<D, kTwo>;
  const DecodeLaunch &p = pf.d;
  // the workgroup's unit (see prefill_kernel)
  const uint32_t C = (uint32_t)max(pf.xcd_chunk, 1);
  const uint32_t xcd = blockIdx.x & 7u, slot = blockIdx.x >> 3;
  const int64_t x = ((int64_t)xcd + 8 * (int64_t)(slot / C)) * C + slot % C;
  const int32_t heads = p.g.kv_heads;
  if (x >= (int64_t)pf.first[pf.n_entries] * heads) return;
  int e = 0;
  while (e + 1 < pf.n_entries && x >= (int64_t)pf.first[e + 1] * heads) ++e;
  const int32_t ns = pf.nseg[e];
  const int32_t nb = (pf.first[e + 1] - pf.first[e]) / ns;
  const int32_t v = (int32_t)(x - (int64_t)pf.first[e] * heads);
  const int32_t sg = v / (heads * nb);
  const int kvh = (v / nb) % heads;
  const int32_t rb = nb - 1 - v % nb;
  const int32_t seq = pf.seq[e], ctx = pf.ctx[e], n = pf.rows[e];
  const int32_t j0 = pf.tq * rb;
  const int32_t jn = min(pf.tq, n - j0);
  const int32_t len = ctx + j0 + jn;
  const int32_t tok0 = min(sg * pf.seg[e], len);
  const int32_t tok_end = ns == 1 ? len : min(len, tok0 + pf.seg[e]);

  const int lane = threadIdx.x & 63, li = lane & 15, lg = lane >> 4;
  const int r0 = 32 * (int)__builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int32_t G = p.q_heads / heads;

  __shared__ v8h vs[2][D / 16][64];
  __shared__ v8b qs[kMx4PrefillWaves][D == 256 ? 2 * 4 * 64 : 1];
  __shared__ uint32_t nans[2][4][Pre::NB / 4];
  Pre pr;
  pr.vs = (__attribute__((address_space(3))) v8h *)&vs[0][0][0];
  pr.q1 = (const __attribute__((address_space(3))) v8b *)qs[r0 / 32];
  pr.nan = (lds_u8 *)&nans[0][0][0];
  pr.wave = r0 / 32;
  pr.lane = lane;
  pr.li = li;
  pr.lg = lg;
  pr.mul = fmaxf(fabsf(p.scale_log2), 1.17549435e-38f);
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    const int r = r0 + 16 * c + li, jl = r / G;
    const int64_t off =
        jl < jn ? ((int64_t)(pf.qoff[e] + j0 + jl) * p.q_heads + kvh * G + r % G) * D : -1;
    Mx4Query<D, false, true> x;
    x.load(p.q, off, p.scale_log2 < 0.0f ? -1.0f : 1.0f, false, lg);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      pr.q0[c][u] = x.b[0][0][u];
      if constexpr (D == 256) qs[r0 / 32][(4 * c + u) * 64 + lane] = x.b[0][1][u];
    }
    pr.rlim[c] = jl < jn ? ctx + j0 + jl + 1 : 0;
    pr.M[c] = kNoMax;
    pr.l[c] = 0.0f;
#pragma unroll
    for (int i = 0; i < D / 16; ++i) pr.acc[c][i] = v4f{0.f, 0.f, 0.f, 0.f};
  }
  pr.whole = ctx + j0 + 1;
  pr.end = len;

  // every wave walks every tile of the block; a tile's V is widened while the
  // one before it is worked on
  Mx4Place at(p, seq, kvh);
  if (tok0 < tok_end) {
    const uint8_t *k = at.tile<D>(tok0);
    pr.load_k(k);
    pr.load_v(k + at.region);
    const uint8_t *next = tok0 + kTile < tok_end ? at.tile<D>(tok0 + kTile) : nullptr;
    pr.widen(0, tok0);
    if (next != nullptr) pr.load_v(next + at.region);
    int buf = 0;
    int32_t tok = tok0;
    auto step = [&](auto masked) {
      const uint8_t *after = tok + 2 * kTile < tok_end ? at.tile<D>(tok + 2 * kTile) : nullptr;
      pr.template compute<decltype(masked)::value>(buf, tok, next, after != nullptr ? after + at.region : nullptr);
      next = after;
      buf ^= 1;
      tok += kTile;
    };
    while (tok < tok_end && tok + kTile <= pr.whole) step(std::false_type{});
    while (tok < tok_end) step(std::true_type{});
  }
  if (at.bad && lane == 0) atomicOr(p.fault, FAULT_BAD_PAGE);

#pragma unroll
  for (int c = 0; c < 2; ++c) {
    float l = pr.l[c];
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    const int r = r0 + 16 * c + li, jl = r / G;
    if (jl >= jn) continue;
    const int64_t erow = (int64_t)(j0 + jl) * p.q_heads + kvh * G + r % G;
    const bool part = ns > 1;
    const int64_t prow = pf.wsoff[e] + erow * ns + sg;
    const int64_t orow = (int64_t)pf.qoff[e] * p.q_heads + erow;
    const float inv = 0x1p-6f * (part ? 1.0f : l == 0.0f ? 0.0f : 1.0f / l);
#pragma unroll
    for (int b = 0; b < Pre::NB; ++b) {
      const v4f ev = pr.acc[c][2 * b] * inv, od = pr.acc[c][2 * b + 1] * inv;
      const int d0 = 32 * b + 8 * lg;
      const v4f o0 = {ev[0], od[0], ev[1], od[1]}, o1 = {ev[2], od[2], ev[3], od[3]};
      if (part) {
        *reinterpret_cast<v4f *>(pf.ws_o + prow * D + d0) = o0;
        *reinterpret_cast<v4f *>(pf.ws_o + prow * D + d0 + 4) = o1;
      } else if (p.out_bf16 != 0) {
        v8b w;
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = (__bf16)(i & 1 ? od[i / 2] : ev[i / 2]);
        *reinterpret_cast<v8b *>(static_cast<uint16_t *>(p.out) + orow * D + d0) = w;
      } else {
        *reinterpret_cast<v4f *>(static_cast<float *>(p.out) + orow * D + d0) = o0;
        *reinterpret_cast<v4f *>(static_cast<float *>(p.out) + orow * D + d0 + 4) = o1;
      }
    }
    // (the combine takes a row whose l is not above 0 for empty)
    if (part && lg == 0)
      *reinterpret_cast<float2 *>(pf.ws_ml + 2 * prow) =
          l == 0.0f ? float2{-INFINITY, 0.0f} : l != l ? float2{0.0f, 1.0f} : float2{pr.M[c], l};
  }
#endif  // __HIP_DEVICE_COMPILE__
}

}  // namespace

hipError_t launch_mx4_prefill(const PrefillLaunch &pf, hipStream_t s) {
  if (pf.n_entries <= 0 || pf.first[pf.n_entries] <= 0) return hipSuccess;
  const int64_t units = (int64_t)pf.first[pf.n_entries] * pf.d.g.kv_heads;
  const int64_t round = 8 * (int64_t)std::max(pf.xcd_chunk, 1);
  const dim3 grid((unsigned)((units + round - 1) / round * round)), block(64 * kMx4PrefillWaves);
  const bool two = pf.d.out_bf16 == 0;
  if (pf.d.g.head_dim == 256) {
    if (two) hipLaunchKernelGGL((mx4_prefill_kernel<256, true>), grid, block, 0, s, pf);
    else hipLaunchKernelGGL((mx4_prefill_kernel<256, false>), grid, block, 0, s, pf);
  } else {
    if (two) hipLaunchKernelGGL((mx4_prefill_kernel<128, true>), grid, block, 0, s, pf);
    else hipLaunchKernelGGL((mx4_prefill_kernel<128, false>), grid, block, 0, s, pf);
  }
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? launch_prefill_combine(pf, s) : e;
}

}  // namespace rkv
