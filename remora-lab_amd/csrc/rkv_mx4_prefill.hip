// rkv_mx4_prefill.hip -- chunked prefill attention over 4-bit pages (rkv_mx4.h)
// for gfx950: the units, causal ranges, split plan and combine of
// rkv_prefill.hip with a kernel of its own.
//
// A workgroup of 4 waves takes a block of 128 query rows of one (entry, kv
// head), wave w rows 32w .. 32w+31 as two column groups of 16.  The waves
// share nothing: each walks the block's tiles by itself, up to the last
// position that its own rows attend, and loads them straight into registers
// (the other waves' loads of the same tile come from the CU's L1 or the L2).
//   QK: bf16 16x16x32 on K codes widened with their scales, exact.
//   PV: f16 16x16x32 on V codes times their scales, exact in f16 too, and held
//     times 2^6: 2^-17 to 6 * 2^13 (the product of a subnormal f16 keeps the
//     bits that its unnormalised exponent leaves: without the 2^6 V of 3e-7
//     came out 1.3e-5 off).  One product of the weights cut to f16 for bf16
//     rows (11 bits: 1.4e-4 of a row beside the 1.7e-3 of its own rounding),
//     two for f32 rows (22 bits).
// The scales cost a multiplication per widened V value and none per weight:
// 64 packed products a tile for all 32 rows at head_dim 256.
#include <algorithm>

#include "rkv_mx4_attn.h"

namespace rkv {
namespace {

constexpr int kMx4PrefillWaves = 4;

#if defined(__HIP_DEVICE_COMPILE__)
template <int D, bool kTwo>
struct Mx4Prefill {
  static constexpr int H = D / 128, NB = D / 32, G = 2;
  using Query = Mx4Query<D, false, true>;
  using Tile = Mx4Tile<D, true>;

  // the query operand of (group, half, step) at 64 lanes * 16 bytes each
  const __attribute__((address_space(3))) v8b *q;
  __attribute__((address_space(3))) uint8_t *vsc;  // the tile's D bytes of V scales, the wave's own
  v4f acc[G][D / 16];  // acc[2b + odd][i]: dim 32*b + 8*lg + 2*i + odd of column li
  float M[G], l[G];
  float mul;
  int32_t rlim[G];     // positions that the lane's row attends
  int32_t end;         // positions that any of the wave's rows attends
  int lane, li, lg;

  template <bool kMasked>
  __device__ __forceinline__ void compute(Tile &t, int32_t tok, const uint8_t *next, uint64_t region) {
    v4f sc[G][2];
#pragma unroll
    for (int g = 0; g < G; ++g) sc[g][0] = sc[g][1] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int h = 0; h < H; ++h) {
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        v8b b[G];
#pragma unroll
        for (int g = 0; g < G; ++g) b[g] = q[((g * H + h) * 4 + u) * 64 + lane];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const float scale = __builtin_bit_cast(float, (t.ks >> (8 * (j * H + h)) & 0xffu) << 23);
          const v8b a = mx4_widen_k((uint32_t)t.kc[j * H + h][u], scale);
#pragma unroll
          for (int g = 0; g < G; ++g)
            sc[g][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b[g], sc[g][j], 0, 0, 0);
        }
      }
    }
    if (next != nullptr) t.load_k(next, lane);
    v8h w[G][kTwo ? 2 : 1];
    float x[G][8];
    bool high = false;
#pragma unroll
    for (int g = 0; g < G; ++g) {
      const int32_t live = rlim[g] - tok - 8 * lg;
      float top = kNoMax;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        x[g][i] = sc[g][i / 4][i % 4];
        if constexpr (kMasked) x[g][i] = i < live ? x[g][i] : -INFINITY;
        top = fmaxf(top, x[g][i]);
      }
      high = high || __builtin_fmaf(top, mul, -M[g]) > 15.0f;
    }
    if (__ballot(high) != 0) rescale(x);
    const v2h one = {(_Float16)1.0f, (_Float16)1.0f};
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(x[g][2 * i], mul, -M[g]));
        const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(x[g][2 * i + 1], mul, -M[g]));
        const v2h hi = __builtin_bit_cast(v2h, __builtin_amdgcn_cvt_pkrtz(p0, p1));
        w[g][0][2 * i] = hi[0];
        w[g][0][2 * i + 1] = hi[1];
        l[g] = __builtin_amdgcn_fdot2(hi, one, l[g], false);
        if constexpr (kTwo) {
          const v2h lo = __builtin_bit_cast(v2h, __builtin_amdgcn_cvt_pkrtz(p0 - (float)hi[0], p1 - (float)hi[1]));
          w[g][1][2 * i] = lo[0];
          w[g][1][2 * i + 1] = lo[1];
          l[g] = __builtin_amdgcn_fdot2(lo, one, l[g], false);
        }
      }
    // every lane's word of the V scales to LDS, its group's blocks from there
    // (a wave's LDS accesses run in order)
    if constexpr (H == 2) *reinterpret_cast<__attribute__((address_space(3))) uint32_t *>(vsc + 4 * lane) = t.vmax;
    else *reinterpret_cast<__attribute__((address_space(3))) uint16_t *>(vsc + 2 * lane) = (uint16_t)t.vmax;
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    const uint32_t keep0 = mx4_keep(end - tok - 8 * lg), keep1 = mx4_keep(end - tok - 8 * lg - 4);
    if constexpr (kMasked) drop_nan(tok, keep0, keep1);
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      const v2u sw = scales(b);
      uint32_t s0 = sw[0], s1 = sw[1];
      if constexpr (kMasked) {  // what lies behind the rows' tokens is nobody's
        s0 &= keep0;
        s1 &= keep1;
      }
      const v8h m = mx4_v_scales(s0, s1);
#pragma unroll
      for (int odd = 0; odd < 2; ++odd) {
        const int dt = 2 * b + odd;
        const v8h a = mx4_widen_v((uint32_t)t.vc[dt / 4][dt % 4], 0x1p-2f) * m;  // V times 2^6
#pragma unroll
        for (int g = 0; g < G; ++g)
#pragma unroll
          for (int k = 0; k < (kTwo ? 2 : 1); ++k)
            acc[g][dt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, w[g][k], acc[g][dt], 0, 0, 0);
      }
    }
    if (next != nullptr) t.load_v(next + region, lane);
  }

  // Bytes of the V scales of block b for the lane's 8 tokens.
  __device__ __forceinline__ v2u scales(int b) const {
    return *reinterpret_cast<const __attribute__((address_space(3))) v2u *>(vsc + 8 * NB * lg + 8 * b);
  }

  // A masked tile with NaN V blocks: rows that attend one get NaN in its
  // dims, and the block's scale goes to 0 for the rows that do not (a weight
  // of 0 times NaN is NaN).
  __device__ __forceinline__ void drop_nan(int32_t tok, uint32_t keep0, uint32_t keep1) {
    auto nans = [](uint32_t s) { return ((s | 0x80808080u) - 0x7c7c7c7cu) & 0x80808080u; };  // bytes of 0x7c and more
    uint32_t any = 0;
#pragma unroll
    for (int b = 0; b < NB; ++b) any |= nans(scales(b)[0] & keep0) | nans(scales(b)[1] & keep1);
    if (__ballot(any != 0) == 0) return;
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      const v2u s = scales(b);
      const uint32_t n0 = nans(s[0] & keep0), n1 = nans(s[1] & keep1);
#pragma unroll
      for (int g = 0; g < G; ++g) {
        const int32_t live = rlim[g] - tok - 8 * lg;
        int hit = ((n0 & mx4_keep(live)) | (n1 & mx4_keep(live - 4))) != 0u;
        hit |= __shfl_xor(hit, 16);
        hit |= __shfl_xor(hit, 32);
        const float add = hit ? __builtin_nanf("") : 0.0f;
        acc[g][2 * b] += add;
        acc[g][2 * b + 1] += add;
      }
      // (every lane of the group holds and writes the same bytes)
      *reinterpret_cast<__attribute__((address_space(3))) v2u *>(vsc + 8 * NB * lg + 8 * b) =
          v2u{s[0] & ~((n0 >> 7) * 0xffu), s[1] & ~((n1 >> 7) * 0xffu)};
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }

  // A score outgrew 2^15 over its row's M: the rows' new M puts their largest
  // at 2^11, and the sums go into its units.
  __device__ __forceinline__ void rescale(const float (&x)[G][8]) {
#pragma unroll
    for (int g = 0; g < G; ++g) {
      float top = x[g][0];
#pragma unroll
      for (int i = 1; i < 8; ++i) top = fmaxf(top, x[g][i]);
      top = fmaxf(top, __shfl_xor(top, 16));
      top = fmaxf(top, __shfl_xor(top, 32));
      float n = __builtin_fmaf(top, mul, -11.0f);
      if (!(n > M[g])) n = M[g];
      const float f = __builtin_amdgcn_exp2f(M[g] - n);
      M[g] = n;
      l[g] *= f;
#pragma unroll
      for (int i = 0; i < D / 16; ++i) acc[g][i] *= f;
    }
  }
};
#endif  // __HIP_DEVICE_COMPILE__

template <int D, bool kTwo>
__global__ __launch_bounds__(64 * kMx4PrefillWaves, 2) void mx4_prefill_kernel(PrefillLaunch pf) {
#if defined(__HIP_DEVICE_COMPILE__)
  using Pre = Mx4Prefill<D, kTwo>;
  const DecodeLaunch &p = pf.d;
  const Geo g = p.g;
  // the workgroup's unit (see prefill_kernel)
  const uint32_t C = (uint32_t)max(pf.xcd_chunk, 1);
  const uint32_t xcd = blockIdx.x & 7u, slot = blockIdx.x >> 3;
  const int64_t x = ((int64_t)xcd + 8 * (int64_t)(slot / C)) * C + slot % C;
  const int32_t heads = g.kv_heads;
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
  if (r0 / G >= jn) return;  // (waves share nothing: no barrier waits for this one)

  __shared__ v8b qs[kMx4PrefillWaves][2 * 4 * Pre::H * 64];
  Pre pr;
  __shared__ __attribute__((aligned(16))) uint8_t vscs[kMx4PrefillWaves][D];
  pr.q = (const __attribute__((address_space(3))) v8b *)qs[r0 / 32];
  pr.vsc = (__attribute__((address_space(3))) uint8_t *)vscs[r0 / 32];
  pr.lane = lane;
  pr.li = li;
  pr.lg = lg;
  pr.mul = fmaxf(fabsf(p.scale_log2), 1.17549435e-38f);
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    const int r = r0 + 16 * c + li, jl = r / G;
    const int64_t off =
        jl < jn ? ((int64_t)(pf.qoff[e] + j0 + jl) * p.q_heads + kvh * G + r % G) * D : -1;
    typename Pre::Query q;
    q.load(p.q, off, p.scale_log2 < 0.0f ? -1.0f : 1.0f, false, lg);
#pragma unroll
    for (int i = 0; i < 4 * Pre::H; ++i) qs[r0 / 32][(c * 4 * Pre::H + i) * 64 + lane] = q.b[0][i / 4][i % 4];
    pr.rlim[c] = jl < jn ? ctx + j0 + jl + 1 : 0;
    pr.M[c] = kNoMax;
    pr.l[c] = 0.0f;
#pragma unroll
    for (int i = 0; i < D / 16; ++i) pr.acc[c][i] = v4f{0.f, 0.f, 0.f, 0.f};
  }
  // positions attended by all, and by any, of the wave's rows
  const int32_t all = ctx + j0 + r0 / G + 1;
  pr.end = ctx + j0 + min((r0 + 31) / G, jn - 1) + 1;
  const int32_t last = min(tok_end, pr.end);

  const uint64_t PB = mx4_page_bytes(g), RB = mx4_region_bytes(g);
  const uint8_t *base = p.pages + (uint64_t)kvh * 2u * RB;
  const int32_t *bt = p.bt + (int64_t)seq * p.bt_stride;
  bool bad = false;
  auto place = [&](int32_t tok) -> const uint8_t * {
    int32_t page = bt[tok / g.page_tokens];
    if (page < 0 || page >= g.num_pages) {
      bad = true;
      page = 0;
    }
    return base + (uint64_t)page * PB + (uint64_t)(tok % g.page_tokens / kTile) * mx4_tile_bytes(D);
  };
  typename Pre::Tile t;
  if (tok0 < last) {
    const uint8_t *at = place(tok0);
    t.load_k(at, lane);
    t.load_v(at + RB, lane);
    // two loops and not one with a choice: each keeps the sums in place
    int32_t tok = tok0;
    const int32_t whole = min(all, last);
    for (; tok + kTile <= whole; tok += kTile) {
      at = tok + kTile < last ? place(tok + kTile) : nullptr;
      pr.template compute<false>(t, tok, at, RB);
    }
    for (; tok < last; tok += kTile) {
      at = tok + kTile < last ? place(tok + kTile) : nullptr;
      pr.template compute<true>(t, tok, at, RB);
    }
  }
  if (bad && lane == 0) atomicOr(p.fault, FAULT_BAD_PAGE);

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
