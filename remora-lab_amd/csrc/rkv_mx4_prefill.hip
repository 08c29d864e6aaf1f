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

template <int D, bool kTwo>
__global__ __launch_bounds__(64 * kMx4PrefillWaves, 2) void mx4_prefill_kernel(PrefillLaunch pf) {
#if defined(__HIP_DEVICE_COMPILE__)
  using Pre = Mx4Wide<D, 2, kTwo, true>;
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
  if (r0 / G >= jn) return;  // (waves share nothing: no barrier waits for this one)

  __shared__ v8b qs[kMx4PrefillWaves][Pre::kQuery];
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
    pr.put_query(qs[r0 / 32], c, p.q, off, p.scale_log2 < 0.0f ? -1.0f : 1.0f);
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

  Mx4Place at(p, seq, kvh);
  mx4_walk<D>(pr, at, tok0, kTile, min(all, last), last, [] {});
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
