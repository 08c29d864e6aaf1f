// rkv_mx4_decode.hip -- paged flash-decode attention over 4-bit pages
// (rkv_mx4.h) for gfx950: GQA, causal multi-query verify, split-K partitions
// with the combine of rkv_decode.hip.
//
// For every row r of a kv head (q_len * q_heads/kv_heads of them, up to 32):
//   s_t = scale * q_r . k_t,  o_r = sum_t 2^(s_t - M) v_t / sum_t 2^(s_t - M)
// in base 2 (scale * log2 e folded into s), M following the largest s lazily.
//
// A workgroup of NW waves takes a partition of one entry and kv head; its
// waves take 32-token tiles in turn and merge at the end through LDS, so a
// short context needs neither partials nor a second launch.  Everything a
// tile needs comes straight from memory into the registers of the matrix
// instructions in whole 1 KiB loads, one tile ahead; LDS is only the merge.
//
//   QK: bf16 16x16x32, A = K codes widened with their power of two (exact in
//     bf16, one instruction for two), B = the query, an f32 one as three bf16
//     terms; products are exact and summed in f32.  Up to 8 rows columns 8-15
//     hold the rows again (f32: their second terms).  (The scaled E2M1 x E4M3
//     product needs no widening, but keeps only about 13 bits below its
//     largest term: with channels eight times the others the outputs of 32k
//     tokens were off by 1.5e-5, 2e-6 in f32.)
//   PV: f16 16x16x32, A = V codes widened (exact, one instruction for two),
//     B = p * 2^e_v as two f16 terms, p = hi + lo to 22 bits, both times the
//     block's power of two (exact).  Up to 8 rows lo takes columns 8-15.
//
// f16 range: M is kept so that p * 2^e_v <= 2^15, i.e. with vcap the largest V
// exponent met (at least 2^0 in the units of the stored byte) the row maximum
// maps to 2^(11 - vcap) and may rise by 2^4 before the sums are rescaled.
#include <algorithm>

#include "rkv_mx4_attn.h"

namespace rkv {
namespace {

#if defined(__HIP_DEVICE_COMPILE__)

// NG: 0: up to 8 rows (the second terms in columns 8-15), 1: up to 16, 2: up
// to 32 (two column groups).
template <int D, int NG, bool kBf16, int NW>
struct Mx4Decoder {
  static constexpr int H = D / 128, NB = D / 32;
  static constexpr bool kSplit = NG == 0;
  static constexpr int G = NG == 2 ? 2 : 1;  // column groups
  using Query = Mx4Query<D, kSplit, kBf16>;
  using Tile = Mx4Tile<D>;

  Query q[G];
  v4f acc[G][D / 16];  // acc[2b + odd][i]: dim 32*b + 8*lg + 2*i + odd of column li
  float M[G], l[G];
  float mul;           // |scale| * log2 e
  int32_t rlim[G];     // positions that the lane's row attends
  int32_t vcap;        // exponent of the largest V scale met, in the stored byte's units, >= 0
  float losel;         // kSplit: -1 in the columns of the second term
  int32_t end;         // tokens of the partition's entry that are live up to here
  int lane, li, lg;

  // The tile at position tok, held in t; the wave's next one, at `next` (NULL:
  // none), is loaded into t's registers as they come free.
  template <bool kMasked>
  __device__ __forceinline__ void compute(Tile &t, int32_t tok, const uint8_t *next, uint64_t region) {
    v8h w[G][kSplit ? 1 : 2];  // the tokens' weights: first terms (kSplit: by column), second terms
    uint32_t keep[G][2];       // masked tiles: bytes of the live tokens' V scales
    float x[G][8];
    v4f sc[G][2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
#pragma unroll
      for (int g = 0; g < G; ++g) sc[g][j] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int h = 0; h < H; ++h) {
        const float scale = __builtin_bit_cast(float, (t.ks >> (8 * (j * H + h)) & 0xffu) << 23);
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const uint32_t c = (uint32_t)t.kc[j * H + h][u];
          const v8b a = mx4_widen_k(c, scale);
#pragma unroll
          for (int g = 0; g < G; ++g)
#pragma unroll
            for (int s = Query::kSets - 1; s >= 0; --s)
              sc[g][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, q[g].b[s][h][u], sc[g][j], 0, 0, 0);
        }
      }
    }
#pragma unroll
    for (int g = 0; g < G; ++g) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float a = sc[g][i / 4][i % 4];
        x[g][i] = kSplit && !kBf16 ? a + dpp_ror8(a) : a;
      }
      if constexpr (kMasked) {
        const int32_t live = min(max(rlim[g] - tok - 8 * lg, 0), 8);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[g][i] = i < live ? x[g][i] : -INFINITY;
        keep[g][0] = mx4_keep(live);
        keep[g][1] = mx4_keep(live - 4);
      }
    }
    if (next != nullptr) t.load_k(next, lane);
    // s - M of the largest score, and the V scales against vcap
    const uint32_t vmax = kMasked ? t.vmax & vlive(end - tok) : t.vmax;
    const uint32_t cap = (uint32_t)(4 * (vcap + 15)) * 0x01010101u;
    bool high = (((vmax | 0x80808080u) - cap - 0x01010101u) & 0x80808080u) != 0u;
#pragma unroll
    for (int g = 0; g < G; ++g) {
      float top = x[g][0];
#pragma unroll
      for (int i = 1; i < 8; ++i) top = fmaxf(top, x[g][i]);
      high = high || __builtin_fmaf(top, mul, -M[g]) > (float)(15 - vcap);
    }
    if (__ballot(high) != 0) rescale(vmax, x);
#pragma unroll
    for (int g = 0; g < G; ++g) {
      float p[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) p[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[g][i], mul, -M[g]));
      const v2h one = {(_Float16)1.0f, (_Float16)1.0f};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const v2h hi = __builtin_bit_cast(v2h, __builtin_amdgcn_cvt_pkrtz(p[2 * i], p[2 * i + 1]));
        const float m1 = kSplit ? losel : -1.0f;
        const float r0 = __builtin_fmaf((float)hi[0], m1, p[2 * i]);
        const float r1 = __builtin_fmaf((float)hi[1], m1, p[2 * i + 1]);
        const v2h lo = __builtin_bit_cast(v2h, __builtin_amdgcn_cvt_pkrtz(r0, r1));
        if constexpr (kSplit) {
          w[g][0][2 * i] = lo[0];
          w[g][0][2 * i + 1] = lo[1];
        } else {
          w[g][0][2 * i] = hi[0];
          w[g][0][2 * i + 1] = hi[1];
          w[g][1][2 * i] = lo[0];
          w[g][1][2 * i + 1] = lo[1];
          l[g] = __builtin_amdgcn_fdot2(hi, one, l[g], false);
        }
        l[g] = __builtin_amdgcn_fdot2(lo, one, l[g], false);
      }
    }
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      v8h ws[G][kSplit ? 1 : 2];
#pragma unroll
      for (int g = 0; g < G; ++g) {
        uint32_t s0 = (uint32_t)t.vs[b / 2][2 * (b & 1)], s1 = (uint32_t)t.vs[b / 2][2 * (b & 1) + 1];
        if constexpr (kMasked) {
          s0 &= keep[g][0];
          s1 &= keep[g][1];
        }
        const v8h mh = mx4_v_scales(s0, s1);
#pragma unroll
        for (int k = 0; k < (kSplit ? 1 : 2); ++k) ws[g][k] = w[g][k] * mh;
      }
#pragma unroll
      for (int odd = 0; odd < 2; ++odd) {
        const int dt = 2 * b + odd;
        const uint32_t c = (uint32_t)t.vc[dt / 4][dt % 4];
        const v8h a = mx4_widen_v(c, 1.0f);
#pragma unroll
        for (int g = 0; g < G; ++g)
#pragma unroll
          for (int k = 0; k < (kSplit ? 1 : 2); ++k)
            acc[g][dt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, ws[g][k], acc[g][dt], 0, 0, 0);
      }
    }
    if (next != nullptr) t.load_v(next + region, lane);
  }

  // The bytes of vmax that belong to the tile's first n tokens: what a page
  // holds behind them is nobody's, and no result may follow it.
  __device__ __forceinline__ uint32_t vlive(int32_t n) const {
    constexpr int kPer = H == 2 ? 4 : 2;  // tokens of a lane, of group lane / 16
    return mx4_keep(min(n - 8 * lg - kPer * (lane % (8 / kPer)), kPer));
  }

  // A score or a V scale outgrew what M allows: the rows' new M, and the sums in its units.
  __device__ __forceinline__ void rescale(uint32_t v, const float (&x)[G][8]) {
    v = max(max(v & 0xffu, (v >> 8) & 0xffu), max((v >> 16) & 0xffu, v >> 24));
    // (a NaN scale's byte reads as 16; NaN outgrows no range)
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) v = max(v, (uint32_t)__shfl_xor((int)v, off));
    const int32_t cap = min(max((int32_t)(v >> 2) - 15, vcap), 15);
#pragma unroll
    for (int g = 0; g < G; ++g) {
      float top = x[g][0];
#pragma unroll
      for (int i = 1; i < 8; ++i) top = fmaxf(top, x[g][i]);
      top = fmaxf(top, __shfl_xor(top, 16));
      top = fmaxf(top, __shfl_xor(top, 32));
      // s_max * 2^(vcap - 11), and no lower than what held before
      float n = fmaxf(__builtin_fmaf(top, mul, (float)(cap - 11)), M[g] + (float)(cap - vcap));
      if (!(n > M[g])) n = M[g];  // (a row without a live token stays where it was)
      const float f = __builtin_amdgcn_exp2f(M[g] - n);
      M[g] = n;
      l[g] *= f;
#pragma unroll
      for (int i = 0; i < D / 16; ++i) acc[g][i] *= f;
    }
    vcap = cap;
  }
};
#endif  // __HIP_DEVICE_COMPILE__

template <int D, int NG, bool kBf16, int NW>
__global__ __launch_bounds__(64 * NW, NG == 2 || (NG == 1 && !kBf16) ? 1 : 2) void mx4_decode_kernel(DecodeLaunch p) {
#if defined(__HIP_DEVICE_COMPILE__)
  using Dec = Mx4Decoder<D, NG, kBf16, NW>;
  constexpr int kRows = NG == 0 ? 8 : 16 * Dec::G;
  constexpr int kStride = D + 4;  // floats between a row's sums in LDS
  __shared__ __attribute__((aligned(16))) float sums[NW][kRows][kStride];
  __shared__ float ms[NW][kRows], ls[NW][kRows];
  Dec dc;
  const int lane = threadIdx.x & 63;
  const int wave = (int)__builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int li = lane & 15, lg = lane >> 4;
  dc.lane = lane;
  dc.li = li;
  dc.lg = lg;
  const int kvh = blockIdx.y;
  const Geo g = p.g;

  int32_t pt, b, seq, lenc, part, nb;
  if (!locate(p, lane, (int32_t)blockIdx.x, pt, b, seq, lenc, part, nb, 1 << 24)) return;
  if (p.ws_hdr != nullptr && kvh == 0 && threadIdx.x == 0) {
    if (blockIdx.x == 0) p.ws_hdr[0] = pt;
    if (part == 0) {
      p.ws_hdr[1 + 2 * b] = (int32_t)blockIdx.x;
      p.ws_hdr[2 + 2 * b] = nb;
    }
  }
  int32_t len = lenc;
  if (seq < 0 || seq >= p.n_seqs) {
    if (threadIdx.x == 0) atomicOr(p.fault, FAULT_BAD_SEQ);
    len = 0;
  } else if (lenc == 0 && p.seq_lens[seq] != 0) {  // out of range: locate() takes it as 0
    if (threadIdx.x == 0) atomicOr(p.fault, FAULT_BAD_POSITION);
  } else if ((int64_t)len > (int64_t)p.bt_stride * g.page_tokens) {
    if (threadIdx.x == 0) atomicOr(p.fault, FAULT_BAD_POSITION);
    len = 0;
  }
  const int32_t tok0 = min(part * pt, len);
  const int32_t tok_end = part == nb - 1 ? len : min(len, tok0 + pt);

  const int32_t q_per_kv = p.q_heads / g.kv_heads;
  const int32_t R = p.q_len * q_per_kv;
  const float sign = p.scale_log2 < 0.0f ? -1.0f : 1.0f;
  // at least the smallest normal: a masked -inf times it stays -inf with a scale of 0
  dc.mul = fmaxf(fabsf(p.scale_log2), 1.17549435e-38f);
  dc.vcap = 0;
  dc.losel = li >= 8 ? -1.0f : 0.0f;
#pragma unroll
  for (int c = 0; c < Dec::G; ++c) {
    const int row = Dec::kSplit ? (li & 7) : 16 * c + li;
    const int j = row / q_per_kv;
    const int64_t off =
        row < R ? (((int64_t)b * p.q_len + j) * p.q_heads + kvh * q_per_kv + row % q_per_kv) * D : -1;
    dc.q[c].load(p.q, off, sign, Dec::kSplit && li >= 8, lg);
    dc.rlim[c] = row < R ? len - p.q_len + j + 1 : 0;
    dc.M[c] = kNoMax;
    dc.l[c] = 0.0f;
#pragma unroll
    for (int i = 0; i < D / 16; ++i) dc.acc[c][i] = v4f{0.f, 0.f, 0.f, 0.f};
  }
  dc.end = tok_end;
  const int32_t rlim_min = len - p.q_len + 1;  // positions that every row attends

  // ---- the wave's tiles: tok0 + 32*wave, then every NW-th -----------------
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
  typename Dec::Tile t;
  constexpr int32_t kStep = kTile * NW;
  int32_t tok = tok0 + kTile * wave;
  if (tok < tok_end) {
    const uint8_t *at = place(tok);
    t.load_k(at, lane);
    t.load_v(at + RB, lane);
    for (; tok < tok_end; tok += kStep) {
      at = tok + kStep < tok_end ? place(tok + kStep) : nullptr;
      if (tok + kTile > min(rlim_min, tok_end)) dc.template compute<true>(t, tok, at, RB);
      else dc.template compute<false>(t, tok, at, RB);
    }
  }
  if (bad && lane == 0) atomicOr(p.fault, FAULT_BAD_PAGE);

  // ---- merge of the waves -------------------------------------------------
#pragma unroll
  for (int c = 0; c < Dec::G; ++c) {
    float l = dc.l[c];
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    if constexpr (Dec::kSplit) {
      l += dpp_ror8(l);
#pragma unroll
      for (int i = 0; i < D / 16; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k) dc.acc[c][i][k] += dpp_ror8(dc.acc[c][i][k]);
    }
    const int row = 16 * c + li;
    if (row < kRows) {
      if (lg == 0) {
        ms[wave][row] = dc.M[c];
        ls[wave][row] = l;
      }
#pragma unroll
      for (int i = 0; i < Dec::NB; ++i) {
        const v4f e = dc.acc[c][2 * i], o = dc.acc[c][2 * i + 1];
        float *dst = &sums[wave][row][32 * i + 8 * lg];
        *reinterpret_cast<v4f *>(dst) = v4f{e[0], o[0], e[1], o[1]};
        *reinterpret_cast<v4f *>(dst + 4) = v4f{e[2], o[2], e[3], o[3]};
      }
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < R * (D / 4); i += 64 * NW) {
    const int row = i / (D / 4), d0 = 4 * (i % (D / 4));
    float m = ms[0][row];
#pragma unroll
    for (int w = 1; w < NW; ++w) m = fmaxf(m, ms[w][row]);
    float l = 0.0f;
    v4f o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const float f = __builtin_amdgcn_exp2f(ms[w][row] - m);
      l += ls[w][row] * f;
      o += *reinterpret_cast<const v4f *>(&sums[w][row][d0]) * (f * 0x1p-8f);  // V scales are stored times 2^8
    }
    const int j = row / q_per_kv;
    const int64_t orow = ((int64_t)b * p.q_len + j) * p.q_heads + kvh * q_per_kv + row % q_per_kv;
    if (p.ws_o == nullptr) {
      // l is 0 where no token is live, NaN where a key of the row's is
      const float inv = l == 0.0f ? 0.0f : 1.0f / l;
      if (l == 0.0f) o = v4f{0.f, 0.f, 0.f, 0.f};
      o *= inv;
      if (p.out_bf16 != 0) {
        const uint32_t w0 = (uint32_t)f32_to_bf16_rtne(o[0]) | ((uint32_t)f32_to_bf16_rtne(o[1]) << 16);
        const uint32_t w1 = (uint32_t)f32_to_bf16_rtne(o[2]) | ((uint32_t)f32_to_bf16_rtne(o[3]) << 16);
        *reinterpret_cast<uint2 *>(static_cast<uint16_t *>(p.out) + orow * D + d0) = uint2{w0, w1};
      } else {
        *reinterpret_cast<v4f *>(static_cast<float *>(p.out) + orow * D + d0) = o;
      }
    } else {
      const int64_t prow = ((int64_t)kvh * p.n_wg + (int64_t)blockIdx.x) * R + row;
      *reinterpret_cast<v4f *>(p.ws_o + prow * D + d0) = o;
      // the combine takes a row whose l is not above 0 for empty: a NaN row keeps l = 1 beside its NaN sums
      const float2 ml = l == 0.0f ? float2{-INFINITY, 0.0f} : l != l ? float2{0.0f, 1.0f} : float2{m, l};
      if (d0 == 0) *reinterpret_cast<float2 *>(p.ws_ml + 2 * prow) = ml;
    }
  }
#endif  // __HIP_DEVICE_COMPILE__
}

template <int D, int NG>
void launch_rows(const DecodeLaunch &d, hipStream_t s) {
  const dim3 grid((unsigned)d.n_grid, (unsigned)d.g.kv_heads);
  if (d.q_bf16 != 0)
    hipLaunchKernelGGL((mx4_decode_kernel<D, NG, true, kMx4Waves>), grid, dim3(64 * kMx4Waves), 0, s, d);
  else
    hipLaunchKernelGGL((mx4_decode_kernel<D, NG, false, kMx4Waves>), grid, dim3(64 * kMx4Waves), 0, s, d);
}

}  // namespace

hipError_t launch_mx4_decode(const DecodeLaunch &d, hipStream_t s) {
  if (d.batch == 0 || d.n_grid == 0) return hipSuccess;
  const int R = d.q_len * (d.q_heads / d.g.kv_heads);
  if (d.g.head_dim == 256) {
    if (R <= 8) launch_rows<256, 0>(d, s);
    else if (R <= 16) launch_rows<256, 1>(d, s);
    else launch_rows<256, 2>(d, s);
  } else {
    if (R <= 8) launch_rows<128, 0>(d, s);
    else if (R <= 16) launch_rows<128, 1>(d, s);
    else launch_rows<128, 2>(d, s);
  }
  return hipGetLastError();
}

}  // namespace rkv
