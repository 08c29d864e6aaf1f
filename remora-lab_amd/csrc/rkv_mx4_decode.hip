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
// Up to 8 rows (Mx4Narrow):
//   QK: bf16 16x16x32, A = K codes widened with their power of two (exact in
//     bf16, one instruction for two), B = the query, an f32 one as three bf16
//     terms; products are exact and summed in f32.  Columns 8-15 hold the rows
//     again (f32: their second terms).  (The scaled E2M1 x E4M3
//     product needs no widening, but keeps only about 13 bits below its
//     largest term: with channels eight times the others the outputs of 32k
//     tokens were off by 1.5e-5, 2e-6 in f32.)
//   PV: f16 16x16x32, A = V codes widened (exact, one instruction for two),
//     B = p * 2^e_v as two f16 terms, p = hi + lo to 22 bits, both times the
//     block's power of two (exact); lo takes columns 8-15.
//   f16 range: M is kept so that p * 2^e_v <= 2^15, i.e. with vcap the largest V
//   exponent met (at least 2^0 in the units of the stored byte) the row maximum
//   maps to 2^(11 - vcap) and may rise by 2^4 before the sums are rescaled.
// 9 to 32 rows (Mx4Wide): one or two groups of 16 columns, V widened with its
// scales once for all of them, the query in LDS.
//
// Measured (2 kv heads of 256, bf16 queries): 64 x 32k tokens of 8 rows 180 us
// a call, 6.4 TB/s (a read of the same pages in the same order 165); one
// sequence of 262,145 tokens 35 us, 16 of 4k..16k 26, one of 300 8: locating
// the partition, its page ids and its first tile come one after the other, and
// a second launch joins partials (4.5 us).  32 x 32k tokens of 32 rows 131 us
// (memory alone 83): 2 waves a SIMD issue 380 vector and 96 matrix instructions
// a tile, counted.  Not faster: two tiles in flight, a third wave a SIMD, 8 waves a
// workgroup.
#include <algorithm>

#include "rkv_mx4_attn.h"

namespace rkv {
namespace {

#if defined(__HIP_DEVICE_COMPILE__)

template <int D, bool kBf16>
struct Mx4Narrow {
  static constexpr int H = D / 128, NB = D / 32;
  using Query = Mx4Query<D, true, kBf16>;
  using Tile = Mx4Tile<D>;

  Query q;
  __attribute__((address_space(3))) uint8_t *vsc;  // the tile's D bytes of V scales, the wave's own
  v4f acc[D / 16];  // acc[2b + odd][i]: dim 32*b + 8*lg + 2*i + odd of column li
  float M, l;
  float mul;        // |scale| * log2 e
  int32_t rlim;     // positions that the lane's row attends
  int32_t vcap;     // exponent of the largest V scale met, in the stored byte's units, >= 0
  float losel;      // -1 in the columns of the second term
  int32_t end;      // positions that any row attends
  int lane, li, lg;

  // The tile at position tok, held in t; the wave's next one, at `next` (NULL:
  // none), is loaded into t's registers as they come free.
  template <bool kMasked>
  __device__ __forceinline__ void compute(Tile &t, int32_t tok, const uint8_t *next, uint64_t region) {
    v4f sc[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      sc[j] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int h = 0; h < H; ++h) {
        const float scale = __builtin_bit_cast(float, (t.ks >> (8 * (j * H + h)) & 0xffu) << 23);
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const v8b a = mx4_widen_k((uint32_t)t.kc[j * H + h][u], scale);
#pragma unroll
          for (int s = Query::kSets - 1; s >= 0; --s)
            sc[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, q.b[s][h][u], sc[j], 0, 0, 0);
        }
      }
    }
    if (next != nullptr) t.load_k(next, lane);
    float x[8];
    const int32_t live = rlim - tok - 8 * lg;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      x[i] = sc[i / 4][i % 4];
      if constexpr (!kBf16) x[i] += dpp_ror8(x[i]);
      if constexpr (kMasked) x[i] = i < live ? x[i] : -INFINITY;
    }
    // s - M of the largest score, and the V scales against vcap
    const uint32_t vmax = kMasked ? t.vsw & vlive(end - tok) : t.vsw;
    const uint32_t cap = (uint32_t)(4 * (vcap + 15)) * 0x01010101u;
    float top = x[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) top = fmaxf(top, x[i]);
    const bool high = (((vmax | 0x80808080u) - cap - 0x01010101u) & 0x80808080u) != 0u ||
                      __builtin_fmaf(top, mul, -M) > (float)(15 - vcap);
    if (__ballot(high) != 0) rescale(vmax, top);
    const v2h one = {(_Float16)1.0f, (_Float16)1.0f};
    v8h w;  // the tokens' weights: first terms, in columns 8-15 second terms
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(x[2 * i], mul, -M));
      const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(x[2 * i + 1], mul, -M));
      const v2h hi = __builtin_bit_cast(v2h, __builtin_amdgcn_cvt_pkrtz(p0, p1));
      const v2h own = __builtin_bit_cast(
          v2h, __builtin_amdgcn_cvt_pkrtz(__builtin_fmaf((float)hi[0], losel, p0), __builtin_fmaf((float)hi[1], losel, p1)));
      w[2 * i] = own[0];
      w[2 * i + 1] = own[1];
      l = __builtin_amdgcn_fdot2(own, one, l, false);
    }
    mx4_put_scales<D>(vsc, t.vsw, lane);
    // masked tiles: the row's own tokens' scales only (a weight of 0 times NaN is NaN)
    const uint32_t keep0 = mx4_keep(live), keep1 = mx4_keep(live - 4);
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      const v2u sw = mx4_get_scales<D>(vsc, b, lg);
      uint32_t s0 = sw[0], s1 = sw[1];
      if constexpr (kMasked) {
        s0 &= keep0;
        s1 &= keep1;
      }
      const v8h ws = w * mx4_v_scales(s0, s1);
#pragma unroll
      for (int odd = 0; odd < 2; ++odd) {
        const int dt = 2 * b + odd;
        acc[dt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(mx4_widen_v((uint32_t)t.vc[dt / 4][dt % 4], 1.0f), ws, acc[dt],
                                                         0, 0, 0);
      }
    }
    if (next != nullptr) t.load_v(next + region, lane);
  }

  // The bytes of vsw that belong to the tile's first n tokens: what a page
  // holds behind them is nobody's, and no result may follow it.
  __device__ __forceinline__ uint32_t vlive(int32_t n) const {
    constexpr int kPer = H == 2 ? 4 : 2;  // tokens of a lane, of group lane / 16
    return mx4_keep(min(n - 8 * lg - kPer * (lane % (8 / kPer)), kPer));
  }

  // A score or a V scale outgrew what M allows: the rows' new M, and the sums in its units.
  __device__ __forceinline__ void rescale(uint32_t v, float top) {
    v = max(max(v & 0xffu, (v >> 8) & 0xffu), max((v >> 16) & 0xffu, v >> 24));
    // (a NaN scale's byte reads as 16; NaN outgrows no range)
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) v = max(v, (uint32_t)__shfl_xor((int)v, off));
    const int32_t cap = min(max((int32_t)(v >> 2) - 15, vcap), 15);
    top = fmaxf(top, __shfl_xor(top, 16));
    top = fmaxf(top, __shfl_xor(top, 32));
    // s_max * 2^(vcap - 11), and no lower than what held before
    float n = fmaxf(__builtin_fmaf(top, mul, (float)(cap - 11)), M + (float)(cap - vcap));
    if (!(n > M)) n = M;  // (a row without a live token stays where it was)
    const float f = __builtin_amdgcn_exp2f(M - n);
    M = n;
    l *= f;
#pragma unroll
    for (int i = 0; i < D / 16; ++i) acc[i] *= f;
    vcap = cap;
  }
};

// A workgroup's partition: entry b's tokens [tok0, tok_end) of sequence seq.
struct Mx4Part {
  int32_t b, seq, len, tok0, tok_end;
};
// false: the grid's spare workgroup, or the entry is reported (its partition is
// then empty and its rows 0: part.len is 0).
__device__ __forceinline__ bool find_part(const DecodeLaunch &p, int lane, int kvh, Mx4Part &o) {
  int32_t pt, lenc, part, nb;
  if (!locate(p, lane, (int32_t)blockIdx.x, pt, o.b, o.seq, lenc, part, nb, 1 << 24)) return false;
  if (p.ws_hdr != nullptr && kvh == 0 && threadIdx.x == 0) {
    if (blockIdx.x == 0) p.ws_hdr[0] = pt;
    if (part == 0) {
      p.ws_hdr[1 + 2 * o.b] = (int32_t)blockIdx.x;
      p.ws_hdr[2 + 2 * o.b] = nb;
    }
  }
  o.len = lenc;
  int32_t bad = 0;
  if (o.seq < 0 || o.seq >= p.n_seqs) bad = FAULT_BAD_SEQ;
  else if (lenc == 0 && p.seq_lens[o.seq] != 0) bad = FAULT_BAD_POSITION;  // out of range: locate() takes it as 0
  else if ((int64_t)lenc > (int64_t)p.bt_stride * p.g.page_tokens) bad = FAULT_BAD_POSITION;
  if (bad != 0) {
    if (threadIdx.x == 0) atomicOr(p.fault, bad);
    o.len = 0;
  }
  o.tok0 = min(part * pt, o.len);
  o.tok_end = part == nb - 1 ? o.len : min(o.len, o.tok0 + pt);
  return true;
}

// First element of the entry's query row `row` (q_len rows of the kv head's q
// heads), -1 past the last one.
__device__ __forceinline__ int64_t query_row(const DecodeLaunch &p, int32_t b, int kvh, int row) {
  const int32_t G = p.q_heads / p.g.kv_heads;
  if (row >= p.q_len * G) return -1;
  return ((int64_t)b * p.q_len + row / G) * p.q_heads + kvh * G + row % G;
}

// 4 dims from d0 of a row whose weighted sum is o and weight l at M = m: the
// row itself, or the partition's partial of it.
template <int D>
__device__ __forceinline__ void store_row(const DecodeLaunch &p, int32_t b, int kvh, int row, int d0, v4f o, float m,
                                          float l) {
  if (p.ws_o == nullptr) {
    // l is 0 where no token is live, NaN where a key of the row's is
    if (l == 0.0f) o = v4f{0.f, 0.f, 0.f, 0.f};
    else o *= 1.0f / l;
    const int64_t at = query_row(p, b, kvh, row) * D + d0;
    if (p.out_bf16 != 0) {
      const v2b w0 = {(__bf16)o[0], (__bf16)o[1]}, w1 = {(__bf16)o[2], (__bf16)o[3]};
      *reinterpret_cast<v2u *>(static_cast<uint16_t *>(p.out) + at) =
          v2u{__builtin_bit_cast(uint32_t, w0), __builtin_bit_cast(uint32_t, w1)};
    } else {
      *reinterpret_cast<v4f *>(static_cast<float *>(p.out) + at) = o;
    }
    return;
  }
  const int32_t R = p.q_len * (p.q_heads / p.g.kv_heads);
  const int64_t prow = ((int64_t)kvh * p.n_wg + (int64_t)blockIdx.x) * R + row;
  *reinterpret_cast<v4f *>(p.ws_o + prow * D + d0) = o;
  // the combine takes a row whose l is not above 0 for empty: a NaN row keeps l = 1 beside its NaN sums
  const float2 ml = l == 0.0f ? float2{-INFINITY, 0.0f} : l != l ? float2{0.0f, 1.0f} : float2{m, l};
  if (d0 == 0) *reinterpret_cast<float2 *>(p.ws_ml + 2 * prow) = ml;
}

// A group's sums in this lane, 8 dims of each block of row `row`, times f to dst.
template <int D, bool kAdd>
__device__ __forceinline__ void put_sums(float *dst, const v4f *acc, int lg, float f) {
#pragma unroll
  for (int i = 0; i < D / 32; ++i) {
    const v4f e = acc[2 * i] * f, o = acc[2 * i + 1] * f;
    v4f *at = reinterpret_cast<v4f *>(dst + 32 * i + 8 * lg);
    const v4f a = {e[0], o[0], e[1], o[1]}, b = {e[2], o[2], e[3], o[3]};
    at[0] = kAdd ? at[0] + a : a;
    at[1] = kAdd ? at[1] + b : b;
  }
}
#endif  // __HIP_DEVICE_COMPILE__

template <int D, bool kBf16, int NW>
__global__ __launch_bounds__(64 * NW, kMx4WgsPerCu) void mx4_decode_kernel(DecodeLaunch p) {
#if defined(__HIP_DEVICE_COMPILE__)
  using Dec = Mx4Narrow<D, kBf16>;
  constexpr int kStride = D + 4;  // floats between a row's sums in LDS
  __shared__ __attribute__((aligned(16))) float sums[NW][8][kStride];
  __shared__ float ms[NW][8], ls[NW][8];
  __shared__ __attribute__((aligned(16))) uint8_t vscs[NW][D];
  Dec dc;
  const int lane = threadIdx.x & 63, li = lane & 15, lg = lane >> 4;
  const int wave = (int)__builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int kvh = blockIdx.y;
  dc.lane = lane;
  dc.li = li;
  dc.lg = lg;
  Mx4Part part;
  if (!find_part(p, lane, kvh, part)) return;
  const int32_t G = p.q_heads / p.g.kv_heads, R = p.q_len * G;
  // at least the smallest normal: a masked -inf times it stays -inf with a scale of 0
  dc.mul = fmaxf(fabsf(p.scale_log2), 1.17549435e-38f);
  dc.vsc = (__attribute__((address_space(3))) uint8_t *)vscs[wave];
  dc.vcap = 0;
  dc.losel = li >= 8 ? -1.0f : 0.0f;
  dc.end = part.tok_end;
  const int64_t row = query_row(p, part.b, kvh, li & 7);
  dc.rlim = row < 0 ? 0 : part.len - p.q_len + (li & 7) / G + 1;
  dc.M = kNoMax;
  dc.l = 0.0f;
#pragma unroll
  for (int i = 0; i < D / 16; ++i) dc.acc[i] = v4f{0.f, 0.f, 0.f, 0.f};

  // the wave's tiles: tok0 + 32*wave, then every NW-th; row 0 attends len - q_len + 1 positions
  Mx4Place at(p, part.seq, kvh);
  mx4_walk<D>(dc, at, part.tok0 + kTile * wave, kTile * NW, min(part.len - p.q_len + 1, part.tok_end), part.tok_end,
              [&] { dc.q.load(p.q, row < 0 ? -1 : row * D, p.scale_log2 < 0.0f ? -1.0f : 1.0f, li >= 8, lg); });
  if (at.bad && lane == 0) atomicOr(p.fault, FAULT_BAD_PAGE);

  // ---- merge of the waves: second terms onto the first, then every wave's rows side by side
  float l = dc.l;
  l += __shfl_xor(l, 16);
  l += __shfl_xor(l, 32);
  l += dpp_ror8(l);
#pragma unroll
  for (int i = 0; i < D / 16; ++i)
#pragma unroll
    for (int k = 0; k < 4; ++k) dc.acc[i][k] += dpp_ror8(dc.acc[i][k]);
  if (li < 8) {
    if (lg == 0) {
      ms[wave][li] = dc.M;
      ls[wave][li] = l;
    }
    put_sums<D, false>(sums[wave][li], dc.acc, lg, 0x1p-8f);  // (V scales are stored times 2^8)
  }
  __syncthreads();
  for (int i = threadIdx.x; i < R * (D / 4); i += 64 * NW) {
    const int r = i / (D / 4), d0 = 4 * (i % (D / 4));
    float m = ms[0][r];
#pragma unroll
    for (int w = 1; w < NW; ++w) m = fmaxf(m, ms[w][r]);
    float sum = 0.0f;
    v4f o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const float f = __builtin_amdgcn_exp2f(ms[w][r] - m);
      sum += ls[w][r] * f;
      o += *reinterpret_cast<const v4f *>(&sums[w][r][d0]) * f;
    }
    store_row<D>(p, part.b, kvh, r, d0, o, m, sum);
  }
#endif  // __HIP_DEVICE_COMPILE__
}

// G groups of 16 rows.  The query (and, when the waves are done with it, the
// rows' sums, wave after wave) is the workgroup's.
template <int D, int G, bool kBf16, int NW>
__global__ __launch_bounds__(64 * NW, kMx4WgsPerCu) void mx4_decode_wide_kernel(DecodeLaunch p) {
#if defined(__HIP_DEVICE_COMPILE__)
  using Dec = Mx4Wide<D, G, kBf16>;  // (weights of two terms cost a verify of 32 x 32k rows 1 us of 152)
  constexpr int kStride = D + 4;
  constexpr int kShared = Dec::kQuery * 16 > 16 * G * kStride * 4 ? Dec::kQuery * 16 : 16 * G * kStride * 4;
  __shared__ __attribute__((aligned(16))) uint8_t shared[kShared];
  __shared__ __attribute__((aligned(16))) uint8_t vscs[NW][D];
  __shared__ float ms[NW][16 * G], ls[NW][16 * G];
  Dec dc;
  const int lane = threadIdx.x & 63, li = lane & 15, lg = lane >> 4;
  const int wave = (int)__builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int kvh = blockIdx.y;
  dc.lane = lane;
  dc.li = li;
  dc.lg = lg;
  Mx4Part part;
  if (!find_part(p, lane, kvh, part)) return;
  const int32_t heads = p.q_heads / p.g.kv_heads, R = p.q_len * heads;
  dc.q = (const __attribute__((address_space(3))) v8b *)(v8b *)shared;
  dc.vsc = (__attribute__((address_space(3))) uint8_t *)vscs[wave];
  dc.mul = fmaxf(fabsf(p.scale_log2), 1.17549435e-38f);
  dc.end = part.tok_end;
#pragma unroll
  for (int c = 0; c < G; ++c) {
    dc.rlim[c] = 16 * c + li >= R ? 0 : part.len - p.q_len + (16 * c + li) / heads + 1;
    dc.M[c] = kNoMax;
    dc.l[c] = 0.0f;
#pragma unroll
    for (int i = 0; i < D / 16; ++i) dc.acc[c][i] = v4f{0.f, 0.f, 0.f, 0.f};
  }
  Mx4Place at(p, part.seq, kvh);
  mx4_walk<D>(dc, at, part.tok0 + kTile * wave, kTile * NW, min(part.len - p.q_len + 1, part.tok_end), part.tok_end, [&] {
    if (wave < G) {
      const int64_t row = query_row(p, part.b, kvh, 16 * wave + li);
      dc.put_query(reinterpret_cast<v8b *>(shared), wave, p.q, row < 0 ? -1 : row * D, p.scale_log2 < 0.0f ? -1.0f : 1.0f);
    }
    __syncthreads();
  });
  if (at.bad && lane == 0) atomicOr(p.fault, FAULT_BAD_PAGE);

#pragma unroll
  for (int c = 0; c < G; ++c) {
    float l = dc.l[c];
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    if (lg == 0) {
      ms[wave][16 * c + li] = dc.M[c];
      ls[wave][16 * c + li] = l;
    }
  }
  float *sums = reinterpret_cast<float *>(shared);
#pragma unroll 1
  for (int w = 0; w < NW; ++w) {
    __syncthreads();
    if (wave != w) continue;
#pragma unroll
    for (int c = 0; c < G; ++c) {
      const int r = 16 * c + li;
      float m = ms[0][r];
#pragma unroll
      for (int k = 1; k < NW; ++k) m = fmaxf(m, ms[k][r]);
      const float f = __builtin_amdgcn_exp2f(dc.M[c] - m) * 0x1p-6f;  // (V is held times 2^6)
      if (w == 0) put_sums<D, false>(sums + r * kStride, dc.acc[c], lg, f);
      else put_sums<D, true>(sums + r * kStride, dc.acc[c], lg, f);
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < R * (D / 4); i += 64 * NW) {
    const int r = i / (D / 4), d0 = 4 * (i % (D / 4));
    float m = ms[0][r];
#pragma unroll
    for (int w = 1; w < NW; ++w) m = fmaxf(m, ms[w][r]);
    float sum = 0.0f;
#pragma unroll
    for (int w = 0; w < NW; ++w) sum += ls[w][r] * __builtin_amdgcn_exp2f(ms[w][r] - m);
    store_row<D>(p, part.b, kvh, r, d0, *reinterpret_cast<const v4f *>(sums + r * kStride + d0), m, sum);
  }
#endif  // __HIP_DEVICE_COMPILE__
}

template <int D, bool kBf16>
void launch_rows(const DecodeLaunch &d, hipStream_t s) {
  const dim3 grid((unsigned)d.n_grid, (unsigned)d.g.kv_heads);
  const int R = d.q_len * (d.q_heads / d.g.kv_heads);
  if (R <= 8)
    hipLaunchKernelGGL((mx4_decode_kernel<D, kBf16, kMx4Waves>), grid, dim3(64 * kMx4Waves), 0, s, d);
  else if (R <= 16)
    hipLaunchKernelGGL((mx4_decode_wide_kernel<D, 1, kBf16, kMx4Waves>), grid, dim3(64 * kMx4Waves), 0, s, d);
  else
    hipLaunchKernelGGL((mx4_decode_wide_kernel<D, 2, kBf16, kMx4Waves>), grid, dim3(64 * kMx4Waves), 0, s, d);
}

}  // namespace

hipError_t launch_mx4_decode(const DecodeLaunch &d, hipStream_t s) {
  if (d.batch == 0 || d.n_grid == 0) return hipSuccess;
  if (d.g.head_dim == 256) {
    if (d.q_bf16) launch_rows<256, true>(d, s);
    else launch_rows<256, false>(d, s);
  } else {
    if (d.q_bf16) launch_rows<128, true>(d, s);
    else launch_rows<128, false>(d, s);
  }
  return hipGetLastError();
}

}  // namespace rkv
