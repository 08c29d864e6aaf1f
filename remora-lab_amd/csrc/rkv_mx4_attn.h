// rkv_mx4_attn.h -- what attention over 4-bit pages holds in registers: a tile
// of K and V as it lies in memory, and the query operand (gfx950).
#pragma once

#include "rkv_decode_kernel.h"
#include "rkv_mx4.h"

namespace rkv {
namespace {

typedef uint32_t v2u __attribute__((ext_vector_type(2)));
typedef __bf16 v2b __attribute__((ext_vector_type(2)));
typedef __bf16 v8b __attribute__((ext_vector_type(8)));
typedef uint32_t v4u __attribute__((ext_vector_type(4)));

constexpr float kNoMax = -3.0e38f;  // M before the first live token; finite, so M - M is 0

#if defined(__HIP_DEVICE_COMPILE__)

__device__ __forceinline__ v4i load16_nt(const uint8_t *p) {
  return __builtin_nontemporal_load(reinterpret_cast<const v4i *>(p));
}

// What a wave holds of one tile.  Of the V scales each lane has others, which
// the wave passes round through LDS when it needs them (loaded by every lane
// that needs them they would take 16 registers and four loads more).
template <int D>
struct Mx4Tile {
  static constexpr int H = D / 128, NB = D / 32;
  v4i kc[2 * H];      // K codes of (j, h)
  uint32_t ks;        // their E8M0 bytes
  v4i vc[D / 64];     // V codes
  uint32_t vsw;       // 4 (D 128: 2) of the tile's V scale bytes

  __device__ __forceinline__ void load_k(const uint8_t *k, int lane) {
#pragma unroll
    for (int i = 0; i < 2 * H; ++i) kc[i] = load16_nt(k + 1024 * i + 16 * lane);
    if constexpr (H == 2)
      ks = *reinterpret_cast<const uint32_t *>(k + 16 * D + 4 * lane);
    else
      ks = *reinterpret_cast<const uint16_t *>(k + 16 * D + 2 * lane);
  }
  __device__ __forceinline__ void load_v(const uint8_t *v, int lane) {
#pragma unroll
    for (int i = 0; i < D / 64; ++i) vc[i] = load16_nt(v + 1024 * i + 16 * lane);
    if constexpr (H == 2)
      vsw = *reinterpret_cast<const uint32_t *>(v + 16 * D + 4 * lane);
    else
      vsw = *reinterpret_cast<const uint16_t *>(v + 16 * D + 2 * lane);
  }
};

// The query operand of one lane: dims 128*h + 32*lg + 8*u .. +7 of its column
// for step u of half h, the dims of dword u of its K codes.
template <int D, bool kSplit, bool kBf16>
struct Mx4Query {
  static constexpr int H = D / 128;
  // products per step: a bf16 query is one term, an f32 one three, of which
  // the first two share a product where columns 8-15 are free
  static constexpr int kSets = kBf16 ? 1 : kSplit ? 2 : 3;
  v8b b[kSets][H][4];

  // off: the row's first element, -1: no row (zeros)
  __device__ __forceinline__ void load(const void *q, int64_t off, float sign, bool second, int lg) {
#pragma unroll
    for (int h = 0; h < H; ++h)
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int64_t at = off + 128 * h + 32 * lg + 8 * u;
        if constexpr (kBf16) {
          v4u w = {0, 0, 0, 0};
          if (off >= 0) w = *reinterpret_cast<const v4u *>(static_cast<const uint16_t *>(q) + at);
          b[0][h][u] = __builtin_bit_cast(v8b, w ^ (sign < 0.0f ? 0x80008000u : 0u));
        } else {
          v4f w[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
          if (off >= 0) {
            w[0] = reinterpret_cast<const v4f *>(static_cast<const float *>(q) + at)[0];
            w[1] = reinterpret_cast<const v4f *>(static_cast<const float *>(q) + at)[1];
          }
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float x = w[i / 4][i % 4] * sign;
            const __bf16 t0 = (__bf16)x;
            const float r1 = x - (float)t0;
            const __bf16 t1 = (__bf16)r1;
            const __bf16 t2 = (__bf16)(r1 - (float)t1);
            if constexpr (kSplit) {
              b[0][h][u][i] = second ? t1 : t0;
              b[1][h][u][i] = second ? (__bf16)0.0f : t2;
            } else {
              b[0][h][u][i] = t0;
              b[1][h][u][i] = t1;
              b[2][h][u][i] = t2;
            }
          }
        }
      }
  }
};

// The 8 f16 values of a V code word: tokens 0..7 of the lane's group for one
// dim, times `scale` (a power of two).
__device__ __forceinline__ v8h mx4_widen_v(uint32_t c, float scale) {
  const v2h a0 = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c, scale, 0);
  const v2h a1 = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c, scale, 1);
  const v2h a2 = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c, scale, 2);
  const v2h a3 = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c, scale, 3);
  return v8h{a0[0], a0[1], a1[0], a1[1], a2[0], a2[1], a3[0], a3[1]};
}

// The 8 bf16 values of a K code word: 8 dims of a token, times its scale.
__device__ __forceinline__ v8b mx4_widen_k(uint32_t c, float scale) {
  const v2b a0 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, scale, 0);
  const v2b a1 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, scale, 1);
  const v2b a2 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, scale, 2);
  const v2b a3 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, scale, 3);
  return v8b{a0[0], a0[1], a1[0], a1[1], a2[0], a2[1], a3[0], a3[1]};
}

// The V scales of a lane's 8 tokens in one block as f16 values times 2^8, from
// their bytes.
__device__ __forceinline__ v8h mx4_v_scales(uint32_t s0, uint32_t s1) {
  const v4u m = {__builtin_amdgcn_perm(s0, s0, 0x010c000cu), __builtin_amdgcn_perm(s0, s0, 0x030c020cu),
                 __builtin_amdgcn_perm(s1, s1, 0x010c000cu), __builtin_amdgcn_perm(s1, s1, 0x030c020cu)};
  return __builtin_bit_cast(v8h, m);
}

// Bytes of a word of V scales that mark NaN blocks (0x7c and more): their bit 7.
__device__ __forceinline__ uint32_t mx4_nans(uint32_t s) { return ((s | 0x80808080u) - 0x7c7c7c7cu) & 0x80808080u; }

// Bytes of a word of scales that belong to the first n of its 4 tokens.
__device__ __forceinline__ uint32_t mx4_keep(int32_t n) { return n >= 4 ? ~0u : n <= 0 ? 0u : (1u << (8 * n)) - 1u; }

// A tile's V scales in LDS, the wave's own D bytes: every lane's word in (a
// wave's LDS accesses run in order), and the bytes of block b for the 8 tokens
// of a lane's group out.
template <int D>
__device__ __forceinline__ void mx4_put_scales(__attribute__((address_space(3))) uint8_t *vsc, uint32_t w, int lane) {
  if constexpr (D == 256) *reinterpret_cast<__attribute__((address_space(3))) uint32_t *>(vsc + 4 * lane) = w;
  else *reinterpret_cast<__attribute__((address_space(3))) uint16_t *>(vsc + 2 * lane) = (uint16_t)w;
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
}
template <int D>
__device__ __forceinline__ v2u mx4_get_scales(const __attribute__((address_space(3))) uint8_t *vsc, int b, int lg) {
  return *reinterpret_cast<const __attribute__((address_space(3))) v2u *>(vsc + D / 4 * lg + 8 * b);
}

// A kv head's tiles of one sequence.  A page id outside the pool reads page 0
// and is remembered.
struct Mx4Place {
  const uint8_t *base;  // the kv head's K region of page 0
  const int32_t *bt;    // the sequence's block-table row
  uint64_t page_bytes, region;
  int32_t page_tokens, num_pages;
  bool bad;
  __device__ __forceinline__ Mx4Place(const DecodeLaunch &p, int32_t seq, int kvh)
      : base(p.pages + (uint64_t)kvh * 2u * mx4_region_bytes(p.g)), bt(p.bt + (int64_t)seq * p.bt_stride),
        page_bytes(mx4_page_bytes(p.g)), region(mx4_region_bytes(p.g)), page_tokens(p.g.page_tokens),
        num_pages(p.g.num_pages), bad(false) {}
  // the K tile that holds position tok (V's is `region` bytes on)
  template <int D>
  __device__ __forceinline__ const uint8_t *tile(int32_t tok) {
    int32_t page = bt[tok / page_tokens];
    if (page < 0 || page >= num_pages) {
      bad = true;
      page = 0;
    }
    return base + (uint64_t)page * page_bytes + (uint64_t)(tok % page_tokens / kTile) * mx4_tile_bytes(D);
  }
};

// A wave's walk over the tiles at tok, tok + step, .. below `end`, those that
// end at or before `whole` unmasked.  `ready` runs when the first tile's loads
// are on their way.  (Two loops and not one with a choice: each keeps the sums
// in place.)
template <int D, typename Work, typename Ready>
__device__ __forceinline__ void mx4_walk(Work &w, Mx4Place &at, int32_t tok, int32_t step, int32_t whole, int32_t end,
                                         Ready ready) {
  typename Work::Tile t;
  if (tok < end) {
    const uint8_t *k = at.tile<D>(tok);
    t.load_k(k, w.lane);
    t.load_v(k + at.region, w.lane);
  }
  ready();
  for (; tok + kTile <= whole && tok < end; tok += step)
    w.template compute<false>(t, tok, tok + step < end ? at.tile<D>(tok + step) : nullptr, at.region);
  for (; tok < end; tok += step)
    w.template compute<true>(t, tok, tok + step < end ? at.tile<D>(tok + step) : nullptr, at.region);
}

// G groups of 16 query rows, a row per column: their sums and softmax state.
// kTwo: softmax weights of two f16 terms.
template <int D, int G, bool kTwo>
struct Mx4Rows {
  static constexpr int kTerms = kTwo ? 2 : 1;
  v4f acc[G][D / 16];  // acc[2b + odd][i]: dim 32*b + 8*lg + 2*i + odd of column li
  float M[G], l[G];
  float mul;
  int32_t rlim[G];     // positions that the lane's row attends
  int lane, li, lg;

  // The weights of a tile at position tok, from its scores.
  template <bool kMasked>
  __device__ __forceinline__ void weights(const v4f (&sc)[G][2], int32_t tok, v8h (&w)[G][kTerms]) {
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
    float minus = -1.0f;
    asm("" : "+s"(minus));  // (a factor to the compiler: one mixed fma and not a conversion and a difference)
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
          const v2h lo = __builtin_bit_cast(v2h, __builtin_amdgcn_cvt_pkrtz(
              __builtin_fmaf((float)hi[0], minus, p0), __builtin_fmaf((float)hi[1], minus, p1)));
          w[g][1][2 * i] = lo[0];
          w[g][1][2 * i + 1] = lo[1];
          l[g] = __builtin_amdgcn_fdot2(lo, one, l[g], false);
        }
      }
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

// G groups of rows that share the widened K and V of a tile.
template <int D, int G, bool kBf16>
struct Mx4Wide : Mx4Rows<D, G, true> {
  using Rows = Mx4Rows<D, G, true>;
  using Rows::acc, Rows::rlim, Rows::lane, Rows::lg;
  static constexpr int H = D / 128, NB = D / 32;
  using Query = Mx4Query<D, false, kBf16>;
  static constexpr int kQuery = G * H * 4 * Query::kSets * 64;  // the query operand's 16-byte words in LDS
  using Tile = Mx4Tile<D>;

  // the query operand of (group, half, step, term), 64 lanes' words each
  const __attribute__((address_space(3))) v8b *q;
  __attribute__((address_space(3))) uint8_t *vsc;  // the tile's D bytes of V scales, the wave's own
  int32_t end;  // positions that any of the wave's rows attends

  // Column li's row of group g (its first element at off, -1: none) into the
  // operand at `to`.
  __device__ __forceinline__ void put_query(v8b *to, int g, const void *src, int64_t off, float sign) const {
    Query x;
    x.load(src, off, sign, false, lg);
#pragma unroll
    for (int i = 0; i < 4 * H; ++i)
#pragma unroll
      for (int s = 0; s < Query::kSets; ++s) to[((g * H * 4 + i) * Query::kSets + s) * 64 + lane] = x.b[s][i / 4][i % 4];
  }

  // The tile at position tok, held in t; the wave's next one, at `next` (NULL:
  // none), is loaded into t's registers as they come free.
  template <bool kMasked>
  __device__ __forceinline__ void compute(Tile &t, int32_t tok, const uint8_t *next, uint64_t region) {
    v4f sc[G][2];
#pragma unroll
    for (int g = 0; g < G; ++g) sc[g][0] = sc[g][1] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int h = 0; h < H; ++h) {
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        v8b b[G][Query::kSets];
#pragma unroll
        for (int g = 0; g < G; ++g)
#pragma unroll
          for (int s = 0; s < Query::kSets; ++s) b[g][s] = q[(((g * H + h) * 4 + u) * Query::kSets + s) * 64 + lane];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const float scale = __builtin_bit_cast(float, (t.ks >> (8 * (j * H + h)) & 0xffu) << 23);
          const v8b a = mx4_widen_k((uint32_t)t.kc[j * H + h][u], scale);
#pragma unroll
          for (int g = 0; g < G; ++g)
#pragma unroll
            for (int s = Query::kSets - 1; s >= 0; --s)
              sc[g][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b[g][s], sc[g][j], 0, 0, 0);
        }
      }
    }
    if (next != nullptr) t.load_k(next, lane);
    v8h w[G][Rows::kTerms];
    Rows::template weights<kMasked>(sc, tok, w);
    mx4_put_scales<D>(vsc, t.vsw, lane);
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
          for (int k = 0; k < Rows::kTerms; ++k)
            acc[g][dt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, w[g][k], acc[g][dt], 0, 0, 0);
      }
    }
    if (next != nullptr) t.load_v(next + region, lane);
  }

  __device__ __forceinline__ v2u scales(int b) const { return mx4_get_scales<D>(vsc, b, lg); }

  // A masked tile with NaN V blocks: rows that attend one get NaN in its
  // dims, and the block's scale goes to 0 for the rows that do not (a weight
  // of 0 times NaN is NaN).
  __device__ __forceinline__ void drop_nan(int32_t tok, uint32_t keep0, uint32_t keep1) {
    uint32_t any = 0;
#pragma unroll
    for (int b = 0; b < NB; ++b) any |= mx4_nans(scales(b)[0] & keep0) | mx4_nans(scales(b)[1] & keep1);
    if (__ballot(any != 0) == 0) return;
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      const v2u s = scales(b);
      const uint32_t n0 = mx4_nans(s[0] & keep0), n1 = mx4_nans(s[1] & keep1);
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
};
#endif  // __HIP_DEVICE_COMPILE__

}  // namespace
}  // namespace rkv
