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

// What a wave holds of one tile.  kScalesInLds: of the V scales only its share
// of vmax, which the wave passes round through LDS when it needs them.
template <int D, bool kScalesInLds = false>
struct Mx4Tile {
  static constexpr int H = D / 128, NB = D / 32;
  v4i kc[2 * H];      // K codes of (j, h)
  uint32_t ks;        // their E8M0 bytes
  v4i vc[D / 64];     // V codes
  v4i vs[kScalesInLds ? 1 : NB / 2];  // V scale bytes of the lane's 8 tokens, 8 per block
  uint32_t vmax;      // 2 or 4 of the tile's V scale bytes, each lane others

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
#pragma unroll
    for (int i = 0; i < (kScalesInLds ? 0 : NB / 2); ++i)
      vs[i] = *reinterpret_cast<const v4i *>(v + 16 * D + 8 * NB * (lane >> 4) + 16 * i);
    if constexpr (H == 2)
      vmax = *reinterpret_cast<const uint32_t *>(v + 16 * D + 4 * lane);
    else
      vmax = *reinterpret_cast<const uint16_t *>(v + 16 * D + 2 * lane);
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

// Bytes of a word of scales that belong to the first n of its 4 tokens.
__device__ __forceinline__ uint32_t mx4_keep(int32_t n) { return n >= 4 ? ~0u : n <= 0 ? 0u : (1u << (8 * n)) - 1u; }
#endif  // __HIP_DEVICE_COMPILE__

}  // namespace
}  // namespace rkv
