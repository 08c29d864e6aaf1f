// rkv_mx4.h -- the 4-bit page format: 32 values of a row as E2M1 codes under a
// power-of-two scale (17 bytes), laid out for the gfx950 matrix instructions.
//
// A block's scale is 2^e, e the smallest exponent with max|v| <= 7 * 2^e (7
// still rounds to the largest code, 6, with the error of half a step), kept
// within [kMx4KMin, kMx4KMax] for K and [kMx4VMin, kMx4VMax] for V; a code is
// v / 2^e rounded to nearest, ties to the even code, saturating at 6.  A block
// with a value that is not finite holds NaN: codes 0 under a NaN scale.
//
// Page = [kv_head][kind K|V][tile], a tile 32 tokens in 17*D contiguous bytes,
// 16*D of codes and D of scales:
//   K codes  [j][h][b][m] 16 bytes: token 8*(m/4) + 4*j + m%4, dims
//            128*h + 32*b .. +31, even dim in the low nibble
//   K scales [b][m][j][h] bytes, E8M0: e + 127 (NaN 255)
//   V codes  [c][g][n][t] 4 bytes: dim 64*c + 32*(t/2) + 2*n + t%2, tokens
//            8*g .. 8*g+7, even token in the low nibble
//   V scales [g][block][8 tokens] bytes: the high byte of the f16 2^(e+8)
//            (NaN 0x7e)
// with j < 2, h < D/128, b < 4, m < 16, c < D/64, g < 4, n < 16, t < 4.
//
// K codes [j][h] are 1 KiB: lane 16*b + m of a wave holds the A operand of
// mfma_scale 16x16x128 (32 E2M1 values of one token) as it lies in memory, and
// its scale dword holds the E8M0 bytes of all the tile's products.  V codes
// [c] are 1 KiB of A operands of the f16 16x16x32 product: lane 16*g + n holds
// the 8 tokens of group g for 4 dims.  The even and odd dims of a block are
// two products, so that one pair of rows fits the 4 + 4 values a lane keeps of
// it into 8 consecutive dims.
#pragma once

#include "rkv_device.h"

namespace rkv {

constexpr int32_t kMx4KMin = -24, kMx4KMax = 15;
constexpr int32_t kMx4VMin = -22, kMx4VMax = 7;
constexpr int32_t kMx4Tile = 32;

__host__ __device__ constexpr uint64_t mx4_tile_bytes(int32_t head_dim) { return 17u * (uint64_t)head_dim; }
__host__ __device__ inline uint64_t mx4_region_bytes(const Geo &g) {
  return (uint64_t)(g.page_tokens / kMx4Tile) * mx4_tile_bytes(g.head_dim);
}
__host__ __device__ inline uint64_t mx4_page_bytes(const Geo &g) {
  return (uint64_t)g.kv_heads * 2u * mx4_region_bytes(g);
}
__host__ __device__ inline uint64_t mx4_region_base(const Geo &g, int32_t page, int32_t kvh, int32_t kind) {
  return (uint64_t)page * mx4_page_bytes(g) + (uint64_t)(kvh * 2 + kind) * mx4_region_bytes(g);
}

}  // namespace rkv
