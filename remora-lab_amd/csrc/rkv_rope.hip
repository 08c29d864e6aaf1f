// rkv_rope.hip -- per-head norm and position rotation of query and key rows,
// the same on the way into the paged cache (Q8_0 or 4-bit pages), and cached
// rows read back as values (gfx950).
//
//   n = x / sqrt(mean(x^2) + eps) * w            (head by head, if a weight is given)
//   a_i = position[axis_i] * freq_i              (pair i of the rotated dims)
//   (x_i, x_j) -> (x_i cos a_i - x_j sin a_i, x_j cos a_i + x_i sin a_i)
//
// Angles are exact in f64 (24 + 31 bits) and reduced there, so a position of a
// million keeps every bit.  A key on its way into the cache is normed and
// rotated in f64 and rounded to f32 once, before the quantizer: f64 runs at
// half the f32 rate here, and a page byte then follows from the definition alone,
// not from an order of sums (an f32 rotation moves about one code in 10^6 over
// a border).  Rows that are returned go in f32.
//
// A head is held by D/8 lanes, 8 values each: lane c of a rotated pair of
// halves takes dims 4c..4c+3 and rot/2 + 4c.., so both values of its 4 pairs
// are its own and their cosines serve every head of the row.
#include <algorithm>
#include <type_traits>

#include "rkv_launch.h"
#include "rkv_mx4.h"

namespace rkv {
namespace {

typedef uint32_t v2u __attribute__((ext_vector_type(2)));
typedef uint32_t v4u __attribute__((ext_vector_type(4)));
typedef float v2f __attribute__((ext_vector_type(2)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef __bf16 v2b __attribute__((ext_vector_type(2)));

#if defined(__HIP_DEVICE_COMPILE__)

// ---- angles -------------------------------------------------------------------

// sin and cos of a by their Taylor series on [-pi/4, pi/4], whose first terms
// left out are below 5e-17.  Reduction: a - n*pi/2 with pi/2 in two parts, each
// step one fma, for |a| up to 2^31 and more.
__device__ __forceinline__ void sin_cos(double a, double &s, double &c) {
  const double n = __builtin_rint(a * 0.63661977236758134308);
  double r = __builtin_fma(-n, 0x1.921fb54442d18p+0, a);
  r = __builtin_fma(-n, 0x1.1a62633145c07p-54, r);
  const double z = r * r;
  double ps = -1.0 / 1307674368000.0;  // 15!
  ps = __builtin_fma(ps, z, 1.0 / 6227020800.0);
  ps = __builtin_fma(ps, z, -1.0 / 39916800.0);
  ps = __builtin_fma(ps, z, 1.0 / 362880.0);
  ps = __builtin_fma(ps, z, -1.0 / 5040.0);
  ps = __builtin_fma(ps, z, 1.0 / 120.0);
  ps = __builtin_fma(ps, z, -1.0 / 6.0);
  ps = __builtin_fma(r * z, ps, r);
  double pc = 1.0 / 20922789888000.0;  // 16!
  pc = __builtin_fma(pc, z, -1.0 / 87178291200.0);
  pc = __builtin_fma(pc, z, 1.0 / 479001600.0);
  pc = __builtin_fma(pc, z, -1.0 / 3628800.0);
  pc = __builtin_fma(pc, z, 1.0 / 40320.0);
  pc = __builtin_fma(pc, z, -1.0 / 720.0);
  pc = __builtin_fma(pc, z, 1.0 / 24.0);
  pc = __builtin_fma(pc, z, -0.5);
  pc = __builtin_fma(pc, z, 1.0);
  const int q = (int)(n - 4.0 * __builtin_floor(n * 0.25));  // quadrant
  s = q & 1 ? pc : ps;
  c = q & 1 ? ps : pc;
  s = q & 2 ? -s : s;
  c = (q + 1) & 2 ? -c : c;
}

// The angle of a pair, from the row's positions on the axes.
__device__ __forceinline__ double angle(const RopeLaunch &r, int pair, const int32_t (&at)[4]) {
  int32_t axis = r.pair_axis != nullptr ? r.pair_axis[pair] : 0;
  if (axis < 0 || axis >= r.n_axes) {
    atomicOr(r.fault, FAULT_BAD_POSITION);
    axis = 0;
  }
  return (double)(axis == 0 ? at[0] : axis == 1 ? at[1] : axis == 2 ? at[2] : at[3]) * (double)r.freqs[pair];
}

// Cosines and sines of lane c's 4 pairs of a row (1 and 0 past the rotated
// dims).  The loads of a row are independent of each other: its positions on
// every axis, and the axes that choose among them.
struct Turn {
  double c[4], s[4];
  __device__ __forceinline__ void load(const RopeLaunch &r, int64_t row, int32_t pos, int lane) {
    int32_t at[4] = {pos, pos, pos, pos};
    if (r.positions != nullptr)
#pragma unroll
      for (int a = 0; a < 4; ++a) at[a] = r.positions[(int64_t)min(a, r.n_axes - 1) * r.n_rows + row];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      c[i] = 1.0;
      s[i] = 0.0;
    }
    if (8 * lane < r.rot_dim)
#pragma unroll
      for (int i = 0; i < 4; ++i) sin_cos(angle(r, 4 * lane + i, at), s[i], c[i]);
  }
};

// ---- sums over a head's lanes ----------------------------------------------------

template <int kCtrl>
__device__ __forceinline__ float dpp(float x) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), kCtrl, 0xf, 0xf, false));
}
template <int kCtrl>
__device__ __forceinline__ double dpp(double x) {
  const uint64_t u = __builtin_bit_cast(uint64_t, x);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, kCtrl, 0xf, 0xf, false);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(u >> 32), kCtrl, 0xf, 0xf, false);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
// The value of the lane 16 away, in the neighbouring row of 16: a row swap
// leaves it in one of two registers and the lane's own in the other.
__device__ __forceinline__ uint32_t next_row(uint32_t x) {
  const auto r = __builtin_amdgcn_permlane16_swap(x, x, false, false);
  return (threadIdx.x & 16u) ? r[0] : r[1];
}
__device__ __forceinline__ float next_row(float x) {
  return __builtin_bit_cast(float, next_row(__builtin_bit_cast(uint32_t, x)));
}
__device__ __forceinline__ double next_row(double x) {
  const uint64_t u = __builtin_bit_cast(uint64_t, x);
  return __builtin_bit_cast(double, (uint64_t)next_row((uint32_t)(u >> 32)) << 32 | next_row((uint32_t)u));
}
// Over kLanes (16 or 32) consecutive lanes: swaps within quads, halves of a
// row and the row, then the neighbouring row.
template <int kLanes, typename T>
__device__ __forceinline__ T lanes_sum(T x) {
  x += dpp<0xb1>(x);   // quad_perm 1 0 3 2
  x += dpp<0x4e>(x);   // quad_perm 2 3 0 1
  x += dpp<0x141>(x);  // row_half_mirror
  x += dpp<0x140>(x);  // row_mirror
  if constexpr (kLanes == 32) x += next_row(x);
  return x;
}

__device__ __forceinline__ float inv_sqrt(float x) { return __builtin_amdgcn_rsqf(x); }
__device__ __forceinline__ double inv_sqrt(double x) {
  double y = __builtin_amdgcn_rsq(x);
#pragma unroll
  for (int i = 0; i < 2; ++i) y = __builtin_fma(y * __builtin_fma(-x * y, y, 1.0), 0.5, y);
  return x == __builtin_inf() ? 0.0 : y;
}

// ---- one head ------------------------------------------------------------------

// The dims of lane c: 4 from first(), 4 from second().
struct Dims {
  int a, b;
  __device__ __forceinline__ Dims(const RopeLaunch &r, int c) {
    const bool halves = r.on && !r.adjacent && 8 * c < r.rot_dim;
    a = halves ? 4 * c : 8 * c;
    b = halves ? r.rot_dim / 2 + 4 * c : 8 * c + 4;
  }
};

__device__ __forceinline__ void load4(const void *src, int64_t at, bool bf16, float (&v)[8], int to) {
  if (bf16) {
    const v2u w = *reinterpret_cast<const v2u *>(static_cast<const uint16_t *>(src) + at);
    v[to] = __builtin_bit_cast(float, w[0] << 16);
    v[to + 1] = __builtin_bit_cast(float, w[0] & 0xffff0000u);
    v[to + 2] = __builtin_bit_cast(float, w[1] << 16);
    v[to + 3] = __builtin_bit_cast(float, w[1] & 0xffff0000u);
  } else {
    const v4f w = *reinterpret_cast<const v4f *>(static_cast<const float *>(src) + at);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[to + i] = w[i];
  }
}
__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
  const v2b r = {(__bf16)a, (__bf16)b};
  return __builtin_bit_cast(uint32_t, r);
}
__device__ __forceinline__ void store4(void *out, int64_t at, bool bf16, const float (&v)[8], int from) {
  if (bf16)
    *reinterpret_cast<v2u *>(static_cast<uint16_t *>(out) + at) =
        v2u{pack_bf16(v[from], v[from + 1]), pack_bf16(v[from + 2], v[from + 3])};
  else
    *reinterpret_cast<v4f *>(static_cast<float *>(out) + at) = v4f{v[from], v[from + 1], v[from + 2], v[from + 3]};
}

// A norm weight's values at a lane's dims, 4 at a time (a choice for each
// value would wait for eight loads one after the other).  A weight lies where
// its own type may.
typedef uint32_t v2u_any __attribute__((ext_vector_type(2), aligned(2)));
typedef float v4f_any __attribute__((ext_vector_type(4), aligned(4)));
__device__ __forceinline__ void load_weight(const void *w, bool bf16, const Dims &d, float (&v)[8]) {
  if (w == nullptr) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = 1.0f;
  } else if (bf16) {
    const uint16_t *p = static_cast<const uint16_t *>(w);
    const v2u_any x[2] = {*reinterpret_cast<const v2u_any *>(p + d.a), *reinterpret_cast<const v2u_any *>(p + d.b)};
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = bf16_bits_to_f32((uint16_t)(x[i / 4][i % 4 / 2] >> (16 * (i & 1))));
  } else {
    const float *p = static_cast<const float *>(w);
    const v4f_any x[2] = {*reinterpret_cast<const v4f_any *>(p + d.a), *reinterpret_cast<const v4f_any *>(p + d.b)};
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = x[i / 4][i % 4];
  }
}

// Norm and rotation of a head's 8 values in this lane, in T.  kAdjacent, which
// names the registers of a pair, is a branch of the caller's.
template <typename T, int D, bool kAdjacent>
__device__ __forceinline__ void turn_head(float (&v)[8], const RopeLaunch &r, bool norm, const float (&w)[8],
                                          const Turn &t, bool rotated) {
  T x[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = (T)v[i];
  if (norm) {
    T q = x[0] * x[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) q = __builtin_elementwise_fma(x[i], x[i], q);
    const T f = inv_sqrt(lanes_sum<D / 8>(q) * (T)(1.0 / D) + (T)r.eps);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] *= f * (T)w[i];
  }
  if (rotated) {
    T y[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int a = kAdjacent ? 2 * i : i, b = kAdjacent ? 2 * i + 1 : i + 4;
      const T c = (T)t.c[i], s = (T)t.s[i];
      y[a] = __builtin_elementwise_fma(x[a], c, -(x[b] * s));
      y[b] = __builtin_elementwise_fma(x[b], c, x[a] * s);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = y[i];
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = (float)x[i];
}

// A row's heads [h0, h1) of one kind.
struct HeadRange {
  HeadRows m;
  const void *weight;
  int h0, h1;
};

// A lane's 8 values of a head as they lie in memory.
template <bool kBf16>
struct HeadValues {
  using Half = typename std::conditional<kBf16, v2u, v4f>::type;
  Half w[2];
  __device__ __forceinline__ void load(const void *src, int64_t at, const Dims &d) {
    using T = typename std::conditional<kBf16, uint16_t, float>::type;
    const T *p = static_cast<const T *>(src) + at;
    w[0] = *reinterpret_cast<const Half *>(p + d.a);
    w[1] = *reinterpret_cast<const Half *>(p + d.b);
  }
  __device__ __forceinline__ float operator[](int i) const {
    if constexpr (!kBf16) return w[i / 4][i % 4];
    else return __builtin_bit_cast(float, i & 1 ? w[i / 4][i % 4 / 2] & 0xffff0000u : w[i / 4][i % 4 / 2] << 16);
  }
};

// Heads of one row, by one wave, 512/D at a time: those of `one`, then those
// of `two`, kAhead steps of loads on their way.  The first go out before the
// row's cosines are computed, a pair or two a lane, and passed round through
// `turns` (the wave's own).  A pair's values, weights, cosine and sine meet in
// four products that are the row's, so a head costs two products a value and
// its norm one more.
template <int D, bool kIn16, bool kOut16, bool kAdjacent>
__device__ __forceinline__ void turn_row(const RopeLaunch &r, const HeadRange &one, const HeadRange &two, int64_t row,
                                         int32_t pos, int lane, float2 (&turns)[D / 2]) {
  constexpr int L = D / 8, kHeads = 64 / L, kAhead = 4;
  const int c = lane % L;
  const Dims d(r, c);
  const bool rotated = 8 * c < r.rot_dim;
  const int n1 = (max(one.h1 - one.h0, 0) + kHeads - 1) / kHeads;
  const int n = n1 + (max(two.h1 - two.h0, 0) + kHeads - 1) / kHeads;
  if (n == 0) return;
  HeadValues<kIn16> v[kAhead];
  auto head = [&](int i) { return (i < n1 ? one.h0 + i * kHeads : two.h0 + (i - n1) * kHeads) + lane / L; };
  auto load = [&](int i) {
    const int h = min(head(i), (i < n1 ? one.h1 : two.h1) - 1);
    v[i % kAhead].load(i < n1 ? one.m.src : two.m.src, row * (i < n1 ? one.m.stride : two.m.stride) + (int64_t)h * D, d);
  };
#pragma unroll
  for (int i = 0; i < kAhead; ++i)
    if (i < n) load(i);
  float w[2][8];
  load_weight(one.weight, r.norm_bf16 != 0, d, w[0]);
  load_weight(two.weight, r.norm_bf16 != 0, d, w[1]);
  int32_t at[4] = {pos, pos, pos, pos};
  if (r.positions != nullptr)
#pragma unroll
    for (int a = 0; a < 4; ++a) at[a] = r.positions[(int64_t)min(a, r.n_axes - 1) * r.n_rows + row];
#pragma unroll
  for (int pair = lane; pair < D / 2; pair += 64) {
    if (2 * pair >= r.rot_dim) break;
    double si, co;
    sin_cos(angle(r, pair, at), si, co);
    turns[pair] = float2{(float)co, (float)si};
  }
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  // y[a] = x[a] * ca + x[b] * -sb, y[b] = x[b] * cb + x[a] * sa
  float ca[4], cb[4], sa[4], sb[4];
  auto weigh = [&](const float (&x)[8]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float wa = x[kAdjacent ? 2 * i : i], wb = x[kAdjacent ? 2 * i + 1 : i + 4];
      const float2 u = rotated ? turns[4 * c + i] : float2{1.0f, 0.0f};
      ca[i] = u.x * wa;
      cb[i] = u.x * wb;
      sa[i] = u.y * wa;
      sb[i] = u.y * wb;
    }
  };
  weigh(w[0]);
  for (int base = 0; base < n; base += kAhead)
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int i = base + k;
      if (i >= n) break;
      if (i == n1) weigh(w[1]);
      const HeadValues<kIn16> &x = v[k];
      const bool norm = (i < n1 ? one.weight : two.weight) != nullptr;
      float f = 1.0f;
      if (norm) {
        float q = x[0] * x[0];
#pragma unroll
        for (int e = 1; e < 8; ++e) q = __builtin_fmaf(x[e], x[e], q);
        f = inv_sqrt(lanes_sum<L>(q) * (1.0f / D) + r.eps);
      }
      float y[8];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int a = kAdjacent ? 2 * e : e, b = kAdjacent ? 2 * e + 1 : e + 4;
        y[a] = x[a] * ca[e];
        y[b] = x[b] * cb[e];
        if (rotated) {  // (not a sine of 0: it would make NaN of an infinite partner)
          y[a] = __builtin_fmaf(x[b], -sb[e], y[a]);
          y[b] = __builtin_fmaf(x[a], sa[e], y[b]);
        }
      }
      if (norm) {
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] *= f;
      }
      if (i + kAhead < n) load(i + kAhead);
      const int h = head(i);
      if (h < (i < n1 ? one.h1 : two.h1)) {
        void *out = i < n1 ? one.m.out : two.m.out;
        const int64_t to = row * (i < n1 ? one.m.out_stride : two.m.out_stride) + (int64_t)h * D;
        store4(out, to + d.a, kOut16, y, 0);
        store4(out, to + d.b, kOut16, y, 4);
      }
    }
}

template <int D, bool kIn16, bool kOut16>
__device__ __forceinline__ void turn_row(const RopeLaunch &r, const HeadRange &one, const HeadRange &two, int64_t row,
                                         int32_t pos, int lane, float2 (&turns)[D / 2]) {
  if (r.adjacent) turn_row<D, kIn16, kOut16, true>(r, one, two, row, pos, lane, turns);
  else turn_row<D, kIn16, kOut16, false>(r, one, two, row, pos, lane, turns);
}
#endif  // __HIP_DEVICE_COMPILE__

// Bound by memory from about 8000 rows on: 32,768 rows of 18 heads of 128 bf16
// values 52.5 us, 5.8 TB/s read and written; 4099 rows 8.9 us, 4.2 TB/s; a
// single row is a launch.  Four rows a workgroup, a row a wave; blockIdx.y: which `chunk` of the row's
// query heads and then key heads, counted through.
template <int D, bool kIn16, bool kOut16>
__global__ __launch_bounds__(256) void rope_rows_kernel(RopeLaunch r, HeadRows q, HeadRows k, int32_t chunk) {
#if defined(__HIP_DEVICE_COMPILE__)
  __shared__ __attribute__((aligned(16))) float2 turns[4][D / 2];
  const int wave = (int)__builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t row = (int64_t)blockIdx.x * 4 + wave;
  if (row >= r.n_rows) return;
  const int h0 = (int)blockIdx.y * chunk, h1 = h0 + chunk;
  turn_row<D, kIn16, kOut16>(r, HeadRange{q, r.q_norm, h0, min(h1, q.heads)},
                             HeadRange{k, r.k_norm, max(h0 - q.heads, 0), min(h1 - q.heads, k.heads)}, row,
                             r.own != nullptr ? r.own[row] : 0, threadIdx.x & 63, turns[wave]);
#endif
}

// ---- append ------------------------------------------------------------------------
// kv heads of a workgroup, which share a row's cosines: two of a large call's
// rows (65,619 rows of 2 heads into 4-bit pages 82 -> 74 us without queries, 38
// unrotated), one of a small call's, where the second would wait for the first
// (64 rows 9.1 -> 12.8 us a call).
constexpr int append_heads(int rows) { return rows == 32 ? 2 : 1; }

#if defined(__HIP_DEVICE_COMPILE__)

// E2M1 codes of this lane's 8 values of a block held by 4 consecutive lanes,
// and the block's exponent (999: not finite).
template <int kKind>
__device__ __forceinline__ uint32_t mx4_quantize8(const float (&v)[8], int32_t &e) {
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) top = max(top, __builtin_bit_cast(uint32_t, v[i]) & 0x7fffffffu);
  top = max(top, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, 0xb1, 0xf, 0xf, false));
  top = max(top, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, 0x4e, 0xf, 0xf, false));
  // |v| = m * 2^x, m in [1, 2): at most 7 * 2^(x-2) up to m = 1.75
  e = (int32_t)(top >> 23) - 127 - ((top & 0x7fffffu) <= 0x600000u ? 2 : 1);
  e = min(max(e, kKind == 0 ? kMx4KMin : kMx4VMin), kKind == 0 ? kMx4KMax : kMx4VMax);
  const float scale = __builtin_bit_cast(float, (uint32_t)(e + 127) << 23);
  uint32_t w = 0;
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[0], v[1], scale, 0);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[2], v[3], scale, 1);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[4], v[5], scale, 2);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[6], v[7], scale, 3);
  if (top >= 0x7f800000u) {
    e = 999;
    w = 0;
  }
  return w;
}

// The low nibbles of 8 bytes, byte k to nibble k.
__device__ __forceinline__ uint32_t low_nibbles(uint32_t w0, uint32_t w1) {
  w0 &= 0x0f0f0f0fu;
  w1 &= 0x0f0f0f0fu;
  w0 = (w0 | w0 >> 4) & 0x00ff00ffu;
  w1 = (w1 | w1 >> 4) & 0x00ff00ffu;
  return ((w0 | w0 >> 8) & 0xffffu) | (w1 | w1 >> 8) << 16;
}
#endif  // __HIP_DEVICE_COMPILE__

// Workgroup x = i * every, i < append_blocks, takes input rows [ROWS*(i /
// groups), +ROWS) and kv heads [kHeads*(i % groups), +kHeads); the others are
// the query waves (rope_rows_kernel's, keys none).
//  1. wave 0 finds each row's page and slot; rows that have none are reported
//     and skipped.
//  2. 512/D rows a wave: K normed and rotated in f64, through LDS into 8
//     consecutive dims a lane, V as it is, both quantized by 4 lanes a block;
//     codes and scales to LDS.
//  3. Runs to the pages, a wave each.  A run is the rows that follow each other
//     inside one group of slots whose V codes share words of a page (4 tokens
//     of a Q8_0 tile's dim, 8 of a 4-bit one's); the workgroup that holds its
//     first row takes all of it (rows past its own among them), and stores
//     whole words, 16 bytes a lane.  A run that does not fill its group leaves
//     the other tokens' bits alone: bytes, and in 4-bit pages an atomic xor of
//     the V words' own bits (another run of the call may hold the rest).
// Bound by memory but for the f64 of the rotation: 65,619 rows of 16 query and
// 2 kv heads of 256 bf16 values into 4-bit pages 232 us, 5.3 TB/s read and
// written; their keys and values alone 75 us, 39 unrotated.  4096 rows into
// Q8_0 pages 21 us, 64 rows 9 us (latency: page ids, rows, runs).
template <int D, bool kMx4, int ROWS, bool kBf16>
__global__ __launch_bounds__(256) void append_rope_kernel(AppendRopeLaunch p, int32_t groups, uint32_t append_blocks,
                                                          uint32_t every, int32_t chunk) {
#if defined(__HIP_DEVICE_COMPILE__)
  constexpr int L = D / 8, RW = 64 / L, NB = D / 32, H = D / 128;
  constexpr int GROUP = kMx4 ? 8 : 4;        // tokens of a V word
  constexpr int VR = ROWS + GROUP - 1;       // rows a workgroup may take
  constexpr int CB = kMx4 ? D / 2 : D;       // code bytes of a row
  constexpr int CS = CB + 16;                // LDS row stride
  constexpr int kHeads = append_heads(ROWS);
  __shared__ __attribute__((aligned(16))) float turned[4][RW][D];
  __shared__ __attribute__((aligned(16))) uint8_t codes[kHeads][2][VR][CS];
  __shared__ uint16_t scales[kHeads][2][VR][NB];
  __shared__ int64_t rbase[VR + 1];  // the row's page, bytes into the pool; -1: skip
  __shared__ int32_t rslot[VR + 1], rpos[VR + 1];
  __shared__ uint64_t starts;        // rows that start a run
  __shared__ int32_t vend;           // end of the rows that this workgroup's runs take
  const AppendLaunch &a = p.a;
  const Geo g = a.g;
  const int tid = (int)threadIdx.x, lane = tid & 63;
  const int wave = (int)__builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t nth = blockIdx.x / every;
  if (nth >= append_blocks || blockIdx.x % every != 0) {
    const uint32_t nq = (uint32_t)(p.q.heads + chunk - 1) / (uint32_t)chunk, x = blockIdx.x - min(nth + 1, append_blocks);
    const int64_t row = (int64_t)(x / nq) * 4 + wave;
    const int at = (int)(x % nq) * chunk;
    if (row < a.n_rows)
      turn_row<D, kBf16, kBf16>(p.r, HeadRange{p.q, p.r.q_norm, at, min(p.q.heads, at + chunk)},
                                HeadRange{p.q, nullptr, 0, 0}, row, a.positions[row], lane,
                                *reinterpret_cast<float2(*)[D / 2]>(&turned[wave][0][0]));
    return;
  }
  const int64_t row0 = (int64_t)(nth / groups) * ROWS;
  const int h0 = (int)(nth % groups) * kHeads, nh = min(g.kv_heads - h0, kHeads);
  const int nr = (int)min<int64_t>(ROWS, (int64_t)a.n_rows - row0);
  const uint64_t PB = kMx4 ? mx4_page_bytes(g) : page_bytes(g);
  const uint64_t RB = kMx4 ? mx4_region_bytes(g) : region_bytes(g);

  if (wave == 0) {
    const bool in = lane <= VR && row0 + lane < a.n_rows;
    int32_t seq = -1, pos = -1;
    if (in) {
      seq = a.seq_ids[row0 + lane];
      pos = a.positions[row0 + lane];
    }
    int32_t pseq = __shfl_up(seq, 1), ppos = __shfl_up(pos, 1);
    if (lane == 0 && row0 > 0) {
      pseq = a.seq_ids[row0 - 1];
      ppos = a.positions[row0 - 1];
    }
    int64_t base = -1;
    int32_t bad = 0;
    if (in) {
      if (seq < 0 || seq >= a.n_seqs) bad = FAULT_BAD_SEQ;
      else if (pos < 0 || pos / g.page_tokens >= a.bt_stride) bad = FAULT_BAD_POSITION;
      else {
        const int32_t page = a.bt[(int64_t)seq * a.bt_stride + pos / g.page_tokens];
        if (page < 0 || page >= g.num_pages) bad = FAULT_BAD_PAGE;
        else base = (int64_t)((uint64_t)page * PB);
      }
      if (bad != 0 && h0 == 0 && lane < nr) atomicOr(a.fault, bad);
    }
    const bool follows = (lane > 0 || row0 > 0) && seq == pseq && pos > 0 && pos - 1 == ppos && pos % GROUP != 0;
    const uint64_t s = __ballot(in && !follows);
    if (lane <= VR) {
      rbase[lane] = base;
      rslot[lane] = pos % g.page_tokens;
      rpos[lane] = pos;
    }
    if (lane == 0) {
      const int avail = (int)min<int64_t>(VR, (int64_t)a.n_rows - row0);
      const uint64_t mine = s & ((1ull << nr) - 1ull), later = s & ~((1ull << nr) - 1ull);
      starts = mine;
      vend = mine == 0 ? 0 : later == 0 ? avail : min(avail, (int)__builtin_ctzll(later));
    }
  }
  __syncthreads();
  const uint64_t runs = starts;
  const int v0 = runs != 0 ? (int)__builtin_ctzll(runs) : 0, v1 = vend;

  // ---- quantized rows to LDS ------------------------------------------------------
  const int c = lane % L, sub = lane / L;
  const Dims d(p.r, c);
  const bool rotated = p.r.on && 8 * c < p.r.rot_dim;
  float w[8];
  load_weight(p.r.on ? p.r.k_norm : nullptr, p.r.norm_bf16 != 0, d, w);
  for (int i = v0 + RW * wave; i < v1; i += 4 * RW) {
    const int r = min(i + sub, v1 - 1);
    float k[kHeads][8], v[kHeads][8];
#pragma unroll
    for (int h = 0; h < kHeads; ++h) {
      const int64_t hd = (int64_t)(h0 + min(h, nh - 1)) * D;
      const int64_t ka = (row0 + r) * p.k_stride + hd, va = (row0 + r) * p.v_stride + hd + 8 * c;
      load4(a.k_src, ka + d.a, kBf16, k[h], 0);
      load4(a.k_src, ka + d.b, kBf16, k[h], 4);
      load4(a.v_src, va, kBf16, v[h], 0);
      load4(a.v_src, va + 4, kBf16, v[h], 4);
    }
    Turn t;
    if (p.r.on) t.load(p.r, row0 + r, rpos[r], c);
#pragma unroll
    for (int h = 0; h < kHeads; ++h) {
      if (h >= nh) break;
      if (p.r.on && p.r.adjacent) turn_head<double, D, true>(k[h], p.r, p.r.k_norm != nullptr, w, t, rotated);
      else if (p.r.on) turn_head<double, D, false>(k[h], p.r, p.r.k_norm != nullptr, w, t, rotated);
      // K to 8 consecutive dims a lane, within the wave
      float *row = turned[wave][sub];
      *reinterpret_cast<v4f *>(row + d.a) = v4f{k[h][0], k[h][1], k[h][2], k[h][3]};
      *reinterpret_cast<v4f *>(row + d.b) = v4f{k[h][4], k[h][5], k[h][6], k[h][7]};
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
      __builtin_amdgcn_wave_barrier();
      const v4f x0 = *reinterpret_cast<const v4f *>(row + 8 * c), x1 = *reinterpret_cast<const v4f *>(row + 8 * c + 4);
      __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        k[h][e] = x0[e];
        k[h][4 + e] = x1[e];
      }
      uint16_t ks, vs;
      if constexpr (kMx4) {
        int32_t ke, ve;
        const uint32_t kq = mx4_quantize8<0>(k[h], ke), vq = mx4_quantize8<1>(v[h], ve);
        *reinterpret_cast<uint32_t *>(&codes[h][0][r][4 * c]) = kq;
        *reinterpret_cast<uint32_t *>(&codes[h][1][r][4 * c]) = vq;
        ks = ke == 999 ? 255 : (uint16_t)(ke + 127);
        vs = ve == 999 ? 0x7e : (uint16_t)(4 * (ve + 23));
      } else {
        const uint64_t kq = q8_quantize_values<8>(k[h], a.rule, ks), vq = q8_quantize_values<8>(v[h], a.rule, vs);
        *reinterpret_cast<uint64_t *>(&codes[h][0][r][8 * c]) = kq;
        *reinterpret_cast<uint64_t *>(&codes[h][1][r][8 * c]) = vq ^ 0x8080808080808080ull;  // stored biased (code_bias)
      }
      if (c % 4 == 0) {
        scales[h][0][r][c / 4] = ks;
        scales[h][1][r][c / 4] = vs;
      }
    }
  }
  __syncthreads();

  // ---- runs to the pages ------------------------------------------------------------
  int at = 0;
  for (uint64_t left = runs; left != 0; left &= left - 1, ++at) {
    const int r = (int)__builtin_ctzll(left);
    const uint64_t next = left & (left - 1);
    const int n = (next != 0 ? (int)__builtin_ctzll(next) : v1) - r;  // 1..GROUP rows
    const int64_t base = rbase[r];
    if (base < 0) continue;
    const int slot = rslot[r], first = slot % GROUP;
    for (int h = 0; h < nh; ++h) {
      if ((at * nh + h) % 4 != wave) continue;
      uint8_t *kr = a.pages + base + (uint64_t)(2 * (h0 + h)) * RB, *vr = kr + RB;
      const auto &kc = codes[h][0], &vc = codes[h][1];
      const auto &ks = scales[h][0], &vs = scales[h][1];
      if constexpr (kMx4) {
        const uint64_t tile = (uint64_t)(slot / 32) * mx4_tile_bytes(D);
        const int grp = slot % 32 / 8;
        if (lane < 32 * H) {  // K: (j, h, b, token of 4), a block each
          const int jh = lane / 16, b = lane / 4 % 4, m = lane % 4, k = 4 * (jh / H) + m - first;
          if (k >= 0 && k < n)
            *reinterpret_cast<v4u *>(kr + tile + (jh * 4 + b) * 256 + (4 * grp + m) * 16) =
                *reinterpret_cast<const v4u *>(&kc[r + k][16 * (jh % H * 4 + b)]);
        }
        if (lane < 32 * H) {  // K scales: (b, token of 4, j, h), bytes that lie side by side
          const int b = lane / (8 * H), m = lane / (2 * H) % 4, jh = lane % (2 * H), k = 4 * (jh / H) + m - first;
          if (k >= 0 && k < n)
            kr[tile + 16 * D + (b * 16 + 4 * grp + m) * 2 * H + jh] = (uint8_t)ks[r + k][jh % H * 4 + b];
        }
        if (lane < D / 4) {  // V: (c, n), 4 words, of the even and odd dims 2n of blocks 2c and 2c + 1
          const int cc = lane / 16, nn = lane % 16;
          uint32_t b[2][2] = {{0, 0}, {0, 0}};
#pragma unroll
          for (int t = 0; t < 8; ++t) {
            if (t < first || t >= first + n) continue;
#pragma unroll
            for (int u = 0; u < 2; ++u)
              b[u][t / 4] |= (uint32_t)vc[r + t - first][32 * cc + 16 * u + nn] << (8 * (t % 4));
          }
          const v4u q = {low_nibbles(b[0][0], b[0][1]), low_nibbles(b[0][0] >> 4, b[0][1] >> 4),
                         low_nibbles(b[1][0], b[1][1]), low_nibbles(b[1][0] >> 4, b[1][1] >> 4)};
          uint32_t *dst = reinterpret_cast<uint32_t *>(vr + tile + cc * 1024 + (grp * 16 + nn) * 16);
          if (n == 8) {
            *reinterpret_cast<v4u *>(dst) = q;
          } else {
            const uint32_t own = ((1u << (4 * n)) - 1u) << (4 * first);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const uint32_t was = __hip_atomic_load(dst + k, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
              const uint32_t flip = (was ^ q[k]) & own;
              if (flip != 0) atomicXor(dst + k, flip);
            }
          }
        }
        if (lane < NB * 8) {
          const int blk = lane / 8, k = lane % 8 - first;
          if (k >= 0 && k < n) vr[tile + 16 * D + (grp * NB + blk) * 8 + lane % 8] = (uint8_t)vs[r + k][blk];
        }
      } else {
        // K rows of neighbouring slots lie one behind the other
        if (16 * lane < n * D) {
          const int k = 16 * lane / D, x = 16 * lane % D;
          *reinterpret_cast<v4u *>(kr + (uint64_t)slot * D + 16 * lane) = *reinterpret_cast<const v4u *>(&kc[r + k][x]);
        }
        for (int x = lane; x < D; x += 64) {
          uint8_t *dst = vr + code_offset(g, 1, slot, x);
          if (n == 4) {
            *reinterpret_cast<uint32_t *>(dst) = (uint32_t)vc[r][x] | (uint32_t)vc[r + 1][x] << 8 |
                                                 (uint32_t)vc[r + 2][x] << 16 | (uint32_t)vc[r + 3][x] << 24;
          } else {
            for (int k = 0; k < n; ++k) dst[k] = vc[r + k][x];
          }
        }
        if (lane < NB * 8) {
          const int kind = lane / (NB * 4), blk = lane / 4 % NB, k = lane % 4;
          if (k < n)
            *reinterpret_cast<uint16_t *>((kind ? vr : kr) + scale_offset(g, slot + k, blk)) =
                kind ? vs[r + k][blk] : ks[r + k][blk];
        }
      }
    }
  }
#endif  // __HIP_DEVICE_COMPILE__
}

// ---- rows read back -----------------------------------------------------------------

// One thread per 8 consecutive dims of a row; blockIdx.y: (kv head, kind).  A
// V row's values lie 8 (Q8_0: 32) tokens apart, so rows that follow each other
// share their lines in the L1.  65,619 rows of 4-bit pages into bf16 50 us (170
// MB in all), 4096 of Q8_0 9 us.
template <int D, bool kMx4>
__global__ __launch_bounds__(256) void read_rows_kernel(ReadRowsLaunch p) {
#if defined(__HIP_DEVICE_COMPILE__)
  constexpr int L = D / 8, NB = D / 32;
  const AppendLaunch &a = p.a;
  const Geo g = a.g;
  const int c = (int)threadIdx.x % L;
  const int kind = (int)blockIdx.y & 1, h = (int)blockIdx.y >> 1;
  const int64_t row = (int64_t)blockIdx.x * (256 / L) + threadIdx.x / L;
  void *out = kind == 0 ? p.k_out : p.v_out;
  if (row >= a.n_rows) return;
  const int32_t seq = a.seq_ids[row], pos = a.positions[row];
  int32_t bad = 0, page = 0;
  const uint32_t upos = (uint32_t)pos, PT = (uint32_t)g.page_tokens;
  if (seq < 0 || seq >= a.n_seqs) bad = FAULT_BAD_SEQ;
  else if (pos < 0 || upos / PT >= (uint32_t)a.bt_stride) bad = FAULT_BAD_POSITION;
  else {
    page = a.bt[(int64_t)seq * a.bt_stride + upos / PT];
    if (page < 0 || page >= g.num_pages) bad = FAULT_BAD_PAGE;
  }
  if (bad != 0 && c == 0 && blockIdx.y == 0) atomicOr(a.fault, bad);
  if (out == nullptr) return;
  const int64_t at = (row * g.kv_heads + h) * D + 8 * c;
  const int slot = (int)(upos % PT), blk = c / 4;
  if constexpr (kMx4) {
    uint32_t q = 0, s = 0;
    if (bad == 0) {
      const uint8_t *tile = a.pages + mx4_region_base(g, page, h, kind) + (uint64_t)(slot / 32) * mx4_tile_bytes(D);
      const int tok = slot % 32;
      if (kind == 0) {
        const int j = tok % 8 / 4, m = 4 * (tok / 8) + tok % 4, jh = j * (D / 128) + blk / 4;
        q = *reinterpret_cast<const uint32_t *>(tile + (jh * 4 + blk % 4) * 256 + m * 16 + 4 * (c % 4));
        s = tile[16 * D + (blk % 4 * 16 + m) * (D / 64) + jh];
      } else {
        const int grp = tok / 8, nib = 4 * (tok % 8);
        v2u w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)  // dims 32*blk + 8*(c % 4) + 2*i, +1
          w[i] = *reinterpret_cast<const v2u *>(tile + blk / 2 * 1024 + (grp * 16 + 4 * (c % 4) + i) * 16 + 8 * (blk % 2));
        s = tile[16 * D + (grp * NB + blk) * 8 + tok % 8];
#pragma unroll
        for (int i = 0; i < 4; ++i) q |= (w[i][0] >> nib & 15u) << (8 * i) | (w[i][1] >> nib & 15u) << (8 * i + 4);
        s = s >= 0x7c ? 255 : s / 4 - 23 + 127;  // as K's
      }
    }
    const float scale = __builtin_bit_cast(float, s << 23);  // (255: NaN)
    if (p.out_bf16 != 0) {
      const v2b w0 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, scale, 0), w1 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, scale, 1),
                w2 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, scale, 2), w3 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, scale, 3);
      *reinterpret_cast<v4u *>(static_cast<uint16_t *>(out) + at) =
          v4u{__builtin_bit_cast(uint32_t, w0), __builtin_bit_cast(uint32_t, w1), __builtin_bit_cast(uint32_t, w2),
              __builtin_bit_cast(uint32_t, w3)};
    } else {
      const v2f w0 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, scale, 0), w1 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, scale, 1),
                w2 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, scale, 2), w3 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, scale, 3);
      v4f *dst = reinterpret_cast<v4f *>(static_cast<float *>(out) + at);
      dst[0] = v4f{w0[0], w0[1], w1[0], w1[1]};
      dst[1] = v4f{w2[0], w2[1], w3[0], w3[1]};
    }
  } else {
    float v[8] = {};
    if (bad == 0) {
      const uint8_t *region = a.pages + region_base(g, page, h, kind);
      const float scale = f16_bits_to_f32(*reinterpret_cast<const uint16_t *>(region + scale_offset(g, slot, blk)));
      uint64_t q;  // the 8 codes
      if (kind == 0) {
        q = *reinterpret_cast<const uint64_t *>(region + (uint32_t)slot * D + 8 * c);
      } else {
        const uint32_t TT = (uint32_t)tile_tokens(g.page_tokens);
        const uint8_t *from = region + code_offset(g, 1, slot, 8 * c);
        q = 0x8080808080808080ull;  // stored biased (code_bias)
#pragma unroll
        for (int i = 0; i < 8; ++i) q ^= (uint64_t)from[TT * i] << (8 * i);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = scale * (float)(int8_t)(q >> (8 * i));
    }
    store4(out, at, p.out_bf16 != 0, v, 0);
    store4(out, at + 4, p.out_bf16 != 0, v, 4);
  }
#endif  // __HIP_DEVICE_COMPILE__
}

// Heads of a wave: a row's heads over so many waves that the launch has about
// 4096 (16 a CU), as each computes its row's cosines for all of them (2048 or
// 8192 waves: the same within 0.6 us from 1024 to 32,768 rows of 18 heads).
int32_t head_chunk(int64_t rows, int32_t heads, int32_t per) {
  const int64_t want = std::max<int64_t>(1, (int64_t)heads * rows / 4096);
  return (int32_t)std::min<int64_t>((want + per - 1) / per * per, (heads + per - 1) / per * per);
}

template <int D, bool kMx4, int ROWS>
void launch_append_rope_r(const AppendRopeLaunch &p, hipStream_t s) {
  const int64_t row_blocks = ((int64_t)p.a.n_rows + ROWS - 1) / ROWS;
  const int32_t groups = (p.a.g.kv_heads + append_heads(ROWS) - 1) / append_heads(ROWS);
  const uint32_t blocks = (uint32_t)(row_blocks * groups);
  uint32_t q_blocks = 0;
  int32_t chunk = 1;
  if (p.q.src != nullptr && p.q.bf16 == p.q.out_bf16) {
    chunk = head_chunk(p.a.n_rows, p.q.heads, 512 / D);
    q_blocks = (uint32_t)((p.a.n_rows + 3LL) / 4 * ((p.q.heads + chunk - 1) / chunk));
  }
  // A small call's append goes first, a large one's is spread over the launch:
  // its f64 then runs beside the queries' loads (65,619 rows in one launch 232
  // us, in two 256; an odd step, as every 8th workgroup is on one XCD: 449).
  uint32_t every = ROWS == 8 ? 1 : (blocks + q_blocks) / blocks;
  every -= every % 2 == 0;
  if (p.a.src_bf16)
    hipLaunchKernelGGL((append_rope_kernel<D, kMx4, ROWS, true>), dim3(blocks + q_blocks), dim3(256), 0, s, p, groups,
                       blocks, every, chunk);
  else
    hipLaunchKernelGGL((append_rope_kernel<D, kMx4, ROWS, false>), dim3(blocks + q_blocks), dim3(256), 0, s, p, groups,
                       blocks, every, chunk);
}
// 32-row workgroups once there are at least 8 per CU, else 8-row ones.
bool small_call(const AppendRopeLaunch &p) {
  return (int64_t)p.a.n_rows * p.a.g.kv_heads < (int64_t)32 * 8 * kComputeUnits;
}
// Queries of another type than the rows' go by themselves.
bool queries_with(const AppendRopeLaunch &p) { return p.q.bf16 == p.q.out_bf16; }
template <int D, bool kMx4>
void launch_append_rope_d(const AppendRopeLaunch &p, hipStream_t s) {
  if (small_call(p)) launch_append_rope_r<D, kMx4, 8>(p, s);
  else launch_append_rope_r<D, kMx4, 32>(p, s);
}

}  // namespace

hipError_t launch_rope_rows(const RopeLaunch &r, const HeadRows &q, const HeadRows &k, int32_t head_dim,
                            hipStream_t s) {
  if (r.n_rows <= 0 || q.heads + k.heads <= 0) return hipSuccess;
  const int32_t chunk = head_chunk(r.n_rows, q.heads + k.heads, 512 / head_dim);
  const dim3 grid((unsigned)((r.n_rows + 3LL) / 4), (unsigned)((q.heads + k.heads + chunk - 1) / chunk));
  const HeadRows &m = q.heads > 0 ? q : k;
  auto go = [&](auto d) {
    constexpr int D = decltype(d)::value;
    if (m.bf16 && m.out_bf16) hipLaunchKernelGGL((rope_rows_kernel<D, true, true>), grid, dim3(256), 0, s, r, q, k, chunk);
    else if (m.bf16) hipLaunchKernelGGL((rope_rows_kernel<D, true, false>), grid, dim3(256), 0, s, r, q, k, chunk);
    else if (m.out_bf16) hipLaunchKernelGGL((rope_rows_kernel<D, false, true>), grid, dim3(256), 0, s, r, q, k, chunk);
    else hipLaunchKernelGGL((rope_rows_kernel<D, false, false>), grid, dim3(256), 0, s, r, q, k, chunk);
  };
  if (head_dim == 256) go(std::integral_constant<int, 256>{});
  else go(std::integral_constant<int, 128>{});
  return hipGetLastError();
}

hipError_t launch_append_rope(const AppendRopeLaunch &p, hipStream_t s) {
  if (p.a.n_rows <= 0) return hipSuccess;
  if (p.q.src != nullptr && !queries_with(p)) {
    const hipError_t e = launch_rope_rows(p.r, p.q, HeadRows{}, p.a.g.head_dim, s);
    if (e != hipSuccess) return e;
  }
  if (p.a.g.head_dim == 256) {
    if (p.mx4) launch_append_rope_d<256, true>(p, s);
    else launch_append_rope_d<256, false>(p, s);
  } else {
    if (p.mx4) launch_append_rope_d<128, true>(p, s);
    else launch_append_rope_d<128, false>(p, s);
  }
  return hipGetLastError();
}

hipError_t launch_read_rows(const ReadRowsLaunch &p, hipStream_t s) {
  if (p.a.n_rows <= 0) return hipSuccess;
  const int rows = 256 / (p.a.g.head_dim / 8);  // of a workgroup
  const dim3 grid((unsigned)(((int64_t)p.a.n_rows + rows - 1) / rows), (unsigned)p.a.g.kv_heads * 2);
  if (p.a.g.head_dim == 256) {
    if (p.mx4) hipLaunchKernelGGL((read_rows_kernel<256, true>), grid, dim3(256), 0, s, p);
    else hipLaunchKernelGGL((read_rows_kernel<256, false>), grid, dim3(256), 0, s, p);
  } else {
    if (p.mx4) hipLaunchKernelGGL((read_rows_kernel<128, true>), grid, dim3(256), 0, s, p);
    else hipLaunchKernelGGL((read_rows_kernel<128, false>), grid, dim3(256), 0, s, p);
  }
  return hipGetLastError();
}

}  // namespace rkv
