// Helpers of the microscaled 4-bit format (gfx950 only): blocks of 32 E2M1
// codes along a row, one E8M0 scale byte each.
//
//   value = grid(code) * 2^(scale - 127), scale 255: NaN
//   scale = max(floor(log2 max|x|) - 2, -127) + 127, code = the nearest grid
//   value of x * 2^(127 - scale) (ties to the even code), at most 6
//
// Two codes a byte, the lower half first; a row holds KB = ceil(K / 32)
// blocks, 16 * KB bytes and KB scale bytes, and its last block is padded
// with zero codes.
#pragma once

#include "mxk_internal.h"

namespace mxk {

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2f __attribute__((ext_vector_type(2)));
typedef float f32x4f __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

inline int64_t fp4_blocks(int64_t cols) { return (cols + 31) / 32; }

// Scale byte s as the conversions' scale operand, of which they read the
// exponent field alone: 2^(s - 127), also for s = 0, and NaN for s = 255
__device__ __forceinline__ float e8m0_operand(uint32_t s) { return __uint_as_float(s << 23); }

// N elements of type T as the dwords that hold them
template <typename T, int N>
struct FpWords {
  static constexpr int NW = N * (int)sizeof(T) / 4;
  uint32_t w[NW];
};

// N elements at p, which needs no more alignment than an element's: global
// memory takes wide loads at any address (unaligned mode), at one
// instruction per 16 bytes
template <typename T, int N>
__device__ __forceinline__ void fp4_load(const T* p, FpWords<T, N>& v) {
  __builtin_memcpy(v.w, p, sizeof(v.w));
}
// the first `live` of them (the others read as +0), element by element
template <typename T, int N>
__device__ __forceinline__ void fp4_load_tail(const T* p, int live, FpWords<T, N>& v) {
  T e[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    uint32_t z = 0;
    __builtin_memcpy(&e[i], &z, sizeof(T));
    if (i < live) e[i] = p[i];
  }
  __builtin_memcpy(v.w, e, sizeof(v.w));
}

// Largest magnitude of the elements, as the bits of its float32 value (so
// that NaN and infinity compare above every number).  16-bit types compare
// as pairs of 16-bit integers.
typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
template <typename T, int N>
__device__ __forceinline__ uint32_t fp4_amax_bits(const FpWords<T, N>& v) {
  if constexpr (sizeof(T) == 4) {
    uint32_t m = v.w[0] & 0x7FFFFFFFu;
#pragma unroll
    for (int i = 1; i < N; ++i) m = max(m, v.w[i] & 0x7FFFFFFFu);
    return m;
  } else {
    u16x2 m = __builtin_bit_cast(u16x2, v.w[0] & 0x7FFF7FFFu);
#pragma unroll
    for (int i = 1; i < N / 2; ++i)
      m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, v.w[i] & 0x7FFF7FFFu));
    const uint32_t h = max((uint32_t)m[0], (uint32_t)m[1]);
    if constexpr (__is_same(T, __half))
      return __float_as_uint((float)__builtin_bit_cast(_Float16, (uint16_t)h));
    else
      return h << 16;
  }
}

// Scale byte of a block from the bits of its largest magnitude: the exponent
// field less 2 (E2M1's largest binade), at least 0; 255 for NaN and infinity
__device__ __forceinline__ uint32_t fp4_scale_byte(uint32_t amax_bits) {
  const uint32_t e = amax_bits >> 23;
  return e == 255u ? 255u : max(e, 2u) - 2u;
}

// Codes of the N elements (N / 8 dwords) for scale s = e8m0_operand(byte): the
// conversion divides by the power of two, rounds to the nearest even code
// and saturates at 6 (checked against the grid's midpoints)
template <typename T, int N>
__device__ __forceinline__ void fp4_codes(const FpWords<T, N>& v, float s, uint32_t (&q)[N / 8]) {
#pragma unroll
  for (int d = 0; d < N / 8; ++d) {
    uint32_t o = 0u;
    if constexpr (sizeof(T) == 4) {
      const float* f = reinterpret_cast<const float*>(v.w) + 8 * d;
      o = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(o, f[0], f[1], s, 0);
      o = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(o, f[2], f[3], s, 1);
      o = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(o, f[4], f[5], s, 2);
      o = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(o, f[6], f[7], s, 3);
    } else if constexpr (__is_same(T, __half)) {
      const uint32_t* w = v.w + 4 * d;
      o = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(o, __builtin_bit_cast(f16x2, w[0]), s, 0);
      o = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(o, __builtin_bit_cast(f16x2, w[1]), s, 1);
      o = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(o, __builtin_bit_cast(f16x2, w[2]), s, 2);
      o = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(o, __builtin_bit_cast(f16x2, w[3]), s, 3);
    } else {
      const uint32_t* w = v.w + 4 * d;
      o = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(o, __builtin_bit_cast(bf16x2, w[0]), s, 0);
      o = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(o, __builtin_bit_cast(bf16x2, w[1]), s, 1);
      o = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(o, __builtin_bit_cast(bf16x2, w[2]), s, 2);
      o = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(o, __builtin_bit_cast(bf16x2, w[3]), s, 3);
    }
    q[d] = o;
  }
}

// a float32 result as T, rounded to nearest even
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) {
  return __builtin_bit_cast(__half, (_Float16)v);
}
template <>
__device__ __forceinline__ hip_bfloat16 from_f32<hip_bfloat16>(float v) {
  return __builtin_bit_cast(hip_bfloat16, (__bf16)v);
}

// Slot s of the tiles of BM rows of all segments (the experts', then the rows
// behind the last of them and those in front of the first, which a part of a
// larger plan has): its segment and rows.  Offsets are brought into [0, M], so
// that no row outside the product is named whatever they hold.
struct Segment {
  int e;  // E: rows without an expert; E + 1: no tile
  int64_t lo, hi;
};
template <int BM>
__device__ __forceinline__ Segment find_segment(int64_t slot, const int* offsets, int E, int64_t M) {
  // one segment per lane, 64 at a time: tiles of the segments before by a scan
  const int lane = threadIdx.x & 63;
  Segment g = {E + 1, 0, 0};
  int64_t before = 0;
  for (int e0 = 0; e0 <= E + 1; e0 += 64) {
    const int e = e0 + lane;
    int64_t lo = 0, hi = 0;
    if (e <= E + 1) {
      lo = e > E ? 0 : (int64_t)offsets[e];
      hi = e == E ? M : (int64_t)offsets[e > E ? 0 : e + 1];
      lo = lo < 0 ? 0 : (lo > M ? M : lo);
      hi = hi < lo ? lo : (hi > M ? M : hi);
    }
    const int tiles = (int)((hi - lo + BM - 1) / BM);
    int upto = tiles;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int v = __shfl_up(upto, d);
      if (lane >= d) upto += v;
    }
    const int64_t at = slot - before;
    const uint64_t here = __ballot(at >= upto - tiles && at < upto);
    if (here) {
      const int src = __builtin_ctzll(here);
      const int first = __shfl(upto - tiles, src);
      const int64_t slo = __shfl((int)lo, src), shi = __shfl((int)hi, src);
      g.e = __builtin_amdgcn_readfirstlane(min(e0 + src, E));
      g.lo = __builtin_amdgcn_readfirstlane((int)(slo + (at - first) * BM));
      g.hi = __builtin_amdgcn_readfirstlane((int)(shi < slo + (at - first + 1) * BM ? shi : slo + (at - first + 1) * BM));
      return g;
    }
    before += __shfl(upto, 63);
  }
  return g;
}
// Slots that cover every case of M rows in E segments and the two of rows without
// an expert: each segment wastes less than a tile, and no tile is empty
inline int64_t segment_slots(int64_t M, int E, int BM) {
  return std::min<int64_t>(M, (M + (int64_t)(E + 2) * (BM - 1)) / BM);
}

// Tile t of a grid of tm x tn, taken so that the workgroups of one XCD
// (blockIdx % 8) are consecutive tiles of an order that walks 8 rows of tiles
// down before it goes right: the 32 tiles an XCD holds at once share 8 row
// and 4 column panels in its L2.
__device__ __forceinline__ void place_tile(uint32_t id, uint32_t tm, uint32_t tn, uint32_t& m, uint32_t& n) {
  const uint32_t total = tm * tn, xcd = id & 7u, local = id >> 3;
  const uint32_t per = total >> 3, rest = total & 7u;
  const uint32_t t = xcd * per + min(xcd, rest) + local;
  const uint32_t group = t / (8u * tn), in = t - group * 8u * tn;
  const uint32_t high = min(8u, tm - group * 8u);
  n = in / high;
  m = group * 8u + (in - n * high);
}

// The same for products by expert, of whose tm rows of tiles only the first
// ones are in use (how many is not known on the host): blocks of 8 x 4 tiles in
// turn to the XCDs, so that each has its share of those.  false: no such tile.
__device__ __forceinline__ bool place_block_tile(uint32_t id, uint32_t tm, uint32_t tn, uint32_t& m, uint32_t& n) {
  const uint32_t local = id >> 3, block = (local >> 5) * 8u + (id & 7u), in = local & 31u;
  const uint32_t across = (tn + 3u) >> 2, row = block / across;
  m = row * 8u + (in & 7u);
  n = (block - row * across) * 4u + (in >> 3);
  return m < tm && n < tn;
}
// how many ids that takes
inline int64_t block_tile_ids(int64_t tm, int64_t tn) {
  return ceil_div(ceil_div(tm, 8) * ceil_div(tn, 4), 8) * 256;
}

}  // namespace mxk
