// Products of microscaled 4-bit operands for gfx950, dense and by expert:
//
//   y[m, n] = sum_k a[m, k] b[n, k] (+ bias[n])           (both packed along k)
//
// v_mfma_scale_f32_16x16x128_f8f6f4 takes the codes and their scale bytes as
// stored: a lane holds the 32 codes of one row and block (16 bytes) and that
// block's scale, so nothing is decoded, and products and sums are exact up to
// the float32 accumulator.
//
// By expert: rows [offsets[e], offsets[e + 1]) of a go through b[e], and rows
// past the last expert's are written as zeros; with `order` row r of the
// product is row order[r] / top of a.
#include "mxk_mxfp4.h"

namespace mxk {

struct Fp4Gemm {
  const uint8_t *a, *as, *b, *bs;
  int64_t a_rows, M, N, KB;  // rows of a, of the product, of b (per expert); blocks of a row
  const float* bias;         // [N] or, by expert, [E][N]; null: none
  void* y;
  const int* offsets;        // by expert: [E + 1]
  int E;
  const int* order;          // by expert: [M] or null
  DivU32 top;
};

// Slot s of the tiles of BM rows of all segments (the experts', then the rows
// without one): its segment and rows.  Offsets are brought into [0, M], so
// that no row outside the product is named whatever they hold.
struct Segment {
  int e;  // E: rows without an expert; E + 1: no tile
  int64_t lo, hi;
};
template <int BM>
__device__ __forceinline__ Segment find_segment(int64_t s, const int* offsets, int E, int64_t M) {
  Segment g;
  int64_t lo = 0;
  for (int e = 0; e <= E; ++e) {
    int64_t hi = e < E ? (int64_t)offsets[e + 1] : M;
    hi = hi < lo ? lo : (hi > M ? M : hi);
    const int64_t tiles = (hi - lo + BM - 1) / BM;
    if (s < tiles) {
      g.e = e;
      g.lo = lo + s * BM;
      g.hi = hi < g.lo + BM ? hi : g.lo + BM;
      return g;
    }
    s -= tiles;
    lo = hi;
  }
  g.e = E + 1;
  g.lo = g.hi = 0;
  return g;
}
// Slots that cover every case of M rows in E segments and the rows without an
// expert: each segment wastes less than a tile, and no tile is empty
static int64_t segment_slots(int64_t M, int E, int BM) {
  return std::min<int64_t>(M, (M + (int64_t)(E + 1) * (BM - 1)) / BM);
}

// Row of a that row r of the product reads, -1: none
__device__ __forceinline__ int64_t source_row(const Fp4Gemm& p, int64_t r) {
  if (!p.order) return r < p.a_rows ? r : -1;
  const int pick = p.order[r];
  if (pick < 0) return -1;
  const int64_t t = divu32((uint32_t)pick, p.top);
  return t < p.a_rows ? t : -1;
}

// 64 x 64 tiles of four waves (32 x 32 each), operands straight from memory.
template <typename T, bool EXPERT>
__global__ __launch_bounds__(256) void k_fp4_gemm(Fp4Gemm p) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int r = lane & 15, g = lane >> 4;
  const int64_t tiles_n = (p.N + 63) / 64;
  const int64_t slot = blockIdx.x / tiles_n, n0 = (blockIdx.x % tiles_n) * 64 + (wave & 1) * 32;
  int64_t lo = slot * 64, hi = p.M < lo + 64 ? p.M : lo + 64;
  int e = 0;
  if (EXPERT) {
    const Segment s = find_segment<64>(slot, p.offsets, p.E, p.M);
    e = s.e;
    lo = s.lo;
    hi = s.hi;
    if (e > p.E) return;
  }
  const bool none = EXPERT && e == p.E;
  const int64_t m0 = lo + (wave >> 1) * 32;
  const uint8_t *ap[2], *asp[2], *bp[2], *bsp[2];
  bool al[2], bl[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int64_t m = m0 + 16 * i + r, n = n0 + 16 * i + r;
    const int64_t src = m < hi && !none ? source_row(p, m) : -1;
    al[i] = src >= 0;
    ap[i] = p.a + (al[i] ? src : 0) * p.KB * 16;
    asp[i] = p.as + (al[i] ? src : 0) * p.KB;
    bl[i] = n < p.N && !none;
    const int64_t row = bl[i] ? (int64_t)e * p.N + n : 0;
    bp[i] = p.b + row * p.KB * 16;
    bsp[i] = p.bs + row * p.KB;
  }
  f32x4f acc[2][2];
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j) acc[i][j] = f32x4f{0, 0, 0, 0};
  if (!none) {
    for (int64_t k = g; k - g < p.KB; k += 4) {
      i32x8 A[2], B[2];
      int sa[2], sb[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        i32x4 va = {0, 0, 0, 0}, vb = {0, 0, 0, 0};
        sa[i] = sb[i] = 0;
        if (al[i] && k < p.KB) {
          va = *reinterpret_cast<const i32x4*>(ap[i] + k * 16);
          sa[i] = asp[i][k];
        }
        if (bl[i] && k < p.KB) {
          vb = *reinterpret_cast<const i32x4*>(bp[i] + k * 16);
          sb[i] = bsp[i][k];
        }
        A[i] = i32x8{va[0], va[1], va[2], va[3], 0, 0, 0, 0};
        B[i] = i32x8{vb[0], vb[1], vb[2], vb[3], 0, 0, 0, 0};
      }
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
          acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(B[j], A[i], acc[i][j], 4, 4, 0, sb[j], 0, sa[i]);
    }
  }
  T* y = reinterpret_cast<T*>(p.y);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int64_t m = m0 + 16 * i + r;
    if (m >= hi) continue;
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int64_t n = n0 + 16 * j + 4 * g + q;
        if (n >= p.N) continue;
        float v = acc[i][j][q];
        if (p.bias && !none) v += p.bias[(int64_t)e * p.N + n];
        y[m * p.N + n] = from_f32<T>(v);
      }
  }
}

static int launch_gemm(const Fp4Gemm& p, int y_type, hipStream_t st) {
  const bool ex = p.offsets != nullptr;
  const int64_t slots = ex ? segment_slots(p.M, p.E, 64) : ceil_div(p.M, 64);
  const int64_t n = slots * ceil_div(p.N, 64);
  if (n >= ((int64_t)1 << 31)) return fail(MXK_EINVAL, "mxfp4 product: too many tiles");
#define MXK_L(T)                                                                                         \
  do {                                                                                                   \
    if (ex) hipLaunchKernelGGL((k_fp4_gemm<T, true>), dim3((unsigned)n), dim3(256), 0, st, p);           \
    else hipLaunchKernelGGL((k_fp4_gemm<T, false>), dim3((unsigned)n), dim3(256), 0, st, p);             \
  } while (0)
  if (y_type == MXK_IN_F32) MXK_L(float);
  else if (y_type == MXK_IN_F16) MXK_L(__half);
  else MXK_L(hip_bfloat16);
#undef MXK_L
  return check_launch("mxfp4 product");
}

}  // namespace mxk

using namespace mxk;

extern "C" {

int mxk_mxfp4_matmul(const void* a_codes, const void* a_scales, int64_t a_rows, const void* b_codes,
                     const void* b_scales, int64_t M, int64_t N, int64_t K, const float* bias, int y_type, void* y,
                     const int32_t* offsets, int experts, const int32_t* order, int top, void* stream) {
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (a_rows < 0 || M < 0 || N < 0 || K < 0) return fail(MXK_EINVAL, "mxfp4_matmul: negative size");
  if (M >= ((int64_t)1 << 31) || N >= ((int64_t)1 << 31) || K >= ((int64_t)1 << 28) || a_rows >= ((int64_t)1 << 31))
    return fail(MXK_EINVAL, "mxfp4_matmul: rows below 2^31, K below 2^28");
  if (y_type != MXK_IN_F32 && y_type != MXK_IN_F16 && y_type != MXK_IN_BF16)
    return fail(MXK_EINVAL, "mxfp4_matmul: unknown y_type");
  if (offsets ? (experts < 1 || experts > 1000) : (order != nullptr || a_rows != M))
    return fail(MXK_EINVAL, "mxfp4_matmul: 1 to 1000 experts with offsets; without them no order and a_rows = M");
  if (order ? (top < 1) : (offsets && a_rows != M))
    return fail(MXK_EINVAL, "mxfp4_matmul: top at least 1 with an order, a_rows = M without one");
  if (M == 0 || N == 0) return MXK_OK;
  if (!y || (K > 0 && (!b_codes || !b_scales || (a_rows > 0 && (!a_codes || !a_scales)))))
    return fail(MXK_EINVAL, "mxfp4_matmul: null pointer");
  if (!aligned16(a_codes) || !aligned16(b_codes)) return fail(MXK_EINVAL, "mxfp4_matmul: codes must be 16-byte aligned");
  Fp4Gemm p;
  p.a = reinterpret_cast<const uint8_t*>(a_codes);
  p.as = reinterpret_cast<const uint8_t*>(a_scales);
  p.b = reinterpret_cast<const uint8_t*>(b_codes);
  p.bs = reinterpret_cast<const uint8_t*>(b_scales);
  p.a_rows = a_rows;
  p.M = M;
  p.N = N;
  p.KB = fp4_blocks(K);
  p.bias = bias;
  p.y = y;
  p.offsets = offsets;
  p.E = experts;
  p.order = order;
  p.top = make_divu32((uint32_t)(top < 1 ? 1 : top));
  return launch_gemm(p, y_type, st);
}

}  // extern "C"
