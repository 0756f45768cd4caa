// Gradients of the microscaled 4-bit products for gfx950 (straight through
// the quantizer): with y = a b^T over packed a [M][K] and b [N][K],
//
//   da[m, k] = sum_n dy[m, n] b[n, k]        db[n, k] = sum_m dy[m, n] a[m, k]
//
// dy is not quantized.  A code times its power-of-two scale has two
// significant bits and is exact in bfloat16, so the product runs on bf16
// MFMAs with dy as one bf16 term (bf16), two (f16) or three (f32) that add
// up to it exactly: every product is exact, sums are in float32.
#include "mxk_mxfp4.h"

namespace mxk {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

template <typename T> struct Planes { static constexpr int N = 1; };
template <> struct Planes<__half> { static constexpr int N = 2; };
template <> struct Planes<float> { static constexpr int N = 3; };

// v as the sum of N bf16 terms (16 bits each), truncated so that no term
// overflows; a NaN or infinity is the first term alone
template <int N>
__device__ __forceinline__ void split_bf16(float v, uint16_t (&t)[N]) {
  const bool finite = (__float_as_uint(v) & 0x7F800000u) != 0x7F800000u;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    uint32_t b = __float_as_uint(v);
    if (!finite) b = i ? 0u : (b & 0x007FFFFFu ? b | 0x00400000u : b);
    b &= 0xFFFF0000u;
    t[i] = (uint16_t)(b >> 16);
    v = v - __uint_as_float(b);
  }
}

// out[i, j] = sum_t L[i, t] V[t, j]: L = dy at l + i * si + t * st, V the
// packed rows, J = K columns
struct Fp4Grad {
  const void* l;
  int64_t si, st;
  const uint8_t *v, *vs;
  int64_t I, T, J, KB;
  void* out;
  const int* offsets;  // by expert: the segments of I (gradient of a) or of T (of b)
  int E;
  int64_t rows;        // by expert: rows of all segments
};

template <typename T, typename O, bool OF_B>
__global__ __launch_bounds__(256) void k_fp4_grad(Fp4Grad p) {
  constexpr int P = Planes<T>::N;
  __shared__ uint16_t Ls[P][64][40];
  __shared__ uint16_t Vs[64][40];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int r = lane & 15, g = lane >> 4;
  const int64_t tiles_j = (p.J + 63) / 64;
  const int64_t j0 = (blockIdx.x % tiles_j) * 64;
  int64_t slot = blockIdx.x / tiles_j;
  int64_t i0 = slot * 64, i1 = p.I, t0 = 0, t1 = p.T, vrow = 0, orow = 0;
  if (p.offsets) {
    if (OF_B) {
      const int64_t tiles_i = (p.I + 63) / 64;
      const int e = (int)(slot / tiles_i);
      i0 = (slot % tiles_i) * 64;
      t0 = p.offsets[e];
      t1 = p.offsets[e + 1];
      t0 = t0 < 0 ? 0 : t0;
      t1 = t1 > p.rows ? p.rows : t1;
      orow = (int64_t)e * p.I;
    } else {
      int64_t lo = 0;
      int e = 0;
      for (; e <= p.E; ++e) {
        int64_t hi = e < p.E ? (int64_t)p.offsets[e + 1] : p.I;
        hi = hi < lo ? lo : (hi > p.I ? p.I : hi);
        const int64_t n = (hi - lo + 63) / 64;
        if (slot < n) {
          i0 = lo + slot * 64;
          i1 = hi;
          break;
        }
        slot -= n;
        lo = hi;
      }
      if (e > p.E) return;
      if (e == p.E) t1 = 0;
      vrow = (int64_t)e * p.T;
    }
  }
  f32x4f acc[2][2];
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j) acc[i][j] = f32x4f{0, 0, 0, 0};
  const T* l = reinterpret_cast<const T*>(p.l);
  for (int64_t tb = t0; tb < t1; tb += 32) {
    __syncthreads();
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      const int f = tid + 256 * q;
      // consecutive lanes along the contiguous dimension of dy
      const int ii = OF_B ? (f & 63) : (f >> 5), tt = OF_B ? (f >> 6) : (f & 31);
      float x = 0.0f;
      if (i0 + ii < i1 && tb + tt < t1) x = ElemT<T>::cvt(l[(i0 + ii) * p.si + (tb + tt) * p.st]);
      uint16_t t[P];
      split_bf16<P>(x, t);
#pragma unroll
      for (int k = 0; k < P; ++k) Ls[k][ii][tt] = t[k];
    }
    {
      const int tt = tid >> 3, d = tid & 7;
      const int64_t blk = (j0 >> 5) + (d >> 2);
      uint32_t q = 0, s = 0;
      if (tb + tt < t1 && blk < p.KB) {
        const int64_t row = vrow + tb + tt;
        q = reinterpret_cast<const uint32_t*>(p.v + (row * p.KB + blk) * 16)[d & 3];
        s = p.vs[row * p.KB + blk];
      }
      const float f = e8m0_value(s);
      uint32_t w[4];
      w[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, f, 0));
      w[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, f, 1));
      w[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, f, 2));
      w[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, f, 3));
#pragma unroll
      for (int k = 0; k < 8; ++k) Vs[8 * d + k][tt] = (uint16_t)(w[k >> 1] >> (16 * (k & 1)));
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < P; ++k) {
      bf16x8 A[2], B[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        A[i] = *reinterpret_cast<const bf16x8*>(&Ls[k][(wave >> 1) * 32 + 16 * i + r][8 * g]);
        B[i] = *reinterpret_cast<const bf16x8*>(&Vs[(wave & 1) * 32 + 16 * i + r][8 * g]);
      }
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
          acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(B[j], A[i], acc[i][j], 0, 0, 0);
    }
  }
  O* out = reinterpret_cast<O*>(p.out);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int64_t ii = i0 + (wave >> 1) * 32 + 16 * i + r;
    if (ii >= i1) continue;
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int64_t jj = j0 + (wave & 1) * 32 + 16 * j + 4 * g + q;
        if (jj < p.J) out[(orow + ii) * p.J + jj] = from_f32<O>(acc[i][j][q]);
      }
  }
}

template <typename T, typename O>
static void launch_grad_t(const Fp4Grad& p, bool of_b, unsigned n, hipStream_t st) {
  if (of_b) hipLaunchKernelGGL((k_fp4_grad<T, O, true>), dim3(n), dim3(256), 0, st, p);
  else hipLaunchKernelGGL((k_fp4_grad<T, O, false>), dim3(n), dim3(256), 0, st, p);
}

static int launch_grad(const Fp4Grad& p, bool of_b, int dy_type, int out_type, hipStream_t st) {
  const int64_t ti = ceil_div(p.I, 64);
  int64_t slots = ti;
  if (p.offsets) slots = of_b ? ti * p.E : std::min<int64_t>(p.I, (p.I + (int64_t)(p.E + 1) * 63) / 64);
  const int64_t n = slots * ceil_div(p.J, 64);
  if (n >= ((int64_t)1 << 31)) return fail(MXK_EINVAL, "mxfp4 gradient: too many tiles");
#define MXK_O(T)                                                                          \
  do {                                                                                    \
    if (out_type == MXK_IN_F32) launch_grad_t<T, float>(p, of_b, (unsigned)n, st);        \
    else if (out_type == MXK_IN_F16) launch_grad_t<T, __half>(p, of_b, (unsigned)n, st);  \
    else launch_grad_t<T, hip_bfloat16>(p, of_b, (unsigned)n, st);                        \
  } while (0)
  if (dy_type == MXK_IN_F32) MXK_O(float);
  else if (dy_type == MXK_IN_F16) MXK_O(__half);
  else MXK_O(hip_bfloat16);
#undef MXK_O
  return check_launch("mxfp4 gradient");
}

static bool known(int t) { return t == MXK_IN_F32 || t == MXK_IN_F16 || t == MXK_IN_BF16; }

static int check_grad(const void* dy, int dy_type, int64_t M, int64_t N, int64_t K, const void* codes,
                      const void* scales, int out_type, const void* out, const int32_t* offsets, int experts) {
  if (M < 0 || N < 0 || K < 0) return fail(MXK_EINVAL, "mxfp4 gradient: negative size");
  if (M >= ((int64_t)1 << 31) || N >= ((int64_t)1 << 31) || K >= ((int64_t)1 << 28))
    return fail(MXK_EINVAL, "mxfp4 gradient: rows below 2^31, K below 2^28");
  if (!known(dy_type) || !known(out_type)) return fail(MXK_EINVAL, "mxfp4 gradient: unknown type");
  if (offsets && (experts < 1 || experts > 1000)) return fail(MXK_EINVAL, "mxfp4 gradient: 1 to 1000 experts");
  if (!out && M * N * K > 0) return fail(MXK_EINVAL, "mxfp4 gradient: null pointer");
  if (M > 0 && N > 0 && K > 0 && (!dy || !codes || !scales)) return fail(MXK_EINVAL, "mxfp4 gradient: null pointer");
  if ((reinterpret_cast<uintptr_t>(codes) & 15u) != 0)
    return fail(MXK_EINVAL, "mxfp4 gradient: codes must be 16-byte aligned");
  return MXK_OK;
}

}  // namespace mxk

using namespace mxk;

extern "C" {

int mxk_mxfp4_grad_a(const void* dy, int dy_type, int64_t M, int64_t N, const void* b_codes, const void* b_scales,
                     int64_t K, int out_type, void* da, const int32_t* offsets, int experts, void* stream) {
  int rc = check_grad(dy, dy_type, M, N, K, b_codes, b_scales, out_type, da, offsets, experts);
  if (rc != MXK_OK || M == 0 || K == 0) return rc;
  Fp4Grad p;
  p.l = dy;
  p.si = N;
  p.st = 1;
  p.v = reinterpret_cast<const uint8_t*>(b_codes);
  p.vs = reinterpret_cast<const uint8_t*>(b_scales);
  p.I = M;
  p.T = N;
  p.J = K;
  p.KB = fp4_blocks(K);
  p.out = da;
  p.offsets = offsets;
  p.E = experts;
  p.rows = M;
  return launch_grad(p, false, dy_type, out_type, reinterpret_cast<hipStream_t>(stream));
}

int mxk_mxfp4_grad_b(const void* dy, int dy_type, int64_t M, int64_t N, const void* a_codes, const void* a_scales,
                     int64_t K, int out_type, void* db, const int32_t* offsets, int experts, void* stream) {
  int rc = check_grad(dy, dy_type, M, N, K, a_codes, a_scales, out_type, db, offsets, experts);
  if (rc != MXK_OK || N == 0 || K == 0) return rc;
  Fp4Grad p;
  p.l = dy;
  p.si = 1;
  p.st = N;
  p.v = reinterpret_cast<const uint8_t*>(a_codes);
  p.vs = reinterpret_cast<const uint8_t*>(a_scales);
  p.I = N;
  p.T = M;
  p.J = K;
  p.KB = fp4_blocks(K);
  p.out = db;
  p.offsets = offsets;
  p.E = experts;
  p.rows = M;
  return launch_grad(p, true, dy_type, out_type, reinterpret_cast<hipStream_t>(stream));
}

}  // extern "C"
