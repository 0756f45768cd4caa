// Microscaled 4-bit floating point for gfx950: quantize and dequantize.
//
// Both are one pass over the data and bound by HBM: quantize reads a row's
// elements once and writes 17 bytes per 32 of them, dequantize the other way
// round.  A lane holds 8 elements (one 16-byte load of a 16-bit type), the 4
// lanes of a block share its largest magnitude by two lane exchanges, and a
// wave stores 64 consecutive dwords of codes.  There is nothing to divide:
// the scale is a power of two, so its exponent field comes from the bits of
// the maximum and v_cvt_scalef32_pk_fp4_* rounds two elements at a time.
// 16383x8192 bf16 (268 MB and 71 MB): quantize 56 us, dequantize 48, 6.0 and
// 7.0 TB/s, above the 5.1 of a large copy.
#include "mxk_mxfp4.h"

namespace mxk {

// Task i (one lane, 8 elements): element group i % lanes of row i / lanes,
// lanes = 4 * KB.  FLAT: rows follow each other without padding and hold
// whole blocks, so that task i is elements 8i and no row is looked up.
// U tasks per thread, 256 apart, with all loads issued before the first use.
template <typename T, bool FLAT, int U>
__global__ __launch_bounds__(256) void k_fp4_quantize(const T* __restrict__ x, int64_t ld, uint32_t total, int cols,
                                                      DivU32 by_lanes, uint32_t lanes, uint32_t* __restrict__ codes,
                                                      uint8_t* __restrict__ scales) {
  const uint64_t first = (uint64_t)blockIdx.x * (256u * U) + threadIdx.x;
  FpWords<T, 8> v[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const uint64_t i = first + 256u * u;
    if (i < total) {
      if constexpr (FLAT) {
        fp4_load(x + 8 * i, v[u]);
      } else {
        const uint32_t r = divu32((uint32_t)i, by_lanes), c = 8u * ((uint32_t)i - r * lanes);
        const T* p = x + (int64_t)r * ld + c;
        const int live = cols - (int)c;
        if (live >= 8) fp4_load(p, v[u]);
        else fp4_load_tail(p, live, v[u]);
      }
    } else {
#pragma unroll
      for (int q = 0; q < FpWords<T, 8>::NW; ++q) v[u].w[q] = 0u;
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const uint64_t i = first + 256u * u;
    // total is a multiple of 4: the lanes of a block are all in range or all out of it
    const uint32_t byte = fp4_scale_byte(group_max_u<4>(fp4_amax_bits(v[u])));
    uint32_t q[1];
    fp4_codes(v[u], e8m0_operand(byte), q);
    if (i < total) {
      codes[i] = byte == 255u ? 0u : q[0];
      if ((threadIdx.x & 3u) == 0u) scales[i >> 2] = (uint8_t)byte;
    }
  }
}

// Task i, one a thread: one dword (8 codes).  Four a thread, as above, were no faster
// anywhere (4000x4096 bf16 7.3 us against 6.5).  f16 results go through
// float32, where the value is exact, so that subnormal and overflowing ones
// round once.
template <typename T, bool FLAT>
__global__ __launch_bounds__(256) void k_fp4_dequantize(const uint32_t* __restrict__ codes,
                                                        const uint8_t* __restrict__ scales, uint32_t total, int cols,
                                                        DivU32 by_lanes, uint32_t lanes, T* __restrict__ y) {
  const uint64_t i = (uint64_t)blockIdx.x * 256u + threadIdx.x;
  if (i >= total) return;
  const uint32_t q = codes[i];
  const float f = e8m0_operand(scales[i >> 2]);
  FpWords<T, 8> o;
  if constexpr (__is_same(T, hip_bfloat16)) {
    o.w[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, f, 0));
    o.w[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, f, 1));
    o.w[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, f, 2));
    o.w[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, f, 3));
  } else {
    f32x2f p[4];
    p[0] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, f, 0);
    p[1] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, f, 1);
    p[2] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, f, 2);
    p[3] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, f, 3);
    T t[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) t[e] = from_f32<T>(p[e >> 1][e & 1]);
    __builtin_memcpy(o.w, t, sizeof(o.w));
  }
  if constexpr (FLAT) {
    u32x4* d = reinterpret_cast<u32x4*>(y + 8 * i);
#pragma unroll
    for (int k = 0; k < FpWords<T, 8>::NW / 4; ++k)
      __builtin_nontemporal_store(u32x4{o.w[4 * k], o.w[4 * k + 1], o.w[4 * k + 2], o.w[4 * k + 3]}, d + k);
  } else {
    const uint32_t r = divu32((uint32_t)i, by_lanes), c = 8u * ((uint32_t)i - r * lanes);
    T* p = y + (int64_t)r * cols + c;
    const int live = cols - (int)c;
    if (live >= 8) {
      __builtin_memcpy(p, o.w, sizeof(o.w));
    } else {
      const T* t = reinterpret_cast<const T*>(o.w);
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (e < live) p[e] = t[e];
    }
  }
}

// Rows a launch covers: its task index has to fit 31 bits
static int64_t rows_per_launch(int64_t lanes) { return std::max<int64_t>(1, ((int64_t)1 << 31) / lanes - 1); }

template <typename T>
static void launch_quantize(const T* x, int64_t rows, int64_t cols, int64_t ld, uint8_t* codes, uint8_t* scales,
                            hipStream_t st) {
  const int64_t kb = fp4_blocks(cols), lanes = 4 * kb, step = rows_per_launch(lanes);
  // 16-byte loads at their natural alignment only where rows have it too
  const bool flat = cols % 32 == 0 && ld == cols && aligned16(x);
  const DivU32 dv = make_divu32((uint32_t)lanes);
  for (int64_t r0 = 0; r0 < rows; r0 += step) {
    const int64_t n = std::min(step, rows - r0);
    const uint32_t total = (uint32_t)(n * lanes);
    const T* xp = x + r0 * ld;
    uint32_t* cp = reinterpret_cast<uint32_t*>(codes + r0 * kb * 16);
    uint8_t* sp = scales + r0 * kb;
    // four tasks a thread hide the loads' latency (4000x4096 bf16 6.2 us against
    // 8.2 with one; 16383x8192 the same); below 4 workgroups a CU of that size, more
    // workgroups do (2000x2000 3.4 us against 4.1 with four)
    const bool big = total >= 256u * 4u * 1024u;
    const dim3 grid((unsigned)ceil_div(total, big ? 1024 : 256));
#define MXK_Q(F, U)                                                                                              \
  hipLaunchKernelGGL((k_fp4_quantize<T, F, U>), grid, dim3(256), 0, st, xp, ld, total, (int)cols, dv,           \
                     (uint32_t)lanes, cp, sp)
    if (flat && big) MXK_Q(true, 4);
    else if (flat) MXK_Q(true, 1);
    else if (big) MXK_Q(false, 4);
    else MXK_Q(false, 1);
#undef MXK_Q
  }
}

template <typename T>
static void launch_dequantize(const uint8_t* codes, const uint8_t* scales, int64_t rows, int64_t cols, T* y,
                              hipStream_t st) {
  const int64_t kb = fp4_blocks(cols), lanes = 4 * kb, step = rows_per_launch(lanes);
  const bool flat = cols % 32 == 0 && aligned16(y);
  const DivU32 dv = make_divu32((uint32_t)lanes);
  for (int64_t r0 = 0; r0 < rows; r0 += step) {
    const int64_t n = std::min(step, rows - r0);
    const uint32_t total = (uint32_t)(n * lanes);
    const uint32_t* cp = reinterpret_cast<const uint32_t*>(codes + r0 * kb * 16);
    const uint8_t* sp = scales + r0 * kb;
    T* yp = y + r0 * cols;
    const dim3 grid((unsigned)ceil_div(total, 256));
    hipLaunchKernelGGL((flat ? k_fp4_dequantize<T, true> : k_fp4_dequantize<T, false>), grid, dim3(256), 0, st, cp, sp,
                       total, (int)cols, dv, (uint32_t)lanes, yp);
  }
}

}  // namespace mxk

using namespace mxk;

extern "C" {

int mxk_mxfp4_quantize(const void* x, int x_type, int64_t rows, int64_t cols, int64_t row_stride, void* codes,
                       void* scales, void* stream) {
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (rows < 0 || cols < 0 || row_stride < 0) return fail(MXK_EINVAL, "mxfp4_quantize: negative size");
  if (cols >= ((int64_t)1 << 28)) return fail(MXK_EINVAL, "mxfp4_quantize: rows of 2^28 elements or more");
  if (rows == 0 || cols == 0) return MXK_OK;
  if (!x || !codes || !scales) return fail(MXK_EINVAL, "mxfp4_quantize: null pointer");
  if ((reinterpret_cast<uintptr_t>(codes) & 3u) != 0)
    return fail(MXK_EINVAL, "mxfp4_quantize: codes must be 4-byte aligned");
  uint8_t* c = reinterpret_cast<uint8_t*>(codes);
  uint8_t* s = reinterpret_cast<uint8_t*>(scales);
  if (x_type == MXK_IN_F32) launch_quantize(reinterpret_cast<const float*>(x), rows, cols, row_stride, c, s, st);
  else if (x_type == MXK_IN_F16) launch_quantize(reinterpret_cast<const __half*>(x), rows, cols, row_stride, c, s, st);
  else if (x_type == MXK_IN_BF16)
    launch_quantize(reinterpret_cast<const hip_bfloat16*>(x), rows, cols, row_stride, c, s, st);
  else return fail(MXK_EINVAL, "mxfp4_quantize: unknown x_type");
  return check_launch("mxfp4_quantize");
}

int mxk_mxfp4_dequantize(const void* codes, const void* scales, int64_t rows, int64_t cols, int y_type, void* y,
                         void* stream) {
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (rows < 0 || cols < 0) return fail(MXK_EINVAL, "mxfp4_dequantize: negative size");
  if (cols >= ((int64_t)1 << 28)) return fail(MXK_EINVAL, "mxfp4_dequantize: rows of 2^28 elements or more");
  if (rows == 0 || cols == 0) return MXK_OK;
  if (!codes || !scales || !y) return fail(MXK_EINVAL, "mxfp4_dequantize: null pointer");
  if ((reinterpret_cast<uintptr_t>(codes) & 3u) != 0)
    return fail(MXK_EINVAL, "mxfp4_dequantize: codes must be 4-byte aligned");
  const uint8_t* c = reinterpret_cast<const uint8_t*>(codes);
  const uint8_t* s = reinterpret_cast<const uint8_t*>(scales);
  if (y_type == MXK_IN_F32) launch_dequantize(c, s, rows, cols, reinterpret_cast<float*>(y), st);
  else if (y_type == MXK_IN_F16) launch_dequantize(c, s, rows, cols, reinterpret_cast<__half*>(y), st);
  else if (y_type == MXK_IN_BF16) launch_dequantize(c, s, rows, cols, reinterpret_cast<hip_bfloat16*>(y), st);
  else return fail(MXK_EINVAL, "mxfp4_dequantize: unknown y_type");
  return check_launch("mxfp4_dequantize");
}

}  // extern "C"
