// Gradients of the microscaled 4-bit products for gfx950 (straight through
// the quantizer): with y = a b^T over packed a [M][K] and b [N][K],
//
//   da[m, k] = sum_n dy[m, n] b[n, k]        db[n, k] = sum_m dy[m, n] a[m, k]
//
// dy is not quantized.  A code times its power-of-two scale has two
// significant bits and is exact in bfloat16, so the product runs on bf16
// MFMAs with dy as one bf16 term (bf16), two (f16) or three (f32) that add
// up to it exactly: every product is exact, sums are in float32.  (Of an f32 dy
// below 2^-110 what lies under 2^-133, the smallest bf16, is left out.)
//
// The terms of f16 and f32 (and rows of bf16 that do not start on 16 bytes)
// are laid out first as planes of aligned bf16 rows, whose sums simply
// continue one after the other.
#include "mxk_mxfp4.h"

#include <type_traits>

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

// planes[k][M][pitch] = term k of dy [M][N], zeros in columns N .. pitch - 1
// (pitch: N rounded up to 8).  One pass, 8 columns a thread, bound by HBM: 4000x4096
// f32 27 us, f16 17 (6.1 and 5.7 TB/s).
template <typename T>
__global__ __launch_bounds__(256) void k_fp4_planes(const T* __restrict__ dy, int64_t M, int64_t N, int64_t pitch,
                                                    uint16_t* __restrict__ planes) {
  constexpr int P = Planes<T>::N;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, per = pitch >> 3;
  if (i >= M * per) return;
  const int64_t r = i / per, c = (i - r * per) * 8;
  FpWords<T, 8> w;
  const int live = N - c >= 8 ? 8 : (int)(N - c);
  if (live >= 8) fp4_load(dy + r * N + c, w);
  else fp4_load_tail(dy + r * N + c, live, w);
  T v[8];
  __builtin_memcpy(v, w.w, sizeof(v));
  uint16_t t[P][8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    uint16_t s[P];
    split_bf16<P>(ElemT<T>::cvt(v[e]), s);
#pragma unroll
    for (int k = 0; k < P; ++k) t[k][e] = s[k];
  }
#pragma unroll
  for (int k = 0; k < P; ++k) __builtin_memcpy(planes + (k * M + r) * pitch + c, t[k], 16);
}

// out[i, j] = sum over planes and t of L[i, t] V[t, j]: L = dy (rows i) or its
// transpose (rows t), V the packed rows, J = K columns
struct Fp4Grad {
  const uint16_t* l;   // [planes][l_rows][pitch] bf16
  int64_t l_rows, pitch;
  int planes;
  const uint8_t *v, *vs;
  int64_t I, T, J, KB;
  void* out;
  const int* offsets;  // by expert: the segments of I (gradient of a) or of T (of b)
  int E;
};

#define MXK_FAR 0x80000000u  // past every buffer

// Tiles of (64 F)^2 of (i, j), four waves of F x F fragments of 32 x 32
// (v_mfma_f32_32x32x16_bf16), stages of 64 t in two LDS buffers of rows of
// 64 bf16 of t.
//
// V comes packed along j and is wanted along t: a thread takes 8 codes of j
// from 8 rows t, turns them into bf16 pairs along j (the scale of a row and
// block in the conversion), and transposes the 8 x 8 block with byte
// permutes, 8 conversions and 8 permutes per two rows of LDS.  L of the
// gradient of b is transposed the same way; L of the gradient of a is copied.
// Both pass through registers: a stage's operands are requested while the stage
// two before it multiplies, and written to LDS between the MFMAs of the stage before.
// 16-byte chunk c of LDS row r sits at c ^ (r & 7) ^ (r >> 3 & 7): reads
// take 8 consecutive rows, the transposing writes every eighth row.
//
// Bound by the matrix unit and by the conversions beside it (115 VALU a wave and
// stage): 4000x4096x4096 of bf16 131 us for the gradient of a, 134 of b, 1.0
// PFLOP/s (115 and 116 us in a row of calls without the profiler; 8192x8192x4096
// 426 us, 1.3), where the instruction alone runs at 1.75 on random values.  MFMAs
// take 56% of the cycles, waits 15%.  f16 takes two, f32 three times that.  The
// sum over t is one workgroup's whatever I is: 1 to 256 rows of 8192x8192 115 us.
template <typename O, int F, bool OF_B>
__global__ __launch_bounds__(256, 1) void k_fp4_grad(Fp4Grad p, uint32_t tm, uint32_t tn) {
  // LDS: L of either buffer, then V of either, so that a buffer and a fragment
  // are an immediate offset
  constexpr int B = 64 * F, OP = B * 128;
  constexpr int NW = 32 * F, CB = F == 4 ? 128 : 64;
  constexpr int CH = CB / 16, CC = CB / (int)sizeof(O), PASS = NW / CC;
  __shared__ __align__(16) uint8_t lds[4 * OP];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r32 = lane & 31, h = lane >> 5;
  uint32_t it, jt;
  if (OF_B || !p.offsets) place_tile(blockIdx.x, tm, tn, it, jt);
  else if (!place_block_tile(blockIdx.x, tm, tn, it, jt)) return;
  const int64_t j0 = (int64_t)jt * B;
  int64_t i0 = (int64_t)it * B, i1 = p.I < i0 + B ? p.I : i0 + B, t0 = 0, t1 = p.T, v0 = 0, o0 = 0;
  if (p.offsets) {
    if (OF_B) {
      const uint32_t per = (uint32_t)((p.I + B - 1) / B);
      const uint32_t e = it / per;
      i0 = (int64_t)(it - e * per) * B;
      i1 = p.I < i0 + B ? p.I : i0 + B;
      const int64_t lo = p.offsets[e], hi = p.offsets[e + 1];
      t0 = lo < 0 ? 0 : (lo > p.T ? p.T : lo);
      t1 = hi < t0 ? t0 : (hi > p.T ? p.T : hi);
      v0 = 0;
      o0 = (int64_t)e * p.I;
    } else {
      const Segment s = find_segment<B>(it, p.offsets, p.E, p.I);
      if (s.e > p.E) return;
      if (s.e == p.E) t1 = 0;  // rows without an expert: zeros
      i0 = s.lo;
      i1 = s.hi;
      v0 = (int64_t)s.e * p.T;
    }
  }
  const uint32_t row_bytes = (uint32_t)p.KB * 16u, KB = (uint32_t)p.KB;
  const uint32_t pitch = (uint32_t)p.pitch * 2u;  // bytes
  const uint32_t per_plane = (uint32_t)((t1 - t0 + 63) >> 6), stages = per_plane * (uint32_t)p.planes;

  // what this thread stages: V in 8 x 8 blocks (F = 2: waves 0, 1), L in 8 x
  // 8 blocks of dy's transpose (F = 2: waves 2, 3) or in rows of 16-byte chunks
  constexpr int G = B / 8;  // blocks across
  const bool does_v = F == 4 || wave < 2, does_lt = F == 4 || wave >= 2;
  const int g8 = tid % G, tg = (tid / G) & 7;
  const uint32_t vblk = (uint32_t)(j0 >> 5) + (g8 >> 2);
  const uint32_t v_off = vblk < KB ? (uint32_t)(8 * tg) * row_bytes + vblk * 16u + (g8 & 3) * 4u : MXK_FAR;
  const uint32_t s_off = vblk < KB ? (uint32_t)(8 * tg) * KB + vblk : MXK_FAR;
  const uint32_t lt_off = (uint32_t)(8 * tg) * pitch + g8 * 16u;
  const uint32_t ld_off = (uint32_t)(tid >> 3) * pitch + (tid & 7) * 16u;

  uint32_t vw[8], vsc[8];
  u32x4 lw[OF_B ? 8 : B / 32];
  // the buffers of stage s, and whether this thread's chunk of a copied L is past its end
  __amdgpu_buffer_rsrc_t rv, rs, rl;
  uint32_t far = 0;
  auto prepare = [&](uint32_t s) {
    const uint32_t plane = s / per_plane, st = s - plane * per_plane;
    const int64_t t = t0 + 64 * (int64_t)st;
    const int64_t left = s < stages ? (t1 - t < 64 ? t1 - t : 64) : 0;
    rv = make_rsrc(p.v + (v0 + t) * row_bytes, (uint32_t)left * row_bytes);
    rs = make_rsrc(p.vs + (v0 + t) * KB, (uint32_t)left * KB);
    if constexpr (OF_B) {
      const int64_t cols = p.pitch - i0;  // of dy from this tile on
      rl = make_rsrc(p.l + (plane * p.l_rows + t) * p.pitch + i0,
                     left > 0 ? (uint32_t)((left - 1) * pitch + cols * 2) : 0u);
    } else {
      const int64_t rows = p.I - i0 < B ? p.I - i0 : B;
      rl = make_rsrc(p.l + (plane * p.l_rows + i0) * p.pitch + t, left > 0 ? (uint32_t)(rows * pitch - (t * 2)) : 0u);
      far = (tid & 7) * 8 < left ? 0u : MXK_FAR;
    }
  };
  // request half q (0, 1) of its operands
  auto request = [&](int q) {
    if (does_v) {
#pragma unroll
      for (int k = 4 * q; k < 4 * q + 4; ++k) {
        vw[k] = buf_load_b32(rv, v_off + k * row_bytes, 0);
        vsc[k] = (uint32_t)__builtin_amdgcn_raw_buffer_load_b8(rs, (int)(s_off + k * KB), 0, 0);
      }
    }
    if constexpr (OF_B) {
      if (does_lt) {
#pragma unroll
        for (int k = 4 * q; k < 4 * q + 4; ++k) lw[k] = buf_load_b128(rl, lt_off + k * pitch, 0);
      }
    } else {
#pragma unroll
      for (int k = q * B / 64; k < (q + 1) * B / 64; ++k)
        lw[k] = buf_load_b128(rl, (ld_off + k * 32u * pitch) | far, 0);
    }
  };
  // where this thread's rows of LDS are: chunk tg of rows 8 g8 + k of a
  // transposed operand, chunk tid % 8 of rows tid / 8 + 32 k of a copied one
  // (those with k even and odd differ by 4 in bits 3 .. 5 of the row)
  uint8_t* put_t[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) put_t[k] = lds + (8 * g8 + k) * 128 + ((tg ^ k ^ (g8 & 7)) << 4);
  uint8_t* put_c[2];
#pragma unroll
  for (int k = 0; k < 2; ++k)
    put_c[k] = lds + (tid >> 3) * 128 + (((tid & 7) ^ ((tid >> 3) & 7) ^ (((tid >> 6) + 4 * k) & 7)) << 4);
  // two LDS rows of the transpose of an 8 x 8 block of 16-bit values: low and high halves of eight pairs
  auto put_pairs = [&](int base, int q, const uint32_t (&a)[8]) {
    u32x4 lo, hi;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      lo[k] = __builtin_amdgcn_perm(a[2 * k + 1], a[2 * k], 0x05040100u);
      hi[k] = __builtin_amdgcn_perm(a[2 * k + 1], a[2 * k], 0x07060302u);
    }
    *reinterpret_cast<u32x4*>(put_t[2 * q] + base) = lo;
    *reinterpret_cast<u32x4*>(put_t[2 * q + 1] + base) = hi;
  };
#define MXK_VPAIR(k, q) \
  __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(vw[k], e8m0_operand(vsc[k]), q))
  // quarter q of the staged V, of the staged L
  auto stage_v = [&](int buf, int q) {
    if (!does_v) return;
    uint32_t a[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      if (q == 0) a[k] = MXK_VPAIR(k, 0);
      else if (q == 1) a[k] = MXK_VPAIR(k, 1);
      else if (q == 2) a[k] = MXK_VPAIR(k, 2);
      else a[k] = MXK_VPAIR(k, 3);
    }
    put_pairs((2 + buf) * OP, q, a);
  };
  auto stage_l = [&](int buf, int q) {
    if constexpr (OF_B) {
      if (!does_lt) return;
      uint32_t a[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) a[k] = lw[k][q];
      put_pairs(buf * OP, q, a);
    } else {
#pragma unroll
      for (int k = q * B / 128; k < (q + 1) * B / 128; ++k)
        *reinterpret_cast<u32x4*>(put_c[k & 1] + buf * OP + 4096 * k) = lw[k];
    }
  };

  const int ra = (wave >> 1) * NW + r32, rb = (wave & 1) * NW + r32;
  f32x16 acc[F][F];  // [V fragment][L fragment]: rows of the result are j
#pragma unroll
  for (int i = 0; i < F; ++i)
#pragma unroll
    for (int j = 0; j < F; ++j)
#pragma unroll
      for (int q = 0; q < 16; ++q) acc[i][j][q] = 0.0f;
  bf16x8 fa[2][F], fb[2][F];
  // chunk 2 s + h of rows ra + 32 i; bits 3 .. 5 of the row change with i by 4 (i & 1)
  const uint8_t *get_l[4], *get_v[4];
#pragma unroll
  for (int s = 0; s < 4; ++s) {
    get_l[s] = lds + ra * 128 + (((2 * s + h) ^ (ra & 7) ^ ((ra >> 3) & 7)) << 4);
    get_v[s] = lds + 2 * OP + rb * 128 + (((2 * s + h) ^ (rb & 7) ^ ((rb >> 3) & 7)) << 4);
  }
  auto read_frag = [&](int buf, int s, int i, bf16x8 (&xa)[F], bf16x8 (&xb)[F]) {
    // chunk c ^ 4 is that of step s ^ 2
    const int at = i & 1 ? s ^ 2 : s;
    xa[i] = *reinterpret_cast<const bf16x8*>(get_l[at] + buf * OP + i * 4096);
    xb[i] = *reinterpret_cast<const bf16x8*>(get_v[at] + buf * OP + i * 4096);
  };
  // A row of F MFMAs and what is issued between them: the conversions of a
  // stage fit into the MFMAs' shadows only if they alternate with them
#define MXK_STEP(XA, XB, BETWEEN)                                                              \
  _Pragma("unroll") for (int i = 0; i < F; ++i) {                                              \
    BETWEEN;                                                                                   \
    _Pragma("unroll") for (int j = 0; j < F; ++j)                                              \
        acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(XB[i], XA[j], acc[i][j], 0, 0, 0); \
    _Pragma("unroll") for (int j = 0; j < F; ++j) {                                            \
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0); /* MFMA */                            \
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 0); /* LDS read */                        \
      __builtin_amdgcn_sched_group_barrier(0x002, SHADOW, 0); /* VALU */                       \
      __builtin_amdgcn_sched_group_barrier(0x200, 1, 0); /* LDS write */                       \
      __builtin_amdgcn_sched_group_barrier(0x020, 4, 0); /* loads */                           \
    }                                                                                          \
    __builtin_amdgcn_sched_barrier(0);                                                         \
  }
  constexpr int SHADOW = 24 / F;  // a row's share of the conversions, spread over its MFMAs (48 / F was 2% slower)
  // Quarters per row of MFMAs
  constexpr int Q = 4 / F;
  if (stages > 0) {
    prepare(0);
    request(0);
    request(1);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      stage_v(0, q);
      stage_l(0, q);
    }
    prepare(1);
    request(0);
    request(1);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
#pragma unroll
    for (int i = 0; i < F; ++i) read_frag(0, 0, i, fa[0], fb[0]);
    // two stages a turn, one in each buffer; where their number is odd the last one's operands are zeros
    auto stage = [&](auto which, uint32_t s) {
      constexpr int buf = decltype(which)::value;
      MXK_STEP(fa[0], fb[0], {
        read_frag(buf, 1, i, fa[1], fb[1]);
        _Pragma("unroll") for (int q = i * Q; q < (i + 1) * Q; ++q) stage_v(buf ^ 1, q);
      })
      MXK_STEP(fa[1], fb[1], {
        read_frag(buf, 2, i, fa[0], fb[0]);
        _Pragma("unroll") for (int q = i * Q; q < (i + 1) * Q; ++q) stage_l(buf ^ 1, q);
        if (i == F - 1) prepare(s + 2);
      })
      MXK_STEP(fa[0], fb[0], {
        read_frag(buf, 3, i, fa[1], fb[1]);
        if (i < 2) request(i);
      })
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
      MXK_STEP(fa[1], fb[1], read_frag(buf ^ 1, 0, i, fa[0], fb[0]))
    };
    for (uint32_t s = 0; s < stages; s += 2) {
      stage(std::integral_constant<int, 0>(), s);
      stage(std::integral_constant<int, 1>(), s + 1);
    }
  }
#undef MXK_STEP
#undef MXK_VPAIR
  __syncthreads();

  // The result through LDS, as the products' (32 rows of i and CB bytes of j at a time and wave)
  O* out = reinterpret_cast<O*>(p.out) + o0 * p.J;
  const bool whole = p.J * (int)sizeof(O) % 16 == 0 && (reinterpret_cast<uintptr_t>(p.out) & 15u) == 0;
  uint8_t* mine = lds + wave * 32 * CB;
  const int64_t jw = j0 + (wave & 1) * NW, iw = i0 + (wave >> 1) * NW;
  const uint32_t el = (uint32_t)lane;
#pragma unroll
  for (int j = 0; j < F; ++j)
#pragma unroll
    for (int s = 0; s < PASS; ++s) {
#pragma unroll
      for (int u = 0; u < CC / 8; ++u) {
        const int iq = s * (CC / 8) + u, i = iq >> 2, q = iq & 3;
        O t[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) t[k] = from_f32<O>(acc[i][j][4 * q + k]);
        const uint32_t byte = (8 * u + 4 * (el >> 5)) * (uint32_t)sizeof(O);
        uint8_t* d = mine + (el & 31u) * CB + (((byte >> 4) ^ (el & (CH - 1))) << 4) + (byte & 15);
        __builtin_memcpy(__builtin_assume_aligned(d, 4 * sizeof(O)), t, sizeof(t));
      }
      __builtin_amdgcn_wave_barrier();
      u32x4 w[CH / 2];
#pragma unroll
      for (int k = 0; k < CH / 2; ++k) {
        const uint32_t row = k * (64 / CH) + el / CH, ch = el % CH;
        w[k] = *reinterpret_cast<const u32x4*>(mine + row * CB + ((ch ^ (row & (CH - 1))) << 4));
      }
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int k = 0; k < CH / 2; ++k) {
        const int64_t i = iw + 32 * j + k * (64 / CH) + el / CH;
        const int64_t n = jw + s * CC + (el % CH) * (16 / (int)sizeof(O));
        if (i < i1 && n < p.J) {
          O* d = out + i * p.J + n;
          if (whole) {
            *reinterpret_cast<u32x4*>(d) = w[k];
          } else {
            O t[16 / sizeof(O)];
            __builtin_memcpy(t, &w[k], 16);
#pragma unroll
            for (int q = 0; q < 16 / (int)sizeof(O); ++q)
              if (n + q < p.J) d[q] = t[q];
          }
        }
      }
    }
}

// bf16 rows that are read where they lie: 16-byte rows at 16-byte addresses
static bool direct_rows(const void* dy, int dy_type, int64_t N) {
  return dy_type == MXK_IN_BF16 && N % 8 == 0 && aligned16(dy);
}
static int planes_of(int dy_type) { return dy_type == MXK_IN_BF16 ? 1 : (dy_type == MXK_IN_F16 ? 2 : 3); }
static int64_t planes_bytes(int dy_type, int64_t M, int64_t N) {
  return planes_of(dy_type) * M * ceil_div(N, 8) * 16;
}

static int launch_planes(const void* dy, int dy_type, int64_t M, int64_t N, uint16_t* planes, hipStream_t st) {
  const int64_t pitch = ceil_div(N, 8) * 8, n = ceil_div(M * (pitch / 8), 256);
  if (n >= ((int64_t)1 << 31)) return fail(MXK_EINVAL, "mxfp4 gradient: dy too large");
#define MXK_P(T)                                                                                                    \
  hipLaunchKernelGGL((k_fp4_planes<T>), dim3((unsigned)n), dim3(256), 0, st, reinterpret_cast<const T*>(dy), M, N, \
                     pitch, planes)
  if (dy_type == MXK_IN_F32) MXK_P(float);
  else if (dy_type == MXK_IN_F16) MXK_P(__half);
  else MXK_P(hip_bfloat16);
#undef MXK_P
  return check_launch("mxfp4 gradient: planes");
}

static int launch_grad(const Fp4Grad& p, bool of_b, int out_type, hipStream_t st) {
  const bool ex = p.offsets != nullptr;
  auto tiles = [&](int B) {
    const int64_t ti = ceil_div(p.I, B);
    return (ex ? (of_b ? ti * p.E : segment_slots(p.I, p.E, B)) : ti) * ceil_div(p.J, B);
  };
  // large tiles where they occupy most CUs (192 of them, 3000x4096x4096: 103 us
  // against 130; 128, 2048x4096x4096: 101 against 80)
  const int F = tiles(256) >= 160 ? 4 : 2;
  const int64_t B = 64 * F, n = tiles((int)B), tn = ceil_div(p.J, B);
  if (n >= ((int64_t)1 << 31)) return fail(MXK_EINVAL, "mxfp4 gradient: too many tiles");
  const uint32_t tm = (uint32_t)(n / tn);
  const int64_t ids = ex && !of_b ? block_tile_ids(tm, tn) : n;
  if (ids >= ((int64_t)1 << 31)) return fail(MXK_EINVAL, "mxfp4 gradient: too many tiles");
  const dim3 grid((unsigned)ids);
#define MXK_G(O, F, OB) hipLaunchKernelGGL((k_fp4_grad<O, F, OB>), grid, dim3(256), 0, st, p, tm, (uint32_t)tn)
#define MXK_O(O)                     \
  do {                               \
    if (F == 4) {                    \
      if (of_b) MXK_G(O, 4, true);   \
      else MXK_G(O, 4, false);       \
    } else {                         \
      if (of_b) MXK_G(O, 2, true);   \
      else MXK_G(O, 2, false);       \
    }                                \
  } while (0)
  if (out_type == MXK_IN_F32) MXK_O(float);
  else if (out_type == MXK_IN_F16) MXK_O(__half);
  else MXK_O(hip_bfloat16);
#undef MXK_O
#undef MXK_G
  return check_launch("mxfp4 gradient");
}

static bool known(int t) { return t == MXK_IN_F32 || t == MXK_IN_F16 || t == MXK_IN_BF16; }

static int check_grad(bool of_b, const void* dy, int dy_type, int64_t M, int64_t N, int64_t K, const void* codes,
                      const void* scales, int out_type, const void* out, const int32_t* offsets, int experts,
                      const void* ws, size_t ws_bytes) {
  if (M < 0 || N < 0 || K < 0) return fail(MXK_EINVAL, "mxfp4 gradient: negative size");
  // 256 rows of dy and 64 packed rows within a buffer of 2^31 bytes
  if (M >= ((int64_t)1 << 31) || N >= ((int64_t)1 << 22) || K >= ((int64_t)1 << 26))
    return fail(MXK_EINVAL, "mxfp4 gradient: M below 2^31, N below 2^22, K below 2^26");
  if (!known(dy_type) || !known(out_type)) return fail(MXK_EINVAL, "mxfp4 gradient: unknown type");
  if (offsets && (experts < 1 || experts > 1000)) return fail(MXK_EINVAL, "mxfp4 gradient: 1 to 1000 experts");
  // an empty sum is written too: the result is there wherever it has elements
  if (!out && (of_b ? N : M) > 0 && K > 0) return fail(MXK_EINVAL, "mxfp4 gradient: null pointer");
  if (M > 0 && N > 0 && K > 0 && (!dy || !codes || !scales)) return fail(MXK_EINVAL, "mxfp4 gradient: null pointer");
  if ((reinterpret_cast<uintptr_t>(codes) & 15u) != 0)
    return fail(MXK_EINVAL, "mxfp4 gradient: codes must be 16-byte aligned");
  if (M > 0 && N > 0 && K > 0 && !direct_rows(dy, dy_type, N) &&
      (!ws || !aligned16(ws) || ws_bytes < (size_t)planes_bytes(dy_type, M, N)))
    return fail(MXK_EINVAL, "mxfp4 gradient: workspace too small or not 16-byte aligned");
  return MXK_OK;
}

static int run_grad(Fp4Grad& p, bool of_b, const void* dy, int dy_type, int64_t M, int64_t N, int out_type, void* ws,
                    hipStream_t st) {
  p.l_rows = M;
  p.planes = planes_of(dy_type);
  p.pitch = N;
  p.l = reinterpret_cast<const uint16_t*>(dy);
  if (M > 0 && N > 0 && !direct_rows(dy, dy_type, N)) {
    p.pitch = ceil_div(N, 8) * 8;
    p.l = reinterpret_cast<const uint16_t*>(ws);
    const int rc = launch_planes(dy, dy_type, M, N, reinterpret_cast<uint16_t*>(ws), st);
    if (rc != MXK_OK) return rc;
  }
  return launch_grad(p, of_b, out_type, st);
}

}  // namespace mxk

using namespace mxk;

extern "C" {

size_t mxk_mxfp4_grad_workspace(const void* dy, int dy_type, int64_t M, int64_t N) {
  if (M <= 0 || N <= 0 || !known(dy_type) || direct_rows(dy, dy_type, N)) return 0;
  return (size_t)planes_bytes(dy_type, M, N);
}

int mxk_mxfp4_grad_a(const void* dy, int dy_type, int64_t M, int64_t N, const void* b_codes, const void* b_scales,
                     int64_t K, int out_type, void* da, const int32_t* offsets, int experts, void* workspace,
                     size_t workspace_nbytes, void* stream) {
  int rc = check_grad(false, dy, dy_type, M, N, K, b_codes, b_scales, out_type, da, offsets, experts, workspace,
                      workspace_nbytes);
  if (rc != MXK_OK || M == 0 || K == 0) return rc;
  Fp4Grad p;
  p.v = reinterpret_cast<const uint8_t*>(b_codes);
  p.vs = reinterpret_cast<const uint8_t*>(b_scales);
  p.I = M;
  p.T = N;
  p.J = K;
  p.KB = fp4_blocks(K);
  p.out = da;
  p.offsets = offsets;
  p.E = experts;
  return run_grad(p, false, dy, dy_type, M, N, out_type, workspace, reinterpret_cast<hipStream_t>(stream));
}

int mxk_mxfp4_grad_b(const void* dy, int dy_type, int64_t M, int64_t N, const void* a_codes, const void* a_scales,
                     int64_t K, int out_type, void* db, const int32_t* offsets, int experts, void* workspace,
                     size_t workspace_nbytes, void* stream) {
  int rc = check_grad(true, dy, dy_type, M, N, K, a_codes, a_scales, out_type, db, offsets, experts, workspace,
                      workspace_nbytes);
  if (rc != MXK_OK || N == 0 || K == 0) return rc;
  Fp4Grad p;
  p.v = reinterpret_cast<const uint8_t*>(a_codes);
  p.vs = reinterpret_cast<const uint8_t*>(a_scales);
  p.I = N;
  p.T = M;
  p.J = K;
  p.KB = fp4_blocks(K);
  p.out = db;
  p.offsets = offsets;
  p.E = experts;
  return run_grad(p, true, dy, dy_type, M, N, out_type, workspace, reinterpret_cast<hipStream_t>(stream));
}

}  // extern "C"
