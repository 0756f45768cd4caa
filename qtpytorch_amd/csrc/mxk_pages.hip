// Rotary positions, and rows into, out of and within a paged 8-bit key-value
// cache, for gfx950.
//
// Rotation: pair i of a head's first R = 2 * pairs elements, (u, w) =
// (x[i], x[i + R/2]) or, interleaved, (x[2i], x[2i+1]), becomes
// (u cos a - w sin a, w cos a + u sin a) with a = position[axis[i]] *
// freqs[i]; elements from R on stay as they are.
#include "mxk_pages.h"

#include <algorithm>

namespace mxk {

struct Rotation {
  const double* __restrict__ freqs;  // radians per position
  const int* __restrict__ axis;      // null: axis 0
  const void* __restrict__ pos;      // [T][axes], one axis: for all pairs; null: the token's own place
  int wide;                          // int64 positions
  int pairs, axes, interleaved;
  float sign;
};

// cos and sin of a pair's angle.  The angle of a far position has few bits
// left in float32 (10^6 radians: 1/16), so it is reduced in float64, as turns:
// the rest of a turn is exact there, and float32 holds it to 2^-26 of a turn.
__device__ __forceinline__ float2 rot_turn(const Rotation& r, int64_t at, int t, int i) {
  int64_t p = at;
  if (r.pos) {
    const int ax = r.axis && r.axes > 1 ? r.axis[i] : 0;
    const int64_t e = (int64_t)t * r.axes + ax;
    p = (uint32_t)ax >= (uint32_t)r.axes ? 0
        : r.wide ? reinterpret_cast<const int64_t*>(r.pos)[e] : (int64_t) reinterpret_cast<const int*>(r.pos)[e];
  }
  double a = (double)p * r.freqs[i] * 0.15915494309189535;
  a -= __builtin_rint(a);
  float s, c;
  sincospif(2.0f * (float)a, &s, &c);
  return make_float2(c, s * r.sign);
}

// V elements at p as float and back; no alignment beyond an element's
template <typename T, int V>
__device__ __forceinline__ void row_load(const T* p, float (&v)[V]) {
  T e[V];
  __builtin_memcpy(e, p, sizeof(e));
#pragma unroll
  for (int i = 0; i < V; ++i) v[i] = ElemT<T>::cvt(e[i]);
}
template <typename T>
__device__ __forceinline__ T row_cvt(float v) {
  if constexpr (__is_same(T, float)) return v;
  else if constexpr (__is_same(T, __half)) return __float2half_rn(v);
  else return __builtin_bit_cast(hip_bfloat16, (__bf16)v);
}
template <typename T, int V>
__device__ __forceinline__ void row_store(T* p, const float (&v)[V]) {
  T e[V];
#pragma unroll
  for (int i = 0; i < V; ++i) e[i] = row_cvt<T>(v[i]);
  __builtin_memcpy(p, e, sizeof(e));
}

// ---------------------------------------------------------------- rotary
// TB tokens a workgroup: their angles once into LDS, then V pairs (or V
// elements that are not rotated) a thread and step.  The angles, ~100
// instructions each, are shared by all heads of a token.  Bound by memory: 8190
// tokens of 32 heads of 128 in bfloat16, 134 MB in 24.3 us, 5.5 TB/s.
template <typename T, int V>
__global__ __launch_bounds__(256) void k_rotary(const T* __restrict__ x, int64_t token_stride, int64_t head_stride,
                                                Rotation r, int T_, int D, int TB, uint32_t per_token, DivU32 by_token,
                                                uint32_t per_head, DivU32 by_head, int H, T* __restrict__ y) {
  extern __shared__ float2 cs[];  // [TB][pairs]
  const int t0 = kv_block() * TB, tn = min(TB, T_ - t0);
  if (tn <= 0) return;  // blocks past the last
  for (int i = threadIdx.x; i < tn * r.pairs; i += 256) {
    const int t = i / r.pairs;
    cs[i] = rot_turn(r, t0 + t, t0 + t, i - t * r.pairs);
  }
  __syncthreads();
  const uint32_t turned = (uint32_t)r.pairs / V;  // items of a head that are pairs
  const uint32_t total = (uint32_t)tn * per_token;
  for (uint32_t it = blockIdx.y * 256u + threadIdx.x; it < total; it += gridDim.y * 256u) {
    const uint32_t t = divu32(it, by_token), rest = it - t * per_token;
    const uint32_t h = divu32(rest, by_head), c = rest - h * per_head;
    const T* src = x + (int64_t)(t0 + t) * token_stride + (int64_t)h * head_stride;
    T* dst = y + ((int64_t)(t0 + t) * H + h) * D;
    if (c >= turned) {
      const int e = 2 * r.pairs + (int)(c - turned) * V;
      T keep[V];
      __builtin_memcpy(keep, src + e, sizeof(keep));
      __builtin_memcpy(dst + e, keep, sizeof(keep));
      continue;
    }
    const float2* a = cs + t * r.pairs + c * V;
    if (r.interleaved) {
      const int e = (int)c * 2 * V;
      float v[2 * V], o[2 * V];
      row_load<T, 2 * V>(src + e, v);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        o[2 * i] = __builtin_fmaf(v[2 * i], a[i].x, -(v[2 * i + 1] * a[i].y));
        o[2 * i + 1] = __builtin_fmaf(v[2 * i + 1], a[i].x, v[2 * i] * a[i].y);
      }
      row_store<T, 2 * V>(dst + e, o);
    } else {
      const int e = (int)c * V;
      float u[V], w[V], ou[V], ow[V];
      row_load<T, V>(src + e, u);
      row_load<T, V>(src + r.pairs + e, w);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        ou[i] = __builtin_fmaf(u[i], a[i].x, -(w[i] * a[i].y));
        ow[i] = __builtin_fmaf(w[i], a[i].x, u[i] * a[i].y);
      }
      row_store<T, V>(dst + e, ou);
      row_store<T, V>(dst + r.pairs + e, ow);
    }
  }
}

// ---------------------------------------------------------------- append
// A lane's eight elements e..e+7 of the rotated rows of one token: y[i] = x[i] * c[i] + x[partner(i)] * s[i].
// The partners are eight in a row too where pairs lie half a head apart and R/2 is a multiple of 8 (they are read
// with a load of their own, which the L1 serves), or within the eight where pairs are neighbours; else
// they are read one by one.
struct Turn8 {
  float c[8], s[8];
  int first;  // of the partners in a row; -1: within the eight, -2: one by one, -3: nothing is rotated
};

__device__ __forceinline__ Turn8 turn8(const Rotation& r, int e, const float2* __restrict__ cs) {
  Turn8 t;
  const int R = 2 * r.pairs;
  t.first = e >= R ? -3 : r.interleaved ? (e + 8 <= R ? -1 : -2) : r.pairs % 8 ? -2 : e < r.pairs ? e + r.pairs : e - r.pairs;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int k = e + i;
    const bool low = r.interleaved ? (i & 1) == 0 : k < r.pairs;  // the pair's first element
    const float2 a = k >= R ? make_float2(1.0f, 0.0f) : cs[r.interleaved ? k >> 1 : low ? k : k - r.pairs];
    t.c[i] = a.x;
    t.s[i] = low ? -a.y : a.y;
  }
  return t;
}

// turn: this lane's row is rotated
template <typename T>
__device__ __forceinline__ void row_values(const T* __restrict__ row, int e, const Rotation& r, bool turn, const Turn8& t,
                                           float (&x)[8]) {
  row_load<T, 8>(row + e, x);
  if (!turn || t.first == -3) return;
  float w[8];
  if (t.first >= 0) {
    row_load<T, 8>(row + t.first, w);
  } else if (t.first == -1) {
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = x[i ^ 1];
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int k = e + i;
      const int other = r.interleaved ? k ^ 1 : k < r.pairs ? k + r.pairs : k - r.pairs;
      w[i] = k < 2 * r.pairs ? ElemT<T>::cvt(row[other]) : 0.0f;
    }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = __builtin_fmaf(x[i], t.c[i], w[i] * t.s[i]);
}

// Keys, values and queries of new tokens: keys and queries rotated, keys and
// values to their places in the pages as 8-bit codes, scale = max|x| / 127 of
// a head's row (at least 1e-12 / 127), code = the rounded quotient; a row
// with a NaN or an infinity has a scale of NaN and codes of zero.  A rotated
// key goes to its codes unrounded.
//
// A wave a token: it finds the token's place and angles (which pass through LDS of its own: no barrier) and takes
// its rows, or blockIdx.y's part of them.  D / 8 lanes a row, so that a lane has the same elements of all of the
// rows and keeps their angles in registers.  11172 tokens of 32 + 8 + 8 heads of 128 in bfloat16: 60 us, 4.2 TB/s, at 74
// registers; bound by the latency of a step's reads at the waves that fit (two or three steps' rows requested at
// once: 66 to 68 us at 90 to 104 registers; four tokens shared by a workgroup's waves: 69).
template <typename T, int D>
__global__ __launch_bounds__(256) void k_kv_append_pages(
    const T* __restrict__ k, int64_t k_token, int64_t k_head, const T* __restrict__ v, int64_t v_token, int64_t v_head,
    const T* __restrict__ q, int64_t q_token, int64_t q_head, int Hq, Rotation r, KvBatch s, KvPool p,
    T* __restrict__ q_out) {
  constexpr int LPR = D / 8, RPW = 64 / LPR;  // lanes a row, rows a wave and step
  __shared__ float2 angles[4][D / 2];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int t = kv_block() * 4 + wave;
  if (t >= s.T) return;
  const int b = kv_sequence(s, t);
  const int64_t place = b < 0 ? 0 : kv_place(s, b, t);
  for (int i = lane; i < r.pairs; i += 64) angles[wave][i] = rot_turn(r, place, t, i);
  // the wave's lanes read each other's angles
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
  const int page = b < 0 || place < 0 ? -1 : kv_page(s, p, b, place >> p.shift);
  const int rows = 2 * p.H + Hq, li = lane % LPR, e = li * 8, sub = lane / LPR;
  const Turn8 turn = turn8(r, e, angles[wave]);
  const T *kt = k + (int64_t)t * k_token, *vt = v + (int64_t)t * v_token, *qt = q + (int64_t)t * q_token;
  T* qo = q_out + (int64_t)t * Hq * D;
  const int64_t values = (int64_t)p.H << p.shift;
  const int64_t key0 = kv_row(p, max(page, 0), 0, 0, (int)(place & ((1 << p.shift) - 1)));
  // every lane of a wave takes part in the reductions: a row past the end is the last one again, not stored
  for (int first = blockIdx.y * RPW; first < rows; first += gridDim.y * RPW) {
    const int row = min(first + sub, rows - 1);
    const bool is_q = row >= 2 * p.H, is_v = !is_q && row >= p.H, live = first + sub < rows;
    float x[8];
    row_values<T>(is_q ? qt + (row - 2 * p.H) * q_head : is_v ? vt + (row - p.H) * v_head : kt + row * k_head, e, r, !is_v,
                  turn, x);
    if (is_q && live) {
      float y[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] = b < 0 ? 0.0f : x[i];
      row_store<T, 8>(qo + (row - 2 * p.H) * D + e, y);
    }
    if (first >= 2 * p.H) continue;  // queries alone
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, mag_bits(x[i]));
    m = group_max_u<LPR>(m);
    const bool whole = m < 0x7F800000u;
    const float scale = amax_clamped(m) / 127.0f;
    div_rn_all<8>(x, scale, 1.0f / scale);
    uint32_t w[2] = {0u, 0u};
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i >> 2] |= ((uint32_t)encode_vec_q(x[i], 127.0f) & 255u) << (8 * (i & 3));
    if (!is_q && page >= 0 && live) {
      const int64_t dst = key0 + (is_v ? values : 0) + ((int64_t)(is_v ? row - p.H : row) << p.shift);
      *reinterpret_cast<u32x2*>(p.codes + dst * D + e) = whole ? u32x2{w[0], w[1]} : u32x2{0u, 0u};
      if (li == 0) p.scales[dst] = whole ? scale : __uint_as_float(0x7FC00000u);
    }
  }
}

// ---------------------------------------------------------------- read
// Values of the T positions lengths[b] + i as rows of k and v; zeros for a
// token without a place.  A wave a token (and part of its rows), 8 codes a lane.  11172 tokens of 8 heads of 128 as
// bfloat16: 15 us, 4.6 TB/s; of one token, latency (3 us).
template <typename T, int D>
__global__ __launch_bounds__(256) void k_kv_read(KvBatch s, KvPool p, T* __restrict__ k, T* __restrict__ v) {
  constexpr int LPR = D / 8;
  const int t = kv_block() * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (t >= s.T) return;
  const int b = kv_sequence(s, t);
  const int64_t at = b < 0 ? -1 : kv_place(s, b, t);
  const int page = at < 0 ? -1 : kv_page(s, p, b, at >> p.shift);
  const int pos = (int)(at & ((1 << p.shift) - 1));
  const int step = gridDim.y * 64, items = 2 * p.H * LPR;
  for (int first = blockIdx.y * 64 + lane; first < items; first += 4 * step) {
    u32x2 c[4];
    float scale[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {  // four requests in flight
      const int row = min(first + u * step, items - 1) / LPR, e = (first + u * step) % LPR * 8;
      const int which = row >= p.H, h = which ? row - p.H : row;
      c[u] = u32x2{0u, 0u};
      scale[u] = 0.0f;
      if (page >= 0) {
        const int64_t src = kv_row(p, page, which, h, pos);
        c[u] = *reinterpret_cast<const u32x2*>(p.codes + src * D + e);
        scale[u] = p.scales[src];
      }
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int it = first + u * step, row = it / LPR, e = it % LPR * 8;
      if (it >= items) break;
      const int which = row >= p.H, h = which ? row - p.H : row;
      float x[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = (float)((int)(c[u][i >> 2] << (24 - 8 * (i & 3))) >> 24) * scale[u];
      row_store<T, 8>((which ? v : k) + ((int64_t)t * p.H + h) * D + e, x);
    }
  }
}

// ---------------------------------------------------------------- keep
// Position lengths[b] + j takes the row of new token path[b][j], for every
// entry inside [0, its sequence's new tokens).  One workgroup a sequence and
// head holds all the rows in LDS before it writes any, so that a row may be
// read by one entry and written by another, in any order.  250 paths of 1 to 16, 8.5 on average, in 16
// heads of 128: 8.5 us for 18 MB, bound by the latency of look-up, reads and writes one after the other.
#define MXK_KEEP_MOST 64
template <int D>
__global__ __launch_bounds__(256) void k_kv_keep(KvBatch s, KvPool p, const int* __restrict__ path, int L) {
  constexpr int C = D / 16;
  extern __shared__ u32x4 held[];  // [2][L][C]
  __shared__ float scale[2][MXK_KEEP_MOST];
  __shared__ int64_t from[MXK_KEEP_MOST], to[MXK_KEEP_MOST];  // row of the key; -1: none
  const int b = blockIdx.x, h = blockIdx.y;
  const int64_t values = (int64_t)p.H << p.shift;  // rows between a page's keys and its values
  for (int j = threadIdx.x; j < L; j += 256) {
    const int pick = path[(int64_t)b * L + j];
    const int64_t held_at = s.lengths[b], src = held_at + pick, dst = held_at + j;
    from[j] = to[j] = -1;
    if (held_at >= 0 && pick >= 0 && pick < kv_count(s, b)) {
      const int sp = kv_page(s, p, b, src >> p.shift), dp = kv_page(s, p, b, dst >> p.shift);
      const int in = (1 << p.shift) - 1;
      if (sp >= 0 && dp >= 0) {
        from[j] = kv_row(p, sp, 0, h, (int)(src & in));
        to[j] = kv_row(p, dp, 0, h, (int)(dst & in));
      }
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < 2 * L * C; i += 256) {
    const int which = i >= L * C, rest = which ? i - L * C : i, j = rest / C, c = rest - j * C;
    if (from[j] < 0) continue;
    const int64_t row = from[j] + (which ? values : 0);
    held[i] = *reinterpret_cast<const u32x4*>(p.codes + row * D + c * 16);
    if (c == 0) scale[which][j] = p.scales[row];
  }
  __syncthreads();
  for (int i = threadIdx.x; i < 2 * L * C; i += 256) {
    const int which = i >= L * C, rest = which ? i - L * C : i, j = rest / C, c = rest - j * C;
    if (to[j] < 0) continue;
    const int64_t row = to[j] + (which ? values : 0);
    *reinterpret_cast<u32x4*>(p.codes + row * D + c * 16) = held[i];
    if (c == 0) p.scales[row] = scale[which][j];
  }
}

// ---------------------------------------------------------------- host
static int check_pool(const char* who, const void* codes, const void* scales, int64_t pages, int page, int H, int D) {
  const std::string w(who);
  if (pages < 0 || pages >= ((int64_t)1 << 31) || H < 1 || H > 1024 || !kv_page_ok(page))
    return fail(MXK_EINVAL, w + ": pages below 2^31 of a power of two of positions from 16 on, 1 to 1024 heads");
  if (D != 64 && D != 128 && D != 256) return fail(MXK_EUNSUPPORTED, w + ": heads of 64, 128 or 256 elements");
  if (pages > 0 && (!codes || !scales)) return fail(MXK_EINVAL, w + ": null pointer");
  if (!aligned16(codes) || !aligned16(scales)) return fail(MXK_EINVAL, w + ": codes and scales start on 16 bytes");
  return MXK_OK;
}

static int check_batch(const char* who, const int32_t* table, const int32_t* lengths, const int32_t* offsets,
                       int64_t B, int64_t width, int64_t T) {
  const std::string w(who);
  if (B < 0 || width < 0 || T < 0 || B >= ((int64_t)1 << 24) || width >= ((int64_t)1 << 31) ||
      T > (int64_t)1 << 30)
    return fail(MXK_EINVAL, w + ": bad sizes (sequences below 2^24, pages of one below 2^31, at most 2^30 tokens)");
  if (!offsets || (B > 0 && (!lengths || (width > 0 && !table)))) return fail(MXK_EINVAL, w + ": null pointer");
  return MXK_OK;
}

static int check_rotation(const char* who, const double* freqs, int pairs, int64_t axes, int pos_bytes,
                          const void* pos, int64_t D, bool own_place) {
  const std::string w(who);
  if (pairs < 0 || 2 * (int64_t)pairs > D) return fail(MXK_EINVAL, w + ": more rotated elements than a head has");
  if (pairs == 0) return MXK_OK;
  if (!freqs || (!pos && !own_place)) return fail(MXK_EINVAL, w + ": null pointer");
  if (pos && (axes < 1 || axes > 1024 || (pos_bytes != 4 && pos_bytes != 8)))
    return fail(MXK_EINVAL, w + ": positions of 4 or 8 bytes on 1 to 1024 axes");
  return MXK_OK;
}

static KvPool make_pool(void* codes, float* scales, int64_t pages, int page, int H) {
  return KvPool{reinterpret_cast<int8_t*>(codes), scales, (uint32_t)pages, H, log2_of(page)};
}
static KvBatch make_batch(const int32_t* table, const int32_t* lengths, const int32_t* offsets, int64_t B,
                          int64_t width, int64_t T) {
  return KvBatch{table, lengths, offsets, (int)B, (int)width, (int)T};
}

template <typename T>
static int launch_rotary(const void* x, int64_t ts, int64_t hs, const Rotation& r, int64_t T_, int H, int D, void* y,
                         hipStream_t st) {
  const int rest = D - 2 * r.pairs;
  int V = 8;
  while (V > 1 && (r.pairs % V || rest % V)) V >>= 1;
  const uint32_t per_head = (uint32_t)(r.pairs / V + rest / V), per_token = per_head * (uint32_t)H;
  // Tokens a workgroup: as many as give each thread an angle, if that leaves two workgroups a CU; never
  // more than LDS holds or 2^31 items.
  int64_t TB = std::max<int64_t>(1, 256 / std::max(1, r.pairs));
  TB = std::max<int64_t>(1, std::min(TB, T_ / (2 * num_cus())));
  TB = std::min<int64_t>(TB, std::max<int64_t>(1, ((int64_t)1 << 30) / per_token));
  const int64_t blocks = ceil_div(T_, TB);
  // few tokens of many heads: a workgroup takes a part of a token's items
  const int64_t parts = std::min<int64_t>(ceil_div((int64_t)per_token * TB, 256),
                                          std::max<int64_t>(1, (2 * num_cus()) / std::max<int64_t>(1, blocks)));
  const dim3 grid = kv_grid(blocks, std::min<int64_t>(parts, 65535));
  const size_t lds = (size_t)TB * r.pairs * sizeof(float2);
  const T* xp = reinterpret_cast<const T*>(x);
  T* yp = reinterpret_cast<T*>(y);
  const DivU32 bt = make_divu32(per_token), bh = make_divu32(per_head);
#define MXK_R(V_)                                                                                                    \
  hipLaunchKernelGGL((k_rotary<T, V_>), grid, dim3(256), lds, st, xp, ts, hs, r, (int)T_, D, (int)TB, per_token, bt, \
                     per_head, bh, H, yp)
  if (V == 8) MXK_R(8);
  else if (V == 4) MXK_R(4);
  else if (V == 2) MXK_R(2);
  else MXK_R(1);
#undef MXK_R
  return check_launch("rotary");
}

template <typename T, int D>
static int launch_append(const void* k, int64_t kt, int64_t kh, const void* v, int64_t vt, int64_t vh, const void* q,
                         int64_t qt, int64_t qh, int Hq, const Rotation& r, const KvBatch& s, const KvPool& p,
                         void* q_out, hipStream_t st) {
  const int steps = (int)ceil_div(2 * p.H + Hq, 64 / (D / 8));
  const int64_t blocks = ceil_div(s.T, 4);
  // few tokens: a wave takes a part of a token's rows, down to one step of them
  const int64_t parts = std::min<int64_t>(steps, std::max<int64_t>(1, 4 * num_cus() / blocks));
  const dim3 grid = kv_grid(blocks, parts);
  hipLaunchKernelGGL((k_kv_append_pages<T, D>), grid, dim3(256), 0, st, reinterpret_cast<const T*>(k), kt, kh,
                     reinterpret_cast<const T*>(v), vt, vh, reinterpret_cast<const T*>(q), qt, qh, Hq, r, s, p,
                     reinterpret_cast<T*>(q_out));
  return check_launch("kv_append");
}

template <typename T>
static int launch_append_d(int D, const void* k, int64_t kt, int64_t kh, const void* v, int64_t vt, int64_t vh,
                           const void* q, int64_t qt, int64_t qh, int Hq, const Rotation& r, const KvBatch& s,
                           const KvPool& p, void* q_out, hipStream_t st) {
  if (D == 64) return launch_append<T, 64>(k, kt, kh, v, vt, vh, q, qt, qh, Hq, r, s, p, q_out, st);
  if (D == 128) return launch_append<T, 128>(k, kt, kh, v, vt, vh, q, qt, qh, Hq, r, s, p, q_out, st);
  return launch_append<T, 256>(k, kt, kh, v, vt, vh, q, qt, qh, Hq, r, s, p, q_out, st);
}

template <typename T>
static int launch_read(int D, const KvBatch& s, const KvPool& p, void* k, void* v, hipStream_t st) {
  const int64_t blocks = ceil_div(s.T, 4);
  const int64_t parts = std::min<int64_t>(ceil_div((int64_t)2 * p.H * D / 8, 64),
                                          std::max<int64_t>(1, 2 * num_cus() / blocks));
  const dim3 grid = kv_grid(blocks, parts);
  T *kp = reinterpret_cast<T*>(k), *vp = reinterpret_cast<T*>(v);
  if (D == 64) hipLaunchKernelGGL((k_kv_read<T, 64>), grid, dim3(256), 0, st, s, p, kp, vp);
  else if (D == 128) hipLaunchKernelGGL((k_kv_read<T, 128>), grid, dim3(256), 0, st, s, p, kp, vp);
  else hipLaunchKernelGGL((k_kv_read<T, 256>), grid, dim3(256), 0, st, s, p, kp, vp);
  return check_launch("kv_read");
}

}  // namespace mxk

using namespace mxk;

extern "C" {

int mxk_rotary(const void* x, int x_type, int64_t tokens, int heads, int64_t D, int64_t token_stride,
               int64_t head_stride, const double* freqs, const int32_t* axis, int pairs, int interleaved,
               const void* pos, int pos_bytes, int axes, int backward, void* y, void* stream) {
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (tokens < 0 || heads < 0 || D < 0 || tokens > (int64_t)1 << 30 || heads > 65536 || D > 4096 ||
      (int64_t)heads * D >= ((int64_t)1 << 28))
    return fail(MXK_EINVAL, "rotary: bad sizes (at most 2^30 tokens, at most 65536 heads of 4096, below 2^28 elements)");
  if (tokens == 0 || heads == 0 || D == 0) return MXK_OK;
  if (const int rc = check_rotation("rotary", freqs, pairs, axes, pos_bytes, pos, D, false)) return rc;
  if (!x || !y) return fail(MXK_EINVAL, "rotary: null pointer");
  const Rotation r{freqs, axis, pos, pos_bytes == 8, pairs, axes, interleaved != 0, backward ? -1.0f : 1.0f};
  if (x_type == MXK_IN_F32)
    return launch_rotary<float>(x, token_stride, head_stride, r, tokens, heads, (int)D, y, st);
  if (x_type == MXK_IN_F16)
    return launch_rotary<__half>(x, token_stride, head_stride, r, tokens, heads, (int)D, y, st);
  if (x_type == MXK_IN_BF16)
    return launch_rotary<hip_bfloat16>(x, token_stride, head_stride, r, tokens, heads, (int)D, y, st);
  return fail(MXK_EINVAL, "rotary: unknown x_type");
}

int mxk_kv_pages_append(const void* k, int64_t k_token, int64_t k_head, const void* v, int64_t v_token,
                        int64_t v_head, const void* q, int64_t q_token, int64_t q_head, int q_heads, int x_type,
                        void* codes, float* scales, int64_t pages, int page, int heads, int D, const int32_t* table,
                        const int32_t* lengths, const int32_t* offsets, int64_t B, int64_t width, int64_t tokens,
                        const double* freqs, const int32_t* axis, int pairs, int interleaved, const void* pos,
                        int pos_bytes, int axes, void* q_out, void* stream) {
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (const int rc = check_pool("kv_append", codes, scales, pages, page, heads, D)) return rc;
  if (const int rc = check_batch("kv_append", table, lengths, offsets, B, width, tokens)) return rc;
  if (const int rc = check_rotation("kv_append", freqs, pairs, axes, pos_bytes, pos, D, true)) return rc;
  if (x_type != MXK_IN_F32 && x_type != MXK_IN_F16 && x_type != MXK_IN_BF16)
    return fail(MXK_EINVAL, "kv_append: unknown x_type");
  if (q_heads < 0 || q_heads > 65536) return fail(MXK_EINVAL, "kv_append: at most 65536 query heads");
  if (tokens == 0) return MXK_OK;
  if (!k || !v || (q_heads > 0 && (!q || !q_out))) return fail(MXK_EINVAL, "kv_append: null pointer");
  const Rotation r{freqs, axis, pos, pos_bytes == 8, pairs, axes, interleaved != 0, 1.0f};
  const KvBatch s = make_batch(table, lengths, offsets, B, width, tokens);
  const KvPool p = make_pool(codes, scales, pages, page, heads);
  if (x_type == MXK_IN_F32)
    return launch_append_d<float>(D, k, k_token, k_head, v, v_token, v_head, q, q_token, q_head, q_heads, r, s, p,
                                  q_out, st);
  if (x_type == MXK_IN_F16)
    return launch_append_d<__half>(D, k, k_token, k_head, v, v_token, v_head, q, q_token, q_head, q_heads, r, s, p,
                                   q_out, st);
  return launch_append_d<hip_bfloat16>(D, k, k_token, k_head, v, v_token, v_head, q, q_token, q_head, q_heads, r, s,
                                       p, q_out, st);
}

int mxk_kv_pages_read(const void* codes, const float* scales, int64_t pages, int page, int heads, int D,
                      const int32_t* table, const int32_t* lengths, const int32_t* offsets, int64_t B, int64_t width,
                      int64_t tokens, int y_type, void* k, void* v, void* stream) {
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (const int rc = check_pool("kv_read", codes, scales, pages, page, heads, D)) return rc;
  if (const int rc = check_batch("kv_read", table, lengths, offsets, B, width, tokens)) return rc;
  if (tokens == 0) return MXK_OK;
  if (!k || !v) return fail(MXK_EINVAL, "kv_read: null pointer");
  const KvBatch s = make_batch(table, lengths, offsets, B, width, tokens);
  const KvPool p = make_pool(const_cast<void*>(codes), const_cast<float*>(scales), pages, page, heads);
  if (y_type == MXK_IN_F32) return launch_read<float>(D, s, p, k, v, st);
  if (y_type == MXK_IN_F16) return launch_read<__half>(D, s, p, k, v, st);
  if (y_type == MXK_IN_BF16) return launch_read<hip_bfloat16>(D, s, p, k, v, st);
  return fail(MXK_EINVAL, "kv_read: unknown y_type");
}

int mxk_kv_pages_keep(void* codes, float* scales, int64_t pages, int page, int heads, int D, const int32_t* table,
                      const int32_t* lengths, const int32_t* offsets, int64_t B, int64_t width, int64_t tokens,
                      const int32_t* path, int steps, void* stream) {
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (const int rc = check_pool("kv_keep", codes, scales, pages, page, heads, D)) return rc;
  if (const int rc = check_batch("kv_keep", table, lengths, offsets, B, width, tokens)) return rc;
  if (steps < 0 || steps > MXK_KEEP_MOST) return fail(MXK_EINVAL, "kv_keep: paths of at most 64 tokens");
  if (B == 0 || steps == 0) return MXK_OK;
  if (!path) return fail(MXK_EINVAL, "kv_keep: null pointer");
  const KvBatch s = make_batch(table, lengths, offsets, B, width, tokens);
  const KvPool p = make_pool(codes, scales, pages, page, heads);
  const dim3 grid((unsigned)B, (unsigned)heads);
  const size_t lds = (size_t)2 * steps * D;
  if (D == 64) hipLaunchKernelGGL((k_kv_keep<64>), grid, dim3(256), lds, st, s, p, path, steps);
  else if (D == 128) hipLaunchKernelGGL((k_kv_keep<128>), grid, dim3(256), lds, st, s, p, path, steps);
  else hipLaunchKernelGGL((k_kv_keep<256>), grid, dim3(256), lds, st, s, p, path, steps);
  return check_launch("kv_keep");
}

}  // extern "C"
