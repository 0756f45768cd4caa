// Attention of new tokens over a paged 8-bit key-value cache, for gfx950.
//
//   o = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale <q, k_j> - m)
//
// over the keys j that a token sees: those held before the call, and of the
// call's own tokens the ones up to itself, or those whose bit its mask has.
// One pass over the keys with a running maximum m.
//
// Keys.  The codes go to the int8 MFMA as they are stored.  A query row is
// taken to integers of 16 bits (24 for float32 queries) against its largest
// element, as two (three) int8 terms, so that <q, k> is an exact integer:
// the only error is the query's, 2^-16 (2^-24) of its largest element, and a
// key costs no conversion.
//
// Values.  S^T = K Q^T leaves a lane with 8 keys of one query row, which is
// the B operand of O^T = V^T P^T with the keys in an order of their own; the
// lane reads D/16 codes of the same 8 keys, and a byte permute per pair of
// keys transposes them.  code + 128 in the low byte of a float16 is
// (code + 128) * 2^-24; one packed fma makes it code * 2^-9, exact.  The
// probabilities carry the values' scales: p_j * scale_j * 2^(10 - e), e the
// exponent of the largest scale so far, is at most 2^15, and keeps 11 bits (22
// for float32 queries: a second term) down to 2^-24 of the largest.
//
// Work.  The blocks of 128 keys of all sequences, heads and tiles of rows
// lie on one line, which is cut into equal shares, one a workgroup: uneven
// contexts, one long context and a thousand short ones fill the card alike.
// A workgroup's four waves take 32 keys of a block each and are joined in LDS;
// a tile that crosses a cut is left in parts, which a second kernel joins
// in the order of the keys.
#include "mxk_pages.h"

#include <algorithm>
#include <cmath>

namespace mxk {

typedef int i32x4a __attribute__((ext_vector_type(4)));
typedef float f32x4a __attribute__((ext_vector_type(4)));
typedef float f32x16a __attribute__((ext_vector_type(16)));
typedef _Float16 f16x2a __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8a __attribute__((ext_vector_type(8)));


struct AttendArgs {
  const void* q;
  int64_t q_token, q_head;
  KvPool pool;
  KvBatch batch;
  const uint64_t* mask;  // [T][words], null: causal
  int words;
  float scale;  // of the scores, times log2(e)
  int Hq, G;    // query heads; of one key head
  int keys;            // of a block: 128 or 256
  int TT, GC, chunks;  // a tile: TT tokens (a power of two, at most keys) of GC heads, chunks of them over G
  void* out;
  float* part_o;  // [shares][2][rows][D], of their own maximum
  float2* part_s;  // [shares][2][rows]: maximum, sum
};

// ---------------------------------------------------------------- the line of blocks
// sum of floor(i / 2^s) over i < x
__device__ __forceinline__ int64_t sum_floor(int64_t x, int s) {
  const int64_t q = x >> s;
  return ((q * (q - 1) / 2) << s) + q * (x - (q << s));
}

struct Line {
  int rs;  // log2(keys / TT)
  int ts;  // log2(TT)
  int64_t cap;   // positions of the table
  int64_t most;  // blocks that a tile has at most: the table's, at least one.  The workspace is sized by it.
};

// A sequence on the line: per key head, its tiles' blocks one after the other
struct SeqWork {
  int first, n;    // new tokens
  int64_t ctx;     // keys held
  int64_t a;       // causal: token tile t has floor((a + t) / 2^rs) blocks, at most Line::most
  int64_t full;    // causal: the first token tile that has that many
  int64_t blocks;  // masked: of every tile
  int tiles;       // token tiles
  int64_t head;    // blocks of one key head
};

__device__ __forceinline__ int64_t tile_blocks(const AttendArgs& A, const Line& L, const SeqWork& w, int t) {
  return A.mask ? w.blocks : min((w.a + t) >> L.rs, L.most);
}

// Blocks of a key head's token tiles below t
__device__ __forceinline__ int64_t blocks_below(const AttendArgs& A, const Line& L, const SeqWork& w, int t) {
  if (A.mask) return A.chunks * (t * w.blocks);
  const int64_t some = min((int64_t)t, w.full);
  return A.chunks * (sum_floor(w.a + some, L.rs) - sum_floor(w.a, L.rs) + (t - some) * L.most);
}

__device__ __forceinline__ SeqWork seq_work(const AttendArgs& A, const Line& L, int b) {
  SeqWork w;
  w.first = kv_first(A.batch, b);
  w.n = kv_count(A.batch, b);
  w.ctx = min(max((int64_t)A.batch.lengths[b], (int64_t)0), L.cap);
  w.tiles = (w.n + A.TT - 1) >> L.ts;
  w.a = (w.ctx + A.TT + A.keys - 1) >> L.ts;
  w.full = max((int64_t)0, (L.most << L.rs) - w.a);
  w.blocks = min((w.ctx + w.n + A.keys - 1) >> (L.ts + L.rs), L.most);
  w.head = blocks_below(A, L, w, w.tiles);
  return w;
}

__device__ __forceinline__ Line make_line(const AttendArgs& A) {
  Line L;
  L.ts = 31 - __builtin_clz(A.TT);
  L.rs = 31 - __builtin_clz(A.keys) - L.ts;
  L.cap = (int64_t)A.batch.width << A.pool.shift;
  L.most = max((int64_t)1, (L.cap + A.keys - 1) >> (L.ts + L.rs));
  return L;
}

__device__ __forceinline__ int64_t uniform64(int64_t v) {
  const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)v);
  const uint32_t hi = __builtin_amdgcn_readfirstlane((uint32_t)(v >> 32));
  return (int64_t)((uint64_t)hi << 32 | lo);
}

// Blocks of all sequences; every lane of every wave ends with the sum
__device__ __forceinline__ int64_t line_length(const AttendArgs& A, const Line& L) {
  const int lane = threadIdx.x & 63;
  int64_t sum = 0;
  for (int b = lane; b < A.batch.B; b += 64) sum += seq_work(A, L, b).head * A.pool.H;
#pragma unroll
  for (int i = 1; i < 64; i <<= 1) sum += __shfl_xor(sum, i);
  return uniform64(sum);
}

// Share of the line that each of `shares` workgroups takes
__device__ __forceinline__ int64_t line_share(int64_t total, int shares) {
  int64_t per = (int64_t)((double)total / (double)shares);
  while (per * shares < total) ++per;
  return per;
}

// A place on the line: the tile it lies in and the tile's own blocks
struct Place {
  int b, h, x;       // sequence, key head, tile (token tile * chunks + chunk)
  int64_t k;         // block within the tile
  int64_t blocks;    // of the tile
};

// at: below line_length; found by a whole wave, uniform in it
__device__ __forceinline__ Place line_place(const AttendArgs& A, const Line& L, int64_t at, SeqWork& w) {
  const int lane = threadIdx.x & 63;
  int b = 0;
  for (int b0 = 0; b0 < A.batch.B; b0 += 64) {
    const int64_t own = b0 + lane < A.batch.B ? seq_work(A, L, b0 + lane).head * A.pool.H : 0;
    int64_t upto = own;
#pragma unroll
    for (int i = 1; i < 64; i <<= 1) {
      const int64_t o = __shfl_up(upto, i);
      if (lane >= i) upto += o;
    }
    const uint64_t beyond = __ballot(upto > at);
    if (beyond) {
      const int l = __builtin_ctzll(beyond);
      at -= __shfl(upto - own, l);
      b = b0 + l;
      break;
    }
    at -= __shfl(upto, 63);
  }
  Place p;
  p.b = __builtin_amdgcn_readfirstlane(b);
  at = uniform64(at);
  w = seq_work(A, L, p.b);
  p.h = 0;
  while (at >= w.head && p.h < A.pool.H - 1) {  // at most 1024 heads, 64 at once below
    if (at >= 64 * w.head && p.h + 64 < A.pool.H) p.h += 64, at -= 64 * w.head;
    else ++p.h, at -= w.head;
  }
  int lo = 0, hi = w.tiles - 1;  // the last token tile that begins at or before `at`
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (blocks_below(A, L, w, mid) <= at) lo = mid;
    else hi = mid - 1;
  }
  const int t = lo;
  at -= blocks_below(A, L, w, t);
  p.blocks = tile_blocks(A, L, w, t);
  int c = 0;
  while (at >= p.blocks && c < A.chunks - 1) ++c, at -= p.blocks;
  p.x = t * A.chunks + c;
  p.k = at;
  return p;
}

// ---------------------------------------------------------------- query rows
// QT int8 terms of a lane's D/4 elements of query row `row` (null: zeros): elements
// i*64 + g*16 + 0..15 for i < D/64.  unit: what one step of the last term stands for.
template <typename T, int D, int QT>
__device__ __forceinline__ void query_terms(const T* __restrict__ row, int g, i32x4a (&term)[QT][D / 64], float& unit) {
  constexpr float TOP = QT == 2 ? 32512.0f : 8323072.0f;  // 127 * 2^8, 127 * 2^16
  float x[D / 64][16];
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < D / 64; ++i) {
    T e[16];
    if (row) __builtin_memcpy(e, row + i * 64 + g * 16, sizeof(e));
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      x[i][j] = row ? ElemT<T>::cvt(e[j]) : 0.0f;
      m = max(m, mag_bits(x[i][j]));
    }
  }
  m = max(m, (uint32_t)__shfl_xor((int)m, 16));
  m = max(m, (uint32_t)__shfl_xor((int)m, 32));
  const float top = __uint_as_float(m);
  // rows below 2^-100 count as zeros, rows with a NaN or an infinity as NaN
  const bool some = m >= 0x0D800000u && m < 0x7F800000u;
  const float inv = some ? TOP / top : 0.0f;
  unit = m >= 0x7F800000u ? __uint_as_float(0x7FC00000u) : some ? top / TOP : 0.0f;
#pragma unroll
  for (int i = 0; i < D / 64; ++i)
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      uint32_t t[QT] = {};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        int v = some ? (int)rne(x[i][4 * w + j] * inv) : 0;
#pragma unroll
        for (int n = QT - 1; n >= 0; --n) {  // the last term is the lowest
          const int low = n ? ((v + 128) & 255) - 128 : v;
          t[n] |= ((uint32_t)low & 255u) << (8 * j);
          v = (v - low) >> 8;
        }
      }
#pragma unroll
      for (int n = 0; n < QT; ++n) term[n][i][w] = (int)t[n];
    }
}

// ---------------------------------------------------------------- 32 keys
template <int D>
struct Keys32 {
  i32x4a k[2][D / 64];      // codes of key lane%16 (+16): elements i*64 + g*16 + 0..15
  uint32_t v[8][D / 64];    // codes of keys g*4 + 0..3 (+16): elements (lane%16)*(D/16) on
  f32x4a ks[2], vs[2];      // scales of keys g*4 + 0..3 (+16)
  bool ok[2];               // a page is there
};

template <int D>
__device__ __forceinline__ void load_keys(const KvPool& p, int h, int64_t key, const int (&page)[2], int lane,
                                          Keys32<D>& s) {
  const int l = lane & 15, g = lane >> 4;
  const int64_t values = (int64_t)p.H << p.shift;
#pragma unroll
  for (int a = 0; a < 2; ++a) {
    s.ok[a] = page[a] >= 0;
    // without a page: some row of the pool, whose keys nobody sees
    const int64_t row = kv_row(p, max(page[a], 0), 0, h, (int)((key + 16 * a) & ((1 << p.shift) - 1)));
    const int8_t* kc = p.codes + row * D;
#pragma unroll
    for (int i = 0; i < D / 64; ++i)
      s.k[a][i] = *reinterpret_cast<const i32x4a*>(kc + l * D + i * 64 + g * 16);
    const int8_t* vc = p.codes + (row + values) * D;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      __builtin_memcpy(s.v[4 * a + j], vc + (g * 4 + j) * D + l * (D / 16), D / 16);
    s.ks[a] = *reinterpret_cast<const f32x4a*>(p.scales + row + g * 4);
    s.vs[a] = *reinterpret_cast<const f32x4a*>(p.scales + row + values + g * 4);
  }
}

__device__ __forceinline__ float scale_of_exp(int e) {  // 2^e, zero below the normal range
  return e < -126 ? 0.0f : __uint_as_float((uint32_t)(min(e, 127) + 127) << 23);
}

// One tile over blocks [k0, k1): four waves, 32 keys of a block each
template <typename T, int D, int QT, int PT>
struct TileState {
  f32x4a o[D / 16];  // row lane%16, elements (g*4 + r) * (D/16) + j in o[j][r], times 2^(1 - e)
  float m, l;        // maximum (log2 units), the lane's own sum
  int e;             // exponent of the largest value scale, wave-uniform
};

template <typename T, int D, int QT, int PT>
__device__ __forceinline__ void step32(const AttendArgs& A, const i32x4a (&q)[QT][D / 64], float unit, Keys32<D>& s,
                                       int64_t key, int64_t ctx, int64_t end, int tok, const uint64_t* __restrict__ bits,
                                       int lane, TileState<T, D, QT, PT>& st) {
  const int g = lane >> 4;
  float t[8];
#pragma unroll
  for (int a = 0; a < 2; ++a) {
    i32x4a acc[QT];
#pragma unroll
    for (int n = 0; n < QT; ++n) {
      acc[n] = i32x4a{0, 0, 0, 0};
#pragma unroll
      for (int i = 0; i < D / 64; ++i) acc[n] = __builtin_amdgcn_mfma_i32_16x16x64_i8(s.k[a][i], q[n][i], acc[n], 0, 0, 0);
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      float f = (float)(acc[0][r] * 256 + acc[1][r]);
      if constexpr (QT == 3) f = __builtin_fmaf(f, 256.0f, (float)acc[2][r]);
      t[4 * a + r] = f * s.ks[a][r] * unit;
    }
  }
  float vs[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) vs[i] = s.vs[i >> 2][i & 3];
  if (key + 32 > min(ctx, end) || !s.ok[0] || !s.ok[1]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int64_t at = key + 16 * (i >> 2) + 4 * g + (i & 3), j = at - ctx;
      bool see = at < end && s.ok[i >> 2];
      if (see && j >= 0) see = bits ? j < 64 * (int64_t)A.words && (bits[j >> 6] >> (j & 63) & 1) : j <= tok;
      if (!see) t[i] = -__builtin_inff(), vs[i] = 0.0f;
    }
  }
  // A new maximum or a new largest scale: the sums so far are taken to it.  Up to 2^4 above the
  // maximum in use needs no step (the probabilities' range has room for it), so that after the
  // first blocks a wave seldom takes one.
  float top = t[0];
  uint32_t big = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    top = fmaxf(top, t[i]);
    const uint32_t b = mag_bits(vs[i]);
    big = max(big, b < 0x7F800000u ? b : 0u);
  }
  const int eb = (int)(big >> 23) - 127;
  if (__ballot(top > st.m + 4.0f || eb > st.e)) {
    top = fmaxf(top, __shfl_xor(top, 16));
    top = fmaxf(top, __shfl_xor(top, 32));
    int e = eb;
#pragma unroll
    for (int i = 1; i < 64; i <<= 1) e = max(e, __shfl_xor(e, i));
    e = max(e, st.e);
    const float m = fmaxf(st.m, top);
    const float shrink = m == st.m ? 1.0f : __builtin_amdgcn_exp2f(st.m - m);
    const float both = shrink * scale_of_exp(st.e - e);
    st.l *= shrink;
#pragma unroll
    for (int j = 0; j < D / 16; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r) st.o[j][r] *= both;
    st.m = m;
    st.e = e;
  }
  const float m = st.m == -__builtin_inff() ? 0.0f : st.m;
  const float up = scale_of_exp(10 - st.e);
  f16x8a p[PT];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float w = __builtin_amdgcn_exp2f(t[i] - m);
    st.l += w;
    float c = w * (vs[i] * up);
    // One rounding of c for both of its uses: the compiler fuses the product into one of two conversions, which then
    // differ where c lies between two float16 (a probability 2^-11 off in 1 of 2^14)
    if constexpr (PT == 2) asm("" : "+v"(c));
    p[0][i] = (_Float16)c;
    if constexpr (PT == 2) p[1][i] = (_Float16)(c - (float)p[0][i]);
  }
#pragma unroll
  for (int j = 0; j < D / 16; ++j) {
    typedef uint32_t u32x4v __attribute__((ext_vector_type(4)));
    u32x4v w;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t sel = 0x0C000C00u | (uint32_t)(j & 3) | (uint32_t)(4 + (j & 3)) << 16;
      const uint32_t pair = __builtin_amdgcn_perm(s.v[2 * i + 1][j >> 2] ^ 0x80808080u, s.v[2 * i][j >> 2] ^ 0x80808080u, sel);
      const f16x2a h = __builtin_elementwise_fma(__builtin_bit_cast(f16x2a, pair), f16x2a{32768.0f, 32768.0f},
                                                 f16x2a{-0.25f, -0.25f});
      w[i] = __builtin_bit_cast(uint32_t, h);
    }
    const f16x8a v = __builtin_bit_cast(f16x8a, w);
#pragma unroll
    for (int n = 0; n < PT; ++n) st.o[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, p[n], st.o[j], 0, 0, 0);
  }
}

template <typename T>
__device__ __forceinline__ T out_cvt(float v) {
  if constexpr (__is_same(T, float)) return v;
  else if constexpr (__is_same(T, __half)) return __float2half_rn(v);
  else return __builtin_bit_cast(hip_bfloat16, (__bf16)v);
}

// Row r of a tile: its token in the sequence and its query head; false: none
__device__ __forceinline__ bool tile_row(const AttendArgs& A, const SeqWork& w, const Place& p, int r, int& tok,
                                         int& head) {
  const int t = p.x / A.chunks, c = p.x - t * A.chunks;
  const int i = r / A.GC, hh = c * A.GC + (r - i * A.GC);
  tok = t * A.TT + i;
  head = p.h * A.G + hh;
  return i < A.TT && tok < w.n && hh < A.G;
}

// Rows of tokens that no sequence has
template <typename T, int D, int THREADS>
__device__ __forceinline__ void zero_padding(const AttendArgs& A, int shares) {
  const int B = A.batch.B;
  const int lo = B ? min(max(A.batch.offsets[0], 0), A.batch.T) : 0;
  const int hi = B ? min(max(A.batch.offsets[B], 0), A.batch.T) : 0;
  const int64_t row = (int64_t)A.Hq * D, n = (lo + (A.batch.T - hi)) * row;
  T* out = reinterpret_cast<T*>(A.out);
  for (int64_t i = (int64_t)blockIdx.x * THREADS + threadIdx.x; i < n; i += (int64_t)shares * THREADS)
    out[i < lo * row ? i : i - lo * row + hi * row] = out_cvt<T>(0.0f);
}

// The next tile on the line (there is one)
__device__ __forceinline__ void next_tile(const AttendArgs& A, const Line& L, SeqWork& w, Place& p) {
  p.k = 0;
  if (++p.x == w.tiles * A.chunks) {
    p.x = 0;
    if (++p.h == A.pool.H) {
      p.h = 0;
      do ++p.b, w = seq_work(A, L, p.b);
      while (w.head == 0);
    }
  }
  p.blocks = tile_blocks(A, L, w, p.x / A.chunks);
}

// Tiles of 16 rows
template <typename T, int D, int QT, int PT>
__global__ __launch_bounds__(256, D == 256 ? 1 : 2) void k_attend(AttendArgs A, int shares) {
  constexpr int LD = D + 4;
  __shared__ float so[4][16][LD];
  __shared__ float sm[4][16], sl[4][16];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int l16 = lane & 15, g = lane >> 4;
  const Line L = make_line(A);
  const int64_t total = line_length(A, L);
  const int64_t per = line_share(total, shares);
  const int64_t from = (int64_t)blockIdx.x * per, to = min(total, from + per);

  zero_padding<T, D, 256>(A, shares);
  if (from >= to) return;

  SeqWork w;
  Place p = line_place(A, L, from, w);
  int64_t at = from;
  while (true) {
    const int64_t k1 = min(p.blocks, p.k + (to - at));
    const bool whole = p.k == 0 && k1 == p.blocks;
    int tok, head;
    const bool row_ok = tile_row(A, w, p, l16, tok, head);
    i32x4a q[QT][D / 64];
    float unit;
    query_terms<T, D, QT>(row_ok ? reinterpret_cast<const T*>(A.q) + (int64_t)(w.first + tok) * A.q_token +
                                       (int64_t)head * A.q_head
                                 : nullptr,
                          g, q, unit);
    unit *= A.scale;
    const uint64_t* bits = A.mask && row_ok ? A.mask + (int64_t)(w.first + tok) * A.words : A.mask;
    const int64_t end = min(L.cap, w.ctx + (A.mask ? w.n : min(w.n, (p.x / A.chunks + 1) * A.TT)));
    TileState<T, D, QT, PT> st;
#pragma unroll
    for (int j = 0; j < D / 16; ++j) st.o[j] = f32x4a{0, 0, 0, 0};
    st.m = -__builtin_inff();
    st.l = 0.0f;
    st.e = -100;  // smaller scales lose bits
    int64_t key = p.k * 128 + wave * 32;
    const int64_t stop = min(end, k1 * 128);
    if (key < stop) {
      Keys32<D> cur, nxt;
      int page[2];
#pragma unroll
      for (int a = 0; a < 2; ++a) page[a] = kv_page(A.batch, A.pool, p.b, (key + 16 * a) >> A.pool.shift);
      load_keys<D>(A.pool, p.h, key, page, lane, cur);
      while (true) {
        const int64_t next = key + 128;
        const bool more = next < stop;
        if (more) {
#pragma unroll
          for (int a = 0; a < 2; ++a) page[a] = kv_page(A.batch, A.pool, p.b, (next + 16 * a) >> A.pool.shift);
          load_keys<D>(A.pool, p.h, next, page, lane, nxt);
        }
        step32<T, D, QT, PT>(A, q, unit, cur, key, w.ctx, end, tok, bits, lane, st);
        if (!more) break;
        cur = nxt;
        key = next;
      }
    }
    // the four waves' sums, each of its own maximum
    float l = st.l;
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    const float down = scale_of_exp(st.e - 1);
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int j = 0; j < D / 16; ++j) so[wave][l16][(g * 4 + r) * (D / 16) + j] = st.o[j][r] * down;
    if (g == 0) sm[wave][l16] = st.m, sl[wave][l16] = l;
    __syncthreads();
    {
      const int r = threadIdx.x >> 4, d0 = (threadIdx.x & 15) * (D / 16);
      float m = -__builtin_inff();
#pragma unroll
      for (int i = 0; i < 4; ++i) m = fmaxf(m, sm[i][r]);
      float sum = 0.0f, acc[D / 16];
#pragma unroll
      for (int j = 0; j < D / 16; ++j) acc[j] = 0.0f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        // a wave whose keys the row does not see adds nothing; NaN scores leave m at -inf and their sum NaN
        const float f = sm[i][r] == m ? 1.0f : __builtin_amdgcn_exp2f(sm[i][r] - m);
        sum += f * sl[i][r];
#pragma unroll
        for (int j = 0; j < D / 16; ++j) acc[j] = __builtin_fmaf(f, so[i][r][d0 + j], acc[j]);
      }
      int rt, rh;
      if (tile_row(A, w, p, r, rt, rh)) {
        if (whole) {
          T* dst = reinterpret_cast<T*>(A.out) + ((int64_t)(w.first + rt) * A.Hq + rh) * D + d0;
          const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
          T e[D / 16];
#pragma unroll
          for (int j = 0; j < D / 16; ++j) e[j] = out_cvt<T>(acc[j] * inv);
          __builtin_memcpy(dst, e, sizeof(e));
        } else {
          const int64_t slot = ((int64_t)blockIdx.x * 2 + (p.k == 0 ? 1 : 0)) * 16 + r;
          __builtin_memcpy(A.part_o + slot * D + d0, acc, sizeof(acc));
          if ((threadIdx.x & 15) == 0) A.part_s[slot] = make_float2(m, sum);
        }
      }
    }
    at += k1 - p.k;
    if (at >= to) break;
    __syncthreads();
    next_tile(A, L, w, p);
  }
}

// ---------------------------------------------------------------- tiles of many rows
// NW waves of 32 rows each share the keys, 64 at a time: their codes are
// made float16 (code * 2^-9, exact) once for the workgroup on the way into LDS,
// values transposed, and both products run on the 32x32x16 MFMA.  As above S^T
// leaves a lane with one row's keys, which are the second product's operand as
// they are; only the keys' order in LDS follows it: values lie by element, and
// there 16 keys s of a block as two runs of 8, keys 16s + 4h + {0..3, 8..11} for
// the lanes' half h.
//
// Element d of the values is row (d % 4) * (D/4) + d / 4 of LDS: a thread reads
// four elements of four keys, and its writes, like the MFMA's reads, take
// rows that follow each other.  16-byte pieces are swizzled so that neither
// meets itself in a bank.
#define MXK_TILE 64

template <typename T, int D, int QT>
__device__ __forceinline__ void query_halves(const T* __restrict__ row, int h, f16x8a (&q)[QT][D / 16], float& unit) {
  float x[D / 16][8];
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < D / 16; ++i) {
    T e[8];
    if (row) __builtin_memcpy(e, row + i * 16 + h * 8, sizeof(e));
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      x[i][j] = row ? ElemT<T>::cvt(e[j]) : 0.0f;
      m = max(m, mag_bits(x[i][j]));
    }
  }
  m = max(m, (uint32_t)__shfl_xor((int)m, 32));
  // a power of two takes the largest to 2^14 .. 2^15; zeros and NaN as in query_terms
  const bool some = m >= 0x0D800000u && m < 0x7F800000u;
  const int e = some ? (int)(m >> 23) - 127 : 0;
  const float up = some ? scale_of_exp(14 - e) : 0.0f;
  unit = m >= 0x7F800000u ? __uint_as_float(0x7FC00000u) : scale_of_exp(e - 14 + 9);
#pragma unroll
  for (int i = 0; i < D / 16; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      float v = some ? x[i][j] * up : 0.0f;
      if constexpr (QT == 2) asm("" : "+v"(v));  // one rounding for both terms, as for the probabilities
      q[0][i][j] = (_Float16)v;
      if constexpr (QT == 2) q[1][i][j] = (_Float16)(v - (float)q[0][i][j]);
    }
}

// two codes, in the low bytes of the halves (plus 128), as float16 code * 2^-9
__device__ __forceinline__ uint32_t codes_f16(uint32_t pair) {
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(__builtin_bit_cast(f16x2a, pair),
                                                                f16x2a{32768.0f, 32768.0f}, f16x2a{-0.25f, -0.25f}));
}

// Swizzle of the 16-byte pieces of a key's row (D * 2 bytes): 16 rows in a row
// take 16 places of the 256 bytes of all banks
template <int D>
__device__ __forceinline__ int key_swizzle(int row) {
  return D == 64 ? (row >> 1) & 7 : row & 15;
}

template <int D, int NW>
struct TileLds {
  uint32_t k[2][MXK_TILE * D / 2];  // [key][D] float16, pieces of 8 swizzled
  uint32_t v[2][MXK_TILE * D / 2];  // [row][64 keys] float16, pieces of 8 swizzled
  float ks[2][MXK_TILE], vs[2][MXK_TILE];  // vs times 2^(10 - e)
  int e[2];
  uint32_t ok[2];  // bits of the block's runs of 16 keys that have a page
};

template <typename T, int D, int QT, int PT, int NW>
__global__ __launch_bounds__(64 * NW, NW == 8 || D == 256 ? 1 : 2) void k_attend_tile(AttendArgs A, int shares) {
  constexpr int P = 8 / NW;          // pieces of 16 bytes of keys (and of values) a thread and D = 128
  constexpr int KP = P * D / 128 > 0 ? P * D / 128 : 1;
  constexpr int CPR = D / 16;        // 16-byte pieces of a row of codes
  constexpr int PIECES = MXK_TILE * CPR;
  __shared__ TileLds<D, NW> S;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l32 = lane & 31, h = lane >> 5;
  const Line L = make_line(A);
  const int64_t total = line_length(A, L);
  const int64_t per = line_share(total, shares);
  // neighbours on the line read the same keys: they go to one XCD
  const int share = shares % 8 == 0 ? (blockIdx.x & 7) * (shares >> 3) + (blockIdx.x >> 3) : blockIdx.x;
  const int64_t from = (int64_t)share * per, to = min(total, from + per);
  zero_padding<T, D, 64 * NW>(A, shares);
  if (from >= to) return;

  SeqWork w;
  Place p = line_place(A, L, from, w);
  int64_t at = from;
  while (true) {
    const int64_t k1 = min(p.blocks, p.k + (to - at));
    const bool whole = p.k == 0 && k1 == p.blocks;
    int tok, head;
    const bool row_ok = tile_row(A, w, p, wave * 32 + l32, tok, head);
    const bool busy = __ballot(row_ok) != 0;
    f16x8a q[QT][D / 16];
    float unit;
    query_halves<T, D, QT>(row_ok ? reinterpret_cast<const T*>(A.q) + (int64_t)(w.first + tok) * A.q_token +
                                        (int64_t)head * A.q_head
                                  : nullptr,
                           h, q, unit);
    unit *= A.scale;
    const uint64_t* bits = A.mask && row_ok ? A.mask + (int64_t)(w.first + tok) * A.words : A.mask;
    const int64_t end = min(L.cap, w.ctx + (A.mask ? w.n : min(w.n, (p.x / A.chunks + 1) * A.TT)));
    const int64_t key0 = p.k * A.keys, stop = min(end, k1 * A.keys);
    // the wave's first and last token: between them a causal block needs its mask
    int lo_tok = row_ok ? tok : 0x7FFFFFFF, hi_tok = row_ok ? tok : -1;
#pragma unroll
    for (int i = 1; i < 32; i <<= 1) lo_tok = min(lo_tok, __shfl_xor(lo_tok, i)), hi_tok = max(hi_tok, __shfl_xor(hi_tok, i));
    lo_tok = __builtin_amdgcn_readfirstlane(lo_tok);
    hi_tok = __builtin_amdgcn_readfirstlane(hi_tok);

    f32x16a o[D / 32];
#pragma unroll
    for (int j = 0; j < D / 32; ++j)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[j][i] = 0.0f;
    float m = -__builtin_inff(), l = 0.0f;
    int e = -100;

    // codes of a block on their way: the thread's pieces of keys, and four keys by four elements of values
    u32x4 kr[KP];
    uint32_t vr[KP][4];
    float sr = 0.0f;
    int run_ok = 0;
    auto fetch = [&](int64_t key) {
#pragma unroll
      for (int i = 0; i < KP; ++i) {
        const int piece = tid + i * 64 * NW, row = piece / CPR, c = piece % CPR;
        if (piece >= PIECES) break;
        const int64_t kk = key + row;
        const int page = kv_page(A.batch, A.pool, p.b, kk >> A.pool.shift);
        const int64_t src = kv_row(A.pool, max(page, 0), 0, p.h, (int)(kk & ((1 << A.pool.shift) - 1)));
        kr[i] = *reinterpret_cast<const u32x4*>(A.pool.codes + src * D + c * 16);
      }
#pragma unroll
      for (int i = 0; i < KP; ++i) {
        const int piece = tid + i * 64 * NW, four = piece / (D / 4), c = piece % (D / 4);
        if (piece >= PIECES) break;
        const int64_t kk = key + four * 4;
        const int page = kv_page(A.batch, A.pool, p.b, kk >> A.pool.shift);
        const int64_t src = kv_row(A.pool, max(page, 0), 1, p.h, (int)(kk & ((1 << A.pool.shift) - 1)));
#pragma unroll
        for (int r = 0; r < 4; ++r)
          vr[i][r] = *reinterpret_cast<const uint32_t*>(A.pool.codes + (src + r) * D + c * 4);
      }
      if (wave < 2) {
        const int64_t kk = key + lane;
        const int page = kk < end ? kv_page(A.batch, A.pool, p.b, kk >> A.pool.shift) : -1;
        sr = 0.0f;
        if (page >= 0) sr = A.pool.scales[kv_row(A.pool, page, wave, p.h, (int)(kk & ((1 << A.pool.shift) - 1)))];
        run_ok = page >= 0;
      }
    };
    int e_run = -100;  // of wave 1, which finds the exponent for all
    auto put = [&](int buf) {
#pragma unroll
      for (int i = 0; i < KP; ++i) {
        const int piece = tid + i * 64 * NW, row = piece / CPR, c = piece % CPR;
        if (piece >= PIECES) break;
        u32x4 half[2];
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const uint32_t u = kr[i][x] ^ 0x80808080u;
          half[x >> 1][2 * (x & 1)] = codes_f16(__builtin_amdgcn_perm(0u, u, 0x0C010C00u));
          half[x >> 1][2 * (x & 1) + 1] = codes_f16(__builtin_amdgcn_perm(0u, u, 0x0C030C02u));
        }
#pragma unroll
        for (int x = 0; x < 2; ++x)
          *reinterpret_cast<u32x4*>(&S.k[buf][row * (D / 2) + (((2 * c + x) ^ key_swizzle<D>(row)) * 4)]) = half[x];
      }
#pragma unroll
      for (int i = 0; i < KP; ++i) {
        const int piece = tid + i * 64 * NW, four = piece / (D / 4), c = piece % (D / 4);
        if (piece >= PIECES) break;
        // keys 16s + 8b + 4h': run s*2 + h', its half b
        const int run = (four >> 2) * 2 + (four & 1), b = (four >> 1) & 1;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t sel = 0x0C000C00u | (uint32_t)j | (uint32_t)(4 + j) << 16;
          u32x2 two;
#pragma unroll
          for (int x = 0; x < 2; ++x)
            two[x] = codes_f16(__builtin_amdgcn_perm(vr[i][2 * x + 1] ^ 0x80808080u, vr[i][2 * x] ^ 0x80808080u, sel));
          const int row = j * (D / 4) + c;
          *reinterpret_cast<u32x2*>(&S.v[buf][row * (MXK_TILE / 2) + ((run ^ ((row >> 1) & 7)) * 4) + b * 2]) = two;
        }
      }
      if (wave == 0) S.ks[buf][lane] = sr;
      if (wave == 1) {
        const uint32_t bb = mag_bits(sr);
        int top = (int)((bb < 0x7F800000u ? bb : 0u) >> 23) - 127;
#pragma unroll
        for (int i = 1; i < 64; i <<= 1) top = max(top, __shfl_xor(top, i));
        e_run = max(e_run, top);
        S.vs[buf][lane] = sr * scale_of_exp(10 - e_run);
        const uint64_t b = __ballot(run_ok);
        if (lane == 0) {
          S.e[buf] = e_run;
          S.ok[buf] = (uint32_t)(b & 1) | (uint32_t)(b >> 16 & 1) << 1 | (uint32_t)(b >> 32 & 1) << 2 |
                      (uint32_t)(b >> 48 & 1) << 3;
        }
      }
    };

    __syncthreads();  // the tile before is read
    if (key0 < stop) {
      fetch(key0);
      put(0);
    }
    __syncthreads();
    int buf = 0;
    for (int64_t key = key0; key < stop; key += MXK_TILE, buf ^= 1) {
      const bool more = key + MXK_TILE < stop;
      if (more) fetch(key + MXK_TILE);
      const int e_new = __builtin_amdgcn_readfirstlane(S.e[buf]);
      const uint32_t ok = __builtin_amdgcn_readfirstlane(S.ok[buf]);
      const int64_t j0 = key - w.ctx;  // the first key among the new tokens
      // rows of tokens before the whole block see none of it
      if (busy && (A.mask || j0 <= hi_tok)) {
        const bool open = key + MXK_TILE <= end && ok == 15 && (j0 + MXK_TILE <= 0 || (!A.mask && j0 + MXK_TILE - 1 <= lo_tok));
        uint64_t see = ~0ull;
        if (!open) {
          if (A.mask) {
            const int64_t word = j0 >= 0 ? j0 >> 6 : -1;
            const uint64_t none = 0;
            if (j0 >= 0) {
              const int sh = (int)(j0 & 63);
              const uint64_t one = word < A.words ? bits[word] : none;
              const uint64_t two = word + 1 < A.words ? bits[word + 1] : none;
              see = sh ? one >> sh | two << (64 - sh) : one;
            } else if (j0 > -MXK_TILE) {
              see = bits[0] << (int)-j0 | ((1ull << (int)-j0) - 1);
            }
          } else {
            const int64_t last = tok - j0;  // the last key of the block that the row sees
            see = last < 0 ? 0 : last >= 63 ? ~0ull : (2ull << (int)last) - 1;
          }
          if (key + MXK_TILE > end) see &= (1ull << (int)(end - key)) - 1;
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (!(ok >> i & 1)) see &= ~(0xFFFFull << (16 * i));
          see >>= 4 * h;
        }
        float t[2][16];
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) {
          f32x16a acc;
#pragma unroll
          for (int i = 0; i < 16; ++i) acc[i] = 0.0f;
          const int row = kt * 32 + l32;
#pragma unroll
          for (int i = 0; i < D / 16; ++i) {
            const f16x8a kf = *reinterpret_cast<const f16x8a*>(&S.k[buf][row * (D / 2) + (((2 * i + h) ^ key_swizzle<D>(row)) * 4)]);
#pragma unroll
            for (int n = 0; n < QT; ++n) acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf, q[n][i], acc, 0, 0, 0);
          }
#pragma unroll
          for (int a = 0; a < 4; ++a) {
            const f32x4a s4 = *reinterpret_cast<const f32x4a*>(&S.ks[buf][kt * 32 + a * 8 + h * 4]);
#pragma unroll
            for (int r = 0; r < 4; ++r) t[kt][4 * a + r] = acc[4 * a + r] * s4[r];
          }
        }
        if (!open) {
#pragma unroll
          for (int kt = 0; kt < 2; ++kt)
#pragma unroll
            for (int i = 0; i < 16; ++i)
              if (!((uint32_t)(see >> (32 * kt)) >> (8 * (i >> 2) + (i & 3)) & 1)) t[kt][i] = -__builtin_inff();
        }
        float top = t[0][0];
#pragma unroll
        for (int kt = 0; kt < 2; ++kt)
#pragma unroll
          for (int i = 0; i < 16; ++i) top = fmaxf(top, t[kt][i]);
        top *= unit;
        if (__ballot(top > m + 4.0f) || e_new != e) {
          top = fmaxf(top, __shfl_xor(top, 32));
          const float mm = fmaxf(m, top);
          const float shrink = mm == m ? 1.0f : __builtin_amdgcn_exp2f(m - mm);
          const float both = shrink * scale_of_exp(e - e_new);
          l *= shrink;
#pragma unroll
          for (int j = 0; j < D / 32; ++j)
#pragma unroll
            for (int i = 0; i < 16; ++i) o[j][i] *= both;
          m = mm;
          e = e_new;
        }
        const float ms = m == -__builtin_inff() ? 0.0f : m;
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) {
          f16x8a pr[PT][2];
#pragma unroll
          for (int a = 0; a < 4; ++a) {
            const f32x4a s4 = *reinterpret_cast<const f32x4a*>(&S.vs[buf][kt * 32 + a * 8 + h * 4]);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              float x = __builtin_amdgcn_exp2f(__builtin_fmaf(t[kt][4 * a + r], unit, -ms));
              float c = x * s4[r];
              if (!open && !((uint32_t)(see >> (32 * kt)) >> (8 * a + r) & 1)) x = c = 0.0f;
              l += x;
              if constexpr (PT == 2) asm("" : "+v"(c));
              const int s = a >> 1, i = 4 * (a & 1) + r;
              pr[0][s][i] = (_Float16)c;
              if constexpr (PT == 2) pr[1][s][i] = (_Float16)(c - (float)pr[0][s][i]);
            }
          }
#pragma unroll
          for (int j = 0; j < D / 32; ++j) {
            const int row = j * 32 + l32;
#pragma unroll
            for (int s = 0; s < 2; ++s) {
              const int run = (kt * 2 + s) * 2 + h;
              const f16x8a vf =
                  *reinterpret_cast<const f16x8a*>(&S.v[buf][row * (MXK_TILE / 2) + ((run ^ ((row >> 1) & 7)) * 4)]);
#pragma unroll
              for (int n = 0; n < PT; ++n) o[j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf, pr[n][s], o[j], 0, 0, 0);
            }
          }
        }
      }
      if (more) put(buf ^ 1);
      __syncthreads();
    }

    // a lane has its row's elements 4c .. 4c+3 for every c with bit 2 of c equal to h
    l += __shfl_xor(l, 32);
    if (row_ok) {
      const float down = scale_of_exp(e - 1), inv = l == 0.0f ? 0.0f : 1.0f / l;
      const int64_t slot = ((int64_t)share * 2 + (p.k == 0 ? 1 : 0)) * (32 * NW) + wave * 32 + l32;
      T* dst = reinterpret_cast<T*>(A.out) + ((int64_t)(w.first + tok) * A.Hq + head) * D;
#pragma unroll
      for (int a = 0; a < D / 32; ++a)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          float x[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int row = j * (D / 4) + 8 * a + r;
            x[j] = o[row / 32][(row % 32 / 8) * 4 + row % 4] * down;
          }
          const int d = 4 * (8 * a + 4 * h + r);
          if (whole) {
            T y[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) y[j] = out_cvt<T>(x[j] * inv);
            __builtin_memcpy(dst + d, y, sizeof(y));
          } else {
            __builtin_memcpy(A.part_o + slot * D + d, x, sizeof(x));
          }
        }
      if (!whole && h == 0) A.part_s[slot] = make_float2(m, l);
    }
    at += k1 - p.k;
    if (at >= to) break;
    next_tile(A, L, w, p);
  }
}

// A tile whose first block lies in share s and whose last one does not: its
// parts are share s's second one and the first ones of the shares after it, up to the one
// with its last block.  A wave a row.
template <typename T, int D>
__global__ __launch_bounds__(64) void k_attend_join(AttendArgs A, int shares, int rows) {
  constexpr int E = D / 64;
  const Line L = make_line(A);
  const int64_t total = line_length(A, L);
  const int64_t per = line_share(total, shares);
  const int s = blockIdx.x, r = blockIdx.y;
  const int64_t from = s * per, to = min(total, from + per);
  if (from >= to || to == total) return;
  SeqWork w;
  const Place p = line_place(A, L, to - 1, w);
  const int64_t begin = to - 1 - p.k, end = begin + p.blocks;
  if (end <= to || begin < from) return;
  int tok, head;
  if (!tile_row(A, w, p, r, tok, head)) return;
  const int last = (int)((end - 1) / per);
  const int lane = threadIdx.x;
  float m = -__builtin_inff();
  for (int i = s + lane; i <= last; i += 64) m = fmaxf(m, A.part_s[((int64_t)i * 2 + (i == s)) * rows + r].x);
#pragma unroll
  for (int i = 1; i < 64; i <<= 1) m = fmaxf(m, __shfl_xor(m, i));
  float sum = 0.0f, acc[E];
#pragma unroll
  for (int j = 0; j < E; ++j) acc[j] = 0.0f;
  for (int i = s; i <= last; ++i) {
    const int64_t slot = ((int64_t)i * 2 + (i == s)) * rows + r;
    const float2 ms = A.part_s[slot];
    const float f = ms.x == m ? 1.0f : __builtin_amdgcn_exp2f(ms.x - m);
    sum += f * ms.y;
    float v[E];
    __builtin_memcpy(v, A.part_o + slot * D + lane * E, sizeof(v));
#pragma unroll
    for (int j = 0; j < E; ++j) acc[j] = __builtin_fmaf(f, v[j], acc[j]);
  }
  const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
  T e[E];
#pragma unroll
  for (int j = 0; j < E; ++j) e[j] = out_cvt<T>(acc[j] * inv);
  __builtin_memcpy(reinterpret_cast<T*>(A.out) + ((int64_t)(w.first + tok) * A.Hq + head) * D + lane * E, e, sizeof(e));
}

// ---------------------------------------------------------------- host
struct AttendPlan {
  int rows, keys, TT, GC, chunks, shares;
  bool cut;  // a tile may be cut
};

static AttendPlan plan_attend(int64_t T, int64_t B, int64_t width, int page, int H, int G, int D) {
  AttendPlan a;
  // rows of a sequence and key head, on average
  const double each = B > 0 ? (double)T * G / (double)std::min(B, T) : 0.0;
  a.rows = each <= 32 ? 16 : each <= 128 || D == 256 ? 128 : 256;
  a.keys = a.rows == 16 ? 128 : 256;
  a.GC = std::min(G, a.rows);
  a.chunks = (int)ceil_div(G, a.GC);
  a.TT = 1;
  while (a.TT * 2 * a.GC <= a.rows) a.TT *= 2;
  // no more shares than blocks there can be
  const double tiles = ((double)T / a.TT + (double)std::min(B, T)) * a.chunks * H;
  const double blocks = std::ceil((double)width * page / a.keys);
  a.cut = blocks > 1 && B > 0;
  const double most = (a.rows == 256 || D == 256 ? 1.0 : 2.0) * num_cus();  // workgroups that run at once
  a.shares = (int)std::max(1.0, std::min(most, tiles * std::max(1.0, blocks)));
  return a;
}

template <typename T, int D, int QT, int PT>
static int launch_attend(const AttendArgs& A, const AttendPlan& a, hipStream_t st) {
  constexpr int QH = sizeof(T) == 4 ? 2 : 1;  // float16 terms of a query
  if (a.rows == 16) {
    hipLaunchKernelGGL((k_attend<T, D, QT, PT>), dim3(a.shares), dim3(256), 0, st, A, a.shares);
  } else if (a.rows == 128) {
    hipLaunchKernelGGL((k_attend_tile<T, D, QH, PT, 4>), dim3(a.shares), dim3(256), 0, st, A, a.shares);
  } else {
    if constexpr (D < 256)
      hipLaunchKernelGGL((k_attend_tile<T, D, QH, PT, 8>), dim3(a.shares), dim3(512), 0, st, A, a.shares);
  }
  if (a.cut && a.shares > 1)
    hipLaunchKernelGGL((k_attend_join<T, D>), dim3(a.shares - 1, a.rows), dim3(64), 0, st, A, a.shares, a.rows);
  return check_launch("kv_attend");
}

template <typename T, int QT, int PT>
static int launch_attend_d(int D, const AttendArgs& A, const AttendPlan& a, hipStream_t st) {
  if (D == 64) return launch_attend<T, 64, QT, PT>(A, a, st);
  if (D == 128) return launch_attend<T, 128, QT, PT>(A, a, st);
  return launch_attend<T, 256, QT, PT>(A, a, st);
}

}  // namespace mxk

using namespace mxk;

extern "C" {

size_t mxk_kv_pages_attend_workspace(int64_t tokens, int64_t B, int64_t width, int page, int heads, int q_heads,
                                     int D) {
  if (tokens <= 0 || B <= 0 || width < 0 || heads < 1 || q_heads < heads || q_heads % heads || !kv_page_ok(page))
    return 0;
  const AttendPlan a = plan_attend(tokens, B, width, page, heads, q_heads / heads, D);
  return a.cut ? (size_t)a.shares * 2 * a.rows * ((size_t)D * 4 + 8) : 0;
}

int mxk_kv_pages_attend(const void* q, int q_type, int64_t q_token, int64_t q_head, int q_heads, const void* codes,
                        const float* scales, int64_t pages, int page, int heads, int D, const int32_t* table,
                        const int32_t* lengths, const int32_t* offsets, int64_t B, int64_t width, int64_t tokens,
                        const void* mask, int words, float scale, void* out, void* workspace,
                        size_t workspace_nbytes, void* stream) {
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (pages < 0 || pages >= ((int64_t)1 << 31) || heads < 1 || heads > 1024 || !kv_page_ok(page))
    return fail(MXK_EINVAL, "kv_attend: pages below 2^31 of a power of two of positions from 16 on, 1 to 1024 heads");
  if (D != 64 && D != 128 && D != 256) return fail(MXK_EUNSUPPORTED, "kv_attend: heads of 64, 128 or 256 elements");
  if (q_heads < heads || q_heads % heads || q_heads > 65536)
    return fail(MXK_EINVAL, "kv_attend: query heads are a multiple of the cache's, at most 65536");
  if (B < 0 || width < 0 || tokens < 0 || B >= ((int64_t)1 << 24) || width >= ((int64_t)1 << 31) ||
      tokens >= ((int64_t)1 << 31) - 64)
    return fail(MXK_EINVAL, "kv_attend: bad sizes (sequences below 2^24, pages of one and tokens below 2^31)");
  if (!(scale > 0.0f) || !std::isfinite(scale)) return fail(MXK_EINVAL, "kv_attend: the scale is a positive number");
  if (q_type != MXK_IN_F32 && q_type != MXK_IN_F16 && q_type != MXK_IN_BF16)
    return fail(MXK_EINVAL, "kv_attend: unknown q_type");
  if (mask && (words < 1 || words > (1 << 20))) return fail(MXK_EINVAL, "kv_attend: 1 to 2^20 words of mask a token");
  if (tokens == 0) return MXK_OK;
  if (!q || !out || !offsets || (B > 0 && (!lengths || (width > 0 && !table))))
    return fail(MXK_EINVAL, "kv_attend: null pointer");
  if (pages == 0) return fail(MXK_EINVAL, "kv_attend: a pool without pages");
  if (!codes || !scales) return fail(MXK_EINVAL, "kv_attend: null pointer");
  if (!aligned16(codes) || !aligned16(scales))
    return fail(MXK_EINVAL, "kv_attend: codes and scales start on 16 bytes");
  const int G = q_heads / heads;
  const AttendPlan a = plan_attend(tokens, B, width, page, heads, G, D);
  const size_t part = (size_t)a.shares * 2 * a.rows;
  if (a.cut && a.shares > 1 && (!workspace || workspace_nbytes < part * ((size_t)D * 4 + 8) || !aligned16(workspace)))
    return fail(MXK_EINVAL, "kv_attend: workspace too small (mxk_kv_pages_attend_workspace) or not on 16 bytes");
  AttendArgs A;
  A.q = q;
  A.q_token = q_token;
  A.q_head = q_head;
  A.pool = KvPool{const_cast<int8_t*>(reinterpret_cast<const int8_t*>(codes)), const_cast<float*>(scales),
                  (uint32_t)pages, heads, log2_of(page)};
  A.batch = KvBatch{table, lengths, offsets, (int)B, (int)width, (int)tokens};
  A.mask = reinterpret_cast<const uint64_t*>(mask);
  A.words = words;
  A.scale = scale * 1.4426950408889634f;
  A.Hq = q_heads;
  A.G = G;
  A.keys = a.keys;
  A.TT = a.TT;
  A.GC = a.GC;
  A.chunks = a.chunks;
  A.out = out;
  A.part_o = reinterpret_cast<float*>(workspace);
  A.part_s = workspace ? reinterpret_cast<float2*>(A.part_o + part * D) : nullptr;
  if (q_type == MXK_IN_F32) return launch_attend_d<float, 3, 2>(D, A, a, st);
  if (q_type == MXK_IN_F16) return launch_attend_d<__half, 2, 1>(D, A, a, st);
  return launch_attend_d<hip_bfloat16, 2, 1>(D, A, a, st);
}

}  // extern "C"
