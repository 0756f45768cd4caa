// Attention of new tokens over a paged 8-bit key-value cache, for gfx950.
//
//   o = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale <q, k_j> - m)
//
// over the keys j that a token sees: those held before the call, and of the
// call's own tokens the ones up to itself, or those whose bit its mask has.
// One pass over the keys with a running maximum m.  Few rows a sequence and
// head take tiles of 16 rows (k_attend), which are bound by the cache's bytes;
// more take tiles of up to 256 (k_attend_tile), bound by their arithmetic.
//
// Tiles of 16 rows, keys.  The codes go to the int8 MFMA as they are stored.  A query row is
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
// exponent of the largest scale that the row has seen so far, is at most 2^15, and keeps 11 bits (22
// for float32 and float16 queries: a second term) down to 2^-24 of the largest.
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
  int keys;     // of a block: 128 or 256
  int TT, GC, chunks;  // a tile: TT tokens (a power of two, at most keys) of GC heads, chunks of them over G
  int cap, most;       // positions of the table (below 2^31 - 2^16); blocks of a tile at most, at least one
  int rows, shares;    // of a tile; the line's
  void* out;
  // of tiles that are cut, null where none can be: sums [shares][2][rows][D] of their own maximum, the maximum and
  // weight of each row, and the tile that a share leaves to the shares after it
  float* part_o;
  float2* part_s;
  struct PartTile* part_t;
  // of tiles of many rows, [shares]: bit i (31: any from there on) of the share's tile i whose value scales or queries are
  // too far apart for a common largest one
  uint32_t* apart;
};

struct PartTile {
  int first, n, h, x;  // of the sequence's new tokens; key head, tile
  int last;            // share with the tile's last block, -1: no tile
  int pad[3];
};

// ---------------------------------------------------------------- the line of blocks
// All places on the line are below 2^31 (the host has seen to it).

// sum of floor(i / 2^s) over i < x, modulo 2^32: differences of two are exact
__device__ __forceinline__ uint32_t sum_floor(uint32_t x, int s) {
  const uint32_t q = x >> s;
  const uint32_t half = q & 1 ? q * ((q - 1) >> 1) : (q >> 1) * (q - 1);
  return (half << s) + q * (x - (q << s));
}

struct Line {
  int ts, rs;  // log2 of TT and of keys / TT
};

// A sequence on the line: per key head, its tiles' blocks one after the other
struct SeqWork {
  int first, n, ctx;  // new tokens, keys held
  int a;              // causal: token tile t has floor((a + t) / 2^rs) blocks, at most AttendArgs::most
  int full;           // causal: the first token tile that has that many
  int blocks;         // masked: of every tile
  int tiles;          // token tiles
  uint32_t head;      // blocks of one key head
};

__device__ __forceinline__ int tile_blocks(const AttendArgs& A, const Line& L, const SeqWork& w, int t) {
  return A.mask ? w.blocks : t >= w.full ? A.most : (w.a + t) >> L.rs;
}

// Blocks of a key head's token tiles below t
__device__ __forceinline__ uint32_t blocks_below(const AttendArgs& A, const Line& L, const SeqWork& w, int t) {
  if (A.mask) return (uint32_t)A.chunks * ((uint32_t)t * (uint32_t)w.blocks);
  const int some = min(t, w.full);
  return (uint32_t)A.chunks * (sum_floor((uint32_t)(w.a + some), L.rs) - sum_floor((uint32_t)w.a, L.rs) +
                               (uint32_t)(t - some) * (uint32_t)A.most);
}

__device__ __forceinline__ SeqWork seq_work(const AttendArgs& A, const Line& L, int b) {
  SeqWork w;
  const int held = A.batch.lengths[b];
  w.first = kv_offset(A.batch, b);
  w.n = kv_count(A.batch, b);
  w.ctx = min(max(held, 0), A.cap);
  w.tiles = (w.n + A.TT - 1) >> L.ts;
  w.a = (w.ctx + A.TT + A.keys - 1) >> L.ts;
  w.full = max(0, (int)(((int64_t)A.most << L.rs) - w.a));
  w.blocks = min((int)(((int64_t)w.ctx + w.n + A.keys - 1) >> (L.ts + L.rs)), A.most);
  w.head = blocks_below(A, L, w, w.tiles);
  return w;
}

__device__ __forceinline__ Line make_line(const AttendArgs& A) {
  Line L;
  L.ts = 31 - __builtin_clz(A.TT);
  L.rs = 31 - __builtin_clz(A.keys) - L.ts;
  return L;
}

// A place on the line: the tile it lies in and the block of the tile
struct Place {
  int b, h, x;  // sequence, key head, tile (token tile * chunks + chunk)
  int k;        // block within the tile
  int blocks;   // of the tile
};

__device__ __forceinline__ uint32_t wave_scan(uint32_t v) {  // inclusive
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int i = 1; i < 64; i <<= 1) {
    const uint32_t o = __shfl_up(v, i);
    if (lane >= i) v += o;
  }
  return v;
}
__device__ __forceinline__ uint32_t lane_of(uint32_t v, int lane) { return __builtin_amdgcn_readlane(v, lane); }
__device__ __forceinline__ int lane_of(int v, int lane) { return (int)__builtin_amdgcn_readlane((uint32_t)v, lane); }

// Share `share` of the line, [from, to), and the place it begins at.  Found by
// every wave for itself, which holds a sequence a lane: for up to 64 of them one round of loads.
// More are first summed by the workgroup's THREADS threads, a run of sequences each (1024 sequences of 256 keys, one head: 30 us,
// and 39 where each wave walks them 64 at a time; 4096 of 64: 57 and 106).
// false: an empty share.
template <int THREADS>
__device__ __forceinline__ bool line_share(const AttendArgs& A, const Line& L, int share, uint32_t& from, uint32_t& to,
                                           uint32_t& per, SeqWork& w, Place& p) {
  const int lane = threadIdx.x & 63, B = A.batch.B;
  __shared__ uint32_t sums[THREADS];
  if (B == 0) return false;
  uint32_t total, upto4 = 0, four = 0;
  const int run = (B + THREADS - 1) / THREADS;
  SeqWork mine;
  uint32_t own = 0, upto = 0;
  if (B <= 64) {
    mine = seq_work(A, L, min(lane, B - 1));
    own = lane < B ? mine.head * (uint32_t)A.pool.H : 0;
    upto = wave_scan(own);
    total = lane_of(upto, 63);
  } else {
    uint32_t sum = 0;
    const int first = (int)threadIdx.x * run, end = min(first + run, B);
#pragma unroll 4
    for (int b = first; b < end; ++b) sum += seq_work(A, L, b).head * (uint32_t)A.pool.H;
    sums[threadIdx.x] = sum;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < THREADS / 64; ++i) four += sums[lane * (THREADS / 64) + i];
    upto4 = wave_scan(four);
    total = lane_of(upto4, 63);
  }
  per = (total + (uint32_t)A.shares - 1) / (uint32_t)A.shares;
  from = (uint32_t)share * per;
  to = min(total, from + per);
  if (from >= to) return false;
  uint32_t at = from;
  int b0 = 0;
  if (B > 64) {
    const int l = __builtin_ctzll(__ballot(upto4 > at));
    at -= lane_of(upto4 - four, l);
    int i = l * (THREADS / 64);
    while (i < THREADS - 1 && at >= sums[i]) at -= sums[i++];
    b0 = __builtin_amdgcn_readfirstlane(i) * run;
    at = __builtin_amdgcn_readfirstlane(at);
    if (b0 >= B) return false;  // of sums that have wrapped, as below
    mine = seq_work(A, L, min(b0 + lane, B - 1));
    own = b0 + lane < B ? mine.head * (uint32_t)A.pool.H : 0;
    upto = wave_scan(own);
  }
  while (at >= lane_of(upto, 63)) {
    at -= lane_of(upto, 63);
    b0 += 64;
    if (b0 >= B) return false;  // offsets that do not ascend, and so many tokens that the sum has wrapped
    mine = seq_work(A, L, min(b0 + lane, B - 1));
    own = b0 + lane < B ? mine.head * (uint32_t)A.pool.H : 0;
    upto = wave_scan(own);
  }
  const int l = __builtin_ctzll(__ballot(upto > at));
  at -= lane_of(upto - own, l);
  w.first = lane_of(mine.first, l);
  w.n = lane_of(mine.n, l);
  w.ctx = lane_of(mine.ctx, l);
  w.a = lane_of(mine.a, l);
  w.full = lane_of(mine.full, l);
  w.blocks = lane_of(mine.blocks, l);
  w.tiles = lane_of(mine.tiles, l);
  w.head = lane_of(mine.head, l);
  p.b = b0 + l;
  p.h = (int)__builtin_amdgcn_readfirstlane(at / w.head);
  at -= (uint32_t)p.h * w.head;
  int lo = 0, hi = w.tiles - 1;  // the last token tile that begins at or before `at`
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (blocks_below(A, L, w, mid) <= at) lo = mid;
    else hi = mid - 1;
  }
  at -= blocks_below(A, L, w, lo);
  p.blocks = tile_blocks(A, L, w, lo);
  int c = 0;
  while (at >= (uint32_t)p.blocks) ++c, at -= (uint32_t)p.blocks;  // below chunks
  p.x = lo * A.chunks + c;
  p.k = (int)at;
  return true;
}

// The next tile on the line; false: none, which ascending offsets do not come to
__device__ __forceinline__ bool next_tile(const AttendArgs& A, const Line& L, SeqWork& w, Place& p) {
  p.k = 0;
  if (++p.x == w.tiles * A.chunks) {
    p.x = 0;
    if (++p.h == A.pool.H) {
      p.h = 0;
      do {
        if (++p.b >= A.batch.B) return false;
        w = seq_work(A, L, p.b);
      } while (w.head == 0);
    }
  }
  p.blocks = tile_blocks(A, L, w, p.x / A.chunks);
  return true;
}

// The workgroup's share.  Neighbours on the line may read the same keys: they go to one XCD.  Tiles of 16 rows, 16 trees of 64
// tokens on 4000 keys of 8 heads: 65 us, 91 in the order of the blocks.
__device__ __forceinline__ int share_of_block(const AttendArgs& A) {
  return A.shares % 8 == 0 ? (blockIdx.x & 7) * (A.shares >> 3) + (blockIdx.x >> 3) : blockIdx.x;
}

// The tile that a share ends in and does not end, if it begins there too
__device__ __forceinline__ void leave_part(const AttendArgs& A, int share, bool some, uint32_t end, uint32_t per,
                                           const SeqWork& w, const Place& p) {
  if (!A.part_t || threadIdx.x != 0) return;
  PartTile t = {};
  t.last = -1;
  if (some) t = PartTile{w.first, w.n, p.h, p.x, min((int)((end - 1) / per), A.shares - 1), {0, 0, 0}};
  A.part_t[share] = t;
}

// First position past the keys that a tile's last token may see
__device__ __forceinline__ int tile_end(const AttendArgs& A, const SeqWork& w, const Place& p) {
  const int new_ones = A.mask ? w.n : min(w.n, (p.x / A.chunks + 1) * A.TT);
  return w.ctx + min(A.cap - w.ctx, new_ones);
}

// Pages of a tile's runs of 16 keys, 64 runs a lane each, a batch ahead of its use
struct RunPages {
  int cur, next;
  __device__ __forceinline__ int load(const AttendArgs& A, int b, int run) const {
    return kv_page(A.batch, A.pool, b, ((int64_t)run << 4) >> A.pool.shift);
  }
  __device__ __forceinline__ void start(const AttendArgs& A, int b, int run) {
    cur = load(A, b, run + (int)(threadIdx.x & 63));
    next = load(A, b, run + 64 + (int)(threadIdx.x & 63));
  }
  __device__ __forceinline__ void advance(const AttendArgs& A, int b, int run) {  // run: of the batch after the next
    cur = next;
    next = load(A, b, run + (int)(threadIdx.x & 63));
  }
};

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
__device__ __forceinline__ void load_keys(const KvPool& p, int h, int key, int page0, int page1, int lane, Keys32<D>& s) {
  const int l = lane & 15, g = lane >> 4;
  const int64_t values = (int64_t)p.H << p.shift;
#pragma unroll
  for (int a = 0; a < 2; ++a) {
    const int page = a ? page1 : page0;
    s.ok[a] = page >= 0;
    // without a page: some row of the pool, whose keys nobody sees
    const int64_t row = kv_row(p, max(page, 0), 0, h, (key + 16 * a) & ((1 << p.shift) - 1));
    const int8_t* kc = p.codes + row * D;
#pragma unroll
    for (int i = 0; i < D / 64; ++i)
      s.k[a][i] = *reinterpret_cast<const i32x4a*>(kc + (uint32_t)(l * D + i * 64 + g * 16));
    const int8_t* vc = p.codes + (row + values) * D;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      __builtin_memcpy(s.v[4 * a + j], __builtin_assume_aligned(vc + (uint32_t)((g * 4 + j) * D + l * (D / 16)), D / 16),
                       D / 16);
    s.ks[a] = *reinterpret_cast<const f32x4a*>(p.scales + row + g * 4);
    s.vs[a] = *reinterpret_cast<const f32x4a*>(p.scales + row + values + g * 4);
  }
}

__device__ __forceinline__ float scale_of_exp(int e) {  // 2^e, zero below the normal range
  return e < -126 ? 0.0f : __uint_as_float((uint32_t)(min(e, 127) + 127) << 23);
}

// Exponent of a scale, -127 of one that is not finite
__device__ __forceinline__ int scale_exp(float s) {
  const uint32_t b = mag_bits(s);
  return (int)((b < 0x7F800000u ? b : 0u) >> 23) - 127;
}
__device__ __forceinline__ int wave_max(int v) {
#pragma unroll
  for (int i = 1; i < 64; i <<= 1) v = max(v, __shfl_xor(v, i));
  return v;
}

// One tile over blocks [k0, k1): four waves, 32 keys of a block each
template <typename T, int D, int QT, int PT>
struct TileState {
  f32x4a o[D / 16];  // row lane%16, elements (g*4 + r) * (D/16) + j in o[j][r], times 2^(1 - e)
  float m, l;        // maximum (log2 units), the lane's own sum
  int e;             // exponent of the largest value scale that the row sees
};

template <typename T, int D, int QT, int PT>
__device__ __forceinline__ void step32(const AttendArgs& A, const i32x4a (&q)[QT][D / 64], float unit, Keys32<D>& s,
                                       int key, int ctx, int end, int tok, const uint64_t* __restrict__ bits,
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
      const int at = key + 16 * (i >> 2) + 4 * g + (i & 3), j = at - ctx;
      bool see = at < end && s.ok[i >> 2];
      if (see && j >= 0) see = bits ? (j >> 6) < A.words && (bits[j >> 6] >> (j & 63) & 1) : j <= tok;
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
    // of the row's own keys: a scale that only other rows see would take its bits from the row's
    int e = max(eb, st.e);
    e = max(e, __shfl_xor(e, 16));
    e = max(e, __shfl_xor(e, 32));
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
__device__ __forceinline__ void zero_padding(const AttendArgs& A) {
  const int B = A.batch.B;
  const int64_t lo = B ? kv_offset(A.batch, 0) : 0, hi = B ? kv_offset(A.batch, B) : 0;
  const int64_t row = (int64_t)A.Hq * D, n = (lo + (A.batch.T - hi)) * row;
  T* out = reinterpret_cast<T*>(A.out);
  for (int64_t i = (int64_t)blockIdx.x * THREADS + threadIdx.x; i < n; i += (int64_t)A.shares * THREADS)
    out[i < lo * row ? i : i - lo * row + hi * row] = out_cvt<T>(0.0f);
}

// Tiles of 16 rows, four waves that take 32 keys of each block of 128 and are
// joined in LDS; two workgroups a CU.  Bound by memory: 64 sequences of up to
// 8192 keys, 8 heads of 128 with 4 of queries each, bfloat16, 598 MB of cache:
// 126 us, 4.75 TB/s of the 5.0 that a large copy reaches; 2 sequences of up to 130003, 447 MB:
// 84 us, 5.3 TB/s.  A wave asks for the next block's keys and values before it
// computes the present one's; pages come a batch of 32 blocks ahead.
template <typename T, int D, int QT, int PT>
__global__ __launch_bounds__(256, D == 256 ? 1 : 2) void k_attend(AttendArgs A) {
  constexpr int LD = D + 4;
  __shared__ float so[4][16][LD];
  __shared__ float sm[4][16], sl[4][16];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int l16 = lane & 15, g = lane >> 4, share = share_of_block(A);
  const Line L = make_line(A);
  zero_padding<T, D, 256>(A);
  uint32_t from, to, per;
  SeqWork w;
  Place p;
  if (!line_share<256>(A, L, share, from, to, per, w, p)) {
    leave_part(A, share, false, 0, 1, w, p);
    return;
  }
  uint32_t at = from;
  // a wave's keys: 32 of each block, so its runs of 16 are blocks * 8 + wave * 2 + 0, 1; lane i holds run i & 1 of
  // the block i / 2 after the first
  auto pages_of = [&](int block) {
    return kv_page(A.batch, A.pool, p.b, ((int64_t)(block + (lane >> 1)) * 128 + wave * 32 + (lane & 1) * 16) >> A.pool.shift);
  };
  int k1, end, stop, pages, ahead;  // of the tile at hand: blocks up to k1, keys up to end and of these blocks
  Keys32<D> cur;
  auto find = [&]() {
    k1 = (int)min((uint32_t)p.blocks, (uint32_t)p.k + (to - at));
    end = tile_end(A, w, p);
    stop = (int)min((int64_t)end, (int64_t)k1 * 128);
    pages = pages_of(p.k);
    ahead = pages_of(p.k + 32);
  };
  auto begin = [&]() {
    const int key = p.k * 128 + wave * 32;
    if (key < stop) load_keys<D>(A.pool, p.h, key, lane_of(pages, 0), lane_of(pages, 1), lane, cur);
  };
  find();
  begin();
  while (true) {
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
    TileState<T, D, QT, PT> st;
#pragma unroll
    for (int j = 0; j < D / 16; ++j) st.o[j] = f32x4a{0, 0, 0, 0};
    st.m = -__builtin_inff();
    st.l = 0.0f;
    st.e = -100;  // smaller scales lose bits
    int key = p.k * 128 + wave * 32;
    if (key < stop) {
      Keys32<D> nxt;
      for (int i = 1;; ++i) {
        const int next = key + 128;
        const bool more = next < stop;
        if (more) {
          if ((i & 31) == 0) {
            pages = ahead;
            ahead = pages_of(p.k + i + 32);
          }
          load_keys<D>(A.pool, p.h, next, lane_of(pages, 2 * (i & 31)), lane_of(pages, 2 * (i & 31) + 1), lane, nxt);
        }
        step32<T, D, QT, PT>(A, q, unit, cur, key, w.ctx, end, tok, bits, lane, st);
        if (!more) break;
        cur = nxt;
        key = next;
      }
    }
    // the next tile's pages are on their way while this one's sums go to LDS, its first keys while they are joined
    // (64 sequences of 2000 keys: 49 us, 50.5 without)
    const SeqWork w0 = w;
    const Place p0 = p;
    const int done = k1;
    at += (uint32_t)(k1 - p.k);
    const bool again = at < to && next_tile(A, L, w, p);
    if (again) find();
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
    if (again) begin();
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
      if (tile_row(A, w0, p0, r, rt, rh)) {
        if (whole) {
          T* dst = reinterpret_cast<T*>(A.out) + ((int64_t)(w0.first + rt) * A.Hq + rh) * D + d0;
          const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
          T e[D / 16];
#pragma unroll
          for (int j = 0; j < D / 16; ++j) e[j] = out_cvt<T>(acc[j] * inv);
          __builtin_memcpy(dst, e, sizeof(e));
        } else {
          const int64_t slot = ((int64_t)share * 2 + (p0.k == 0 ? 1 : 0)) * 16 + r;
          __builtin_memcpy(A.part_o + slot * D + d0, acc, sizeof(acc));
          if ((threadIdx.x & 15) == 0) A.part_s[slot] = make_float2(m, sum);
        }
      }
    }
    if (!again) {
      leave_part(A, share, p0.k == 0 && done < p0.blocks, at + (uint32_t)(p0.blocks - done), per, w0, p0);
      break;
    }
    __syncthreads();
  }
}

// ---------------------------------------------------------------- tiles of many rows
// NW waves of 32 rows each (4 or 8) share the keys, 64 at a time: their codes are
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
//
// Roundings: a query is one float16 term (two for float32), which holds
// float16 and bfloat16 queries whole as far as the tile's largest element allows (a row of less than 2^-8 of
// it is computed by its own, k_attend_tile);
// probabilities times the values' scales are one float16 term (two for
// float32), 2^-11 of a weight: half the matrix work of two, against results of 8 and 11 bits (the float16 cases' error
// grows from 2.1e-4, the result's own rounding, to 3.0e-4).  For bfloat16 the probability and the scale go to
// float16 before their product (three roundings of 2^-11 against the result's 2^-8), the row's weight is the float32 sum of
// these float16 probabilities, whose roundings so are in both parts of the quotient, and a
// scale keeps 11 bits down to 2^-14 of the largest one so far, one less for each power of two
// below; the other forms' do down to 2^-24.
//
// Bound by issue: matrix and vector instructions of a SIMD's two waves
// hardly overlap (matrix 35 % of the cycles, vector 45 %).  2 sequences with up to 2000 new
// tokens behind up to 6000 keys, 8 heads of 128 with 4 of queries each, bfloat16: 281 GFLOP in
// 355 us with the join, 0.79 PFLOP/s of the 1.20 that a large bfloat16 product reaches.
//
// Registers: the sums of a wave's rows (D / 2), the queries (D / 4, float32 twice) and a step's keys on their way fill 256.  Heads
// of 128 spill two, outside the loop over the steps; float32 and heads of 256 take accumulation registers too, so that a
// SIMD has one wave, which nothing runs beside; both together also spill 16, some in the loop.

// A lane's elements i*16 + h*8 + 0..7 of a query row (null: zeros), and the exponent of the row's largest; rows below
// 2^-100 count as zeros, and so do, at first, those with a NaN or an infinity.
template <typename T, int D>
struct QueryHalf {
  T x[D / 16][8];
  int e;
  bool some, nan;
};

template <typename T, int D>
__device__ __forceinline__ void query_load(const T* __restrict__ row, int h, QueryHalf<T, D>& q) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < D / 16; ++i) {
    __builtin_memset(q.x[i], 0, sizeof(q.x[i]));
    if (row) __builtin_memcpy(q.x[i], row + i * 16 + h * 8, sizeof(q.x[i]));
#pragma unroll
    for (int j = 0; j < 8; ++j) m = max(m, mag_bits(ElemT<T>::cvt(q.x[i][j])));
  }
  m = max(m, (uint32_t)__shfl_xor((int)m, 32));
  q.some = m >= 0x0D800000u && m < 0x7F800000u;
  q.nan = m >= 0x7F800000u;
  q.e = q.some ? (int)(m >> 23) - 127 : -100;
}

// The row times 2^(14 - e), e the exponent of the largest element of the workgroup's rows: float16 has 11 bits of it (22
// in two terms) down to 2^-28 of that element.
template <typename T, int D, int QT>
__device__ __forceinline__ void query_terms16(const QueryHalf<T, D>& q, int e, f16x8a (&term)[QT][D / 16]) {
  const float up = q.some ? scale_of_exp(14 - e) : 0.0f;
#pragma unroll
  for (int i = 0; i < D / 16; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      float v = q.some ? ElemT<T>::cvt(q.x[i][j]) * up : 0.0f;
      if constexpr (QT == 2) asm("" : "+v"(v));  // one rounding for both terms, as for the probabilities
      term[0][i][j] = (_Float16)v;
      if constexpr (QT == 2) term[1][i][j] = (_Float16)(v - (float)term[0][i][j]);
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

// Keys of a step: at heads of 256 half as many, so that two steps fit LDS and the registers
template <int D>
constexpr int tile_keys() { return D == 256 ? 32 : 64; }

template <int D, int NW>
struct TileLds {
  static constexpr int K = tile_keys<D>();
  u32x4 k[2][K * D / 8];  // [key][D] float16, pieces of 8 swizzled
  u32x4 v[2][K * D / 8];  // [row][K keys] float16, pieces of 8 swizzled
  float ks[2][K];    // times the queries' unit (own: but for the row's exponent)
  float vs[2][K];    // times 2^(10 - e); coarse: float16, times 2^-e, in the order of a lane's weights; own: as they are
  int e[2];
  int top[NW], low[NW];  // exponents of the waves' largest query elements: of all rows, the smallest of a row's own
  uint32_t ok[2];  // bits of the step's runs of 16 keys that have a page; bit 31: a value's scale is not finite
};

// Swizzle of the 16-byte pieces of a value row (K * 2 bytes)
template <int D>
__device__ __forceinline__ int value_swizzle(int row) {
  return D == 256 ? (row >> 2) & 3 : (row >> 1) & 7;
}

// What a thread fetches of a step, on its way from memory to LDS
template <int D, int NW>
struct Fetched {
  static constexpr int PIECES = tile_keys<D>() * D / 16, N = PIECES / (64 * NW) > 0 ? PIECES / (64 * NW) : 1;
  u32x4 k[N];        // 16 elements of a key
  uint32_t v[N][4];  // four elements of four keys
  float scale;       // wave 0: of a key, wave 1: of a value
  int page;          // of that key, waves 0 and 1
};

template <int D, int NW>
__device__ __forceinline__ void tile_fetch(const AttendArgs& A, int h, int key, int end, int pages, int first_run,
                                           Fetched<D, NW>& f) {
  using F = Fetched<D, NW>;
  const uint32_t tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int in = (1 << A.pool.shift) - 1;
  const int64_t values = (int64_t)A.pool.H << A.pool.shift;
#pragma unroll
  for (int i = 0; i < F::N; ++i) {
    // D pieces are 16 keys: a wave's lie in one run, with one page
    const uint32_t first = (wave + i * NW) * 64, run = first / D, piece = (first + lane) % D;
    if (first >= F::PIECES) break;
    const int page = lane_of(pages, first_run + (int)run);
    const int64_t row = kv_row(A.pool, max(page, 0), 0, h, (key + (int)run * 16) & in);
    const int8_t* k = A.pool.codes + row * D;
    const int8_t* v = k + values * D;
    f.k[i] = *reinterpret_cast<const u32x4*>(k + (uint32_t)(piece * 16));
    const uint32_t four = piece / (D / 4), c = piece % (D / 4);
#pragma unroll
    for (int r = 0; r < 4; ++r)
      f.v[i][r] = *reinterpret_cast<const uint32_t*>(v + (uint32_t)((four * 4 + r) * D + c * 4));
  }
  if (wave < 2) {
    const int l = (int)lane & (tile_keys<D>() - 1), at = key + l;
    const int there = __shfl(pages, first_run + (l >> 4));  // with all lanes: they hold each other's pages
    const int page = at < end ? there : -1;
    f.page = page;
    f.scale = 0.0f;
    if (page >= 0) f.scale = A.pool.scales[kv_row(A.pool, page, (int)wave, h, at & in)];
  }
}

// Of wave 1, which finds it for all: the exponent of the largest value scale of the tile's keys so far, and one that no
// row's own largest is below (of the keys that all rows see; if there are none, of the smallest)
struct ScaleRange {
  int top, low;
};

// key: the step's first, bound: the first that not all rows see
template <int D, int NW, bool COARSE, bool OWN>
__device__ __forceinline__ void tile_put(const Fetched<D, NW>& f, TileLds<D, NW>& S, int step, float unit, int key, int bound,
                                         ScaleRange& range) {
  using F = Fetched<D, NW>;
  constexpr int K = tile_keys<D>(), RUNS = K / 16;
  const uint32_t tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int buf = step & 1;
#pragma unroll
  for (int i = 0; i < F::N; ++i) {
    const uint32_t first = (wave + i * NW) * 64, piece = first + lane;
    if (first >= F::PIECES) break;
    {
      const uint32_t row = piece / (D / 16), c = piece % (D / 16);
      u32x4 half[2];
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const uint32_t u = f.k[i][x] ^ 0x80808080u;
        half[x >> 1][2 * (x & 1)] = codes_f16(__builtin_amdgcn_perm(0u, u, 0x0C010C00u));
        half[x >> 1][2 * (x & 1) + 1] = codes_f16(__builtin_amdgcn_perm(0u, u, 0x0C030C02u));
      }
#pragma unroll
      for (int x = 0; x < 2; ++x) S.k[buf][row * (D / 8) + ((2 * c + x) ^ key_swizzle<D>(row))] = half[x];
    }
    // keys 16s + 8b + 4h': run s*2 + h', its half b
    const uint32_t four = piece / (D / 4), c = piece % (D / 4);
    const uint32_t run = (four >> 2) * 2 + (four & 1), b = (four >> 1) & 1;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t sel = 0x0C000C00u | (uint32_t)j | (uint32_t)(4 + j) << 16;
      u32x2 two;
#pragma unroll
      for (int x = 0; x < 2; ++x)
        two[x] = codes_f16(__builtin_amdgcn_perm(f.v[i][2 * x + 1] ^ 0x80808080u, f.v[i][2 * x] ^ 0x80808080u, sel));
      const uint32_t row = j * (D / 4) + c;
      reinterpret_cast<u32x2*>(&S.v[buf][row * (K / 8) + (run ^ value_swizzle<D>(row))])[b] = two;
    }
  }
  if (wave == 0 && lane < K) S.ks[buf][lane] = f.scale * unit;
  if (wave == 1) {
    const uint32_t bb = mag_bits(f.scale);
    if constexpr (!OWN) {
      const int e = scale_exp(f.scale), top = wave_max(e), shared = bound - key;
      if (shared < K) {
        if (shared > 0) range.low = max(range.top, wave_max((int)lane < shared ? e : -127));
        else if (shared + step * K <= 0) range.low = min(range.low, -wave_max(e > -127 ? -e : -127));
      }
      range.top = max(range.top, top);
      if (shared >= K) range.low = range.top;
    }
    const int e_run = range.top;
    if (lane < K) {
      if constexpr (OWN) {
        S.vs[buf][lane] = f.scale;
      } else if constexpr (COARSE) {
        // key 32 kt + 8 a + 4 h + r is weight 4 a + r of half h
        const int to = (lane & 32) + (lane >> 2 & 1) * 16 + (lane >> 3 & 3) * 4 + (lane & 3);
        reinterpret_cast<_Float16*>(S.vs[buf])[to] = (_Float16)(f.scale * scale_of_exp(-e_run));
      } else {
        S.vs[buf][lane] = f.scale * scale_of_exp(10 - e_run);
      }
    }
    const uint64_t there = __ballot(f.page >= 0);
    uint32_t ok = 0;
#pragma unroll
    for (int i = 0; i < RUNS; ++i) ok |= (uint32_t)(there >> (16 * i) & 1) << i;
    if (__ballot(bb >= 0x7F800000u)) ok |= 1u << 31;
    if (lane == 0) {
      S.e[buf] = e_run;
      S.ok[buf] = ok;
    }
  }
}

// Sums of a lane's row: o[j][i] is row j * 32 + (i / 4) * 8 + h * 4 + i % 4 of the values in LDS
template <int D>
struct RowState {
  f32x16a o[D / 32];
  float m, l;
  int e;  // exponent of the largest value scale: of the tile's keys so far, own: of those that the row sees
};

// Scores of a wave's 32 rows against a step's keys, but for the row's unit.  The stages' LDS reads are issued
// a stage ahead and held there: left to itself the compiler waits for each of them in front of its MFMA.
template <int D, int QT, int NW>
__device__ __forceinline__ void tile_scores(const TileLds<D, NW>& S, int step, const f16x8a (&q)[QT][D / 16],
                                            f32x16a (&t)[tile_keys<D>() / 32]) {
  constexpr int KT = tile_keys<D>() / 32, N = D / 16;
  const int lane = threadIdx.x & 63, l32 = lane & 31, h = lane >> 5;
  auto key = [&](int kt, int i) {
    const int row = kt * 32 + l32;
    return __builtin_bit_cast(f16x8a, S.k[step & 1][row * (D / 8) + ((2 * i + h) ^ key_swizzle<D>(row))]);
  };
  constexpr int AHEAD = 4;  // reads in front of their MFMAs
  f16x8a f[N][KT];
#pragma unroll
  for (int i = 0; i < AHEAD; ++i)
#pragma unroll
    for (int kt = 0; kt < KT; ++kt) f[i][kt] = key(kt, i);
  __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (int kt = 0; kt < KT; ++kt)
#pragma unroll
    for (int i = 0; i < 16; ++i) t[kt][i] = 0.0f;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if (i + AHEAD < N) {
#pragma unroll
      for (int kt = 0; kt < KT; ++kt) f[i + AHEAD][kt] = key(kt, i + AHEAD);
    }
#pragma unroll
    for (int n = 0; n < QT; ++n)
#pragma unroll
      for (int kt = 0; kt < KT; ++kt)
        t[kt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(f[i][kt], q[n][i], t[kt], 0, 0, 0);
    __builtin_amdgcn_sched_barrier(0);
  }
}

// Scores to probabilities and their product with the step's values.  see: a bit for each key that the
// row sees (shifted down by the lane's 4h), used where not `all` of the rows see all keys.
//
// VALU work bounds the kernel (it does not overlap with MFMAs here), so that its instructions per score
// are counted: one fma takes the product with the key's scale and from the maximum; then the
// maximum (half), exponential, conversion (half).  COARSE (bfloat16 results): the probability itself goes to
// float16, the value's scale is applied to pairs, and the weight is a dot product of pairs with ones, 1.5 where the
// exact form takes 2.5 with products and sums in float32.
// OWN: value scales relative to the largest that the row sees, scores times the row's own unit.
template <int D, int PT, int NW, bool COARSE, bool OWN>
__device__ __forceinline__ void tile_values(const TileLds<D, NW>& S, int step, f32x16a (&t)[tile_keys<D>() / 32], bool all,
                                            bool finite, uint64_t see, float own_unit, RowState<D>& st) {
  constexpr int K = tile_keys<D>(), KT = K / 32, N = D / 16;  // N fragments of values for 32 keys
  const int lane = threadIdx.x & 63, l32 = lane & 31, h = lane >> 5, buf = step & 1;
  int e_new = OWN ? st.e : __builtin_amdgcn_readfirstlane(S.e[buf]);
  if constexpr (OWN) {
#pragma unroll
    for (int i = 0; i < 16 * KT; ++i) {
      const int k = (i >> 2) * 8 + (i & 3);
      if (see >> k & 1) e_new = max(e_new, scale_exp(S.vs[buf][k + h * 4]));
    }
    e_new = max(e_new, __shfl_xor(e_new, 32));
  }
  constexpr float UP = COARSE ? 10.0f : 0.0f;  // log2 of the factor that the exact form has in the values' scales
  const float from = st.m == -__builtin_inff() ? 0.0f : st.m;
#pragma unroll
  for (int kt = 0; kt < KT; ++kt)
#pragma unroll
    for (int a = 0; a < 4; ++a) {
      const f32x4a ks = *reinterpret_cast<const f32x4a*>(&S.ks[buf][kt * 32 + a * 8 + h * 4]);
#pragma unroll
      for (int r = 0; r < 4; ++r)
        t[kt][4 * a + r] = OWN ? __builtin_fmaf(t[kt][4 * a + r] * ks[r], own_unit, UP - from)
                               : __builtin_fmaf(t[kt][4 * a + r], ks[r], UP - from);
    }
  if (!all) {
#pragma unroll
    for (int kt = 0; kt < KT; ++kt)
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (!((uint32_t)(see >> (32 * kt)) >> (8 * (i >> 2) + (i & 3)) & 1)) t[kt][i] = -__builtin_inff();
  }
  float top = -__builtin_inff();
#pragma unroll
  for (int kt = 0; kt < KT; ++kt)
#pragma unroll
    for (int i = 0; i < 16; ++i) top = fmaxf(top, t[kt][i]);
  // the running maximum follows the largest score by steps of at least 2^4, as in step32; a row's first score sets it
  if (__ballot(top > UP + 4.0f || (st.m == -__builtin_inff() && top > -__builtin_inff())) ||
      (OWN ? __ballot(e_new != st.e) != 0 : e_new != st.e)) {
    top = fmaxf(top, __shfl_xor(top, 32));
    const bool first = st.m == -__builtin_inff();
    const float rise = first ? (top > -__builtin_inff() ? top - UP : 0.0f) : fmaxf(top - UP, 0.0f);
    const float shrink = first ? 1.0f : __builtin_amdgcn_exp2f(-rise);
    const float both = shrink * scale_of_exp(st.e - e_new);
    st.l *= shrink;
#pragma unroll
    for (int j = 0; j < D / 32; ++j)
#pragma unroll
      for (int i = 0; i < 16; ++i) st.o[j][i] *= both;
#pragma unroll
    for (int kt = 0; kt < KT; ++kt)
#pragma unroll
      for (int i = 0; i < 16; ++i) t[kt][i] -= rise;
    if (!first || top > -__builtin_inff()) st.m = from + rise;
    st.e = e_new;
  }
  f16x8a p[KT][PT][2];
#pragma unroll
  for (int kt = 0; kt < KT; ++kt) {
    f16x8a sc[2];
    f32x4a vs[4];
    if constexpr (COARSE) {
#pragma unroll
      for (int x = 0; x < 2; ++x)
        sc[x] = *reinterpret_cast<const f16x8a*>(reinterpret_cast<const _Float16*>(S.vs[buf]) + kt * 32 + h * 16 + x * 8);
    } else {
#pragma unroll
      for (int x = 0; x < 4; ++x) vs[x] = *reinterpret_cast<const f32x4a*>(&S.vs[buf][kt * 32 + x * 8 + h * 4]);
    }
    if constexpr (OWN) {
      const float up = scale_of_exp(10 - st.e);
#pragma unroll
      for (int i = 0; i < 16; ++i)  // what the row does not see may be past its own
        vs[i >> 2][i & 3] = (uint32_t)(see >> (32 * kt)) >> (8 * (i >> 2) + (i & 3)) & 1 ? vs[i >> 2][i & 3] * up : 0.0f;
    }
    if constexpr (COARSE) {
#pragma unroll
      for (int i = 0; i < 16; i += 2) {
        const f16x2a x = {(_Float16)__builtin_amdgcn_exp2f(t[kt][i]), (_Float16)__builtin_amdgcn_exp2f(t[kt][i + 1])};
        st.l = __builtin_amdgcn_fdot2(x, f16x2a{(_Float16)1.0f, (_Float16)1.0f}, st.l, false);
        const f16x2a c = x * f16x2a{sc[i >> 3][i & 7], sc[i >> 3][(i & 7) + 1]};
        p[kt][0][i >> 3][i & 7] = c[0];
        p[kt][0][i >> 3][(i & 7) + 1] = c[1];
      }
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float x = __builtin_amdgcn_exp2f(t[kt][i]);
        float c = x * vs[i >> 2][i & 3];
        st.l += x;
        if constexpr (PT == 2) asm("" : "+v"(c));
        p[kt][0][i >> 3][i & 7] = (_Float16)c;
        if constexpr (PT == 2) p[kt][1][i >> 3][i & 7] = (_Float16)(c - (float)p[kt][0][i >> 3][i & 7]);
      }
    }
    if (!OWN && !finite) {  // zero times such a scale: what a row does not see adds nothing to it all the same
#pragma unroll
      for (int n = 0; n < PT; ++n)
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (!((uint32_t)(see >> (32 * kt)) >> (8 * (i >> 2) + (i & 3)) & 1)) p[kt][n][i >> 3][i & 7] = (_Float16)0.0f;
    }
  }
  auto value = [&](int x) {  // fragment x: keys x / (N / 2) * 16 on, elements x % (N / 2) * 32 on
    const int row = x % (N / 2) * 32 + l32, run = x / (N / 2) * 2 + h;
    return __builtin_bit_cast(f16x8a, S.v[buf][row * (K / 8) + (run ^ value_swizzle<D>(row))]);
  };
  constexpr int F = KT * N, AHEAD = 8 < F ? 8 : F;
  f16x8a vf[F];
#pragma unroll
  for (int x = 0; x < AHEAD; ++x) vf[x] = value(x);
  __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (int x = 0; x < F; ++x) {
    if (x + AHEAD < F) vf[x + AHEAD] = value(x + AHEAD);
#pragma unroll
    for (int n = 0; n < PT; ++n)
      st.o[x % (N / 2)] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf[x], p[x / N][n][x / (N / 2) % 2], st.o[x % (N / 2)], 0, 0, 0);
    if (x & 1) __builtin_amdgcn_sched_barrier(0);
  }
  __builtin_amdgcn_sched_barrier(0);
}

// Which of a step's K keys from `key` on a row sees, a bit each
template <int K>
__device__ __forceinline__ uint64_t row_sees(const AttendArgs& A, const uint64_t* __restrict__ bits, int key, int ctx, int end,
                                             int tok, uint32_t ok) {
  const int j0 = key - ctx;  // the first key among the new tokens
  uint64_t see = ~0ull;
  if (!A.mask) {
    const int64_t last = (int64_t)tok - j0;  // the last key of the step that the row sees
    see = last < 0 ? 0 : last >= 63 ? ~0ull : (2ull << (int)last) - 1;
  } else if (j0 >= 0) {
    const int word = j0 >> 6, sh = j0 & 63;
    const uint64_t one = word < A.words ? bits[word] : 0, two = word + 1 < A.words ? bits[word + 1] : 0;
    see = sh ? one >> sh | two << (64 - sh) : one;
  } else if (j0 > -64) {
    see = bits[0] << -j0 | ((1ull << -j0) - 1);
  }
  if (end - key < 64) see &= (1ull << (end - key)) - 1;  // keys past the end; there is one before it
#pragma unroll
  for (int i = 0; i < K / 16; ++i)
    if (!(ok >> i & 1)) see &= ~(0xFFFFull << (16 * i));
  return see;
}

// Place in a part of the four elements 32 a + 16 h + 4 r .. of row `wave` * 32 + lane % 32 (a lane's 4 r follow by 256): a
// wave writes and reads 1 KB in a row.
template <int D>
__device__ __forceinline__ int tile_part(int wave, int a, int lane) { return ((wave * (D / 32) + a) * 256 + lane) * 4; }

// The value scales of a tile's keys are taken relative to one exponent, which costs a row bits where its own largest scale is
// far below it: keys that it does not see must not do that.  So are the queries of a tile's rows.  The first launch (not OWN)
// notes tiles where a row's own may be below 2^-4 of the largest scale, or its query below 2^-8 of the largest; a second one
// computes these again with exponents of each row's own, in the exact form for bfloat16 too, and ends at once where there are
// none.  Both forms in one kernel cost it registers: 16 trees of 16 tokens with 8 queries a head behind 4000 keys 71 us without,
// 73 in two launches, 77 in one; 4 of 64 tokens behind 30000 180, 189, 195.
template <typename T, int D, int QT, int PT, int NW, bool OWN>
__global__ __launch_bounds__(64 * NW, D == 256 || QT == 2 ? 1 : 2) void k_attend_tile(AttendArgs A) {
  constexpr int K = tile_keys<D>(), RUNS = K / 16, BATCH = 64 / RUNS;  // runs of a step, steps of a batch of pages
  constexpr bool COARSE = __is_same(T, hip_bfloat16) && !OWN;
  __shared__ TileLds<D, NW> S;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int l32 = lane & 31, h = lane >> 5;
  const int share = share_of_block(A);
  const Line L = make_line(A);
  uint32_t apart = 0;  // OWN: the share's tiles to compute; else found by wave 1
  if constexpr (OWN) {
    apart = A.apart[share];
    if (apart == 0) return;
  } else {
    zero_padding<T, D, 64 * NW>(A);
  }
  uint32_t from, to, per;
  SeqWork w;
  Place p;
  if (!line_share<64 * NW>(A, L, share, from, to, per, w, p)) {
    if constexpr (!OWN) {
      leave_part(A, share, false, 0, 1, w, p);
      if (threadIdx.x == 0) A.apart[share] = 0;
    }
    return;
  }
  uint32_t at = from;
  for (int tile = 0;; tile = min(tile + 1, 31)) {
    const int k1 = (int)min((uint32_t)p.blocks, (uint32_t)p.k + (to - at));
    const bool whole = p.k == 0 && k1 == p.blocks;
    const int end = tile_end(A, w, p);
    const int key0 = p.k * A.keys, stop = (int)min((int64_t)end, (int64_t)k1 * A.keys);
    if (OWN && !(apart >> tile & 1)) {
      at += (uint32_t)(k1 - p.k);
      if (at >= to || !next_tile(A, L, w, p)) break;
      continue;
    }
    RunPages pages;
    pages.start(A, p.b, key0 >> 4);
    int tok, head;
    const bool row_ok = tile_row(A, w, p, wave * 32 + l32, tok, head);
    const bool busy = __ballot(row_ok) != 0;
    QueryHalf<T, D> raw;
    query_load<T, D>(row_ok ? reinterpret_cast<const T*>(A.q) + (int64_t)(w.first + tok) * A.q_token + (int64_t)head * A.q_head
                            : nullptr,
                     h, raw);
    int e_q = raw.e;
#pragma unroll
    for (int i = 1; i < 32; i <<= 1) e_q = max(e_q, __shfl_xor(e_q, i));
    int e_low = raw.some ? raw.e : 127;
    if constexpr (!OWN) {
#pragma unroll
      for (int i = 1; i < 32; i <<= 1) e_low = min(e_low, __shfl_xor(e_low, i));
    }
    const uint64_t* bits = A.mask && row_ok ? A.mask + (int64_t)(w.first + tok) * A.words : A.mask;
    // the wave's first token: it sees all keys up to it, and a causal step past it needs its mask
    int lo_tok = row_ok ? tok : 0x7FFFFFFF;
#pragma unroll
    for (int i = 1; i < 32; i <<= 1) lo_tok = min(lo_tok, __shfl_xor(lo_tok, i));
    lo_tok = __builtin_amdgcn_readfirstlane(lo_tok);

    RowState<D> st;
#pragma unroll
    for (int j = 0; j < D / 32; ++j)
#pragma unroll
      for (int i = 0; i < 16; ++i) st.o[j][i] = 0.0f;
    st.m = -__builtin_inff();
    st.l = 0.0f;
    st.e = -100;
    // keys in front of this one are seen by all rows: the ones held, causal also those up to the tile's first token
    const int bound = A.mask ? w.ctx : w.ctx + min(end - w.ctx, p.x / A.chunks * A.TT + 1);
    ScaleRange range = {-100, 127};
    Fetched<D, NW> f;
    const int steps = stop > key0 ? (stop - key0 + K - 1) / K : 0;
    auto fetch = [&](int n) {
      if (n >= steps) return;
      if (n % BATCH == 0 && n) pages.advance(A, p.b, (key0 >> 4) + (n + BATCH) * RUNS);
      tile_fetch<D, NW>(A, p.h, key0 + n * K, end, pages.cur, (n % BATCH) * RUNS, f);
    };
    fetch(0);
    __syncthreads();  // the tile before is read
    if (lane == 0) S.top[wave] = e_q, S.low[wave] = e_low;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NW; ++i) e_q = max(e_q, S.top[i]), e_low = min(e_low, S.low[i]);
    e_q = __builtin_amdgcn_readfirstlane(e_q);
    if (!OWN && __builtin_amdgcn_readfirstlane(e_low) < e_q - 8) apart |= 1u << tile;
    f16x8a q[QT][D / 16];
    query_terms16<T, D, QT>(raw, OWN ? raw.e : e_q, q);
    // of a product of a query's terms and a key's code * 2^-9
    const float unit = OWN ? 0x1p-5f * A.scale : scale_of_exp(e_q - 14 + 9) * A.scale, own_unit = OWN ? scale_of_exp(raw.e) : 0.0f;
    if (steps) tile_put<D, NW, COARSE, OWN>(f, S, 0, unit, key0, bound, range);
    __syncthreads();
    fetch(1);
    for (int n = 0; n < steps; ++n) {
      if (busy) {
        const int key = key0 + n * K, j0 = key - w.ctx;
        f32x16a t[K / 32];
        tile_scores<D, QT, NW>(S, n, q, t);
        const uint32_t ok = __builtin_amdgcn_readfirstlane(S.ok[n & 1]);
        const bool all = key + K <= end && (ok & 0xFFFFu) == (1u << RUNS) - 1 &&
                         (j0 + K <= 0 || (!A.mask && j0 + K - 1 <= lo_tok));
        uint64_t see = ~0ull;
        if (!all) see = row_sees<K>(A, bits, key, w.ctx, end, tok, ok) >> (4 * h);
        tile_values<D, PT, NW, COARSE, OWN>(S, n, t, all, ok >> 31 == 0, see, own_unit, st);
      }
      if (n + 1 < steps) tile_put<D, NW, COARSE, OWN>(f, S, n + 1, unit, key0 + (n + 1) * K, bound, range);
      __syncthreads();
      fetch(n + 2);
    }

    // a lane has its row's elements 4c .. 4c+3 for every c with bit 2 of c equal to h
    float l = st.l;
    l += __shfl_xor(l, 32);
    if constexpr (COARSE) l *= 0x1p-10f;
    if (raw.nan && l != 0.0f) l = __uint_as_float(0x7FC00000u);  // of a row that sees a key
    if (row_ok) {
      const float down = scale_of_exp(st.e - 1), inv = l == 0.0f ? 0.0f : 1.0f / l;
      const int64_t slot = (int64_t)share * 2 + (p.k == 0 ? 1 : 0);
      T* dst = reinterpret_cast<T*>(A.out) + ((int64_t)(w.first + tok) * A.Hq + head) * D;
      float* part = A.part_o + slot * (32 * NW * D) + tile_part<D>(wave, 0, lane);
#pragma unroll
      for (int a = 0; a < D / 32; ++a) {  // 16 elements in a row
        T y[16];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          f32x4a x;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int row = j * (D / 4) + 8 * a + r;
            x[j] = st.o[row / 32][(row % 32 / 8) * 4 + row % 4] * down;
          }
          if (!whole) *reinterpret_cast<f32x4a*>(part + a * 1024 + r * 256) = x;
#pragma unroll
          for (int j = 0; j < 4; ++j) y[4 * r + j] = out_cvt<T>(x[j] * inv);
        }
        if (whole) __builtin_memcpy(dst + 32 * a + 16 * h, y, sizeof(y));
      }
      if (!whole && h == 0) A.part_s[slot * (32 * NW) + wave * 32 + l32] = make_float2(st.m, l);
    }
    if (!OWN && wave == 1 && range.top > range.low + 4) apart |= 1u << tile;
    at += (uint32_t)(k1 - p.k);
    const bool some = p.k == 0 && k1 < p.blocks;  // then at >= to
    const uint32_t last = at + (uint32_t)(p.blocks - k1);
    if (at >= to || !next_tile(A, L, w, p)) {
      if constexpr (!OWN) {
        leave_part(A, share, some, last, per, w, p);
        if (threadIdx.x == 64) A.apart[share] = apart;
      }
      break;
    }
  }
}

// A tile that share s begins and does not end: its parts are share s's second
// one and the first ones of the shares after it, up to the one with its last
// block.  Tiles of 16 rows, which may have many parts: a wave a row; a lane finds the weight of
// every 64th part, all lanes add the parts' sums in their order.
template <typename T, int D>
__global__ __launch_bounds__(256) void k_attend_join(AttendArgs A) {
  constexpr int E = D / 64, U = 16;  // elements of a lane, parts in flight
  const int s = blockIdx.x, lane = threadIdx.x & 63, r = blockIdx.y * 4 + (threadIdx.x >> 6);
  const PartTile t = A.part_t[s];
  if (t.last < 0) return;
  SeqWork w;
  w.first = t.first;
  w.n = t.n;
  Place p;
  p.h = t.h;
  p.x = t.x;
  int tok, head;
  if (!tile_row(A, w, p, r, tok, head)) return;
  const int parts = t.last - s + 1;
  auto slot = [&](int i) { return ((int64_t)(s + i) * 2 + (i == 0)) * A.rows + r; };
  float m = -__builtin_inff(), sum = 0.0f, acc[E];
#pragma unroll
  for (int j = 0; j < E; ++j) acc[j] = 0.0f;
  for (int i0 = 0; i0 < parts; i0 += 64) {
    const int n = min(64, parts - i0);
    float v[U][E];
    auto load = [&](int i) {  // past the last part: it again, not added
#pragma unroll
      for (int u = 0; u < U; ++u)
        __builtin_memcpy(v[u], A.part_o + slot(i0 + min(i + u, n - 1)) * D + lane * E, sizeof(v[u]));
    };
    const float2 ms = A.part_s[slot(i0 + min(lane, n - 1))];
    load(0);  // on its way while the weights are found
    float top = fmaxf(m, ms.x);
#pragma unroll
    for (int i = 1; i < 64; i <<= 1) top = fmaxf(top, __shfl_xor(top, i));
    const float shrink = m == top ? 1.0f : __builtin_amdgcn_exp2f(m - top);
    m = top;
    const float f = lane >= n ? 0.0f : ms.x == m ? 1.0f : __builtin_amdgcn_exp2f(ms.x - m);
    sum *= shrink;
    if (lane < n) sum += f * ms.y;
#pragma unroll
    for (int j = 0; j < E; ++j) acc[j] *= shrink;
    for (int i = 0;;) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const float g = __shfl(f, min(i + u, 63));
        if (i + u < n) {
#pragma unroll
          for (int j = 0; j < E; ++j) acc[j] = __builtin_fmaf(g, v[u][j], acc[j]);
        }
      }
      if ((i += U) >= n) break;
      load(i);
    }
  }
#pragma unroll
  for (int i = 1; i < 64; i <<= 1) sum += __shfl_xor(sum, i);
  const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
  T e[E];
#pragma unroll
  for (int j = 0; j < E; ++j) e[j] = out_cvt<T>(acc[j] * inv);
  __builtin_memcpy(reinterpret_cast<T*>(A.out) + ((int64_t)(w.first + tok) * A.Hq + head) * D + lane * E, e, sizeof(e));
}

// The same for tiles of many rows, which have few parts: a lane has 16 elements of a row as in k_attend_tile and finds the
// parts' weights itself.  Bound by the parts' bytes: 256 shares of 256 rows of 128, 7.5 to 13.5 us at 5 to 6 TB/s.
template <typename T, int D>
__global__ __launch_bounds__(256) void k_attend_join_tile(AttendArgs A) {
  const int s = blockIdx.x, lane = threadIdx.x & 63, unit = blockIdx.y * 4 + (threadIdx.x >> 6);
  const int wave = unit / (D / 32), a = unit % (D / 32), r = wave * 32 + (lane & 31);
  const PartTile t = A.part_t[s];
  if (t.last < 0) return;
  SeqWork w;
  w.first = t.first;
  w.n = t.n;
  Place p;
  p.h = t.h;
  p.x = t.x;
  int tok, head;
  if (!tile_row(A, w, p, r, tok, head)) return;
  const int parts = t.last - s + 1;
  auto slot = [&](int i) { return (int64_t)(s + i) * 2 + (i == 0); };
  constexpr int U = 4;  // parts in flight
  float m = -__builtin_inff(), sum = 0.0f;
  f32x4a acc[4];
#pragma unroll
  for (int x = 0; x < 4; ++x) acc[x] = f32x4a{0, 0, 0, 0};
  for (int i = 0; i < parts; i += U) {
    float2 ms[U];
    f32x4a v[U][4];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      ms[u].x = -__builtin_inff();
      if (i + u < parts) {
        ms[u] = A.part_s[slot(i + u) * A.rows + r];
        const float* part = A.part_o + slot(i + u) * A.rows * D + tile_part<D>(wave, a, lane);
#pragma unroll
        for (int x = 0; x < 4; ++x) v[u][x] = *reinterpret_cast<const f32x4a*>(part + x * 256);
      }
    }
    float top = m;
#pragma unroll
    for (int u = 0; u < U; ++u) top = fmaxf(top, ms[u].x);
    const float shrink = m == top ? 1.0f : __builtin_amdgcn_exp2f(m - top);
    m = top;
    sum *= shrink;
#pragma unroll
    for (int x = 0; x < 4; ++x) acc[x] *= shrink;
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (i + u < parts) {
        const float f = ms[u].x == m ? 1.0f : __builtin_amdgcn_exp2f(ms[u].x - m);
        sum += f * ms[u].y;
#pragma unroll
        for (int x = 0; x < 4; ++x)
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[x][j] = __builtin_fmaf(f, v[u][x][j], acc[x][j]);
      }
  }
  const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
  T e[16];
#pragma unroll
  for (int x = 0; x < 4; ++x)
#pragma unroll
    for (int j = 0; j < 4; ++j) e[4 * x + j] = out_cvt<T>(acc[x][j] * inv);
  __builtin_memcpy(reinterpret_cast<T*>(A.out) + ((int64_t)(w.first + tok) * A.Hq + head) * D + 32 * a + 16 * (lane >> 5), e,
                   sizeof(e));
}

// ---------------------------------------------------------------- host
struct AttendPlan {
  int rows, keys, TT, GC, chunks, shares, cap, most;
  bool cut;  // a tile may be cut
  bool fits;  // the line is below 2^31 blocks
};

static AttendPlan plan_attend(int64_t T, int64_t B, int64_t width, int page, int H, int G, int D, bool wide) {
  AttendPlan a;
  // rows of a sequence and key head, on average
  const double each = B > 0 ? (double)T * G / (double)std::min(B, T) : 0.0;
  // Tiles of 16 rows, whose waves need no barrier, though several of them read the same keys from the L2, then of 128 (two
  // workgroups a CU but for float32 and heads of 256), then of 256.  us by tiles of 16 / 128 / 256, 8 heads with 4 queries each:
  // heads of 128, bfloat16, 16 sequences of 4000 keys: 48 rows 75 / 66 / 88, 64 rows 70 / 66 / 89, 80 rows 109 / 71 / 88, 128 rows
  // 127 / 74 / 89, 160 rows 161 / 113 / 93, 192 rows 178 / 112 / 98; 2 of 60000: 64 rows 128 / 114 / 157, 80 rows 147 / 124 / 158, 128
  // rows 224 / 129 / 156, 160 rows 265 / 199 / 163; 16 of 300: 48 rows 17 / 28 / 24, 64 rows 18 / 30 / 26, 80 rows 31 / 32 / 27, 128 rows
  // 29 / 35 / 30.  float32 by 16 / 128, 4000 keys: 80 rows 110 / 124, 96 rows 104 / 126, 112 rows 148 / 126, 128 rows 125 / 129; 60000: 96
  // rows 174 / 220, 112 rows 254 / 225.  Heads of 256, bfloat16 by 16 / 128, 4000 keys: 64 rows 125 / 197, 80 rows 199 / 198, 96 rows
  // 182 / 199, 112 rows 272 / 201; 60000: 80 rows 420 / 360, 96 rows 334 / 360, 112 rows 559 / 363; float32, 4000 keys: 80 rows 201 / 249, 96
  // rows 204 / 248, 112 rows 275 / 251.
  // (Up to 64 rows short contexts would lose more by 128 than long ones win.)
  a.rows = each <= (wide || D == 256 ? 96 : 64) ? 16 : D == 256 || wide || each <= 128 ? 128 : 256;
  a.keys = a.rows == 16 ? 128 : 256;
  a.GC = std::min(G, a.rows);
  a.chunks = (int)ceil_div(G, a.GC);
  a.TT = 1;
  while (a.TT * 2 * a.GC <= a.rows) a.TT *= 2;
  // no more shares than blocks there can be
  const double tiles = ((double)T / a.TT + (double)std::min(B, T)) * a.chunks * H;
  a.cap = (int)std::min<int64_t>(width * page, ((int64_t)1 << 31) - ((int64_t)1 << 16));
  a.most = std::max(1, (a.cap + a.keys - 1) / a.keys);
  a.cut = a.most > 1 && B > 0;
  a.fits = tiles * a.most < 2147483648.0;
  const double most = (a.rows == 256 || D == 256 || (a.rows == 128 && wide) ? 1.0 : 2.0) * num_cus();  // workgroups that run at once
  a.shares = (int)std::max(1.0, std::min(most, tiles * a.most));
  return a;
}

static bool has_parts(const AttendPlan& a) { return a.cut && a.shares > 1; }

static size_t attend_bytes(const AttendPlan& a, int D) {
  return (size_t)a.shares * ((has_parts(a) ? 2 * (size_t)a.rows * ((size_t)D * 4 + sizeof(float2)) + sizeof(PartTile) : 0) +
                             (a.rows > 16 ? sizeof(uint32_t) : 0));
}

template <typename T, int D, int QT, int PT>
static int launch_attend(const AttendArgs& A, const AttendPlan& a, hipStream_t st) {
  constexpr int QH = sizeof(T) == 4 ? 2 : 1;  // float16 terms of a query and of the probabilities in the tile kernel
  if (a.rows == 16) {
    hipLaunchKernelGGL((k_attend<T, D, QT, PT>), dim3(a.shares), dim3(256), 0, st, A);
  } else if (a.rows == 128) {
    hipLaunchKernelGGL((k_attend_tile<T, D, QH, QH, 4, false>), dim3(a.shares), dim3(256), 0, st, A);
    hipLaunchKernelGGL((k_attend_tile<T, D, QH, QH, 4, true>), dim3(a.shares), dim3(256), 0, st, A);
  } else {
    if constexpr (D < 256 && QH == 1) {
      hipLaunchKernelGGL((k_attend_tile<T, D, QH, QH, 8, false>), dim3(a.shares), dim3(512), 0, st, A);
      hipLaunchKernelGGL((k_attend_tile<T, D, QH, QH, 8, true>), dim3(a.shares), dim3(512), 0, st, A);
    }
  }
  if (has_parts(a)) {
    if (a.rows == 16) hipLaunchKernelGGL((k_attend_join<T, D>), dim3(a.shares - 1, 4), dim3(256), 0, st, A);
    else hipLaunchKernelGGL((k_attend_join_tile<T, D>), dim3(a.shares - 1, a.rows * D / 4096), dim3(256), 0, st, A);
  }
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

size_t mxk_kv_pages_attend_workspace(int q_type, int64_t tokens, int64_t B, int64_t width, int page, int heads,
                                     int q_heads, int D) {
  if (tokens <= 0 || B <= 0 || width < 0 || heads < 1 || q_heads < heads || q_heads % heads || !kv_page_ok(page))
    return 0;
  const AttendPlan a = plan_attend(tokens, B, width, page, heads, q_heads / heads, D, q_type == MXK_IN_F32);
  return attend_bytes(a, D);
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
      tokens > (int64_t)1 << 30)
    return fail(MXK_EINVAL, "kv_attend: bad sizes (sequences below 2^24, pages of one below 2^31, at most 2^30 tokens)");
  if (!(scale > 0.0f) || !std::isfinite(scale * 1.4426950408889634f))
    return fail(MXK_EINVAL, "kv_attend: the scale is a positive number");
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
  const AttendPlan a = plan_attend(tokens, B, width, page, heads, G, D, q_type == MXK_IN_F32);
  if (!a.fits) return fail(MXK_EINVAL, "kv_attend: more than 2^31 blocks of keys that the table has room for");
  const size_t need = attend_bytes(a, D), part = (size_t)a.shares * 2 * a.rows;
  if (need && (!workspace || workspace_nbytes < need || !aligned16(workspace)))
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
  A.cap = a.cap;
  A.most = a.most;
  A.rows = a.rows;
  A.shares = a.shares;
  const bool parts = has_parts(a);
  A.part_o = parts ? reinterpret_cast<float*>(workspace) : nullptr;
  A.part_s = parts ? reinterpret_cast<float2*>(A.part_o + part * D) : nullptr;
  A.part_t = parts ? reinterpret_cast<PartTile*>(A.part_s + part) : nullptr;
  A.apart = reinterpret_cast<uint32_t*>(parts ? static_cast<void*>(A.part_t + a.shares) : workspace);
  if (q_type == MXK_IN_F32) return launch_attend_d<float, 3, 2>(D, A, a, st);
  if (q_type == MXK_IN_F16) return launch_attend_d<__half, 2, 2>(D, A, a, st);
  return launch_attend_d<hip_bfloat16, 2, 1>(D, A, a, st);
}

}  // extern "C"
