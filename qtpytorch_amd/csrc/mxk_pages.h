// Paged 8-bit key-value cache (gfx950 only): layout and look-ups.
//
//   codes  int8  [pages][2][H][page][D]   keys (0) and values (1)
//   scales float [pages][2][H][page]      value = code * scale
//
// A page is a power of two of at least 16 positions; D is 64, 128 or 256.  A
// batch of B sequences: table [B][width] (the page of each run of positions),
// lengths [B] (positions held), offsets [B+1] (first of each one's new tokens
// among the T of a call).  All of it is device data that the host has not
// seen: a page outside the pool, a position outside the table and a token of
// no sequence are left out by every kernel, so that no access leaves its
// buffer whatever the values are.
#pragma once

#include "mxk_internal.h"

namespace mxk {

struct KvPool {
  int8_t* codes;
  float* scales;
  uint32_t pages;
  int H, shift;  // page = 1 << shift positions
};

struct KvBatch {
  const int* __restrict__ table;
  const int* __restrict__ lengths;
  const int* __restrict__ offsets;
  int B, width, T;
};

// Page of run `run` of sequence b, or -1
__device__ __forceinline__ int kv_page(const KvBatch& s, const KvPool& p, int b, int64_t run) {
  if ((uint64_t)run >= (uint64_t)s.width) return -1;
  const int page = s.table[(int64_t)b * s.width + run];
  return (uint32_t)page < p.pages ? page : -1;
}

// New tokens of sequences: offset i taken into [0, T], and how many tokens sequence b has (with its first one inside [0, T])
__device__ __forceinline__ int kv_offset(const KvBatch& s, int i) { return min(max(s.offsets[i], 0), s.T); }
__device__ __forceinline__ int kv_count(const KvBatch& s, int b) { return max(0, kv_offset(s, b + 1) - kv_offset(s, b)); }

// Position of token t in sequence b
__device__ __forceinline__ int64_t kv_place(const KvBatch& s, int b, int t) {
  return (int64_t)s.lengths[b] + ((int64_t)t - s.offsets[b]);
}

// Blocks of a launch over tokens: x and z, since the threads of one dimension stay below 2^32.  Up to 2^22 - 1 of them lie
// past the last: their kernels end at once.
inline dim3 kv_grid(int64_t blocks, int64_t parts) {
  const int64_t x = blocks < ((int64_t)1 << 22) ? blocks : (int64_t)1 << 22;
  return dim3((unsigned)x, (unsigned)parts, (unsigned)ceil_div(blocks, x));
}
__device__ __forceinline__ int kv_block() { return (int)(blockIdx.z * gridDim.x + blockIdx.x); }

// Sequence of token t, found by a whole wave: the number of sequences that
// end at or before t; -1 for a token of none.  A lane looks at the end of one of 64 runs of
// sequences, so that up to 64 take one load and up to 4096 two, where a binary search takes 6 and 12 dependent ones
// (4096 tokens of as many sequences appended in 5 us, 14 with a walk of 64 at a time).
__device__ __forceinline__ int kv_sequence(const KvBatch& s, int t) {
  const int lane = threadIdx.x & 63;
  int b = 0, n = s.B;  // the runs still in question: sequences [b, b + n)
  while (n > 0) {
    const int run = (n + 63) >> 6;
    const int last = min((lane + 1) * run, n);  // past the lane's run
    const bool mine = lane * run < n;
    const int ends = __builtin_popcountll(__ballot(mine && s.offsets[b + last] <= t));
    b += min(ends * run, n);
    n = run == 1 ? 0 : min(run, n - ends * run);
  }
  return b < s.B && s.offsets[b] <= t ? b : -1;
}

// A row of the cache: which = 0 key, 1 value
__device__ __forceinline__ int64_t kv_row(const KvPool& p, int page, int which, int h, int at) {
  return ((((int64_t)page * 2 + which) * p.H + h) << p.shift) + at;
}

inline bool kv_page_ok(int page) { return page >= 16 && page <= (1 << 20) && is_pow2(page); }
inline int log2_of(int64_t v) {
  int l = 0;
  while (((int64_t)1 << l) < v) ++l;
  return l;
}

}  // namespace mxk
