// Tokens to experts and back, for gfx950: the order of picks by expert, the
// copy of token rows in that order, their weighted sum and its gradients.
//
// P = tokens * top picks, pick i = t * top + j of token t.  The plan of a
// routing is three int32 arrays:
//   order[P]      pick at each sorted place (stable: by expert, then by
//                 pick), -1 past the last pick that has an expert
//   place[P]      where each pick went, -1 for one without an expert (an id
//                 outside [0, E): another device's, or a padded token's)
//   offsets[E+1]  first place of each expert; offsets[E] is the number in use
// Every kernel here gathers: each output element is written by one thread in
// a fixed order of additions, so results do not depend on timing.
#include "mxk_mxfp4.h"

namespace mxk {

#define MXK_SORT_THREADS 1024
#define MXK_SORT_WAVES (MXK_SORT_THREADS / 64)

// expert of a pick, E for one without
template <typename I>
__device__ __forceinline__ uint32_t expert_of(I id, uint32_t E) {
  return (uint64_t)(int64_t)id < (uint64_t)E ? (uint32_t)id : E;
}

// Counts of each expert in each chunk of picks: hist[chunk][E].
template <typename I>
__global__ __launch_bounds__(MXK_SORT_THREADS) void k_expert_count(const I* __restrict__ ids, uint32_t P, uint32_t E,
                                                                   uint32_t chunk, int* __restrict__ hist) {
  extern __shared__ int cnt[];  // [E + 1]
  for (uint32_t e = threadIdx.x; e <= E; e += MXK_SORT_THREADS) cnt[e] = 0;
  __syncthreads();
  const uint32_t lo = blockIdx.x * chunk, hi = min(P, lo + chunk);
  for (uint32_t i = lo + threadIdx.x; i < hi; i += MXK_SORT_THREADS) atomicAdd(&cnt[expert_of(ids[i], E)], 1);
  __syncthreads();
  for (uint32_t e = threadIdx.x; e < E; e += MXK_SORT_THREADS) hist[(int64_t)blockIdx.x * E + e] = cnt[e];
}

// One chunk of picks to their places.  Bounded by latency (the ids are a few
// hundred KB at most): each wave counts its own contiguous share in LDS, the
// shares' first places follow from the counts of the chunks before (`hist`,
// which a single chunk does not need) and of the waves before, and a wave
// then places 64 picks at a time, ranked among the lanes with the same expert by
// ballots over the bits of the expert's number.  64 picks 3.5 us; 65536 picks of 128
// experts 7.2 us and 3.1 for the counts.
template <typename I>
__global__ __launch_bounds__(MXK_SORT_THREADS) void k_expert_place(const I* __restrict__ ids, uint32_t P, uint32_t E,
                                                                   uint32_t chunk, const int* __restrict__ hist,
                                                                   int* __restrict__ order, int* __restrict__ place,
                                                                   int* __restrict__ offsets) {
  extern __shared__ int sh[];
  int* start = sh;                                  // [waves][E + 1]: counts, then next places
  int* sums = sh + MXK_SORT_WAVES * (E + 1);        // [waves]: scan over waves of experts
  const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6;
  for (uint32_t k = tid; k < MXK_SORT_WAVES * (E + 1); k += MXK_SORT_THREADS) start[k] = 0;
  __syncthreads();
  const uint32_t share = (chunk / MXK_SORT_WAVES + 63u) & ~63u;  // a multiple of 64 per wave
  const uint32_t first = blockIdx.x * chunk, last = min(P, first + chunk);
  const uint32_t lo = min(last, first + wave * share), hi = min(last, lo + share);
  int* mine = start + wave * (E + 1);
  for (uint32_t i = lo + lane; i < hi; i += 64) atomicAdd(&mine[expert_of(ids[i], E)], 1);
  __syncthreads();
  // an expert per thread (there are at most 1000): totals, exclusive scan, first places
  int before = 0, total = 0;
  if (tid < E) {
    if (gridDim.x > 1) {
      for (uint32_t c0 = 0; c0 < gridDim.x; c0 += 16) {  // sixteen chunks' counts at a time
        int n[16];
#pragma unroll
        for (uint32_t k = 0; k < 16; ++k) n[k] = c0 + k < gridDim.x ? hist[(int64_t)(c0 + k) * E + tid] : 0;
#pragma unroll
        for (uint32_t k = 0; k < 16; ++k) {
          total += n[k];
          before += c0 + k < blockIdx.x ? n[k] : 0;
        }
      }
    } else {
      for (int w = 0; w < MXK_SORT_WAVES; ++w) total += start[w * (E + 1) + tid];
    }
  }
  int scan = total;  // inclusive over the wave
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int up = __shfl_up(scan, d);
    if ((int)lane >= d) scan += up;
  }
  if (lane == 63) sums[wave] = scan;
  __syncthreads();
  int left = 0, used = 0;
  for (uint32_t w = 0; w < MXK_SORT_WAVES; ++w) {
    if (w < wave) left += sums[w];
    used += sums[w];
  }
  if (tid < E) {
    const int at = left + scan - total;
    if (blockIdx.x == 0) offsets[tid] = at;
    int next = at + before;
    for (int w = 0; w < MXK_SORT_WAVES; ++w) {
      const int n = start[w * (E + 1) + tid];
      start[w * (E + 1) + tid] = next;
      next += n;
    }
  }
  __syncthreads();
  if (blockIdx.x == 0 && tid == 0) offsets[E] = used;
  // places past the last one in use
  for (uint32_t i = first + tid; i < last; i += MXK_SORT_THREADS)
    if (i >= (uint32_t)used) order[i] = -1;
  const int bits = 32 - __builtin_clz(E | 1u);  // of 0 .. E
  for (uint32_t i0 = lo; i0 < hi; i0 += 64) {
    const uint32_t i = i0 + lane;
    const bool live = i < hi;
    const uint32_t e = live ? expert_of(ids[i], E) : E;
    uint64_t same = __ballot(live);
    for (int b = 0; b < bits; ++b) {
      const uint64_t set = __ballot((e >> b) & 1u);
      same &= ((e >> b) & 1u) ? set : ~set;
    }
    const int rank = __popcll(same & ((1ull << lane) - 1ull));
    const bool picked = live && e < E;
    int at = -1;
    if (picked) at = mine[e] + rank;
    // every lane has read its counter before the first of each expert moves it
    __builtin_amdgcn_wave_barrier();
    if (picked && rank == 0) mine[e] += __popcll(same);
    __builtin_amdgcn_wave_barrier();
    if (live) place[i] = at;
    if (picked) order[at] = (int)i;
  }
}

// out[r] = x[order[r] / top], zeros where order[r] < 0: a copy, bound by
// HBM's write rate (a token's row is read `top` times, from the caches after
// the first).  A thread copies one piece of 16 bytes: four a thread with their loads
// first took as long for large copies and longer for small ones (32000 rows of
// 4096 bf16 63 us both, 4000 rows 7.7 against 6.5).  WHOLE: rows of whole aligned
// pieces, written past the caches; else any alignment, and the last piece of a
// row may be shorter.
template <bool WHOLE>
__global__ __launch_bounds__(256) void k_expert_gather(const uint8_t* __restrict__ x, int64_t x_stride,
                                                       const int* __restrict__ order, DivU32 by_top, uint32_t tokens,
                                                       uint32_t total, DivU32 by_pieces, uint32_t pieces,
                                                       uint32_t row_bytes, uint32_t slices, uint8_t* __restrict__ out) {
  // slices = 8: workgroup b, on XCD b % 8, copies that eighth of the columns
  // (pieces and total are a slice's), so that an XCD's L2 sees an eighth of each
  // token (32000 rows of 4096 bf16, 4 a token: 63 us against 74); slices = 1: whole rows
  const uint32_t slice = slices > 1 ? blockIdx.x & 7u : 0u, block = slices > 1 ? blockIdx.x >> 3 : blockIdx.x;
  const uint64_t i = (uint64_t)block * 256u + threadIdx.x;
  if (i >= total) return;
  const uint32_t r = divu32((uint32_t)i, by_pieces);
  const uint32_t c = (slice * pieces + (uint32_t)i - r * pieces) * 16u;
  const int pick = order[r];
  const uint32_t token = divu32((uint32_t)pick, by_top);
  const bool some = pick >= 0 && token < tokens;
  const uint8_t* p = x + (int64_t)token * x_stride + c;
  uint8_t* o = out + (int64_t)r * row_bytes + c;
  u32x4 v = {0u, 0u, 0u, 0u};
  if (WHOLE) {
    if (some) v = *reinterpret_cast<const u32x4*>(p);
    __builtin_nontemporal_store(v, reinterpret_cast<u32x4*>(o));
  } else if (c + 16u <= row_bytes) {
    if (some) __builtin_memcpy(&v, p, 16);
    __builtin_memcpy(o, &v, 16);
  } else {  // elements have an even number of bytes
    for (uint32_t k = c; k < row_bytes; k += 2, p += 2, o += 2) {
      uint16_t t = 0;
      if (some) __builtin_memcpy(&t, p, 2);
      __builtin_memcpy(o, &t, 2);
    }
  }
}

// 8 results at p (the first `live` where fewer are left)
template <typename T>
__device__ __forceinline__ void store8(T* p, int live, const float (&v)[8]) {
  T t[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) t[e] = from_f32<T>(v[e]);
  if (live >= 8) {
    __builtin_memcpy(p, t, sizeof(t));
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < live) p[e] = t[e];
  }
}

// 8 elements on 16 bytes that are read once, or written past the caches
template <typename T>
__device__ __forceinline__ void load8_nt(const T* p, FpWords<T, 8>& v) {
#pragma unroll
  for (int k = 0; k < FpWords<T, 8>::NW / 4; ++k) {
    const u32x4 w = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(p) + k);
    __builtin_memcpy(&v.w[4 * k], &w, 16);
  }
}
template <typename T>
__device__ __forceinline__ void store8_nt(T* p, const float (&v)[8]) {
  T t[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) t[e] = from_f32<T>(v[e]);
  u32x4 w[sizeof(t) / 16];
  __builtin_memcpy(w, t, sizeof(t));
#pragma unroll
  for (int k = 0; k < (int)sizeof(t) / 16; ++k) __builtin_nontemporal_store(w[k], reinterpret_cast<u32x4*>(p) + k);
}

// y[t] = sum over j of gate[t, j] * h[place[t, j]] (gate = 1 where gates is
// null), in float32 by ascending j, picks without an expert left out.  Bound
// by HBM: one read of the rows in use, one write of the tokens.  A thread
// holds 8 columns of a token and requests the rows of Q picks at a time (eight in
// place of four were no faster for 8 picks a token, 101 us for 8000 tokens of
// 4096 bf16, and slower for 4: 68 against 54): a pick without an expert reads row 0 in
// place of a branch, and its values are replaced by zeros.  8000 tokens of 4096
// bf16, 4 picks (328 MB): 53 us, 6.1 TB/s.
// The result's type O is the rows' or, for float32 rows, any: rounded once.
// WHOLE: columns in whole groups of 8 on 16 bytes.
template <typename T, typename O, bool GATED, bool WHOLE>
__global__ __launch_bounds__(256) void k_expert_combine(const T* __restrict__ h, const int* __restrict__ place,
                                                        const float* __restrict__ gates, int top, int rows,
                                                        uint32_t total, DivU32 by_pieces, uint32_t pieces, int cols,
                                                        O* __restrict__ y) {
  const uint64_t i = (uint64_t)blockIdx.x * 256u + threadIdx.x;
  if (i >= total) return;
  const uint32_t t = divu32((uint32_t)i, by_pieces), c = 8u * ((uint32_t)i - t * pieces);
  const int live = WHOLE ? 8 : cols - (int)c;
  constexpr int Q = 4;
  float acc[8] = {0, 0, 0, 0, 0, 0, 0, 0};
  const int64_t p0 = (int64_t)t * top;
  if (rows > 0) {
    for (int j0 = 0; j0 < top; j0 += Q) {
      FpWords<T, 8> v[Q];
      float g[Q];
      bool ok[Q];
#pragma unroll
      for (int q = 0; q < Q; ++q) {
        const int j = j0 + q < top ? j0 + q : top - 1;
        const int at = place[p0 + j];
        ok[q] = j0 + q < top && at >= 0 && at < rows;
        g[q] = GATED ? gates[p0 + j] : 1.0f;
        const T* row = h + (int64_t)(ok[q] ? at : 0) * cols + c;
        if (WHOLE) load8_nt(row, v[q]);
        else if (live >= 8) fp4_load(row, v[q]);
        else fp4_load_tail(row, live, v[q]);
      }
#pragma unroll
      for (int q = 0; q < Q; ++q) {
        T e8[8];
        __builtin_memcpy(e8, v[q].w, sizeof(e8));
        // an exact zero for a pick that is not there, whatever row 0 and its gate hold
        const float w = ok[q] ? g[q] : 0.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e) acc[e] = __builtin_fmaf(w, ok[q] ? ElemT<T>::cvt(e8[e]) : 0.0f, acc[e]);
      }
    }
  }
  store8(y + (int64_t)t * cols + c, live, acc);
}

// Zeros in the rows of dh that no place names: the picks dropped from a plan, the
// rows past the last in use.  A place names row r if it is that of the pick
// order[r]; should a plan's order not be the inverse of its places, the row of a place is
// written over by the launch behind this one.  A workgroup looks at 32 rows: 1.5 to 2.7 us
// for 32000 rows that are all named, 15 where a quarter of them, 8 KB each, are not.
// WHOLE: rows of whole aligned 16-byte pieces.
template <bool WHOLE>
__global__ __launch_bounds__(256) void k_expert_unnamed(const int* __restrict__ order, const int* __restrict__ place,
                                                        int rows, int64_t row_bytes, uint8_t* __restrict__ dh) {
  const int64_t r0 = (int64_t)blockIdx.x * 32, r = r0 + (threadIdx.x & 31);
  bool none = false;
  if (r < rows) {
    const int pick = order[r];
    none = pick < 0 || pick >= rows || place[pick] != r;
  }
  // the halves of a wave hold the same rows
  for (uint32_t left = (uint32_t)__ballot(none); left; left &= left - 1u) {
    uint8_t* row = dh + (r0 + __builtin_ctz(left)) * row_bytes;
    if (WHOLE) {
      for (int64_t c = threadIdx.x * 16; c < row_bytes; c += 4096)
        __builtin_nontemporal_store(u32x4{0u, 0u, 0u, 0u}, reinterpret_cast<u32x4*>(row + c));
    } else {  // elements have an even number of bytes
      const uint16_t z = 0;
      for (int64_t c = threadIdx.x * 2; c < row_bytes; c += 512) __builtin_memcpy(row + c, &z, 2);
    }
  }
}

// Gradients of the weighted sum: dh[place[t, j]] = gate[t, j] * dy[t] and
// dgate[t, j] = <dy[t], h[place[t, j]]>; zero for picks without an expert.  Rows
// that no place names are k_expert_unnamed's.  Not GATED: gates of 1, no dgate, h
// is not read.  Bound by HBM: dy is read once per
// token and group of four picks, h read and dh written once.  W waves share a
// token, one for each 512 columns (up to 8), so that a lane mostly has one
// set of loads and stores and many tokens are under way (8 waves against 4 and
// 1 for 4096 bf16: 8000 tokens of 4 picks 102, 106 and 125 us, 16 of 8 picks
// 7.2, 8.3 and 20.7; 4000 of 2 picks 35, 30 and 30).  8000 tokens of 4 picks are
// 590 MB, 99 us, 6.0 TB/s.  The products of a lane are added in order of its columns,
// then over the lanes of a wave and the waves of a token in a fixed order.
// WHOLE: columns in whole groups of 8 on 16 bytes; dh is then written past the
// caches.
template <typename T, int W, bool WHOLE, bool GATED>
__global__ __launch_bounds__(W > 4 ? 64 * W : 256) void k_expert_combine_grad(
    const T* __restrict__ dy, const T* __restrict__ h, const int* __restrict__ place, const float* __restrict__ gates,
    int tokens, int top, int rows, int cols, T* __restrict__ dh, float* __restrict__ dg) {
  constexpr int PER = W > 4 ? 1 : 4 / W;  // tokens per workgroup
  __shared__ float part[PER * W][4];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t t = (int64_t)blockIdx.x * PER + wave / W;
  const int w = wave % W;
  const bool live_t = t < tokens;
  const int64_t p0 = t * top;
  const T* dyt = dy + t * cols;
  for (int j0 = 0; j0 < top; j0 += 4) {
    float dot[4] = {0, 0, 0, 0};
    if (live_t) {
      int at[4];
      float g[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const bool in = j0 + q < top;
        // the same for the whole wave: branches on it are scalar
        at[q] = __builtin_amdgcn_readfirstlane(in ? place[p0 + j0 + q] : -1);
        if (at[q] >= rows) at[q] = -1;
        g[q] = GATED && in ? gates[p0 + j0 + q] : 1.0f;
      }
      for (int c = (w * 64 + lane) * 8; c < cols; c += W * 512) {
        const int live = WHOLE ? 8 : cols - c;
        FpWords<T, 8> d, v[4];
        if (live >= 8) fp4_load(dyt + c, d);
        else fp4_load_tail(dyt + c, live, d);
        if (GATED) {
#pragma unroll
          for (int q = 0; q < 4; ++q)
            if (at[q] >= 0) {
              const T* row = h + (int64_t)at[q] * cols + c;
              if (WHOLE) load8_nt(row, v[q]);
              else if (live >= 8) fp4_load(row, v[q]);
              else fp4_load_tail(row, live, v[q]);
            }
        }
        T d8[8];
        __builtin_memcpy(d8, d.w, sizeof(d8));
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          if (at[q] >= 0) {
            float o[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) o[e] = g[q] * ElemT<T>::cvt(d8[e]);
            if (GATED) {
              T v8[8];
              __builtin_memcpy(v8, v[q].w, sizeof(v8));
#pragma unroll
              for (int e = 0; e < 8; ++e)
                dot[q] = __builtin_fmaf(ElemT<T>::cvt(d8[e]), ElemT<T>::cvt(v8[e]), dot[q]);
            }
            if (WHOLE) store8_nt(dh + (int64_t)at[q] * cols + c, o);
            else store8(dh + (int64_t)at[q] * cols + c, live, o);
          }
        }
      }
      if (GATED) {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
#pragma unroll
          for (int s = 32; s > 0; s >>= 1) dot[q] += __shfl_xor(dot[q], s);
          if (at[q] < 0) dot[q] = 0.0f;
        }
      }
    }
    if constexpr (GATED && W == 1) {
      if (live_t && lane == 0) {
#pragma unroll
        for (int q = 0; q < 4; ++q)
          if (j0 + q < top) dg[p0 + j0 + q] = dot[q];
      }
    } else if constexpr (GATED) {
      if (lane == 0) {
#pragma unroll
        for (int q = 0; q < 4; ++q) part[wave][q] = dot[q];
      }
      __syncthreads();
      if (live_t && w == 0 && lane < 4 && j0 + lane < top) {
        float sum = part[wave][lane];
#pragma unroll
        for (int k = 1; k < W; ++k) sum += part[wave + k][lane];
        dg[p0 + j0 + lane] = sum;
      }
      __syncthreads();
    }
  }
}

// Picks per chunk: one chunk (one launch) up to 2048 (2000 picks of 32 experts 6.3
// us; chunks of 1024 and their counts 7.3); above it at most 128 chunks of at least
// 2048 picks, whose counts every workgroup reads (128000 picks of 128 experts 11.7
// us, in chunks of 1024 13.2, of 8192 16.4; 16000 of 256 9.6, 8.6 and 16.5)
static int64_t sort_chunk(int64_t P) {
  if (P <= 2048) return 2048;
  const int64_t c = std::max<int64_t>(2048, ceil_div(P, 128));
  return ceil_div(c, MXK_SORT_THREADS) * MXK_SORT_THREADS;
}

template <typename I>
static int launch_sort(const I* ids, int64_t P, int E, int* order, int* place, int* offsets, int* hist,
                       hipStream_t st) {
  const int64_t chunk = sort_chunk(P), n = std::max<int64_t>(1, ceil_div(P, chunk));
  if (n > 1)
    hipLaunchKernelGGL((k_expert_count<I>), dim3((unsigned)n), dim3(MXK_SORT_THREADS), (E + 1) * sizeof(int), st, ids,
                       (uint32_t)P, (uint32_t)E, (uint32_t)chunk, hist);
  const size_t lds = ((size_t)MXK_SORT_WAVES * (E + 1) + MXK_SORT_WAVES) * sizeof(int);
  hipLaunchKernelGGL((k_expert_place<I>), dim3((unsigned)n), dim3(MXK_SORT_THREADS), lds, st, ids, (uint32_t)P,
                     (uint32_t)E, (uint32_t)chunk, hist, order, place, offsets);
  return check_launch("expert_sort");
}

}  // namespace mxk

using namespace mxk;

extern "C" {

size_t mxk_expert_sort_workspace(int64_t picks, int experts) {
  if (picks <= 0 || experts <= 0) return 0;
  const int64_t n = ceil_div(picks, sort_chunk(picks));
  return n > 1 ? (size_t)n * experts * sizeof(int) : 0;
}

int mxk_expert_sort(const void* ids, int id_bytes, int64_t picks, int experts, int32_t* order, int32_t* place,
                    int32_t* offsets, void* workspace, size_t workspace_nbytes, void* stream) {
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (picks < 0 || picks >= ((int64_t)1 << 31) - 65536)
    return fail(MXK_EINVAL, "expert_sort: 0 <= picks < 2^31 - 2^16");
  // the waves' counters have to fit 64 KiB of LDS
  if (experts < 1 || experts > 1000) return fail(MXK_EINVAL, "expert_sort: 1 to 1000 experts");
  if (id_bytes != 4 && id_bytes != 8) return fail(MXK_EINVAL, "expert_sort: ids of 4 or 8 bytes");
  if (!offsets || (picks > 0 && (!ids || !order || !place))) return fail(MXK_EINVAL, "expert_sort: null pointer");
  const size_t need = mxk_expert_sort_workspace(picks, experts);
  if (need > 0 && (!workspace || workspace_nbytes < need)) return fail(MXK_EINVAL, "expert_sort: workspace too small");
  int* hist = reinterpret_cast<int*>(workspace);
  if (id_bytes == 4)
    return launch_sort(reinterpret_cast<const int32_t*>(ids), picks, experts, order, place, offsets, hist, st);
  return launch_sort(reinterpret_cast<const int64_t*>(ids), picks, experts, order, place, offsets, hist, st);
}

int mxk_expert_gather(const void* x, int elem_bytes, int64_t tokens, int64_t cols, int64_t row_stride,
                      const int32_t* order, int64_t rows, int top, void* out, void* stream) {
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (elem_bytes != 2 && elem_bytes != 4) return fail(MXK_EINVAL, "expert_gather: elements of 2 or 4 bytes");
  if (tokens < 0 || cols < 0 || rows < 0 || top < 1 || row_stride < 0 || rows >= ((int64_t)1 << 31) ||
      tokens >= ((int64_t)1 << 31) || cols >= ((int64_t)1 << 28) || rows > tokens * top)
    return fail(MXK_EINVAL, "expert_gather: bad sizes (rows at most tokens * top, below 2^31; cols below 2^28)");
  if (rows == 0 || cols == 0) return MXK_OK;
  if (!x || !order || !out) return fail(MXK_EINVAL, "expert_gather: null pointer");
  const int64_t row_bytes = cols * elem_bytes;
  const bool whole = row_bytes % 16 == 0 && row_stride * elem_bytes % 16 == 0 && aligned16(x) && aligned16(out);
  // eighths of whole lines
  const int64_t slices = whole && row_bytes % 1024 == 0 ? 8 : 1;
  const int64_t pieces = ceil_div(row_bytes, 16) / slices;
  const int64_t step = std::max<int64_t>(1, ((int64_t)1 << 28) / pieces - 1);
  const DivU32 bt = make_divu32((uint32_t)top), bp = make_divu32((uint32_t)pieces);
  const uint8_t* xp = reinterpret_cast<const uint8_t*>(x);
  for (int64_t r0 = 0; r0 < rows; r0 += step) {
    const uint32_t total = (uint32_t)(std::min(step, rows - r0) * pieces);
    hipLaunchKernelGGL((whole ? k_expert_gather<true> : k_expert_gather<false>),
                       dim3((unsigned)(ceil_div(total, 256) * slices)), dim3(256), 0, st, xp, row_stride * elem_bytes,
                       order + r0, bt, (uint32_t)tokens, total, bp, (uint32_t)pieces, (uint32_t)row_bytes,
                       (uint32_t)slices, reinterpret_cast<uint8_t*>(out) + r0 * row_bytes);
  }
  return check_launch("expert_gather");
}

int mxk_expert_combine(const void* h, int h_type, int64_t rows, const int32_t* place, const float* gates,
                       int64_t tokens, int top, int64_t cols, int y_type, void* y, void* stream) {
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (tokens < 0 || top < 1 || cols < 0 || rows < 0 || rows >= ((int64_t)1 << 31) ||
      tokens >= ((int64_t)1 << 31) || tokens * top >= ((int64_t)1 << 31) || cols >= ((int64_t)1 << 28))
    return fail(MXK_EINVAL, "expert_combine: bad sizes (tokens * top below 2^31, cols below 2^28)");
  if (tokens == 0 || cols == 0) return MXK_OK;
  if ((rows > 0 && !h) || !place || !y) return fail(MXK_EINVAL, "expert_combine: null pointer");
  if (h_type != MXK_IN_F32 && h_type != MXK_IN_F16 && h_type != MXK_IN_BF16)
    return fail(MXK_EINVAL, "expert_combine: unknown h_type");
  if (y_type != h_type && (h_type != MXK_IN_F32 || (y_type != MXK_IN_F16 && y_type != MXK_IN_BF16)))
    return fail(MXK_EINVAL, "expert_combine: y of the rows' type, or any for float32 rows");
  const bool whole = cols % 8 == 0 && aligned16(h) && aligned16(y);
  const int64_t pieces = ceil_div(cols, 8), step = std::max<int64_t>(1, ((int64_t)1 << 31) / pieces - 1);
  const DivU32 bp = make_divu32((uint32_t)pieces);
  for (int64_t t0 = 0; t0 < tokens; t0 += step) {
    const uint32_t total = (uint32_t)(std::min(step, tokens - t0) * pieces);
    const dim3 grid((unsigned)ceil_div(total, 256));
    const int* pl = place + t0 * top;
    const float* gt = gates ? gates + t0 * top : nullptr;
#define MXK_CG(T, O, G)                                                                                             \
  hipLaunchKernelGGL((whole ? k_expert_combine<T, O, G, true> : k_expert_combine<T, O, G, false>), grid, dim3(256), \
                     0, st, hp, pl, gt, top, (int)rows, total, bp, (uint32_t)pieces, (int)cols, yp)
#define MXK_C(T, O)                                                                                               \
  do {                                                                                                            \
    const T* hp = reinterpret_cast<const T*>(h);                                                                  \
    O* yp = reinterpret_cast<O*>(y) + t0 * cols;                                                                  \
    if (gt) MXK_CG(T, O, true);                                                                                   \
    else MXK_CG(T, O, false);                                                                                     \
  } while (0)
    if (h_type == MXK_IN_F16) MXK_C(__half, __half);
    else if (h_type == MXK_IN_BF16) MXK_C(hip_bfloat16, hip_bfloat16);
    else if (y_type == MXK_IN_F16) MXK_C(float, __half);
    else if (y_type == MXK_IN_BF16) MXK_C(float, hip_bfloat16);
    else MXK_C(float, float);
#undef MXK_C
#undef MXK_CG
  }
  return check_launch("expert_combine");
}

int mxk_expert_combine_grad(const void* dy, const void* h, int h_type, int64_t rows, const int32_t* order,
                            const int32_t* place, const float* gates, int64_t tokens, int top, int64_t cols, void* dh,
                            float* dgates, void* stream) {
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (tokens < 0 || top < 1 || cols < 0 || rows < 0 || rows >= ((int64_t)1 << 31) ||
      tokens >= ((int64_t)1 << 31) || tokens * top >= ((int64_t)1 << 31) || cols >= ((int64_t)1 << 28))
    return fail(MXK_EINVAL, "expert_combine_grad: bad sizes (tokens * top below 2^31, cols below 2^28)");
  if (tokens == 0) return MXK_OK;
  if (rows != tokens * top) return fail(MXK_EINVAL, "expert_combine_grad: rows must be tokens * top");
  if (!order || !place || (gates && !dgates) || (cols > 0 && (!dy || !dh || (gates && !h))))
    return fail(MXK_EINVAL, "expert_combine_grad: null pointer");
  if (h_type != MXK_IN_F32 && h_type != MXK_IN_F16 && h_type != MXK_IN_BF16)
    return fail(MXK_EINVAL, "expert_combine_grad: unknown h_type");
  const int64_t waves = ceil_div(cols, 512);
  const bool whole = cols % 8 == 0 && aligned16(dy) && aligned16(h) && aligned16(dh);
  if (cols > 0) {
    const int64_t row_bytes = cols * (h_type == MXK_IN_F32 ? 4 : 2);
    hipLaunchKernelGGL((whole ? k_expert_unnamed<true> : k_expert_unnamed<false>), dim3((unsigned)ceil_div(rows, 32)),
                       dim3(256), 0, st, order, place, (int)rows, row_bytes, reinterpret_cast<uint8_t*>(dh));
  }
#define MXK_GG(T, W, G)                                                                                        \
  hipLaunchKernelGGL((whole ? k_expert_combine_grad<T, W, true, G> : k_expert_combine_grad<T, W, false, G>),   \
                     dim3((unsigned)ceil_div(tokens, W > 4 ? 1 : 4 / W)), dim3(W > 4 ? 64 * W : 256), 0, st,  \
                     reinterpret_cast<const T*>(dy), reinterpret_cast<const T*>(h), place, gates, (int)tokens, \
                     top, (int)rows, (int)cols, reinterpret_cast<T*>(dh), dgates)
#define MXK_GW(T, W)                    \
  do {                                  \
    if (gates) MXK_GG(T, W, true);      \
    else MXK_GG(T, W, false);           \
  } while (0)
#define MXK_G(T)                        \
  do {                                  \
    if (waves <= 1) MXK_GW(T, 1);       \
    else if (waves <= 2) MXK_GW(T, 2);  \
    else if (waves <= 4) MXK_GW(T, 4);  \
    else MXK_GW(T, 8);                  \
  } while (0)
  if (h_type == MXK_IN_F32) MXK_G(float);
  else if (h_type == MXK_IN_F16) MXK_G(__half);
  else MXK_G(hip_bfloat16);
#undef MXK_G
#undef MXK_GW
#undef MXK_GG
  return check_launch("expert_combine_grad");
}

}  // extern "C"
