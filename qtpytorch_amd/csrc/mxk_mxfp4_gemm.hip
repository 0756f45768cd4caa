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
// in front of the first expert's and past the last's are written as zeros; with `order` row r of the
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
  const void* x;             // float rows in place of a (k_fp4_few), x_stride elements apart
  int64_t x_stride;
  int K;
};

// Row of a that row r of the product reads, -1: none
__device__ __forceinline__ int64_t source_row(const Fp4Gemm& p, int64_t r) {
  if (!p.order) return r < p.a_rows ? r : -1;
  const int pick = p.order[r];
  if (pick < 0) return -1;
  const int64_t t = divu32((uint32_t)pick, p.top);
  return t < p.a_rows ? t : -1;
}

// 64 x 64 tiles of four waves (32 x 32 each), operands straight from memory.  For
// what the kernels below do not take: K = 0 (the result is the bias), and
// operands whose offsets pass their 32 bits (tile_of).  4000x4096x4096 takes it 458 us (44).
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


// ---------------------------------------------------------------- tiles through LDS
// What the tile kernel reads in its own order, in one launch (products of few
// stages read scales where they lie instead, tile_of):
//  - scale bytes by stages of 8 blocks (256 values of K): ta[kt][row of the
//    product][8], tb[kt][row of b][8], zeros past KB; 17/16 of a byte moved
//    per 32 values;
//  - by expert, each slot's segment and rows, and the row of a behind each row
//    of the product, which a tile would otherwise look up while nothing else is
//    under way.
// Latency: 5.6 us for 16384 rows of 8192, 7.4 for 32 experts of 4096x2048; four
// rows a lane or a whole row a lane took as long.
struct Fp4Staged {
  uint8_t *ta, *tb;
  int4* slot;  // {expert, first row, end, 0}
  int* row;    // -1: none
};
__global__ __launch_bounds__(256) void k_fp4_stage(Fp4Gemm p, Fp4Staged out, int64_t b_rows, int64_t a_blocks,
                                                   int64_t b_blocks, int64_t slots, int tile) {
  int64_t block = blockIdx.x;
  if (block >= a_blocks + b_blocks) {  // a slot per wave
    const int64_t slot = (block - a_blocks - b_blocks) * 4 + (threadIdx.x >> 6);
    if (slot >= slots) return;
    const Segment s = tile == 256 ? find_segment<256>(slot, p.offsets, p.E, p.M)
                                  : find_segment<128>(slot, p.offsets, p.E, p.M);
    if ((threadIdx.x & 63) == 0) out.slot[slot] = make_int4(s.e, (int)s.lo, (int)s.hi, 0);
    return;
  }
  const bool of_a = block < a_blocks;
  if (!of_a) block -= a_blocks;
  const int64_t rows = of_a ? p.M : b_rows;
  const int64_t r = block * 32 + (threadIdx.x >> 3);
  if (r >= rows) return;
  const int64_t src = of_a ? source_row(p, r) : r;
  if (of_a && p.offsets && (threadIdx.x & 7) == 0) out.row[r] = (int)src;
  const uint8_t* s = (of_a ? p.as : p.bs) + (src < 0 ? 0 : src) * p.KB;
  uint8_t* to = of_a ? out.ta : out.tb;
  for (int64_t k = 8 * (threadIdx.x & 7); k < p.KB; k += 64) {
    uint64_t v = 0;
    if (src >= 0) {
      if (k + 8 <= p.KB) {
        __builtin_memcpy(&v, s + k, 8);
      } else {
        for (int i = 0; i < 8; ++i)
          if (k + i < p.KB) v |= (uint64_t)s[k + i] << (8 * i);
      }
    }
    *reinterpret_cast<uint64_t*>(to + ((k >> 3) * rows + r) * 8) = v;
  }
}

// Raw buffer resource over [p, p + bytes), wave-uniform: loads past the end return 0
__device__ __forceinline__ i32x4 buffer_words(const void* p, uint32_t bytes) {
  const uint64_t a = reinterpret_cast<uint64_t>(p);
  return i32x4{__builtin_amdgcn_readfirstlane((int)(uint32_t)a),
               __builtin_amdgcn_readfirstlane((int)(uint32_t)(a >> 32) & 0xFFFF),
               __builtin_amdgcn_readfirstlane((int)bytes), 0x00020000};
}
// 16 bytes per lane from a buffer into LDS at `lds` + 16 * lane.  In
// assembly, so that the compiler does not order the tile's LDS reads behind
// loads of the other buffer; the kernel waits for them itself (wait_loads).
// A load into LDS needs one wait state behind the write of m0, which the
// hardware does not insert, nor the compiler within assembly: the s_nop.  The
// build checks it on the result (check_lds_loads.py).
__device__ __forceinline__ void load_to_lds(i32x4 r, uint32_t off, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
               :
               : "s"(lds), "v"(off), "s"(r)
               : "memory");
}
// The scales of R rows, 8 bytes each, by one instruction of the wave
template <int R>
__device__ __forceinline__ void load_scales_to_lds(i32x4 r, int lane, uint32_t lds) {
  if constexpr (R == 128) {
    load_to_lds(r, 16u * lane, lds);
  } else {
    static_assert(R == 64, "16 or 8 bytes per lane");
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dword %1, %2, 0 offen lds\n\t"
                 "s_mov_b32 m0, %3\n\ts_nop 0\n\tbuffer_load_dword %4, %2, 0 offen lds"
                 :
                 : "s"(lds), "v"(4u * lane), "s"(r), "s"(lds + 256u), "v"(4u * lane + 256u)
                 : "memory");
  }
}
template <int N>
__device__ __forceinline__ void wait_loads() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" : : "i"(N) : "memory");
}

// wait_loads<N> where `counted`, else wait_loads<0>; the choice is made inside
// the assembly, which keeps the compiler from doubling the loop around it
template <int N>
__device__ __forceinline__ void wait_loads_if(uint32_t counted) {
  asm volatile("s_cmp_eq_u32 %0, 0\n\ts_cbranch_scc1 1f\n\ts_waitcnt vmcnt(%1) lgkmcnt(0)\n\ts_branch 2f\n"
               "1:\ts_waitcnt vmcnt(0) lgkmcnt(0)\n2:"
               :
               : "s"(__builtin_amdgcn_readfirstlane(counted)), "i"(N)
               : "memory", "scc");
}

#define MXK_FAR_ROW 0x80000000u   // offset of a row that is not there: past every buffer (at most 2^30 bytes)
#define MXK_FAR_BLOCK 0x40000000u // added for blocks past KB

// Tiles of (2 * 32 * F)^2, four waves of F x F fragments of 32 x 32, stages
// of 256 values of K (128 bytes a row) in two LDS buffers.
//
// v_mfma_scale_f32_32x32x64_f8f6f4: lane l holds row l % 32 and one of the two
// blocks of a step; the four steps of a stage give lane half h the blocks
// 4h .. 4h+3, so one dword per row holds its four scale bytes and a step
// selects its byte.  (Any order of K is right as long as both operands share it.)
//
// LDS rows are 128 bytes, half of the banks: 16-byte chunk c of row r sits at
// c ^ (r & 7) ^ (r >> 3 & 7), so that 16 lanes of consecutive rows read all
// banks once (with c ^ (r & 7) rows r and r + 8 meet).  The loads write LDS in
// lane order, so the lane picks the chunk that belongs at its place.
//
// The barrier of a stage sits before its last step: by then the next stage
// has landed and this stage's last fragments are in registers, so the loads of the
// stage after next go into the buffer just read, and the next stage's first
// fragments are read while the last step multiplies.
//
// A workgroup takes tile after tile.  Its next tile's place (and, by expert,
// its rows) is looked up before the products of this one, and that tile's first
// two stages are requested between the stores of this one's result.  The
// stores are not hidden behind its products, though: the compiler waits for all of
// vector memory in front of a tile's first MFMA, where the sums start from a
// bias that may be there or not, and by expert for the look-up's loads too.
//
// What an instruction loads and reads stands between single MFMAs, in their
// shadow: in front of rows of four it took 5% longer.
//
// Bound by the matrix unit, whose rate falls with what the operands hold: this
// instruction alone on random codes in registers 6.4 PFLOP/s, on zeros 9.1.
// 8192x8192x8192 255 to 299 us (4.3 to 3.7 PFLOP/s; MFMAs 59% of the cycles,
// waits 20%), 4000x4096x4096 43 us (3.1; MFMAs 45%, waits 30%), 16000 rows over
// 32 experts of 4096x2048 116 us (2.3; MFMAs 35%, waits 26%: of a tile's
// cycles its eight stages take some 29000, the stores of all CUs at once 11000).
// 1500x1800x2080, one tile of 9 stages on 180 CUs, 13.9 us: MFMAs 11%, waits 48%.
template <typename T, int F, bool EXPERT, bool STAGED>
__global__ __launch_bounds__(256, 1) void k_fp4_gemm_tile(Fp4Gemm p, Fp4Staged in, int64_t b_rows, uint32_t tm,
                                                          uint32_t tn, uint32_t splits, uint32_t ids) {
  constexpr int B = 64 * F;                 // rows of a tile
  constexpr int OP = B * 128, SC = B * 8;   // bytes of an operand's stage and of its scales
  constexpr int BUF = 2 * OP, SBUF = 2 * SC;
  constexpr int LI = B / 32;                // load instructions per wave, operand and stage
  // scales in stage order by k_fp4_stage, or each thread brings its row's of a stage
  static_assert(STAGED || (F == 2 && !EXPERT), "rows of a and b as threads");
  constexpr int LOADS = 2 * LI + (STAGED && F == 2 ? 2 : 1);  // all of a wave and stage
  constexpr int NW = 32 * F;                // columns of a wave
  constexpr int CB = F == 4 ? 128 : 64;     // bytes of a row that the result passes through LDS at once
  constexpr int CH = CB / 16, CC = CB / (int)sizeof(T), PASS = NW / CC;
  // passes of the result, each with CH / 2 stores; every STEP of them one of
  // the 2 F parts of the next tile's first two stages
  constexpr int PASSES = F * PASS, STEP = PASSES / (2 * F);
  // memory operations of a wave complete in order: what may be due behind the
  // last load of stage 0 (the stores from its pass on and stage 1), of stage 1.
  // They are right by themselves; the compiler's own wait of today, which comes
  // behind the first, leaves nothing due at the second.
  constexpr int BEHIND0 = LOADS + (PASSES - (F - 1) * STEP) * (CH / 2);
  constexpr int BEHIND1 = (PASSES - (2 * F - 1) * STEP) * (CH / 2);
  static_assert(STEP >= 1 && BEHIND0 <= 63, "a part for every pass, counts that the wait can hold");
  __shared__ __align__(16) uint8_t lds[2 * BUF + 2 * SBUF + 4 * 32 * CB];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r32 = lane & 31, h = lane >> 5;
  const uint32_t row_bytes = (uint32_t)p.KB * 16u;
  const uint32_t KB = (uint32_t)p.KB, stages = (KB + 7u) >> 3;
  // whole 16-byte pieces of y: stores by buffer, as many for every tile
  const bool whole = p.N * (int)sizeof(T) % 16 == 0 && (reinterpret_cast<uintptr_t>(p.y) & 15u) == 0;

  // a tile: rows lo .. hi of the product, columns from n0, stages from .. to
  struct Tile {
    int lo, hi, e;
    int64_t n0;
    uint32_t from, to;
    T* y;
  };
  Tile cur = {}, next = {};
  // loads of this wave: rows (wave * LI + i) * 8 + lane / 8 of either operand,
  // chunk (lane & 7) ^ (lane / 8) ^ (wave * LI + i & 7) of the stage
  const int lr = lane >> 3, chunk = (lane & 7) ^ lr;
  const int flip = wave * LI & 7;
  const uint32_t off0 = (uint32_t)(wave * LI * 8 + lr) * row_bytes, step8 = 8u * row_bytes;
  i32x4 ra, rb;
  uint32_t off_a[EXPERT ? LI : 1];  // by expert: of any rows
  int src[EXPERT ? LI : 1];         // those of the next tile
  // not STAGED: this thread's row of scales, the bytes from there to the last
  // eight of all, and the stage's bytes that are on the way (of a tile's first
  // stage in sc0).  Eight bytes are read wherever they are there; those of other
  // rows and stages are taken out at their use.
  const uint8_t* srow = nullptr;
  int room = 0;
  uint64_t sc = 0, sc0 = 0;
  auto put_scales = [&](uint32_t t, uint32_t buf, uint64_t v) {
    const int past = 8 * (int)t - room;  // 8 or more only where no block is left
    const uint32_t live = KB > 8u * t ? KB - 8u * t : 0u;
    const uint64_t mask = live >= 8u ? ~0ull : (1ull << (8u * live)) - 1u;
    *reinterpret_cast<uint64_t*>(lds + 2 * BUF + buf * SBUF + threadIdx.x * 8u) =
        (v >> (8 * (past > 0 ? past & 7 : 0))) & mask;
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  };

  // the next tile from `id` on that has products (rows without an expert are
  // written here): true, or false at the end
  auto look_ahead = [&](uint32_t& id) -> bool {
    for (; id < ids; id += gridDim.x) {
      uint32_t mt, nt;
      next.from = 0;
      next.to = stages;
      next.y = reinterpret_cast<T*>(p.y);
      if constexpr (EXPERT) {
        if (!place_block_tile(id, tm, tn, mt, nt)) continue;
        next.n0 = (int64_t)nt * B;
        const int4 s = in.slot[mt];
        next.e = __builtin_amdgcn_readfirstlane(s.x);
        next.lo = __builtin_amdgcn_readfirstlane(s.y);
        next.hi = __builtin_amdgcn_readfirstlane(s.z);
        if (next.e > p.E) continue;
        if (next.e == p.E) {
          const int64_t w = p.N - next.n0 < B ? p.N - next.n0 : B;
          for (int64_t r = next.lo + wave; r < next.hi; r += 4)
            for (int64_t c = lane; c < w; c += 64) next.y[r * p.N + next.n0 + c] = from_f32<T>(0.0f);
          continue;
        }
#pragma unroll
        for (int i = 0; i < LI; ++i) {
          const int r = next.lo + (wave * LI + i) * 8 + lr;
          src[i] = in.row[r < next.hi ? r : next.hi - 1];
        }
      } else {
        place_tile(id, tm, tn * splits, mt, nt);
        if (splits > 1) {
          const uint32_t part = nt % splits;
          nt /= splits;
          next.from = part * stages / splits;
          next.to = (part + 1u) * stages / splits;
          next.y += (int64_t)part * p.M * p.N;
        }
        next.n0 = (int64_t)nt * B;
        next.lo = (int)mt * B;
        next.hi = p.M < (int64_t)next.lo + B ? (int)p.M : next.lo + B;
      }
      return true;
    }
    return false;
  };
  // that tile is the one to load now
  auto advance = [&]() {
    cur = next;
    const int64_t rows_b = p.N - cur.n0 < B ? p.N - cur.n0 : B;
    rb = buffer_words(p.b + ((int64_t)cur.e * p.N + cur.n0) * row_bytes, (uint32_t)(rows_b * row_bytes));
    if constexpr (EXPERT) {
      // with an order, rows of all of a; without, of this tile's part of it
      const bool picked = p.order != nullptr;
      ra = buffer_words(picked ? p.a : p.a + cur.lo * (int64_t)row_bytes,
                        (uint32_t)(picked ? p.a_rows : (int64_t)(cur.hi - cur.lo)) * row_bytes);
#pragma unroll
      for (int i = 0; i < LI; ++i)
        off_a[i] = src[i] < 0 ? MXK_FAR_ROW : (uint32_t)(src[i] - (picked ? 0 : cur.lo)) * row_bytes;
    } else {
      ra = buffer_words(p.a + cur.lo * (int64_t)row_bytes, (uint32_t)(cur.hi - cur.lo) * row_bytes);
      if constexpr (!STAGED) {
        const bool of_b = threadIdx.x >= B;
        const int64_t row = (of_b ? cur.n0 : cur.lo) + (threadIdx.x & (B - 1)), rows = of_b ? p.N : p.M;
        const int64_t first = (row < rows ? row : rows - 1) * KB, last = rows * KB - 8 - first;
        srow = (of_b ? p.bs : p.as) + first;
        room = (int)(last < (1 << 24) ? last : (1 << 24));  // a row has at most 2^18 blocks
      }
    }
  };
  // load k of 2 LI of a stage's codes: of a and b in turn
  auto issue_load = [&](uint32_t t, uint32_t buf, int k) {
    const int i = k >> 1;
    const uint32_t blk = 8u * t + (chunk ^ flip ^ i);
    const uint32_t ok = blk < KB && t < cur.to ? blk * 16u : MXK_FAR_BLOCK;
    if (k & 1) load_to_lds(rb, off0 + i * step8 + ok, buf * BUF + OP + (wave * LI + i) * 1024u);
    else load_to_lds(ra, (EXPERT ? off_a[EXPERT ? i : 0] : off0 + i * step8) + ok, buf * BUF + (wave * LI + i) * 1024u);
  };
  // its scales: planes of [rows][8] bytes, B / 128 kilobytes an operand; waves 0, 1
  // take a's, 2, 3 b's (F = 2: each wave half a kilobyte, the upper lanes nothing)
  auto issue_scales = [&](uint32_t t, uint32_t buf, uint64_t& by_thread) {
    if (!STAGED) {
      __builtin_memcpy(&by_thread, srow + min(8 * (int)t, room), 8);
    } else {
      constexpr int R = B / 2;  // rows per wave
      const bool of_b = wave >= 2;
      const int64_t rows = of_b ? b_rows : p.M;
      const int64_t first = (of_b ? (int64_t)cur.e * p.N + cur.n0 : cur.lo) + R * (wave & 1);
      // past the last row: bytes of the next plane or of the kilobytes kept after the
      // last, for rows whose codes are zeros or whose results are not stored
      const i32x4 rs =
          buffer_words((of_b ? in.tb : in.ta) + ((int64_t)t * rows + first) * 8, t < cur.to ? R * 8u : 0u);
      load_scales_to_lds<R>(rs, lane, 2u * BUF + buf * SBUF + (of_b ? SC : 0) + R * 8u * (wave & 1));
    }
  };
  // part q of F of the loads of a stage
  auto issue = [&](uint32_t t, uint32_t buf, int q, uint64_t& by_thread) {
#pragma unroll
    for (int k = q * 2 * LI / F; k < (q + 1) * 2 * LI / F; ++k) issue_load(t, buf, k);
    if (q == F - 1) issue_scales(t, buf, by_thread);
  };

  // fragment reads: rows of this wave's half of a (wave / 2) and of b (wave % 2)
  const uint32_t rd_a = (uint32_t)((wave >> 1) * 32 * F + r32) * 128u;
  const uint32_t rd_b = OP + (uint32_t)((wave & 1) * 32 * F + r32) * 128u;
  uint32_t at[4];
#pragma unroll
  for (int s = 0; s < 4; ++s) at[s] = (uint32_t)((4 * h + s) ^ (lane & 7) ^ (r32 >> 3)) * 16u;
  const uint32_t rs_a = 2 * BUF + ((wave >> 1) * 32 * F + r32) * 8 + 4 * h;
  const uint32_t rs_b = 2 * BUF + SC + ((wave & 1) * 32 * F + r32) * 8 + 4 * h;

  f32x16 acc[F][F];  // [b fragment][a fragment]: rows of the result are n
  i32x4 fa[2][F], fb[2][F];
  int sa[2][F], sb[2][F];
  auto read_frag = [&](uint32_t buf, int s, int i, i32x4 (&xa)[F], i32x4 (&xb)[F]) {
    const uint32_t c = at[s] ^ (i & 1 ? 64u : 0u);  // rows 32 i: bit 2 of r >> 3
    xa[i] = *reinterpret_cast<const i32x4*>(lds + buf * BUF + rd_a + c + i * 4096);
    xb[i] = *reinterpret_cast<const i32x4*>(lds + buf * BUF + rd_b + c + i * 4096);
  };
  auto read_scale = [&](uint32_t buf, int i, int (&xa)[F], int (&xb)[F]) {
    xa[i] = *reinterpret_cast<const int*>(lds + buf * SBUF + rs_a + i * 256);
    xb[i] = *reinterpret_cast<const int*>(lds + buf * SBUF + rs_b + i * 256);
  };
  // One step: F x F MFMAs, before each what `between` issues there, which fits
  // into the shadow of the one before
#define MXK_STEP(SEL, XA, XB, BETWEEN)                                                                       \
  _Pragma("unroll") for (int i = 0; i < F; ++i) {                                                           \
    _Pragma("unroll") for (int j = 0; j < F; ++j) {                                                         \
      BETWEEN;                                                                                              \
      __builtin_amdgcn_sched_barrier(0);                                                                    \
      const i32x8 va = {XA[j][0], XA[j][1], XA[j][2], XA[j][3], 0, 0, 0, 0};                                \
      const i32x8 vb = {XB[i][0], XB[i][1], XB[i][2], XB[i][3], 0, 0, 0, 0};                                \
      acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(vb, va, acc[i][j], 4, 4, SEL, sb[0][i],   \
                                                                  SEL, sa[0][j]);                           \
      __builtin_amdgcn_sched_barrier(0);                                                                    \
    }                                                                                                       \
  }

  uint32_t id = blockIdx.x;
  if (!look_ahead(id)) return;
  advance();
#pragma unroll
  for (int q = 0; q < 2 * F; ++q) issue(cur.from + q / F, q / F, q % F, q < F ? sc0 : sc);
  uint32_t behind = 0;  // whether stores are due behind and between this tile's first loads
  for (;;) {
    // sums start from the bias, which every row of a fragment shares
#pragma unroll
    for (int i = 0; i < F; ++i) {
      float b[16];
#pragma unroll
      for (int q = 0; q < 16; ++q) b[q] = 0.0f;
      if (p.bias) {
        const int64_t n = cur.n0 + (wave & 1) * NW + 32 * i + 4 * h;
#pragma unroll
        for (int q = 0; q < 16; ++q) {
          const int64_t at = n + 8 * (q >> 2) + (q & 3);
          b[q] = p.bias[(int64_t)cur.e * p.N + (at < p.N ? at : p.N - 1)];
        }
      }
#pragma unroll
      for (int j = 0; j < F; ++j)
#pragma unroll
        for (int q = 0; q < 16; ++q) acc[i][j][q] = b[q];
    }
    if (behind) wait_loads<BEHIND0>();
    else wait_loads<LOADS>();
    if constexpr (!STAGED) put_scales(cur.from, 0, sc0);
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
#pragma unroll
    for (int i = 0; i < F; ++i) {
      read_scale(0, i, sa[0], sb[0]);
      read_frag(0, 0, i, fa[0], fb[0]);
    }
    id += gridDim.x;
    const bool more = look_ahead(id);
    // past the last stage the loads bring zeros and the reads are not used
    uint32_t buf = 0;
    for (uint32_t t = cur.from; t < cur.to; ++t) {
      MXK_STEP(0, fa[0], fb[0], if (j == 0) read_frag(buf, 1, i, fa[1], fb[1]))
      MXK_STEP(1, fa[1], fb[1], if (j == 0) read_frag(buf, 2, i, fa[0], fb[0]))
      MXK_STEP(2, fa[0], fb[0], if (j == 0) read_frag(buf, 3, i, fa[1], fb[1]))
      wait_loads_if<BEHIND1>(t == cur.from ? behind : 0u);
      if constexpr (!STAGED) put_scales(t + 1, buf ^ 1u, sc);
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
      buf ^= 1u;
      MXK_STEP(3, fa[1], fb[1], {
        if (j == 0) read_frag(buf, 0, i, fa[0], fb[0]);
        if (j == 1) read_scale(buf, i, sa[1], sb[1]);
        // 2 LI loads over F x F MFMAs
        _Pragma("unroll") for (int k = (i * F + j) * 2 * LI / (F * F); k < (i * F + j + 1) * 2 * LI / (F * F); ++k)
            issue_load(t + 2, buf ^ 1u, k);
        if (i == F - 1 && j == F - 1) issue_scales(t + 2, buf ^ 1u, sc);
      })
#pragma unroll
      for (int i = 0; i < F; ++i) {
        sa[0][i] = sa[1][i];
        sb[0][i] = sb[1][i];
      }
    }
    wait_loads<0>();
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");

    // The result through LDS, 32 rows of m and CB bytes of n at a time and
    // wave: a lane holds four consecutive n of one m; whole 64- or 128-byte
    // pieces of rows leave in 16-byte stores.
    uint8_t* mine = lds + 2 * BUF + 2 * SBUF + wave * 32 * CB;
    const int64_t nw = cur.n0 + (wave & 1) * NW, mw = cur.lo + (wave >> 1) * NW, m1 = cur.hi;
    T* const y = cur.y;
    if (more) advance();
    // the sums stay where they are until here: read earlier, they would push the loads' addresses into scratch
#pragma unroll
    for (int i = 0; i < F; ++i)
#pragma unroll
      for (int j = 0; j < F; ++j) asm volatile("" : "+a"(acc[i][j]));
    // a buffer over this wave's rows; its offsets stay below 2^31 (N checked on the host)
    const int64_t left = m1 - mw;
    const uint32_t pitch = (uint32_t)p.N * (uint32_t)sizeof(T);
    const __amdgpu_buffer_rsrc_t ry =
        make_rsrc(y + mw * p.N, left <= 0 ? 0u : (uint32_t)(left < NW ? left : NW) * pitch);
    uint32_t el = (uint32_t)lane;
    asm volatile("" : "+v"(el));  // the addresses below are not worth registers during the products
    const uint32_t col = (uint32_t)nw * (uint32_t)sizeof(T) + (el % CH) * 16u, out0 = (el / CH) * pitch + col;
    uint8_t* put = mine + (el & 31u) * CB;
#pragma unroll
    for (int j = 0; j < F; ++j)
#pragma unroll
      for (int s = 0; s < PASS; ++s) {
        const int part = (j * PASS + s) / STEP;
        if (more && (j * PASS + s) % STEP == 0 && part < 2 * F) 
          issue(cur.from + part / F, part / F, part % F, part < F ? sc0 : sc);
#pragma unroll
        for (int u = 0; u < CC / 8; ++u) {
          const int iq = s * (CC / 8) + u, i = iq >> 2, q = iq & 3;
          T t[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) t[k] = from_f32<T>(acc[i][j][4 * q + k]);
          const uint32_t byte = (8 * u + 4 * (el >> 5)) * (uint32_t)sizeof(T);
          uint8_t* d = put + (((byte >> 4) ^ (el & (CH - 1))) << 4) + (byte & 15);
          __builtin_memcpy(__builtin_assume_aligned(d, 4 * sizeof(T)), t, sizeof(t));
        }
        __builtin_amdgcn_wave_barrier();
        u32x4 v[CH / 2];
#pragma unroll
        for (int k = 0; k < CH / 2; ++k) {
          const uint32_t row = k * (64 / CH) + el / CH, ch = el % CH;
          v[k] = *reinterpret_cast<const u32x4*>(mine + row * CB + ((ch ^ (row & (CH - 1))) << 4));
        }
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int k = 0; k < CH / 2; ++k) {
          if (whole) {
            const uint32_t o = col + s * CB < pitch ? out0 + (32 * j + k * (64 / CH)) * pitch + s * CB : 0x80000000u;
            __builtin_amdgcn_raw_buffer_store_b128(v[k], ry, (int)o, 0, 0);
          } else if (const uint32_t row = 32 * j + k * (64 / CH) + el / CH; mw + row < m1) {
            const int64_t n = nw + s * CC + (el % CH) * (16 / sizeof(T));
            T t[16 / sizeof(T)];
            __builtin_memcpy(t, &v[k], 16);
#pragma unroll
            for (int q = 0; q < 16 / (int)sizeof(T); ++q)
              if (n + q < p.N) y[(mw + row) * p.N + n + q] = t[q];
          }
        }
      }
    if (!more) return;
    behind = whole ? 1u : 0u;
  }
#undef MXK_STEP
}

// ---------------------------------------------------------------- few rows
// 16 * MT rows of a by NT tiles of 16 rows of b per workgroup, K shared out
// over its waves in chunks of 512 and the waves' sums added through LDS in
// their order.
//
// Bound by HBM (17/32 byte per weight, each read once): 16x8192x8192 with x in
// bf16 11.2 us, packed 9.6 (3.8 TB/s of weights), 8 tokens to 4 of 32 experts
// of 4096x4096 29 us (5.6 TB/s of the busy experts').  A wave requests its
// chunk of a tile of b, 256 bytes a row, straight into LDS of its own, in
// whole lines (lanes of an MFMA operand lie in different rows: read in that
// order, each lane's 16 bytes would be a request by itself, 64 a wave
// instruction), then reads it as v_mfma_scale_f32_16x16x128 wants it: lane l
// row l % 16, block 4 s + l / 16 of step s.  16-byte chunk c of row r sits at
// c ^ r.  The next tile is on its way while one is multiplied.
//
// Float rows of x (MT = 1) are packed while the first tiles of b travel: the
// loads of x come first, 4 lanes to a block and 4 registers to 4 rows; the
// lanes share the block's largest magnitude, and a 4 x 4 transpose between
// those lanes and registers (8 VALU) leaves each lane with one whole block of
// its own row.
template <typename X> struct IsPacked { static constexpr bool V = false; };
template <> struct IsPacked<uint8_t> { static constexpr bool V = true; };

template <typename X, typename T, int MT, int NT, bool EXPERT>
__global__ __launch_bounds__(MT > 2 ? 512 : 1024) void k_fp4_few(Fp4Gemm p) {
  constexpr bool PACKED = IsPacked<X>::V;
  constexpr int OWN = NT > 1 ? 8192 : 4096;           // bytes of LDS of a wave: two tiles, or the only one
  extern __shared__ __align__(16) uint8_t few_lds[];  // then the sums: [waves][MT * NT][64][4] floats
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
  const int r = lane & 15, g = lane >> 4;
  const int64_t tiles_n = (p.N + 16 * NT - 1) / (16 * NT);
  const int64_t slot = blockIdx.x / tiles_n, n0 = (blockIdx.x - slot * tiles_n) * (16 * NT);
  int64_t lo = slot * 16 * MT, hi = p.M < lo + 16 * MT ? p.M : lo + 16 * MT;
  int e = 0;
  if (EXPERT) {
    const Segment sg = find_segment<16 * MT>(slot, p.offsets, p.E, p.M);
    e = sg.e;
    lo = sg.lo;
    hi = sg.hi;
    if (e > p.E) return;
  }
  T* y = reinterpret_cast<T*>(p.y);
  if (EXPERT && e == p.E) {
    for (int i = threadIdx.x; i < (int)(hi - lo) * 16 * NT; i += blockDim.x) {
      const int64_t n = n0 + i % (16 * NT);
      if (n < p.N) y[(lo + i / (16 * NT)) * p.N + n] = from_f32<T>(0.0f);
    }
    return;
  }
  const int KB = (int)p.KB, chunks = (KB + 15) >> 4;
  const uint32_t row_bytes = (uint32_t)KB * 16u;
  const int64_t rows_b = p.N - n0 < 16 * NT ? p.N - n0 : 16 * NT;
  const __amdgpu_buffer_rsrc_t rb =
      make_rsrc(p.b + ((int64_t)e * p.N + n0) * row_bytes, (uint32_t)rows_b * row_bytes);
  uint8_t* own = few_lds + wave * OWN;
  // tile i of b into LDS: 4 rows an instruction; row 4 k + lane / 16 has its chunk (lane % 16) ^ row at lane % 16
  auto fetch_b = [&](int chunk, int i) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int row = 4 * k + g, c = r ^ row;
      const uint32_t blk = 16u * chunk + c;
      const uint32_t off = (uint32_t)(16 * i + row) * row_bytes + (blk < (uint32_t)KB ? blk * 16u : MXK_FAR_BLOCK);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          rb, (__attribute__((address_space(3))) void*)(own + 4096 * (i & 1) + 1024 * k), 16, (int)off, 0, 0, 2);
    }
  };
  // a row's 16 scale bytes of a chunk; of them this lane's four, byte s that of step s
  auto load_scales = [&](const uint8_t* row, int chunk, uint32_t (&w)[4]) {
    if (16 * chunk + 16 <= KB) {
      __builtin_memcpy(w, row + 16 * chunk, 16);
    } else {
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        w[s] = 0;
        if (16 * chunk + 4 * s + g < KB) w[s] = (uint32_t)row[16 * chunk + 4 * s + g] << (8 * g);
      }
    }
  };
  auto pick_scales = [&](const uint32_t (&w)[4]) -> uint32_t {
    const uint32_t sel = 0x0C0C0000u | (uint32_t)((4 + g) << 8) | (uint32_t)g;
    return __builtin_amdgcn_perm(w[1], w[0], sel) | (__builtin_amdgcn_perm(w[3], w[2], sel) << 16);
  };
  f32x4f acc[MT][NT];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) acc[i][j] = f32x4f{0, 0, 0, 0};
  // this lane's row of scales of tile i (columns past N are not stored)
  auto scales_of = [&](int i) -> const uint8_t* {
    const int64_t n = n0 + 16 * i + r;
    return p.bs + ((int64_t)e * p.N + (n < p.N ? n : p.N - 1)) * KB;
  };
  uint32_t bw[2][4];
  // requests of a tile: in whole chunks one load of scales, then 4 into LDS, in
  // that order, which the waits below count on
  auto request = [&](int chunk, int i) {
    load_scales(scales_of(i), chunk, bw[i & 1]);
    asm volatile("" ::: "memory");
    fetch_b(chunk, i);
    asm volatile("" ::: "memory");
  };
  // the products of a chunk, once its first two tiles are requested
  auto multiply = [&](int chunk, const u32x4 (&xc)[MT][4], const uint32_t (&xs)[MT]) {
    const bool full = 16 * chunk + 16 <= KB;
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      // tile i is in LDS when only tile i + 1's requests are due (the
      // compiler does not know of that dependence)
      if (i + 1 < NT && full) wait_loads<5>();
      else wait_loads<0>();
      const uint8_t* tile = own + 4096 * (i & 1) + r * 256;
      const int sb = (int)pick_scales(bw[i & 1]);
      i32x8 vb[4];
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        const i32x4 w = *reinterpret_cast<const i32x4*>(tile + (((4 * s + g) ^ r) << 4));
        vb[s] = i32x8{w[0], w[1], w[2], w[3], 0, 0, 0, 0};
      }
#define MXK_FEW(S)                                                                                               \
  _Pragma("unroll") for (int m = 0; m < MT; ++m) {                                                              \
    const i32x8 va = {(int)xc[m][S][0], (int)xc[m][S][1], (int)xc[m][S][2], (int)xc[m][S][3], 0, 0, 0, 0};      \
    acc[m][i] =                                                                                                 \
        __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(vb[S], va, acc[m][i], 4, 4, S, sb, S, (int)xs[m]);     \
  }
      MXK_FEW(0)
      MXK_FEW(1)
      MXK_FEW(2)
      MXK_FEW(3)
#undef MXK_FEW
      if (i + 2 < NT) {
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // tile i has been read
        request(chunk, i + 2);
      }
    }
  };
  if constexpr (PACKED) {
    const uint8_t *ap[MT], *asp[MT];
    bool al[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      const int64_t m = lo + 16 * i + r;
      const int64_t src = m < hi ? source_row(p, m) : -1;
      al[i] = src >= 0;
      ap[i] = p.a + (al[i] ? src : 0) * p.KB * 16;
      asp[i] = p.as + (al[i] ? src : 0) * p.KB;
    }
    for (int chunk = wave; chunk < chunks; chunk += waves) {
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the chunk before has been read
      uint32_t xs[MT], xw[MT][4];
      u32x4 xc[MT][4];
#pragma unroll
      for (int i = 0; i < MT; ++i) {
#pragma unroll
        for (int s = 0; s < 4; ++s) {
          xw[i][s] = 0;
          xc[i][s] = u32x4{0u, 0u, 0u, 0u};
        }
        if (al[i]) {
          load_scales(asp[i], chunk, xw[i]);
#pragma unroll
          for (int s = 0; s < 4; ++s) {
            const int blk = 16 * chunk + 4 * s + g;
            if (blk < KB) xc[i][s] = *reinterpret_cast<const u32x4*>(ap[i] + (int64_t)blk * 16);
          }
        }
      }
      request(chunk, 0);
      if (NT > 1) request(chunk, 1);
#pragma unroll
      for (int i = 0; i < MT; ++i) xs[i] = pick_scales(xw[i]);
      multiply(chunk, xc, xs);
    }
  } else {
    static_assert(MT == 1, "float rows: one tile");
    // rows 4 (lane / 4 % 4) + k of x, k = 0 .. 3, as a buffer (the host keeps x below
    // 2^31 bytes): a row that is not there lies past its end and reads as zeros
    const __amdgpu_buffer_rsrc_t rx =
        make_rsrc(p.x, (uint32_t)(((p.a_rows - 1) * p.x_stride + p.K) * (int)sizeof(X)));
    uint32_t x_off[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int64_t m = lo + (r & 12) + k;
      const int64_t src = m < hi ? source_row(p, m) : -1;
      x_off[k] = src >= 0 ? (uint32_t)(src * p.x_stride * (int)sizeof(X)) : MXK_FAR_ROW;
    }
    constexpr int W = (int)sizeof(X) * 2 / 4;  // 16-byte loads of 8 elements
    constexpr int AT = sizeof(X) == 4 ? 1 : 4; // steps whose elements are in registers at once
    const bool odd = lane & 1, high = lane & 2;
    for (int chunk = wave; chunk < chunks; chunk += waves) {
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      uint32_t xs[1] = {0};
      u32x4 xc[1][4];
#pragma unroll
      for (int s0 = 0; s0 < 4; s0 += AT) {
        FpWords<X, 8> v[AT][4];  // of step s0 + t, row (r & 12) + k: elements 8 (r & 3) .. + 7 of block g
        const int c0 = 512 * chunk + 128 * s0 + 32 * g + 8 * (r & 3);
#pragma unroll
        for (int t = 0; t < AT; ++t)
#pragma unroll
          for (int k = 0; k < 4; ++k)
#pragma unroll
            for (int q = 0; q < W; ++q) {
              const u32x4 w4 = buf_load_b128(rx, x_off[k] + (uint32_t)(c0 + 128 * t) * (uint32_t)sizeof(X) + 16u * q, 0);
              __builtin_memcpy(&v[t][k].w[4 * q], &w4, 16);
            }
        if (s0 + AT >= 4) {  // behind the last loads of x, which are waited for alone
          __builtin_amdgcn_sched_barrier(0);
          request(chunk, 0);
          if (NT > 1) request(chunk, 1);
          __builtin_amdgcn_sched_barrier(0);
        }
        if (512 * chunk + 512 > p.K) {  // the elements past the end of a row are the next one's: whole dwords of zeros
#pragma unroll
          for (int t = 0; t < AT; ++t)
#pragma unroll
            for (int q = 0; q < 4 * W; ++q) {
              const bool in = c0 + 128 * t + q * 4 / (int)sizeof(X) < p.K;
#pragma unroll
              for (int k = 0; k < 4; ++k) v[t][k].w[q] = in ? v[t][k].w[q] : 0u;
            }
        }
#pragma unroll
        for (int t = 0; t < AT; ++t) {
          uint32_t a[4], byte[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            byte[k] = fp4_scale_byte(group_max_u<4>(fp4_amax_bits(v[t][k])));
            uint32_t q[1];
            fp4_codes(v[t][k], e8m0_operand(byte[k]), q);
            a[k] = byte[k] == 255u ? 0u : q[0];
          }
          // out[d] of lane k = a[k] of lane d (lanes of four), one bit of the two at a time
#define MXK_SWAP(A, B, CTRL, UP)                                                        \
  {                                                                                     \
    const uint32_t x = (uint32_t)__builtin_amdgcn_mov_dpp((int)B, CTRL, 0xF, 0xF, true); \
    const uint32_t z = (uint32_t)__builtin_amdgcn_mov_dpp((int)A, CTRL, 0xF, 0xF, true); \
    A = UP ? x : A;                                                                     \
    B = UP ? B : z;                                                                     \
  }
          MXK_SWAP(a[0], a[1], 0xB1, odd)
          MXK_SWAP(a[2], a[3], 0xB1, odd)
          MXK_SWAP(a[0], a[2], 0x4E, high)
          MXK_SWAP(a[1], a[3], 0x4E, high)
#undef MXK_SWAP
          xc[0][s0 + t] = u32x4{a[0], a[1], a[2], a[3]};
          const uint32_t mine = high ? (odd ? byte[3] : byte[2]) : (odd ? byte[1] : byte[0]);
          xs[0] |= mine << (8 * (s0 + t));
        }
      }
      multiply(chunk, xc, xs);
    }
  }
  __syncthreads();  // every wave has read its rows of b: the sums take their place
  float* part = reinterpret_cast<float*>(few_lds);
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j)
      *reinterpret_cast<f32x4f*>(&part[(((wave * MT + i) * NT + j) * 64 + lane) * 4]) = acc[i][j];
  __syncthreads();
  for (int o = threadIdx.x; o < MT * NT * 256; o += blockDim.x) {
    const int nl = o % (16 * NT), ml = o / (16 * NT);
    const int64_t m = lo + ml, n = n0 + nl;
    if (m >= hi || n >= p.N) continue;
    const int at = (((ml >> 4) * NT + (nl >> 4)) * 64 + ((nl & 15) >> 2) * 16 + (ml & 15)) * 4 + (nl & 3);
    float v = p.bias ? p.bias[(int64_t)e * p.N + n] : 0.0f;
    for (int w = 0; w < waves; ++w) v += part[w * MT * NT * 256 + at];
    y[m * p.N + n] = from_f32<T>(v);
  }
}

// y = bias + the sum of the parts of K, in their order, four values a thread;
// eight parts are requested at a time.  128x8192, four parts: 5.2 us for 19 MB
// that are mostly still in the caches.
template <typename T>
__global__ __launch_bounds__(256) void k_fp4_join(const float* __restrict__ parts, int splits, int64_t total, int64_t N,
                                                  const float* __restrict__ bias, T* __restrict__ y) {
  const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
  if (i >= total) return;
  float v[4] = {0, 0, 0, 0};
  if (bias) {
    uint32_t n = (uint32_t)(i % N);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      v[k] = bias[n];
      n = n + 1 == (uint32_t)N ? 0u : n + 1;
    }
  }
  if (i + 4 <= total) {
    for (int s0 = 0; s0 < splits; s0 += 8) {
      float w[8][4];
#pragma unroll
      for (int s = 0; s < 8; ++s) {
#pragma unroll
        for (int k = 0; k < 4; ++k) w[s][k] = 0.0f;
        if (s0 + s < splits) __builtin_memcpy(w[s], parts + (s0 + s) * total + i, 16);
      }
#pragma unroll
      for (int s = 0; s < 8; ++s)
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] += w[s][k];
    }
    T t[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) t[k] = from_f32<T>(v[k]);
    __builtin_memcpy(y + i, t, sizeof(t));
  } else {
    for (int k = 0; i + k < total; ++k) {
      float w = v[k];
      for (int s = 0; s < splits; ++s) w += parts[s * total + i + k];
      y[i + k] = from_f32<T>(w);
    }
  }
}

// Bytes of the scales of `rows` rows in stage order, with room for the last tile's reads past the end
static int64_t stage_bytes(int64_t rows, int64_t KB) { return ceil_div(ceil_div(KB, 8) * rows, 2) * 16 + 4096; }

// Tiles of 16 rows of k_fp4_few for a problem (0: another kernel).  Dense:
// while one set of tiles holds every row, so that b is read once (64x8192x8192
// 17.7 us against the tile kernel's 19.5, 64x4096x4096 9.2 against 13.4,
// 32x8192x8192 12.7 against 18.3; two sets of 64 rows, 128x8192x8192: 33
// against 22).  By expert the rows of one are known on average only, and those
// above a set read the expert again: 32 experts of 4096x4096 with 16 rows each
// 72 us against 86, with 25 rows 84 against 88, with 32 rows 108 against 91; one
// tile of rows is best to 16 (12 rows 58 us, with two tiles 68).
static int few_of(const Fp4Gemm& p) {
  if (p.KB == 0 || p.KB > (1 << 18)) return 0;  // 64 rows of b in a buffer of at most 2^28 bytes
  if (p.offsets) {
    const int64_t rows = ceil_div(p.M, p.E);
    return rows <= 16 ? 1 : (rows <= 24 ? 2 : 0);
  }
  return p.M <= 16 ? 1 : (p.M <= 32 ? 2 : (p.M <= 64 ? 4 : 0));
}

// The tile kernel's shape for a problem: fragments a side of its waves (0:
// the plain kernel) and parts of K
struct Shape {
  int F, splits;
  bool staged;
};
static Shape tile_of(const Fp4Gemm& p) {
  const int64_t row_bytes = p.KB * 16;
  if (p.KB == 0 || few_of(p) || row_bytes > (1 << 22)) return {0, 1, false};
  if (p.order && p.a_rows * row_bytes > ((int64_t)1 << 30)) return {0, 1, false};
  if (p.N >= ((int64_t)1 << 21)) return {0, 1, false};  // 256 rows of 4-byte results within 2^31 bytes
  auto tiles = [&](int B) { return (p.offsets ? segment_slots(p.M, p.E, B) : ceil_div(p.M, B)) * ceil_div(p.N, B); };
  // large tiles where they occupy most CUs (2048x8192x8192, 256 of them: 76 us
  // against 92; 1024x8192x8192, 128: 61 against 48) and where experts fill one (32 of
  // 4096x4096: 250 rows each 129 us against 132, 62 rows 89 against 74)
  if (tiles(256) >= 192 && (!p.offsets || p.M > 128 * (int64_t)p.E)) return {4, 1, true};
  if (p.offsets) return {2, 1, true};
  // K in parts where tiles leave CUs idle and the stages saved, some 0.45 us
  // each, outweigh a launch and the parts' way through memory (128x8192x8192
  // in 4: 20 us against 33, 256x8192x8192 in 2: 27 against 30, 1000x500x4096
  // in 4: 14 against 16; 256x4096x4096 in 4: 22 against 16)
  const int64_t stages = ceil_div(p.KB, 8), n = tiles(128);
  const int64_t parts = std::max<int64_t>(1, std::min<int64_t>({num_cus() / n, stages / 4, 16}));
  const double saved = 0.45 * (double)(stages - stages / parts), cost = 3.0 + (double)(parts * p.M * p.N) * 0.8e-6;
  const int64_t splits = parts > 1 && saved > cost ? parts : 1;
  // scales straight from their rows, eight bytes of a line at a time, save a launch and
  // cost some 0.1 us a stage where every CU takes part: up to 12 stages of a tile per
  // CU on average (1500x1800x2080, 6 of them: 13.7 us against 15.3, 256x4096x4096, 4:
  // 13.8 against 16.3; 1024x4096x4096, 16: 21.3 against 20.6, 1024x8192x8192, 64: 57
  // against 50); they need eight bytes
  return {2, (int)splits, n * stages > 12 * num_cus() || p.N * p.KB < 8};
}
static int64_t tile_bytes(const Fp4Gemm& p, const Shape& t) {
  int64_t n = t.splits > 1 ? ceil_div(t.splits * p.M * p.N, 4) * 16 : 0;
  if (t.staged) n += stage_bytes(p.M, p.KB) + stage_bytes(p.offsets ? p.E * p.N : p.N, p.KB);
  return p.offsets ? n + 16 * segment_slots(p.M, p.E, 64 * t.F) + 4 * p.M : n;
}

// Whether the kernel of few rows packs float x itself: a dense product of at
// most 16 rows and one chunk of K per wave, whole dwords a row, x a buffer of
// less than 2^31 bytes.  The GPU takes as long either way (16x8192x8192 11.2
// us against 9.6 and 2.4, 1x4096x4096 6.3 against 5.9), the call 3 us less with one launch and no
// workspace.  By expert, where many workgroups would each pack mostly rows
// that are not there, packing first is faster: 8 tokens to 4 of 32 experts of
// 4096x4096 44 us against 29 and 2.5 for packing.
static bool packs_inside(const Fp4Gemm& p, int64_t x_stride, int x_type, int64_t K) {
  const int64_t size = x_type == MXK_IN_F32 ? 4 : 2;
  return !p.offsets && few_of(p) == 1 && p.KB <= 256 && K * size % 4 == 0 &&
         p.a_rows * std::max(x_stride, p.KB * 32) < ((int64_t)1 << 31) / size;
}

template <typename X, typename T, int MT, int NT>
static int launch_few_t(const Fp4Gemm& p, hipStream_t st) {
  const bool ex = p.offsets != nullptr;
  const int64_t n = (ex ? segment_slots(p.M, p.E, 16 * MT) : ceil_div(p.M, 16 * MT)) * ceil_div(p.N, 16 * NT);
  if (n >= ((int64_t)1 << 31)) return fail(MXK_EINVAL, "mxfp4 product: too many tiles");
  const int waves = (int)std::min<int64_t>(MT > 2 ? 8 : 16, ceil_div(p.KB, 16));
  const size_t own = NT > 1 ? 8192 : 4096, sums = MT * NT * 1024;
  const size_t lds = waves * std::max(own, sums);
  if constexpr (IsPacked<X>::V && MT < 4) {
    if (ex) {
      hipLaunchKernelGGL((k_fp4_few<X, T, MT, NT, true>), dim3((unsigned)n), dim3(64 * waves), lds, st, p);
      return check_launch("mxfp4 product of few rows by expert");
    }
  }
  hipLaunchKernelGGL((k_fp4_few<X, T, MT, NT, false>), dim3((unsigned)n), dim3(64 * waves), lds, st, p);
  return check_launch("mxfp4 product of few rows");
}
template <typename X, typename T, int MT>
static int launch_few_n(const Fp4Gemm& p, hipStream_t st) {
  // tiles of b per workgroup: as many as leave each CU a workgroup (by expert
  // four, since how many experts have rows is not known here), and as the
  // registers hold (four only for one packed tile of rows)
  const int64_t tiles = ceil_div(p.N, 16) * (p.offsets ? std::min<int64_t>(p.M, p.E) : 1);
  const int64_t per = tiles / (num_cus() * (p.offsets ? 4 : 1));
  if constexpr (IsPacked<X>::V && MT == 1)
    if (per >= 4) return launch_few_t<X, T, MT, 4>(p, st);
  if constexpr (IsPacked<X>::V || sizeof(X) == 2)
    if (per >= 2) return launch_few_t<X, T, MT, 2>(p, st);
  return launch_few_t<X, T, MT, 1>(p, st);
}
template <typename T>
static int launch_few_packed(const Fp4Gemm& p, int mt, hipStream_t st) {
  if (mt == 1) return launch_few_n<uint8_t, T, 1>(p, st);
  if (mt == 4) return launch_few_n<uint8_t, T, 4>(p, st);
  return launch_few_n<uint8_t, T, 2>(p, st);
}

static int launch_gemm(const Fp4Gemm& p, int y_type, uint8_t* ws, size_t ws_bytes, hipStream_t st) {
  const bool ex = p.offsets != nullptr;
  if (const int mt = few_of(p)) {
    if (y_type == MXK_IN_F32) return launch_few_packed<float>(p, mt, st);
    if (y_type == MXK_IN_F16) return launch_few_packed<__half>(p, mt, st);
    return launch_few_packed<hip_bfloat16>(p, mt, st);
  }
  const Shape t = tile_of(p);
  const int64_t B = t.F ? 64 * t.F : 64;
  const int64_t slots = ex ? segment_slots(p.M, p.E, (int)B) : ceil_div(p.M, B);
  const int64_t tn = ceil_div(p.N, B), n = ex && t.F ? block_tile_ids(slots, tn) : slots * tn * t.splits;
  if (n >= ((int64_t)1 << 31)) return fail(MXK_EINVAL, "mxfp4 product: too many tiles");
  const size_t need = t.F ? (size_t)tile_bytes(p, t) : 0;
  if (need > 0 && (!ws || !aligned16(ws) || ws_bytes < need))
    return fail(MXK_EINVAL, "mxfp4 product: workspace too small or not 16-byte aligned");
  const int64_t b_rows = ex ? p.E * p.N : p.N;
  Fp4Staged in = {};
  if (t.staged) {
    const int64_t na = stage_bytes(p.M, p.KB), nb = stage_bytes(b_rows, p.KB);
    const int64_t ga = ceil_div(p.M, 32), gb = ceil_div(b_rows, 32), gs = ex ? ceil_div(slots, 4) : 0;
    if (ga + gb + gs >= ((int64_t)1 << 31)) return fail(MXK_EINVAL, "mxfp4 product: too many rows");
    in.ta = ws;
    in.tb = ws + na;
    in.slot = reinterpret_cast<int4*>(ws + na + nb);
    in.row = reinterpret_cast<int*>(in.slot + slots);
    hipLaunchKernelGGL(k_fp4_stage, dim3((unsigned)(ga + gb + gs)), dim3(256), 0, st, p, in, b_rows, ga, gb, slots,
                       (int)B);
  }
  const int64_t cus = (num_cus() + 7) & ~7;  // a multiple of the XCDs: a workgroup's tiles stay on its own
#define MXK_TILE(T, F, EX, ST, P)                                                                                    \
  hipLaunchKernelGGL((k_fp4_gemm_tile<T, F, EX, ST>), dim3((unsigned)std::min<int64_t>(n, (F == 4 ? 1 : 2) * cus)), \
                     dim3(256), 0, st, P, in, b_rows, (uint32_t)slots, (uint32_t)tn, (uint32_t)t.splits, (uint32_t)n)
#define MXK_L(T, EX)                                                                                     \
  do {                                                                                                   \
    if (t.F == 4) MXK_TILE(T, 4, EX, true, p);                                                           \
    else if (t.F == 2 && (EX || t.staged)) MXK_TILE(T, 2, EX, true, p);                                  \
    else if (t.F == 2) MXK_TILE(T, 2, false, false, p);                                                  \
    else hipLaunchKernelGGL((k_fp4_gemm<T, EX>), dim3((unsigned)n), dim3(256), 0, st, p);                \
  } while (0)
#define MXK_T(T)                \
  do {                          \
    if (ex) MXK_L(T, true);     \
    else MXK_L(T, false);       \
  } while (0)
  if (t.splits > 1) {
    // behind the scales
    float* parts = reinterpret_cast<float*>(t.staged ? ws + stage_bytes(p.M, p.KB) + stage_bytes(p.N, p.KB) : ws);
    Fp4Gemm q = p;
    q.y = parts;
    q.bias = nullptr;
    if (t.staged) MXK_TILE(float, 2, false, true, q);
    else MXK_TILE(float, 2, false, false, q);
    const int64_t total = p.M * p.N;
    const dim3 grid((unsigned)ceil_div(total, 1024));
#define MXK_J(T)                                                                                                    \
  hipLaunchKernelGGL((k_fp4_join<T>), grid, dim3(256), 0, st, parts, t.splits, total, p.N, p.bias,                  \
                     reinterpret_cast<T*>(p.y))
    if (y_type == MXK_IN_F32) MXK_J(float);
    else if (y_type == MXK_IN_F16) MXK_J(__half);
    else MXK_J(hip_bfloat16);
#undef MXK_J
  } else if (y_type == MXK_IN_F32) {
    MXK_T(float);
  } else if (y_type == MXK_IN_F16) {
    MXK_T(__half);
  } else {
    MXK_T(hip_bfloat16);
  }
#undef MXK_T
#undef MXK_L
#undef MXK_TILE
  return check_launch("mxfp4 product");
}

// Sizes of a problem whose tensors are not known yet
static bool sizes(Fp4Gemm& p, int64_t a_rows, int64_t M, int64_t N, int64_t K, int experts, int picked) {
  static const int some = 0;
  if (a_rows < 0 || M <= 0 || N <= 0 || K <= 0 || experts < 0) return false;
  p.a_rows = a_rows;
  p.M = M;
  p.N = N;
  p.KB = fp4_blocks(K);
  p.offsets = experts > 0 ? &some : nullptr;
  p.order = picked ? &some : nullptr;
  p.E = experts;
  return true;
}
static int64_t packed_bytes(int64_t rows, int64_t KB) { return ceil_div(rows * KB * 17, 16) * 16; }

static int describe(Fp4Gemm& p, const char* what, const void* a, const void* as, int64_t a_rows, const void* b,
                    const void* bs, int64_t M, int64_t N, int64_t K, const float* bias, int y_type, void* y,
                    const int32_t* offsets, int experts, const int32_t* order, int top) {
  const std::string w = std::string(what) + ": ";
  if (a_rows < 0 || M < 0 || N < 0 || K < 0) return fail(MXK_EINVAL, w + "negative size");
  if (M >= ((int64_t)1 << 31) || N >= ((int64_t)1 << 31) || K >= ((int64_t)1 << 28) || a_rows >= ((int64_t)1 << 31))
    return fail(MXK_EINVAL, w + "rows below 2^31, K below 2^28");
  if (y_type != MXK_IN_F32 && y_type != MXK_IN_F16 && y_type != MXK_IN_BF16)
    return fail(MXK_EINVAL, w + "unknown type");
  if (offsets ? (experts < 1 || experts > 1000) : (order != nullptr || a_rows != M))
    return fail(MXK_EINVAL, w + "1 to 1000 experts with offsets; without them no order and as many rows as results");
  if (order ? (top < 1) : (offsets && a_rows != M))
    return fail(MXK_EINVAL, w + "top at least 1 with an order, as many rows as results without one");
  if (M == 0 || N == 0) return MXK_OK;
  if (!y || (K > 0 && (!b || !bs || (a_rows > 0 && (!a || !as))))) return fail(MXK_EINVAL, w + "null pointer");
  if (!aligned16(b)) return fail(MXK_EINVAL, w + "codes must be 16-byte aligned");
  p = {};
  p.a = reinterpret_cast<const uint8_t*>(a);
  p.as = reinterpret_cast<const uint8_t*>(as);
  p.b = reinterpret_cast<const uint8_t*>(b);
  p.bs = reinterpret_cast<const uint8_t*>(bs);
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
  return MXK_OK;
}

}  // namespace mxk

using namespace mxk;

extern "C" {

size_t mxk_mxfp4_matmul_workspace(int64_t a_rows, int64_t M, int64_t N, int64_t K, int experts, int picked) {
  Fp4Gemm p = {};
  if (!sizes(p, a_rows, M, N, K, experts, picked)) return 0;
  const Shape t = tile_of(p);
  return t.F ? (size_t)tile_bytes(p, t) : 0;
}

int mxk_mxfp4_matmul(const void* a_codes, const void* a_scales, int64_t a_rows, const void* b_codes,
                     const void* b_scales, int64_t M, int64_t N, int64_t K, const float* bias, int y_type, void* y,
                     const int32_t* offsets, int experts, const int32_t* order, int top, void* workspace,
                     size_t workspace_nbytes, void* stream) {
  Fp4Gemm p;
  const int rc = describe(p, "mxfp4_matmul", a_codes, a_scales, a_rows, b_codes, b_scales, M, N, K, bias, y_type, y,
                          offsets, experts, order, top);
  if (rc != MXK_OK || M == 0 || N == 0) return rc;
  if (!aligned16(a_codes)) return fail(MXK_EINVAL, "mxfp4_matmul: codes must be 16-byte aligned");
  return launch_gemm(p, y_type, reinterpret_cast<uint8_t*>(workspace), workspace_nbytes,
                     reinterpret_cast<hipStream_t>(stream));
}

size_t mxk_mxfp4_linear_workspace(int x_type, int64_t x_rows, int64_t x_stride, int64_t M, int64_t N, int64_t K,
                                  int experts, int picked) {
  Fp4Gemm p = {};
  if (!sizes(p, x_rows, M, N, K, experts, picked) || packs_inside(p, x_stride, x_type, K)) return 0;
  return (size_t)packed_bytes(x_rows, p.KB) + mxk_mxfp4_matmul_workspace(x_rows, M, N, K, experts, picked);
}

int mxk_mxfp4_linear(const void* x, int x_type, int64_t x_rows, int64_t x_stride, const void* b_codes,
                     const void* b_scales, int64_t M, int64_t N, int64_t K, const float* bias, void* y,
                     const int32_t* offsets, int experts, const int32_t* order, int top, void* workspace,
                     size_t workspace_nbytes, void* stream) {
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  Fp4Gemm p;
  int rc = describe(p, "mxfp4_linear", x, x, x_rows, b_codes, b_scales, M, N, K, bias, x_type, y, offsets, experts,
                    order, top);
  if (rc != MXK_OK || M == 0 || N == 0) return rc;
  if (x_stride < K) return fail(MXK_EINVAL, "mxfp4_linear: x_stride below K");
  if (packs_inside(p, x_stride, x_type, K)) {
    p.x = x;
    p.x_stride = x_stride;
    p.K = (int)K;
    if (x_type == MXK_IN_F32) return launch_few_n<float, float, 1>(p, st);
    if (x_type == MXK_IN_F16) return launch_few_n<__half, __half, 1>(p, st);
    return launch_few_n<hip_bfloat16, hip_bfloat16, 1>(p, st);
  }
  const size_t own = (size_t)packed_bytes(x_rows, p.KB);
  uint8_t* ws = reinterpret_cast<uint8_t*>(workspace);
  if (own > 0 && (!ws || !aligned16(ws) || workspace_nbytes < own))
    return fail(MXK_EINVAL, "mxfp4_linear: workspace too small or not 16-byte aligned");
  uint8_t* scales = ws + x_rows * p.KB * 16;
  rc = mxk_mxfp4_quantize(x, x_type, x_rows, K, x_stride, ws, scales, stream);
  if (rc != MXK_OK) return rc;
  p.a = ws;
  p.as = scales;
  return launch_gemm(p, x_type, ws + own, workspace_nbytes - own, st);
}

}  // extern "C"
