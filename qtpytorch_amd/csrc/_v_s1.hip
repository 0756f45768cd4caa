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


// ---------------------------------------------------------------- tiles through LDS
// Scale bytes in the order in which the tile kernel's stages read them:
// out[kt][row][8], kt = stages of 8 blocks (256 values of K), zeros past KB,
// for the rows of the product (picked by `order` where there is one) and those of b.  One
// launch for both operands: 17/16 of a byte moved per 32 values.
__global__ __launch_bounds__(256) void k_fp4_stage_scales(Fp4Gemm p, int64_t b_rows, int64_t a_blocks,
                                                          uint8_t* __restrict__ ta, uint8_t* __restrict__ tb) {
  const bool of_a = (int64_t)blockIdx.x < a_blocks;
  const int64_t rows = of_a ? p.M : b_rows;
  const int64_t r = (of_a ? (int64_t)blockIdx.x : (int64_t)blockIdx.x - a_blocks) * 32 + (threadIdx.x >> 3);
  if (r >= rows) return;
  const int64_t src = of_a ? source_row(p, r) : r;
  const uint8_t* s = (of_a ? p.as : p.bs) + (src < 0 ? 0 : src) * p.KB;
  uint8_t* out = of_a ? ta : tb;
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
    *reinterpret_cast<uint64_t*>(out + ((k >> 3) * rows + r) * 8) = v;
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
__device__ __forceinline__ void load_to_lds(i32x4 r, uint32_t off, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
               :
               : "s"(lds), "v"(off), "s"(r)
               : "memory");
}
template <int N>
__device__ __forceinline__ void wait_loads() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" : : "i"(N) : "memory");
}

// Tile t of a grid of tm x tn, taken so that the workgroups of one XCD
// (blockIdx % 8) are consecutive tiles of an order that walks 8 rows of tiles
// down before it goes right: the 32 tiles an XCD holds at once share 8 row
// and 4 column panels in its L2.
__device__ __forceinline__ void place_tile(uint32_t id, uint32_t tm, uint32_t tn, uint32_t& m, uint32_t& n) {
  const uint32_t total = tm * tn, xcd = id & 7u, local = id >> 3;
  const uint32_t per = total >> 3, rest = total & 7u;
  const uint32_t t = xcd * per + min(xcd, rest) + local;
  const uint32_t group = t / (8u * tn), in = t - group * 8u * tn;
  const uint32_t high = min(8u, tm - group * 8u);
  n = in / high;
  m = group * 8u + (in - n * high);
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
// LDS rows are 128 bytes: 16-byte chunk c of row r sits at c ^ (r & 7), so
// that 8 lanes of consecutive rows read all banks once.  The loads write LDS
// in lane order, so the lane picks the chunk that belongs at its place.
//
// The barrier of a stage sits before its last step: by then the next stage
// has landed and this stage's last fragments are in registers, so the loads of the
// stage after next go into the buffer just read, and the next stage's first
// fragments are read while the last step multiplies.
template <typename T, int F, bool EXPERT>
__global__ __launch_bounds__(256, 1) void k_fp4_gemm_tile(Fp4Gemm p, const uint8_t* __restrict__ ta,
                                                          const uint8_t* __restrict__ tb, int64_t b_rows, uint32_t tm,
                                                          uint32_t tn) {
  constexpr int B = 64 * F;                 // rows of a tile
  constexpr int OP = B * 128, SC = B * 8;   // bytes of an operand's stage and of its scales
  constexpr int BUF = 2 * OP, SBUF = 2 * SC;
  constexpr int LI = B / 32;                // load instructions per wave, operand and stage
  __shared__ __align__(16) uint8_t lds[2 * BUF + 2 * SBUF];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r32 = lane & 31, h = lane >> 5;
  uint32_t mt, nt;
  place_tile(blockIdx.x, tm, tn, mt, nt);
  int64_t lo = (int64_t)mt * B, hi = p.M < lo + B ? p.M : lo + B;
  int e = 0;
  if (EXPERT) {
    const Segment s = find_segment<B>(mt, p.offsets, p.E, p.M);
    e = s.e;
    lo = s.lo;
    hi = s.hi;
    if (e > p.E) return;
  }
  const int64_t n0 = (int64_t)nt * B;
  T* y = reinterpret_cast<T*>(p.y);
  if (EXPERT && e == p.E) {  // rows without an expert
    const int64_t w = p.N - n0 < B ? p.N - n0 : B;
    for (int64_t i = threadIdx.x; i < (hi - lo) * w; i += 256)
      y[(lo + i / w) * p.N + n0 + i % w] = from_f32<T>(0.0f);
    return;
  }
  const uint32_t row_bytes = (uint32_t)p.KB * 16u;
  const int64_t rows_b = p.N - n0 < B ? p.N - n0 : B;
  const bool picked = EXPERT && p.order != nullptr;
  const uint8_t* a0 = picked ? p.a : p.a + lo * (int64_t)row_bytes;
  const int64_t rows_a = picked ? p.a_rows : (p.M - lo < B ? p.M - lo : B);
  const i32x4 ra = buffer_words(a0, (uint32_t)(rows_a * row_bytes));
  const i32x4 rb =
      buffer_words(p.b + ((int64_t)e * p.N + n0) * row_bytes, (uint32_t)(rows_b * row_bytes));
  // scales: planes of [rows][8] bytes; a lane's 16 bytes are those of two rows
  const int64_t sr_a = lo, sr_b = (int64_t)e * p.N + n0;

  // loads of this wave: rows (wave * LI + i) * 8 + lane / 8 of either operand
  const int lr = lane >> 3, chunk = (lane & 7) ^ lr;
  uint32_t off_a[LI], off_b[LI];
#pragma unroll
  for (int i = 0; i < LI; ++i) {
    const int row = (wave * LI + i) * 8 + lr;
    off_b[i] = (uint32_t)row * row_bytes;
    off_a[i] = off_b[i];
    if (picked) {
      const int64_t src = lo + row < hi ? source_row(p, lo + row) : -1;
      off_a[i] = src >= 0 ? (uint32_t)src * row_bytes : MXK_FAR_ROW;
    }
  }
  const uint32_t KB = (uint32_t)p.KB, stages = (KB + 7u) >> 3;
  // Workgroups start at different stages and wrap around.  Rows of 4096 bytes
  // (K = 8192), or a multiple, put one stage of every row into the same
  // channel of L2; in step, all workgroups of an XCD would wait for that one.
  const uint32_t skew = (mt const uint32_t skew = (2u * ((mt & 7u) + 8u * ((nt >> 1) & 1u))) % stages; 7u) % stages;
  auto issue = [&](uint32_t step, uint32_t buf) {
    const uint32_t turn = step + skew < stages ? step + skew : step + skew - stages;
    const uint32_t t = step < stages ? turn : stages;
    const uint32_t blk = 8u * t + chunk;
    const uint32_t ok = blk < KB ? blk * 16u : MXK_FAR_BLOCK;
#pragma unroll
    for (int i = 0; i < LI; ++i) load_to_lds(ra, off_a[i] + ok, buf * BUF + (wave * LI + i) * 1024u);
#pragma unroll
    for (int i = 0; i < LI; ++i) load_to_lds(rb, off_b[i] + ok, buf * BUF + OP + (wave * LI + i) * 1024u);
    // scales: B / 128 kilobytes an operand; waves 0, 1 take a's, 2, 3 b's (F = 2: waves 0 and 2)
    if (F == 4 || (wave & 1) == 0) {
      const bool of_b = wave >= 2;
      const int64_t rows = of_b ? b_rows : p.M, first = (of_b ? sr_b : sr_a) + 128 * (wave & 1);
      // past the last row: bytes of the next plane or of the kilobyte kept after the
      // last, for rows whose codes are zeros or whose results are not stored
      const i32x4 rs = buffer_words((of_b ? tb : ta) + ((int64_t)t * rows + first) * 8, t < stages ? 1024u : 0u);
      load_to_lds(rs, 16u * lane, 2u * BUF + buf * SBUF + (of_b ? SC : 0) + 1024u * (wave & 1));
    }
  };

  // fragment reads: rows of this wave's half of a (wave / 2) and of b (wave % 2)
  const uint32_t rd_a = (uint32_t)((wave >> 1) * 32 * F + r32) * 128u;
  const uint32_t rd_b = OP + (uint32_t)((wave & 1) * 32 * F + r32) * 128u;
  uint32_t at[4];
#pragma unroll
  for (int s = 0; s < 4; ++s) at[s] = (uint32_t)((4 * h + s) ^ (lane & 7)) * 16u;
  const uint32_t rs_a = 2 * BUF + ((wave >> 1) * 32 * F + r32) * 8 + 4 * h;
  const uint32_t rs_b = 2 * BUF + SC + ((wave & 1) * 32 * F + r32) * 8 + 4 * h;

  f32x16 acc[F][F];  // [b fragment][a fragment]: rows of the result are n
#pragma unroll
  for (int i = 0; i < F; ++i)
#pragma unroll
    for (int j = 0; j < F; ++j)
#pragma unroll
      for (int q = 0; q < 16; ++q) acc[i][j][q] = 0.0f;
  i32x4 fa[2][F], fb[2][F];
  int sa[2][F], sb[2][F];
  auto read_frags = [&](uint32_t buf, int s, i32x4 (&xa)[F], i32x4 (&xb)[F]) {
#pragma unroll
    for (int i = 0; i < F; ++i) {
      xa[i] = *reinterpret_cast<const i32x4*>(lds + buf * BUF + rd_a + at[s] + i * 4096);
      xb[i] = *reinterpret_cast<const i32x4*>(lds + buf * BUF + rd_b + at[s] + i * 4096);
    }
  };
  auto read_scales = [&](uint32_t buf, int (&xa)[F], int (&xb)[F]) {
#pragma unroll
    for (int i = 0; i < F; ++i) {
      xa[i] = *reinterpret_cast<const int*>(lds + buf * SBUF + rs_a + i * 256);
      xb[i] = *reinterpret_cast<const int*>(lds + buf * SBUF + rs_b + i * 256);
    }
  };
#define MXK_STEP(SEL, XA, XB, SA, SB)                                                                           \
  _Pragma("unroll") for (int i = 0; i < F; ++i) _Pragma("unroll") for (int j = 0; j < F; ++j) {                \
    const i32x8 va = {XA[j][0], XA[j][1], XA[j][2], XA[j][3], 0, 0, 0, 0};                                      \
    const i32x8 vb = {XB[i][0], XB[i][1], XB[i][2], XB[i][3], 0, 0, 0, 0};                                      \
    acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(vb, va, acc[i][j], 4, 4, SEL, SB[i], SEL, SA[j]); \
  }

  issue(0, 0);
  issue(1, 1);
  if (F == 4 || (wave & 1) == 0) wait_loads<2 * LI + 1>();
  else wait_loads<2 * LI>();
  __builtin_amdgcn_s_barrier();
  read_scales(0, sa[0], sb[0]);
  read_frags(0, 0, fa[0], fb[0]);
  // past the last stage the loads bring zeros and the reads are not used
  uint32_t buf = 0;
  for (uint32_t t = 0; t < stages; ++t) {
    read_frags(buf, 1, fa[1], fb[1]);
    MXK_STEP(0, fa[0], fb[0], sa[0], sb[0])
    read_frags(buf, 2, fa[0], fb[0]);
    MXK_STEP(1, fa[1], fb[1], sa[0], sb[0])
    read_frags(buf, 3, fa[1], fb[1]);
    MXK_STEP(2, fa[0], fb[0], sa[0], sb[0])
    wait_loads<0>();
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    issue(t + 2, buf);
    buf ^= 1u;
    read_scales(buf, sa[1], sb[1]);
    read_frags(buf, 0, fa[0], fb[0]);
    MXK_STEP(3, fa[1], fb[1], sa[0], sb[0])
#pragma unroll
    for (int i = 0; i < F; ++i) {
      sa[0][i] = sa[1][i];
      sb[0][i] = sb[1][i];
    }
  }
  wait_loads<0>();
#undef MXK_STEP

  // The result through LDS, 32 rows of m at a time and wave: a lane holds
  // four consecutive n of one m; rows leave in 16-byte pieces of whole lines.
  __syncthreads();
  constexpr int NW = 32 * F;                          // columns of a wave
  constexpr int ROW = NW * (int)sizeof(T), CH = ROW / 16;  // bytes and 16-byte chunks of a row of them
  static_assert(32 * ROW * 4 <= (int)sizeof(lds), "four waves' rows");
  uint8_t* mine = lds + wave * 32 * ROW;
  const int64_t nw = n0 + (wave & 1) * NW;
  if (p.bias) {
    const float* bias = p.bias + (int64_t)e * p.N;
#pragma unroll
    for (int i = 0; i < F; ++i)
#pragma unroll
      for (int q = 0; q < 16; ++q) {
        const int64_t n = nw + 32 * i + 8 * (q >> 2) + 4 * h + (q & 3);
        const float b = n < p.N ? bias[n] : 0.0f;
#pragma unroll
        for (int j = 0; j < F; ++j) acc[i][j][q] += b;
      }
  }
#pragma unroll
  for (int j = 0; j < F; ++j) {
#pragma unroll
    for (int i = 0; i < F; ++i)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int c = 32 * i + 8 * q + 4 * h;  // first of the lane's four columns
        float v[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = acc[i][j][4 * q + k];
        T t[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) t[k] = from_f32<T>(v[k]);
        const int byte = c * (int)sizeof(T);
        uint8_t* d = mine + r32 * ROW + (((byte >> 4) ^ (r32 & (CH - 1))) << 4) + (byte & 15);
        __builtin_memcpy(__builtin_assume_aligned(d, 4 * sizeof(T)), t, sizeof(t));
      }
    __builtin_amdgcn_wave_barrier();
    constexpr int PER = 64 / CH > 0 ? 64 / CH : 1;  // rows per instruction
#pragma unroll
    for (int k = 0; k < 32 / PER; ++k) {
      const int row = k * PER + lane / CH, ch = lane % CH;
      const u32x4 v = *reinterpret_cast<const u32x4*>(mine + row * ROW + ((ch ^ (row & (CH - 1))) << 4));
      const int64_t m = lo + (wave >> 1) * NW + 32 * j + row, n = nw + ch * (16 / (int)sizeof(T));
      if (m < hi) {
        T* dst = y + m * p.N + n;
        if (n + 16 / (int)sizeof(T) <= p.N) {
          __builtin_memcpy(dst, &v, 16);
        } else {
          T t[16 / sizeof(T)];
          __builtin_memcpy(t, &v, 16);
#pragma unroll
          for (int k2 = 0; k2 < 16 / (int)sizeof(T); ++k2)
            if (n + k2 < p.N) dst[k2] = t[k2];
        }
      }
    }
    __builtin_amdgcn_wave_barrier();
  }
}

// Bytes of the scales of `rows` rows in stage order, with room for the last tile's reads past the end
static int64_t stage_bytes(int64_t rows, int64_t KB) { return ceil_div(KB, 8) * rows * 8 + 4096; }

// Fragments a side of the tile kernel's waves for a problem, 0: the plain kernel
static int tile_of(const Fp4Gemm& p) {
  const int64_t row_bytes = p.KB * 16;
  if (p.KB == 0 || p.M < 64 || p.N < 64 || row_bytes > (1 << 22)) return 0;
  if (p.order && p.a_rows * row_bytes > ((int64_t)1 << 30)) return 0;
  const int64_t m4 = p.offsets ? segment_slots(p.M, p.E, 256) : ceil_div(p.M, 256);
  if (p.offsets && p.M < 64 * (int64_t)p.E) return 0;
  return m4 * ceil_div(p.N, 256) >= 192 ? 4 : 2;
}

static int launch_gemm(const Fp4Gemm& p, int y_type, uint8_t* ws, size_t ws_bytes, hipStream_t st) {
  const bool ex = p.offsets != nullptr;
  const int F = tile_of(p);
  const int64_t B = F ? 64 * F : 64;
  const int64_t slots = ex ? segment_slots(p.M, p.E, (int)B) : ceil_div(p.M, B);
  const int64_t tn = ceil_div(p.N, B), n = slots * tn;
  if (n >= ((int64_t)1 << 31)) return fail(MXK_EINVAL, "mxfp4 product: too many tiles");
  const int64_t b_rows = ex ? p.E * p.N : p.N, na = stage_bytes(p.M, p.KB), nb = stage_bytes(b_rows, p.KB);
  if (F && (!ws || ws_bytes < (size_t)(na + nb))) return fail(MXK_EINVAL, "mxfp4 product: workspace too small");
  if (F) {
    const int64_t ga = ceil_div(p.M, 32), gb = ceil_div(b_rows, 32);
    if (ga + gb >= ((int64_t)1 << 31)) return fail(MXK_EINVAL, "mxfp4 product: too many rows");
    hipLaunchKernelGGL(k_fp4_stage_scales, dim3((unsigned)(ga + gb)), dim3(256), 0, st, p, b_rows, ga, ws, ws + na);
  }
#define MXK_L(T, EX)                                                                                              \
  do {                                                                                                            \
    if (F == 4)                                                                                                   \
      hipLaunchKernelGGL((k_fp4_gemm_tile<T, 4, EX>), dim3((unsigned)n), dim3(256), 0, st, p, ws, ws + na,       \
                         b_rows, (uint32_t)slots, (uint32_t)tn);                                                  \
    else if (F == 2)                                                                                              \
      hipLaunchKernelGGL((k_fp4_gemm_tile<T, 2, EX>), dim3((unsigned)n), dim3(256), 0, st, p, ws, ws + na,       \
                         b_rows, (uint32_t)slots, (uint32_t)tn);                                                  \
    else                                                                                                          \
      hipLaunchKernelGGL((k_fp4_gemm<T, EX>), dim3((unsigned)n), dim3(256), 0, st, p);                           \
  } while (0)
#define MXK_T(T)                \
  do {                          \
    if (ex) MXK_L(T, true);     \
    else MXK_L(T, false);       \
  } while (0)
  if (y_type == MXK_IN_F32) MXK_T(float);
  else if (y_type == MXK_IN_F16) MXK_T(__half);
  else MXK_T(hip_bfloat16);
#undef MXK_T
#undef MXK_L
  return check_launch("mxfp4 product");
}

}  // namespace mxk

using namespace mxk;

extern "C" {

size_t mxk_mxfp4_matmul_workspace(int64_t a_rows, int64_t M, int64_t N, int64_t K, int experts, int picked) {
  if (a_rows < 0 || M <= 0 || N <= 0 || K <= 0 || experts < 0) return 0;
  Fp4Gemm p = {};
  static const int some = 0;
  p.a_rows = a_rows;
  p.M = M;
  p.N = N;
  p.KB = fp4_blocks(K);
  p.offsets = experts > 0 ? &some : nullptr;
  p.order = picked ? &some : nullptr;
  p.E = experts;
  if (!tile_of(p)) return 0;
  return (size_t)(stage_bytes(M, p.KB) + stage_bytes(experts > 0 ? experts * N : N, p.KB));
}

int mxk_mxfp4_matmul(const void* a_codes, const void* a_scales, int64_t a_rows, const void* b_codes,
                     const void* b_scales, int64_t M, int64_t N, int64_t K, const float* bias, int y_type, void* y,
                     const int32_t* offsets, int experts, const int32_t* order, int top, void* workspace,
                     size_t workspace_nbytes, void* stream) {
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
  return launch_gemm(p, y_type, reinterpret_cast<uint8_t*>(workspace), workspace_nbytes, st);
}

}  // extern "C"
