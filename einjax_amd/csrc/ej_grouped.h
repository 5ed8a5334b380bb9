// Products grouped by expert with ragged sizes: the geometry, the LDS tiles
// and the main loops.
//
//   rows product:    C[s, n] = sum_k A[row(s), k] B_e[k, n]   for s in group e
//   weight gradient: D_e[i, j] = sum over s in group e of P[p(s), i] Q[q(s), j]
//
// Group e holds the slots [offsets[e], offsets[e + 1]).  The offsets are read
// on the device: the grid is sized for a bound, every workgroup finds its
// group and row block with one scan of the group sizes (no plan kernel, no
// host wait), and workgroups beyond the live blocks exit.
//
// An operand tile is either contraction-contiguous ("K": rows of 128 bytes of
// consecutive k) or contraction-major ("M": one LDS row for each k, as W [k][n]
// and as both operands of the weight gradient lie in memory).  Tiles keep that
// layout in LDS, so nothing is transposed on the way in: K tiles are read as
// 16-byte fragments, 16-bit M tiles by the transposing LDS read and fp32 M
// tiles by single words.  16-byte chunks are XOR-swizzled so that one read
// instruction touches every bank equally.
#pragma once

#include "ej_gemm.h"

namespace ej {

typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef int i32v2_t __attribute__((ext_vector_type(2)));
typedef int i32v4_t __attribute__((ext_vector_type(4)));
typedef short i16x4_t __attribute__((ext_vector_type(4)));

// Storage types of the operands.  kStep = elements of k in a 128-byte row.
struct OpBf16 {
  using elem = uint16_t;
  using acc = f32x4_t;
  static constexpr bool kInt = false;
};
struct OpF16 {
  using elem = uint16_t;
  using acc = f32x4_t;
  static constexpr bool kInt = false;
};
struct OpF32 {
  using elem = float;
  using acc = f32x4_t;
  static constexpr bool kInt = false;
};
struct OpI8 {
  using elem = int8_t;
  using acc = i32v4_t;
  static constexpr bool kInt = true;
};

template <class Op>
constexpr int kElem = static_cast<int>(sizeof(typename Op::elem));
constexpr int kRowB = 128;                       // bytes of a K tile's row
template <class Op>
constexpr int kStep = kRowB / kElem<Op>;         // elements of k per stage
template <class Op>
constexpr int kChunk = 16 / kElem<Op>;           // elements of a 16-byte chunk

struct GroupedArgs {
  const char *a;            // A [n_a][k], or P [n_a][m] of the weight gradient
  const char *b;            // B [e][k][n] or [e][n][k], or Q [n_b][n]
  void *c;                  // C [slots][n], or D [e][m][n]
  const int32_t *a_rows;    // row of each slot in A (null: the slot itself)
  const int32_t *b_rows;    // weight gradient: row of each slot in Q
  const int32_t *offsets;   // [n_groups + 1] (null: one group of every slot)
  const float *a_scale;     // 8-bit: scale of each row of A
  const float *b_scale;     // 8-bit: scales [e][n]
  int64_t lda, ldb, ldc;    // row strides, elements
  int64_t b_group, c_group; // elements between the groups of B and of D
  int64_t n_a, n_b;         // rows of A; rows of Q
  int64_t slots;
  int32_t n_groups, m, n, k;
  int32_t out;              // EJ_F32, EJ_BF16 or EJ_F16
  uint32_t row_blocks, col_blocks;  // bound on live row blocks; column blocks
};

// A 16-byte chunk of zeros: what lanes beyond an operand's extent load.
static __device__ const uint4 grouped_zeros = {0, 0, 0, 0};

// ---- matrix instructions ---------------------------------------------------
// acc += X Y^T over one 64-byte slab of k: X holds 16 rows (the accumulator's
// register rows), Y 16 rows (its lanes).
template <class Op>
__device__ inline void mma(typename Op::acc &acc, const i32v4_t &x, const i32v4_t &y) {
  if constexpr (__is_same(Op, OpBf16)) {
    acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, x),
                                                  __builtin_bit_cast(bf16x8_t, y), acc, 0, 0, 0);
  } else if constexpr (__is_same(Op, OpF16)) {
    acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, x),
                                                 __builtin_bit_cast(f16x8_t, y), acc, 0, 0, 0);
  } else if constexpr (__is_same(Op, OpI8)) {
    acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(x, y, acc, 0, 0, 0);
  } else {
    const f32x4_t xf = __builtin_bit_cast(f32x4_t, x), yf = __builtin_bit_cast(f32x4_t, y);
#pragma unroll
    for (int c = 0; c < 4; ++c)
      acc = __builtin_amdgcn_mfma_f32_16x16x4f32(xf[c], yf[c], acc, 0, 0, 0);
  }
}

// ---- LDS tiles --------------------------------------------------------------
typedef __attribute__((address_space(3))) unsigned char lds_u8;

// Chunk c of row r of a K tile lies at chunk c ^ swz_k(r): the 16 rows of a
// fragment read then cover all 64 banks.
__device__ inline int swz_k(int row) { return (row >> 1) & 7; }

// The same for an M tile (row = one k).  16-bit: the four k-rows that a
// 16-lane group of the transposing read takes go to distinct 32-byte groups,
// and the two halves of the wave to distinct halves.  fp32: the four k-rows
// that the lane groups read go to distinct 64-byte groups.
template <class Op, int CHUNKS>
__device__ inline int swz_m(int krow) {
  if constexpr (kElem<Op> == 4) return 4 * ((krow >> 2) & 3);
  else if constexpr (CHUNKS >= 16) return (2 * (krow & 3)) ^ (8 * ((krow >> 3) & 1));
  else return 2 * (krow & 3);
}

// One operand's tile: ROWS rows (of the output's extent) by kStep of k.
template <class Op, int ROWS, bool KC>
struct Tile {
  static constexpr int kBytes = ROWS * kRowB;
  static constexpr int kLine = KC ? kRowB : ROWS * kElem<Op>;  // bytes of an LDS row
  static constexpr int kChunks = kLine / 16;                   // chunks of an LDS row
  static_assert(KC || kChunks >= (kElem<Op> == 4 ? 16 : 8), "M tiles: swizzle range");

  // Line (row or k) and unswizzled chunk that the 16 bytes at LDS position
  // `pos` (in chunks) hold.
  __device__ static inline void at(int pos, int *line, int *chunk) {
    *line = pos / kChunks;
    *chunk = (pos % kChunks) ^ (KC ? swz_k(*line) : swz_m<Op, kChunks>(*line));
  }

  // This lane's part of the fragment of 16 rows from row0 on, 64-byte slab
  // `slab` of the stage's k, from the tile at LDS address `base`.
  __device__ static inline i32v4_t frag(uint32_t base, int row0, int slab, int lane) {
    if constexpr (KC) {
      const int row = row0 + (lane & 15);
      const int chunk = (slab * 4 + (lane >> 4)) ^ swz_k(row);
      return *reinterpret_cast<const __attribute__((address_space(3))) i32v4_t *>(
          (lds_u8 *)(size_t)(base + row * kRowB + chunk * 16));
    } else if constexpr (kElem<Op> == 2) {
      const int t = (lane & 15) >> 2, q = lane & 3;
      i32v2_t h[2];
#pragma unroll
      for (int hh = 0; hh < 2; ++hh) {
        const int krow = slab * 32 + (lane >> 4) * 8 + hh * 4 + t;
        const int chunk = ((row0 >> 3) + (q >> 1)) ^ swz_m<Op, kChunks>(krow);
        h[hh] = __builtin_bit_cast(
            i32v2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                         (__attribute__((address_space(3))) i16x4_t *)(size_t)(
                             base + krow * kLine + chunk * 16 + (q & 1) * 8)));
      }
      return i32v4_t{h[0][0], h[0][1], h[1][0], h[1][1]};
    } else {
      i32v4_t v;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int krow = slab * 16 + (lane >> 4) * 4 + c;
        const int col = row0 + (lane & 15);
        const int chunk = (col >> 2) ^ swz_m<Op, kChunks>(krow);
        v[c] = *reinterpret_cast<const __attribute__((address_space(3))) int *>(
            (lds_u8 *)(size_t)(base + krow * kLine + chunk * 16 + (col & 3) * 4));
      }
      return v;
    }
  }
};

// ---- groups -----------------------------------------------------------------
// Slots of group e, clamped to the slots there are whatever the offsets hold.
__device__ inline void group_range(const GroupedArgs &g, int e, int *lo, int *hi) {
  const int s = static_cast<int>(g.slots);
  if (!g.offsets) {
    *lo = 0;
    *hi = s;
    return;
  }
  int a = g.offsets[e], b = g.offsets[e + 1];
  a = a < 0 ? 0 : a > s ? s : a;
  b = b < a ? a : b > s ? s : b;
  *lo = a;
  *hi = b;
}

// Inclusive prefix sum of 32-bit values across a wave.
__device__ inline int wave_inclusive_sum32(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);
  return v;
}

// Row blocks of `block` slots that the groups have in all.
__device__ inline int live_row_blocks(const GroupedArgs &g, int block) {
  const int lane = threadIdx.x & 63;
  int total = 0;
  for (int e0 = 0; e0 < g.n_groups; e0 += 64) {
    int lo = 0, hi = 0;
    if (e0 + lane < g.n_groups) group_range(g, e0 + lane, &lo, &hi);
    const int inc = wave_inclusive_sum32((hi - lo + block - 1) / block);
    total += __builtin_amdgcn_readlane(inc, 63);
  }
  return total;
}

// Group and slots of row block `rb` (below the live count).
struct RowBlock {
  int group, lo, hi;  // slots [lo, hi) of the block
};
__device__ inline RowBlock find_row_block(const GroupedArgs &g, int block, int rb) {
  const int lane = threadIdx.x & 63;
  int before = 0;
  for (int e0 = 0; e0 < g.n_groups; e0 += 64) {
    int lo = 0, hi = 0;
    if (e0 + lane < g.n_groups) group_range(g, e0 + lane, &lo, &hi);
    const int mine = (hi - lo + block - 1) / block;
    const int inc = before + wave_inclusive_sum32(mine);
    const uint64_t past = __ballot(inc > rb);
    if (past) {
      const int l = __builtin_ctzll(past);
      const int first = __builtin_amdgcn_readlane(inc - mine, l);
      RowBlock r;
      r.group = e0 + l;
      r.lo = __builtin_amdgcn_readlane(lo, l) + (rb - first) * block;
      const int end = __builtin_amdgcn_readlane(hi, l);
      r.hi = r.lo + block < end ? r.lo + block : end;
      return r;
    }
    before = __builtin_amdgcn_readlane(inc, 63);
  }
  return RowBlock{0, 0, 0};
}

// Row of A that slot s takes; an index outside A is clamped, so that no
// content of the index array leads out of bounds.
__device__ inline int64_t slot_row(const int32_t *rows, int64_t n_rows, int s) {
  if (!rows) return s < n_rows ? s : n_rows - 1;
  const int64_t r = rows[s];
  return r < 0 ? 0 : r < n_rows ? r : n_rows - 1;
}

// ---- results ----------------------------------------------------------------
__device__ inline uint16_t to_16(float v, int code) {
  return code == EJ_BF16 ? __builtin_bit_cast(uint16_t, static_cast<__bf16>(v))
                         : __builtin_bit_cast(uint16_t, static_cast<_Float16>(v));
}

// Stores v[0..3] as columns col .. col + 3 of a row at element offset `at`
// (of column 0); vec: the row's groups of four columns are aligned and whole.
__device__ inline void put4(void *c, int code, int64_t at, int col, int n, bool vec,
                            const float (&v)[4]) {
  if (code == EJ_F32) {
    float *p = static_cast<float *>(c) + at + col;
    if (vec && col + 4 <= n) {
      *reinterpret_cast<f32x4_t *>(p) = f32x4_t{v[0], v[1], v[2], v[3]};
    } else {
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (col + r < n) p[r] = v[r];
    }
  } else {
    uint16_t *p = static_cast<uint16_t *>(c) + at + col;
    if (vec && col + 4 <= n) {
      ushort4 o;
      o.x = to_16(v[0], code);
      o.y = to_16(v[1], code);
      o.z = to_16(v[2], code);
      o.w = to_16(v[3], code);
      *reinterpret_cast<ushort4 *>(p) = o;
    } else {
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (col + r < n) p[r] = to_16(v[r], code);
    }
  }
}

// Whether groups of four columns can be stored as one vector.
__device__ inline bool vec_rows(const GroupedArgs &g) {
  const int b = g.out == EJ_F32 ? 4 : 2;
  return g.ldc % 4 == 0 && g.c_group % 4 == 0 && reinterpret_cast<size_t>(g.c) % (4 * b) == 0;
}

// Zeroes the rows of C that no group covers (slots before the first offset
// and past the last), by the `nb` workgroups of which this is number `b`.
__device__ inline void zero_dead_rows(const GroupedArgs &g, int b, int nb) {
  const int s = static_cast<int>(g.slots);
  if (!g.offsets) return;
  int first = g.offsets[0], last = g.offsets[g.n_groups];
  first = first < 0 ? 0 : first > s ? s : first;
  last = last < first ? first : last > s ? s : last;
  const int dead = first + (s - last);
  for (int i = b; i < dead; i += nb) {
    const int64_t row = i < first ? i : last + (i - first);
    for (int col = threadIdx.x; col < g.n; col += blockDim.x) {
      if (g.out == EJ_F32) static_cast<float *>(g.c)[row * g.ldc + col] = 0.f;
      else static_cast<uint16_t *>(g.c)[row * g.ldc + col] = 0;
    }
  }
}
constexpr int kZeroBlocks = 64;  // workgroups appended to a grid for zero_dead_rows


// ---- operand loads ------------------------------------------------------------
#define EJ_LDS_PTR(p) ((__attribute__((address_space(3))) void *)(p))

// 16 bytes at any element alignment, the first `valid` elements of them (the
// rest zero).
template <class Op>
__device__ inline i32v4_t load_chunk(const char *p, int valid) {
  using E = typename Op::elem;
  constexpr int N = kChunk<Op>;
  i32v4_t v = {0, 0, 0, 0};
  if (valid >= N) {
    __builtin_memcpy(&v, __builtin_assume_aligned(p, alignof(E)), 16);
  } else {
    E e[N] = {};
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (i < valid) e[i] = reinterpret_cast<const E *>(p)[i];
    __builtin_memcpy(&v, e, 16);
  }
  return v;
}

// One operand's loads of a stage, split over NW waves; lane positions are
// fixed for the kernel, the sources advance stage by stage.  DIRECT: 16-byte
// loads straight into LDS (rows 16-byte aligned, extents whole chunks);
// otherwise loads into registers, at any alignment, stored to LDS a stage
// later.
template <class Op, int ROWS, bool KC, int NW, bool DIRECT>
struct Loader {
  using T = Tile<Op, ROWS, KC>;
  static constexpr int kLoads = T::kBytes / 1024 / NW;  // load instructions per wave and stage
  static_assert(T::kBytes % (1024 * NW) == 0, "whole loads per wave");

  const char *src[kLoads];  // this lane's source in the next stage
  int line[kLoads];         // K: first k element of the lane's chunk; M: its k-row
  int valid[kLoads];        // M, not DIRECT: elements of the lane's chunk inside the extent
  i32v4_t reg[DIRECT ? 1 : kLoads];

  // K tiles: row_at(i) is the address of output row i's first k element.
  template <class RowAt>
  __device__ inline void init_k(int wave, int lane, RowAt row_at) {
#pragma unroll
    for (int v = 0; v < kLoads; ++v) {
      int row, chunk;
      T::at((v * NW + wave) * 64 + lane, &row, &chunk);
      line[v] = chunk * kChunk<Op>;
      src[v] = row_at(row) + chunk * 16;
    }
  }
  // M tiles: column col0 + i of the operand is output row i; extent `ext`.
  __device__ inline void init_m(int wave, int lane, const char *base, int64_t ld, int col0,
                                int ext) {
#pragma unroll
    for (int v = 0; v < kLoads; ++v) {
      int chunk;
      T::at((v * NW + wave) * 64 + lane, &line[v], &chunk);
      int col = col0 + chunk * kChunk<Op>;
      if constexpr (DIRECT) {
        if (col > ext - kChunk<Op>) col = ext - kChunk<Op>;
      } else {
        valid[v] = ext - col;
        if (col >= ext) col = 0;
      }
      src[v] = base + (line[v] * ld + col) * kElem<Op>;
    }
  }

  // Loads the next stage, of which `left` elements of k exist (>= 1), to the
  // tile at `tile`, and advances the sources by `step` bytes.
  __device__ inline void load(unsigned char *tile, int wave, int left, int64_t step) {
#pragma unroll
    for (int v = 0; v < kLoads; ++v) {
      if constexpr (DIRECT) {
        const char *p = src[v];
        if (left < kStep<Op>)
          p = line[v] < left ? p : reinterpret_cast<const char *>(&grouped_zeros);
        __builtin_amdgcn_global_load_lds(p, EJ_LDS_PTR(tile + (v * NW + wave) * 1024), 16, 0, 0);
      } else {
        const int n = KC ? left - line[v] : line[v] < left ? valid[v] : 0;
        reg[v] = load_chunk<Op>(src[v], n);
      }
      src[v] += step;
    }
  }
  // Not DIRECT: what load() fetched, into the tile at `tile`.
  __device__ inline void store(unsigned char *tile, int wave, int lane) {
#pragma unroll
    for (int v = 0; v < kLoads; ++v)
      *reinterpret_cast<i32v4_t *>(tile + ((v * NW + wave) * 64 + lane) * 16) = reg[v];
  }

  // M tiles whose rows are slots (weight gradient): the sources of the stage
  // that starts at slot s0, rows through the index array if there is one.
  __device__ inline void seek_slots(const char *base, int64_t ld, const int32_t *rows,
                                    int64_t n_rows, int s0, int s_end, const int (&col)[kLoads]) {
#pragma unroll
    for (int v = 0; v < kLoads; ++v) {
      const int s = s0 + line[v];
      src[v] = base + (slot_row(rows, n_rows, s < s_end ? s : s_end - 1) * ld + col[v]) *
                          kElem<Op>;
    }
  }
};

}  // namespace ej
