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
typedef int i32v8_t __attribute__((ext_vector_type(8)));
typedef int i32v4_any_t __attribute__((ext_vector_type(4), aligned(1)));
typedef float f32x2_t __attribute__((ext_vector_type(2)));
typedef short i16x4_t __attribute__((ext_vector_type(4)));
// vectors at any element's alignment
typedef float f32x4_any_t __attribute__((ext_vector_type(4), aligned(4)));
typedef uint16_t u16x4_any_t __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t u32x4_any_t __attribute__((ext_vector_type(4), aligned(2)));

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

// 8-bit floating point (e4m3) with a scale for each 128 of k: kBlocks.  FINE:
// by the 16-bit matrix instructions, see mma_block.
template <bool FINE>
struct OpBlocks {
  using elem = uint8_t;
  using acc = f32x4_t;
  static constexpr bool kInt = false;
};
using OpF8 = OpBlocks<false>;
using OpF8Fine = OpBlocks<true>;
template <class Op>
constexpr bool kBlocks = __is_same(Op, OpF8) || __is_same(Op, OpF8Fine);

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
  const float *a_scale;     // 8-bit: scale of each row of A; blocks: [n_a][k blocks]
  const float *b_scale;     // 8-bit: scales [e][n]; blocks: [e][n blocks][k blocks]
  int64_t lda, ldb, ldc;    // row strides, elements
  int64_t b_group, c_group; // elements between the groups of B and of D
  int64_t n_a, n_b;         // rows of A; rows of Q
  int64_t slots;
  int32_t n_groups, m, n, k;
  int32_t out;              // EJ_F32, EJ_BF16 or EJ_F16
  uint32_t row_blocks, col_blocks;  // bound on live row blocks; column blocks
  // The contraction in `splits` parts (grid.y), each into fp32 sums of its own,
  // [splits][slots][n] or [splits][n_groups][m][n]; 1: none.
  float *partial;
  int32_t splits;
  // Gated products: n columns of results from the 2 n of B, the gate's first.
  float *gate_up;           // [slots][2 n] (null: not kept)
  int32_t activation;       // EJ_SILU, EJ_GELU or EJ_GELU_TANH
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

// A fragment's 128 of k in 8-bit floats, 32 a lane (16 of each 64-byte slab),
// and X Y^T over it.  Which of k lies in which lane is the same for X and Y, so
// the sum does not depend on it.  The form without scales: those of the blocks
// are fp32, not powers of two, and are applied to the sum.
//
// The 8-bit matrix instruction aligns the products of 8 consecutive k to the
// largest of them and drops what lies below 2^-13 of it (measured: 65536 + v
// keeps the multiples of 8 of v, toward zero); the eights are added in fp32.  A
// sum loses at most 7 2^-13 of the sum of its eights' largest magnitudes: 0.22 of
// bf16's unit roundoff, but 1.75 of fp16's.  Measured by sums that cancel but for
// the losses (root mean squares): normally distributed values lose 2^-16.7 of the
// sums, a 170th of what rounding to bf16 does and a 22nd of fp16's; such values
// times exp of others twice as wide 2^-14.4, a 35th and a fourth.  16-bit results
// take these sums for their rate.  Results in fp32 take FINE: e4m3 values are bf16
// values, and the sum of those is formed in fp32, at half the rate.
template <class Op>
struct BlockFragment {
  i32v8_t v;
  __device__ inline void set(const i32v4_t &lo, const i32v4_t &hi) {
    v = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
  }
};
template <>
struct BlockFragment<OpF8Fine> {
  bf16x8_t v[4];
  __device__ inline void set(const i32v4_t &lo, const i32v4_t &hi) {
#if defined(__HIP_DEVICE_COMPILE__)
    typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
#pragma unroll
    for (int w = 0; w < 8; ++w) {
      const uint32_t word = w < 4 ? lo[w] : hi[w - 4];
      const bf16x2_t a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(word, 1.f, false);
      const bf16x2_t b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(word, 1.f, true);
      v[w / 2][w % 2 * 4] = a[0];
      v[w / 2][w % 2 * 4 + 1] = a[1];
      v[w / 2][w % 2 * 4 + 2] = b[0];
      v[w / 2][w % 2 * 4 + 3] = b[1];
    }
#endif
  }
};
__device__ inline f32x4_t mma_block(const BlockFragment<OpF8> &x, const BlockFragment<OpF8> &y) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(x.v, y.v, f32x4_t{0.f, 0.f, 0.f, 0.f}, 0,
                                                          0, 0, 0, 0, 0);
}
__device__ inline f32x4_t mma_block(const BlockFragment<OpF8Fine> &x,
                                    const BlockFragment<OpF8Fine> &y) {
  f32x4_t sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int c = 0; c < 4; ++c)
    sum = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x.v[c], y.v[c], sum, 0, 0, 0);
  return sum;
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
  if constexpr (kElem<Op> == 4) return 4 * ((krow >> 2) & (CHUNKS >= 16 ? 3 : 1));
  else if constexpr (CHUNKS >= 16) return (2 * (krow & 3)) ^ (8 * ((krow >> 3) & 1));
  else return 2 * (krow & 3);
}

// One operand's tile: ROWS rows (of the output's extent) by kStep of k.
template <class Op, int ROWS, bool KC>
struct Tile {
  static constexpr int kBytes = ROWS * kRowB;
  static constexpr int kLine = KC ? kRowB : ROWS * kElem<Op>;  // bytes of an LDS row
  static constexpr int kChunks = kLine / 16;                   // chunks of an LDS row
  static constexpr int kReads = KC ? 1 : kElem<Op>;            // LDS reads of a fragment
  static_assert(KC || kChunks >= 8, "M tiles: swizzle range");

  // Line (row or k) and unswizzled chunk that the 16 bytes at LDS position
  // `pos` (in chunks) hold.
  __device__ static inline void at(int pos, int *line, int *chunk) {
    *line = pos / kChunks;
    *chunk = (pos % kChunks) ^ (KC ? swz_k(*line) : swz_m<Op, kChunks>(*line));
  }
};

// This lane's places in the fragments of F x 16 rows from row0 on: K tiles
// need one address for each 64-byte slab of the stage's k (the swizzle repeats
// every 16 rows), M tiles one for each fragment; the rest are constant offsets.
template <class Op, class T, bool KC, int F>
struct Fragments {
  static constexpr int kAddr = KC ? 2 : F;
  uint32_t addr[kAddr];

  __device__ inline void init(uint32_t base, int row0, int lane) {
    if constexpr (KC) {
      const int row = row0 + (lane & 15);
#pragma unroll
      for (int s = 0; s < 2; ++s)
        addr[s] = base + row * kRowB + ((s * 4 + (lane >> 4)) ^ swz_k(row)) * 16;
    } else {
#pragma unroll
      for (int i = 0; i < F; ++i) {
        if constexpr (kElem<Op> == 2) {
          const int krow = (lane >> 4) * 8 + ((lane & 15) >> 2);
          const int chunk = ((row0 + i * 16) >> 3) + ((lane & 3) >> 1);
          addr[i] = base + krow * T::kLine + (chunk ^ swz_m<Op, T::kChunks>(krow)) * 16 +
                    (lane & 1) * 8;
        } else {
          const int krow = (lane >> 4) * 4, col = row0 + i * 16 + (lane & 15);
          addr[i] = base + krow * T::kLine + ((col >> 2) ^ swz_m<Op, T::kChunks>(krow)) * 16 +
                    (col & 3) * 4;
        }
      }
    }
  }
  // The fragment of rows row0 + 16 i .. + 15, slab `slab`, of the tile `off`
  // bytes past the base.
  __device__ inline i32v4_t read(uint32_t off, int i, int slab) const {
    if constexpr (KC) {
      return *reinterpret_cast<const __attribute__((address_space(3))) i32v4_t *>(
          (lds_u8 *)(size_t)(addr[slab] + off) + i * 16 * kRowB);
    } else if constexpr (kElem<Op> == 2) {
      lds_u8 *p = (lds_u8 *)(size_t)(addr[i] + off) + slab * 32 * T::kLine;
      const i32v2_t h0 = __builtin_bit_cast(
          i32v2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                       (__attribute__((address_space(3))) i16x4_t *)p));
      const i32v2_t h1 = __builtin_bit_cast(
          i32v2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                       (__attribute__((address_space(3))) i16x4_t *)(p + 4 * T::kLine)));
      return i32v4_t{h0[0], h0[1], h1[0], h1[1]};
    } else {
      lds_u8 *p = (lds_u8 *)(size_t)(addr[i] + off) + slab * 16 * T::kLine;
      i32v4_t v;
#pragma unroll
      for (int c = 0; c < 4; ++c)
        v[c] = *reinterpret_cast<const __attribute__((address_space(3))) int *>(p + c * T::kLine);
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

// An 8-bit product's sum times (a b), without the range of fp32 for the scales'
// product: the result leaves it only where sum a b does; elsewhere its bits are
// those of sum * (a * b).  16384 rows in 8 groups, k = n = 4096: 269 us, 267 with
// sum * (a * b), 273 with the smaller scale picked as the first factor.
__device__ inline float scaled(float sum, float a, float b) {
  return ldexpf(sum * (__builtin_amdgcn_frexp_mantf(a) * __builtin_amdgcn_frexp_mantf(b)),
                __builtin_amdgcn_frexp_expf(a) + __builtin_amdgcn_frexp_expf(b));
}
// Stores v[0..3] as columns col .. col + 3 of a row at element offset `at`
// (of column 0), as one vector at any element's alignment.
__device__ inline void put4(void *c, int code, int64_t at, int col, int n, const float (&v)[4]) {
  if (code == EJ_F32) {
    float *p = static_cast<float *>(c) + at + col;
    if (col + 4 <= n) {
      *reinterpret_cast<f32x4_any_t *>(p) = f32x4_any_t{v[0], v[1], v[2], v[3]};
    } else {
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (col + r < n) p[r] = v[r];
    }
  } else {
    uint16_t *p = static_cast<uint16_t *>(c) + at + col;
    const u16x4_any_t o = {to_16(v[0], code), to_16(v[1], code), to_16(v[2], code),
                           to_16(v[3], code)};
    if (col + 4 <= n) {
      *reinterpret_cast<u16x4_any_t *>(p) = o;
    } else {
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (col + r < n) p[r] = o[r];
    }
  }
}

// 16-bit results of two fragments of a row, at columns col and col + 16 on, in
// pieces of 16 bytes: lanes 16 apart exchange four columns, so that each holds
// eight of one fragment.  Stores of 8 bytes a lane take the large blocks of
// 16384 x 512 x 4096 bf16 96 us, these 80; in rows off 16 bytes (3022 x 771 x
// 1283) single elements 37 us, these 33.
__device__ inline void put8(void *c, int code, int64_t at, int col, int n, int lane, bool there,
                            const float (&v)[2][4]) {
#if defined(__HIP_DEVICE_COMPILE__)
  u32x4_any_t w;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    uint32_t p[2];
#pragma unroll
    for (int f = 0; f < 2; ++f)
      p[f] = to_16(v[f][2 * h], code) | static_cast<uint32_t>(to_16(v[f][2 * h + 1], code)) << 16;
    const auto both = __builtin_amdgcn_permlane16_swap(p[0], p[1], false, false);
    w[h] = both[0];
    w[2 + h] = both[1];
  }
  const int first = col + (lane >> 4 & 1) * 16 + (lane >> 5) * 8;
  uint16_t *p = static_cast<uint16_t *>(c) + at + first;
  if (there && first + 8 <= n) {
    *reinterpret_cast<u32x4_any_t *>(p) = w;
  } else if (there) {
#pragma unroll
    for (int r = 0; r < 8; ++r)
      if (first + r < n) p[r] = static_cast<uint16_t>(w[r / 2] >> 16 * (r & 1));
  }
#endif
}

// Stages [first, last) of part `part` of `parts`.
__device__ inline void part_of(int stages, int part, int parts, int *first, int *last) {
  *first = static_cast<int>(static_cast<int64_t>(stages) * part / parts);
  *last = static_cast<int>(static_cast<int64_t>(stages) * (part + 1) / parts);
}

// Zeroes the rows of C that no group covers (slots before the first offset
// and past the last), by the `nb` workgroups of which this is number `b`.
__device__ inline void zero_dead_rows(const GroupedArgs &g, int b, int nb) {
  const int s = static_cast<int>(g.slots);
  if (!g.offsets || !g.c) return;
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
// Loads 16 bytes for each lane straight into LDS, lane l's to `lds` + 16 l
// (m0 holds the address and needs one wait state before it is used).  As asm,
// because the compiler holds back every transposing LDS read until all such
// loads it knows of have landed; the loops wait for them by count (s_waitcnt
// vmcnt) before the barrier after which a stage is read.  The load has no
// output register.
__device__ inline void load_to_lds(const char *src, uint32_t lds) {
#if defined(__HIP_DEVICE_COMPILE__)
  asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %0, off" : : "v"(src), "{m0}"(lds));
#endif
}
// The same for 4 bytes, lane l's to `lds` + 4 l.
__device__ inline void load_word_to_lds(const float *src, uint32_t lds) {
#if defined(__HIP_DEVICE_COMPILE__)
  asm volatile("s_nop 0\n\tglobal_load_lds_dword %0, off" : : "v"(src), "{m0}"(lds));
#endif
}
// The same from a uniform address and 32 bits of offset for each lane, which take
// no vector instruction to move on.
__device__ inline void load_to_lds(const char *base, uint32_t off, uint32_t lds) {
#if defined(__HIP_DEVICE_COMPILE__)
  asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" : : "v"(off), "s"(base), "{m0}"(lds));
#endif
}
__device__ inline void load_word_to_lds(const char *base, uint32_t off, uint32_t lds) {
#if defined(__HIP_DEVICE_COMPILE__)
  asm volatile("s_nop 0\n\tglobal_load_lds_dword %0, %1" : : "v"(off), "s"(base), "{m0}"(lds));
#endif
}
__device__ inline uint32_t lds_address(const void *p) {
  return static_cast<uint32_t>(reinterpret_cast<size_t>((lds_u8 *)p));
}

// How tiles are loaded:
//   kLoadDirect   16 bytes straight into LDS: rows 16-byte aligned, extents whole
//                 chunks
//   kLoadPieces   16 bytes into registers, at any element's alignment, stored to
//                 LDS a stage later.  A chunk that a row ends in is loaded from
//                 the row's last 16 bytes and shifted down when it is stored.
//   kLoadElements the same, element by element: rows shorter than 16 bytes
// In the first two no load stands behind a branch, which would have it waited
// for before the next one.
constexpr int kLoadPieces = 0, kLoadDirect = 1, kLoadElements = 2;

// v moved down by n elements (0 to a chunk of them), zeros on top.
template <class Op>
__device__ inline i32v4_t shift_down(const i32v4_t &v, int n) {
  const int bits = n * kElem<Op> * 8;
  uint64_t w[2];
  __builtin_memcpy(w, &v, 16);
  const uint64_t hi = bits < 64 ? w[1] >> bits : 0;
  const uint64_t lo = bits == 0    ? w[0]
                      : bits < 64  ? w[0] >> bits | w[1] << (64 - bits)
                      : bits < 128 ? w[1] >> (bits - 64)
                                   : 0;
  w[0] = lo;
  w[1] = hi;
  i32v4_t r;
  __builtin_memcpy(&r, w, 16);
  return r;
}

// The first `valid` elements from p on (any number), zeros behind them.
template <class Op>
__device__ inline i32v4_t load_elements(const char *p, int valid) {
  using E = typename Op::elem;
  E e[kChunk<Op>] = {};
#pragma unroll
  for (int i = 0; i < kChunk<Op>; ++i)
    if (i < valid) e[i] = reinterpret_cast<const E *>(p)[i];
  i32v4_t v;
  __builtin_memcpy(&v, e, 16);
  return v;
}

// One operand's loads of a stage, split over NW waves; lane positions are
// fixed for the kernel, the sources advance stage by stage.
template <class Op, int ROWS, bool KC, int NW, int LOADS>
struct Loader {
  using T = Tile<Op, ROWS, KC>;
  static constexpr int kLoads = T::kBytes / 1024 / NW;  // load instructions per wave and stage
  static_assert(T::kBytes % (1024 * NW) == 0, "whole loads per wave");

  // k-rows between a lane's places in two loads of an M tile.  Its swizzle
  // repeats after that many, or after twice as many: then a lane has one
  // column in even loads and one in odd ones.
  static constexpr int kApart = KC ? 0 : NW * 64 / T::kChunks;
  static constexpr int kPeriod = T::kChunks >= 16 ? 16 : 8;
  static constexpr int kCols = KC || kLoads == 1 || kApart % kPeriod == 0 ? 1 : 2;
  static_assert(kCols == 1 || kApart * 2 % kPeriod == 0, "places repeat");

  const char *src[kLoads];  // this lane's source in the next stage
  int line;                 // K: first k element of the lane's chunk; M: its k-row in load 0
  int col[kCols];           // M: first column of the lane's chunk (in pieces: of what is loaded)
  int valid[kCols];         // M, not direct: elements from the chunk's first column to the extent
  bool edge;                // M, pieces: the tile reaches past the extent
  int held_left;            // K, pieces: elements of k of the stage that is held
  i32v4_t reg[LOADS == kLoadDirect ? 1 : kLoads];

  // k element (K) or k-row (M) of the lane's place in load v; in K tiles the
  // swizzle repeats every 16 rows, and differs by 4 between its halves.
  __device__ inline int line_at(int v) const {
    if constexpr (KC) return NW % 2 == 0 || v % 2 == 0 ? line : line ^ (4 * kChunk<Op>);
    else return line + v * kApart;
  }

  // K tiles: row_at(i) is the address of output row i's first k element.
  template <class RowAt>
  __device__ inline void init_k(int wave, int lane, RowAt row_at) {
#pragma unroll
    for (int v = 0; v < kLoads; ++v) {
      int row, chunk;
      T::at((v * NW + wave) * 64 + lane, &row, &chunk);
      if (v == 0) line = chunk * kChunk<Op>;
      src[v] = row_at(row) + chunk * 16;
    }
  }
  // M tiles: column col0 + i of the operand is output row i; extent `ext`.
  __device__ inline void init_m(int wave, int lane, const char *base, int64_t ld, int col0,
                                int ext) {
    init_m(wave, lane, base, ld, ext, [&](int i, int *shift) {
      *shift = 0;
      return col0 + i;
    });
  }
  // M tiles: output row i is column col_at(i, &shift) of an extent `ext` that
  // begins at column shift; a chunk's columns follow each other.
  template <class ColAt>
  __device__ inline void init_m(int wave, int lane, const char *base, int64_t ld, int ext,
                                ColAt col_at) {
    edge = false;
#pragma unroll
    for (int v = 0; v < kLoads; ++v) {
      int krow, chunk;
      T::at((v * NW + wave) * 64 + lane, &krow, &chunk);
      if (v == 0) line = krow;
      if (v < kCols) {
        int shift, c = col_at(chunk * kChunk<Op>, &shift);
        valid[v] = ext - c;
        if (LOADS != kLoadElements && c > ext - kChunk<Op>) {
          c = ext - kChunk<Op>;
          edge = true;
        }
        col[v] = c + shift;
      }
      src[v] = base + (line_at(v) * ld + col[v % kCols]) * kElem<Op>;
    }
    if constexpr (LOADS == kLoadPieces) edge = __any(edge);
  }

  // Starts load v of the next stage, of which `left` elements of k exist
  // (>= 1), to the tile at `tile`, and advances its source by `step` bytes.
  // part: the stage may end short of kStep elements.
  __device__ inline void load(int v, unsigned char *tile, int wave, int left, int64_t step,
                              bool part) {
    const char *zeros = reinterpret_cast<const char *>(&grouped_zeros), *p = src[v];
    if constexpr (LOADS == kLoadDirect) {
      if (part && left < kStep<Op>) p = line_at(v) < left ? p : zeros;
      load_to_lds(p, lds_address(tile) + (v * NW + wave) * 1024);
    } else if constexpr (LOADS == kLoadPieces) {
      const int there = left - line_at(v);
      if constexpr (KC) {
        p -= there < kChunk<Op> ? (kChunk<Op> - there) * kElem<Op> : 0;
        held_left = left;
      }
      p = there > 0 ? p : zeros;
      // as global memory: a load that might be of LDS is waited for with the
      // LDS reads
      reg[v] = *(const __attribute__((address_space(1))) i32v4_any_t *)(p);
    } else {
      if constexpr (KC) reg[v] = load_elements<Op>(p, left - line_at(v));
      else reg[v] = load_elements<Op>(p, line_at(v) < left ? valid[v % kCols] : 0);
    }
    src[v] += step;
  }
  // Not direct: what load() fetched, into the tile at `tile`.
  __device__ inline void store(unsigned char *tile, int wave, int lane) {
    constexpr int N = kChunk<Op>;
    if constexpr (LOADS == kLoadPieces && KC) {
      if (held_left < kStep<Op>)
#pragma unroll
        for (int v = 0; v < kLoads; ++v) {
          const int there = held_left - line_at(v);
          reg[v] = shift_down<Op>(reg[v], there < N && there > 0 ? N - there : 0);
        }
    }
    if constexpr (LOADS == kLoadPieces && !KC) {
      if (edge)
#pragma unroll
        for (int v = 0; v < kLoads; ++v) {
          const int there = valid[v % kCols];
          reg[v] = shift_down<Op>(reg[v], there < N && there > 0 ? N - there : 0);
        }
    }
#pragma unroll
    for (int v = 0; v < kLoads; ++v)
      *reinterpret_cast<i32v4_t *>(tile + ((v * NW + wave) * 64 + lane) * 16) = reg[v];
  }

  // M tiles of gathered rows (weight gradient): the sources of the stage whose
  // rows' places in the operand lie in the lanes of `row` (lane i: k-row i).
  __device__ inline void seek(const char *base, int64_t ld, int row) {
    int r[kLoads];
#pragma unroll
    for (int v = 0; v < kLoads; ++v) r[v] = __shfl(row, line_at(v));
#pragma unroll
    for (int v = 0; v < kLoads; ++v) src[v] = base + (r[v] * ld + col[v % kCols]) * kElem<Op>;
  }
};

}  // namespace ej
