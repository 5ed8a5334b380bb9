// Blocks of 128 in 8-bit floats (e4m3) with a scale each.
#include <type_traits>

#include "ej_internal.h"

namespace ej {
namespace {

constexpr int kThreads = 256;
constexpr float kMax = 448.f;  // the largest e4m3 value

// N values of a row from column `col` on, zeros past its end, in 32 bits.  A row's
// last values are loaded with those before them, N together, and only rows of
// fewer than N (FEW) one by one: no load stands behind a branch.
template <int N, bool FEW, class T>
__device__ inline void load_piece(const T *row, int col, int n, float (&v)[N]) {
  if constexpr (FEW) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = col + i < n ? static_cast<float>(row[col + i]) : 0.f;
  } else {
    const int from = col <= n - N ? col : n - N;
    T e[N];
    __builtin_memcpy(e, __builtin_assume_aligned(row + from, alignof(T)), sizeof(e));
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = static_cast<float>(e[i]);
    if (__any(from < col)) {
      // values of the piece before: the last `there` are this one's
      const int there = from == col ? N : n > col ? n - col : 0;
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = i >= N - there ? v[i] : 0.f;
    }
  }
}

// Magnitudes as the integers of their bits, which order them with infinity
// and then NaN on top.
template <int N>
__device__ inline uint32_t largest(const float (&v)[N], uint32_t most) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const uint32_t m = __float_as_uint(v[i]) & 0x7fffffffu;
    most = m > most ? m : most;
  }
  return most;
}

// Over a row of 16 lanes, in every one of them: the other of a pair, of a pair of
// pairs, and the mirrored places of eight and of sixteen.
__device__ inline uint32_t largest_of_16(uint32_t most) {
  auto with = [&](uint32_t other) { most = other > most ? other : most; };
  with(__builtin_amdgcn_update_dpp(0, most, 0xb1, 0xf, 0xf, false));
  with(__builtin_amdgcn_update_dpp(0, most, 0x4e, 0xf, 0xf, false));
  with(__builtin_amdgcn_update_dpp(0, most, 0x141, 0xf, 0xf, false));
  with(__builtin_amdgcn_update_dpp(0, most, 0x140, 0xf, 0xf, false));
  return most;
}

__device__ inline float scale_of(uint32_t most) {
  const float s = __uint_as_float(most) * static_cast<float>(1.0 / 448.0);
  return most < 0x7f800000u ? s : __uint_as_float(0x7fc00000u);
}

// v / s to the nearest e4m3 values, stored from column `col` of a row on.
//
// The quotient is that of a division: v times the rounded reciprocal is within two
// units in the last place, and with the remainder, which a fused multiply-add
// gives exactly, times the reciprocal added it is the rounded quotient.  (A
// product alone misses ties: 16-bit values are often an exact tie between two
// e4m3 values apart.)  Remainders are exact for scales from 2^-90 on; below, and
// for those that keep no values, it is divided.
template <int N, bool FEW>
__device__ inline void put_piece(uint8_t *row, int col, int n, const float (&v)[N], float s) {
  static_assert(N % 4 == 0, "words");
  const float inv = 1.f / s;
  float f[N];
  if (s >= 0x1p-90f) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      f[i] = v[i] * inv;
      f[i] = fmaf(fmaf(-f[i], s, v[i]), inv, f[i]);
    }
  } else {
    const bool plain = s > 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float x = plain ? v[i] / s : 0.f;
      // the quotients by a subnormal scale may pass the largest value
      f[i] = fminf(fmaxf(x, -kMax), kMax);
    }
  }
  uint32_t w[N / 4];
#pragma unroll
  for (int i = 0; i < N; i += 4) {
    const int word = __builtin_amdgcn_cvt_pk_fp8_f32(f[i], f[i + 1], 0, false);
    w[i / 4] = __builtin_amdgcn_cvt_pk_fp8_f32(f[i + 2], f[i + 3], word, true);
  }
  if (col <= n - N) {
    __builtin_memcpy(row + col, w, N);
  } else {
    // a short piece's values lie first (FEW) or last
    const int there = n > col ? n - col : 0, skip = FEW ? 0 : N - there;
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (i >= skip && i < skip + there)
        row[col + i - skip] = static_cast<uint8_t>(w[i / 4] >> 8 * (i % 4));
  }
}

// Rows and matrices of what is quantized.
template <class T>
struct Values {
  const T *x;
  int64_t mat_ld, ld, n_rows;  // rows of a matrix
  int64_t total;               // rows in all
  int32_t n;
  uint8_t *q;
  float *scale;
};

// 1 x 128: sixteen lanes a block, eight values each.  MATS: rows of more than one
// matrix.  Bound by memory: 8192 x 4096 bf16 20 us (5.0 TB/s; by division 27 to 32), in
// rows off 16 bytes 21.
template <class T, bool FEW, bool MATS>
__global__ __launch_bounds__(kThreads) void quantize_rows_of_blocks_kernel(Values<T> a) {
  constexpr int N = 8;
  const uint32_t k_blocks = (static_cast<uint32_t>(a.n) + 127) / 128;
  const uint32_t at = blockIdx.x * (kThreads / 16) + threadIdx.x / 16;
  const uint32_t row = at / k_blocks, block = at - row * k_blocks;
  const int col = static_cast<int>(block) * 128 + (threadIdx.x & 15) * N;
  const int64_t in = row < a.total ? row : a.total - 1;
  int64_t off = in * a.ld;
  if constexpr (MATS) off = in / a.n_rows * a.mat_ld + in % a.n_rows * a.ld;
  float v[N];
  load_piece<N, FEW>(a.x + off, col, a.n, v);
  const uint32_t most = largest_of_16(largest(v, 0));
  if (row >= a.total) return;
  const float s = scale_of(most);
  if ((threadIdx.x & 15) == 0) a.scale[at] = s;
  put_piece<N, FEW>(a.q + row * static_cast<int64_t>(a.n), col, a.n, v, s);
}

// 128 x 128: a workgroup a block, each thread eight columns of eight rows.  Bound by
// memory: 8 x 4096 x 4096 bf16 80 us (5.0 TB/s).
template <class T, bool FEW>
__global__ __launch_bounds__(kThreads) void quantize_blocks_kernel(Values<T> a) {
  constexpr int N = 8, R = 8;
  const int64_t k_blocks = (a.n + 127) / 128, r_blocks = (a.n_rows + 127) / 128;
  const int64_t b = blockIdx.x, mat = b / (r_blocks * k_blocks), in = b % (r_blocks * k_blocks);
  const int64_t row0 = in / k_blocks * 128 + threadIdx.x / 16;
  const int col = static_cast<int>(in % k_blocks) * 128 + (threadIdx.x & 15) * N;
  float v[R][N];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    // rows past the end: the last one again
    const int64_t row = row0 + r * 16 < a.n_rows ? row0 + r * 16 : a.n_rows - 1;
    load_piece<N, FEW>(a.x + mat * a.mat_ld + row * a.ld, col, a.n, v[r]);
  }
  uint32_t most = 0;
#pragma unroll
  for (int r = 0; r < R; ++r) most = largest(v[r], most);
  most = largest_of_16(most);
#pragma unroll
  for (int m = 16; m < 64; m <<= 1) {
    const uint32_t other = __shfl_xor(most, m);
    most = other > most ? other : most;
  }
  __shared__ uint32_t part[kThreads / 64];
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = most;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kThreads / 64; ++w) most = part[w] > most ? part[w] : most;
  const float s = scale_of(most);
  if (threadIdx.x == 0) a.scale[b] = s;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int64_t row = row0 + r * 16;
    if (row < a.n_rows)
      put_piece<N, FEW>(a.q + (mat * a.n_rows + row) * a.n, col, a.n, v[r], s);
  }
}

}  // namespace
}  // namespace ej

using namespace ej;

extern "C" int ej_quantize_blocks(const void *x, int32_t dtype, int64_t n_mats, int64_t mat_ld,
                                  int64_t n_rows, int64_t ld, int32_t n, int32_t block_rows,
                                  uint8_t *q, float *scale, ej_stream_t stream) {
  EJ_CHECK_ARG(dtype == EJ_F32 || dtype == EJ_BF16 || dtype == EJ_F16,
               "values of dtype %d: expected EJ_F32, EJ_BF16 or EJ_F16", dtype);
  EJ_CHECK_ARG(block_rows == 1 || block_rows == 128, "blocks of %d rows: expected 1 or 128",
               block_rows);
  EJ_CHECK_ARG(n_mats >= 0 && n_rows >= 0 && n >= 0, "negative size");
  if (n_mats == 0 || n_rows == 0 || n == 0) return EJ_OK;
  EJ_CHECK_ARG(x && q && scale, "null argument");
  EJ_CHECK_ARG(ld >= n, "row stride %lld below n = %d", (long long)ld, n);
  // a launch holds fewer than 2^32 threads
  const int64_t k_blocks = (static_cast<int64_t>(n) + 127) / 128;
  const int64_t most = (int64_t{1} << 32) / kThreads;
  const int64_t per_mat = block_rows == 1 ? n_rows : ceil_div(n_rows, 128);
  const int64_t held = (block_rows == 1 ? kThreads / 16 : 1) * (most - 1);
  if (n > INT32_MAX - 256 || n_rows > held || n_mats > held || per_mat > held / k_blocks / n_mats) {
    set_error("%lld matrices of %lld x %d: too many blocks for one launch", (long long)n_mats,
              (long long)n_rows, n);
    return EJ_E_UNSUPPORTED;
  }
  auto run = [&](auto *tp) {
    using T = std::remove_pointer_t<decltype(tp)>;
    Values<T> a = {static_cast<const T *>(x), mat_ld, ld, n_rows, n_mats * n_rows, n, q, scale};
    const int64_t blocks = n_mats * per_mat * k_blocks;
    auto launch = [&](auto kernel, int64_t grid) {
      hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(grid)), dim3(kThreads), 0,
                         as_stream(stream), a);
    };
    const bool few = n < 8;
    if (block_rows == 128) {
      if (few) launch(quantize_blocks_kernel<T, true>, blocks);
      else launch(quantize_blocks_kernel<T, false>, blocks);
    } else {
      const bool mats = n_mats > 1 && mat_ld != n_rows * ld;
      const int64_t grid = ceil_div(blocks, kThreads / 16);
      if (few) launch(quantize_rows_of_blocks_kernel<T, true, true>, grid);
      else if (mats) launch(quantize_rows_of_blocks_kernel<T, false, true>, grid);
      else launch(quantize_rows_of_blocks_kernel<T, false, false>, grid);
    }
    EJ_LAUNCH_CHECK();
    return EJ_OK;
  };
  if (dtype == EJ_F32) return run(static_cast<float *>(nullptr));
  if (dtype == EJ_BF16) return run(static_cast<__bf16 *>(nullptr));
  return run(static_cast<_Float16 *>(nullptr));
}
