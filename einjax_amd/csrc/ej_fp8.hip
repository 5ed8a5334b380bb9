// Blocks of 128 in 8-bit floats (e4m3) with a scale each.
#include <type_traits>

#include "ej_internal.h"

namespace ej {
namespace {

constexpr int kThreads = 256;
constexpr float kMax = 448.f;  // the largest e4m3 value

// N values of T in 32 bits, from any place in a row; zero past its end.
template <int N, class T>
__device__ inline void load_piece(const T *p, int there, float (&v)[N]) {
  T e[N];
  if (there >= N) {
    __builtin_memcpy(e, __builtin_assume_aligned(p, alignof(T)), sizeof(e));
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = static_cast<float>(e[i]);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = i < there ? static_cast<float>(p[i]) : 0.f;
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

__device__ inline float scale_of(uint32_t most) {
  const float s = __uint_as_float(most) * static_cast<float>(1.0 / 448.0);
  return most < 0x7f800000u ? s : __uint_as_float(0x7fc00000u);
}

// v / s to the nearest e4m3 values.  s is zero or NaN for blocks whose values
// are all 0 here.
template <int N>
__device__ inline void put_piece(uint8_t *q, int there, const float (&v)[N], float s) {
  static_assert(N % 4 == 0, "words");
  uint32_t w[N / 4];
  const bool plain = s > 0.f;
#pragma unroll
  for (int i = 0; i < N; i += 4) {
    float f[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      f[c] = plain ? v[i + c] / s : 0.f;
      f[c] = fminf(fmaxf(f[c], -kMax), kMax);
    }
    int word = __builtin_amdgcn_cvt_pk_fp8_f32(f[0], f[1], 0, false);
    w[i / 4] = __builtin_amdgcn_cvt_pk_fp8_f32(f[2], f[3], word, true);
  }
  if (there >= N) {
    __builtin_memcpy(q, w, N);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (i < there) q[i] = static_cast<uint8_t>(w[i / 4] >> 8 * (i % 4));
  }
}

// 1 x 128: sixteen lanes a block, eight values each.
template <class T>
__global__ __launch_bounds__(kThreads) void quantize_rows_of_blocks_kernel(
    const T *x, int64_t mat_ld, int64_t ld, int64_t n_rows, int64_t total, int32_t n, uint8_t *q,
    float *scale) {
  constexpr int N = 8;
  const uint32_t k_blocks = (static_cast<uint32_t>(n) + 127) / 128;
  const uint32_t at = blockIdx.x * (kThreads / 16) + threadIdx.x / 16;
  const uint32_t row = at / k_blocks, block = at - row * k_blocks;
  const bool live = row < total;
  const int col = static_cast<int>(block) * 128 + (threadIdx.x & 15) * N;
  const int64_t mat = row / n_rows, in = row - mat * n_rows;
  float v[N];
  load_piece<N>(x + mat * mat_ld + in * ld + col, live ? n - col : 0, v);
  uint32_t most = largest(v, 0);
#pragma unroll
  for (int m = 1; m < 16; m <<= 1) {
    const uint32_t other = __shfl_xor(most, m);
    most = other > most ? other : most;
  }
  if (!live) return;
  const float s = scale_of(most);
  if ((threadIdx.x & 15) == 0) scale[row * static_cast<int64_t>(k_blocks) + block] = s;
  put_piece<N>(q + row * static_cast<int64_t>(n) + col, n - col, v, s);
}

// 128 x 128: a workgroup a block, each thread eight columns of eight rows.
template <class T>
__global__ __launch_bounds__(kThreads) void quantize_blocks_kernel(const T *x, int64_t mat_ld,
                                                                   int64_t ld, int64_t n_rows,
                                                                   int32_t n, uint8_t *q,
                                                                   float *scale) {
  constexpr int N = 8, R = 8;
  const int64_t k_blocks = (n + 127) / 128, r_blocks = (n_rows + 127) / 128;
  const int64_t b = blockIdx.x, mat = b / (r_blocks * k_blocks), in = b % (r_blocks * k_blocks);
  const int64_t row0 = in / k_blocks * 128 + threadIdx.x / 16;
  const int col = static_cast<int>(in % k_blocks) * 128 + (threadIdx.x & 15) * N;
  float v[R][N];
  uint32_t most = 0;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int64_t row = row0 + r * 16;
    load_piece<N>(x + mat * mat_ld + row * ld + col, row < n_rows ? n - col : 0, v[r]);
    most = largest(v[r], most);
  }
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) {
    const uint32_t other = __shfl_xor(most, m);
    most = other > most ? other : most;
  }
  __shared__ uint32_t part[kThreads / 64];
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = most;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kThreads / 64; ++w) most = part[w] > most ? part[w] : most;
  const float s = scale_of(most);
  if (threadIdx.x == 0) scale[b] = s;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int64_t row = row0 + r * 16;
    if (row < n_rows) put_piece<N>(q + (mat * n_rows + row) * n + col, n - col, v[r], s);
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
  const int64_t k_blocks = (static_cast<int64_t>(n) + 127) / 128, most = (int64_t{1} << 32) / kThreads;
  const int64_t per_mat = block_rows == 1 ? n_rows : ceil_div(n_rows, 128);
  const int64_t held = (block_rows == 1 ? kThreads / 16 : 1) * (most - 1);
  if (n > INT32_MAX - 256 || n_rows > held || n_mats > held || per_mat > held / k_blocks / n_mats) {
    set_error("%lld matrices of %lld x %d: too many blocks for one launch", (long long)n_mats,
              (long long)n_rows, n);
    return EJ_E_UNSUPPORTED;
  }
  auto run = [&](auto *tp) {
    using T = std::remove_pointer_t<decltype(tp)>;
    const T *xt = static_cast<const T *>(x);
    const int64_t blocks = n_mats * per_mat * k_blocks;
    if (block_rows == 1)
      hipLaunchKernelGGL(quantize_rows_of_blocks_kernel<T>,
                         dim3(static_cast<unsigned>(ceil_div(blocks, kThreads / 16))),
                         dim3(kThreads), 0, as_stream(stream), xt, mat_ld, ld, n_rows,
                         n_mats * n_rows, n, q, scale);
    else
      hipLaunchKernelGGL(quantize_blocks_kernel<T>, dim3(static_cast<unsigned>(blocks)),
                         dim3(kThreads), 0, as_stream(stream), xt, mat_ld, ld, n_rows, n, q,
                         scale);
    EJ_LAUNCH_CHECK();
    return EJ_OK;
  };
  if (dtype == EJ_F32) return run(static_cast<float *>(nullptr));
  if (dtype == EJ_BF16) return run(static_cast<__bf16 *>(nullptr));
  return run(static_cast<_Float16 *>(nullptr));
}
