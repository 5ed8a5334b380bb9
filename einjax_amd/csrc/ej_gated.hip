// Gradient of the gated products' activation and product.
#include "ej_gated.h"

#include <type_traits>

namespace ej {
namespace {

constexpr int kThreads = 256;

// N values of T, anywhere in a row.
template <class T, int N>
struct Piece {
  T e[N];
  __device__ inline void load(const T *p, int there) {
    if (there >= N) {
      __builtin_memcpy(e, __builtin_assume_aligned(p, alignof(T)), sizeof(e));
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (i < there) e[i] = p[i];
    }
  }
  __device__ inline void store(T *p, int there) const {
    if (there >= N) {
      __builtin_memcpy(__builtin_assume_aligned(p, alignof(T)), e, sizeof(e));
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (i < there) p[i] = e[i];
    }
  }
};

// With h = act(g) u and its gradient dh: dg = dh u act'(g), du = dh act(g).  A
// thread takes a piece of one row: bound by memory (14 bytes of traffic for a
// column of 16-bit results, 20 in fp32): 16384 x 2048 bf16 80 to 84 us (5.6 to 5.9
// TB/s).  g and u come in fp32, so that the gradient is rounded once, to the
// operands' type, as the products after it take it: kept in more bits it would go
// through the matrix instructions twice (error of a bf16 training step's gradients
// 0.0023 of their norm, 0.0017 with fp32 gradients).
template <class T>
__global__ __launch_bounds__(kThreads) void gated_vjp_kernel(const float *gate_up, const T *grad,
                                                             int64_t rows, int32_t n, int64_t ld,
                                                             int32_t activation, T *out) {
  constexpr int N = 16 / sizeof(T);
  const uint32_t pieces = (static_cast<uint32_t>(n) + N - 1) / N;
  const uint32_t at = blockIdx.x * kThreads + threadIdx.x;
  const int64_t row = at / pieces;
  if (row >= rows) return;
  const int32_t col = static_cast<int32_t>(at - static_cast<uint32_t>(row) * pieces) * N;
  const int there = n - col;
  const int64_t first = row * (2 * static_cast<int64_t>(n)) + col;
  Piece<float, N> g, u;
  Piece<T, N> dh, dg, du;
  g.load(gate_up + first, there);
  u.load(gate_up + first + n, there);
  dh.load(grad + row * ld + col, there);
  by_activation<sizeof(T) == 4>(activation, [&](auto act) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      float value, slope;
      act.both(g.e[i], &value, &slope);
      const float d = static_cast<float>(dh.e[i]);
      dg.e[i] = static_cast<T>(d * u.e[i] * slope);
      du.e[i] = static_cast<T>(d * value);
    }
  });
  dg.store(out + first, there);
  du.store(out + first + n, there);
}

}  // namespace
}  // namespace ej

using namespace ej;

extern "C" int ej_gated_vjp(const float *gate_up, const void *grad, int32_t dtype, int64_t n_rows,
                            int32_t n, int64_t grad_stride, int32_t activation, void *out,
                            ej_stream_t stream) {
  EJ_CHECK_ARG(dtype == EJ_F32 || dtype == EJ_BF16 || dtype == EJ_F16,
               "gradient of dtype %d: expected EJ_F32, EJ_BF16 or EJ_F16", dtype);
  EJ_CHECK_ARG(activation == EJ_SILU || activation == EJ_GELU || activation == EJ_GELU_TANH,
               "activation %d", activation);
  EJ_CHECK_ARG(n_rows >= 0 && n >= 0, "negative size");
  EJ_CHECK_ARG(grad_stride >= n, "row stride %lld below n = %d", (long long)grad_stride, n);
  if (n_rows == 0 || n == 0) return EJ_OK;
  EJ_CHECK_ARG(gate_up && grad && out, "null argument");
  if (n >= (1 << 30)) {
    set_error("n = %d: gated products of fewer than 2^30 columns are supported", n);
    return EJ_E_UNSUPPORTED;
  }
  auto run = [&](auto *tp) {
    using T = std::remove_pointer_t<decltype(tp)>;
    const int64_t pieces = ceil_div(n, static_cast<int64_t>(16 / sizeof(T)));
    // a launch holds fewer than 2^32 threads
    if (n_rows > ((int64_t{1} << 32) - kThreads - 1) / pieces) {
      set_error("%lld rows of %d: too many for one launch", (long long)n_rows, n);
      return EJ_E_UNSUPPORTED;
    }
    const int64_t blocks = ceil_div(n_rows * pieces, kThreads);
    hipLaunchKernelGGL(gated_vjp_kernel<T>, dim3(static_cast<unsigned>(blocks)), dim3(kThreads), 0,
                       as_stream(stream), gate_up, static_cast<const T *>(grad), n_rows, n,
                       grad_stride, activation, static_cast<T *>(out));
    EJ_LAUNCH_CHECK();
    return EJ_OK;
  };
  if (dtype == EJ_F32) return run(static_cast<float *>(nullptr));
  if (dtype == EJ_BF16) return run(static_cast<__bf16 *>(nullptr));
  return run(static_cast<_Float16 *>(nullptr));
}
