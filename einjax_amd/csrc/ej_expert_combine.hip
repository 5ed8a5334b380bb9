// The weighted sum of each token's expert results, its gradients, and rows in
// 8-bit integers with a scale each.
//
// All three are bound by memory: every row is read once (the second pass of
// the quantization over a row comes from the cache) and written once, sixteen
// bytes a lane at any element's alignment.  The last piece of a row that holds
// no whole number of them is moved back over the one before: its elements are
// computed twice, with one result.
#include "ej_internal.h"

#include <type_traits>

namespace ej {
namespace {

constexpr int kThreads = 256;
constexpr int kZeroBlocks = 128;   // workgroups that zero the rows no pair holds
constexpr int kHeldWords = 2048;   // bits of rows that one of them keeps at a time, / 32
// HIP launches hold fewer than 2^32 threads.
constexpr int64_t kMaxBlocks = ((int64_t{1} << 32) - 1) / kThreads;

template <class T>
__device__ inline float widen(T v) {
  return static_cast<float>(v);
}

// Four words at any element's alignment.
typedef uint32_t words_t __attribute__((ext_vector_type(4), aligned(2)));

// First column of the piece of N that begins at col, moved back into the row.
template <int N>
__device__ inline int64_t piece_at(int64_t col, int32_t n) {
  return N == 1 || col + N <= n ? col : n - N;
}

// N consecutive elements (16 bytes when VEC), widened.
template <class T, bool VEC>
struct Piece {
  static constexpr int N = VEC ? 16 / static_cast<int>(sizeof(T)) : 1;
  float v[N];
  __device__ inline void load(const T *p) {
    if constexpr (VEC) {
      struct Chunk { T e[N]; };
      const Chunk w = __builtin_bit_cast(Chunk, *reinterpret_cast<const words_t *>(p));
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = widen(w.e[i]);
    } else {
      v[0] = widen(*p);
    }
  }
  template <class O>
  __device__ inline void store(O *p) const {
    if constexpr (VEC) {
      struct { O e[N]; } w;
#pragma unroll
      for (int i = 0; i < N; ++i) w.e[i] = static_cast<O>(v[i]);
      __builtin_memcpy(p, &w, sizeof(w));
    } else {
      *p = static_cast<O>(v[0]);
    }
  }
};

struct CombineArgs {
  const void *y;
  int64_t ld_y, ld_out;
  int64_t n_slots;
  int32_t k, n;
  const float *weights;  // null: every weight is 1
  const int32_t *slots;
  void *out;
};

// out[t] = sum_j weights[t, j] y[slots[t, j]]: summed in fp32 in the order of
// the picks, rounded once.  One workgroup a token and stretch of columns, so a
// token's indices and weights are read once for 256 lanes.  16384 tokens of 4
// picks, 4096 columns of bf16, 1 pair in 20 left out: 139 us (0.65 GB, 4.6
// TB/s; a large copy reaches 5.2).  4095 columns take as long (element by
// element 3 times that).
template <class T, class O, bool VEC>
__global__ __launch_bounds__(kThreads) void combine_kernel(CombineArgs a, unsigned col_blocks) {
  constexpr int N = Piece<T, VEC>::N;
  const int64_t t = blockIdx.x / col_blocks;
  const int64_t begin =
      (static_cast<int64_t>(blockIdx.x % col_blocks) * kThreads + threadIdx.x) * N;
  if (begin >= a.n) return;
  const int64_t col = piece_at<N>(begin, a.n);
  float sum[N] = {};
  for (int j = 0; j < a.k; ++j) {
    const int64_t s = a.slots[t * a.k + j];
    if (s < 0 || s >= a.n_slots) continue;
    const float w = a.weights ? a.weights[t * a.k + j] : 1.f;
    Piece<T, VEC> y;
    y.load(static_cast<const T *>(a.y) + s * a.ld_y + col);
#pragma unroll
    for (int i = 0; i < N; ++i) sum[i] += w * y.v[i];
  }
  Piece<T, VEC> o;
#pragma unroll
  for (int i = 0; i < N; ++i) o.v[i] = sum[i];
  o.store(static_cast<O *>(a.out) + t * a.ld_out + col);
}

// Zeroes the rows of grad_y that no pair holds.  Which those are goes by the
// slots alone (a caller may take pairs out by a slot of -1).  Workgroup `block`
// of kZeroBlocks looks after every kZeroBlocks-th row: it notes in LDS which of
// its rows the n_pairs pairs hold, then zeroes the others, a wave a row.  So all
// pairs' slots are read by each of them, from the L2 and beside the gradients:
// 16384 tokens of 4 picks, bf16, gradients alone and with the rows (none, all
// unheld): 4096 columns 250, 250 and 128 us, 512 columns 75, 77 and 36, 64
// columns 43, 45 and 29.  64 workgroups are 1 us faster with no such row and up
// to 17 slower with half of them, 256 the other way round.  Numbers left in the
// rows by a launch before and looked at by another took 5 to 13 us more.
template <class T>
__device__ inline void zero_unheld_rows(const CombineArgs &a, int64_t n_pairs, T *grad_y,
                                        int block) {
  constexpr int N = 16 / static_cast<int>(sizeof(T)), W = kThreads / 64;
  __shared__ uint32_t held[kHeldWords];
  const int lane = threadIdx.x & 63;
  const int64_t mine = (a.n_slots - block + kZeroBlocks - 1) / kZeroBlocks;
  for (int64_t i0 = 0; i0 < mine; i0 += 32 * kHeldWords) {
    const int count = static_cast<int>(mine - i0 < 32 * kHeldWords ? mine - i0 : 32 * kHeldWords);
    const int words = (count + 31) / 32;
    for (int w = threadIdx.x; w < words; w += kThreads) held[w] = 0;
    __syncthreads();
    auto look = [&](int64_t s) {
      if ((s & (kZeroBlocks - 1)) != block || s < 0) return;
      const int64_t i = s / kZeroBlocks - i0;
      if (i >= 0 && i < count) atomicOr(&held[i >> 5], 1u << (i & 31));
    };
    const int64_t quads = n_pairs / 4;
#pragma unroll 4
    for (int64_t q = threadIdx.x; q < quads; q += kThreads) {
      const words_t v = *reinterpret_cast<const words_t *>(a.slots + 4 * q);
#pragma unroll
      for (int c = 0; c < 4; ++c) look(static_cast<int32_t>(v[c]));
    }
    if (threadIdx.x < n_pairs - 4 * quads) look(a.slots[4 * quads + threadIdx.x]);
    __syncthreads();
    for (int w = threadIdx.x >> 6; w < words; w += W) {
      const int last = count - 32 * w;
      uint32_t left = __builtin_amdgcn_readfirstlane(~held[w] &
                                                     (last < 32 ? (1u << last) - 1 : ~0u));
      for (; left; left &= left - 1) {
        T *row = grad_y + ((i0 + 32 * w + __builtin_ctz(left)) * kZeroBlocks + block) * a.n;
        if (a.n >= N) {
          const words_t zero = {0, 0, 0, 0};
          for (int64_t col = lane * N; col < a.n; col += 64 * N)
            *reinterpret_cast<words_t *>(row + piece_at<N>(col, a.n)) = zero;
        } else if (lane < a.n) {
          row[lane] = static_cast<T>(0.f);
        }
      }
    }
    __syncthreads();
  }
}

// grad_y[slots[t, j]] = weights[t, j] grad[t]; grad_w[t, j] = grad[t] . y[slots[t, j]].
// One workgroup a token, so every dot product is summed in a fixed order; the
// first `zeroing` workgroups zero grad_y's rows that no pair of the n_pairs holds.
// At the sizes above 230 us (1.18 GB, 5.1 TB/s).
// WHOLE: rows of whole pieces; otherwise the last one is moved back.
template <class T, bool VEC, bool WHOLE>
__global__ __launch_bounds__(kThreads) void combine_vjp_kernel(CombineArgs a, const void *grad,
                                                               int64_t ld_grad, void *grad_y,
                                                               float *grad_w, int zeroing,
                                                               int64_t n_pairs) {
  constexpr int N = Piece<T, VEC>::N, W = kThreads / 64;
  if (blockIdx.x < zeroing) {
    zero_unheld_rows(a, n_pairs, static_cast<T *>(grad_y), blockIdx.x);
    return;
  }
  __shared__ float part[W][EJ_MAX_PICKS];
  const int64_t t = blockIdx.x - zeroing;
  const T *g = static_cast<const T *>(grad) + t * ld_grad;
  for (int j = 0; j < a.k; ++j) {
    const int64_t s = a.slots[t * a.k + j];
    float dot = 0.f;
    if (s >= 0 && s < a.n_slots) {
      const float w = a.weights ? a.weights[t * a.k + j] : 1.f;
      const T *y = static_cast<const T *>(a.y) + s * a.ld_y;
      T *d = static_cast<T *>(grad_y) + s * a.n;
      for (int64_t begin = threadIdx.x * N; begin < a.n; begin += kThreads * N) {
        const int64_t col = WHOLE ? begin : piece_at<N>(begin, a.n);
        // elements of the piece before
        const int twice = WHOLE ? 0 : static_cast<int>(begin - col);
        Piece<T, VEC> gv;
        gv.load(g + col);
        if (grad_w) {
          Piece<T, VEC> yv;
          yv.load(y + col);
          if (twice > 0) {
#pragma unroll
            for (int i = 0; i < N; ++i)
              if (i >= twice) dot += gv.v[i] * yv.v[i];
          } else {
#pragma unroll
            for (int i = 0; i < N; ++i) dot += gv.v[i] * yv.v[i];
          }
        }
        if (grad_y) {
#pragma unroll
          for (int i = 0; i < N; ++i) gv.v[i] *= w;
          gv.store(d + col);
        }
      }
    }
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) dot += __shfl_xor(dot, m);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6][j] = dot;
  }
  __syncthreads();
  if (grad_w && threadIdx.x < a.k) {
    float sum = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) sum += part[w][threadIdx.x];
    grad_w[t * a.k + threadIdx.x] = sum;
  }
}

// q = round(x / scale), scale = max |x| / 127 (as max |x| times the nearest
// fp32 to 1/127); ties to even.  A row of zeros has scale 0 and zeros; a row
// with a NaN or an infinity has scale NaN and zeros, so that whatever is
// computed with it is NaN.
//
// TPR threads a row hold P pieces of it each in registers between the two
// passes; what a longer row has beyond is read twice (from the cache).  The
// arithmetic would take longer than the memory if it were written down as
// above, so
//   - the maximum is taken of the bits without their signs, two 16-bit values
//     an instruction (the order of the magnitudes; infinities and NaN are the
//     largest);
//   - the rounded quotient comes from x times 1 / scale plus 1.5 2^23, whose
//     low byte is the result; where that product lies near a tie, which it can
//     be off by less than 2^-14 of, the piece is divided properly.
// 8192 x 4096 bf16: 31 us (0.1 GB, 3.2 TB/s; 26 with the rows in the cache, as
// 8192 x 4095, which takes 34 element by element).
template <class T>
struct Raw {
  static constexpr int N = 16 / static_cast<int>(sizeof(T));
  uint32_t w[4];
  __device__ inline void load(const T *p) {
    const words_t v = *reinterpret_cast<const words_t *>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = v[i];
  }
  __device__ inline float at(int i) const {
    if constexpr (sizeof(T) == 4) {
      return __uint_as_float(w[i]);
    } else {
      const uint32_t u = w[i / 2];
      if constexpr (std::is_same_v<T, __bf16>)
        return __uint_as_float(i & 1 ? u & 0xffff0000u : u << 16);
      else
        return widen(__builtin_bit_cast(_Float16, static_cast<uint16_t>(i & 1 ? u >> 16 : u)));
    }
  }
};
template <class T>
struct Scalar {  // one element, for rows below 16 bytes
  static constexpr int N = 1;
  T v;
  __device__ inline void load(const T *p) { v = *p; }
  __device__ inline float at(int) const { return widen(v); }
};

typedef unsigned short u16x2_t __attribute__((ext_vector_type(2)));

// Largest magnitude seen, as bits.
template <class T>
struct Magnitude {
  uint32_t bits = 0;
  __device__ inline void look(const Raw<T> &r) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (sizeof(T) == 4) {
        const uint32_t u = r.w[i] & 0x7fffffffu;
        bits = u > bits ? u : bits;
      } else {
        bits = __builtin_bit_cast(
            uint32_t, __builtin_elementwise_max(
                          __builtin_bit_cast(u16x2_t, bits),
                          __builtin_bit_cast(u16x2_t, r.w[i] & 0x7fff7fffu)));
      }
    }
  }
  __device__ inline void look(const Scalar<T> &r) {
    if constexpr (sizeof(T) == 4) {
      const uint32_t u = __float_as_uint(r.v) & 0x7fffffffu;
      bits = u > bits ? u : bits;
    } else {
      const uint32_t u = __builtin_bit_cast(uint16_t, r.v) & 0x7fffu;
      bits = u > bits ? u : bits;
    }
  }
  // As a float; infinity for NaN.
  __device__ inline float value() const {
    if constexpr (sizeof(T) == 4) {
      return __uint_as_float(bits > 0x7f800000u ? 0x7f800000u : bits);
    } else {
      const uint32_t u = (bits & 0xffff) > (bits >> 16) ? bits & 0xffff : bits >> 16;
      constexpr uint32_t inf = std::is_same_v<T, __bf16> ? 0x7f80u : 0x7c00u;
      return u >= inf ? INFINITY : widen(__builtin_bit_cast(T, static_cast<uint16_t>(u)));
    }
  }
};

template <class T, class R, int TPR, int P>
__global__ __launch_bounds__(kThreads) void quantize_kernel(const T *x, int64_t n_rows, int64_t ld,
                                                            int32_t n, int8_t *q, float *scale) {
  constexpr int N = R::N, W = kThreads / 64;
  const int64_t r = static_cast<int64_t>(blockIdx.x) * (kThreads / TPR) + threadIdx.x / TPR;
  if (TPR == 64 && r >= n_rows) return;  // whole waves; no barrier below then
  const int64_t first = threadIdx.x % TPR * N;
  const T *row = x + r * ld;
  R held[P];
  Magnitude<T> seen;
#pragma unroll
  for (int p = 0; p < P; ++p)
    if (first + p * TPR * N < n) held[p].load(row + piece_at<N>(first + p * TPR * N, n));
#pragma unroll
  for (int p = 0; p < P; ++p)
    if (first + p * TPR * N < n) seen.look(held[p]);
  for (int64_t col = first + P * TPR * N; col < n; col += TPR * N) {
    R v;
    v.load(row + piece_at<N>(col, n));
    seen.look(v);
  }
  float most = seen.value();
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) most = fmaxf(most, __shfl_xor(most, m));
  if constexpr (TPR > 64) {
    __shared__ float part[W];
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = most;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < W; ++w) most = fmaxf(most, part[w]);
  }
  const float s = most * static_cast<float>(1.0 / 127.0);
  const bool plain = s > 0.f && most < INFINITY;
  if (first == 0) scale[r] = most < INFINITY ? s : __uint_as_float(0x7fc00000u);
  // 0: divide (a scale so small that its reciprocal overflows)
  const float inv = s >= 1e-37f ? 1.f / s : 0.f;
  auto put = [&](int64_t begin, const R &v) {
    struct { int8_t e[N]; } o;
    float off = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float f = v.at(i) * inv, t = f + 12582912.f;
      off = fmaxf(off, fabsf(f - (t - 12582912.f)));
      o.e[i] = static_cast<int8_t>(__float_as_uint(t));
    }
    if (!(off < 0.4999f) || inv == 0.f || !plain) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float f = plain ? rintf(v.at(i) / s) : 0.f;
        // a subnormal scale may round so far down that a quotient passes 127
        o.e[i] = static_cast<int8_t>(fminf(fmaxf(f, -127.f), 127.f));
      }
    }
    __builtin_memcpy(q + r * n + piece_at<N>(begin, n), &o, N);
  };
#pragma unroll
  for (int p = 0; p < P; ++p)
    if (first + p * TPR * N < n) put(first + p * TPR * N, held[p]);
  for (int64_t col = first + P * TPR * N; col < n; col += TPR * N) {
    R v;
    v.load(row + piece_at<N>(col, n));
    put(col, v);
  }
}

template <class F>
int by_type(int32_t dtype, F f) {
  if (dtype == EJ_F32) return f(static_cast<float *>(nullptr));
  if (dtype == EJ_BF16) return f(static_cast<__bf16 *>(nullptr));
  if (dtype == EJ_F16) return f(static_cast<_Float16 *>(nullptr));
  set_error("values of dtype %d: expected EJ_F32, EJ_BF16 or EJ_F16", dtype);
  return EJ_E_INVAL;
}

int check_combine(int64_t n_slots, int64_t n_tokens, int32_t k, int32_t n) {
  EJ_CHECK_ARG(n_slots >= 0 && n_tokens >= 0 && n >= 0, "negative size");
  EJ_CHECK_ARG(k >= 1, "k = %d, expected at least 1", k);
  if (k > EJ_MAX_PICKS || n_tokens >= ((int64_t{1} << 31) + k - 1) / k ||
      n_slots >= (int64_t{1} << 31)) {
    set_error("%lld tokens of %d picks, %lld slots: at most %d picks and fewer than 2^31 pairs "
              "and slots are supported", (long long)n_tokens, k, (long long)n_slots, EJ_MAX_PICKS);
    return EJ_E_UNSUPPORTED;
  }
  return EJ_OK;
}

// launch(first, count) for ranges of tokens, of which a launch holds `most`
// (a first range also where there are none).
template <class F>
int by_tokens(int64_t n_tokens, int64_t most, F launch) {
  int64_t first = 0;
  do {
    const int64_t count = n_tokens - first < most ? n_tokens - first : most;
    launch(first, count);
    EJ_LAUNCH_CHECK();
    first += count;
  } while (first < n_tokens);
  return EJ_OK;
}

}  // namespace
}  // namespace ej

using namespace ej;

extern "C" int ej_expert_combine(const void *y, int32_t dtype, int64_t n_slots, int64_t ld_y,
                                 const float *weights, const int32_t *slots, int64_t n_tokens,
                                 int32_t k, int32_t n, void *out, int32_t out_dtype,
                                 ej_stream_t stream) {
  EJ_TRY(check_combine(n_slots, n_tokens, k, n));
  EJ_CHECK_ARG(out_dtype == dtype || dtype == EJ_F32, "a sum of dtype %d from values of dtype %d",
               out_dtype, dtype);
  return by_type(dtype, [&](auto *tp) {
    return by_type(out_dtype, [&](auto *op) {
      using T = std::remove_pointer_t<decltype(tp)>;
      using O = std::remove_pointer_t<decltype(op)>;
      if constexpr (std::is_same_v<T, O> || std::is_same_v<T, float>) {
        if (n_tokens == 0 || n == 0) return EJ_OK;
        EJ_CHECK_ARG(slots && out && (y || n_slots == 0), "null argument");
        EJ_CHECK_ARG(ld_y >= n, "row stride %lld below n = %d", (long long)ld_y, n);
        CombineArgs a{y, ld_y, n, n_slots, k, n, weights, slots, out};
        constexpr int N = 16 / sizeof(T);
        const bool vec = n >= N;
        const int64_t cols = ceil_div(n, static_cast<int64_t>(kThreads) * (vec ? N : 1));
        return by_tokens(n_tokens, kMaxBlocks / cols, [&](int64_t first, int64_t count) {
          CombineArgs b = a;
          b.slots += first * k;
          if (b.weights) b.weights += first * k;
          b.out = static_cast<O *>(out) + first * n;
          hipLaunchKernelGGL((vec ? combine_kernel<T, O, true> : combine_kernel<T, O, false>),
                             dim3(static_cast<unsigned>(count * cols)), dim3(kThreads), 0,
                             as_stream(stream), b, static_cast<unsigned>(cols));
        });
      }
      return EJ_OK;
    });
  });
}

extern "C" int ej_expert_combine_vjp(const void *y, int32_t dtype, int64_t n_slots, int64_t ld_y,
                                     const float *weights, const int32_t *slots,
                                     const int32_t *offsets, int32_t n_groups, int64_t n_tokens,
                                     int32_t k, int32_t n, const void *grad, int64_t ld_grad,
                                     void *grad_y, float *grad_weights, ej_stream_t stream) {
  EJ_TRY(check_combine(n_slots, n_tokens, k, n));
  EJ_CHECK_ARG(n_groups >= 0, "negative n_groups");
  return by_type(dtype, [&](auto *tp) {
    using T = std::remove_pointer_t<decltype(tp)>;
    if (!grad_y && !grad_weights) return EJ_OK;
    if (n_slots == 0 && n_tokens == 0) return EJ_OK;
    EJ_CHECK_ARG(offsets && (n_tokens == 0 || (slots && (grad || n == 0))), "null argument");
    EJ_CHECK_ARG(ld_y >= n && ld_grad >= n, "row stride below n = %d", n);
    CombineArgs a{y, ld_y, n, n_slots, k, n, weights, slots, nullptr};
    auto run = [&](auto kernel) {
      return by_tokens(n_tokens, kMaxBlocks - kZeroBlocks, [&](int64_t first, int64_t count) {
        CombineArgs b = a;
        b.slots += first * k;
        if (b.weights) b.weights += first * k;
        const int zeroing = first == 0 && grad_y ? kZeroBlocks : 0;
        if (count + zeroing == 0) return;
        hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(count + zeroing)), dim3(kThreads), 0,
                           as_stream(stream), b,
                           static_cast<const T *>(grad) + first * ld_grad, ld_grad, grad_y,
                           grad_weights ? grad_weights + first * k : nullptr, zeroing,
                           n_tokens * k);
      });
    };
    // Rows of no whole pieces, 16384 tokens of 4 picks, with the last piece moved
    // back and element by element: bf16 4095 columns 311 and 609 us, f16 1001
    // 109 and 155, 501 57 and 61, 150 53 and 39; fp32 2047 276 and 280, 501 110
    // and 81.
    if (n % (16 / static_cast<int>(sizeof(T))) == 0)
      return run(combine_vjp_kernel<T, true, true>);
    if (sizeof(T) == 2 && n >= 512)
      return run(combine_vjp_kernel<T, sizeof(T) == 2, false>);
    return run(combine_vjp_kernel<T, false, true>);
  });
}

extern "C" int ej_quantize_rows(const void *x, int32_t dtype, int64_t n_rows, int64_t ld,
                                int32_t n, int8_t *q, float *scale, ej_stream_t stream) {
  EJ_CHECK_ARG(n_rows >= 0 && n >= 0, "negative size");
  return by_type(dtype, [&](auto *tp) {
    using T = std::remove_pointer_t<decltype(tp)>;
    if (n_rows == 0) return EJ_OK;
    EJ_CHECK_ARG(scale && (n == 0 || (x && q)), "null argument");
    EJ_CHECK_ARG(ld >= n, "row stride %lld below n = %d", (long long)ld, n);
    if (n_rows > kMaxBlocks) {
      set_error("%lld rows: too many for one launch", (long long)n_rows);
      return EJ_E_UNSUPPORTED;
    }
    constexpr int N = 16 / sizeof(T);
    const bool vec = n >= N;
    const T *xt = static_cast<const T *>(x);
    auto run = [&](auto kernel, int64_t blocks) {
      hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(blocks)), dim3(kThreads), 0,
                         as_stream(stream), xt, n_rows, ld, n, q, scale);
    };
    // a wave a row where there are rows enough to fill the CUs and a row fits
    // its registers; otherwise a workgroup a row
    constexpr int kHeld = 8;
    if (vec && n_rows >= 1024 && n <= 64 * N * kHeld)
      run(quantize_kernel<T, Raw<T>, 64, kHeld>, ceil_div(n_rows, kThreads / 64));
    else if (vec)
      run(quantize_kernel<T, Raw<T>, kThreads, 4>, n_rows);
    else
      run(quantize_kernel<T, Scalar<T>, kThreads, 8>, n_rows);
    EJ_LAUNCH_CHECK();
    return EJ_OK;
  });
}
