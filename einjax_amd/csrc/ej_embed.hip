// Rows of a table for tokens, and the gradient to the table.
//
//   out[t] = scale table[tokens[t]]
//   grad_table[v] = scale sum over t with tokens[t] = v of grad[t]
//
// A token outside the table (padding) has a row of zeros and no gradient.  The
// lookup is a relation of tokens and rows; its gradient is the segment sum over
// the tokens in the order of their rows, and of equal ones in their own, so the
// sums are formed in one order whatever ran when, without atomics.
#include <type_traits>

#include "ej_internal.h"

namespace ej {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxBlocks = (1 << 24) - 1;  // of 256 threads in a launch

template <class T>
constexpr int kPiece = 16 / static_cast<int>(sizeof(T));

// A 16-byte piece of a row, anywhere in it; `there` of its values exist.
template <class T>
struct Piece {
  T e[kPiece<T>];
  __device__ inline void load(const T *p, int there) {
    if (there >= kPiece<T>) {
      __builtin_memcpy(e, __builtin_assume_aligned(p, alignof(T)), 16);
    } else {
#pragma unroll
      for (int i = 0; i < kPiece<T>; ++i)
        if (i < there) e[i] = p[i];
    }
  }
  __device__ inline void store(T *p, int there) const {
    if (there >= kPiece<T>) {
      __builtin_memcpy(__builtin_assume_aligned(p, alignof(T)), e, 16);
    } else {
#pragma unroll
      for (int i = 0; i < kPiece<T>; ++i)
        if (i < there) p[i] = e[i];
    }
  }
};

// The row of a token, n_rows for those outside the table.
__device__ inline uint32_t row_of(int64_t token, uint32_t n_rows) {
  return token >= 0 && token < n_rows ? static_cast<uint32_t>(token) : n_rows;
}

// Threads that take one row's pieces side by side: a power of two.
inline int row_threads(int64_t pieces) {
  int t = 1;
  while (t < kThreads && t < pieces) t *= 2;
  return t;
}

// ---- the lookup -------------------------------------------------------------

template <class T, class Token>
__global__ __launch_bounds__(kThreads) void embed_kernel(const T *table, uint32_t n_rows,
                                                         int64_t ld, int32_t n,
                                                         const Token *tokens, int64_t n_tokens,
                                                         float scale, int32_t across, T *out) {
  constexpr int N = kPiece<T>;
  const int64_t t = static_cast<int64_t>(blockIdx.x) * (kThreads / across) + threadIdx.x / across;
  if (t >= n_tokens) return;
  const uint32_t row = row_of(tokens[t], n_rows);
  const bool held = row < n_rows;
  const T *src = table + (held ? row : 0) * ld;
  T *dst = out + t * n;
#pragma unroll 2
  for (int32_t c = (threadIdx.x & (across - 1)) * N; c < n; c += across * N) {
    Piece<T> v;
    if (held) v.load(src + c, n - c);
#pragma unroll
    for (int i = 0; i < N; ++i)
      v.e[i] = held ? static_cast<T>(static_cast<float>(v.e[i]) * scale) : static_cast<T>(0.f);
    v.store(dst + c, n - c);
  }
}

// ---- the order of the tokens -------------------------------------------------

// Zeros, 16 bytes a thread: the workgroups of a launch from `first` on.
template <class T>
__device__ inline void fill_zero(T *p, int64_t count, uint32_t first) {
  constexpr int N = kPiece<T>;
  const int64_t threads = static_cast<int64_t>(gridDim.x - first) * blockDim.x;
  Piece<T> zero;
#pragma unroll
  for (int i = 0; i < N; ++i) zero.e[i] = static_cast<T>(0.f);
  for (int64_t i = (static_cast<int64_t>(blockIdx.x - first) * blockDim.x + threadIdx.x) * N;
       i < count; i += threads * N)
    zero.store(p + i, count - i < N ? static_cast<int>(count - i) : N);
}

// Few tokens: each token's place is the number of tokens before it, by
// comparison with every other one, in one launch.  A workgroup places 64 tokens,
// one a lane; its 16 waves share out the tokens to compare with, which are
// uniform and come through the scalar cache.  The workgroups behind those clear
// the gradient meanwhile.
constexpr int kRankWaves = 16;
constexpr int64_t kRankTokens = 16384;

template <class T, class Token>
__global__ __launch_bounds__(kRankWaves * 64) void rank_kernel(
    const Token *tokens, int32_t n_tokens, uint32_t n_rows, uint32_t *keys, int32_t *perm,
    uint32_t rank_blocks, T *clear, int64_t clear_count) {
  if (blockIdx.x >= rank_blocks) {
    fill_zero(clear, clear_count, rank_blocks);
    return;
  }
  __shared__ int32_t counts[kRankWaves][64];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int32_t first = blockIdx.x * 64, i = first + lane;
  const uint32_t mine = i < n_tokens ? row_of(tokens[i], n_rows) : n_rows;
  const auto *all = (const __attribute__((address_space(4))) Token *)(tokens);
  const int32_t per = (n_tokens + kRankWaves - 1) / kRankWaves;
  const int32_t lo = wave * per, hi = lo + per < n_tokens ? lo + per : n_tokens;
  int32_t count = 0;
  auto span = [&](int32_t a, int32_t b, uint32_t below) {
    int32_t j = a;
    for (; j + 16 <= b; j += 16)
#pragma unroll
      for (int u = 0; u < 16; ++u) count += row_of(all[j + u], n_rows) < below;
    for (; j < b; ++j) count += row_of(all[j], n_rows) < below;
  };
  // tokens before this workgroup's, equal ones counted; its own; those behind
  span(lo, hi < first ? hi : first, mine + 1);
  for (int32_t j = lo > first ? lo : first; j < hi && j < first + 64; ++j)
    count += row_of(all[j], n_rows) < mine + (j < i ? 1 : 0);
  span(lo > first + 64 ? lo : first + 64, hi, mine);
  counts[wave][lane] = count;
  __syncthreads();
  if (wave == 0 && i < n_tokens) {
    int32_t place = 0;
#pragma unroll
    for (int w = 0; w < kRankWaves; ++w) place += counts[w][lane];
    keys[place] = mine;
    perm[place] = i;
  }
}

// More: keys for the radix sort, and its result in 32 bits.
template <class T, class Token>
__global__ __launch_bounds__(kThreads) void sort_keys_kernel(const Token *tokens, int32_t n_tokens,
                                                             uint32_t n_rows, uint64_t *keys,
                                                             int32_t *perm, uint32_t key_blocks,
                                                             T *clear, int64_t clear_count) {
  if (blockIdx.x >= key_blocks) {
    fill_zero(clear, clear_count, key_blocks);
    return;
  }
  const int32_t i = blockIdx.x * kThreads + threadIdx.x;
  if (i >= n_tokens) return;
  keys[i] = row_of(tokens[i], n_rows);
  perm[i] = i;
}

__global__ __launch_bounds__(kThreads) void narrow_keys_kernel(const uint64_t *from,
                                                               int32_t n_tokens, uint32_t *to) {
  const int32_t i = blockIdx.x * kThreads + threadIdx.x;
  if (i < n_tokens) to[i] = static_cast<uint32_t>(from[i]);
}

// ---- the sums -----------------------------------------------------------------

// The sorted tokens in chunks of equal length.  A row whose tokens lie in one
// chunk is written at once; of one that spans several, each chunk leaves its
// part in fp32: `head` where the row began in an earlier chunk, `tail` where it
// began in this one.
struct Sums {
  const uint32_t *keys;
  const int32_t *perm;
  int32_t n_tokens, chunk;
  uint32_t n_rows;
  int32_t n, across;
  int64_t ld;  // of the gradient's rows
  float scale;
  float *parts;  // [chunks][head, tail][n]
  __device__ inline float *part(int64_t c, int tail) const { return parts + (c * 2 + tail) * n; }
};

template <class T>
__device__ inline void put_row(const Sums &s, T *out, uint32_t row, int32_t col,
                               const float (&sum)[kPiece<T>]) {
  Piece<T> v;
#pragma unroll
  for (int i = 0; i < kPiece<T>; ++i) v.e[i] = static_cast<T>(s.scale * sum[i]);
  v.store(out + static_cast<int64_t>(row) * s.n + col, s.n - col);
}

template <int N>
__device__ inline void put_part(float *p, int there, const float (&sum)[N]) {
  if (there >= N) {
    __builtin_memcpy(__builtin_assume_aligned(p, 4), sum, sizeof(sum));
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (i < there) p[i] = sum[i];
  }
}
template <int N>
__device__ inline void add_part(const float *p, int there, float (&sum)[N]) {
  float v[N] = {};
  if (there >= N) {
    __builtin_memcpy(v, __builtin_assume_aligned(p, 4), sizeof(v));
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (i < there) v[i] = p[i];
  }
#pragma unroll
  for (int i = 0; i < N; ++i) sum[i] += v[i];
}

template <class T>
__global__ __launch_bounds__(kThreads) void sum_chunks_kernel(Sums s, const T *grad, T *out) {
  constexpr int N = kPiece<T>, kAhead = 8;
  const int64_t c = static_cast<int64_t>(blockIdx.x) * (kThreads / s.across) +
                    threadIdx.x / s.across;
  const int32_t col = (blockIdx.y * s.across + (threadIdx.x & (s.across - 1))) * N;
  const int64_t p0 = c * s.chunk;
  if (p0 >= s.n_tokens || col >= s.n) return;
  const int32_t p1 = p0 + s.chunk < s.n_tokens ? static_cast<int32_t>(p0) + s.chunk : s.n_tokens;
  const int there = s.n - col;
  uint32_t row = s.keys[p0];
  bool head = p0 > 0 && s.keys[p0 - 1] == row;
  float sum[N] = {};
  auto finish = [&](bool goes_on) {
    if (row >= s.n_rows) return;
    if (head) put_part(s.part(c, 0) + col, there, sum);
    else if (goes_on) put_part(s.part(c, 1) + col, there, sum);
    else put_row(s, out, row, col, sum);
  };
  for (int32_t p = static_cast<int32_t>(p0); p < p1; p += kAhead) {
    uint32_t key[kAhead];
    Piece<T> v[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      key[u] = p + u < p1 ? s.keys[p + u] : s.n_rows;
      if (key[u] < s.n_rows) v[u].load(grad + s.perm[p + u] * s.ld + col, there);
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      if (p + u >= p1) break;
      if (key[u] != row) {
        finish(false);
        row = key[u];
        head = false;
#pragma unroll
        for (int i = 0; i < N; ++i) sum[i] = 0.f;
      }
      if (row >= s.n_rows) return;  // padding sorts last
#pragma unroll
      for (int i = 0; i < N; ++i) sum[i] += static_cast<float>(v[u].e[i]);
    }
  }
  finish(p1 < s.n_tokens && s.keys[p1] == row);
}

// Rows that span chunks: the tail of the chunk that a row began in and the heads
// of the next ones, added in their order.
template <class T>
__global__ __launch_bounds__(kThreads) void join_chunks_kernel(Sums s, T *out) {
  constexpr int N = kPiece<T>;
  const int64_t c = static_cast<int64_t>(blockIdx.x) * (kThreads / s.across) +
                    threadIdx.x / s.across;
  const int32_t col = (blockIdx.y * s.across + (threadIdx.x & (s.across - 1))) * N;
  const int64_t p0 = c * s.chunk, p1 = p0 + s.chunk;
  if (p1 >= s.n_tokens || col >= s.n) return;
  const uint32_t row = s.keys[p1 - 1];
  const bool began = s.keys[p0] != row || p0 == 0 || s.keys[p0 - 1] != row;
  if (row >= s.n_rows || !began || s.keys[p1] != row) return;
  const int there = s.n - col;
  float sum[N] = {};
  add_part(s.part(c, 1) + col, there, sum);
  for (int64_t next = c + 1; next * s.chunk < s.n_tokens && s.keys[next * s.chunk] == row;
       ++next)
    add_part(s.part(next, 0) + col, there, sum);
  put_row(s, out, row, col, sum);
}

// ---- host ------------------------------------------------------------------------

// Tokens of a chunk: 32, more where that gives above 2048 chunks (whose parts
// one thread may have to add up).
int32_t chunk_of(int64_t n_tokens) {
  int64_t c = 32;
  while (ceil_div(n_tokens, c) > 2048) c *= 2;
  return static_cast<int32_t>(c);
}

struct Plan {
  uint32_t *keys;
  int32_t *perm;
  float *parts;
  uint64_t *keys64, *keys_alt;
  int32_t *perm_alt;
  char *sort;
  size_t bytes;
};

Plan carve(void *base, int64_t n_tokens, int64_t n) {
  Carver c(base);
  Plan p = {};
  p.keys = c.take<uint32_t>(n_tokens);
  p.perm = c.take<int32_t>(n_tokens);
  p.parts = c.take<float>(2 * n * ceil_div(n_tokens, chunk_of(n_tokens)));
  if (n_tokens > kRankTokens) {
    p.keys64 = c.take<uint64_t>(n_tokens);
    p.keys_alt = c.take<uint64_t>(n_tokens);
    p.perm_alt = c.take<int32_t>(n_tokens);
    p.sort = c.take<char>(static_cast<int64_t>(sort_workspace_bytes(n_tokens)));
  }
  p.bytes = c.off;
  return p;
}

int check_sizes(int64_t n_tokens, int64_t n_rows, int32_t n) {
  EJ_CHECK_ARG(n_tokens >= 0 && n_rows >= 0 && n >= 0, "negative size");
  if (n_rows >= INT32_MAX || n_tokens > INT32_MAX - kThreads || n > INT32_MAX - 8 * kThreads) {
    set_error("%lld tokens of %lld rows of %d: fewer than 2^31 of each are supported",
              (long long)n_tokens, (long long)n_rows, n);
    return EJ_E_UNSUPPORTED;
  }
  return EJ_OK;
}

template <class F>
int by_types(int32_t dtype, int32_t token_dtype, F f) {
  auto with = [&](auto *t) {
    return token_dtype == EJ_I32 ? f(t, static_cast<const int32_t *>(nullptr))
                                 : f(t, static_cast<const int64_t *>(nullptr));
  };
  EJ_CHECK_ARG(token_dtype == EJ_I32 || token_dtype == EJ_I64,
               "tokens of dtype %d: expected EJ_I32 or EJ_I64", token_dtype);
  if (dtype == EJ_F32) return with(static_cast<float *>(nullptr));
  if (dtype == EJ_BF16) return with(static_cast<__bf16 *>(nullptr));
  if (dtype == EJ_F16) return with(static_cast<_Float16 *>(nullptr));
  set_error("values of dtype %d: expected EJ_F32, EJ_BF16 or EJ_F16", dtype);
  return EJ_E_INVAL;
}

int too_many(const char *what, int64_t n) {
  set_error("%lld %s: too many for one launch", (long long)n, what);
  return EJ_E_UNSUPPORTED;
}

// Workgroups that clear `bytes`: enough to fill the CUs, not more than there is
// for each.
int64_t clear_blocks(int64_t bytes, int threads) {
  const int64_t most = ceil_div(bytes, static_cast<int64_t>(threads) * 64);
  const int64_t full = 256 * 2048 / threads;
  return most < full ? most : full;
}

}  // namespace
}  // namespace ej

using namespace ej;

extern "C" int ej_embed(const void *table, int32_t dtype, int64_t n_rows, int64_t ld, int32_t n,
                        const void *tokens, int32_t token_dtype, int64_t n_tokens, float scale,
                        void *out, ej_stream_t stream) {
  return by_types(dtype, token_dtype, [&](auto *tp, auto *kp) {
    using T = std::remove_pointer_t<decltype(tp)>;
    using Token = std::remove_cv_t<std::remove_pointer_t<decltype(kp)>>;
    EJ_TRY(check_sizes(n_tokens, n_rows, n));
    EJ_CHECK_ARG(ld >= n, "row stride %lld below n = %d", (long long)ld, n);
    if (n_tokens == 0 || n == 0) return EJ_OK;
    EJ_CHECK_ARG(tokens && out && (table || n_rows == 0), "null argument");
    const int across = row_threads(ceil_div(n, kPiece<T>));
    const int64_t blocks = ceil_div(n_tokens, kThreads / across);
    if (blocks > kMaxBlocks) return too_many("tokens", n_tokens);
    hipLaunchKernelGGL((embed_kernel<T, Token>), dim3(static_cast<unsigned>(blocks)),
                       dim3(kThreads), 0, as_stream(stream), static_cast<const T *>(table),
                       static_cast<uint32_t>(n_rows), ld, n, static_cast<const Token *>(tokens),
                       n_tokens, scale, across, static_cast<T *>(out));
    EJ_LAUNCH_CHECK();
    return EJ_OK;
  });
}

extern "C" int ej_embed_vjp_workspace_size(int64_t n_tokens, int64_t n_rows, int32_t n,
                                           size_t *bytes) {
  EJ_TRY(check_sizes(n_tokens, n_rows, n));
  EJ_CHECK_ARG(bytes, "null bytes");
  *bytes = n_tokens && n_rows && n ? carve(nullptr, n_tokens, n).bytes : 0;
  return EJ_OK;
}

extern "C" int ej_embed_vjp(const void *tokens, int32_t token_dtype, int64_t n_tokens,
                            const void *grad, int32_t dtype, int64_t grad_ld, int64_t n_rows,
                            int32_t n, float scale, void *grad_table, void *workspace,
                            size_t workspace_bytes, ej_stream_t stream_) {
  return by_types(dtype, token_dtype, [&](auto *tp, auto *kp) {
    using T = std::remove_pointer_t<decltype(tp)>;
    using Token = std::remove_cv_t<std::remove_pointer_t<decltype(kp)>>;
    EJ_TRY(check_sizes(n_tokens, n_rows, n));
    EJ_CHECK_ARG(grad_ld >= n, "row stride %lld below n = %d", (long long)grad_ld, n);
    if (n_rows == 0 || n == 0) return EJ_OK;
    EJ_CHECK_ARG(grad_table, "null result");
    EJ_CHECK_ARG(n_tokens == 0 || (tokens && grad), "null argument");
    const hipStream_t stream = as_stream(stream_);
    T *out = static_cast<T *>(grad_table);
    const Token *tok = static_cast<const Token *>(tokens);
    const int64_t count = n_rows * static_cast<int64_t>(n);
    const int64_t bytes = count * static_cast<int64_t>(sizeof(T));
    const int32_t m = static_cast<int32_t>(n_tokens);
    const uint32_t rows = static_cast<uint32_t>(n_rows);
    const Plan p = n_tokens ? carve(workspace, n_tokens, n) : Plan{};
    EJ_CHECK_ARG(n_tokens == 0 || (workspace && workspace_bytes >= p.bytes),
                 "workspace of %zu bytes, expected %zu", workspace_bytes, p.bytes);
    Sums s = {p.keys, p.perm, m, chunk_of(n_tokens), rows, n, 0, grad_ld, scale, p.parts};
    s.across = row_threads(ceil_div(n, kPiece<T>));
    const int64_t chunks = ceil_div(n_tokens, s.chunk);
    const int64_t cols = ceil_div(n, static_cast<int64_t>(s.across) * kPiece<T>);
    const int64_t sum_blocks = ceil_div(chunks, kThreads / s.across);
    if (sum_blocks * cols > kMaxBlocks || cols > 65535) return too_many("columns", n);
    if (n_tokens <= kRankTokens) {
      constexpr int kT = kRankWaves * 64;
      const int64_t blocks = ceil_div(n_tokens, 64);
      hipLaunchKernelGGL((rank_kernel<T, Token>),
                         dim3(static_cast<unsigned>(blocks + clear_blocks(bytes, kT))), dim3(kT), 0,
                         stream, tok, m, rows, p.keys, p.perm, static_cast<uint32_t>(blocks), out,
                         count);
      EJ_LAUNCH_CHECK();
    } else {
      const int64_t blocks = ceil_div(n_tokens, kThreads);
      hipLaunchKernelGGL((sort_keys_kernel<T, Token>),
                         dim3(static_cast<unsigned>(blocks + clear_blocks(bytes, kThreads))),
                         dim3(kThreads), 0, stream, tok, m, rows, p.keys64, p.perm,
                         static_cast<uint32_t>(blocks), out, count);
      EJ_LAUNCH_CHECK();
      int bits = 1;
      while (n_rows >> bits) ++bits;  // keys up to n_rows
      EJ_TRY(sort_pairs_u64(p.keys64, p.perm, p.keys_alt, p.perm_alt, n_tokens, bits, p.sort,
                            stream, false, nullptr, false));
      hipLaunchKernelGGL(narrow_keys_kernel, dim3(static_cast<unsigned>(blocks)), dim3(kThreads),
                         0, stream, p.keys64, m, p.keys);
      EJ_LAUNCH_CHECK();
    }
    if (n_tokens == 0) return EJ_OK;
    const dim3 grid(static_cast<unsigned>(sum_blocks), static_cast<unsigned>(cols));
    hipLaunchKernelGGL(sum_chunks_kernel<T>, grid, dim3(kThreads), 0, stream, s,
                       static_cast<const T *>(grad), out);
    EJ_LAUNCH_CHECK();
    if (chunks > 1) {
      hipLaunchKernelGGL(join_chunks_kernel<T>, grid, dim3(kThreads), 0, stream, s, out);
      EJ_LAUNCH_CHECK();
    }
    return EJ_OK;
  });
}
