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

// N values of a row, from any element on.  A row is covered by whole pieces: the
// last one begins N before its end, and what it shares with the one before is
// computed twice.  (A branch for a short piece would have every load waited for
// before the next one.)  Rows of fewer than 16 bytes go by single values.
template <class T, int N>
struct Piece {
  T e[N];
  __device__ inline void load(const T *p) {
    __builtin_memcpy(e, __builtin_assume_aligned(p, alignof(T)), sizeof(e));
  }
  __device__ inline void store(T *p) const {
    __builtin_memcpy(__builtin_assume_aligned(p, alignof(T)), e, sizeof(e));
  }
};
template <int N>
__device__ inline int32_t piece_at(int32_t col, int32_t n) {
  return col <= n - N ? col : n - N;
}

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

// A thread takes a token's pieces, its row's threads apart.  Bound by memory: 16384
// tokens of 32768 x 4096 bf16 41 us, 4096 tokens 12 (two rows a thread at a time
// 42 and 12, four 43 and 12.5, eight 47 and 14); a few tokens: the launch.
template <class T, class Token, int N>
__global__ __launch_bounds__(kThreads) void embed_kernel(const T *table, uint32_t n_rows,
                                                         int64_t ld, int32_t n,
                                                         const Token *tokens, int64_t n_tokens,
                                                         float scale, int32_t across, T *out) {
  const int64_t t = static_cast<int64_t>(blockIdx.x) * (kThreads / across) + threadIdx.x / across;
  if (t >= n_tokens) return;
  const uint32_t row = row_of(tokens[t], n_rows);
  const bool there = row < n_rows;
  for (int32_t c = (threadIdx.x & (across - 1)) * N; c < n; c += across * N) {
    const int32_t col = piece_at<N>(c, n);
    Piece<T, N> v;
    // row 0 for a token outside: a table has one (n_rows 0: none is read)
    if (n_rows) v.load(table + (there ? row : 0) * ld + col);
#pragma unroll
    for (int i = 0; i < N; ++i)
      v.e[i] = there ? static_cast<T>(static_cast<float>(v.e[i]) * scale) : static_cast<T>(0.f);
    v.store(out + t * n + col);
  }
}

// ---- the order of the tokens -------------------------------------------------

// Zeros, 16 bytes a thread at a time: by the workgroups of a launch from `first` on.
template <class T>
__device__ inline void fill_zero(T *p, int64_t count, uint32_t first) {
  constexpr int N = kPiece<T>;
  const int64_t threads = static_cast<int64_t>(gridDim.x - first) * blockDim.x;
  const int64_t mine = static_cast<int64_t>(blockIdx.x - first) * blockDim.x + threadIdx.x;
  Piece<T, N> zero;
#pragma unroll
  for (int i = 0; i < N; ++i) zero.e[i] = static_cast<T>(0.f);
  for (int64_t i = mine; i < count / N; i += threads) zero.store(p + i * N);
  if (mine < count % N) p[count / N * N + mine] = static_cast<T>(0.f);
}

// LDS accesses of the wave's lanes before and behind stay in this order.
__device__ inline void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// Few tokens: one workgroup sorts them in LDS, digit by digit, in one launch; the
// workgroups behind it clear the gradient meanwhile.  Each of its 16 waves takes
// a run of the sequence, 64 tokens at a time.  A pass counts every wave's digits,
// scans the counts by digit and then by wave, and places the tokens in order:
// those of a 64 with the same digit know each other by ballots of its bits.  16384
// tokens of 50000 rows: 40 us with a gradient of 64 columns, where the sort counts
// alone, 59 with one of 4096 (410 MB, whose clearing alone takes 58); 2000 tokens 10.
// 16384 tokens, a power of two, take 112 of the CU's 160 KB.  The whole gradient (us),
// 50000 rows of bf16: 4096 columns 150 and, by the radix sort, 157 for one token more;
// 64 columns, where nothing hides the sort, 50 and 32 (8192 tokens 33, 2000 18): so
// narrow tables lose here from some 8000 tokens on.
constexpr int kSortWaves = 16, kSortThreads = kSortWaves * 64;
constexpr int kSortBits = 8, kSortDigits = 1 << kSortBits;
constexpr int kSortTokens = 16384, kSortRows = kSortTokens / kSortThreads;

template <class T, class Token>
__global__ __launch_bounds__(kSortThreads) void sort_few_kernel(const Token *tokens,
                                                                int32_t n_tokens, uint32_t n_rows,
                                                                int32_t bits, uint32_t *keys,
                                                                int32_t *perm, T *clear,
                                                                int64_t clear_count) {
  if (blockIdx.x > 0) {
    fill_zero(clear, clear_count, 1);
    return;
  }
  __shared__ uint32_t key_of[kSortTokens];
  __shared__ uint16_t token_of[kSortTokens];
  __shared__ int32_t place[kSortDigits * kSortWaves];
  __shared__ int32_t wave_sum[kSortWaves];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // rows of 64 tokens for each wave
  const int rows = (n_tokens + kSortThreads - 1) / kSortThreads;
  const int32_t first = wave * rows * 64 + lane;
  uint32_t key[kSortRows];
  uint16_t token[kSortRows];
#pragma unroll
  for (int r = 0; r < kSortRows; ++r) {
    const int32_t i = first + r * 64;
    if (r < rows && i < n_tokens) {
      key[r] = row_of(tokens[i], n_rows);
      token[r] = static_cast<uint16_t>(i);
    }
  }
  for (int shift = 0; shift < bits; shift += kSortBits) {
    if (shift > 0) {
#pragma unroll
      for (int r = 0; r < kSortRows; ++r) {
        const int32_t i = first + r * 64;
        if (r < rows && i < n_tokens) {
          key[r] = key_of[i];
          token[r] = token_of[i];
        }
      }
    }
    for (int i = threadIdx.x; i < kSortDigits * kSortWaves; i += kSortThreads) place[i] = 0;
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kSortRows; ++r)
      if (r < rows && first + r * 64 < n_tokens)
        atomicAdd(&place[(key[r] >> shift & (kSortDigits - 1)) * kSortWaves + wave], 1);
    __syncthreads();
    // exclusive scan: four counts a thread
    constexpr int kEach = kSortDigits * kSortWaves / kSortThreads;
    int32_t v[kEach], mine = 0;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      v[i] = place[threadIdx.x * kEach + i];
      mine += v[i];
    }
    int32_t upto = mine;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int32_t below = __shfl_up(upto, d);
      upto += lane >= d ? below : 0;
    }
    if (lane == 63) wave_sum[wave] = upto;
    __syncthreads();
    int32_t before = upto - mine;
    for (int w = 0; w < wave; ++w) before += wave_sum[w];
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      place[threadIdx.x * kEach + i] = before;
      before += v[i];
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kSortRows; ++r) {
      if (r >= rows) break;
      const bool there = first + r * 64 < n_tokens;
      const uint32_t digit = key[r] >> shift & (kSortDigits - 1);
      uint64_t same = __ballot(there);
#pragma unroll
      for (int b = 0; b < kSortBits; ++b) {
        const uint64_t set = __ballot(digit >> b & 1);
        same &= digit >> b & 1 ? set : ~set;
      }
      const int rank = __popcll(same & ((uint64_t{1} << lane) - 1));
      int32_t *at = &place[digit * kSortWaves + wave];
      const int32_t base = there ? *at : 0;
      // every lane has read before the first of each digit moves it on
      wave_sync();
      if (there && rank == 0) *at = base + __popcll(same);
      wave_sync();
      if (there) {
        key_of[base + rank] = key[r];
        token_of[base + rank] = token[r];
      }
    }
    __syncthreads();
  }
  for (int32_t i = threadIdx.x; i < n_tokens; i += kSortThreads) {
    keys[i] = key_of[i];
    perm[i] = token_of[i];
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

// The sorted tokens in chunks of equal length, so that a few tokens that make up
// most of a batch do not leave the rest waiting.  A row whose tokens lie in one
// chunk is written at once; of one that spans several, each chunk leaves its
// part in fp32: `head` where the row began in an earlier chunk, `tail` where it
// began in this one.  Bound by memory: 16384 tokens of 4096 columns in bf16 66 us
// and 10 for the joins, while the caches still write out the cleared gradient.
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

template <class T, int N>
__device__ inline void put_row(const Sums &s, T *out, uint32_t row, int32_t col,
                               const float (&sum)[N]) {
  Piece<T, N> v;
#pragma unroll
  for (int i = 0; i < N; ++i) v.e[i] = static_cast<T>(s.scale * sum[i]);
  v.store(out + static_cast<int64_t>(row) * s.n + col);
}

template <int N>
__device__ inline void put_part(float *p, const float (&sum)[N]) {
  __builtin_memcpy(__builtin_assume_aligned(p, 4), sum, sizeof(sum));
}

template <class T, int N>
__global__ __launch_bounds__(kThreads) void sum_chunks_kernel(Sums s, const T *grad, T *out) {
  constexpr int kAhead = 8;
  const int64_t c = static_cast<int64_t>(blockIdx.x) * (kThreads / s.across) +
                    threadIdx.x / s.across;
  const int32_t first = (blockIdx.y * s.across + (threadIdx.x & (s.across - 1))) * N;
  const int64_t p0 = c * s.chunk;
  if (p0 >= s.n_tokens || first >= s.n) return;
  const int32_t col = piece_at<N>(first, s.n);
  const int32_t p1 = p0 + s.chunk < s.n_tokens ? static_cast<int32_t>(p0) + s.chunk : s.n_tokens;
  uint32_t row = s.keys[p0];
  bool head = p0 > 0 && s.keys[p0 - 1] == row;
  float sum[N] = {};
  auto finish = [&](bool goes_on) {
    if (row >= s.n_rows) return;
    if (head) put_part(s.part(c, 0) + col, sum);
    else if (goes_on) put_part(s.part(c, 1) + col, sum);
    else put_row(s, out, row, col, sum);
  };
  uint32_t key[kAhead], key_next[kAhead];
  int32_t from_next[kAhead];
  auto places = [&](int32_t p, uint32_t(&k)[kAhead], int32_t(&f)[kAhead]) {
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int32_t at = p + u < p1 ? p + u : p1 - 1;
      k[u] = s.keys[at];
      f[u] = s.perm[at];
    }
  };
  places(static_cast<int32_t>(p0), key_next, from_next);
  for (int32_t p = static_cast<int32_t>(p0); p < p1; p += kAhead) {
    Piece<T, N> v[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      key[u] = key_next[u];
      v[u].load(grad + from_next[u] * s.ld + col);
    }
    places(p + kAhead, key_next, from_next);
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
template <class T, int N>
__global__ __launch_bounds__(kThreads) void join_chunks_kernel(Sums s, T *out) {
  const int64_t c = static_cast<int64_t>(blockIdx.x) * (kThreads / s.across) +
                    threadIdx.x / s.across;
  const int32_t first = (blockIdx.y * s.across + (threadIdx.x & (s.across - 1))) * N;
  const int64_t p0 = c * s.chunk, p1 = p0 + s.chunk;
  if (p1 >= s.n_tokens || first >= s.n) return;
  const int32_t col = piece_at<N>(first, s.n);
  const uint32_t row = s.keys[p1 - 1];
  const bool began = s.keys[p0] != row || p0 == 0 || s.keys[p0 - 1] != row;
  if (row >= s.n_rows || !began || s.keys[p1] != row) return;
  const int64_t chunks = (s.n_tokens + s.chunk - 1) / s.chunk;
  // the chunk that the row ends in, kAhead looked at together
  constexpr int kAhead = 8;
  int64_t last = c;
  for (int same = kAhead; same == kAhead; last += same) {
    uint32_t key[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int64_t next = last + 1 + u;
      key[u] = s.keys[(next < chunks ? next : c) * s.chunk];
      if (next >= chunks) key[u] = s.n_rows;
    }
    same = 0;
#pragma unroll
    for (int u = 0; u < kAhead; ++u) same += same == u && key[u] == row;
  }
  float sum[N];
  __builtin_memcpy(sum, __builtin_assume_aligned(s.part(c, 1) + col, 4), sizeof(sum));
  for (int64_t next = c + 1; next <= last; next += kAhead) {
    float v[kAhead][N];
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
      __builtin_memcpy(v[u], __builtin_assume_aligned(
                                 s.part(next + u <= last ? next + u : last, 0) + col, 4),
                       sizeof(v[u]));
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
#pragma unroll
      for (int i = 0; i < N; ++i) sum[i] += next + u <= last ? v[u][i] : 0.f;
  }
  put_row(s, out, row, col, sum);
}

// ---- host ------------------------------------------------------------------------

// Tokens of a chunk: 8 to 32, as many as leave the chunks some 64 K threads (16384
// tokens in 16 columns of bf16: 25 us in chunks of 32, 15 in 16), and more where
// there would be above 2048 chunks, whose parts one thread may have to add up.
// Many tokens of a narrow table then have few threads, 2048 for each 16 bytes of
// its rows: the gradient of 131072 tokens in 64 columns of bf16 takes 60 us, of
// 2^21 tokens 324 (their bytes 55).
int32_t chunk_of(int64_t n_tokens, int64_t n) {
  int64_t c = 8;
  while (c < 32 && n_tokens * ceil_div(n, 8) > c * 65536) c *= 2;
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
  p.parts = c.take<float>(2 * n * ceil_div(n_tokens, chunk_of(n_tokens, n)));
  if (n_tokens > kSortTokens) {
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
    constexpr int N = kPiece<T>;
    const int across = row_threads(ceil_div(n, n < N ? 1 : N));
    auto run = [&](auto kernel) {
      const int64_t blocks = ceil_div(n_tokens, kThreads / across);
      if (blocks > kMaxBlocks) return too_many("tokens", n_tokens);
      hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(blocks)), dim3(kThreads), 0,
                         as_stream(stream), static_cast<const T *>(table),
                         static_cast<uint32_t>(n_rows), ld, n, static_cast<const Token *>(tokens),
                         n_tokens, scale, across, static_cast<T *>(out));
      EJ_LAUNCH_CHECK();
      return EJ_OK;
    };
    if (n < N) return run(embed_kernel<T, Token, 1>);
    return run(embed_kernel<T, Token, N>);
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
    Sums s = {p.keys, p.perm, m, chunk_of(n_tokens, n), rows, n, 0, grad_ld, scale, p.parts};
    constexpr int N = kPiece<T>;
    const int piece = n < N ? 1 : N;
    s.across = row_threads(ceil_div(n, piece));
    const int64_t chunks = ceil_div(n_tokens, s.chunk);
    const int64_t cols = ceil_div(n, static_cast<int64_t>(s.across) * piece);
    const int64_t sum_blocks = ceil_div(chunks, kThreads / s.across);
    if (sum_blocks * cols > kMaxBlocks || cols > 65535) return too_many("columns", n);
    int bits = 1;
    while (n_rows >> bits) ++bits;  // keys up to n_rows
    if (n_tokens <= kSortTokens) {
      hipLaunchKernelGGL((sort_few_kernel<T, Token>),
                         dim3(static_cast<unsigned>(1 + clear_blocks(bytes, kSortThreads))),
                         dim3(kSortThreads), 0, stream, tok, m, rows, bits, p.keys, p.perm, out,
                         count);
      EJ_LAUNCH_CHECK();
    } else {
      const int64_t blocks = ceil_div(n_tokens, kThreads);
      hipLaunchKernelGGL((sort_keys_kernel<T, Token>),
                         dim3(static_cast<unsigned>(blocks + clear_blocks(bytes, kThreads))),
                         dim3(kThreads), 0, stream, tok, m, rows, p.keys64, p.perm,
                         static_cast<uint32_t>(blocks), out, count);
      EJ_LAUNCH_CHECK();
      EJ_TRY(sort_pairs_u64(p.keys64, p.perm, p.keys_alt, p.perm_alt, n_tokens, bits, p.sort,
                            stream, false, nullptr, false));
      hipLaunchKernelGGL(narrow_keys_kernel, dim3(static_cast<unsigned>(blocks)), dim3(kThreads),
                         0, stream, p.keys64, m, p.keys);
      EJ_LAUNCH_CHECK();
    }
    if (n_tokens == 0) return EJ_OK;
    const dim3 grid(static_cast<unsigned>(sum_blocks), static_cast<unsigned>(cols));
    auto sums = [&](auto sum, auto join) {
      hipLaunchKernelGGL(sum, grid, dim3(kThreads), 0, stream, s, static_cast<const T *>(grad),
                         out);
      EJ_LAUNCH_CHECK();
      if (chunks == 1) return EJ_OK;
      hipLaunchKernelGGL(join, grid, dim3(kThreads), 0, stream, s, out);
      EJ_LAUNCH_CHECK();
      return EJ_OK;
    };
    if (n < N) return sums(sum_chunks_kernel<T, 1>, join_chunks_kernel<T, 1>);
    return sums(sum_chunks_kernel<T, N>, join_chunks_kernel<T, N>);
  });
}
