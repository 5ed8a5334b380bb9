// Routing of tokens to experts: softmax, top-k and the relation of (token,
// expert) pairs grouped by expert.
//
// For the logits l of a token: m = max l, p = exp(l - m) / sum exp(l - m); the
// k largest logits are its picks (equal ones in the order of their experts),
// with weights p, or p divided by the sum over the picks.  A logit of -inf
// excludes its expert; picks beyond the experts left are -1 with weight 0.
//
// A token's logits stay in registers: 16 or 64 lanes hold V each, two reductions
// (the largest ordered value, the lowest expert that has it) for each pick, no
// sort.  The grouping is a
// stable counting sort (pairs of one expert in token order, so results do not
// depend on scheduling): workgroups count their tokens' picks in LDS, then
// each adds up the counts before its own and places its pairs, ranked among
// the lanes of a wave by ballots on the expert's bits.  Two launches; a batch
// that one workgroup takes is routed and grouped in one.
#include "ej_internal.h"

#include <type_traits>

namespace ej {
namespace {

constexpr int kMaxExperts = 1024;
constexpr int kRouteThreads = 1024;  // a workgroup a CU: one pass of 64 tokens
constexpr int kVjpThreads = 256;
constexpr int kGroupThreads = 512;
constexpr int kGroupWaves = kGroupThreads / 64;
constexpr int kRouteBlocks = 256;   // bound on the workgroups whose counts are added up
// The gradient gives a token a wave at most, and HIP launches hold fewer than
// 2^32 threads.
constexpr int64_t kMaxTokens = (int64_t{1} << 26) - 4;

// Whether one workgroup routes and groups (`routes`), or only groups, a batch.
// Routing takes it a pass for every 32 tokens (8 of more than 256 experts).
// Measured (us) so and in two launches over all CUs, tokens x experts, picks:
//   32 x 128, 8   6.4  8.8      64 x 64, 4   6.0   7.8    128 x 32, 4   7.3  8.0
//   64 x 128, 8   9.6  8.8      96 x 64, 4   7.4   7.9    256 x 32, 4  12.2  7.9
//   256 x 128, 8 29.8 10.0     128 x 64, 4   9.0   7.9    128 x 16, 8   8.5  7.7
//   32 x 256, 8   8.9 10.9     8 x 1024, 16 14.9  17.7    128 x 8, 2    5.6  8.0
//   48 x 256, 8  13.1 10.8    32 x 1024, 16 44.2  24.1    256 x 8, 2    8.4  7.9
// and grouping alone 256 x 128, 8 6.1 and 7.7, 256 x 1024, 2 4.8 and 9.5, 256 x
// 1024, 16 11.9 and 9.7.
bool one_workgroup(int64_t n_tokens, int32_t n_experts, bool routes) {
  if (!routes) return n_tokens <= 256;
  return n_tokens <= kGroupThreads / (n_experts <= 256 ? 16 : 64) ||
         (n_tokens <= 128 && n_tokens * n_experts <= 4096);
}

struct RouteArgs {
  const void *logits;
  int64_t ld;
  int32_t dtype, n_experts, k, renormalize;
  int64_t n_tokens;
  float *weights;
  int32_t *experts, *offsets, *rows, *slots;
  int32_t *counts;         // [blocks][n_experts]
  int32_t tokens_per_block;
};

__device__ inline float load_logit(const RouteArgs &a, int64_t t, int e) {
  const int64_t i = t * a.ld + e;
  if (a.dtype == EJ_F32) return static_cast<const float *>(a.logits)[i];
  const uint16_t h = static_cast<const uint16_t *>(a.logits)[i];
  if (a.dtype == EJ_BF16) return __uint_as_float(static_cast<uint32_t>(h) << 16);
  return static_cast<float>(__builtin_bit_cast(_Float16, h));
}

// Unsigned words in the order of the floats: NaN above +inf, -0 equal to 0,
// never 0 itself (which marks a logit as taken).
__device__ inline uint32_t ordered(float x) {
  if (x != x) return 0xffffffffu;
  const uint32_t u = __float_as_uint(x + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ inline float unordered(uint32_t o) {
  return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o);
}
constexpr uint32_t kExcluded = 0x007fffffu;  // ordered(-inf)

// Reductions over the L lanes of a token, every lane gets the same result:
// within 16 lanes by DPP (neighbours, pairs, then mirrored halves, whose lanes
// agree already), across the rows of 16 by shuffles.
template <int CTRL>
__device__ inline uint32_t moved(uint32_t v) {
  return static_cast<uint32_t>(
      __builtin_amdgcn_update_dpp(0, static_cast<int>(v), CTRL, 0xf, 0xf, false));
}
template <int L, class F>
__device__ inline uint32_t lanes_reduce(uint32_t v, F f) {
  static_assert(L == 16 || L == 64, "whole DPP rows");
  v = f(v, moved<0xb1>(v));   // quad_perm [1, 0, 3, 2]
  v = f(v, moved<0x4e>(v));   // quad_perm [2, 3, 0, 1]
  v = f(v, moved<0x141>(v));  // row_half_mirror
  v = f(v, moved<0x140>(v));  // row_mirror
  if constexpr (L == 64) {
    v = f(v, static_cast<uint32_t>(__shfl_xor(static_cast<int>(v), 16)));
    v = f(v, static_cast<uint32_t>(__shfl_xor(static_cast<int>(v), 32)));
  }
  return v;
}
template <int L>
__device__ inline uint32_t lanes_max(uint32_t v) {
  return lanes_reduce<L>(v, [](uint32_t a, uint32_t b) { return a > b ? a : b; });
}
template <int L>
__device__ inline uint32_t lanes_min(uint32_t v) {
  return lanes_reduce<L>(v, [](uint32_t a, uint32_t b) { return a < b ? a : b; });
}
template <int L>
__device__ inline float lanes_sum(float v) {
  return __uint_as_float(lanes_reduce<L>(__float_as_uint(v), [](uint32_t a, uint32_t b) {
    return __float_as_uint(__uint_as_float(a) + __uint_as_float(b));
  }));
}

// Picks of token t by L lanes holding V logits each (expert v * L + lane);
// lane j of the L returns pick j and its weight.
template <int L, int V>
__device__ inline void route_token(const RouteArgs &a, int64_t t, int lane, int *pick_out,
                                   float *weight_out) {
  uint32_t key[V];
  float x[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int e = v * L + lane;
    x[v] = e < a.n_experts ? load_logit(a, t, e) : -INFINITY;
    key[v] = e < a.n_experts ? ordered(x[v]) : 0;
  }
  int pick = -1;
  uint32_t pick_key = kExcluded;
  float top = 0.f;
  for (int j = 0; j < a.k; ++j) {
    uint32_t best = 0;
    int at = 0;
#pragma unroll
    for (int v = 0; v < V; ++v)
      if (key[v] > best) {
        best = key[v];
        at = v * L + lane;
      }
    // of equal values the lowest expert wins
    const uint32_t wk = lanes_max<L>(best);
    const int we = static_cast<int>(lanes_min<L>(best == wk ? at : 0x7fffffffu));
    if (wk <= kExcluded) break;  // uniform over the L lanes
    if (j == 0) top = wk == 0xffffffffu ? __uint_as_float(0x7fc00000u) : unordered(wk);
    if (lane == j) {
      pick = we;
      pick_key = wk;
    }
#pragma unroll
    for (int v = 0; v < V; ++v)
      if (v * L + lane == we) key[v] = 0;
  }
  float w = 0.f;
  if (pick >= 0)
    w = pick_key == 0xffffffffu ? __uint_as_float(0x7fc00000u) : expf(unordered(pick_key) - top);
  float sum;
  if (a.renormalize) {
    sum = lanes_sum<L>(w);
  } else {
    sum = 0.f;
#pragma unroll
    for (int v = 0; v < V; ++v)
      if (v * L + lane < a.n_experts) sum += expf(x[v] - top);
    sum = lanes_sum<L>(sum);
  }
  *pick_out = pick;
  *weight_out = pick >= 0 ? w / sum : 0.f;
}

// Routes tokens [t0, t1) with the whole workgroup and hands every pair to
// pair(t, j, expert).
template <int L, int V, int NT, class Pair>
__device__ inline void route_tokens(const RouteArgs &a, int64_t t0, int64_t t1, Pair pair) {
  const int sub = threadIdx.x / L, lane = threadIdx.x % L;
  for (int64_t t = t0 + sub; t < t1; t += NT / L) {
    int e;
    float w;
    route_token<L, V>(a, t, lane, &e, &w);
    if (lane < a.k) {
      a.weights[t * a.k + lane] = w;
      a.experts[t * a.k + lane] = e;
      pair(t, lane, e);
    }
  }
}

// ---- grouping ---------------------------------------------------------------
// Places the pairs [p0, p1) (expert_of(p), -1 for none): wave w of the
// workgroup takes the w-th part of them.  base[e] (LDS) = slot of the first
// pair of expert e in this workgroup; cur[kGroupWaves][n_experts] is scratch.
template <class ExpertOf>
__device__ inline void place_pairs(const RouteArgs &a, int64_t p0, int64_t p1, const int *base,
                                   int *cur, ExpertOf expert_of) {
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t part = (p1 - p0 + kGroupThreads - 1) / kGroupThreads * 64;
  const int64_t q0 = p0 + wave * part < p1 ? p0 + wave * part : p1;
  const int64_t q1 = q0 + part < p1 ? q0 + part : p1;
  int *mine = cur + wave * a.n_experts;
  for (int i = threadIdx.x; i < kGroupWaves * a.n_experts; i += kGroupThreads) cur[i] = 0;
  __syncthreads();
  for (int64_t p = q0 + lane; p < q1; p += 64) {
    const int e = expert_of(p);
    if (e >= 0 && e < a.n_experts) atomicAdd(&mine[e], 1);
  }
  __syncthreads();
  for (int e = threadIdx.x; e < a.n_experts; e += kGroupThreads) {
    int run = base[e];
#pragma unroll
    for (int w = 0; w < kGroupWaves; ++w) {
      const int c = cur[w * a.n_experts + e];
      cur[w * a.n_experts + e] = run;
      run += c;
    }
  }
  __syncthreads();
  for (int64_t q = q0; q < q1; q += 64) {
    const int64_t p = q + lane;
    int e = p < q1 ? expert_of(p) : -1;
    if (e >= a.n_experts) e = -1;
    // the lanes with this lane's expert
    uint64_t same = __ballot(e >= 0);
    for (int b = 1; b < a.n_experts; b <<= 1) {
      const uint64_t set = __ballot(e >= 0 && (e & b));
      same &= e & b ? set : ~set;
    }
    int slot = -1;
    if (e >= 0) slot = mine[e] + __popcll(same & ((1ull << lane) - 1));
    // every lane has read its cursor before the last lane of an expert moves it
    asm volatile("" ::: "memory");
    if (e >= 0 && (same >> lane) == 1ull) mine[e] = slot + 1;
    asm volatile("" ::: "memory");
    if (p < q1) {
      a.slots[p] = slot;
      if (slot >= 0) a.rows[slot] = static_cast<int32_t>(p / a.k);
    }
  }
}

// Exclusive prefix of total[0 .. n) (LDS) in place, by the whole workgroup;
// returns the sum.
__device__ inline int scan_experts(int *total, int n) {
  int64_t run = 0;
  for (int e0 = 0; e0 < n; e0 += kGroupThreads) {
    const int e = e0 + threadIdx.x;
    const int c = e < n ? total[e] : 0;
    int64_t sum;
    const int64_t pre = block_exclusive_sum<kGroupThreads>(c, &sum);
    if (e < n) total[e] = static_cast<int>(run + pre);
    run += sum;
  }
  __syncthreads();
  return static_cast<int>(run);
}

// Bound by the vector instructions of the k reductions of a token.  A
// workgroup of 1024 a CU takes 64 tokens in one pass: 16384 x 128 fp32 logits,
// 8 picks 9.3 us (8.4 MB read: 0.9 TB/s); workgroups of 256 in four passes 17.6.
template <int L, int V>
__global__ __launch_bounds__(kRouteThreads) void route_kernel(RouteArgs a) {
  __shared__ int hist[kMaxExperts];
  for (int e = threadIdx.x; e < a.n_experts; e += kRouteThreads) hist[e] = 0;
  __syncthreads();
  const int64_t t0 = static_cast<int64_t>(blockIdx.x) * a.tokens_per_block;
  const int64_t t1 = t0 + a.tokens_per_block < a.n_tokens ? t0 + a.tokens_per_block : a.n_tokens;
  route_tokens<L, V, kRouteThreads>(a, t0, t1, [&](int64_t, int, int e) {
    if (e >= 0) atomicAdd(&hist[e], 1);
  });
  __syncthreads();
  for (int e = threadIdx.x; e < a.n_experts; e += kRouteThreads)
    a.counts[static_cast<int64_t>(blockIdx.x) * a.n_experts + e] = hist[e];
}

// The counts alone, of picks that are given.
__global__ __launch_bounds__(kRouteThreads) void count_kernel(RouteArgs a) {
  __shared__ int hist[kMaxExperts];
  for (int e = threadIdx.x; e < a.n_experts; e += kRouteThreads) hist[e] = 0;
  __syncthreads();
  const int64_t per = static_cast<int64_t>(a.tokens_per_block) * a.k;
  const int64_t p0 = blockIdx.x * per;
  const int64_t p1 = p0 + per < a.n_tokens * a.k ? p0 + per : a.n_tokens * a.k;
  for (int64_t p = p0 + threadIdx.x; p < p1; p += kRouteThreads) {
    const int e = a.experts[p];
    if (e >= 0 && e < a.n_experts) atomicAdd(&hist[e], 1);
  }
  __syncthreads();
  for (int e = threadIdx.x; e < a.n_experts; e += kRouteThreads)
    a.counts[static_cast<int64_t>(blockIdx.x) * a.n_experts + e] = hist[e];
}

// Rows of slots that hold no pair.
__device__ inline void clear_rows(const RouteArgs &a, int64_t live, int64_t first, int64_t step) {
  for (int64_t s = live + first; s < a.n_tokens * a.k; s += step) a.rows[s] = 0;
}

// Offsets, slots and rows.  Every workgroup adds up all counts itself, so that
// there is no launch for their prefix and no order between workgroups: bound by
// latency (256 counts of each expert, then two passes over its own pairs).
// 131072 pairs of 128 experts in 256 workgroups 8.8 us.
__global__ __launch_bounds__(kGroupThreads) void group_kernel(RouteArgs a) {
  extern __shared__ int lds[];
  int *total = lds, *before = lds + a.n_experts, *cur = lds + 2 * a.n_experts;
  // the threads split the blocks' counts: thread i takes expert i % n of every
  // parts-th block
  for (int e = threadIdx.x; e < 2 * a.n_experts; e += kGroupThreads) lds[e] = 0;
  __syncthreads();
  const int ne = a.n_experts, nb = gridDim.x, me = blockIdx.x;
  const int width = ne < kGroupThreads ? ne : kGroupThreads, parts = kGroupThreads / width;
  const int part = threadIdx.x / width;
  if (part < parts) {
    for (int e = threadIdx.x % width; e < ne; e += width) {
      int all = 0, pre = 0;
#pragma unroll 8
      for (int b = part; b < nb; b += parts) {
        const int c = a.counts[static_cast<int64_t>(b) * ne + e];
        all += c;
        pre += b < me ? c : 0;
      }
      atomicAdd(&total[e], all);
      atomicAdd(&before[e], pre);
    }
  }
  __syncthreads();
  const int live = scan_experts(total, ne);
  for (int e = threadIdx.x; e < ne; e += kGroupThreads) {
    if (me == 0) a.offsets[e] = total[e];
    before[e] += total[e];
  }
  if (me == 0 && threadIdx.x == 0) a.offsets[ne] = live;
  __syncthreads();
  const int64_t per = static_cast<int64_t>(a.tokens_per_block) * a.k, n = a.n_tokens * a.k;
  const int64_t p0 = me * per < n ? me * per : n, p1 = p0 + per < n ? p0 + per : n;
  place_pairs(a, p0, p1, before, cur, [&](int64_t p) { return a.experts[p]; });
  clear_rows(a, live, me * kGroupThreads + threadIdx.x,
             static_cast<int64_t>(nb) * kGroupThreads);
}

// Everything by one workgroup.  L == 0: the picks are given.  One token of 64
// experts, 4 picks: 4.2 us, most of it the launch.
template <int L, int V>
__global__ __launch_bounds__(kGroupThreads) void route_small_kernel(RouteArgs a) {
  extern __shared__ int lds[];
  int *total = lds, *cur = lds + a.n_experts, *picks = cur + kGroupWaves * a.n_experts;
  const int n = static_cast<int>(a.n_tokens) * a.k;
  for (int e = threadIdx.x; e < a.n_experts; e += kGroupThreads) total[e] = 0;
  __syncthreads();
  if constexpr (L > 0) {
    route_tokens<L, V, kGroupThreads>(a, 0, a.n_tokens, [&](int64_t t, int j, int e) {
      picks[t * a.k + j] = e;
      if (e >= 0) atomicAdd(&total[e], 1);
    });
  } else {
    for (int p = threadIdx.x; p < n; p += kGroupThreads) {
      const int e = a.experts[p];
      picks[p] = e;
      if (e >= 0 && e < a.n_experts) atomicAdd(&total[e], 1);
    }
  }
  __syncthreads();
  const int live = scan_experts(total, a.n_experts);
  for (int e = threadIdx.x; e < a.n_experts; e += kGroupThreads) a.offsets[e] = total[e];
  if (threadIdx.x == 0) a.offsets[a.n_experts] = live;
  place_pairs(a, 0, n, total, cur, [&](int64_t p) { return picks[p]; });
  clear_rows(a, live, threadIdx.x, kGroupThreads);
}

// ---- gradient -----------------------------------------------------------------
// With d = the weights' gradient and dot = sum_j w_j d_j over the picks:
//   renormalized: dl_e = w_e (d_e - dot) at the picks, 0 elsewhere;
//   otherwise:    dl_e = p_e ([e picked] d_e - dot).
// Bound by memory: 16384 x 128 fp32 8.2 us (17.8 MB: 2.2 TB/s, much of it the
// start and end of a launch this short).
template <int L, int V>
__global__ __launch_bounds__(kVjpThreads) void route_vjp_kernel(RouteArgs a, const float *grad,
                                                                  void *grad_logits) {
  const int lane = threadIdx.x % L;
  const int64_t t =
      static_cast<int64_t>(blockIdx.x) * (kVjpThreads / L) + threadIdx.x / L;
  if (t >= a.n_tokens) return;
  float x[V];
  float top = -INFINITY;
  bool nan = false;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int e = v * L + lane;
    x[v] = e < a.n_experts ? load_logit(a, t, e) : -INFINITY;
    nan |= x[v] != x[v];
    top = fmaxf(top, x[v]);
  }
  top = __uint_as_float(lanes_reduce<L>(__float_as_uint(top), [](uint32_t a, uint32_t b) {
    return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b)));
  }));
  if (lanes_max<L>(nan)) top = __uint_as_float(0x7fc00000u);
  int pick = -1;
  float d = 0.f, w = 0.f;
  if (lane < a.k) {
    pick = a.experts[t * a.k + lane];
    if (pick >= a.n_experts) pick = -1;
    if (pick >= 0) {
      d = grad[t * a.k + lane];
      w = expf(load_logit(a, t, pick) - top);
    }
  }
  const bool any = lanes_sum<L>(pick >= 0 ? 1.f : 0.f) > 0.f;
  float sum;
  if (a.renormalize) {
    sum = lanes_sum<L>(w);
  } else {
    sum = 0.f;
#pragma unroll
    for (int v = 0; v < V; ++v)
      if (v * L + lane < a.n_experts) sum += expf(x[v] - top);
    sum = lanes_sum<L>(sum);
  }
  w = pick >= 0 ? w / sum : 0.f;
  const float dot = lanes_sum<L>(w * d);
  float g[V];
#pragma unroll
  for (int v = 0; v < V; ++v)
    g[v] = a.renormalize || !any || v * L + lane >= a.n_experts
               ? 0.f
               : -(expf(x[v] - top) / sum) * dot;
  const float at_pick = w * (d - dot);
  for (int j = 0; j < a.k; ++j) {
    const int e = __shfl(pick, j, L);
    const float ge = __shfl(at_pick, j, L);
#pragma unroll
    for (int v = 0; v < V; ++v)
      if (e == v * L + lane) g[v] = ge;
  }
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int e = v * L + lane;
    if (e >= a.n_experts) continue;
    const int64_t i = t * a.n_experts + e;
    if (a.dtype == EJ_F32) static_cast<float *>(grad_logits)[i] = g[v];
    else if (a.dtype == EJ_BF16) static_cast<__bf16 *>(grad_logits)[i] = static_cast<__bf16>(g[v]);
    else static_cast<_Float16 *>(grad_logits)[i] = static_cast<_Float16>(g[v]);
  }
}

// Sixteen lanes a token up to 256 experts, a wave beyond.
template <class F>
int by_experts(int n, F f) {
  if (n <= 16) return f(std::integral_constant<int, 16>(), std::integral_constant<int, 1>());
  if (n <= 32) return f(std::integral_constant<int, 16>(), std::integral_constant<int, 2>());
  if (n <= 64) return f(std::integral_constant<int, 16>(), std::integral_constant<int, 4>());
  if (n <= 128) return f(std::integral_constant<int, 16>(), std::integral_constant<int, 8>());
  if (n <= 256) return f(std::integral_constant<int, 16>(), std::integral_constant<int, 16>());
  return f(std::integral_constant<int, 64>(), std::integral_constant<int, 16>());
}

int check_route(int64_t n_tokens, int32_t n_experts, int32_t k) {
  EJ_CHECK_ARG(n_tokens >= 0, "n_tokens = %lld is negative", (long long)n_tokens);
  EJ_CHECK_ARG(n_experts >= 1, "n_experts = %d, expected at least 1", n_experts);
  EJ_CHECK_ARG(k >= 1 && k <= n_experts, "k = %d, expected 1 to n_experts = %d", k, n_experts);
  if (n_experts > kMaxExperts || k > EJ_MAX_PICKS) {
    set_error("%d experts and %d picks: at most %d and %d are supported", n_experts, k,
              kMaxExperts, EJ_MAX_PICKS);
    return EJ_E_UNSUPPORTED;
  }
  if (n_tokens > kMaxTokens || n_tokens * k >= (int64_t{1} << 31)) {
    set_error("%lld tokens of %d picks: at most %lld tokens and fewer than 2^31 pairs are supported",
              (long long)n_tokens, k, (long long)kMaxTokens);
    return EJ_E_UNSUPPORTED;
  }
  return EJ_OK;
}

int check_logits(const void *logits, int32_t dtype, int64_t ld, int32_t n_experts) {
  EJ_CHECK_ARG(dtype == EJ_F32 || dtype == EJ_BF16 || dtype == EJ_F16,
               "logits of dtype %d: expected EJ_F32, EJ_BF16 or EJ_F16", dtype);
  EJ_CHECK_ARG(logits, "null logits");
  EJ_CHECK_ARG(ld >= n_experts, "logits row stride %lld below n_experts = %d", (long long)ld,
               n_experts);
  return EJ_OK;
}

// Routes (logits given) or only groups.
int run_route(RouteArgs a, void *workspace, size_t workspace_bytes, hipStream_t stream) {
  const size_t group_lds = (2 + kGroupWaves) * a.n_experts * sizeof(int);
  if (one_workgroup(a.n_tokens, a.n_experts, a.logits != nullptr)) {
    const size_t lds =
        ((1 + kGroupWaves) * a.n_experts + a.n_tokens * a.k) * sizeof(int);
    auto run = [&](auto L, auto V) {
      hipLaunchKernelGGL((route_small_kernel<decltype(L)::value, decltype(V)::value>), dim3(1),
                         dim3(kGroupThreads), lds, stream, a);
      EJ_LAUNCH_CHECK();
      return EJ_OK;
    };
    if (!a.logits) return run(std::integral_constant<int, 0>(), std::integral_constant<int, 1>());
    return by_experts(a.n_experts, run);
  }
  size_t need;
  EJ_TRY(ej_expert_route_workspace_size(a.n_tokens, a.n_experts, &need));
  EJ_CHECK_ARG(workspace && workspace_bytes >= need, "workspace of %zu bytes, expected %zu",
               workspace_bytes, need);
  a.counts = static_cast<int32_t *>(workspace);
  // as many tokens a workgroup as keep the workgroups at one a CU, in sixteens
  a.tokens_per_block =
      static_cast<int32_t>(ceil_div(ceil_div(a.n_tokens, kRouteBlocks), 16) * 16);
  const unsigned blocks = static_cast<unsigned>(ceil_div(a.n_tokens, a.tokens_per_block));
  if (a.logits) {
    EJ_TRY(by_experts(a.n_experts, [&](auto L, auto V) {
      hipLaunchKernelGGL((route_kernel<decltype(L)::value, decltype(V)::value>), dim3(blocks),
                         dim3(kRouteThreads), 0, stream, a);
      EJ_LAUNCH_CHECK();
      return EJ_OK;
    }));
  } else {
    hipLaunchKernelGGL(count_kernel, dim3(blocks), dim3(kRouteThreads), 0, stream, a);
    EJ_LAUNCH_CHECK();
  }
  hipLaunchKernelGGL(group_kernel, dim3(blocks), dim3(kGroupThreads), group_lds, stream, a);
  EJ_LAUNCH_CHECK();
  return EJ_OK;
}

__global__ __launch_bounds__(256) void zero_offsets_kernel(int32_t *offsets, int n) {
  for (int i = threadIdx.x; i < n; i += 256) offsets[i] = 0;
}

}  // namespace
}  // namespace ej

using namespace ej;

extern "C" int ej_expert_route_workspace_size(int64_t n_tokens, int32_t n_experts, size_t *bytes) {
  EJ_CHECK_ARG(bytes, "null bytes");
  EJ_TRY(check_route(n_tokens, n_experts, 1));
  // what routing needs, grouping alone needs at most
  *bytes = one_workgroup(n_tokens, n_experts, true) ? 0
                                                    : sizeof(int32_t) * kRouteBlocks * n_experts;
  return EJ_OK;
}

extern "C" int ej_expert_route(const void *logits, int32_t dtype, int64_t n_tokens,
                               int32_t n_experts, int64_t ld, int32_t k, int32_t renormalize,
                               float *weights, int32_t *experts, int32_t *offsets, int32_t *rows,
                               int32_t *slots, void *workspace, size_t workspace_bytes,
                               ej_stream_t stream) {
  EJ_TRY(check_route(n_tokens, n_experts, k));
  EJ_CHECK_ARG(offsets, "null offsets");
  RouteArgs a{logits, ld,     dtype,   n_experts, k,     renormalize, n_tokens,
              weights, experts, offsets, rows,      slots, nullptr,     0};
  if (n_tokens == 0) {
    hipLaunchKernelGGL(zero_offsets_kernel, dim3(1), dim3(256), 0, as_stream(stream), offsets,
                       n_experts + 1);
    EJ_LAUNCH_CHECK();
    return EJ_OK;
  }
  EJ_TRY(check_logits(logits, dtype, ld, n_experts));
  EJ_CHECK_ARG(weights && experts && rows && slots, "null output");
  return run_route(a, workspace, workspace_bytes, as_stream(stream));
}

extern "C" int ej_expert_group(const int32_t *experts, int64_t n_tokens, int32_t k,
                               int32_t n_experts, int32_t *offsets, int32_t *rows, int32_t *slots,
                               void *workspace, size_t workspace_bytes, ej_stream_t stream) {
  EJ_TRY(check_route(n_tokens, n_experts, k));
  EJ_CHECK_ARG(offsets, "null offsets");
  RouteArgs a{nullptr, 0,  EJ_F32, n_experts, k, 0, n_tokens, nullptr, const_cast<int32_t *>(experts),
              offsets, rows, slots, nullptr, 0};
  if (n_tokens == 0) {
    hipLaunchKernelGGL(zero_offsets_kernel, dim3(1), dim3(256), 0, as_stream(stream), offsets,
                       n_experts + 1);
    EJ_LAUNCH_CHECK();
    return EJ_OK;
  }
  EJ_CHECK_ARG(experts, "null experts");
  EJ_CHECK_ARG(rows && slots, "null output");
  return run_route(a, workspace, workspace_bytes, as_stream(stream));
}

extern "C" int ej_expert_route_vjp(const void *logits, int32_t dtype, int64_t n_tokens,
                                   int32_t n_experts, int64_t ld, int32_t k, int32_t renormalize,
                                   const int32_t *experts, const float *grad_weights,
                                   void *grad_logits, ej_stream_t stream) {
  EJ_TRY(check_route(n_tokens, n_experts, k));
  if (n_tokens == 0) return EJ_OK;
  EJ_TRY(check_logits(logits, dtype, ld, n_experts));
  EJ_CHECK_ARG(experts && grad_weights && grad_logits, "null argument");
  RouteArgs a{logits, ld, dtype, n_experts, k, renormalize, n_tokens, nullptr,
              const_cast<int32_t *>(experts), nullptr, nullptr, nullptr, nullptr, 0};
  return by_experts(n_experts, [&](auto L, auto V) {
    constexpr int l = decltype(L)::value;
    hipLaunchKernelGGL((route_vjp_kernel<l, decltype(V)::value>),
                       dim3(static_cast<unsigned>(ceil_div(n_tokens, kVjpThreads / l))),
                       dim3(kVjpThreads), 0, as_stream(stream), a, grad_weights, grad_logits);
    EJ_LAUNCH_CHECK();
    return EJ_OK;
  });
}
