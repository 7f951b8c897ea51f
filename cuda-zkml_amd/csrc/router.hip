// The experts' router for gfx950: each token's experts by its scores, their
// softmax weights, the balance of the experts, and the gradients.
//
//   z[t,e] = scale s[t,e],  p[t,:] = softmax(z[t,:])
//   e_1, e_2, ... of a token: the experts of its largest scores, of equal scores
//   the lower expert first;  w_j = p[e_j], or p[e_j] / sum_i p[e_i]
//   count[e] = routes that name e, n = tokens with a score, prob[e] = sum_t p[t,e] / n
//   loss = experts sum_e f_e prob[e],  f_e = count[e] / (n slots)
//
// and, for gradients g_w of the weights and g of the loss (f is a constant to it),
//
//   dz[t,e] = p[t,e] (sum_{j: e_j = e} g_w[j] - sum_j g_w[j] p[t,e_j])        w = p
//   dz[t,e] = sum_{j: e_j = e} w_j (g_w[j] - sum_i g_w[i] w_i)               w normalized
//           + g experts / n p[t,e] (f_e - sum_i f_i p[t,i]),
//   ds = scale dz.
//
// L lanes have a token, V neighbouring scores each, in registers: the row is read
// once, and all that a token needs of it (maximum, sum, the next largest) is a
// reduction over L lanes.
#include <math.h>

#include <type_traits>

#include "rows.hpp"
#include "zk_internal.hpp"

namespace zk {

constexpr int ROUTE_THREADS = 256;

struct RouteArgs {
  const void* scores;
  size_t ld;
  uint32_t tokens, experts, slots;
  float scale;
  int renormalize;
  int32_t* expert;   // tokens x slots; given where the routes are
  float* weight;     // tokens x slots
  float* part_prob;  // of each block: sums of p by expert
  uint32_t* part_count;  // of each block: counts by expert, and tokens with a score
};

// What scores are compared as: floats, or integers; NONE is a masked expert's.
template <class T>
struct Score {
  typedef float W;
  static __device__ __forceinline__ float none() { return -INFINITY; }
  static __device__ __forceinline__ float read(T s) { return (float)s + 0.0f; }  // (-0 and 0 are equal)
  // NaN and infinity leave a row without a softmax
  static __device__ __forceinline__ bool bad(float v) { return !(v < INFINITY); }
  // exp(scale (v - m)); v <= m, m a score
  static __device__ __forceinline__ float ex(float v, float m, float scale) { return expf((v - m) * scale); }
};
template <>
struct Score<int> {
  typedef int W;
  static __device__ __forceinline__ int none() { return INT32_MIN; }
  static __device__ __forceinline__ int read(int s) { return s; }
  static __device__ __forceinline__ bool bad(int) { return false; }
  static __device__ __forceinline__ float ex(int v, int m, float scale) {
    return v == none() ? 0.0f : expf(-(float)((uint32_t)m - (uint32_t)v) * scale);
  }
};

template <int L, class X, class F>
__device__ __forceinline__ X over_lanes(X v, F&& f) {
#pragma unroll
  for (int d = L / 2; d; d >>= 1) v = f(v, __shfl_xor(v, d));
  return v;
}
template <int L, class X>
__device__ __forceinline__ X max_over(X v) {
  return over_lanes<L>(v, [](X a, X b) { return a > b ? a : b; });
}
template <int L, class X>
__device__ __forceinline__ X min_over(X v) {
  return over_lanes<L>(v, [](X a, X b) { return a < b ? a : b; });
}
template <int L>
__device__ __forceinline__ float sum_over(float v) {
  return over_lanes<L>(v, [](float a, float b) { return a + b; });
}

// A lane's V scores of a row; those beyond its end are masked.
template <class T, int V>
__device__ __forceinline__ void load_scores(const T* row, uint32_t first, uint32_t experts,
                                            typename Score<T>::W (&v)[V]) {
  T raw[V];
  if (first + V <= experts) {
    __builtin_memcpy(raw, row + first, sizeof(raw));
#pragma unroll
    for (int i = 0; i < V; i++) v[i] = Score<T>::read(raw[i]);
  } else {
#pragma unroll
    for (int i = 0; i < V; i++) v[i] = first + i < experts ? Score<T>::read(row[first + i]) : Score<T>::none();
  }
}

// CHOOSE: a token's experts and weights are found; else given.  BALANCE: counts
// and sums of p are made.
template <class T, int L, int V, bool CHOOSE, bool BALANCE>
__global__ __launch_bounds__(ROUTE_THREADS) void k_route(RouteArgs a) {
  typedef Score<T> S;
  typedef typename S::W W;
  constexpr uint32_t GROUPS = ROUTE_THREADS / L, WAVES = ROUTE_THREADS / 64;
  constexpr int KEPT = (ZK_MAX_SLOTS + L - 1) / L;
  __shared__ uint32_t count[BALANCE ? L * V + 1 : 1];
  __shared__ float sums[BALANCE ? WAVES * L * V : 1];
  const uint32_t tid = threadIdx.x, l = tid % L, first = l * V;
  if (BALANCE) {
    for (uint32_t e = tid; e <= a.experts; e += ROUTE_THREADS) count[e] = 0;
    __syncthreads();
  }
  float psum[V] = {};
  const bool all = BALANCE || !a.renormalize;  // whether every score's exponential is needed
  for (uint32_t t0 = blockIdx.x * GROUPS; t0 < a.tokens; t0 += gridDim.x * GROUPS) {
    const uint32_t t = t0 + tid / L;
    if (t >= a.tokens) continue;  // (all of the token's lanes)
    W v[V];
    load_scores<T, V>((const T*)a.scores + (size_t)t * a.ld, first, a.experts, v);
    W top = S::none();
    bool bad = false;
#pragma unroll
    for (int i = 0; i < V; i++) {
      top = v[i] > top ? v[i] : top;
      bad |= S::bad(v[i]);
    }
    const W m = max_over<L>(top);
    bad = max_over<L>((int)bad) != 0;
    const bool empty = !bad && m == S::none();
    float inv = 0.0f;
    if (all && !bad && !empty) {
      float p[V], z = 0.0f;
#pragma unroll
      for (int i = 0; i < V; i++) z += p[i] = S::ex(v[i], m, a.scale);
      inv = 1.0f / sum_over<L>(z);
      if (BALANCE) {
#pragma unroll
        for (int i = 0; i < V; i++) psum[i] += p[i] * inv;
      }
    }
    if (BALANCE) {
      if (bad) {
#pragma unroll
        for (int i = 0; i < V; i++) psum[i] = NAN;
      }
      if (l == 0 && !empty) atomicAdd(&count[a.experts], 1u);
    }
    if (!CHOOSE) {
      for (uint32_t j = l; j < a.slots; j += L) {
        const uint32_t e = (uint32_t)a.expert[(size_t)t * a.slots + j];
        if (e < a.experts) atomicAdd(&count[e], 1u);
      }
      continue;
    }
    int kept_e[KEPT];
    float kept_w[KEPT];
#pragma unroll
    for (int k = 0; k < KEPT; k++) kept_e[k] = -1, kept_w[k] = bad ? NAN : 0.0f;
    float total = 0.0f;
    for (uint32_t j = 0; j < a.slots && !bad; j++) {
      // a lane's first largest score, then the lowest expert that has the largest of all
      W b = S::none();
      uint32_t e = a.experts;
#pragma unroll
      for (int i = 0; i < V; i++)
        if (v[i] > b) b = v[i], e = first + i;
      const W best = max_over<L>(b);
      if (best == S::none()) break;
      e = min_over<L>(b == best ? e : a.experts);
#pragma unroll
      for (int i = 0; i < V; i++)
        if (first + i == e) v[i] = S::none();
      const float w = S::ex(best, m, a.scale);
      total += w;
#pragma unroll
      for (int k = 0; k < KEPT; k++)
        if (j == l + k * L) kept_e[k] = (int)e, kept_w[k] = w;
      if (BALANCE && l == 0) atomicAdd(&count[e], 1u);
    }
    const float by = a.renormalize ? (total > 0.0f ? 1.0f / total : 0.0f) : inv;
#pragma unroll
    for (int k = 0; k < KEPT; k++)
      if (l + k * L < a.slots) {
        const size_t at = (size_t)t * a.slots + l + k * L;
        a.expert[at] = kept_e[k];
        a.weight[at] = bad ? kept_w[k] : kept_w[k] * by;
      }
  }
  if (!BALANCE) return;
  // the wave's tokens, then the waves, in a fixed order
#pragma unroll
  for (int i = 0; i < V; i++) {
#pragma unroll
    for (int d = L; d < 64; d <<= 1) psum[i] += __shfl_xor(psum[i], d);
    if (tid % 64 < L) sums[(tid / 64) * L * V + first + i] = psum[i];
  }
  __syncthreads();
  for (uint32_t e = tid; e <= a.experts; e += ROUTE_THREADS) {
    a.part_count[(size_t)blockIdx.x * (a.experts + 1) + e] = count[e];
    if (e == a.experts) break;
    float s = sums[e];
#pragma unroll
    for (uint32_t w = 1; w < WAVES; w++) s += sums[w * L * V + e];
    a.part_prob[(size_t)blockIdx.x * a.experts + e] = s;
  }
}

// The blocks' counts and sums to count, prob and loss; sums in 64 bits, in the
// order of the blocks.
__global__ __launch_bounds__(1024) void k_balance_finish(const float* __restrict__ part_prob,
                                                         const uint32_t* __restrict__ part_count, uint32_t blocks,
                                                         uint32_t experts, uint32_t slots,
                                                         int32_t* __restrict__ count, float* __restrict__ prob,
                                                         float* __restrict__ loss) {
  __shared__ uint32_t tokens;
  __shared__ double part[16];
  const uint32_t e = threadIdx.x;
  uint32_t c = 0;
  double s = 0.0;
  if (e < experts)
    for (uint32_t b = 0; b < blocks; b++) {
      c += part_count[(size_t)b * (experts + 1) + e];
      s += part_prob[(size_t)b * experts + e];
    }
  if (e == 0) {
    uint32_t n = 0;
    for (uint32_t b = 0; b < blocks; b++) n += part_count[(size_t)b * (experts + 1) + experts];
    tokens = n;
    count[experts] = (int32_t)n;
  }
  __syncthreads();
  const uint32_t n = tokens;
  const double mean = n ? s / n : 0.0;
  if (e < experts) {
    count[e] = (int32_t)c;
    prob[e] = (float)mean;
  }
  double x = n && e < experts ? mean * c / ((double)n * slots) : 0.0;
#pragma unroll
  for (int d = 32; d; d >>= 1) x += __shfl_xor(x, d);
  if (e % 64 == 0) part[e / 64] = x;
  __syncthreads();
  if (e == 0) {
    for (int w = 1; w < 16; w++) x += part[w];
    *loss = (float)(x * experts);
  }
}

// ------------------------------------------------------------ gradient
struct RouteGradArgs {
  const void* scores;
  size_t ld, ld_grad;
  uint32_t tokens, experts, slots;
  float scale;
  int renormalize;
  const int32_t* expert;
  const float* grad_weight;  // or null
  const int32_t* count;      // or null
  const float* grad_loss;
  void* grad;
};

template <class T, int L, int V>
__global__ __launch_bounds__(ROUTE_THREADS) void k_route_grad(RouteGradArgs a) {
  typedef Score<T> S;
  constexpr uint32_t GROUPS = ROUTE_THREADS / L;
  const uint32_t tid = threadIdx.x, l = tid % L, first = l * V;
  // the loss's factors of this lane's experts: g experts / n, and f
  float f[V] = {}, c = 0.0f;
  if (a.count) {
    const int n = a.count[a.experts];
    if (n > 0) {
      c = *a.grad_loss * ((float)a.experts / (float)n);
      const float per = 1.0f / ((float)n * (float)a.slots);
#pragma unroll
      for (int i = 0; i < V; i++)
        if (first + i < a.experts) f[i] = (float)a.count[first + i] * per;
    }
  }
  for (uint32_t t0 = blockIdx.x * GROUPS; t0 < a.tokens; t0 += gridDim.x * GROUPS) {
    const uint32_t t = t0 + tid / L;
    if (t >= a.tokens) continue;  // (all of the token's lanes)
    float v[V], p[V], d[V];
    load_scores<T, V>((const T*)a.scores + (size_t)t * a.ld, first, a.experts, v);
    float top = S::none();
    bool bad = false;
#pragma unroll
    for (int i = 0; i < V; i++) {
      top = v[i] > top ? v[i] : top;
      bad |= S::bad(v[i]);
    }
    const float m = max_over<L>(top);
    bad = max_over<L>((int)bad) != 0;
    const bool empty = !bad && m == S::none();
#pragma unroll
    for (int i = 0; i < V; i++) d[i] = bad ? NAN : 0.0f;
    if (!bad && !empty) {
      float z = 0.0f, dot = 0.0f;
#pragma unroll
      for (int i = 0; i < V; i++) z += p[i] = S::ex(v[i], m, a.scale);
      const float inv = 1.0f / sum_over<L>(z);
#pragma unroll
      for (int i = 0; i < V; i++) {
        p[i] *= inv;
        dot += p[i] * f[i];
      }
      if (a.count) dot = sum_over<L>(dot);
#pragma unroll
      for (int i = 0; i < V; i++) d[i] = c * p[i] * (f[i] - dot);
      if (a.grad_weight) {
        float g[V] = {}, times[V] = {};
        for (uint32_t j = 0; j < a.slots; j++) {
          const uint32_t e = (uint32_t)a.expert[(size_t)t * a.slots + j];
          const float gj = a.grad_weight[(size_t)t * a.slots + j];
#pragma unroll
          for (int i = 0; i < V; i++)
            if (first + i < a.experts && first + i == e) g[i] += gj, times[i] += 1.0f;
        }
        if (a.renormalize) {
          // softmax over the chosen alone: their own maximum, sum and mean
          float mc = S::none(), zc = 0.0f, gc = 0.0f;
#pragma unroll
          for (int i = 0; i < V; i++)
            if (times[i] > 0.0f && v[i] > mc) mc = v[i];
          mc = max_over<L>(mc);
#pragma unroll
          for (int i = 0; i < V; i++) {
            p[i] = times[i] > 0.0f && v[i] > S::none() ? S::ex(v[i], mc, a.scale) : 0.0f;
            zc += times[i] * p[i];
            gc += g[i] * p[i];
          }
          zc = sum_over<L>(zc), gc = sum_over<L>(gc);
          const float ic = zc > 0.0f ? 1.0f / zc : 0.0f;
          gc *= ic;
#pragma unroll
          for (int i = 0; i < V; i++) d[i] += p[i] * ic * (g[i] - times[i] * gc);
        } else {
          float gp = 0.0f;
#pragma unroll
          for (int i = 0; i < V; i++) gp += g[i] * p[i];
          gp = sum_over<L>(gp);
#pragma unroll
          for (int i = 0; i < V; i++) d[i] += p[i] * (g[i] - gp);
        }
      }
    }
    T out[V];
#pragma unroll
    for (int i = 0; i < V; i++) out[i] = (T)(d[i] * a.scale);
    T* row = (T*)a.grad + (size_t)t * a.ld_grad + first;
    if (first + V <= a.experts) {
      __builtin_memcpy(row, out, sizeof(out));
    } else {
#pragma unroll
      for (int i = 0; i < V; i++)
        if (first + i < a.experts) row[i] = out[i];
    }
  }
}

// ------------------------------------------------------------ which lanes
// Calls fn with the lanes a token gets and the scores of a lane.
template <class Fn>
static int by_experts(uint32_t experts, Fn&& fn) {
  using std::integral_constant;
  const integral_constant<int, 16> quarter;
  const integral_constant<int, 64> whole;
  if (experts <= 16) return fn(quarter, integral_constant<int, 1>());
  if (experts <= 32) return fn(quarter, integral_constant<int, 2>());
  if (experts <= 64) return fn(quarter, integral_constant<int, 4>());
  if (experts <= 128) return fn(quarter, integral_constant<int, 8>());
  if (experts <= 256) return fn(whole, integral_constant<int, 4>());
  if (experts <= 512) return fn(whole, integral_constant<int, 8>());
  return fn(whole, integral_constant<int, 16>());
}

constexpr uint32_t ROUTE_BLOCKS = 1024;    // of a launch at the most (then a block has several tokens a group)
constexpr uint32_t BALANCE_BLOCKS = 128;   // whose sums one block adds up

static uint32_t route_blocks(size_t tokens, int lanes, uint32_t most) {
  const uint32_t b = cdiv(tokens, ROUTE_THREADS / lanes);
  return b < most ? b : most;
}
static uint32_t balance_blocks(size_t tokens, int experts) {
  return route_blocks(tokens, experts <= 128 ? 16 : 64, BALANCE_BLOCKS);
}

// ------------------------------------------------------------ arguments
static int check_route(zk_context* ctx, const void* scores, int type, size_t ld, size_t tokens, int experts, int slots,
                       float scale) {
  if (!float_type(type) && type != ZK_I32) return ctx->fail(ZK_ERR_INVALID, "experts' route: unknown type of scores");
  if (experts < 1 || experts > ZK_MAX_EXPERTS)
    return ctx->fail(ZK_ERR_SIZE, "experts' route: between 1 and 1024 experts");
  if (slots < 1 || slots > ZK_MAX_SLOTS) return ctx->fail(ZK_ERR_SIZE, "experts' route: between 1 and 32 slots");
  if (tokens > ZK_MAX_EXPERT_ROWS || tokens * (size_t)slots > ZK_MAX_EXPERT_ROWS)
    return ctx->fail(ZK_ERR_SIZE, "experts' route: more than 2^22 pairs");
  if (!(scale > 0.0f) || !(scale < INFINITY))
    return ctx->fail(ZK_ERR_INVALID, "experts' route: scale is positive and finite");
  if (ld < (size_t)experts) return ctx->fail(ZK_ERR_INVALID, "experts' route: a row stride below the row's length");
  if (tokens && !scores) return ctx->fail(ZK_ERR_INVALID, "experts' route: null pointer");
  if (!aligned(scores, type_bytes(type)))
    return ctx->fail(ZK_ERR_INVALID, "experts' route: a pointer is not aligned to its type");
  return ZK_OK;
}

// Arrays of 4-byte words that a call needs.
template <class... P>
static int check_route_words(zk_context* ctx, const P*... p) {
  if (((p == nullptr) || ...)) return ctx->fail(ZK_ERR_INVALID, "experts' route: null pointer");
  if ((!aligned(p, 4) || ...)) return ctx->fail(ZK_ERR_INVALID, "experts' route: a pointer is not aligned to its type");
  return ZK_OK;
}

template <class Fn>
static int by_score_type(int type, Fn&& fn) {
  if (type == ZK_I32) return fn(0);
  return by_type(type, fn);
}

template <bool CHOOSE>
static int route(zk_context* ctx, RouteArgs a, int type, int32_t* count, float* prob, float* loss, void* work,
                 size_t work_bytes, hipStream_t st) {
  const bool balance = count != nullptr;
  const uint32_t blocks = balance_blocks(a.tokens, (int)a.experts);
  if (balance) {
    const size_t need = zk_experts_route_work(a.tokens, (int)a.experts);
    if (need && (!work || !aligned(work, 4) || work_bytes < need))
      return ctx->fail(ZK_ERR_INVALID, "experts' route: workspace missing, too small or not aligned to 4 bytes");
    a.part_prob = (float*)work;
    a.part_count = (uint32_t*)work + (size_t)blocks * a.experts;
  }
  const char* name = CHOOSE ? "experts_route" : "experts_balance";
  if (a.tokens)
    ZK_TRY(by_score_type(type, [&](auto zero) -> int {
      typedef decltype(zero) T;
      return by_experts(a.experts, [&](auto lanes, auto per) -> int {
        constexpr int L = decltype(lanes)::value, V = decltype(per)::value;
        if (balance) {
          ZK_LAUNCH(ctx, st, name, (k_route<T, L, V, CHOOSE, true>), dim3(blocks), dim3(ROUTE_THREADS), 0, a);
        } else if constexpr (CHOOSE) {
          ZK_LAUNCH(ctx, st, name, (k_route<T, L, V, true, false>), dim3(route_blocks(a.tokens, L, ROUTE_BLOCKS)),
                    dim3(ROUTE_THREADS), 0, a);
        }
        return ZK_OK;
      });
    }));
  if (balance)
    ZK_LAUNCH(ctx, st, name, k_balance_finish, dim3(1), dim3(1024), 0, a.part_prob, a.part_count,
              a.tokens ? blocks : 0, a.experts, a.slots, count, prob, loss);
  return ZK_OK;
}

}  // namespace zk

extern "C" {

size_t zk_experts_route_work(size_t tokens, int experts) {
  using namespace zk;
  if (experts < 1 || experts > ZK_MAX_EXPERTS || tokens > ZK_MAX_EXPERT_ROWS) return 0;
  return (size_t)balance_blocks(tokens, experts) * (2 * experts + 1) * 4;
}

int zk_experts_route(zk_context* ctx, const void* d_scores, int type, size_t ld, size_t tokens, int experts, int slots,
                     float scale, int renormalize, int32_t* d_expert, float* d_weight, int32_t* d_count,
                     float* d_prob, float* d_loss, void* d_work, size_t work_bytes, void* stream) {
  using namespace zk;
  if (!ctx) return ZK_ERR_INVALID;
  return guard(ctx, [&]() -> int {
    ZK_TRY(check_route(ctx, d_scores, type, ld, tokens, experts, slots, scale));
    if (tokens) ZK_TRY(check_route_words(ctx, d_expert, d_weight));
    if (d_count || d_prob || d_loss) ZK_TRY(check_route_words(ctx, d_count, d_prob, d_loss));
    OnDevice on(ctx);
    const RouteArgs a = {d_scores, ld, (uint32_t)tokens, (uint32_t)experts, (uint32_t)slots, scale, renormalize != 0,
                         d_expert, d_weight, nullptr, nullptr};
    return route<true>(ctx, a, type, d_count, d_prob, d_loss, d_work, work_bytes, ctx->s(stream));
  });
}

int zk_experts_balance(zk_context* ctx, const void* d_scores, int type, size_t ld, size_t tokens, int experts,
                       int slots, float scale, const int32_t* d_expert, int32_t* d_count, float* d_prob,
                       float* d_loss, void* d_work, size_t work_bytes, void* stream) {
  using namespace zk;
  if (!ctx) return ZK_ERR_INVALID;
  return guard(ctx, [&]() -> int {
    ZK_TRY(check_route(ctx, d_scores, type, ld, tokens, experts, slots, scale));
    if (tokens) ZK_TRY(check_route_words(ctx, d_expert));
    ZK_TRY(check_route_words(ctx, d_count, d_prob, d_loss));
    OnDevice on(ctx);
    const RouteArgs a = {d_scores, ld, (uint32_t)tokens, (uint32_t)experts, (uint32_t)slots, scale, 0,
                         (int32_t*)d_expert, nullptr, nullptr, nullptr};
    return route<false>(ctx, a, type, d_count, d_prob, d_loss, d_work, work_bytes, ctx->s(stream));
  });
}

int zk_experts_route_grad(zk_context* ctx, const void* d_scores, int type, size_t ld, size_t tokens, int experts,
                          int slots, float scale, int renormalize, const int32_t* d_expert,
                          const float* d_grad_weight, const int32_t* d_count, const float* d_grad_loss,
                          void* d_grad_scores, size_t ld_grad, void* stream) {
  using namespace zk;
  if (!ctx) return ZK_ERR_INVALID;
  return guard(ctx, [&]() -> int {
    ZK_TRY(check_route(ctx, d_scores, type, ld, tokens, experts, slots, scale));
    if (type == ZK_I32) return ctx->fail(ZK_ERR_INVALID, "experts' route: integer scores have no gradient");
    if (ld_grad < (size_t)experts)
      return ctx->fail(ZK_ERR_INVALID, "experts' route: a row stride below the row's length");
    if (!d_grad_weight && !d_count)
      return ctx->fail(ZK_ERR_INVALID, "experts' route: neither the weights' gradient nor counts");
    if (d_grad_weight && tokens) ZK_TRY(check_route_words(ctx, d_expert, d_grad_weight));
    if (d_count) ZK_TRY(check_route_words(ctx, d_count, d_grad_loss));
    if (!tokens) return ZK_OK;
    if (!d_grad_scores) return ctx->fail(ZK_ERR_INVALID, "experts' route: null pointer");
    if (!aligned(d_grad_scores, type_bytes(type)))
      return ctx->fail(ZK_ERR_INVALID, "experts' route: a pointer is not aligned to its type");
    OnDevice on(ctx);
    const RouteGradArgs a = {d_scores, ld, ld_grad, (uint32_t)tokens, (uint32_t)experts, (uint32_t)slots, scale,
                             renormalize != 0, d_expert, d_grad_weight, d_count, d_grad_loss, d_grad_scores};
    hipStream_t st = ctx->s(stream);
    return by_type(type, [&](auto zero) -> int {
      typedef decltype(zero) T;
      return by_experts(a.experts, [&](auto lanes, auto per) -> int {
        constexpr int L = decltype(lanes)::value, V = decltype(per)::value;
        ZK_LAUNCH(ctx, st, "experts_route_grad", (k_route_grad<T, L, V>), dim3(route_blocks(tokens, L, ROUTE_BLOCKS)),
                  dim3(ROUTE_THREADS), 0, a);
        return ZK_OK;
      });
    });
  });
}

}  // extern "C"
