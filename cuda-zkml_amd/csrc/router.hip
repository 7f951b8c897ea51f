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
// Threads of a block that also makes counts and sums: many waves, so that few
// blocks' sums are left to be added up.
constexpr int balance_threads(int lanes) { return lanes == 16 ? 1024 : 512; }

constexpr uint32_t ROUTE_BLOCKS = 2048;   // of a launch at the most (then a block has several tokens a group)
constexpr uint32_t BALANCE_BLOCKS = 256;  // one a CU
// Tokens times (experts + 64) that one block takes alone, by the time of a call from Python, to
// which a second launch is about 2.8 us: f32, 2 slots, one block and several, 256 tokens' choice of 60 experts 10.7 and 11.6 us, 500 tokens' given routes 9.7
// and 11.3.  The GPU alone would take several blocks earlier, from about 200 tokens of a
// choice on and 300 of given routes: these two are 10.5 and 8.1, 9.5 and 7.1 there, 256 of 8
// 8.1 and 6.3, 128 of 60 6.8 and 8.2.
constexpr size_t BALANCE_ONE_CHOICE = (size_t)1 << 15, BALANCE_ONE = (size_t)1 << 16;

struct RouteArgs {
  const void* scores;
  size_t ld;
  uint32_t tokens, experts, slots;
  float scale;
  int renormalize;
  int32_t* expert;   // tokens x slots; given where the routes are
  float* weight;     // tokens x slots
};

// exp(2 scale x) for x <= 0, half of a difference of scores, so that none is out of range:
// the hardware's 2^y of y = 2 x scale log2(e), the scale first, since its product with a
// constant may be out of range.  EXACT: y's own rounding is made good, so that what is left
// of an error is that of the hardware (1 ulp), of the factor (2^-26 |y|) and of x scale;
// else y is off by two roundings and the factor, which 16-bit results do not show.  Below
// 2^-126 it gives zero.
template <bool EXACT>
__device__ __forceinline__ float exp_down(float x, float scale) {
  constexpr float TWO_LOG2E = 2.88539008f, LN2 = 0.693147181f;
  if constexpr (!EXACT) return __builtin_amdgcn_exp2f(x * scale * TWO_LOG2E);
  const float a = fmaxf(x * scale, -100.0f);
  const float y = a * TWO_LOG2E, lost = fmaf(a, TWO_LOG2E, -y), p = __builtin_amdgcn_exp2f(y);
  return fmaf(p, lost * LN2, p);
}

// What scores are compared as: floats, or integers; NONE is a masked expert's.
// 16-bit scores have a key each, which orders them and names their expert: no
// two keys of a row are equal, and one maximum finds the next expert.
template <class T>
struct Score {
  typedef float W;
  static constexpr bool KEYED = sizeof(T) == 2;
  static __device__ __forceinline__ float none() { return -INFINITY; }
  static __device__ __forceinline__ float larger(float a, float b) { return __builtin_elementwise_maximum(a, b); }
  static __device__ __forceinline__ float read(T s) { return (float)s + 0.0f; }  // (-0 and 0 are equal)
  // A row whose largest score this is has no softmax: it holds a NaN or an infinity.
  static __device__ __forceinline__ bool bad(float m) { return !(m < INFINITY); }
  // exp(scale (v - m)); v <= m, m a score
  template <bool EXACT>
  static __device__ __forceinline__ float ex(float v, float m, float scale) {
    return exp_down<EXACT>(fmaf(v, 0.5f, -0.5f * m), scale);
  }
  // 0: masked, else the score's rank among all of the type above, the expert below
  static __device__ __forceinline__ uint32_t key(float v, uint32_t e) {
    uint16_t b;
    const T s = (T)v;
    __builtin_memcpy(&b, &s, 2);
    const uint32_t rank = b & 0x8000u ? (uint16_t)~b : b | 0x8000u;
    return v == none() ? 0u : rank << 16 | (0xffffu - e);
  }
  static __device__ __forceinline__ float of_key(uint32_t key) {
    const uint32_t rank = key >> 16;
    const uint16_t b = (uint16_t)(rank & 0x8000u ? rank & 0x7fffu : ~rank);
    T s;
    __builtin_memcpy(&s, &b, 2);
    return (float)s;
  }
};
template <>
struct Score<int> {
  typedef int W;
  static constexpr bool KEYED = false;
  static __device__ __forceinline__ int none() { return INT32_MIN; }
  static __device__ __forceinline__ int larger(int a, int b) { return a > b ? a : b; }
  static __device__ __forceinline__ int read(int s) { return s; }
  static __device__ __forceinline__ bool bad(int) { return false; }
  template <bool EXACT>
  static __device__ __forceinline__ float ex(int v, int m, float scale) {
    return v == none() ? 0.0f : exp_down<EXACT>(-0.5f * (float)((uint32_t)m - (uint32_t)v), scale);
  }
};

// What a lane's partner holds: the lanes of a row of 16 by data-parallel moves, which
// take no trip through LDS; after the steps before, all lanes of the partner's half
// hold the same.
template <int D, class X>
__device__ __forceinline__ X partner(X v) {
  static_assert(sizeof(X) == 4, "one register");
  int b;
  __builtin_memcpy(&b, &v, 4);
  if constexpr (D == 1) b = __builtin_amdgcn_update_dpp(b, b, 0xb1, 0xf, 0xf, false);         // quad: 1 0 3 2
  else if constexpr (D == 2) b = __builtin_amdgcn_update_dpp(b, b, 0x4e, 0xf, 0xf, false);    // quad: 2 3 0 1
  else if constexpr (D == 4) b = __builtin_amdgcn_update_dpp(b, b, 0x141, 0xf, 0xf, false);   // half row, mirrored
  else if constexpr (D == 8) b = __builtin_amdgcn_update_dpp(b, b, 0x140, 0xf, 0xf, false);   // row, mirrored
  else b = __shfl_xor(b, D);
  __builtin_memcpy(&v, &b, 4);
  return v;
}
// f over a token's L lanes; every lane has the result, and the same one.
template <int L, int D = 1, class X, class F>
__device__ __forceinline__ X over_lanes(X v, F&& f) {
  if constexpr (D < L) return over_lanes<L, 2 * D>(f(v, partner<D>(v)), f);
  else return v;
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

// N bytes at an address that is a multiple of an element's, in one piece.
template <int N, class P>
__device__ __forceinline__ void copy_piece(const P* from, P* to) {  // (one of them in registers)
  typedef int word __attribute__((aligned(2)));
  typedef int words2 __attribute__((ext_vector_type(2), aligned(2)));
  typedef int words4 __attribute__((ext_vector_type(4), aligned(2)));
  if constexpr (N == 2) *to = *from;
  else if constexpr (N == 4) *(word*)to = *(const word*)from;
  else if constexpr (N == 8) *(words2*)to = *(const words2*)from;
  else *(words4*)to = *(const words4*)from;
}

// Which of a token's experts a lane has: pieces of up to 16 bytes, so that a
// token's lanes take neighbouring ones.  Their numbers grow with i.
template <class T, int L, int V>
struct Part {
  static constexpr int C = V * sizeof(T) < 16 ? V : 16 / sizeof(T);
  static __device__ __forceinline__ uint32_t expert(uint32_t l, int i) { return (i / C) * (L * C) + l * C + i % C; }
};

// A lane's V scores of a row; those beyond its end are masked.
template <class T, int L, int V>
__device__ __forceinline__ void load_scores(const T* row, uint32_t l, uint32_t experts,
                                            typename Score<T>::W (&v)[V]) {
  typedef Part<T, L, V> P;
  T raw[V];
#pragma unroll
  for (int c = 0; c < V; c += P::C) {
    const uint32_t e = P::expert(l, c);
    if (e + P::C <= experts) {
      copy_piece<P::C * sizeof(T)>(row + e, raw + c);
    } else {
      // (read again the row's last score, so that no load waits for another)
#pragma unroll
      for (int i = 0; i < P::C; i++) raw[c + i] = row[e + i < experts ? e + i : experts - 1];
    }
  }
#pragma unroll
  for (int i = 0; i < V; i++) v[i] = P::expert(l, i) < experts ? Score<T>::read(raw[i]) : Score<T>::none();
}

// Counts and sums of p of all tokens to count, prob and loss, by a block's threads;
// expert e's from get(e) (its count, and its sum of p), loss's part of these experts
// from the first thread.  Counts below 2^24, sums in 64 bits.
template <int THREADS, class Get>
__device__ __forceinline__ double balance_of(uint32_t lo, uint32_t hi, uint32_t n, uint32_t experts, uint32_t slots,
                                             int32_t* count, float* prob, Get&& get) {
  __shared__ double part[THREADS / 64];
  double x = 0.0;
  for (uint32_t e = lo + threadIdx.x; e < hi; e += THREADS) {
    uint32_t c;
    double s;
    get(e, c, s);
    const double mean = n ? s / n : 0.0;
    count[e] = (int32_t)c;
    prob[e] = (float)mean;
    if (n) x += mean * c / ((double)n * slots);
  }
#pragma unroll
  for (int d = 32; d; d >>= 1) x += __shfl_xor(x, d);
  if (threadIdx.x % 64 == 0) part[threadIdx.x / 64] = x;
  __syncthreads();
  if (threadIdx.x == 0)
    for (int w = 1; w < THREADS / 64; w++) x += part[w];
  return x * experts;
}

// Where a call's sums go: of each block, then by expert to the caller's arrays.
struct BalanceOut {
  int32_t* count;
  float* prob;
  float* loss;
  double* loss_part;  // of each block of the last step
  uint32_t* ticket;   // blocks of the last step that are done
  float* part_prob;      // of each block: sums of p by expert
  uint32_t* part_count;  // of each block: counts by expert, and tokens with a score
};

// CHOOSE: a token's experts and weights are found; else given.  BALANCE: counts
// and sums of p are made; one block alone makes the caller's results of them.
// Bound by the launch and the chain of a token's maxima: 16384 tokens, 8 of 128 experts,
// bf16, with the balance 9.6 us (4 MB); 32768 x 256, routes given, 9.2 us (17 MB: 1.8 TB/s),
// traced.
template <class T, int L, int V, bool CHOOSE, bool BALANCE>
__global__ __launch_bounds__(BALANCE ? balance_threads(L) : ROUTE_THREADS) void k_route(RouteArgs a, BalanceOut out) {
  typedef Score<T> S;
  typedef Part<T, L, V> P;
  typedef typename S::W W;
  constexpr uint32_t THREADS = BALANCE ? balance_threads(L) : ROUTE_THREADS, GROUPS = THREADS / L, WAVES = THREADS / 64;
  constexpr int KEPT = (ZK_MAX_SLOTS + L - 1) / L;
  __shared__ uint32_t count[BALANCE ? L * V + 1 : 1];
  __shared__ float sums[BALANCE ? WAVES * L * V : 1];
  const uint32_t tid = threadIdx.x, l = tid % L;
  if (BALANCE) {
    for (uint32_t e = tid; e <= a.experts; e += THREADS) count[e] = 0;
    if (blockIdx.x == 0 && tid == 0 && gridDim.x > 1) *out.ticket = 0;
    __syncthreads();
  }
  float psum[V] = {};
  const bool all = BALANCE || !a.renormalize;  // whether every score's exponential is needed
  for (uint32_t t0 = blockIdx.x * GROUPS; t0 < a.tokens; t0 += gridDim.x * GROUPS) {
    const uint32_t t = t0 + tid / L;
    if (t >= a.tokens) continue;  // (all of the token's lanes)
    int given[KEPT];
    if (!CHOOSE) {
#pragma unroll
      for (int k = 0; k < KEPT; k++) given[k] = l + k * L < a.slots ? a.expert[(size_t)t * a.slots + l + k * L] : -1;
    }
    W v[V];
    load_scores<T, L, V>((const T*)a.scores + (size_t)t * a.ld, l, a.experts, v);
    W top = S::none();
#pragma unroll
    for (int i = 0; i < V; i++) top = S::larger(top, v[i]);
    const W m = over_lanes<L>(top, S::larger);
    const bool bad = S::bad(m), empty = m == S::none();
    float inv = 0.0f;
    if (all && !bad && !empty) {
      float p[V], z = 0.0f;
#pragma unroll
      for (int i = 0; i < V; i++) z += p[i] = S::template ex<true>(v[i], m, a.scale);
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
#pragma unroll
      for (int k = 0; k < KEPT; k++)
        if (!empty && (uint32_t)given[k] < a.experts) atomicAdd(&count[given[k]], 1u);
      continue;
    }
    int kept_e[KEPT];
    W kept[KEPT];
#pragma unroll
    for (int k = 0; k < KEPT; k++) kept_e[k] = -1, kept[k] = S::none();
    uint32_t key[S::KEYED ? V : 1];
    if constexpr (S::KEYED) {
#pragma unroll
      for (int i = 0; i < V; i++) key[i] = S::key(v[i], P::expert(l, i));
    }
    for (uint32_t j = 0; j < a.slots && !bad; j++) {
      W best = S::none();
      uint32_t e = a.experts;
      if constexpr (S::KEYED) {
        uint32_t b = 0;
#pragma unroll
        for (int i = 0; i < V; i++) b = key[i] > b ? key[i] : b;
        b = max_over<L>(b);
        if (!b) break;
#pragma unroll
        for (int i = 0; i < V; i++) key[i] = key[i] == b ? 0u : key[i];
        e = 0xffffu - (b & 0xffffu);
        best = S::of_key(b);
      } else {
        // a lane's first largest score, then the lowest expert that has the largest of all
        W b = S::none();
#pragma unroll
        for (int i = 0; i < V; i++)
          if (v[i] > b) b = v[i], e = P::expert(l, i);
        best = over_lanes<L>(b, S::larger);
        if (best == S::none()) break;
        e = min_over<L>(b == best ? e : a.experts);
#pragma unroll
        for (int i = 0; i < V; i++)
          if (P::expert(l, i) == e) v[i] = S::none();
      }
#pragma unroll
      for (int k = 0; k < KEPT; k++)
        if (j == l + k * L) kept_e[k] = (int)e, kept[k] = best;
    }
    // the weights, each by the lane that keeps it
    float w[KEPT], total = 0.0f;
#pragma unroll
    for (int k = 0; k < KEPT; k++) total += w[k] = kept_e[k] < 0 ? 0.0f : S::template ex<true>(kept[k], m, a.scale);
    float by = inv;
    if (a.renormalize) {
      total = sum_over<L>(total);
      by = total > 0.0f ? 1.0f / total : 0.0f;
    }
    if (bad) by = NAN;
#pragma unroll
    for (int k = 0; k < KEPT; k++)
      if (l + k * L < a.slots) {
        const size_t at = (size_t)t * a.slots + l + k * L;
        a.expert[at] = kept_e[k];
        a.weight[at] = w[k] * by;
        if (BALANCE && kept_e[k] >= 0) atomicAdd(&count[kept_e[k]], 1u);
      }
  }
  if constexpr (BALANCE) {
    // the wave's tokens, then the waves, in a fixed order
#pragma unroll
    for (int i = 0; i < V; i++) {
#pragma unroll
      for (int d = L; d < 64; d <<= 1) psum[i] += __shfl_xor(psum[i], d);
      if (tid % 64 < L) sums[(tid / 64) * L * V + P::expert(l, i)] = psum[i];
    }
    __syncthreads();
    auto sum = [&](uint32_t e) {
      float s = sums[e];
#pragma unroll
      for (uint32_t w = 1; w < WAVES; w++) s += sums[w * L * V + e];
      return s;
    };
    if (gridDim.x == 1) {
      const uint32_t n = count[a.experts];
      const double loss = balance_of<THREADS>(0, a.experts, n, a.experts, a.slots, out.count, out.prob,
                                              [&](uint32_t e, uint32_t& c, double& s) { c = count[e], s = sum(e); });
      if (tid == 0) *out.loss = (float)loss, out.count[a.experts] = (int32_t)n;
      return;
    }
    for (uint32_t e = tid; e <= a.experts; e += THREADS) {
      out.part_count[(size_t)blockIdx.x * (a.experts + 1) + e] = count[e];
      if (e < a.experts) out.part_prob[(size_t)blockIdx.x * a.experts + e] = sum(e);
    }
  }
}

// The blocks' counts and sums to the caller's: a block has 32 experts and shares the
// blocks' rows among eight threads each, in a fixed order; the loss is put together by
// the block that is done last, from all blocks' parts in their order.  256 blocks of 256
// experts: 5.7 us traced, two chains of loads behind a launch.
constexpr uint32_t FINISH_EXPERTS = 32;
__global__ __launch_bounds__(256) void k_balance_finish(BalanceOut out, uint32_t blocks, uint32_t experts,
                                                        uint32_t slots) {
  constexpr uint32_t E = FINISH_EXPERTS, PARTS = 256 / E;
  __shared__ uint32_t c_part[PARTS][E], n_part[4];
  __shared__ double s_part[PARTS][E];
  const uint32_t tid = threadIdx.x, x = tid % E, y = tid / E, e = blockIdx.x * E + x;
  uint32_t c = 0, n = 0;
  double s = 0.0;
  static_assert(BALANCE_BLOCKS <= 256, "a thread a block");
  if (tid < blocks) n = out.part_count[(size_t)tid * (experts + 1) + experts];
  // (loads of rows and experts that are not there are of others, so that 16 rows' are
  // under way together)
  const uint32_t col = e < experts ? e : experts - 1;
  for (uint32_t b0 = y; b0 < blocks; b0 += 16 * PARTS) {
    uint32_t ci[16];
    float si[16];
#pragma unroll
    for (uint32_t i = 0; i < 16; i++) {
      const uint32_t b = b0 + i * PARTS < blocks ? b0 + i * PARTS : b0;
      ci[i] = out.part_count[(size_t)b * (experts + 1) + col];
      si[i] = out.part_prob[(size_t)b * experts + col];
    }
#pragma unroll
    for (uint32_t i = 0; i < 16; i++)
      if (b0 + i * PARTS < blocks) c += ci[i], s += si[i];
  }
#pragma unroll
  for (int d = 32; d; d >>= 1) n += __shfl_xor(n, d);
  if (tid % 64 == 0) n_part[tid / 64] = n;
  c_part[y][x] = c, s_part[y][x] = s;
  __syncthreads();
  n = n_part[0] + n_part[1] + n_part[2] + n_part[3];
  const uint32_t lo = blockIdx.x * E, hi = lo + E < experts ? lo + E : experts;
  double loss = balance_of<256>(lo, hi, n, experts, slots, out.count, out.prob,
                                [&](uint32_t f, uint32_t& fc, double& fs) {
                                  fc = 0, fs = 0.0;
#pragma unroll
                                  for (uint32_t p = 0; p < PARTS; p++) fc += c_part[p][f - lo], fs += s_part[p][f - lo];
                                });
  if (tid) return;
  if (blockIdx.x == 0) out.count[experts] = (int32_t)n;
  if (gridDim.x > 1) {
    __hip_atomic_store(&out.loss_part[blockIdx.x], loss, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    const uint32_t done = __hip_atomic_fetch_add(out.ticket, 1u, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT);
    if (done + 1 < gridDim.x) return;
    loss = 0.0;
    for (uint32_t b = 0; b < gridDim.x; b++)
      loss += __hip_atomic_load(&out.loss_part[b], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  *out.loss = (float)loss;
}

// ------------------------------------------------------------ gradient
// One pass as k_route's: 32768 x 256, bf16, 10.4 us traced (34 MB: 3.3 TB/s).
struct RouteGradArgs {
  const void* scores;
  size_t ld, ld_grad;
  uint32_t tokens, experts, slots;
  float scale;
  float in, out;             // factors of what comes in and of the gradient; their product is the scale
  const int32_t* expert;
  const float* grad_weight;  // or null
  const int32_t* count;      // or null
  const float* grad_loss;
  void* grad;
};

template <class T, int L, int V, bool NORMAL>
__global__ __launch_bounds__(ROUTE_THREADS) void k_route_grad(RouteGradArgs a) {
  typedef Score<T> S;
  typedef Part<T, L, V> P;
  constexpr uint32_t GROUPS = ROUTE_THREADS / L;
  constexpr int KEPT = (ZK_MAX_SLOTS + L - 1) / L;
  constexpr bool EXACT = sizeof(T) == 4;
  const uint32_t tid = threadIdx.x, l = tid % L;
  // the loss's gradients of the mean probabilities, g experts / n f, by way of LDS: a
  // few lines of counts that every lane of the chip asks the L2 for cost 11 us of 20
  // (32768 tokens, 256 experts)
  float f[V] = {};
  if (a.count) {
    __shared__ float shared[L * V];
    const float n = (float)a.count[a.experts], g = *a.grad_loss * a.in;
    const float per = n > 0.0f ? g * ((float)a.experts / (n * n * (float)a.slots)) : 0.0f;
    for (uint32_t e = tid; e < L * V; e += ROUTE_THREADS) shared[e] = e < a.experts ? (float)a.count[e] * per : 0.0f;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < V; i++) f[i] = shared[P::expert(l, i)];
  }
  for (uint32_t t0 = blockIdx.x * GROUPS; t0 < a.tokens; t0 += gridDim.x * GROUPS) {
    const uint32_t t = t0 + tid / L;
    if (t >= a.tokens) continue;  // (all of the token's lanes)
    float v[V], d[V];
    // the token's routes, a lane each (two where there are more than lanes)
    int named[KEPT];
    float gw[KEPT];
#pragma unroll
    for (int k = 0; k < KEPT; k++) {
      const bool on = a.grad_weight && l + k * L < a.slots;
      const size_t at = (size_t)t * a.slots + l + k * L;
      named[k] = on ? a.expert[at] : -1;
      gw[k] = on ? a.grad_weight[at] * a.in : 0.0f;
    }
    load_scores<T, L, V>((const T*)a.scores + (size_t)t * a.ld, l, a.experts, v);
    float top = S::none();
#pragma unroll
    for (int i = 0; i < V; i++) top = S::larger(top, v[i]);
    const float m = over_lanes<L>(top, S::larger);
    const bool bad = S::bad(m);
    // g: gradients of the experts' weights; times: routes that name them
    float g[V] = {}, times[V] = {};
    if (a.grad_weight)
      for (uint32_t j = 0; j < a.slots; j++) {
        int e = __shfl(named[0], j, L);
        float gj = __shfl(gw[0], j, L);
        if constexpr (KEPT > 1) {
          if (j >= L) e = __shfl(named[1], j - L, L), gj = __shfl(gw[1], j - L, L);
        }
        if ((uint32_t)e >= a.experts) continue;
#pragma unroll
        for (int i = 0; i < V; i++)
          if (P::expert(l, i) == (uint32_t)e) {
            g[i] += gj;
            if (NORMAL) times[i] += 1.0f;
          }
      }
    // with p = e / z: all that depends on p has the gradient p (G - sum p G)
    float z = 0.0f, dot = 0.0f, ez[V];
#pragma unroll
    for (int i = 0; i < V; i++) {
      const float G = NORMAL ? f[i] : f[i] + g[i];
      z += ez[i] = S::template ex<EXACT>(v[i], m, a.scale);
      dot = fmaf(ez[i], G, dot);
    }
    const float inv = 1.0f / sum_over<L>(z);
    dot = sum_over<L>(dot) * inv;
    const float by = bad ? NAN : inv * a.out;
#pragma unroll
    for (int i = 0; i < V; i++) d[i] = ez[i] * ((NORMAL ? f[i] : f[i] + g[i]) - dot) * by;
    if constexpr (NORMAL) {
      // softmax over the chosen alone: their own maximum, sum and mean
      float mc = S::none(), zc = 0.0f, gc = 0.0f;
#pragma unroll
      for (int i = 0; i < V; i++) mc = times[i] > 0.0f ? S::larger(mc, v[i]) : mc;
      mc = over_lanes<L>(mc, S::larger);
#pragma unroll
      for (int i = 0; i < V; i++) {
        ez[i] = times[i] > 0.0f && v[i] > S::none() ? S::template ex<EXACT>(v[i], mc, a.scale) : 0.0f;
        zc = fmaf(times[i], ez[i], zc);
        gc = fmaf(g[i], ez[i], gc);
      }
      zc = sum_over<L>(zc), gc = sum_over<L>(gc);
      const float ic = zc > 0.0f ? 1.0f / zc : 0.0f, byc = ic * a.out;
      gc *= ic;
#pragma unroll
      for (int i = 0; i < V; i++) d[i] = fmaf(ez[i] * fmaf(-times[i], gc, g[i]), byc, d[i]);
    }
    T out[V];
    // an impossible row's are NaN, else a masked score's is zero (a masked row's sums are of
    // nothing, and an infinity or a NaN that came in is one times zero too)
    const float gone = bad ? NAN : S::none();
#pragma unroll
    for (int i = 0; i < V; i++) out[i] = (T)(v[i] == gone ? 0.0f : d[i]);
    T* row = (T*)a.grad + (size_t)t * a.ld_grad;
#pragma unroll
    for (int k = 0; k < V; k += P::C) {
      const uint32_t e = P::expert(l, k);
      if (e + P::C <= a.experts) {
        copy_piece<P::C * sizeof(T)>(out + k, row + e);
      } else {
#pragma unroll
        for (int i = 0; i < P::C; i++)
          if (e + i < a.experts) row[e + i] = out[k + i];
      }
    }
  }
}

// ------------------------------------------------------------ which lanes
// Calls fn with the lanes a token gets and the scores of a lane: 16 lanes, whose
// reductions need no LDS, as long as their scores fit the registers.
template <class Fn>
static int by_experts(uint32_t experts, Fn&& fn) {
  using std::integral_constant;
  const integral_constant<int, 16> row;
  if (experts <= 16) return fn(row, integral_constant<int, 1>());
  if (experts <= 32) return fn(row, integral_constant<int, 2>());
  if (experts <= 64) return fn(row, integral_constant<int, 4>());
  if (experts <= 128) return fn(row, integral_constant<int, 8>());
  if (experts <= 256) return fn(row, integral_constant<int, 16>());
  if (experts <= 512) return fn(integral_constant<int, 32>(), integral_constant<int, 16>());
  return fn(integral_constant<int, 64>(), integral_constant<int, 16>());
}
static int lanes_of(int experts) { return experts <= 256 ? 16 : experts <= 512 ? 32 : 64; }

static uint32_t route_blocks(size_t tokens, uint32_t a_block, uint32_t most) {
  const uint32_t b = cdiv(tokens, a_block);
  return b < most ? b : most;
}
static uint32_t balance_blocks(size_t tokens, int experts, bool choose) {
  if (tokens * (experts + 64) <= (choose ? BALANCE_ONE_CHOICE : BALANCE_ONE)) return 1;
  const int lanes = lanes_of(experts);
  return route_blocks(tokens, balance_threads(lanes) / lanes, BALANCE_BLOCKS);
}
// A workspace: the last step's parts of the loss and ticket, then the blocks' sums and
// counts; none for one block.
static size_t balance_work(size_t tokens, int experts, bool choose) {
  const uint32_t blocks = balance_blocks(tokens, experts, choose);
  return blocks > 1 ? 8 * (ZK_MAX_EXPERTS / FINISH_EXPERTS + 1) + (size_t)blocks * (2 * experts + 1) * 4 : 0;
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
static int route(zk_context* ctx, const RouteArgs& a, int type, BalanceOut out, void* work, size_t work_bytes,
                 hipStream_t st) {
  const bool balance = out.count != nullptr;
  const uint32_t blocks = balance_blocks(a.tokens, (int)a.experts, CHOOSE);
  if (balance) {
    const size_t need = balance_work(a.tokens, (int)a.experts, CHOOSE);
    if (need && (!work || !aligned(work, 8) || work_bytes < need))
      return ctx->fail(ZK_ERR_INVALID, "experts' route: workspace missing, too small or not aligned to 8 bytes");
    constexpr size_t PARTS = ZK_MAX_EXPERTS / FINISH_EXPERTS;
    out.loss_part = (double*)work;
    out.ticket = (uint32_t*)(out.loss_part + PARTS);
    out.part_prob = (float*)(out.loss_part + PARTS + 1);
    out.part_count = (uint32_t*)(out.part_prob + (size_t)blocks * a.experts);
  } else if (!a.tokens) {
    return ZK_OK;
  }
  const char* name = CHOOSE ? "experts_route" : "experts_balance";
  ZK_TRY(by_score_type(type, [&](auto zero) -> int {
    typedef decltype(zero) T;
    return by_experts(a.experts, [&](auto lanes, auto per) -> int {
      constexpr int L = decltype(lanes)::value, V = decltype(per)::value;
      if (balance) {
        ZK_LAUNCH(ctx, st, name, (k_route<T, L, V, CHOOSE, true>), dim3(blocks), dim3(balance_threads(L)), 0, a, out);
      } else if constexpr (CHOOSE) {
        ZK_LAUNCH(ctx, st, name, (k_route<T, L, V, true, false>),
                  dim3(route_blocks(a.tokens, ROUTE_THREADS / L, ROUTE_BLOCKS)), dim3(ROUTE_THREADS), 0, a, out);
      }
      return ZK_OK;
    });
  }));
  if (balance && blocks > 1)
    ZK_LAUNCH(ctx, st, name, k_balance_finish, dim3(cdiv(a.experts, FINISH_EXPERTS)), dim3(256), 0, out, blocks,
              a.experts, a.slots);
  return ZK_OK;
}

}  // namespace zk

extern "C" {

size_t zk_experts_route_work(size_t tokens, int experts) {
  using namespace zk;
  if (experts < 1 || experts > ZK_MAX_EXPERTS || tokens > ZK_MAX_EXPERT_ROWS) return 0;
  return balance_work(tokens, experts, true);  // (the more of the two)
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
                         d_expert, d_weight};
    const BalanceOut out = {d_count, d_prob, d_loss, nullptr, nullptr, nullptr, nullptr};
    return route<true>(ctx, a, type, out, d_work, work_bytes, ctx->s(stream));
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
                         (int32_t*)d_expert, nullptr};
    const BalanceOut out = {d_count, d_prob, d_loss, nullptr, nullptr, nullptr, nullptr};
    return route<false>(ctx, a, type, out, d_work, work_bytes, ctx->s(stream));
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
    // a small scale has its product with a probability's sum in 32 bits' normal numbers
    // only if what comes in gives up 64 of the powers of two
    const float in = scale < 0x1p-100f ? 0x1p-64f : 1.0f;
    const RouteGradArgs a = {d_scores, ld, ld_grad, (uint32_t)tokens, (uint32_t)experts, (uint32_t)slots, scale, in,
                             scale / in, d_expert, d_grad_weight, d_count, d_grad_loss, d_grad_scores};
    hipStream_t st = ctx->s(stream);
    return by_type(type, [&](auto zero) -> int {
      typedef decltype(zero) T;
      return by_experts(a.experts, [&](auto lanes, auto per) -> int {
        constexpr int L = decltype(lanes)::value, V = decltype(per)::value;
        const dim3 grid(route_blocks(tokens, ROUTE_THREADS / L, ROUTE_BLOCKS));
        if (renormalize && d_grad_weight)
          ZK_LAUNCH(ctx, st, "experts_route_grad", (k_route_grad<T, L, V, true>), grid, dim3(ROUTE_THREADS), 0, a);
        else
          ZK_LAUNCH(ctx, st, "experts_route_grad", (k_route_grad<T, L, V, false>), grid, dim3(ROUTE_THREADS), 0, a);
        return ZK_OK;
      });
    });
  });
}

}  // extern "C"
