// Routed experts for gfx950: samples sorted by the expert (the class, the
// model) that their route names, their rows gathered in that order, the
// experts' answers put back with the routes' weights, and the gradients.
//
// A pair i = token * slots + j is a token's j-th route.  The sort is a stable
// counting sort of the pairs by expert:
//   offsets[e] = number of pairs with an expert below e
//   place[i]   = offsets[e_i] + number of pairs before i with the same expert
//   order[place[i]] = i
// A pair whose expert is outside [0, experts) is dropped: place -1, and order
// holds -1 behind the last sorted pair.  No result depends on the order in
// which blocks or atomics run.
#include "rows.hpp"
#include "zk_internal.hpp"

namespace zk {

// ------------------------------------------------------------ sort
constexpr int SORT_THREADS = 1024, SORT_WAVES = SORT_THREADS / 64;
// Few pairs are sorted by one block, whose time grows with them (128 experts:
// 2048 pairs 4.9 us, 8192 10.9, 16384 would be 19.6; 66 pairs to 8 experts 3.3); more
// by blocks of 2048 pairs or more, in two launches, the second of which adds up the
// blocks' counts (16384: 2.4 + 5.9 us, 65536: 2.4 + 6.8, 2^20: 4.1 + 17.5, to 1024
// experts 4.9 + 53; a launch costs the host 4 us).
// Bound by the chain launch, loads, counts, scan, loads; the pairs' own bytes are
// nothing beside it (65536: 0.8 MB).
constexpr size_t SORT_ONE = 8192;     // pairs that one block sorts alone
constexpr size_t SORT_SEGMENT = 2048; // least pairs of a block otherwise
constexpr size_t SORT_BLOCKS = 128;   // (more counts to add up cost more than they save)

struct SortPlan {
  uint32_t blocks, segment;
};
static SortPlan sort_plan(size_t pairs) {
  SortPlan p = {1, 0};
  if (pairs > SORT_ONE) {
    p.blocks = cdiv(pairs, SORT_SEGMENT);
    if (p.blocks > SORT_BLOCKS) p.blocks = SORT_BLOCKS;
  }
  p.segment = cdiv(pairs, (size_t)p.blocks * SORT_THREADS) * SORT_THREADS;
  return p;
}

// What a wave's lanes wrote to LDS before it, its other lanes read after it: all
// lanes meet here, and the compiler moves no access across.  No instruction: one
// wave's LDS accesses are in order.
__device__ __forceinline__ void lanes_meet() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// Counts of one block's pairs by expert: tot[block][expert].
__global__ __launch_bounds__(SORT_THREADS) void k_sort_count(const int32_t* __restrict__ expert, uint32_t pairs,
                                                             uint32_t experts, uint32_t segment,
                                                             uint32_t* __restrict__ tot) {
  __shared__ uint32_t c[ZK_MAX_EXPERTS];
  for (uint32_t e = threadIdx.x; e < experts; e += SORT_THREADS) c[e] = 0;
  __syncthreads();
  const uint32_t lo = blockIdx.x * segment, hi = lo + segment < pairs ? lo + segment : pairs;
  for (uint32_t i = lo + threadIdx.x; i < hi; i += SORT_THREADS) {
    const uint32_t e = (uint32_t)expert[i];
    if (e < experts) atomicAdd(&c[e], 1u);
  }
  __syncthreads();
  for (uint32_t e = threadIdx.x; e < experts; e += SORT_THREADS) tot[(size_t)blockIdx.x * experts + e] = c[e];
}

// Places of one block's pairs.  A wave owns a run of the block's segment, so
// its own counts and a prefix over the waves give each run's first place.
__global__ __launch_bounds__(SORT_THREADS) void k_sort_place(const int32_t* __restrict__ expert, uint32_t pairs,
                                                             uint32_t experts, uint32_t segment,
                                                             const uint32_t* __restrict__ tot,
                                                             int32_t* __restrict__ offsets,
                                                             int32_t* __restrict__ order,
                                                             int32_t* __restrict__ place) {
  __shared__ uint32_t cnt[SORT_WAVES * ZK_MAX_EXPERTS];
  __shared__ uint32_t base[ZK_MAX_EXPERTS], sum[ZK_MAX_EXPERTS];
  __shared__ uint32_t scan[SORT_WAVES];
  const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const uint32_t seg0 = blockIdx.x * segment, run = segment / SORT_WAVES;
  const uint32_t lo = seg0 + wave * run;
  uint32_t hi = lo + run;
  if (hi > pairs) hi = pairs;
  uint32_t* mine = cnt + wave * experts;  // read and written by different lanes of the wave
  for (uint32_t e = tid; e < SORT_WAVES * experts; e += SORT_THREADS) cnt[e] = 0;
  if (tid < experts) base[tid] = sum[tid] = 0;
  __syncthreads();
  for (uint32_t i = lo + lane; i < hi; i += 64) {
    const uint32_t e = (uint32_t)expert[i];
    if (e < experts) atomicAdd(&mine[e], 1u);
  }
  __syncthreads();
  // thread e: the pairs of expert e in each wave of this block before the next,
  // and, over the blocks, in all of them and in those before this one
  uint32_t all = 0, before = 0, here = 0;
  if (tid < experts) {
    for (uint32_t w = 0; w < SORT_WAVES; w++) {
      const uint32_t c = cnt[w * experts + tid];
      cnt[w * experts + tid] = here;
      here += c;
    }
    all = here;
  }
  if (tot) {
    // the blocks' counts are shared out over all threads, so that a thread has
    // few loads to wait for; the sums are integers, their order does not matter
    const uint32_t mark = blockIdx.x * experts, last = gridDim.x * experts;
#pragma unroll 4
    for (uint32_t i = tid; i < last; i += SORT_THREADS) {
      const uint32_t c = tot[i], e = i % experts;
      atomicAdd(&sum[e], c);
      if (i < mark) atomicAdd(&base[e], c);
    }
    __syncthreads();
    if (tid < experts) all = sum[tid], before = base[tid];
  }
  // exclusive scan of `all` over the experts
  uint32_t s = all;
  for (int d = 1; d < 64; d <<= 1) {
    const uint32_t o = __shfl_up(s, d);
    if (lane >= (uint32_t)d) s += o;
  }
  if (lane == 63) scan[wave] = s;
  __syncthreads();
  uint32_t carry = 0, total = 0;
  for (int w = 0; w < SORT_WAVES; w++) {
    if ((uint32_t)w < wave) carry += scan[w];
    total += scan[w];
  }
  s += carry;
  if (tid < experts) {
    base[tid] = s - all + before;
    if (blockIdx.x == 0) offsets[tid] = (int32_t)(s - all);
  }
  if (tid == 0 && blockIdx.x == 0) offsets[experts] = (int32_t)total;
  __syncthreads();
  const int bits = 32 - __clz((int)experts);  // experts itself stands for dropped
  for (uint32_t c0 = lo; c0 < hi; c0 += 64) {
    const uint32_t i = c0 + lane;
    uint32_t e = i < hi ? (uint32_t)expert[i] : experts;
    if (e > experts) e = experts;
    // the lanes with the same expert
    uint64_t same = ~0ull;
    for (int b = 0; b < bits; b++) {
      const bool bit = (e >> b) & 1u;
      const uint64_t v = __ballot(bit);
      same &= bit ? v : ~v;
    }
    const uint32_t rank = (uint32_t)__popcll(same & ((1ull << lane) - 1));
    uint32_t first = 0;
    // every lane reads before any writes, and the next 64 pairs' lanes after it
    if (e < experts) first = mine[e];
    lanes_meet();
    if (e < experts && rank == 0) mine[e] = first + (uint32_t)__popcll(same);
    lanes_meet();
    if (i < hi) {
      int32_t p = -1;
      if (e < experts) {
        p = (int32_t)(base[e] + first + rank);
        order[p] = (int32_t)i;
      }
      place[i] = p;
      if (i >= total) order[i] = -1;
    }
  }
}

// ------------------------------------------------------------ rows
// out[p] = x[order[p] / slots], zeros where order[p] names no token: 2^log_w
// threads a row, so that short rows fill a wave.  STREAM: see streams().
// Bound by memory: 65536 rows of 4 KB from 16384 in 73 us, 335 MB at 4.6 TB/s
// (55 us at a copy's 6.05: a token's four rows are wanted far apart in the sorted
// order, so that some are fetched again).
template <class T, bool STREAM>
__global__ __launch_bounds__(256) void k_gather(const T* __restrict__ x, size_t ld_x,
                                                const int32_t* __restrict__ order, uint32_t rows, uint32_t tokens,
                                                uint32_t slots, uint32_t cols, uint32_t log_w, T* __restrict__ out,
                                                size_t ld_out) {
  const uint32_t p = blockIdx.x * (256u >> log_w) + (threadIdx.x >> log_w);
  if (p >= rows) return;
  const int o = order[p];
  const uint32_t t = o < 0 ? tokens : (uint32_t)o / slots;
  const uint32_t pieces = pieces_of<T>(cols);
  for (uint32_t c = threadIdx.x & ((1u << log_w) - 1); c < pieces; c += 1u << log_w) {
    const uint32_t at = piece<T>(c, cols);
    Vec<T> v = {};
    if (t < tokens) v = row_load(x + (size_t)t * ld_x + at, cols - at);
    row_store<T, STREAM>(out + (size_t)p * ld_out + at, cols - at, v);
  }
}

// out[t] = sum_j w[t, j] y[place[t, j]], j ascending, in 32 bits; 2^log_w threads
// a token.  Four slots' indexes, then their rows, are loaded together: a token's
// slots are one chain of two loads per four, not per slot.  Bound by memory: 16384
// tokens' four rows of 4 KB in 53 us, 6.3 TB/s.
template <class T, bool STREAM>
__global__ __launch_bounds__(256) void k_combine(const T* __restrict__ y, size_t ld_y,
                                                 const int32_t* __restrict__ place, const float* __restrict__ weight,
                                                 uint32_t rows, uint32_t tokens, uint32_t slots, uint32_t cols,
                                                 uint32_t log_w, T* __restrict__ out, size_t ld_out) {
  constexpr int K = 4;
  const uint32_t t = blockIdx.x * (256u >> log_w) + (threadIdx.x >> log_w);
  if (t >= tokens) return;
  const uint32_t pieces = pieces_of<T>(cols);
  for (uint32_t c = threadIdx.x & ((1u << log_w) - 1); c < pieces; c += 1u << log_w) {
    const uint32_t at = piece<T>(c, cols);
    float s[Vec<T>::N] = {};
    for (uint32_t j0 = 0; j0 < slots; j0 += K) {
      uint32_t p[K];
      float w[K];
      Vec<T> v[K];
#pragma unroll
      for (int k = 0; k < K; k++) {
        const size_t pair = (size_t)t * slots + j0 + k;
        const bool on = j0 + k < slots;
        p[k] = on ? (uint32_t)place[pair] : rows;
        w[k] = on && weight ? weight[pair] : 1.0f;
      }
#pragma unroll
      for (int k = 0; k < K; k++)
        if (p[k] < rows) v[k] = row_load<T, STREAM>(y + (size_t)p[k] * ld_y + at, cols - at);
#pragma unroll
      for (int k = 0; k < K; k++)
        if (p[k] < rows) {
#pragma unroll
          for (uint32_t e = 0; e < Vec<T>::N; e++) s[e] += w[k] * (float)v[k].v[e];
        }
    }
    Vec<T> r;
#pragma unroll
    for (uint32_t e = 0; e < Vec<T>::N; e++) r.v[e] = (T)s[e];
    row_store<T, STREAM>(out + (size_t)t * ld_out + at, cols - at, r);
  }
}

// dy[place[t, j]] = w[t, j] g[t], dw[t, j] = <g[t], y[place[t, j]]>; rows of dy
// that hold no pair get zeros.  A block has a token, so that g's row is read
// once and each dot product ends in one block, whose order is fixed; four slots
// go together.  Bound by memory: 16384 tokens' four rows of 4 KB in 102 us, 604 MB
// at 5.9 TB/s.
template <class T, bool STREAM>
__global__ __launch_bounds__(256) void k_combine_grad(const T* __restrict__ g, size_t ld_g, const T* __restrict__ y,
                                                      size_t ld_y, const int32_t* __restrict__ order,
                                                      const int32_t* __restrict__ place,
                                                      const float* __restrict__ weight, uint32_t rows,
                                                      uint32_t slots, uint32_t cols, T* __restrict__ dy, size_t ld_dy,
                                                      float* __restrict__ dw) {
  constexpr int K = 4;
  __shared__ float part[K][4];
  const uint32_t t = blockIdx.x, tid = threadIdx.x, pairs = gridDim.x * slots;
  const uint32_t pieces = pieces_of<T>(cols);
  for (uint32_t j0 = 0; j0 < slots; j0 += K) {
    const size_t pair = (size_t)t * slots + j0;
    uint32_t p[K];
    float w[K], s[K] = {};
    bool empty[K];  // does position `pair + k` hold none of the pairs?
#pragma unroll
    for (int k = 0; k < K; k++) {
      const bool on = j0 + k < slots;
      p[k] = on ? (uint32_t)place[pair + k] : rows;
      w[k] = on && weight ? weight[pair + k] : 1.0f;
      empty[k] = on && pair + k < rows && (uint32_t)order[pair + k] >= pairs;
    }
    for (uint32_t c = tid; c < pieces; c += 256) {
      const uint32_t at = piece<T>(c, cols), left = cols - at;
      const uint32_t fresh = c * Vec<T>::N - at;  // elements that the piece before has too
      const Vec<T> gv = row_load(g + (size_t)t * ld_g + at, left);
      Vec<T> yv[K];
#pragma unroll
      for (int k = 0; k < K; k++) {
        yv[k] = Vec<T>{};
        if (dw && p[k] < rows) yv[k] = row_load<T, STREAM>(y + (size_t)p[k] * ld_y + at, left);
      }
#pragma unroll
      for (int k = 0; k < K; k++) {
        if (empty[k]) row_store<T, STREAM>(dy + (pair + k) * ld_dy + at, left, Vec<T>{});
        if (p[k] >= rows) continue;
        Vec<T> r;
#pragma unroll
        for (uint32_t e = 0; e < Vec<T>::N; e++) {
          r.v[e] = (T)(w[k] * (float)gv.v[e]);
          if (e >= fresh) s[k] += (float)gv.v[e] * (float)yv[k].v[e];
        }
        row_store<T, STREAM>(dy + (size_t)p[k] * ld_dy + at, left, r);
      }
    }
    if (!dw) continue;
#pragma unroll
    for (int d = 32; d; d >>= 1)
#pragma unroll
      for (int k = 0; k < K; k++) s[k] += __shfl_xor(s[k], d);
    if (j0) __syncthreads();  // the last four's sums are read
    if ((tid & 63) == 0)
#pragma unroll
      for (int k = 0; k < K; k++) part[k][tid >> 6] = s[k];
    __syncthreads();
    if (tid < K && j0 + tid < slots) dw[pair + tid] = part[tid][0] + part[tid][1] + part[tid][2] + part[tid][3];
  }
}

// Whether a call's rows pass the caches (32 MB of L2): what is read or written
// once then goes around them and leaves them to the rows that are read again
// (in turn, gather of 65536 rows of 4 KB 69 us, 84 through the caches); smaller rows stay
// for whoever reads them next.
static bool streams(size_t rows, size_t cols, size_t size) { return rows * cols * size > (size_t)32 << 20; }

// log2 of the threads that a row gets: its pieces, from 8 to 256.
template <class T>
static uint32_t log_threads(size_t cols) {
  uint32_t l = 3;
  while (l < 8 && (1u << l) < pieces_of<T>((uint32_t)cols)) l++;
  return l;
}

// ------------------------------------------------------------ arguments
static int check_experts(zk_context* ctx, size_t pairs, int experts) {
  if (experts < 1 || experts > ZK_MAX_EXPERTS) return ctx->fail(ZK_ERR_SIZE, "experts: between 1 and 1024 experts");
  if (pairs > ZK_MAX_EXPERT_ROWS) return ctx->fail(ZK_ERR_SIZE, "experts: more than 2^22 pairs");
  return ZK_OK;
}

static int check_rows(zk_context* ctx, int type, size_t rows, size_t tokens, int slots, size_t cols) {
  if (!float_type(type))
    return ctx->fail(ZK_ERR_INVALID, "experts: rows are f32, f16 or bf16");
  if (slots < 1) return ctx->fail(ZK_ERR_INVALID, "experts: slots is at least 1");
  if (rows > ZK_MAX_EXPERT_ROWS || tokens > ZK_MAX_EXPERT_ROWS || tokens * (size_t)slots > ZK_MAX_EXPERT_ROWS)
    return ctx->fail(ZK_ERR_SIZE, "experts: more than 2^22 pairs");
  if (cols > 0x7fffffffu) return ctx->fail(ZK_ERR_SIZE, "experts: rows longer than 2^31 - 1");
  return ZK_OK;
}

static int check_matrix(zk_context* ctx, const void* p, int type, size_t ld, size_t cols) {
  if (ld < cols) return ctx->fail(ZK_ERR_INVALID, "experts: a row stride below the row's length");
  if (!p) return ctx->fail(ZK_ERR_INVALID, "experts: null pointer");
  if (!aligned(p, type_bytes(type))) return ctx->fail(ZK_ERR_INVALID, "experts: a pointer is not aligned to its type");
  return ZK_OK;
}

static int check_words(zk_context* ctx, const void* p, bool may_be_null) {
  if (!p && !may_be_null) return ctx->fail(ZK_ERR_INVALID, "experts: null pointer");
  if (!aligned(p, 4)) return ctx->fail(ZK_ERR_INVALID, "experts: a pointer is not aligned to its type");
  return ZK_OK;
}

}  // namespace zk

extern "C" {

size_t zk_experts_sort_work(size_t pairs, int experts) {
  using namespace zk;
  if (experts < 1 || experts > ZK_MAX_EXPERTS || pairs > ZK_MAX_EXPERT_ROWS) return 0;
  const SortPlan p = sort_plan(pairs);
  return p.blocks > 1 ? (size_t)p.blocks * experts * 4 : 0;
}

int zk_experts_sort(zk_context* ctx, const int32_t* d_expert, size_t pairs, int experts, int32_t* d_offsets,
                    int32_t* d_order, int32_t* d_place, void* d_work, size_t work_bytes, void* stream) {
  using namespace zk;
  if (!ctx) return ZK_ERR_INVALID;
  return guard(ctx, [&]() -> int {
    ZK_TRY(check_experts(ctx, pairs, experts));
    ZK_TRY(check_words(ctx, d_offsets, false));
    ZK_TRY(check_words(ctx, d_expert, !pairs));
    ZK_TRY(check_words(ctx, d_order, !pairs));
    ZK_TRY(check_words(ctx, d_place, !pairs));
    const size_t need = zk_experts_sort_work(pairs, experts);
    if (need && (!d_work || !aligned(d_work, 4) || work_bytes < need))
      return ctx->fail(ZK_ERR_INVALID, "experts: workspace missing, too small or not aligned to 4 bytes");
    const SortPlan p = sort_plan(pairs);
    hipStream_t st = ctx->s(stream);
    uint32_t* tot = p.blocks > 1 ? (uint32_t*)d_work : nullptr;
    if (tot)
      ZK_LAUNCH(ctx, st, "experts_sort", k_sort_count, dim3(p.blocks), dim3(SORT_THREADS), 0, d_expert,
                (uint32_t)pairs, (uint32_t)experts, p.segment, tot);
    ZK_LAUNCH(ctx, st, "experts_sort", k_sort_place, dim3(p.blocks), dim3(SORT_THREADS), 0, d_expert,
              (uint32_t)pairs, (uint32_t)experts, p.segment, tot, d_offsets, d_order, d_place);
    return ZK_OK;
  });
}

int zk_experts_gather(zk_context* ctx, const void* d_x, int type, size_t ld_x, size_t cols, const int32_t* d_order,
                      size_t rows, size_t tokens, int slots, void* d_out, size_t ld_out, void* stream) {
  using namespace zk;
  if (!ctx) return ZK_ERR_INVALID;
  return guard(ctx, [&]() -> int {
    ZK_TRY(check_rows(ctx, type, rows, tokens, slots, cols));
    if (!rows || !cols) return ZK_OK;
    ZK_TRY(check_words(ctx, d_order, false));
    if (tokens) ZK_TRY(check_matrix(ctx, d_x, type, ld_x, cols));
    ZK_TRY(check_matrix(ctx, d_out, type, ld_out, cols));
    hipStream_t st = ctx->s(stream);
    return by_type(type, [&](auto zero) -> int {
      typedef decltype(zero) T;
      const uint32_t log_w = log_threads<T>(cols);
      const dim3 grid(cdiv(rows, 256u >> log_w));
      auto go = [&](auto kernel) -> int {
        ZK_LAUNCH(ctx, st, "experts_gather", kernel, grid, dim3(256), 0, (const T*)d_x, ld_x, d_order, (uint32_t)rows,
                  (uint32_t)tokens, (uint32_t)slots, (uint32_t)cols, log_w, (T*)d_out, ld_out);
        return ZK_OK;
      };
      return streams(rows, cols, sizeof(T)) ? go(k_gather<T, true>) : go(k_gather<T, false>);
    });
  });
}

int zk_experts_combine(zk_context* ctx, const void* d_y, int type, size_t ld_y, size_t cols, const int32_t* d_place,
                       const float* d_weight, size_t rows, size_t tokens, int slots, void* d_out, size_t ld_out,
                       void* stream) {
  using namespace zk;
  if (!ctx) return ZK_ERR_INVALID;
  return guard(ctx, [&]() -> int {
    ZK_TRY(check_rows(ctx, type, rows, tokens, slots, cols));
    if (!tokens || !cols) return ZK_OK;
    ZK_TRY(check_words(ctx, d_place, false));
    ZK_TRY(check_words(ctx, d_weight, true));
    if (rows) ZK_TRY(check_matrix(ctx, d_y, type, ld_y, cols));
    ZK_TRY(check_matrix(ctx, d_out, type, ld_out, cols));
    hipStream_t st = ctx->s(stream);
    return by_type(type, [&](auto zero) -> int {
      typedef decltype(zero) T;
      const uint32_t log_w = log_threads<T>(cols);
      const dim3 grid(cdiv(tokens, 256u >> log_w));
      auto go = [&](auto kernel) -> int {
        ZK_LAUNCH(ctx, st, "experts_combine", kernel, grid, dim3(256), 0, (const T*)d_y, ld_y, d_place, d_weight,
                  (uint32_t)rows, (uint32_t)tokens, (uint32_t)slots, (uint32_t)cols, log_w, (T*)d_out, ld_out);
        return ZK_OK;
      };
      return streams(rows, cols, sizeof(T)) ? go(k_combine<T, true>) : go(k_combine<T, false>);
    });
  });
}

int zk_experts_combine_grad(zk_context* ctx, const void* d_grad, size_t ld_grad, const void* d_y, size_t ld_y,
                            int type, size_t cols, const int32_t* d_order, const int32_t* d_place,
                            const float* d_weight, size_t rows, size_t tokens, int slots, void* d_grad_y,
                            size_t ld_grad_y, float* d_grad_weight, void* stream) {
  using namespace zk;
  if (!ctx) return ZK_ERR_INVALID;
  return guard(ctx, [&]() -> int {
    ZK_TRY(check_rows(ctx, type, rows, tokens, slots, cols));
    if (rows > tokens * (size_t)slots)
      return ctx->fail(ZK_ERR_INVALID, "experts: more rows than the tokens have pairs");
    if (!tokens) return ZK_OK;
    ZK_TRY(check_words(ctx, d_place, false));
    ZK_TRY(check_words(ctx, d_order, !rows));
    ZK_TRY(check_words(ctx, d_weight, true));
    ZK_TRY(check_words(ctx, d_grad_weight, true));
    if (cols) {
      ZK_TRY(check_matrix(ctx, d_grad, type, ld_grad, cols));
      if (rows) ZK_TRY(check_matrix(ctx, d_grad_y, type, ld_grad_y, cols));
      if (rows && d_grad_weight) ZK_TRY(check_matrix(ctx, d_y, type, ld_y, cols));
    }
    hipStream_t st = ctx->s(stream);
    return by_type(type, [&](auto zero) -> int {
      typedef decltype(zero) T;
      auto go = [&](auto kernel) -> int {
        ZK_LAUNCH(ctx, st, "experts_combine_grad", kernel, dim3((uint32_t)tokens), dim3(256), 0, (const T*)d_grad,
                  ld_grad, (const T*)d_y, ld_y, d_order, d_place, d_weight, (uint32_t)rows, (uint32_t)slots,
                  (uint32_t)cols, (T*)d_grad_y, ld_grad_y, d_grad_weight);
        return ZK_OK;
      };
      return streams(rows, cols, sizeof(T)) ? go(k_combine_grad<T, true>) : go(k_combine_grad<T, false>);
    });
  });
}

}  // extern "C"
