// What the products of 8-bit rows share: their arguments, the tile of a block
// (dense, and grouped by expert), copies from memory straight to LDS, the stores
// of neighbouring results, and the rows' quantizer.
#pragma once
#include "rows.hpp"
#include "zk_internal.hpp"

namespace zk {

typedef int v4i __attribute__((ext_vector_type(4)));
typedef int v16i __attribute__((ext_vector_type(16)));

constexpr size_t I8_MAX_TILES = (size_t)1 << 22;  // blocks of one launch (its threads stay below 2^32)

// What a product's kernel is given.
struct I8Args {
  const int8_t* x;
  const int8_t* w;
  const float* sx;  // per token, or null: 1
  const float* sw;  // per channel, or null: 1
  const float* bias;
  void* y;
  size_t ld_x, ld_w, ld_y;
  uint32_t rows, n_out, n_in;
  int relu;
  // grouped form
  const int32_t* offsets;
  const int32_t* order;
  uint32_t experts, slots, tokens;
};

// Four neighbouring results, of which the row has `left` from here on.  (Every
// index is a constant: an array that is indexed by a variable goes to LDS, by way
// of the launch packet in host memory, and a call of 5 us then took 16.)
// ONCE: around the caches.
template <bool ONCE = false, class T>
__device__ __forceinline__ void store4(T* y, uint32_t left, const T (&v)[4]) {
  if (left >= 4) {
    if constexpr (ONCE) {
      row16 b;
      static_assert(sizeof(v) == 16, "whole pieces of 16 bytes");
      __builtin_memcpy(&b, v, 16);
      __builtin_nontemporal_store(b, (row16*)y);
    } else {
      __builtin_memcpy(y, v, sizeof(v));
    }
    return;
  }
#pragma unroll
  for (uint32_t k = 0; k < 3; k++)
    if (k < left) y[k] = v[k];
}

// Offset of expert e, inside [0, rows] whatever the device array holds.
__device__ __forceinline__ uint32_t offset_of(const I8Args& a, uint32_t e) {
  const int v = a.offsets[e];
  return v < 0 ? 0u : (uint32_t)v > a.rows ? a.rows : (uint32_t)v;
}

// Row of x behind position p (grouped form), or -1: the position holds none.
__device__ __forceinline__ int64_t source_row(const I8Args& a, uint32_t p) {
  if (!a.order) return p < a.tokens ? (int64_t)p : -1;
  const int o = a.order[p];
  if (o < 0) return -1;
  const uint32_t t = (uint32_t)o / a.slots;
  return t < a.tokens ? (int64_t)t : -1;
}

// Tile (tt, tn) of block b.  Blocks b, b + 8, b + 16, ... share an XCD and its
// L2: each XCD gets one run of the tiles, and a run goes over 8 token tiles
// before it takes the next channel tile, so that the 32 blocks an XCD holds at
// a time read about 8 + 4 tiles of rows between them.
__device__ __forceinline__ bool tile_of_block(uint32_t b, uint32_t tiles_t, uint32_t tiles_n, uint32_t& tt,
                                              uint32_t& tn) {
  constexpr uint32_t G = 8;
  const uint32_t total = tiles_t * tiles_n, per = (total + 7) / 8;
  const uint32_t t = (b & 7) * per + (b >> 3);
  if ((b >> 3) >= per || t >= total) return false;
  const uint32_t group = t / (G * tiles_n), at = t % (G * tiles_n);
  const uint32_t size = tiles_t - group * G < G ? tiles_t - group * G : G;
  tt = group * G + at % size;
  tn = at / size;
  return true;
}

// A block's tile: rows [r0, r1) from channel n0 on, and their expert.  Grouped,
// the row tiles are counted expert by expert, those of the rows without an
// expert (e = experts) last; the grid is made for the most there can be, and the
// tiles there are are spread over its first blocks, so that no XCD is left with
// the empty ones.  The whole wave takes part; the answer is the same in every
// lane.  False: nothing to do.
template <bool GROUPED>
__device__ __forceinline__ bool block_tile(const I8Args& a, uint32_t bt, uint32_t bn, uint32_t tiles_t,
                                           uint32_t tiles_n, uint32_t& r0, uint32_t& r1, uint32_t& n0, uint32_t& e) {
  uint32_t tt, tn;
  if (!GROUPED) {
    if (!tile_of_block(blockIdx.x, tiles_t, tiles_n, tt, tn)) return false;
    r0 = tt * bt, r1 = a.rows, n0 = tn * bn, e = 0;
    return true;
  }
  const uint32_t lane = threadIdx.x & 63;
  // 64 experts at a time, one a lane: rows [lo, hi), n tiles, s of them up to here
  uint32_t lo, hi, n, s;
  auto look = [&](uint32_t e0) {
    const uint32_t me = e0 + lane;
    lo = hi = 0;
    if (me < a.experts) lo = offset_of(a, me), hi = offset_of(a, me + 1);
    n = hi > lo ? (hi - lo + bt - 1) / bt : 0;
    s = n;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const uint32_t o = __shfl_up(s, d);
      if (lane >= (uint32_t)d) s += o;
    }
  };
  uint32_t all = 0;
  for (uint32_t e0 = 64; e0 < a.experts; e0 += 64) look(e0), all += __shfl(s, 63);
  look(0);
  all += __shfl(s, 63);
  const uint32_t end = offset_of(a, a.experts), rest = (a.rows - end + bt - 1) / bt;
  if (!tile_of_block(blockIdx.x, __builtin_amdgcn_readfirstlane(all + rest), tiles_n, tt, tn)) return false;
  n0 = tn * bn;
  uint32_t run = 0;
  for (uint32_t e0 = 0; e0 < a.experts; e0 += 64) {
    if (e0) look(e0);
    const uint64_t past = __ballot(run + s > tt);
    if (past) {
      const int l = __ffsll((unsigned long long)past) - 1;
      const uint32_t first = run + __shfl(s, l) - __shfl(n, l);
      e = __builtin_amdgcn_readfirstlane(e0 + l);
      r0 = __builtin_amdgcn_readfirstlane(__shfl(lo, l) + (tt - first) * bt);
      r1 = __builtin_amdgcn_readfirstlane(__shfl(hi, l));
      return r0 < r1;
    }
    run += __shfl(s, 63);
  }
  e = a.experts;
  r0 = __builtin_amdgcn_readfirstlane(end + (tt - run) * bt);
  r1 = a.rows;
  return r0 < r1;
}

// What rows are padded with: a lane that has no bytes to load takes these.
__device__ const v4i zeros16 = {0, 0, 0, 0};

// ------------------------------------------------------------ memory to LDS
// 16 bytes a lane from `p` to LDS at `at` + 16 * lane (`at` the same in the
// whole wave).  Only wait_loads() waits for it: to the compiler's own counting
// it is unknown, which makes the compiler's waits longer, never shorter.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"  // m0 is named so that nothing of the compiler's is kept in it
__device__ __forceinline__ void load_to_lds(const int8_t* p, uint32_t at) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(at), "v"(p) : "m0");
}
// The same from `p` + off, p the same in the whole wave: one register for an address.
__device__ __forceinline__ void load_to_lds(const int8_t* p, uint32_t off, uint32_t at) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(at), "v"(off), "s"(p) : "m0");
}
#pragma clang diagnostic pop
// Until at most N of the wave's loads are under way.
template <int N>
__device__ __forceinline__ void wait_loads() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
__device__ __forceinline__ void wait_lds() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }
__device__ __forceinline__ void meet() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// ------------------------------------------------------------ rows to 8 bits
// s = a / 127, q = rint(t / a) with a = max|x| and t = 127 x, rounded to 32 bits
// (f16 and bf16: exact).  The quotient is the correctly rounded one: t times the
// rounded reciprocal of a, and one step of Newton's method on the remainder, which
// two fused operations give exactly (Markstein's division; about 10 operations a
// value, where the compiler's takes 25: 2048 rows of 4096 7.9 us instead of 10.0 in
// turn).  So q is what the elementary operations give, and for 16-bit values, whose
// quotients beside a half are further from it than the rounding, the integer nearest
// to the exact quotient.  An f32 quotient within 2^-16 of a half may go to either
// side: an exact decision would need the remainders of both roundings, and would
// part from the elementary operations.  Rows far from 1 are first multiplied by
// a power of two, so that nothing leaves the normal numbers.  A row of zeros
// gives s = 0 and zeros; a row with an infinity or a NaN gives s = NaN and zeros,
// so that its products show it.
struct RowScale {
  float s;      // the row's scale
  float c, a;   // t = x c, c = 127 times a power of two; a with the same power
  float inv;    // 1 / a; 0: all zeros
};

// From the largest magnitude's bits (as integers magnitudes are in the floats'
// order, NaN above infinity).
__device__ __forceinline__ RowScale row_scale(uint32_t m) {
  const float a = __uint_as_float(m);
  RowScale r = {a / 127.0f, 0.0f, 1.0f, 0.0f};
  if (m >= 0x7f800000u) {
    r.s = __uint_as_float(0x7fc00000u);
  } else if (m) {
    const float c = a >= 0x1p64f ? 0x1p-32f : a < 0x1p-64f ? 0x1p64f : 1.0f;
    r.c = 127.0f * c;
    r.a = a * c;
    r.inv = 1.0f / r.a;
  }
  return r;
}

template <class T>
__device__ __forceinline__ uint32_t magnitude(T x) {
  return __float_as_uint((float)x) & 0x7fffffffu;
}

template <class T>
__device__ __forceinline__ void quantize_piece(const Vec<T>& x, const RowScale& r, int8_t* q) {
  if (r.inv == 0.0f) {  // where x itself may be an infinity or a NaN
#pragma unroll
    for (uint32_t i = 0; i < Vec<T>::N; i++) q[i] = 0;
    return;
  }
#pragma unroll
  for (uint32_t i = 0; i < Vec<T>::N; i++) {
    const float t = (float)x.v[i] * r.c, y = t * r.inv;
    q[i] = (int8_t)rintf(fmaf(fmaf(-y, r.a, t), r.inv, y));
  }
}

template <class T>
__device__ __forceinline__ void look_piece(const Vec<T>& v, uint32_t& m) {
#pragma unroll
  for (uint32_t i = 0; i < Vec<T>::N; i++) {
    const uint32_t u = magnitude(v.v[i]);
    m = u > m ? u : m;
  }
}

// ---- a few rows at a time
constexpr uint32_t FEW_ROWS = 16, FEW_BYTES = 36 * 1024;
// A quantized row's stride in LDS: whole steps, and 16 bytes so that the rows of
// a fragment lie in different banks.
static __host__ __device__ inline uint32_t few_ld(uint32_t n_in) { return (n_in + 127) / 128 * 128 + 16; }

// A block's KW waves quantize a few rows into LDS (FEW_ROWS at the most, at stride ld),
// KW / g rows at a time, g waves a row; part is scratch.  All meet at the end.
template <class X, uint32_t KW>
__device__ __forceinline__ void quantize_rows(const X* __restrict__ x, size_t ld_x, uint32_t rows, uint32_t n_in,
                                              int8_t* q, uint32_t ld, uint32_t (&part)[FEW_ROWS][KW],
                                              float (&scale)[FEW_ROWS]) {
  constexpr int HELD = 4;
  const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  uint32_t g = KW;
  while (g > 1 && KW / g < rows) g /= 2;
  const uint32_t at_once = KW / g, first = wave / g, sub = (wave % g) * 64 + lane;
  const uint32_t pieces = pieces_of<X>(n_in);
  Vec<X> held[HELD];
  for (uint32_t r = first; r < rows; r += at_once) {
    const X* row = x + (size_t)r * ld_x;
    uint32_t m = 0;
#pragma unroll
    for (int h = 0; h < HELD; h++) {
      const uint32_t p = sub + h * g * 64;
      held[h] = Vec<X>{};
      if (p < pieces) held[h] = row_load(row + piece<X>(p, n_in), n_in - piece<X>(p, n_in));
    }
#pragma unroll
    for (int h = 0; h < HELD; h++) look_piece(held[h], m);
    for (uint32_t p = sub + HELD * g * 64; p < pieces; p += g * 64)
      look_piece(row_load(row + piece<X>(p, n_in), n_in - piece<X>(p, n_in)), m);
#pragma unroll
    for (int d = 32; d; d >>= 1) {
      const uint32_t o = (uint32_t)__shfl_xor((int)m, d);
      m = o > m ? o : m;
    }
    if (lane == 0) part[r][wave % g] = m;
  }
  wait_lds();
  meet();
  for (uint32_t r = first; r < rows; r += at_once) {
    const X* row = x + (size_t)r * ld_x;
    int8_t* out = q + r * ld;
    uint32_t m = 0;
    for (uint32_t i = 0; i < g; i++) m = part[r][i] > m ? part[r][i] : m;
    const RowScale rs = row_scale(m);
    if (sub == 0) scale[r] = rs.s;
    auto put = [&](uint32_t p, const Vec<X>& v) {
      const uint32_t at = piece<X>(p, n_in);
      int8_t b[Vec<X>::N];
      quantize_piece(v, rs, b);
      if (n_in - at >= Vec<X>::N) {
        __builtin_memcpy(out + at, b, sizeof(b));
      } else {
#pragma unroll
        for (uint32_t i = 0; i < Vec<X>::N; i++)
          if (i < n_in - at) out[at + i] = b[i];
      }
    };
    const bool again = at_once < rows;  // held is the last of several rows
    if (!again) {
#pragma unroll
      for (int h = 0; h < HELD; h++)
        if (sub + h * g * 64 < pieces) put(sub + h * g * 64, held[h]);
    }
    for (uint32_t p = sub + (again ? 0 : HELD * g * 64); p < pieces; p += g * 64)
      put(p, row_load(row + piece<X>(p, n_in), n_in - piece<X>(p, n_in)));
  }
  wait_lds();
  meet();
}

// ---- rows to 8 bits (i8_matmul.hip)
int i8_quantize(zk_context* ctx, const void* x, int type, size_t ld_x, size_t rows, size_t cols, int8_t* q,
                size_t ld_q, float* scale, hipStream_t st);
int check_quantize(zk_context* ctx, const void* x, int type, size_t ld_x, size_t rows, size_t cols);
// Layout of a quantizing layer's workspace: the rows' scales, then the rows' bytes.
struct LinearWork {
  size_t ld, q, bytes;
};
LinearWork linear_work(size_t rows, size_t n_in);

}  // namespace zk
