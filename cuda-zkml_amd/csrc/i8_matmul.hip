// 8-bit integer layers for gfx950: the linear layer a quantized model's
// statement proves (weights out x in, row major), over whole batches on the
// matrix cores, with the scales that tie its integers to the real-valued model.
//
//   acc[t,n] = sum_k x[t,k] w[n,k]                 int32, exact
//   y[t,n]   = act((float(acc) sx[t]) sw[n] + b[n])  or acc itself
//
// A product of two int8 is at most 2^14, so acc is exact for n_in <= 131071.
// The grouped form takes its weights by expert: rows offsets[e] to
// offsets[e+1] of y use w[e].
#include <type_traits>

#include "i8_product.hpp"

namespace zk {

constexpr size_t I8_MAX_IN = 131071;

// Where a lane takes the 16 bytes of k from byte k on, for rows of n_in >= 16
// bytes: a chunk that passes the rows' end is the last 16 bytes of both x's and
// w's rows, with the bytes before k masked off x.  The same order of k on both
// sides is all that a sum needs, and no byte outside a row is read.
struct Chunk {
  uint32_t at;
  v4i mask;
};
__device__ __forceinline__ Chunk last_chunk(uint32_t k, uint32_t n_in) {
  Chunk c;
  c.at = k < n_in - 16 ? k : n_in - 16;
  const uint32_t skip = k - c.at;
#pragma unroll
  for (uint32_t d = 0; d < 4; d++)
    c.mask[d] = skip <= 4 * d ? -1 : skip >= 4 * d + 4 ? 0 : (int)(~0u << (8 * (skip - 4 * d)));
  return c;
}
// 16 bytes from any address: at full rate from whole words, at a third of it
// from others.
__device__ __forceinline__ v4i load16_any(const int8_t* p) {
  v4i v;
  __builtin_memcpy(&v, p, 16);
  return v;
}
// 16 bytes from a multiple of 4 bytes, or, BYTES, from any address as the words
// that hold them, moved down by the address's part of a word (3 rows, 5569 to
// 7061, in turn: 11 us, 19 with load16_any).  No word is read that holds none of the bytes.
typedef int v4i_words __attribute__((ext_vector_type(4), aligned(4)));
__device__ __forceinline__ v4i move_down(const v4i& v, int next, uint32_t by) {
  return v4i{(int)__builtin_amdgcn_alignbyte((uint32_t)v[1], (uint32_t)v[0], by),
             (int)__builtin_amdgcn_alignbyte((uint32_t)v[2], (uint32_t)v[1], by),
             (int)__builtin_amdgcn_alignbyte((uint32_t)v[3], (uint32_t)v[2], by),
             (int)__builtin_amdgcn_alignbyte((uint32_t)next, (uint32_t)v[3], by)};
}
template <bool BYTES>
__device__ __forceinline__ v4i load16(const int8_t* p) {
  if (!BYTES) return *(const v4i_words*)p;
  const uint32_t by = (uint32_t)(uintptr_t)p & 3u;
  const int8_t* q = p - by;
  const v4i v = *(const v4i_words*)q;
  return move_down(v, *(const int*)(q + (by ? 16 : 12)), by);
}
// The last 16 bytes of a row of any length.
template <bool BYTES>
__device__ __forceinline__ v4i load16_end(const int8_t* p) {
  return BYTES ? load16<true>(p) : load16_any(p);
}
// Lane c's 32 of a step's 128 bytes, the same ones on both sides of a product:
// bytes 16 c on of each half, or, BYTES, 32 c on, so that the second 16 bytes'
// first word is the first ones' next.
template <bool BYTES>
__device__ __forceinline__ void load_pair(const int8_t* p, uint32_t c, v4i (&out)[2]) {
  if (!BYTES) {
    out[0] = load16<false>(p + c * 16);
    out[1] = load16<false>(p + c * 16 + 64);
  } else {
    const uint32_t by = (uint32_t)(uintptr_t)p & 3u;
    const int8_t* q = p + c * 32 - by;
    out[0] = load16<false>(q);
    out[1] = load16<false>(q + 16);
    const int next = *(const int*)(q + (by ? 32 : 28));
    out[0] = move_down(out[0], out[1][0], by);
    out[1] = move_down(out[1], next, by);
  }
}
// A token's scale as the results take it: s * up, where up is a power of two that
// keeps a sum below 2^31 times s inside the 32-bit floats (row maxima from 10^31 on
// have such scales, and a channel's scale may bring them back).
struct TokenScale {
  float s, up;
};
__device__ __forceinline__ TokenScale token_scale(float sx) {
  const bool big = fabsf(sx) >= 0x1p96f;
  return TokenScale{big ? sx * 0x1p-32f : sx, big ? 0x1p32f : 1.0f};
}
// (float(acc) sx) sw + b, each operation rounded to 32 bits, so that the result is
// what the elementary operations in this order give bit for bit; times up is exact,
// and so the fused operation rounds once, as the sum alone does.  (sx sw first could
// leave the 32-bit floats where the result does not.)
template <class T>
__device__ __forceinline__ T finish(int acc, const TokenScale& x, float sw, float b, int relu) {
  float f = fmaf((float)acc * x.s * sw, x.up, b);
  // (else the compiler takes an instruction that rounds the f16 from the exact sum)
  if constexpr (std::is_same<T, _Float16>::value) asm("" : "+v"(f));
  if (relu && f < 0.0f) f = 0.0f;  // a NaN stays
  return (T)f;
}
template <>
__device__ __forceinline__ int finish<int>(int acc, const TokenScale&, float, float, int relu) {
  return relu && acc < 0 ? 0 : acc;
}

// ------------------------------------------------------------ tiles in LDS
// A block computes BT tokens x BN channels, its WT x WN waves a grid of
// FT x FN squares of 32 x 32 each (D rows are channels, so that a lane holds
// four neighbouring channels of one token).  Steps of 128 bytes of k, a whole
// cache line of each row, pass through LDS: byte chunk c of row r lies at chunk
// c ^ (r / 2 % 8), so that the 32 rows of a fragment meet no bank twice (the
// conflict counter does not grow with n_in: what it counts are the results).
//
// Rows of whole 16-byte chunks go straight from memory to LDS, with no register
// and no instruction between, into a ring of five slots of one side's tile each:
// this step's two tiles, the next step's two, and x's of the one after, each slot
// asked for again half a step after everybody has read it.  Loads and LDS reads
// are placed between the matrix instructions, which then have no pause longer
// than a barrier.  8192 x 8192 x 8192: 457 us a call, 2.40 POPS (traced, median of
// sixty in a row 479, 457 to 591); 309 with zeros for data.  The matrix cores are
// busy in 0.67 to 0.73 of the cycles with either data (a tile's first loads and
// results take 0.07 by the fit below, waits within the steps the rest); the clock
// makes the difference, 2.1 to 2.2 GHz on zeros and 1.3 to 1.7 with random data,
// where the card's power limits it.  2048 rows, 4096 to 4096: 40.4 us, 1.70 POPS
// (512 tiles, two for each CU).

// ---- what a tile's sums become
// The tile's scales and biases: a thread holds a few of them from the start,
// so that they are there when the sums are, and puts them into LDS after the
// last step: sx[BT], sw[BN], bias[BN] and, in the grouped form, has[BT] (does
// the row have a token?).
template <bool GROUPED, uint32_t BT, uint32_t BN, uint32_t THREADS>
struct Factors {
  static constexpr uint32_t ALL = BT + 2 * BN + (GROUPED ? BT : 0), N = (ALL + THREADS - 1) / THREADS;
  float v[N];
  __device__ __forceinline__ void load(const I8Args& a, uint32_t r0, uint32_t r1, uint32_t n0, uint32_t e) {
    const bool none = GROUPED && e >= a.experts;
    const size_t ch = none ? 0 : (size_t)e * a.n_out;
#pragma unroll
    for (uint32_t i = 0; i < N; i++) {
      const uint32_t k = threadIdx.x + i * THREADS;
      v[i] = 0.0f;
      if (k < BT || k >= BT + 2 * BN) {
        const uint32_t t = r0 + (k < BT ? k : k - BT - 2 * BN);
        int64_t s = -1;
        if (t < r1 && !none) s = GROUPED ? source_row(a, t) : (int64_t)t;
        v[i] = s < 0 ? 0.0f : k < BT && a.sx ? a.sx[s] : 1.0f;
      } else {
        const bool second = k >= BT + BN;
        const uint32_t n = n0 + k - BT - (second ? BN : 0);
        const float* from = second ? a.bias : a.sw;
        v[i] = from ? (n < a.n_out ? from[ch + n] : 0.0f) : second ? 0.0f : 1.0f;
      }
    }
  }
  __device__ __forceinline__ void store(float* to) const {
#pragma unroll
    for (uint32_t i = 0; i < N; i++) {
      const uint32_t k = threadIdx.x + i * THREADS;
      if (k < ALL) to[k] = v[i];
    }
  }
};

// Writes a wave's FN x FT squares: through LDS of its own, 32 tokens at a time,
// so that a row's results leave in 16-byte pieces side by side (8-byte pieces
// of 32 rows at once took 12 us for a tile of 256 x 256).
// f: the block's factors; t0, c0: the wave's first token and channel in the tile.
template <class T, bool GROUPED, uint32_t BT, uint32_t BN, int FT, int FN>
__device__ __forceinline__ void put_results(const I8Args& a, const v16i (&acc)[FN][FT], const float* f, int8_t* own,
                                            uint32_t r0, uint32_t r1, uint32_t n0, uint32_t t0, uint32_t c0) {
  constexpr uint32_t E = 16 / sizeof(T), PIECES = FN * 32 / E, ROWS = 64 / PIECES;  // of one 16-byte store
  constexpr uint32_t LD = FN * 32 * sizeof(T) + 16;
  const uint32_t lane = threadIdx.x & 63, fr = lane & 31, hi = lane >> 5;
  const float *sw = f + BT + c0, *bias = sw + BN, *has = f + BT + 2 * BN;
#pragma unroll
  for (int j = 0; j < FT; j++) {
    const TokenScale sx = token_scale(f[t0 + j * 32 + fr]);
    const bool zero = GROUPED && has[t0 + j * 32 + fr] == 0.0f;
#pragma unroll
    for (int i = 0; i < FN; i++)
#pragma unroll
      for (int q = 0; q < 4; q++) {
        T v[4];
#pragma unroll
        for (int k = 0; k < 4; k++) {
          const uint32_t c = i * 32 + 8 * q + 4 * hi + k;
          v[k] = zero ? (T)0 : finish<T>(acc[i][j][4 * q + k], sx, sw[c], bias[c], a.relu);
        }
        __builtin_memcpy(own + fr * LD + (i * 32 + 8 * q + 4 * hi) * sizeof(T), v, sizeof(v));
      }
    wait_lds();  // one wave's LDS accesses are in order; this keeps the compiler to it
#pragma unroll
    for (uint32_t s = 0; s < 32; s += ROWS) {
      const uint32_t row = s + lane / PIECES, c = lane % PIECES * E;
      const uint32_t t = r0 + t0 + j * 32 + row, n = n0 + c0 + c;
      if (t < r1 && n < a.n_out) {
        const int8_t* from = own + row * LD + c * sizeof(T);
        T* y = (T*)a.y + (size_t)t * a.ld_y + n;
        if (n + E <= a.n_out) {
          v4i v = *(const v4i*)from;
          __builtin_memcpy(y, &v, 16);
        } else {
          for (uint32_t k = 0; k < a.n_out - n; k++) y[k] = ((const T*)from)[k];
        }
      }
    }
    wait_lds();
  }
}

template <class T, bool GROUPED, int WT, int WN, int FT, int FN>
__global__ __launch_bounds__(64 * WT * WN) void k_i8_ring(I8Args a, uint32_t tiles_t, uint32_t tiles_n) {
  constexpr uint32_t WAVES = WT * WN, BT = WT * FT * 32, BN = WN * FN * 32, BK = 128;
  static_assert(BT == BN, "the ring's slots hold either side's tile");
  constexpr uint32_t SLOT = BT * BK, PER = BT / 8 / WAVES;  // 8-row pieces of 1 KB that a wave fills
  constexpr int FIRST = (PER + 1) / 2;  // of a tile's pieces, those that the first of two quarter steps fills
  constexpr uint32_t OWN = 32 * (FN * 32 * sizeof(T) + 16);  // a wave's part of LDS for its results
  static_assert(WAVES * OWN + 4 * (2 * BT + 2 * BN) <= 5 * SLOT, "the results' LDS is the ring's");
  __shared__ __align__(16) int8_t lds[5 * SLOT];
  auto swz = [](uint32_t row) { return (row >> 1) & 7u; };
  const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  uint32_t r0, r1, n0, e;
  if (!block_tile<GROUPED>(a, BT, BN, tiles_t, tiles_n, r0, r1, n0, e)) return;
  const bool none = GROUPED && e >= a.experts;
  const int8_t* w = a.w + (none ? 0 : (size_t)e * a.n_out * a.ld_w);
  const int8_t *xp[PER], *wp[PER];
  auto chunk = [&](uint32_t piece) { return ((lane & 7) ^ swz(piece * 8 + (lane >> 3))) * 16; };
#pragma unroll
  for (uint32_t i = 0; i < PER; i++) {
    const uint32_t row = (wave * PER + i) * 8 + (lane >> 3);
    const uint32_t n = n0 + row < a.n_out ? n0 + row : a.n_out - 1;
    wp[i] = w + (size_t)n * a.ld_w + chunk(wave * PER + i);
  }
  const uint32_t base = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) int8_t*)lds + wave * PER * 1024;
  const uint32_t full = none ? 0 : a.n_in / BK, tail = none ? 0 : a.n_in % BK;
  const uint32_t steps = full + (tail ? 1 : 0);
  // piece i of one side's tile of `step` into ring slot `slot`
  auto fill = [&](const int8_t*& p, uint32_t i, uint32_t step, uint32_t slot) {
    const uint32_t at = base + slot * SLOT + i * 1024;
    if (step < full) load_to_lds(p, at);
    else if (step < steps) load_to_lds(chunk(wave * PER + i) < tail ? p : (const int8_t*)&zeros16, at);
    p += BK;
  };
  const uint32_t wave_t = wave % WT, wave_n = wave / WT;
  const uint32_t fr = lane & 31;
  const int8_t* fx = lds + (wave_t * FT * 32 + fr) * BK;
  const int8_t* fw = lds + (wave_n * FN * 32 + fr) * BK;
  uint32_t ch[4];
#pragma unroll
  for (uint32_t s = 0; s < 4; s++) ch[s] = ((2 * s + (lane >> 5)) ^ swz(fr)) * 16;
  v16i acc[FN][FT] = {};
  v4i wf[2][FN], xf[2][FT];
  auto read = [&](int set, int r, uint32_t xs, uint32_t ws, uint32_t s) {
    if (r < FN) wf[set][r] = *(const v4i*)(fw + ws * SLOT + r * 32 * BK + ch[s]);
    else xf[set][r - FN] = *(const v4i*)(fx + xs * SLOT + (r - FN) * 32 * BK + ch[s]);
  };
  // w's first tiles wait for no index of the rows; the factors' chain of loads
  // runs beside the tiles'
#pragma unroll
  for (uint32_t i = 0; i < PER; i++) fill(wp[i], i, 0, 1);
#pragma unroll
  for (uint32_t i = 0; i < PER; i++) fill(wp[i], i, 1, 3);
#pragma unroll
  for (uint32_t i = 0; i < PER; i++) {
    const uint32_t row = (wave * PER + i) * 8 + (lane >> 3);
    const uint32_t r = r0 + row < r1 ? r0 + row : r1 - 1;
    int64_t s = GROUPED ? source_row(a, r) : (int64_t)r;
    if (s < 0) s = 0;
    xp[i] = a.x + (size_t)s * a.ld_x + chunk(wave * PER + i);
  }
#pragma unroll
  for (uint32_t i = 0; i < PER; i++) fill(xp[i], i, 0, 0);
#pragma unroll
  for (uint32_t i = 0; i < PER; i++) fill(xp[i], i, 1, 2);
#pragma unroll
  for (uint32_t i = 0; i < PER; i++) fill(xp[i], i, 2, 4);
  Factors<GROUPED, BT, BN, 64 * WAVES> factors;
  factors.load(a, r0, r1, n0, e);
  if (steps) {
    if (steps > 2) wait_loads<2 * PER>();
    else wait_loads<0>();
    meet();
    uint32_t xs = 0;  // slot of this step's x
    auto up = [](uint32_t slot, uint32_t by) { return slot + by < 5 ? slot + by : slot + by - 5; };
#pragma unroll
    for (int r = 0; r < FN + FT; r++) read(0, r, 0, 1, 0);
    // One step.  LONG: it is not the first, and all that it fills lies in full steps.
    auto run = [&](auto is_long, uint32_t step) {
      constexpr bool LONG = decltype(is_long)::value;
      constexpr int M = FN * FT, R = FN + FT, SPREAD = M >= 4 ? M * 3 / 4 : M;
      const uint32_t x0 = xs, w0 = up(xs, 1), x1 = up(xs, 2), w1 = up(xs, 3), x2 = up(xs, 4);
      auto put = [&](const int8_t*& p, uint32_t i, uint32_t of, uint32_t slot) {
        if constexpr (LONG) {
          load_to_lds(p, base + slot * SLOT + i * 1024);
          p += BK;
        } else {
          fill(p, i, of, slot);
        }
      };
#pragma unroll
      for (int s = 0; s < 4; s++) {
        if (s == 3) {
          // the next step's tiles are in, and everybody has read this one's
          if (LONG || step + 2 < steps) wait_loads<PER>();
          else wait_loads<0>();
          wait_lds();
          meet();
        }
#pragma unroll
        for (int m = 0; m < M; m++) {
#pragma unroll
          for (int r = m * R / SPREAD; r < (m + 1) * R / SPREAD && r < R; r++) {
            if (s < 3) read((s + 1) & 1, r, x0, w0, s + 1);
            else if (LONG || step + 1 < steps) read(0, r, x1, w1, 0);
          }
          acc[m / FT][m % FT] =
              __builtin_amdgcn_mfma_i32_32x32x32_i8(wf[s & 1][m / FT], xf[s & 1][m % FT], acc[m / FT][m % FT], 0, 0, 0);
          // the tiles of w two steps on and of x three on, as their slots get free
#pragma unroll
          for (int d = 0; d < FIRST; d++)
            if (d * M / FIRST == m) {
              if (s == 3) put(wp[d], d, step + 2, x0);
              if (s == 1 && (LONG || step)) put(xp[d], d, step + 2, x2);
              if (FIRST + d < (int)PER && (LONG || step)) {
                if (s == 0) put(wp[FIRST + d], FIRST + d, step + 1, w1);
                if (s == 2) put(xp[FIRST + d], FIRST + d, step + 2, x2);
              }
            }
          __builtin_amdgcn_sched_barrier(0);
        }
      }
      xs = x1;
    };
    uint32_t step = 0;
    run(std::false_type(), step++);
    for (; step + 2 < full; step++) run(std::true_type(), step);
    for (; step < steps; step++) run(std::false_type(), step);
  }
  // the last step ended with everybody past its reads: the ring is free
  float* f = (float*)(lds + WAVES * OWN);
  factors.store(f);
  wait_lds();
  meet();
  put_results<T, GROUPED, BT, BN, FT, FN>(a, acc, f, lds + wave * OWN, r0, r1, n0, wave_t * FT * 32, wave_n * FN * 32);
}

// The same tiles where a row may start at any byte, or end inside a chunk: the
// steps pass through registers (masked), loaded a step ahead and stored before
// the stage's turn.  Bound by those loads, which take three times as long from
// addresses inside a word: 777 rows, 1001 to 1234, in 10.6 us, 1194 rows, 4438 to
// 5316 f32, in 65.
// (Loads from any address; word loads with the bytes moved down, as the direct
// kernel has them, hold a register more a piece and made the latter 98 us instead
// of 68, in turn.)
template <class T, bool GROUPED, int WT, int WN, int FT, int FN>
__global__ __launch_bounds__(64 * WT * WN) void k_i8_odd(I8Args a, uint32_t tiles_t, uint32_t tiles_n) {
  constexpr uint32_t WAVES = WT * WN, BT = WT * FT * 32, BN = WN * FN * 32, BK = 128;
  constexpr uint32_t XB = BT * BK, STAGE = XB + BN * BK, XR = BT / 8 / WAVES, WR = BN / 8 / WAVES;
  constexpr uint32_t OWN = 32 * (FN * 32 * sizeof(T) + 16);
  static_assert(WAVES * OWN + 4 * (2 * BT + 2 * BN) <= 2 * STAGE, "the results' LDS is the stages'");
  __shared__ __align__(16) int8_t lds[2 * STAGE];
  auto swz = [](uint32_t row) { return (row >> 1) & 7u; };
  const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  uint32_t r0, r1, n0, e;
  if (!block_tile<GROUPED>(a, BT, BN, tiles_t, tiles_n, r0, r1, n0, e)) return;
  const bool none = GROUPED && e >= a.experts;
  const int8_t* w = a.w + (none ? 0 : (size_t)e * a.n_out * a.ld_w);
  Factors<GROUPED, BT, BN, 64 * WAVES> factors;
  factors.load(a, r0, r1, n0, e);
  const int8_t *xp[XR], *wp[WR];
#pragma unroll
  for (uint32_t i = 0; i < XR; i++) {
    const uint32_t row = (wave * XR + i) * 8 + (lane >> 3);
    const uint32_t r = r0 + row < r1 ? r0 + row : r1 - 1;
    int64_t s = GROUPED ? source_row(a, r) : (int64_t)r;
    if (s < 0) s = 0;
    xp[i] = a.x + (size_t)s * a.ld_x;
  }
#pragma unroll
  for (uint32_t i = 0; i < WR; i++) {
    const uint32_t row = (wave * WR + i) * 8 + (lane >> 3);
    const uint32_t n = n0 + row < a.n_out ? n0 + row : a.n_out - 1;
    wp[i] = w + (size_t)n * a.ld_w;
  }
  const uint32_t steps = none ? 0 : (a.n_in + BK - 1) / BK;
  v4i held[XR + WR];
  auto chunk = [&](uint32_t piece) { return ((lane & 7) ^ swz(piece * 8 + (lane >> 3))) * 16; };
  auto take = [&](uint32_t step) {
    if ((step + 1) * BK <= a.n_in) {
#pragma unroll
      for (uint32_t i = 0; i < XR; i++) held[i] = load16_any(xp[i] + step * BK + chunk(wave * XR + i));
#pragma unroll
      for (uint32_t i = 0; i < WR; i++) held[XR + i] = load16_any(wp[i] + step * BK + chunk(wave * WR + i));
    } else {
#pragma unroll
      for (uint32_t i = 0; i < XR; i++) {
        const Chunk c = last_chunk(step * BK + chunk(wave * XR + i), a.n_in);
        held[i] = load16_any(xp[i] + c.at) & c.mask;
      }
#pragma unroll
      for (uint32_t i = 0; i < WR; i++)
        held[XR + i] = load16_any(wp[i] + last_chunk(step * BK + chunk(wave * WR + i), a.n_in).at);
    }
  };
  auto store = [&](uint32_t stage) {
    int8_t* at = lds + stage * STAGE + lane * 16;
#pragma unroll
    for (uint32_t i = 0; i < XR; i++) *(v4i*)(at + (wave * XR + i) * 1024) = held[i];
#pragma unroll
    for (uint32_t i = 0; i < WR; i++) *(v4i*)(at + XB + (wave * WR + i) * 1024) = held[XR + i];
  };
  const uint32_t wave_t = wave % WT, wave_n = wave / WT;
  const uint32_t fr = lane & 31;
  const int8_t* fx = lds + (wave_t * FT * 32 + fr) * BK;
  const int8_t* fw = lds + XB + (wave_n * FN * 32 + fr) * BK;
  uint32_t ch[4];
#pragma unroll
  for (uint32_t s = 0; s < 4; s++) ch[s] = ((2 * s + (lane >> 5)) ^ swz(fr)) * 16;
  v16i acc[FN][FT] = {};
  v4i wf[2][FN], xf[2][FT];
  auto read = [&](int set, uint32_t stage, uint32_t s) {
#pragma unroll
    for (int j = 0; j < FN; j++) wf[set][j] = *(const v4i*)(fw + stage * STAGE + j * 32 * BK + ch[s]);
#pragma unroll
    for (int j = 0; j < FT; j++) xf[set][j] = *(const v4i*)(fx + stage * STAGE + j * 32 * BK + ch[s]);
  };
  if (steps) {
    take(0);
    store(0);
    if (steps > 1) take(1);
    wait_lds();
    meet();
    read(0, 0, 0);
    for (uint32_t step = 0; step < steps; step++) {
      const uint32_t stage = step & 1;
#pragma unroll
      for (uint32_t s = 0; s < 4; s++) {
        if (s < 3) {
          read((s + 1) & 1, stage, s + 1);
        } else {
          // once all have read this stage and filled the next, it may be filled again
          if (step + 1 < steps) store(stage ^ 1);
          wait_lds();
          meet();
          if (step + 2 < steps) take(step + 2);
          if (step + 1 < steps) read(0, stage ^ 1, 0);
        }
#pragma unroll
        for (int i = 0; i < FN; i++)
#pragma unroll
          for (int j = 0; j < FT; j++)
            acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(wf[s & 1][i], xf[s & 1][j], acc[i][j], 0, 0, 0);
      }
    }
  }
  // the last step ended with everybody past its reads: the ring is free
  float* f = (float*)(lds + WAVES * OWN);
  factors.store(f);
  wait_lds();
  meet();
  put_results<T, GROUPED, BT, BN, FT, FN>(a, acc, f, lds + wave * OWN, r0, r1, n0, wave_t * FT * 32, wave_n * FN * 32);
}

// ------------------------------------------------------------ few rows
// Few tokens (decoding), or a small layer: w is read once and a block needs
// little of x, so fragments come straight from global memory.  A block has
// 16 FT tokens x 16 FN channels; its KW waves split k between them in steps of
// 128 bytes (a cache line of every row) and add up their sums in LDS.  Bound by
// what the L2 hands over: 16 (FT + FN) rows a block, 9.3 TB/s over the chip; one
// row by the chain of the launch, a block's loads (all under way together) and
// its sums: one row, 4096 to 4096, in 5.8 us (17 MB; an empty launch takes 2.4), 5
// tokens at two of 16 experts each, 4096 to 2048, in 13.8 (12.6 to 18.3; 64 MB).
template <class T, bool GROUPED, bool BYTES, int FT, int FN, int KW>
__global__ __launch_bounds__(64 * KW, 4) void k_i8_direct(I8Args a, uint32_t tiles_t, uint32_t tiles_n) {
  constexpr uint32_t BT = 16 * FT, BN = 16 * FN, BK = 128;
  constexpr int U = FT + FN <= 2 ? 4 : 2;  // steps whose loads are under way together
  __shared__ __align__(16) v4i sums[KW][FN * FT][64];
  const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  uint32_t r0, r1, n0, e;
  if (!block_tile<GROUPED>(a, BT, BN, tiles_t, tiles_n, r0, r1, n0, e)) return;
  const bool none = GROUPED && e >= a.experts;
  const int8_t* w = a.w + (none ? 0 : (size_t)e * a.n_out * a.ld_w);
  const uint32_t fr = lane & 15, c = lane >> 4;
  const int8_t *xp[FT], *wp[FN];
  int64_t src[FT];
#pragma unroll
  for (int j = 0; j < FT; j++) {
    const uint32_t t = r0 + j * 16 + fr, r = t < r1 ? t : r1 - 1;
    const int64_t s = GROUPED ? source_row(a, r) : (int64_t)r;
    src[j] = none ? -1 : s;
    xp[j] = a.x + (size_t)(s < 0 ? 0 : s) * a.ld_x;
  }
#pragma unroll
  for (int i = 0; i < FN; i++) {
    const uint32_t n = n0 + i * 16 + fr;
    wp[i] = w + (size_t)(n < a.n_out ? n : a.n_out - 1) * a.ld_w;
  }
  v4i acc[FN][FT] = {};
  const uint32_t steps = none ? 0 : (a.n_in + BK - 1) / BK, full = none ? 0 : a.n_in / BK;
  uint32_t step = wave;
  v4i xf[U][FT][2], wf[U][FN][2];
  auto multiply = [&](int u) {
#pragma unroll
    for (int h = 0; h < 2; h++)
#pragma unroll
      for (int i = 0; i < FN; i++)
#pragma unroll
        for (int j = 0; j < FT; j++)
          acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wf[u][i][h], xf[u][j][h], acc[i][j], 0, 0, 0);
  };
  for (; step + (U - 1) * KW < full; step += U * KW) {
#pragma unroll
    for (int u = 0; u < U; u++) {
      const uint32_t k = (step + u * KW) * BK;
#pragma unroll
      for (int i = 0; i < FN; i++) load_pair<BYTES>(wp[i] + k, c, wf[u][i]);
#pragma unroll
      for (int j = 0; j < FT; j++) load_pair<BYTES>(xp[j] + k, c, xf[u][j]);
    }
#pragma unroll
    for (int u = 0; u < U; u++) multiply(u);
  }
  // the rest, all loads together again
  if (step < steps) {
#pragma unroll
    for (int u = 0; u < U; u++) {
      if (step + u * KW >= steps) break;
      const uint32_t k = (step + u * KW) * BK + c * 32;
#pragma unroll
      for (int h = 0; h < 2; h++) {
        const Chunk part = last_chunk(k + 16 * h, a.n_in);
#pragma unroll
        for (int i = 0; i < FN; i++) wf[u][i][h] = load16_end<BYTES>(wp[i] + part.at);
#pragma unroll
        for (int j = 0; j < FT; j++) xf[u][j][h] = load16_end<BYTES>(xp[j] + part.at) & part.mask;
      }
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
      if (step + u * KW >= steps) break;
      multiply(u);
    }
  }
  // ---- results: lane r + 16 q holds channels 4 q to 4 q + 3 of token r
  auto put = [&](int i, int j, const v4i& sum) {
    const uint32_t t = r0 + j * 16 + fr, n = n0 + i * 16 + 4 * c;
    if (t >= r1 || n >= a.n_out) return;
    const bool zero = GROUPED && src[j] < 0;
    const TokenScale sx = token_scale(a.sx && !zero ? a.sx[src[j]] : 1.0f);
    const size_t ch = (none ? 0 : (size_t)e * a.n_out) + n;
    T v[4];
#pragma unroll
    for (uint32_t k = 0; k < 4; k++) {
      const bool in = n + k < a.n_out;
      const float sw = a.sw && in ? a.sw[ch + k] : 1.0f, b = a.bias && in ? a.bias[ch + k] : 0.0f;
      v[k] = zero ? (T)0 : finish<T>(sum[k], sx, sw, b, a.relu);
    }
    store4((T*)a.y + (size_t)t * a.ld_y + n, a.n_out - n, v);
  };
#pragma unroll
  for (int i = 0; i < FN; i++)
#pragma unroll
    for (int j = 0; j < FT; j++) sums[wave][i * FT + j][lane] = acc[i][j];
  __syncthreads();
  // wave k adds up square k
#pragma unroll
  for (int sq = 0; sq < FN * FT; sq++) {
    if ((uint32_t)sq % KW != wave) continue;
    v4i sum = sums[0][sq][lane];
#pragma unroll
    for (int k = 1; k < KW; k++) sum += sums[k][sq][lane];
    put(sq / FT, sq % FT, sum);
  }
}

// ------------------------------------------------------------ short rows, many of them
// A small layer over a whole data set: a wave keeps the weights, scales and
// biases of all 16 FN channels in registers and goes over the tokens, TILES of 16
// at a time, their rows read once, straight to fragments.  H: halves of 64 bytes
// that a row has.  Bound by memory, once the launch's own 2 us are past: 100003 rows,
// 64 to 32 integers, 5.6 us (19 MB); 500000: 20.3 (96 MB).  Measured in turn at
// 100003: 5.0 here and 9.0 through the tiles in LDS, whose blocks have one step
// each.  Results of 4 bytes leave around the caches, which would write them out only
// at the end (5.0 and 7.6 us); 8-byte pieces do not (4.8 us; 5.2 around the caches,
// 15 and 35 with 48 channels, 500000 rows).
template <class T, bool BYTES, int H, int FN>
__global__ __launch_bounds__(256) void k_i8_thin(I8Args a) {
  constexpr int TILES = 2;
  const uint32_t lane = threadIdx.x & 63, fr = lane & 15, c = lane >> 4;
  Chunk part[H];
  v4i wf[FN][H];
  float sw[FN][4], bias[FN][4];
#pragma unroll
  for (int h = 0; h < H; h++) part[h] = last_chunk(64 * h + 16 * c, a.n_in);
#pragma unroll
  for (int i = 0; i < FN; i++) {
    const uint32_t row = i * 16 + fr, n = i * 16 + 4 * c;
    const int8_t* w = a.w + (size_t)(row < a.n_out ? row : a.n_out - 1) * a.ld_w;
#pragma unroll
    for (int h = 0; h < H; h++) wf[i][h] = load16_end<BYTES>(w + part[h].at);
#pragma unroll
    for (uint32_t k = 0; k < 4; k++) {
      const bool in = n + k < a.n_out;
      sw[i][k] = a.sw && in ? a.sw[n + k] : 1.0f, bias[i][k] = a.bias && in ? a.bias[n + k] : 0.0f;
    }
  }
  const uint32_t wave = threadIdx.x >> 6, stride = gridDim.x * 4 * TILES * 16;
  for (uint32_t t0 = (blockIdx.x * 4 + wave) * TILES * 16; t0 < a.rows; t0 += stride) {
    v4i xf[TILES][H];
    TokenScale sx[TILES];
#pragma unroll
    for (int j = 0; j < TILES; j++) {
      const uint32_t t = t0 + j * 16 + fr, r = t < a.rows ? t : a.rows - 1;
#pragma unroll
      for (int h = 0; h < H; h++) xf[j][h] = load16_end<BYTES>(a.x + (size_t)r * a.ld_x + part[h].at) & part[h].mask;
      sx[j] = token_scale(a.sx ? a.sx[r] : 1.0f);
    }
#pragma unroll
    for (int j = 0; j < TILES; j++) {
      const uint32_t t = t0 + j * 16 + fr;
#pragma unroll
      for (int i = 0; i < FN; i++) {
        v4i acc = {};
#pragma unroll
        for (int h = 0; h < H; h++) acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(wf[i][h], xf[j][h], acc, 0, 0, 0);
        const uint32_t n = i * 16 + 4 * c;
        if (t >= a.rows || n >= a.n_out) continue;
        T v[4];
#pragma unroll
        for (int k = 0; k < 4; k++) v[k] = finish<T>(acc[k], sx[j], sw[i][k], bias[i][k], a.relu);
        store4<sizeof(T) == 4>((T*)a.y + (size_t)t * a.ld_y + n, a.n_out - n, v);
      }
    }
  }
}

// ------------------------------------------------------------ rows under 16 bytes
// A thread takes one result at a time: its sum has 15 terms at the most, or none.
template <class T, bool GROUPED>
__global__ __launch_bounds__(256) void k_i8_short(I8Args a) {
  const uint64_t all = (uint64_t)a.rows * a.n_out, stride = (uint64_t)gridDim.x * 256;
  for (uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x; i < all; i += stride) {
    const uint32_t p = (uint32_t)(i / a.n_out), n = (uint32_t)(i % a.n_out);
    int64_t s = p;
    size_t ch = n;
    if (GROUPED) {
      uint32_t e = 0, hi = a.experts;  // the last expert whose rows begin at p or before, with p among them
      while (e < hi) {
        const uint32_t mid = (e + hi) / 2;
        if (offset_of(a, mid + 1) <= p) e = mid + 1;
        else hi = mid;
      }
      s = e < a.experts ? source_row(a, p) : -1;
      ch += (size_t)e * a.n_out;
    }
    T v = (T)0;
    if (s >= 0) {
      int acc = 0;
      for (uint32_t k = 0; k < a.n_in; k++) acc += (int)a.x[(size_t)s * a.ld_x + k] * (int)a.w[ch * a.ld_w + k];
      v = finish<T>(acc, token_scale(a.sx ? a.sx[s] : 1.0f), a.sw ? a.sw[ch] : 1.0f, a.bias ? a.bias[ch] : 0.0f,
                    a.relu);
    }
    ((T*)a.y)[(size_t)p * a.ld_y + n] = v;
  }
}

// ------------------------------------------------------------ which kernel
// A product's time in ns: `base` once, and for each tile that a CU has to do
// (tiles / 256, rounded up where a tile fills a CU for long) `own` for its first
// loads and its results and `step` for each 128 bytes of k.  Fitted to products
// of 1 to 8192 rows, 16 to 8192 long; `odd`: for rows that are not multiples of
// 16 bytes.
struct TileCost {
  uint32_t bt, bn, base, own, step, odd_own, odd_step;
};
constexpr TileCost TILE_COST[] = {
    {16, 16, 600, 1000, 0, 1000, 0},     {32, 16, 600, 1000, 0, 1000, 0},     {16, 32, 600, 1000, 0, 1000, 0},
    {32, 32, 600, 1000, 0, 1000, 0},     {64, 64, 1200, 500, 200, 800, 300},  {128, 128, 1000, 2000, 500, 2200, 750},
    {256, 256, 500, 8000, 1600, 9000, 2500},
};

// The tile with the least estimated time: few rows are split over small tiles
// that read straight from memory, many go through the tiles that read each row
// fewest times.
static int choose_tile(const I8Args& a, bool grouped, bool odd_rows, bool bytes) {
  const uint64_t groups = grouped ? (a.experts < a.rows ? a.experts : a.rows) : 0;
  const uint64_t steps = (a.n_in + 127) / 128;
  int best = 0;
  uint64_t least = ~0ull;
  for (int i = 0; i < (int)(sizeof(TILE_COST) / sizeof(TILE_COST[0])); i++) {
    const TileCost& c = TILE_COST[i];
    const bool small = c.bt < 64, odd = small ? bytes : odd_rows;
    // an expert's last row tile is half full, or it has only one
    uint64_t tt = cdiv(a.rows, c.bt);
    if (grouped && (tt += groups / 2) < groups) tt = groups;
    uint64_t tiles = tt * cdiv(a.n_out, c.bn);
    if (tiles < 256 || !small) tiles = (tiles + 255) / 256 * 256;
    uint64_t own = odd ? c.odd_own : c.own, step = odd ? c.odd_step : c.step;
    // straight from memory: 128 bytes of each row at 36 bytes/ns a CU, the tile's
    // missing rows of x being one and the same
    if (small) step = (c.bn + (a.rows < tt * c.bt ? (a.rows + tt - 1) / tt : c.bt)) * (bytes ? 43 : 36) / 10;
    if (grouped) own += small ? 1000 : 2000;  // the chain of indexes
    const uint64_t t = c.base + tiles * (own + steps * step) / 256;
    if (t < least) least = t, best = i;
  }
  return best;
}

// Products for k_i8_thin: at 64 channels a token's rows in LDS are worth their
// steps (in turn, 100003 rows, 64 to 64 integers: 9.2 us there, 12.1 here; to 48: 9.2
// and 6.8), and under some thousand rows the tiles that split the channels are level
// with it (4096 rows, 64 to 32: 3.0 and 3.0; 512: 2.8 and 3.0).
constexpr uint32_t THIN_ROWS = 4096, THIN_OUT = 48, THIN_IN = 128;

// A product's kernels; those of tiles in the order of TILE_COST, the tiles in LDS
// by the waves that share one, or for odd rows.
enum ProductKernel {
  K_SHORT, K_THIN, K_DIRECT11, K_DIRECT21, K_DIRECT12, K_DIRECT22, K_RING64, K_ODD64, K_RING128_4, K_RING128_8,
  K_ODD128, K_RING256_8, K_RING256_16, K_ODD256, K_COUNT
};
constexpr const char* KERNEL_NAME[K_COUNT] = {
    "short", "thin", "direct 16x16", "direct 32x16", "direct 16x32", "direct 32x32", "ring 64x64", "odd 64x64",
    "ring 128x128, 4 waves", "ring 128x128, 8 waves", "odd 128x128", "ring 256x256, 8 waves",
    "ring 256x256, 16 waves", "odd 256x256"};

// (Of short sums a larger part is a tile's own, which more waves do faster (in turn,
// 8192 rows, 1024 to 8192: 92 us with eight waves of 128 x 128 and 102 with four, 84
// and 88 with sixteen and eight of 256 x 256); fewer waves read LDS less (8192 to
// 8192: 541 and 513, 441 and 426).  Grouped, all share the chain of indexes before
// the first step (66 us and 83, 4096 x 4 rows, 64 experts).)
struct ProductChoice {
  ProductKernel kernel;
  int tile;    // of TILE_COST
  bool bytes;  // rows at addresses inside a word
};
static ProductChoice choose_kernel(const I8Args& a, bool grouped) {
  if (a.n_in < 16 || (grouped && !a.tokens)) return {K_SHORT, 0, false};  // (without tokens there is no row to read)
  const size_t rows_at = (uintptr_t)a.x | (uintptr_t)a.w | a.ld_x | a.ld_w;
  const bool odd = (rows_at | a.n_in) % 16 != 0, bytes = rows_at % 4 != 0, few_steps = a.n_in <= 2048;
  if (!grouped && a.n_in <= THIN_IN && a.rows >= THIN_ROWS && a.n_out <= THIN_OUT) return {K_THIN, 0, bytes};
  const int c = choose_tile(a, grouped, odd, bytes);
  if (c < 4) return {(ProductKernel)(K_DIRECT11 + c), c, bytes};
  if (c == 4) return {odd ? K_ODD64 : K_RING64, c, bytes};
  if (c == 5) return {odd ? K_ODD128 : grouped || few_steps ? K_RING128_8 : K_RING128_4, c, bytes};
  return {odd ? K_ODD256 : few_steps ? K_RING256_16 : K_RING256_8, c, bytes};
}

template <class T, bool GROUPED>
static int launch_product(zk_context* ctx, const I8Args& a, hipStream_t st) {
  const char* name = GROUPED ? "i8_matmul_experts" : "i8_matmul";
  const ProductChoice c = choose_kernel(a, GROUPED);
  auto thin = [&](auto kernel) -> int {
    const uint32_t blocks = cdiv(a.rows, 128);
    ZK_LAUNCH(ctx, st, name, kernel, dim3(blocks < 2048 ? blocks : 2048), dim3(256), 0, a);
    return ZK_OK;
  };
  auto thin_by = [&](auto by, auto h) -> int {
    constexpr bool B = decltype(by)::value;
    constexpr int H = decltype(h)::value;
    if (a.n_out <= 16) return thin(k_i8_thin<T, B, H, 1>);
    if (a.n_out <= 32) return thin(k_i8_thin<T, B, H, 2>);
    return thin(k_i8_thin<T, B, H, 3>);
  };
  auto go = [&](auto kernel, uint32_t threads) -> int {
    // row tiles of the grouped form: whole ones, and a part of one for each
    // expert and for the rows without an expert
    const uint32_t bt = TILE_COST[c.tile].bt, groups = a.experts + 1 < a.rows ? a.experts + 1 : a.rows;
    const uint32_t tiles_t = GROUPED ? a.rows / bt + groups : cdiv(a.rows, bt);
    const uint32_t tiles_n = cdiv(a.n_out, TILE_COST[c.tile].bn);
    const size_t tiles = (size_t)tiles_t * tiles_n;
    if (tiles > I8_MAX_TILES) return ctx->fail(ZK_ERR_SIZE, "i8 experts: rows and n_out make too many tiles");
    ZK_LAUNCH(ctx, st, name, kernel, dim3(cdiv(tiles, 8) * 8), dim3(threads), 0, a, tiles_t, tiles_n);
    return ZK_OK;
  };
  auto direct = [&](auto ft, auto fn) -> int {
    constexpr int FT = decltype(ft)::value, FN = decltype(fn)::value;
    return c.bytes ? go(k_i8_direct<T, GROUPED, true, FT, FN, 8>, 512) : go(k_i8_direct<T, GROUPED, false, FT, FN, 8>, 512);
  };
  const std::integral_constant<int, 1> one;
  const std::integral_constant<int, 2> two;
  switch (c.kernel) {
    case K_SHORT: {
      const size_t blocks = ((size_t)a.rows * a.n_out + 255) / 256;
      ZK_LAUNCH(ctx, st, name, (k_i8_short<T, GROUPED>), dim3(blocks < 65536 ? (uint32_t)blocks : 65536), dim3(256), 0, a);
      return ZK_OK;
    }
    case K_THIN:
      if constexpr (!GROUPED) {
        if (c.bytes) return a.n_in <= 64 ? thin_by(std::true_type(), one) : thin_by(std::true_type(), two);
        return a.n_in <= 64 ? thin_by(std::false_type(), one) : thin_by(std::false_type(), two);
      }
      break;
    case K_DIRECT11: return direct(one, one);
    case K_DIRECT21: return direct(two, one);
    case K_DIRECT12: return direct(one, two);
    case K_DIRECT22: return direct(two, two);
    case K_RING64: return go(k_i8_ring<T, GROUPED, 2, 2, 1, 1>, 256);
    case K_ODD64: return go(k_i8_odd<T, GROUPED, 2, 2, 1, 1>, 256);
    case K_RING128_4:
      if constexpr (!GROUPED) return go(k_i8_ring<T, false, 2, 2, 2, 2>, 256);
      break;
    case K_RING128_8: return go(k_i8_ring<T, GROUPED, 2, 4, 2, 1>, 512);
    case K_ODD128: return go(k_i8_odd<T, GROUPED, 2, 4, 2, 1>, 512);
    case K_RING256_8: return go(k_i8_ring<T, GROUPED, 2, 4, 4, 2>, 512);
    case K_RING256_16: return go(k_i8_ring<T, GROUPED, 4, 4, 2, 2>, 1024);
    case K_ODD256: return go(k_i8_odd<T, GROUPED, 2, 4, 4, 2>, 512);
    default: break;
  }
  return ctx->fail(ZK_ERR_INVALID, "i8 product: no kernel");
}

template <bool GROUPED>
static int i8_dispatch(zk_context* ctx, const I8Args& a, int type, hipStream_t st) {
  switch (type) {
    case ZK_I32: return launch_product<int, GROUPED>(ctx, a, st);
    case ZK_F32: return launch_product<float, GROUPED>(ctx, a, st);
    case ZK_F16: return launch_product<_Float16, GROUPED>(ctx, a, st);
    default: return launch_product<__bf16, GROUPED>(ctx, a, st);
  }
}

// ------------------------------------------------------------ rows to 8 bits
// THREADS threads a row, ROWS rows a block.  A thread keeps its first HELD
// pieces of 16 bytes from the pass for the maximum to the pass that divides, so
// that rows of up to 64 KB are read once.  Bound by its own chain (load, maximum
// over the block, divide, store): 2048 rows of 4096 bf16 in 9.9 us (8.2 to 10.2), 25 MB
// at 2.5 TB/s.
template <class T, int THREADS, int ROWS>
__global__ __launch_bounds__(THREADS* ROWS) void k_i8_quantize(const T* __restrict__ x, size_t ld_x, uint32_t rows,
                                                               uint32_t cols, int8_t* __restrict__ q, size_t ld_q,
                                                               float* __restrict__ scale) {
  constexpr int HELD = 4;
  constexpr int WAVES = THREADS / 64;
  __shared__ uint32_t part[ROWS * WAVES];
  const uint32_t tid = threadIdx.x % THREADS, sub = threadIdx.x / THREADS;
  const uint32_t r = blockIdx.x * ROWS + sub;
  const bool on = r < rows;
  const T* row = x + (size_t)(on ? r : rows - 1) * ld_x;
  int8_t* out = q + (size_t)(on ? r : rows - 1) * ld_q;
  const uint32_t pieces = pieces_of<T>(cols);
  Vec<T> held[HELD];
  uint32_t m = 0;
  auto look = [&](const Vec<T>& v) { look_piece(v, m); };
#pragma unroll
  for (int h = 0; h < HELD; h++) {
    const uint32_t c = tid + h * THREADS;
    held[h] = Vec<T>{};
    if (c < pieces) held[h] = row_load(row + piece<T>(c, cols), cols - piece<T>(c, cols));
  }
#pragma unroll
  for (int h = 0; h < HELD; h++) look(held[h]);
  for (uint32_t c = tid + HELD * THREADS; c < pieces; c += THREADS)
    look(row_load(row + piece<T>(c, cols), cols - piece<T>(c, cols)));
#pragma unroll
  for (int d = 32; d; d >>= 1) {
    const uint32_t o = (uint32_t)__shfl_xor((int)m, d);
    m = o > m ? o : m;
  }
  if (WAVES > 1) {
    if ((tid & 63) == 0) part[sub * WAVES + (tid >> 6)] = m;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < WAVES; i++) {
      const uint32_t o = part[sub * WAVES + i];
      m = o > m ? o : m;
    }
  }
  if (!on) return;
  const RowScale rs = row_scale(m);
  if (tid == 0) scale[r] = rs.s;
  auto put = [&](uint32_t c, const Vec<T>& v) {
    const uint32_t at = piece<T>(c, cols);
    int8_t b[Vec<T>::N];
    quantize_piece(v, rs, b);
    if (cols - at >= Vec<T>::N) {
      __builtin_memcpy(out + at, b, sizeof(b));
    } else {
#pragma unroll
      for (uint32_t i = 0; i < Vec<T>::N; i++)
        if (i < cols - at) out[at + i] = b[i];
    }
  };
#pragma unroll
  for (int h = 0; h < HELD; h++) {
    const uint32_t c = tid + h * THREADS;
    if (c < pieces) put(c, held[h]);
  }
  for (uint32_t c = tid + HELD * THREADS; c < pieces; c += THREADS)
    put(c, row_load(row + piece<T>(c, cols), cols - piece<T>(c, cols)));
}

int i8_quantize(zk_context* ctx, const void* x, int type, size_t ld_x, size_t rows, size_t cols, int8_t* q,
                size_t ld_q, float* scale, hipStream_t st) {
  return by_type(type, [&](auto zero) -> int {
    typedef decltype(zero) T;
    const uint32_t pieces = pieces_of<T>((uint32_t)cols);
    // runs of rows: a launch stays below 2^32 threads
    for (size_t r = 0; r < rows; r += (size_t)1 << 21) {
      const uint32_t n = (uint32_t)(rows - r < (size_t)1 << 21 ? rows - r : (size_t)1 << 21);
      const T* from = (const T*)x + r * ld_x;
      int8_t* to = q + r * ld_q;
      // one piece a thread where rows are few (their latency counts), else two
      // to four of them a thread
      if (pieces <= 64 || (rows >= 2048 && pieces <= 256))
        ZK_LAUNCH(ctx, st, "i8_quantize", (k_i8_quantize<T, 64, 4>), dim3(cdiv(n, 4)), dim3(256), 0, from, ld_x, n,
                  (uint32_t)cols, to, ld_q, scale + r);
      else if (pieces <= 256 || (rows >= 512 && pieces <= 1024))
        ZK_LAUNCH(ctx, st, "i8_quantize", (k_i8_quantize<T, 256, 1>), dim3(n), dim3(256), 0, from, ld_x, n,
                  (uint32_t)cols, to, ld_q, scale + r);
      else
        ZK_LAUNCH(ctx, st, "i8_quantize", (k_i8_quantize<T, 1024, 1>), dim3(n), dim3(1024), 0, from, ld_x, n,
                  (uint32_t)cols, to, ld_q, scale + r);
    }
    return ZK_OK;
  });
}

// ------------------------------------------------------------ a few rows, quantized on the way
// The linear layer of at most 16 rows in one launch: each block asks for its
// first weights, quantizes all of x's rows into LDS while they come (x is small:
// every block reads it from the L2), and goes on as k_i8_direct with its x
// fragments from LDS.  Bound by the chain of x's maximum, its bytes and the
// product: one row, 8192 to 1024 f16, in 9.9 us, 3.9 + 7.2 in two launches.  x's
// quantization is repeated in every block, which costs more than the host's second
// launch once x is large.  A call, this way and in two launches (medians, us): one
// row, 4096 to 4096 bf16, 13.4 and 16.0; 8 rows, 4062 to 1024 (32 KB), 13.6 and 15.7,
// in f32 14.9 and 15.7; 3 rows, 15000 to 1000 (44 KB), 20.2 and 15.6; 16 rows, 2900 to
// 8195 (46 KB), 19.5 and 15.4.  On the GPU alone, where nothing waits for the host,
// two launches are level from about 16 KB on (4096 to 4096: 4 rows 9.3 and 3.4 + 5.8,
// 8 rows 12.5 and 3.6 + 6.2).
template <class T, class X, int FN>
__global__ __launch_bounds__(512) void k_i8_few(I8Args a, const X* __restrict__ x, size_t ld_x) {
  constexpr uint32_t BN = 16 * FN, BK = 128, KW = 8;
  constexpr int U = FN == 1 ? 4 : 2;
  extern __shared__ __align__(16) int8_t q[];  // rows x few_ld(n_in)
  __shared__ __align__(16) v4i sums[KW][FN][64];
  __shared__ uint32_t part[FEW_ROWS][KW];
  __shared__ float scale[FEW_ROWS];
  const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t n0 = blockIdx.x * BN, fr = lane & 15, c = lane >> 4, ld = few_ld(a.n_in);
  const int8_t* wp[FN];
#pragma unroll
  for (int i = 0; i < FN; i++) {
    const uint32_t n = n0 + i * 16 + fr;
    wp[i] = a.w + (size_t)(n < a.n_out ? n : a.n_out - 1) * a.ld_w;
  }
  const uint32_t steps = (a.n_in + BK - 1) / BK, full = a.n_in / BK;
  v4i wf[U][FN][2];
  const bool words = (((uint32_t)(uintptr_t)a.w | (uint32_t)a.ld_w) & 3u) == 0;
  auto load_as = [&](auto bytes, uint32_t step) {
#pragma unroll
    for (int u = 0; u < U; u++) {
      const uint32_t st = step + u * KW, k = st * BK + c * 32;
      if (st < full) {
#pragma unroll
        for (int i = 0; i < FN; i++) load_pair<decltype(bytes)::value>(wp[i] + st * BK, c, wf[u][i]);
      } else if (st < steps) {
#pragma unroll
        for (int h = 0; h < 2; h++)
#pragma unroll
          for (int i = 0; i < FN; i++) wf[u][i][h] = load16_end<decltype(bytes)::value>(wp[i] + last_chunk(k + 16 * h, a.n_in).at);
      }
    }
  };
  auto load = [&](uint32_t step) {
    if (words) load_as(std::false_type(), step);
    else load_as(std::true_type(), step);
  };
  load(wave);
  quantize_rows<X, KW>(x, ld_x, a.rows, a.n_in, q, ld, part, scale);
  // ---- the product
  const uint32_t row = fr < a.rows ? fr : a.rows - 1;
  const int8_t* xq = q + row * ld;
  v4i acc[FN] = {};
  for (uint32_t step = wave; step < steps; step += U * KW) {
    if (step != wave) load(step);
#pragma unroll
    for (int u = 0; u < U; u++) {
      const uint32_t st = step + u * KW;
      if (st >= steps) break;
#pragma unroll
      for (int h = 0; h < 2; h++) {
        v4i xf;
        if (st < full) {
          xf = *(const v4i*)(xq + st * BK + (words ? c * 16 + 64 * h : c * 32 + 16 * h));
        } else {
          const Chunk part = last_chunk(st * BK + c * 32 + 16 * h, a.n_in);
          __builtin_memcpy(&xf, xq + part.at, 16);
          xf &= part.mask;
        }
#pragma unroll
        for (int i = 0; i < FN; i++) acc[i] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wf[u][i][h], xf, acc[i], 0, 0, 0);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < FN; i++) sums[wave][i][lane] = acc[i];
  wait_lds();
  meet();
  if (wave >= FN) return;
  v4i sum = sums[0][wave][lane];
#pragma unroll
  for (uint32_t k = 1; k < KW; k++) sum += sums[k][wave][lane];
  const uint32_t n = n0 + wave * 16 + 4 * c;
  if (fr >= a.rows || n >= a.n_out) return;
  const TokenScale sx = token_scale(scale[fr]);
  T v[4];
#pragma unroll
  for (uint32_t k = 0; k < 4; k++) {
    const bool in = n + k < a.n_out;
    v[k] = finish<T>(sum[k], sx, a.sw && in ? a.sw[n + k] : 1.0f, a.bias && in ? a.bias[n + k] : 0.0f, a.relu);
  }
  store4((T*)a.y + (size_t)fr * a.ld_y + n, a.n_out - n, v);
}

static bool few_rows(size_t rows, size_t n_in) {
  return rows <= FEW_ROWS && n_in >= 16 && n_in <= I8_MAX_IN && rows * few_ld((uint32_t)n_in) <= FEW_BYTES;
}

static int launch_few(zk_context* ctx, const I8Args& a, const void* x, int x_type, size_t ld_x, int y_type,
                      hipStream_t st) {
  return by_type(x_type, [&](auto xz) -> int {
    return by_type(y_type, [&](auto yz) -> int {
      typedef decltype(xz) X;
      typedef decltype(yz) T;
      const uint32_t lds = a.rows * few_ld(a.n_in);
      // 32 channels a block halve the times that x is quantized; with fewer
      // than 256 such blocks they would leave CUs without one
      if (a.n_out >= 8192)
        ZK_LAUNCH(ctx, st, "i8_linear", (k_i8_few<T, X, 2>), dim3(cdiv(a.n_out, 32)), dim3(512), lds, a, (const X*)x, ld_x);
      else
        ZK_LAUNCH(ctx, st, "i8_linear", (k_i8_few<T, X, 1>), dim3(cdiv(a.n_out, 16)), dim3(512), lds, a, (const X*)x, ld_x);
      return ZK_OK;
    });
  });
}

// ------------------------------------------------------------ arguments
// Checks that the two forms of the product share.  reads_x: x has rows at all.
static int check_product(zk_context* ctx, const I8Args& a, size_t rows, size_t n_out, size_t n_in, int type,
                         bool reads_x = true) {
  if (type != ZK_I32 && !float_type(type)) return ctx->fail(ZK_ERR_INVALID, "i8 product: unknown type of y");
  if (type == ZK_I32 && (a.sx || a.sw || a.bias))
    return ctx->fail(ZK_ERR_INVALID, "i8 product: integer sums take no scales and no bias");
  if (n_in > I8_MAX_IN) return ctx->fail(ZK_ERR_SIZE, "i8 product: n_in above 131071 can pass 32 bits");
  if (rows > 0x7fffffffu || n_out > 0x7fffffffu) return ctx->fail(ZK_ERR_SIZE, "i8 product: sizes above 2^31 - 1");
  if (n_out > 16 * I8_MAX_TILES) return ctx->fail(ZK_ERR_SIZE, "i8 product: n_out above 2^26");
  if (a.ld_x < n_in || a.ld_w < n_in || a.ld_y < n_out)
    return ctx->fail(ZK_ERR_INVALID, "i8 product: a row stride below the row's length");
  if (rows && n_out && (!a.y || (n_in && ((!a.x && reads_x) || !a.w))))
    return ctx->fail(ZK_ERR_INVALID, "i8 product: null pointer");
  if (!aligned(a.y, type_bytes(type)) || !aligned(a.sx, 4) || !aligned(a.sw, 4) || !aligned(a.bias, 4))
    return ctx->fail(ZK_ERR_INVALID, "i8 product: a pointer is not aligned to its type");
  return ZK_OK;
}

int check_quantize(zk_context* ctx, const void* x, int type, size_t ld_x, size_t rows, size_t cols) {
  if (!float_type(type)) return ctx->fail(ZK_ERR_INVALID, "i8 quantize: x is f32, f16 or bf16");
  if (rows > 0x7fffffffu || cols > 0x7fffffffu) return ctx->fail(ZK_ERR_SIZE, "i8 quantize: sizes above 2^31 - 1");
  if (ld_x < cols) return ctx->fail(ZK_ERR_INVALID, "i8 quantize: a row stride below the row's length");
  if (rows && cols && !x) return ctx->fail(ZK_ERR_INVALID, "i8 quantize: null pointer");
  if (!aligned(x, type_bytes(type))) return ctx->fail(ZK_ERR_INVALID, "i8 quantize: x is not aligned to its type");
  return ZK_OK;
}

LinearWork linear_work(size_t rows, size_t n_in) {
  LinearWork w;
  w.ld = (n_in + 63) / 64 * 64;
  w.q = (rows * 4 + 63) / 64 * 64;
  w.bytes = w.q + rows * w.ld;
  return w;
}

static int matmul_impl(zk_context* ctx, const int8_t* x, size_t ld_x, const float* sx, const int8_t* w, size_t ld_w,
                       const float* sw, const float* bias, size_t rows, size_t n_out, size_t n_in, int relu, void* y,
                       int type, size_t ld_y, hipStream_t st) {
  I8Args a = {};
  a.x = x, a.w = w, a.sx = sx, a.sw = sw, a.bias = bias, a.y = y;
  a.ld_x = ld_x, a.ld_w = ld_w, a.ld_y = ld_y;
  ZK_TRY(check_product(ctx, a, rows, n_out, n_in, type));
  if (!rows || !n_out) return ZK_OK;
  a.n_out = (uint32_t)n_out, a.n_in = (uint32_t)n_in, a.relu = relu != 0;
  // rows in runs of at most I8_MAX_TILES tiles of 16 x 16
  const size_t most = I8_MAX_TILES / ((n_out + 15) / 16) * 16;
  for (size_t r = 0; r < rows; r += most) {
    I8Args b = a;
    b.rows = (uint32_t)(rows - r < most ? rows - r : most);
    b.x = x ? x + r * ld_x : x;
    b.sx = sx ? sx + r : sx;
    b.y = (uint8_t*)y + r * ld_y * type_bytes(type);
    ZK_TRY(i8_dispatch<false>(ctx, b, type, st));
  }
  return ZK_OK;
}

}  // namespace zk

extern "C" {

int zk_i8_quantize(zk_context* ctx, const void* d_x, int x_type, size_t ld_x, size_t rows, size_t cols, int8_t* d_q,
                   size_t ld_q, float* d_scale, void* stream) {
  using namespace zk;
  if (!ctx) return ZK_ERR_INVALID;
  return guard(ctx, [&]() -> int {
    ZK_TRY(check_quantize(ctx, d_x, x_type, ld_x, rows, cols));
    if (ld_q < cols) return ctx->fail(ZK_ERR_INVALID, "i8 quantize: a row stride below the row's length");
    if (rows && (!d_scale || (cols && !d_q))) return ctx->fail(ZK_ERR_INVALID, "i8 quantize: null pointer");
    if (!aligned(d_scale, 4)) return ctx->fail(ZK_ERR_INVALID, "i8 quantize: d_scale is not aligned to its type");
    return i8_quantize(ctx, d_x, x_type, ld_x, rows, cols, d_q, ld_q, d_scale, ctx->s(stream));
  });
}

int zk_i8_matmul(zk_context* ctx, const int8_t* d_x, size_t ld_x, const float* d_x_scale, const int8_t* d_w,
                 size_t ld_w, const float* d_w_scale, const float* d_bias, size_t rows, size_t n_out, size_t n_in,
                 int relu, void* d_y, int y_type, size_t ld_y, void* stream) {
  using namespace zk;
  if (!ctx) return ZK_ERR_INVALID;
  return guard(ctx, [&] {
    return matmul_impl(ctx, d_x, ld_x, d_x_scale, d_w, ld_w, d_w_scale, d_bias, rows, n_out, n_in, relu, d_y, y_type,
                       ld_y, ctx->s(stream));
  });
}

const char* zk_debug_i8_kernel(size_t rows, size_t n_out, size_t n_in, size_t ld_x, size_t ld_w, size_t address,
                               int experts) {
  using namespace zk;
  if (rows > 0x7fffffffu || n_out > 0x7fffffffu || n_in > I8_MAX_IN || experts < 0) return nullptr;
  I8Args a = {};
  a.x = (const int8_t*)address, a.ld_x = ld_x, a.ld_w = ld_w;
  a.rows = (uint32_t)rows, a.n_out = (uint32_t)n_out, a.n_in = (uint32_t)n_in;
  a.experts = (uint32_t)experts, a.tokens = a.rows;
  return KERNEL_NAME[choose_kernel(a, experts > 0).kernel];
}

size_t zk_i8_linear_work(size_t rows, size_t n_in) {
  if (rows > 0x7fffffffu || n_in > zk::I8_MAX_IN) return 0;
  return zk::linear_work(rows, n_in).bytes;
}

int zk_i8_linear(zk_context* ctx, const void* d_x, int x_type, size_t ld_x, const int8_t* d_w, size_t ld_w,
                 const float* d_w_scale, const float* d_bias, size_t rows, size_t n_out, size_t n_in, int relu,
                 void* d_y, int y_type, size_t ld_y, void* d_work, size_t work_bytes, void* stream) {
  using namespace zk;
  if (!ctx) return ZK_ERR_INVALID;
  return guard(ctx, [&]() -> int {
    ZK_TRY(check_quantize(ctx, d_x, x_type, ld_x, rows, n_in));
    if (!float_type(y_type)) return ctx->fail(ZK_ERR_INVALID, "i8 linear: y is f32, f16 or bf16");
    if (n_in > I8_MAX_IN) return ctx->fail(ZK_ERR_SIZE, "i8 linear: n_in above 131071 can pass 32 bits");
    if (!rows || !n_out) return ZK_OK;
    const LinearWork lw = linear_work(rows, n_in);
    if (!d_work || !aligned(d_work, 16) || work_bytes < lw.bytes)
      return ctx->fail(ZK_ERR_INVALID, "i8 linear: workspace missing, too small or not aligned to 16 bytes");
    float* scale = (float*)d_work;
    int8_t* q = (int8_t*)d_work + lw.q;
    hipStream_t st = ctx->s(stream);
    I8Args a = {};
    a.x = q, a.w = d_w, a.sx = scale, a.sw = d_w_scale, a.bias = d_bias, a.y = d_y;
    a.ld_x = lw.ld, a.ld_w = ld_w, a.ld_y = ld_y;
    ZK_TRY(check_product(ctx, a, rows, n_out, n_in, y_type));
    if (few_rows(rows, n_in)) {
      a.rows = (uint32_t)rows, a.n_out = (uint32_t)n_out, a.n_in = (uint32_t)n_in, a.relu = relu != 0;
      return launch_few(ctx, a, d_x, x_type, ld_x, y_type, st);
    }
    ZK_TRY(i8_quantize(ctx, d_x, x_type, ld_x, rows, n_in, q, lw.ld, scale, st));
    return matmul_impl(ctx, q, lw.ld, scale, d_w, ld_w, d_w_scale, d_bias, rows, n_out, n_in, relu, d_y, y_type,
                       ld_y, st);
  });
}

int zk_i8_matmul_experts(zk_context* ctx, const int8_t* d_x, size_t ld_x, const float* d_x_scale, size_t tokens,
                         const int8_t* d_w, size_t ld_w, const float* d_w_scale, const float* d_bias,
                         const int32_t* d_offsets, int experts, const int32_t* d_order, int slots, size_t rows,
                         size_t n_out, size_t n_in, int relu, void* d_y, int y_type, size_t ld_y, void* stream) {
  using namespace zk;
  if (!ctx) return ZK_ERR_INVALID;
  return guard(ctx, [&]() -> int {
    I8Args a = {};
    a.x = d_x, a.w = d_w, a.sx = d_x_scale, a.sw = d_w_scale, a.bias = d_bias, a.y = d_y;
    a.ld_x = ld_x, a.ld_w = ld_w, a.ld_y = ld_y;
    if (experts < 1 || experts > ZK_MAX_EXPERTS)
      return ctx->fail(ZK_ERR_SIZE, "i8 experts: between 1 and 1024 experts");
    if (slots < 1) return ctx->fail(ZK_ERR_INVALID, "i8 experts: slots is at least 1");
    ZK_TRY(check_product(ctx, a, rows, n_out, n_in, y_type, tokens > 0));
    if (rows > ZK_MAX_EXPERT_ROWS || tokens > 0x7fffffffu)
      return ctx->fail(ZK_ERR_SIZE, "i8 experts: too many rows");
    if (!rows || !n_out) return ZK_OK;
    if (!d_offsets) return ctx->fail(ZK_ERR_INVALID, "i8 experts: null pointer");
    if (!aligned(d_offsets, 4) || !aligned(d_order, 4))
      return ctx->fail(ZK_ERR_INVALID, "i8 experts: a pointer is not aligned to its type");
    a.rows = (uint32_t)rows, a.n_out = (uint32_t)n_out, a.n_in = (uint32_t)n_in, a.relu = relu != 0;
    a.offsets = d_offsets, a.order = d_order, a.experts = (uint32_t)experts, a.slots = (uint32_t)slots;
    a.tokens = (uint32_t)tokens;
    return i8_dispatch<true>(ctx, a, y_type, ctx->s(stream));
  });
}

}  // extern "C"
