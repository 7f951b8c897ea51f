// Layers with 4-bit weights for gfx950: 8-bit rows (one scale each) times weights
// of 4 bits with a scale for each group of a channel's weights.
//
//   acc[t,n,g] = sum_{k in group g} x[t,k] q[n,k]            exact, -8 <= q <= 7
//   y[t,n]     = act(sx[t] sum_g s[g,n] acc[t,n,g] + b[n])
//
// A run of 128 weights of a channel is 64 bytes, whose byte b holds weight b in
// its low and weight 64 + b in its high four bits: 16 neighbouring bytes are, by a
// shift and a mask, two times 16 neighbouring weights, as the matrix instructions
// take them.  Scales lie by group, so that a group's scales of neighbouring
// channels are neighbours.
#include <math.h>

#include <type_traits>

#include "i8_product.hpp"

namespace zk {

constexpr size_t I4_MAX_IN = (size_t)1 << 24;  // (indexes inside a row stay far below 32 bits)

struct I4Args : I8Args {
  const void* scale;  // groups x n_out, for each expert
  uint32_t group, groups;
  int scale_type, y_type;
};

static __host__ __device__ inline size_t i4_row_bytes(size_t n_in) { return (n_in + 127) / 128 * 64; }

// Rows of x behind N positions, -1 for those that hold none, their loads under way
// together (a chain of branches had them wait for one another).
template <bool GROUPED, int N>
__device__ __forceinline__ void source_rows(const I4Args& a, const uint32_t (&p)[N], int (&s)[N]) {
  if (!GROUPED || !a.order) {
#pragma unroll
    for (int i = 0; i < N; i++) s[i] = !GROUPED || p[i] < a.tokens ? (int)p[i] : -1;
    return;
  }
  int o[N];
#pragma unroll
  for (int i = 0; i < N; i++) o[i] = a.order[p[i]];
#pragma unroll
  for (int i = 0; i < N; i++) {
    const uint32_t t = (uint32_t)o[i] / a.slots;
    s[i] = o[i] >= 0 && t < a.tokens ? (int)t : -1;
  }
}

// sx sum + b in one rounding; what is below zero becomes zero, a NaN stays.
__device__ __forceinline__ float i4_finish(float sum, float sx, float b, int relu) {
  const float f = fmaf(sum, sx, b);
  return relu && f < 0.0f ? 0.0f : f;
}

// Zeros for rows that have no token to read.
template <class T>
__global__ __launch_bounds__(256) void k_i4_zeros(T* __restrict__ y, size_t ld_y, uint32_t rows, uint32_t n_out) {
  const uint64_t all = (uint64_t)rows * n_out, stride = (uint64_t)gridDim.x * 256;
  for (uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x; i < all; i += stride)
    y[(size_t)(i / n_out) * ld_y + i % n_out] = (T)0.0f;
}

// ------------------------------------------------------------ few rows
typedef float v4f __attribute__((ext_vector_type(4)));

// 16 bytes of a row of x from byte k on, zeros from its end on; nothing outside the
// row is read.
__device__ __forceinline__ v4i x_piece(const int8_t* row, uint32_t k, uint32_t n_in) {
  v4i v = {0, 0, 0, 0};
  if (k + 16 <= n_in) {
    __builtin_memcpy(&v, row + k, 16);
  } else if (k < n_in) {
    if (n_in >= 16) {
      unsigned __int128 w;
      __builtin_memcpy(&w, row + n_in - 16, 16);
      w >>= 8 * (16 - (n_in - k));
      __builtin_memcpy(&v, &w, 16);
    } else {
      for (uint32_t j = 0; j < n_in - k; j++) v[j >> 2] |= (int)((uint32_t)(uint8_t)row[k + j] << (8 * (j & 3)));
    }
  }
  return v;
}

// Result of row t's channel n.
__device__ __forceinline__ void i4_put(const I4Args& a, uint32_t t, uint32_t n, float v) {
  const size_t at = (size_t)t * a.ld_y + n;
  if (a.y_type == ZK_F32) ((float*)a.y)[at] = v;
  else if (a.y_type == ZK_F16) ((_Float16*)a.y)[at] = (_Float16)v;
  else ((__bf16*)a.y)[at] = (__bf16)v;
}

// A scale's bits, and a sixteenth of what they are worth (apart, so that a load waits for
// nothing): the products are of 16 times the weights, and sums of scaled groups that were
// too, until the end, left the range of 32 bits 16 times early.  Only f32 and bf16 scales
// below 2^-122 lose bits by it, down to a multiple of 2^-145.
__device__ __forceinline__ uint32_t scale_bits(const I4Args& a, size_t at) {
  return a.scale_type == ZK_F32 ? ((const uint32_t*)a.scale)[at] : ((const uint16_t*)a.scale)[at];
}
__device__ __forceinline__ float scale_of(const I4Args& a, uint32_t bits) {
  if (a.scale_type == ZK_F32) return __uint_as_float(bits) * 0.0625f;
  if (a.scale_type == ZK_BF16) return __uint_as_float(bits << 16) * 0.0625f;
  const uint16_t b = (uint16_t)bits;
  _Float16 h;
  __builtin_memcpy(&h, &b, 2);
  return (float)h * 0.0625f;
}
// Groups behind the row's end (of a last step, if a group is less than one) have scales of
// zero: their sums are zero, but the last group's scale may be an infinity.  Of one scale
// on its way to LDS, and of a wave's window in LDS, from `from` to `to`.
template <int NS>
__device__ __forceinline__ float scale_of_group(const I4Args& a, uint32_t bits, uint32_t g) {
  return NS == 1 || g < a.groups ? scale_of(a, bits) : 0.0f;
}
__device__ __forceinline__ void zero_scales(float* scales, uint32_t from, uint32_t to, uint32_t lane) {
  for (uint32_t k = from + lane; k < to; k += 64) scales[k] = 0.0f;
}

// A step's products of 16 tokens and 16 channels, a sum for each of its groups, 16 times
// too large: p a lane's packed weights, x its two fragments.  Groups of 32: an instruction's
// two are told apart by x, the lanes of the other one hold zeros.
template <int G, int NS>
__device__ __forceinline__ void i4_multiply(const v4i (&x)[2], const v4i& p, uint32_t c, v4i (&sums)[NS]) {
  const v4i high = p & (int)0xf0f0f0f0, low = (p << 4) & (int)0xf0f0f0f0, zero = {0, 0, 0, 0};
  if constexpr (G >= 128) {
    sums[0] = __builtin_amdgcn_mfma_i32_16x16x64_i8(x[0], low, zero, 0, 0, 0);
    sums[0] = __builtin_amdgcn_mfma_i32_16x16x64_i8(x[1], high, sums[0], 0, 0, 0);
  } else if constexpr (G == 64) {
    sums[0] = __builtin_amdgcn_mfma_i32_16x16x64_i8(x[0], low, zero, 0, 0, 0);
    sums[1] = __builtin_amdgcn_mfma_i32_16x16x64_i8(x[1], high, zero, 0, 0, 0);
  } else {
#pragma unroll
    for (int k = 0; k < NS; k++)
      sums[k] = __builtin_amdgcn_mfma_i32_16x16x64_i8((int)c / 2 == k % 2 ? x[k / 2] : zero, k < 2 ? low : high, zero, 0, 0, 0);
  }
}

// Few tokens (decoding), or a small layer: w is read once.  A block has 16 FT tokens x
// 16 FN channels, its KW waves a part of k each, in steps of 128; their sums meet in LDS.
// A wave's rows come by lanes that lie side by side in them, straight from memory into
// LDS of its own, U steps ahead (a fragment's 64 lanes, sixteen rows apart, are sixty-four
// accesses of 16 bytes to the vector cache, which does one a cycle: 48 tokens, 8192 to
// 8192, took 20 us that way), so that waves wait for nobody until the end.
// The matrix instruction takes 16 tokens (D's rows) and 16 channels (its columns): a lane
// holds four tokens of one channel, and needs one scale.  16 packed bytes of a lane are its
// operands of two instructions, 16 times the weights, which the scales take back.  G: 128
// for groups of whole steps, 64 or 32.  D's row 4 c + i is token 4 i + c of the 16, so
// that up to four tokens (NI = 1) are one register of each lane.  ODD: x's rows start at
// any byte or end inside a chunk of 16; they come through registers, masked.
// Traced: 1 row, 4096 to 4096 4.6 us, a launch and one chain of loads (8 MB of weights:
// 1.4 us); 48 rows, 8192 to 8192 13.2 us, 12.3 in a graph (34 MB: 5.9 us).
template <int G, bool GROUPED, bool ODD, int FT, int FN, int NI, int KW, int U>
__global__ __launch_bounds__(64 * KW) void k_i4_wave(I4Args a, uint32_t tiles_t, uint32_t tiles_n) {
  constexpr uint32_t BT = NI < 4 ? 4 * NI : 16 * FT, BN = 16 * FN;
  constexpr uint32_t XROWS = NI < 4 ? 4 : 16 * FT;               // of x in LDS
  constexpr uint32_t XB = XROWS * 128, WB = BN * 64, STEP = XB + WB, OWN = 2 * U * STEP;
  constexpr int XP = U * (int)XB / 1024;                         // 1 KB pieces of x in U steps
  constexpr int LOADS = (ODD ? 0 : XP) + U * FN;
  constexpr int NS = G >= 128 ? 1 : 128 / G;                     // scales of a step
  constexpr uint32_t ROWS = 16, W = ROWS / NS;                   // rows of scales, and steps, of a window
  constexpr uint32_t SUMS = FN * FT * NI * 64 * 4;
  static_assert(XP * 1024 == U * (int)XB && KW * OWN >= KW * SUMS, "whole pieces; the sums' LDS is the rows'");
  __shared__ __align__(16) int8_t lds[KW * OWN];
  __shared__ float scales[KW][ROWS][BN];
  const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  uint32_t r0, r1, n0, e;
  if (!block_tile<GROUPED>(a, BT, BN, tiles_t, tiles_n, r0, r1, n0, e)) return;
  const bool none = GROUPED && e >= a.experts;
  const uint32_t fr = lane & 15, c = lane >> 4;
  const size_t ch = none ? 0 : (size_t)e * a.n_out;
  const uint32_t steps = none ? 0 : (a.n_in + 127) / 128;
  const uint32_t per = (steps + KW - 1) / KW, first = wave * per, last = first + per < steps ? first + per : steps;
  // ---- what a lane fetches: x's piece p is its rows 8 p to 8 p + 7 of the U steps' one after
  // the other; chunk s of a row r lies at s ^ (r / 2 % 8), w's at s ^ (r / 4 % 4)
  const int8_t *xp[XP], *wp[FN];
  auto x_step = [&](int p) { return (p * 8 + (lane >> 3)) / XROWS; };
  auto x_chunk = [&](int p) { return ((lane & 7) ^ (((p * 8 + (lane >> 3)) % XROWS) >> 1 & 7)) * 16; };
#pragma unroll
  for (int i = 0; i < FN; i++) {
    const uint32_t row = i * 16 + (lane >> 2), n = n0 + row < a.n_out ? n0 + row : a.n_out - 1;
    wp[i] = a.w + (ch + n) * a.ld_w + ((lane & 3) ^ (row >> 2 & 3)) * 16;
  }
  // rows of x that the lane fetches, and of the results that it will finish
  constexpr int DONE = (FN * FT * NI + KW - 1) / KW;
  uint32_t place[XP + DONE];
  int from[XP + DONE];
#pragma unroll
  for (int p = 0; p < XP; p++) {
    const uint32_t row = (p * 8 + (lane >> 3)) % XROWS;
    const uint32_t t = r0 + (NI < 4 ? row : row / 16 * 16 + (row & 3) * 4 + (row % 16 >> 2));
    place[p] = t < r1 ? t : r1 - 1;
  }
  bool has[DONE];
#pragma unroll
  for (int d = 0; d < DONE; d++) {
    const uint32_t r = wave + d * KW, sq = r / NI, t = r0 + sq % FT * 16 + 4 * (r % NI) + c, n = n0 + sq / FT * 16 + fr;
    has[d] = r < FN * FT * NI && t < r1 && t < r0 + BT && n < a.n_out && !none;
    place[XP + d] = has[d] ? t : r1 - 1;
  }
  source_rows<GROUPED>(a, place, from);
#pragma unroll
  for (int p = 0; p < XP; p++) xp[p] = a.x + (size_t)(from[p] < 0 ? 0 : from[p]) * a.ld_x;
  // the results' factors
  float fx[DONE], fb[DONE];
#pragma unroll
  for (int d = 0; d < DONE; d++) {
    const uint32_t n = n0 + (wave + d * KW) / NI / FT * 16 + fr;
    has[d] = has[d] && from[XP + d] >= 0;
    fx[d] = has[d] && a.sx ? a.sx[from[XP + d]] : 1.0f;
    fb[d] = has[d] && a.bias ? a.bias[ch + n] : 0.0f;
  }
  int8_t* own = lds + wave * OWN;
  const uint32_t base = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) int8_t*)lds + wave * OWN;
  // U steps from s on into one half of the wave's LDS: x's rows of each, then w's
  auto fetch = [&](uint32_t s, uint32_t half) {
    const uint32_t at = base + half * U * STEP;
    if constexpr (ODD) {
      v4i held[XP];
#pragma unroll
      for (int p = 0; p < XP; p++) held[p] = x_piece(xp[p], (s + x_step(p)) * 128 + x_chunk(p), a.n_in);
#pragma unroll
      for (int p = 0; p < XP; p++) *(v4i*)(own + half * U * STEP + p * 1024 + lane * 16) = held[p];
    } else {
#pragma unroll
      for (int p = 0; p < XP; p++) {
        const uint32_t k = (s + x_step(p)) * 128 + x_chunk(p);
        load_to_lds(k < a.n_in ? xp[p] + k : (const int8_t*)&zeros16, at + p * 1024);
      }
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
      const uint32_t step = s + u < last ? s + u : last - 1;  // (again the last one, not used)
#pragma unroll
      for (int i = 0; i < FN; i++) load_to_lds(wp[i] + (size_t)step * 64, at + U * XB + u * WB + i * 1024);
    }
  };
  float acc[FN][FT][NI] = {};
  const uint32_t whole = G >= 128 ? a.group / 128 : 1;  // steps of a group
  for (uint32_t w0 = first; w0 < last; w0 += W) {
    const uint32_t end = w0 + W < last ? w0 + W : last;
    uint32_t sc[4 * FN];
#pragma unroll
    for (int i = 0; i < 4 * FN; i++) {
      const uint32_t k = lane + i * 64, n = n0 + k % BN < a.n_out ? n0 + k % BN : a.n_out - 1;
      uint32_t g = w0 * NS + k / BN;
      if (G >= 128) g /= whole;
      if (g >= a.groups) g = a.groups - 1;  // (of a step's part behind the row's end, not used)
      sc[i] = scale_bits(a, ch * a.groups + (size_t)g * a.n_out + n);
    }
    fetch(w0, 0);
    if (w0 + U < end) fetch(w0 + U, 1);
#pragma unroll
    for (int i = 0; i < 4 * FN; i++) {
      const uint32_t k = lane + i * 64;
      scales[wave][k / BN][k % BN] = scale_of(a, sc[i]);
    }
    if (NS > 1 && end * NS > a.groups) zero_scales(&scales[wave][0][0], (a.groups - w0 * NS) * BN, ROWS * BN, lane);
    uint32_t half = 0;
    for (uint32_t s0 = w0; s0 < end; s0 += U) {
      if (s0 + U < end) wait_loads<LOADS>();
      else wait_loads<0>();
      wait_lds();
      const int8_t *sx = own + half * U * STEP, *sw = sx + U * XB;
#pragma unroll
      for (int u = 0; u < U; u++) {
        if (s0 + u >= end) break;
        v4i xf[FT][2];
#pragma unroll
        for (int j = 0; j < FT; j++) {
          const uint32_t row = NI < 4 ? fr >> 2 : j * 16 + fr;
#pragma unroll
          for (int h = 0; h < 2; h++)
            xf[j][h] = *(const v4i*)(sx + u * XB + row * 128 + ((4 * h + c) ^ (row >> 1 & 7)) * 16);
        }
#pragma unroll
        for (int i = 0; i < FN; i++) {
          const v4i p = *(const v4i*)(sw + u * WB + (i * 16 + fr) * 64 + (c ^ (fr >> 2)) * 16);
          float ws[NS];
#pragma unroll
          for (int k = 0; k < NS; k++) ws[k] = scales[wave][(s0 - w0 + u) * NS + k][i * 16 + fr];
#pragma unroll
          for (int j = 0; j < FT; j++) {
            v4i part[NS];
            i4_multiply<G>(xf[j], p, c, part);
#pragma unroll
            for (int k = 0; k < NS; k++)
#pragma unroll
              for (int q = 0; q < NI; q++) acc[i][j][q] = fmaf((float)part[k][q], ws[k], acc[i][j][q]);
          }
        }
      }
      wait_lds();  // this half is read
      if (s0 + 2 * U < end) fetch(s0 + 2 * U, half);
      half ^= 1;
    }
  }
  meet();  // (every wave's loads are done and read)
  float(*sums)[FN * FT * NI][64] = (float(*)[FN * FT * NI][64])lds;
#pragma unroll
  for (int i = 0; i < FN; i++)
#pragma unroll
    for (int j = 0; j < FT; j++)
#pragma unroll
      for (int q = 0; q < NI; q++) sums[wave][(i * FT + j) * NI + q][lane] = acc[i][j][q];
  wait_lds();
  meet();
  // a wave adds up every KW-th register of the squares
#pragma unroll
  for (int d = 0; d < DONE; d++) {
    const uint32_t r = wave + d * KW, sq = r / NI, t = r0 + sq % FT * 16 + 4 * (r % NI) + c, n = n0 + sq / FT * 16 + fr;
    if (r >= FN * FT * NI || t >= r1 || t >= r0 + BT || n >= a.n_out) continue;
    float sum = sums[0][r][lane];
#pragma unroll
    for (int k = 1; k < KW; k++) sum += sums[k][r][lane];
    i4_put(a, t, n, has[d] ? i4_finish(sum, fx[d], fb[d], a.relu) : 0.0f);
  }
}

// ------------------------------------------------------------ a few rows, quantized on the way
// The linear layer of at most 16 rows in one launch: each block asks for its first weights,
// quantizes all of x's rows into LDS while they come, and goes on as k_i4_wave with its x
// fragments from there.  Bound by the chain of x's maximum, its bytes and the product.
// That every block quantizes x again pays as long as all blocks run at once (two a CU) and x
// is small: at most 64 KB, 48 above 4096 channels, where a CU has two blocks.  One launch and
// two, bf16, on the GPU: 1 x 8192 to 1024 6.8 and 8.0 us, 8 x 4096 to 4096 9.6 and 7.6, 4 x 8192
// to 8192 14.5 and 10.5; a call from Python, to which a second launch is about 2.7 us: 9.7 and
// 12.6, 10.1 and 12.4, 14.6 and 12.2.  Over 312 sizes the rule's calls take 1% longer than the
// shorter of the two on the average, 21% at the most, their kernels 4 and 59% (16 x 2048 to
// 256), always one launch 3 and 81%, 13 and 117%.
constexpr uint32_t I4_FEW_OUT = 2 * 256 * 16, I4_FEW_X = 64 * 1024, I4_FEW_X_WIDE = 48 * 1024;

template <class X, int G, int NI>
__global__ __launch_bounds__(512) void k_i4_few(I4Args a, const X* __restrict__ x, size_t ld_x) {
  constexpr uint32_t KW = 8, U = 2, BN = 16, WB = BN * 64, OWN = 2 * U * WB;
  constexpr int NS = G >= 128 ? 1 : 128 / G;
  constexpr uint32_t ROWS = 16, W = ROWS / NS;
  extern __shared__ __align__(16) int8_t q[];  // rows x few_ld(n_in)
  __shared__ __align__(16) int8_t lds[KW * OWN];
  __shared__ float scales[KW][ROWS][BN];
  __shared__ uint32_t part[FEW_ROWS][KW];
  __shared__ float sx[FEW_ROWS];
  const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t n0 = blockIdx.x * BN, fr = lane & 15, c = lane >> 4, ld = few_ld(a.n_in);
  const uint32_t steps = (a.n_in + 127) / 128, per = (steps + KW - 1) / KW;
  const uint32_t first = wave * per, last = first + per < steps ? first + per : steps;
  const uint32_t wrow = n0 + (lane >> 2) < a.n_out ? n0 + (lane >> 2) : a.n_out - 1;
  const int8_t* wp = a.w + (size_t)wrow * a.ld_w + ((lane & 3) ^ (lane >> 4)) * 16;
  const int8_t* own = lds + wave * OWN;
  const uint32_t base = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) int8_t*)lds + wave * OWN;
  auto fetch = [&](uint32_t s, uint32_t half) {
#pragma unroll
    for (uint32_t u = 0; u < U; u++) {
      const uint32_t step = s + u < last ? s + u : last - 1;  // (again the last one, not used)
      load_to_lds(wp + (size_t)step * 64, base + (half * U + u) * WB);
    }
  };
  const uint32_t whole = G >= 128 ? a.group / 128 : 1;  // steps of a group
  uint32_t sc[4], end = 0;
  auto begin = [&](uint32_t w0) {
    end = w0 + W < last ? w0 + W : last;
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const uint32_t k = lane + i * 64, n = n0 + k % BN < a.n_out ? n0 + k % BN : a.n_out - 1;
      uint32_t g = w0 * NS + k / BN;
      if (G >= 128) g /= whole;
      if (g >= a.groups) g = a.groups - 1;  // (of a step's part behind the row's end, not used)
      sc[i] = scale_bits(a, (size_t)g * a.n_out + n);
    }
    fetch(w0, 0);
    if (w0 + U < end) fetch(w0 + U, 1);
  };
  if (first < last) begin(first);
  for (uint32_t i = threadIdx.x; i < a.rows * 128; i += 512) {  // behind the rows' ends
    const uint32_t k = (a.n_in - 1) / 128 * 128 + i % 128;
    if (k >= a.n_in) q[i / 128 * ld + k] = 0;
  }
  quantize_rows<X, KW>(x, ld_x, a.rows, a.n_in, q, ld, part, sx);
  // ---- the product
  const uint32_t token = NI < 4 ? fr >> 2 : (fr & 3) * 4 + (fr >> 2);
  const int8_t* xq = q + (token < a.rows ? token : a.rows - 1) * ld + 16 * c;
  float acc[NI] = {};
  for (uint32_t w0 = first; w0 < last; w0 += W) {
    if (w0 != first) begin(w0);
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const uint32_t k = lane + i * 64;
      scales[wave][k / BN][k % BN] = scale_of(a, sc[i]);
    }
    if (NS > 1 && end * NS > a.groups) zero_scales(&scales[wave][0][0], (a.groups - w0 * NS) * BN, ROWS * BN, lane);
    uint32_t half = 0;
    for (uint32_t s0 = w0; s0 < end; s0 += U) {
      if (s0 + U < end) wait_loads<U>();
      else wait_loads<0>();
      wait_lds();
#pragma unroll
      for (uint32_t u = 0; u < U; u++) {
        if (s0 + u >= end) break;
        v4i xf[2];
#pragma unroll
        for (int h = 0; h < 2; h++) xf[h] = *(const v4i*)(xq + (s0 + u) * 128 + 64 * h);
        const v4i p = *(const v4i*)(own + (half * U + u) * WB + fr * 64 + (c ^ (fr >> 2)) * 16);
        v4i sums[NS];
        i4_multiply<G>(xf, p, c, sums);
#pragma unroll
        for (int k = 0; k < NS; k++) {
          const float w = scales[wave][(s0 - w0 + u) * NS + k][fr];
#pragma unroll
          for (int i = 0; i < NI; i++) acc[i] = fmaf((float)sums[k][i], w, acc[i]);
        }
      }
      wait_lds();  // this half is read
      if (s0 + 2 * U < end) fetch(s0 + 2 * U, half);
      half ^= 1;
    }
  }
  meet();  // (every wave's loads are done and read)
  float(*sums)[NI][64] = (float(*)[NI][64])lds;
#pragma unroll
  for (int i = 0; i < NI; i++) sums[wave][i][lane] = acc[i];
  wait_lds();
  meet();
  const uint32_t t = 4 * wave + c, n = n0 + fr;
  if (wave >= NI || t >= a.rows || n >= a.n_out) return;
  float sum = sums[0][wave][lane];
#pragma unroll
  for (uint32_t k = 1; k < KW; k++) sum += sums[k][wave][lane];
  i4_put(a, t, n, i4_finish(sum, sx[t], a.bias ? a.bias[n] : 0.0f, a.relu));
}

static bool i4_few(size_t rows, size_t n_out, size_t n_in, int x_type) {
  return rows <= FEW_ROWS && n_in >= 16 && n_out <= I4_FEW_OUT && rows * few_ld((uint32_t)n_in) <= FEW_BYTES &&
         rows * n_in * type_bytes(x_type) <= (n_out > I4_FEW_OUT / 2 ? I4_FEW_X_WIDE : I4_FEW_X);
}

template <int G>
static int i4_launch_few(zk_context* ctx, const I4Args& a, const void* x, int x_type, size_t ld_x, hipStream_t st) {
  return by_type(x_type, [&](auto xz) -> int {
    typedef decltype(xz) X;
    const dim3 grid(cdiv(a.n_out, 16));
    const uint32_t lds = a.rows * few_ld(a.n_in);
    if (a.rows <= 4) ZK_LAUNCH(ctx, st, "i4_linear", (k_i4_few<X, G, 1>), grid, dim3(512), lds, a, (const X*)x, ld_x);
    else ZK_LAUNCH(ctx, st, "i4_linear", (k_i4_few<X, G, 4>), grid, dim3(512), lds, a, (const X*)x, ld_x);
    return ZK_OK;
  });
}

// ------------------------------------------------------------ many rows
// Eight neighbouring results of a row, of which it has `left` from here on.
template <class T>
__device__ __forceinline__ void put8(T* y, uint32_t left, const float (&v)[8]) {
  T r[8];
#pragma unroll
  for (int k = 0; k < 8; k++) r[k] = (T)v[k];
  if (left >= 8) {
#pragma unroll
    for (int k = 0; k < (int)sizeof(r) / 16; k++) ((row16*)y)[k] = ((const row16*)r)[k];
  } else {
#pragma unroll
    for (uint32_t k = 0; k < 7; k++)
      if (k < left) y[k] = r[k];
  }
}

// A block computes BT tokens x BN channels, its WT x WN waves a grid of FT x FN
// squares of 32 x 32 each (D's rows are tokens, its columns channels, so that a lane
// holds one channel's results and needs one scale).  Steps of 128 of k, a cache line of
// x's rows and half a one of w's, go straight from memory to LDS, into three stages: while one is
// multiplied the next is there and the one after under way.  Chunk c (16 bytes) of x's
// row r lies at c ^ (r / 2 % 8), of w's at c ^ (r / 4 % 4): the rows that a fragment
// reads together meet no bank twice.  w is unpacked in registers, once for the wave's FT
// squares; a group's integer sums become floats and go to the results with its scale,
// which is what bounds this kernel beside the matrix cores: 32 operations a square and
// group for four matrix instructions of a step.  Scales come through registers to LDS, four
// groups' at a time.  ODD: x's rows start at any byte or end inside a chunk; they come
// through registers, masked.  A call among others: 4096 rows, 8192 to 8192 293 us, 1.88 POPS
// (320 traced); 2048 tokens x 4 of 64 experts, 2048 to 1024 45 us (53).  777 rows, 4096 to
// 4096, groups of 64: 39 us traced.  The largest tiles have no register left: 4 of a lane's go
// to memory with groups of 128, 15 with 64, 22 with 32.
template <int G, bool GROUPED, bool ODD, int WT, int WN, int FT, int FN>
__global__ __launch_bounds__(64 * WT * WN, 2) void k_i4_ring(I4Args a, uint32_t tiles_t, uint32_t tiles_n) {
  constexpr uint32_t WAVES = WT * WN, THREADS = 64 * WAVES, BT = WT * FT * 32, BN = WN * FN * 32;
  constexpr uint32_t XB = BT * 128, WB = BN * 64, STAGE = XB + WB, STAGES = 3;
  constexpr uint32_t XR = BT / 8 / WAVES, WR = BN / 16 / WAVES;  // 1 KB pieces of a stage that a wave fills
  constexpr int LOADS = (ODD ? 0 : XR) + WR;                     // of them straight to LDS
  constexpr int NS = G >= 128 ? 1 : 128 / G;                     // scales of a step
  constexpr uint32_t ROWS = 4, W = ROWS / NS;                    // rows of scales, and steps, of a window
  constexpr uint32_t SR = ROWS * BN / THREADS;                   // scales of a window that a thread loads
  constexpr uint32_t LD = FN * 32 + 4, OWN = 32 * LD * 4;        // a wave's results of 32 tokens
  static_assert(WAVES * OWN + 4 * (2 * BT + BN) <= STAGES * STAGE, "the results' LDS is the stages'");
  static_assert(XR * 8 * WAVES == BT && WR * 16 * WAVES == BN && SR * THREADS == ROWS * BN, "whole pieces");
  static_assert(BN % 64 == 0, "a wave's scales are of one row");
  __shared__ __align__(16) int8_t lds[STAGES * STAGE];
  __shared__ float scales[2][ROWS][BN];
  const uint32_t tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  uint32_t r0, r1, n0, e;
  if (!block_tile<GROUPED>(a, BT, BN, tiles_t, tiles_n, r0, r1, n0, e)) return;
  const bool none = GROUPED && e >= a.experts;
  const size_t ch = none ? 0 : (size_t)e * a.n_out;
  const uint32_t steps = none ? 0 : (a.n_in + 127) / 128, full = a.n_in / 128;
  const uint32_t base = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) int8_t*)lds;
  // ---- what a lane fetches: a chunk of x's rows and one of w's.  NEAR: 32 bits from a
  // base that the block has in common.
  const int8_t* wbase = a.w + (ch + n0) * a.ld_w;
  const int8_t* xbase = GROUPED ? a.x : a.x + (size_t)r0 * a.ld_x;
  typedef std::conditional_t<ODD, const int8_t*, uint32_t> Place;
  Place xp[XR], wp[WR];
  auto x_chunk = [&](uint32_t i) { return ((lane & 7) ^ (((wave * XR + i) * 8 + (lane >> 3)) >> 1 & 7)) * 16; };
#pragma unroll
  for (uint32_t i = 0; i < WR; i++) {
    const uint32_t row = (wave * WR + i) * 16 + (lane >> 2), n = n0 + row < a.n_out ? row : a.n_out - 1 - n0;
    const size_t off = (size_t)n * a.ld_w + ((lane & 3) ^ (row >> 2 & 3)) * 16;
    if constexpr (ODD) wp[i] = wbase + off;
    else wp[i] = (uint32_t)off;
  }
  // rows of x: those that the lane fetches, and of the tokens whose scale it loads
  constexpr int TOKENS = (2 * BT + THREADS - 1) / THREADS;
  uint32_t place[XR + TOKENS];
  int from[XR + TOKENS];
#pragma unroll
  for (uint32_t i = 0; i < XR; i++) {
    const uint32_t r = r0 + (wave * XR + i) * 8 + (lane >> 3);
    place[i] = r < r1 ? r : r1 - 1;
  }
#pragma unroll
  for (uint32_t i = 0; i < TOKENS; i++) {
    const uint32_t r = r0 + (tid + i * THREADS) % BT;
    place[XR + i] = r < r1 ? r : r1 - 1;
  }
  source_rows<GROUPED>(a, place, from);
#pragma unroll
  for (uint32_t i = 0; i < XR; i++) {
    const size_t off = (size_t)(from[i] < 0 ? 0 : GROUPED ? (uint32_t)from[i] : from[i] - r0) * a.ld_x;
    if constexpr (ODD) xp[i] = xbase + off;
    else xp[i] = (uint32_t)off + x_chunk(i);
  }
  v4i held[ODD ? XR : 1];
  // LONG: a whole step.
  auto fetch = [&](auto is_long, uint32_t step, uint32_t stage) {
    constexpr bool LONG = decltype(is_long)::value;
    const uint32_t at = base + stage * STAGE;
    if constexpr (ODD) {
#pragma unroll
      for (uint32_t i = 0; i < XR; i++) {
        if (LONG || step < full) __builtin_memcpy(&held[i], xp[i] + step * 128 + x_chunk(i), 16);
        else held[i] = x_piece(xp[i], step * 128 + x_chunk(i), a.n_in);
      }
#pragma unroll
      for (uint32_t i = 0; i < WR; i++) load_to_lds(wp[i] + (size_t)step * 64, at + XB + (wave * WR + i) * 1024);
    } else {
      if (LONG || step < full) {
#pragma unroll
        for (uint32_t i = 0; i < XR; i++) load_to_lds(xbase + (size_t)step * 128, xp[i], at + (wave * XR + i) * 1024);
      } else {
        // chunks behind the row's end: its first one, to be cleared
#pragma unroll
        for (uint32_t i = 0; i < XR; i++) {
          const uint32_t c = x_chunk(i);
          load_to_lds(xbase, step * 128 + c < a.n_in ? xp[i] + step * 128 : xp[i] - c, at + (wave * XR + i) * 1024);
        }
      }
#pragma unroll
      for (uint32_t i = 0; i < WR; i++) load_to_lds(wbase + (size_t)step * 64, wp[i], at + XB + (wave * WR + i) * 1024);
    }
  };
  // (once the wave's own pieces of the last step, which is not a whole one, are there)
  auto clear_end = [&](uint32_t step, uint32_t stage) {
    if constexpr (!ODD) {
#pragma unroll
      for (uint32_t i = 0; i < XR; i++)
        if (step * 128 + x_chunk(i) >= a.n_in)
          *(v4i*)(lds + stage * STAGE + (wave * XR + i) * 1024 + lane * 16) = v4i{0, 0, 0, 0};
    }
  };
  auto put_held = [&](uint32_t stage) {
    if constexpr (ODD) {
#pragma unroll
      for (uint32_t i = 0; i < XR; i++) *(v4i*)(lds + stage * STAGE + (wave * XR + i) * 1024 + lane * 16) = held[i];
    }
  };
  uint32_t sc[SR];
  const uint32_t whole = G >= 128 ? a.group / 128 : 1;  // steps of a group
  auto fetch_scales = [&](uint32_t window) {
#pragma unroll
    for (uint32_t i = 0; i < SR; i++) {
      const uint32_t k = tid + i * THREADS, n = n0 + k % BN < a.n_out ? n0 + k % BN : a.n_out - 1;
      uint32_t g = window * ROWS + k / BN;
      if (G >= 128) g /= whole;
      if (g >= a.groups) g = a.groups - 1;  // (of a step's part behind the row's end, not used)
      sc[i] = scale_bits(a, ch * a.groups + (size_t)g * a.n_out + n);
    }
  };
  // INSIDE: all its steps are whole.
  auto put_scales = [&](auto is_inside, uint32_t window) {
    constexpr bool INSIDE = decltype(is_inside)::value;
#pragma unroll
    for (uint32_t i = 0; i < SR; i++) {
      const uint32_t k = tid + i * THREADS;
      // (a wave's are of one row)
      const uint32_t g = window * ROWS + __builtin_amdgcn_readfirstlane(k / BN);
      scales[window & 1][k / BN][k % BN] = scale_of_group<INSIDE ? 1 : NS>(a, sc[i], g);
    }
  };
  // the results' factors, a few for each thread, there when they are needed
  constexpr uint32_t FACTORS = (2 * BT + BN + THREADS - 1) / THREADS;
  float factor[FACTORS];
#pragma unroll
  for (uint32_t i = 0; i < FACTORS; i++) {
    const uint32_t k = tid + i * THREADS;
    factor[i] = 0.0f;
    if (k < 2 * BT) {  // tokens' scales, and whether they are there
      const int from_k = from[XR + (i < TOKENS ? i : 0)];
      const bool in = r0 + k % BT < r1 && !none && from_k >= 0;
      factor[i] = !in ? 0.0f : k < BT && a.sx ? a.sx[from_k] : 1.0f;
    } else if (k < 2 * BT + BN) {
      const uint32_t n = n0 + k - 2 * BT;
      factor[i] = a.bias && n < a.n_out ? a.bias[ch + n] : 0.0f;
    }
  }
  // ---- where a lane reads its fragments
  const uint32_t wave_t = wave % WT, wave_n = wave / WT, fr = lane & 31, hi = lane >> 5;
  const int8_t* fx = lds + (wave_t * FT * 32 + fr) * 128;
  const int8_t* fw = lds + XB + (wave_n * FN * 32 + fr) * 64;
  uint32_t cx[4], cw[2];
#pragma unroll
  for (uint32_t s = 0; s < 4; s++) cx[s] = ((2 * s + hi) ^ (fr >> 1 & 7)) * 16;
#pragma unroll
  for (uint32_t s = 0; s < 2; s++) cw[s] = ((2 * s + hi) ^ (fr >> 2 & 3)) * 16;
  // A step's units, their matrix instructions, and whether a step's last unit is left
  // to the next step.
  constexpr int UNITS = FN * FT * NS, M = 4 / NS;
  constexpr bool DEFER = UNITS % 2 == 0;
  float acc[FN][FT][16] = {}, last = 0.0f;
  v16i part[2] = {};
  auto add_last = [&] {
#pragma unroll
    for (int r = 0; r < 16; r++)
      acc[FN - 1][FT - 1][r] = fmaf((float)part[(UNITS - 1) & 1][r], last, acc[FN - 1][FT - 1][r]);
  };
  // Stage of step s, in its slot, becomes every wave's to read: its pieces are in, those
  // of the other waves too, and all have read the stage before the last; the one after the
  // next is asked for in that one's place.
  auto up = [](uint32_t slot) { return slot + 1 < STAGES ? slot + 1 : 0; };
  auto turn = [&](auto is_long, uint32_t s, uint32_t slot) {
    constexpr bool LONG = decltype(is_long)::value;
    if (LONG || s + 1 < steps) put_held(up(slot));
    if (s % W == 0) put_scales(std::bool_constant<LONG && W <= 2>(), s / W);  // (LONG: s + 2 is whole)
    if (LONG || s + 1 < steps) wait_loads<LOADS>();
    else wait_loads<0>();
    if (!LONG && s >= full) clear_end(s, slot);
    wait_lds();
    meet();
    if (s % W == 0 && s + W < steps) fetch_scales(s / W + 1);
    if (LONG || s + 2 < steps) fetch(is_long, s + 2, up(up(slot)));
  };
  if (steps) {
    fetch_scales(0);
    fetch(std::false_type(), 0, 0);
    put_held(0);
    if (steps > 1) fetch(std::false_type(), 1, 1);
    uint32_t slot = 0;
    auto run = [&](auto is_long, uint32_t step) {
      turn(is_long, step, slot);
      const int8_t *sx = fx + slot * STAGE, *sw = fw + slot * STAGE;
      v4i wf[FN][4], xf[4];
      float ws[FN][NS];
#pragma unroll
      for (int q = 0; q < 4; q++) xf[q] = *(const v4i*)(sx + cx[q]);
#pragma unroll
      for (int i = 0; i < FN; i++) {
#pragma unroll
        for (int q = 0; q < 2; q++) {
          const v4i p = *(const v4i*)(sw + i * 32 * 64 + cw[q]);
          wf[i][q] = (p << 4) & (int)0xf0f0f0f0;
          wf[i][q + 2] = p & (int)0xf0f0f0f0;
        }
#pragma unroll
        for (int k = 0; k < NS; k++)
          ws[i][k] = scales[step / W & 1][step % W * NS + k][wave_n * FN * 32 + i * 32 + fr];
      }
      // unit u: square u / NS, its group u % NS; the sums of the unit before go to the
      // results between this one's matrix instructions
#pragma unroll
      for (int u = 0; u < UNITS; u++) {
        const int j = u / NS / FN, i = u / NS % FN, k = u % NS;
#pragma unroll
        for (int m = 0; m < M; m++) {
          const int q = k * M + m;
          const v16i zero = {};
          part[u & 1] = __builtin_amdgcn_mfma_i32_32x32x32_i8(xf[q], wf[i][q], m ? part[u & 1] : zero, 0, 0, 0);
          // (the fragment's last use: the next tokens' takes its place)
          if (i == FN - 1 && j + 1 < FT) xf[q] = *(const v4i*)(sx + (j + 1) * 32 * 128 + cx[q]);
          __builtin_amdgcn_sched_barrier(0);
          if (u || DEFER) {
            const int v = u ? u - 1 : UNITS - 1;
            const float w = u ? ws[v / NS % FN][v % NS] : last;
            // (not after the first, whose turn the sums before are not there yet)
            constexpr int SHARE = M > 1 ? M - 1 : 1;
            const int lo = M == 1 || m == 0 ? 0 : (m - 1) * 16 / SHARE, to = M == 1 ? 16 : m * 16 / SHARE;
#pragma unroll
            for (int r = 0; r < 16; r++)
              if (r >= lo && r < to)
                acc[v / NS % FN][v / NS / FN][r] = fmaf((float)part[v & 1][r], w, acc[v / NS % FN][v / NS / FN][r]);
          }
          __builtin_amdgcn_sched_barrier(0);
        }
      }
      last = ws[FN - 1][NS - 1];
      if (!DEFER) add_last();
      slot = up(slot);
    };
    uint32_t step = 0;
    if constexpr (FT * FN < 8)  // (the largest squares' registers do not suffice for two loops)
      for (; step + 2 < full; step++) run(std::true_type(), step);
    for (; step < steps; step++) run(std::false_type(), step);
    if (DEFER) add_last();
  }
  // ---- results: a wave's 32 tokens at a time, by way of its own LDS
  wait_lds();
  meet();
  float* f = (float*)(lds + WAVES * OWN);
#pragma unroll
  for (uint32_t i = 0; i < FACTORS; i++)
    if (tid + i * THREADS < 2 * BT + BN) f[tid + i * THREADS] = factor[i];
  wait_lds();
  meet();
  float* own = (float*)(lds + wave * OWN);
  constexpr uint32_t PIECES = FN * 4, PER = 64 / PIECES;  // of eight channels in a row; rows of one store
  const uint32_t c = lane % PIECES * 8, n = n0 + wave_n * FN * 32 + c;
  float bias[8];
#pragma unroll
  for (int k = 0; k < 8; k++) bias[k] = f[2 * BT + wave_n * FN * 32 + c + k];
#pragma unroll
  for (int j = 0; j < FT; j++) {
#pragma unroll
    for (int i = 0; i < FN; i++)
#pragma unroll
      for (int r = 0; r < 16; r++) own[(8 * (r / 4) + 4 * hi + r % 4) * LD + i * 32 + fr] = acc[i][j][r];
    wait_lds();  // one wave's LDS accesses are in order; this keeps the compiler to it
#pragma unroll 1
    for (uint32_t s = 0; s < 32; s += PER) {
      const uint32_t row = s + lane / PIECES, tt = wave_t * FT * 32 + j * 32 + row, t = r0 + tt;
      if (t < r1 && n < a.n_out) {
        float v[8];
        const float sx = f[tt], has = f[BT + tt];
#pragma unroll
        for (int k = 0; k < 8; k++)
          v[k] = has != 0.0f ? i4_finish(own[row * LD + c + k], sx, bias[k], a.relu) : 0.0f;
        const size_t at = (size_t)t * a.ld_y + n;
        if (a.y_type == ZK_F32) put8((float*)a.y + at, a.n_out - n, v);
        else if (a.y_type == ZK_F16) put8((_Float16*)a.y + at, a.n_out - n, v);
        else put8((__bf16*)a.y + at, a.n_out - n, v);
      }
    }
    wait_lds();
  }
}

// ------------------------------------------------------------ which kernel
// A product's time in ns: that of its first tile on a CU, and of each more, both with a
// part for every step of 128 of k (fitted to products of 1 to 4096 rows, 128 to 8192 long,
// and to 2 to 6400 rows of 8 to 64 experts; the rule's choices took 2, 2.5 and 3% longer
// than the best of all on the average, 27% at the most).  Rows of x of whole chunks, at any
// byte, and grouped by expert; 0: not a choice.  Those forms were measured too, and won little:
// 4 x 32 not grouped at one size in 72, by 7%; grouped, the 16 x 16, 32 x 32 and 48 x 32 at none
// of 40, 256 x 256 at one, by 8%.  Smaller groups lengthen a step.
struct I4Cost {
  uint32_t first, step, more, more_step;
};
struct I4Tile {
  const char* name;
  uint32_t bt, bn;
  I4Cost whole, odd, grouped;
  uint32_t step64, step32;  // percent of a step with groups of 64 and 32
};
enum I4Kernel { I4_4x16, I4_4x32, I4_16x16, I4_16x32, I4_32x32, I4_48x32, I4_32x128, I4_64x128, I4_256, I4_COUNT };
constexpr I4Tile I4_TILES[I4_COUNT] = {
    {"wave 4x16", 4, 16, {3866, 18, 846, 21}, {3681, 34, 810, 26}, {4541, 5, 1260, 23}, 100, 110},
    {"wave 4x32", 4, 32, {}, {}, {4680, 44, 800, 40}, 100, 110},
    {"wave 16x16", 16, 16, {4164, 30, 1896, 41}, {4215, 66, 2237, 67}, {}, 105, 130},
    {"wave 16x32", 16, 32, {4468, 88, 491, 44}, {4404, 129, 393, 64}, {5568, 44, 552, 57}, 105, 130},
    {"wave 32x32", 32, 32, {4757, 79, 3039, 76}, {5149, 125, 3493, 122}, {}, 105, 130},
    {"wave 48x32", 48, 32, {5101, 98, 3758, 96}, {5731, 167, 4720, 156}, {}, 105, 130},
    {"stages 32x128", 32, 128, {4453, 451, 756, 145}, {4514, 505, 1157, 154}, {4874, 457, 993, 186}, 155, 200},
    {"stages 64x128", 64, 128, {5150, 537, 2169, 282}, {5432, 617, 2748, 336}, {5764, 542, 74, 378}, 135, 175},
    {"stages 256x256", 256, 256, {12066, 1852, 21966, 2325}, {}, {}, 160, 290},
};

// Whether x's rows are in whole chunks of 16 bytes, and, for the stages, a block's rows
// within 32 bits of one another.
static bool whole_rows(const I4Args& a) { return (((uintptr_t)a.x | a.ld_x | a.n_in) & 15) == 0; }
static bool near_rows(const I4Args& a, bool grouped) {
  return !(a.ld_w >> 23) && !(a.ld_x >> 23) && (!grouped || !((uint64_t)a.tokens * a.ld_x >> 32));
}

// Row tiles.  Of the grouped form: whole ones, and a part of one for each expert and for
// the rows without an expert.
static uint32_t row_tiles(const I4Args& a, uint32_t bt, bool grouped) {
  return grouped ? a.rows / bt + (a.experts + 1 < a.rows ? a.experts + 1 : a.rows) : cdiv(a.rows, bt);
}

static I4Kernel choose_i4(const I4Args& a, bool grouped) {
  const bool whole = whole_rows(a), near = near_rows(a, grouped);
  const uint64_t steps = (a.n_in + 127) / 128, groups = grouped ? (a.experts < a.rows ? a.experts : a.rows) : 0;
  I4Kernel best = I4_4x16;
  uint64_t least = ~0ull;
  for (int i = 0; i < I4_COUNT; i++) {
    const I4Tile& t = I4_TILES[i];
    const I4Cost& c = grouped ? t.grouped : whole && (near || i < I4_32x128) ? t.whole : t.odd;
    if (!c.first || (uint64_t)row_tiles(a, t.bt, grouped) * cdiv(a.n_out, t.bn) > I8_MAX_TILES) continue;
    // an expert's last row tile is half full, or it has only one
    uint64_t tt = cdiv(a.rows, t.bt);
    if (grouped && (tt += groups / 2) < groups) tt = groups;
    const uint64_t tiles = tt * cdiv(a.n_out, t.bn), more = tiles > 256 ? tiles - 256 : 0;
    const uint64_t k = steps * (a.group == 32 ? t.step32 : a.group == 64 ? t.step64 : 100);
    const uint64_t time = c.first + c.step * k / 100 + (c.more * more + c.more_step * k / 100 * more) / 256;
    if (time < least) least = time, best = (I4Kernel)i;
  }
  return best;
}

template <int G, bool GROUPED, bool ODD>
static int launch_i4_as(zk_context* ctx, const I4Args& a, I4Kernel k, hipStream_t st) {
  auto go = [&](auto kernel, uint32_t threads) -> int {
    const uint32_t tiles_t = row_tiles(a, I4_TILES[k].bt, GROUPED);
    const uint32_t tiles_n = cdiv(a.n_out, I4_TILES[k].bn);
    const size_t tiles = (size_t)tiles_t * tiles_n;
    if (tiles > I8_MAX_TILES) return ctx->fail(ZK_ERR_SIZE, "i4 product: rows and n_out make too many tiles");
    ZK_LAUNCH(ctx, st, GROUPED ? "i4_matmul_experts" : "i4_matmul", kernel, dim3(cdiv(tiles, 8) * 8), dim3(threads), 0,
              a, tiles_t, tiles_n);
    return ZK_OK;
  };
  if (k == I4_4x16) return go(k_i4_wave<G, GROUPED, ODD, 1, 1, 1, 8, 2>, 512);
  if (k == I4_16x32) return go(k_i4_wave<G, GROUPED, ODD, 1, 2, 4, 4, 1>, 256);
  if (k == I4_32x128) return go(k_i4_ring<G, GROUPED, ODD, 1, 4, 1, 1>, 256);
  if (k == I4_64x128) return go(k_i4_ring<G, GROUPED, ODD, 1, 4, 2, 1>, 256);
  if constexpr (GROUPED) {
    if (k == I4_4x32) return go(k_i4_wave<G, true, ODD, 1, 2, 1, 4, 2>, 256);
  } else {
    if (k == I4_16x16) return go(k_i4_wave<G, false, ODD, 1, 1, 4, 8, 2>, 512);
    if (k == I4_32x32) return go(k_i4_wave<G, false, ODD, 2, 2, 4, 8, 1>, 512);
    if (k == I4_48x32) return go(k_i4_wave<G, false, ODD, 3, 2, 4, 8, 1>, 512);
    if constexpr (!ODD)
      if (k == I4_256) return go(k_i4_ring<G, false, false, 2, 4, 4, 2>, 512);
  }
  return ctx->fail(ZK_ERR_INVALID, "i4 product: no kernel");
}

template <bool GROUPED>
static int i4_dispatch(zk_context* ctx, const I4Args& a, hipStream_t st) {
  const I4Kernel k = choose_i4(a, GROUPED);
  const bool odd = !whole_rows(a) || (k >= I4_32x128 && !near_rows(a, GROUPED));
  auto by_odd = [&](auto g) -> int {
    constexpr int G = decltype(g)::value;
    return odd ? launch_i4_as<G, GROUPED, true>(ctx, a, k, st) : launch_i4_as<G, GROUPED, false>(ctx, a, k, st);
  };
  if (a.group == 32) return by_odd(std::integral_constant<int, 32>());
  if (a.group == 64) return by_odd(std::integral_constant<int, 64>());
  return by_odd(std::integral_constant<int, 128>());
}

// ------------------------------------------------------------ weights to 4 bits
// s = a / 7 rounded to the scales' type, a = max|w| over the group; q = the integer
// nearest to w / s (ties to even), at most 7 and at least -8 (s may have been rounded
// down).  A group of zeros has s = 0 and zeros, one that holds an infinity or a NaN
// s = NaN and zeros.  Padding is zero.  Eight lanes have one run of 128 weights (small
// groups), or a whole group of them, and load sixteen neighbours each: a byte's two
// weights lie 64 apart.  Done once for a model; bound by memory and the scales' scattered
// stores: 8192 x 8192 bf16 54 us, 3.1 TB/s (192 with a wave for a run, one weight of each
// half a lane).
template <class T, class S>
__global__ __launch_bounds__(256) void k_i4_quantize(const T* __restrict__ w, size_t ld_w, uint32_t rows,
                                                     uint32_t cols, uint32_t group, uint32_t groups, uint32_t units,
                                                     int8_t* __restrict__ q, size_t ld_q, S* __restrict__ scale) {
  constexpr uint32_t N = Vec<T>::N;
  const uint32_t l = threadIdx.x & 7;
  const uint64_t all = (uint64_t)rows * units, stride = (uint64_t)gridDim.x * 32;
  for (uint64_t i = (uint64_t)blockIdx.x * 32 + (threadIdx.x >> 3); i < all; i += stride) {
    const uint32_t r = (uint32_t)(i / units), u = (uint32_t)(i % units);
    const T* row = w + (size_t)r * ld_w;
    const uint32_t run = group < 128 ? 128 : group, k0 = u * run, end = k0 + run < cols ? k0 + run : cols;
    float v[2][8];
    auto load = [&](uint32_t k) {
#pragma unroll
      for (int h = 0; h < 2; h++)
#pragma unroll
        for (uint32_t c = 0; c < 8 / N; c++) {
          const uint32_t at = k + 64 * h + 8 * l + c * N;
          const Vec<T> x = at < end ? row_load(row + at, end - at) : Vec<T>{};
#pragma unroll
          for (uint32_t j = 0; j < N; j++) v[h][c * N + j] = (float)x.v[j];
        }
    };
    // magnitudes as integers, in the floats' order, NaN above infinity
    uint32_t m[2] = {0, 0};
    for (uint32_t k = k0; k < end; k += 128) {
      load(k);
#pragma unroll
      for (int h = 0; h < 2; h++)
#pragma unroll
        for (int j = 0; j < 8; j++) {
          const uint32_t b = __float_as_uint(v[h][j]) & 0x7fffffffu;
          m[h] = b > m[h] ? b : m[h];
        }
    }
    if (group > 64) m[0] = m[1] = m[0] > m[1] ? m[0] : m[1];
    for (uint32_t d = group < 64 ? 2 : 4; d; d >>= 1)
#pragma unroll
      for (int h = 0; h < 2; h++) {
        const uint32_t o = (uint32_t)__shfl_xor((int)m[h], (int)d);
        m[h] = o > m[h] ? o : m[h];
      }
    float s[2];
#pragma unroll
    for (int h = 0; h < 2; h++) {
      const S rounded = m[h] >= 0x7f800000u ? (S)NAN : (S)(__uint_as_float(m[h]) / 7.0f);
      s[h] = (float)rounded;
      const uint32_t k = k0 + 64 * h + 8 * l, g = k / group;
      // the group's first lane writes its scale
      if (g < groups && k % group == 0) scale[(size_t)g * rows + r] = rounded;
    }
    for (uint32_t k = k0; k < end; k += 128) {
      if (group > 128) load(k);
      uint32_t packed[2] = {0, 0};
#pragma unroll
      for (int h = 0; h < 2; h++)
#pragma unroll
        for (int j = 0; j < 8; j++) {
          float f = s[h] > 0.0f && m[h] < 0x7f800000u ? rintf(v[h][j] / s[h]) : 0.0f;
          f = f > 7.0f ? 7.0f : f < -8.0f ? -8.0f : f;
          packed[j / 4] |= ((uint32_t)(int)f & 15) << (j % 4 * 8 + 4 * h);
        }
      *(uint2*)(q + (size_t)r * ld_q + k / 2 + 8 * l) = make_uint2(packed[0], packed[1]);
    }
  }
}

// ------------------------------------------------------------ arguments
static bool group_size(int group) { return group == 32 || group == 64 || (group >= 128 && group % 128 == 0); }

static int check_group(zk_context* ctx, size_t n_in, int group) {
  if (!group_size(group))
    return ctx->fail(ZK_ERR_INVALID, "i4: a group is 32, 64 or a multiple of 128 weights");
  if (n_in > I4_MAX_IN) return ctx->fail(ZK_ERR_SIZE, "i4: rows longer than 2^24");
  return ZK_OK;
}

static int check_i4(zk_context* ctx, const I4Args& a, size_t rows, size_t n_out, size_t n_in, int group, int scale_type,
                    int type, bool reads_x = true) {
  ZK_TRY(check_group(ctx, n_in, group));
  if (!float_type(type)) return ctx->fail(ZK_ERR_INVALID, "i4 product: y is f32, f16 or bf16");
  if (!float_type(scale_type)) return ctx->fail(ZK_ERR_INVALID, "i4 product: scales are f32, f16 or bf16");
  if (rows > 0x7fffffffu || n_out > 16 * I8_MAX_TILES)
    return ctx->fail(ZK_ERR_SIZE, "i4 product: more than 2^31 - 1 rows or 2^26 channels");
  if (a.ld_x < n_in || a.ld_w < i4_row_bytes(n_in) || a.ld_y < n_out)
    return ctx->fail(ZK_ERR_INVALID, "i4 product: a row stride below the row's length");
  if (rows && n_out && (!a.y || (n_in && ((!a.x && reads_x) || !a.w || !a.scale))))
    return ctx->fail(ZK_ERR_INVALID, "i4 product: null pointer");
  if (!aligned(a.w, 16) || a.ld_w % 16)
    return ctx->fail(ZK_ERR_INVALID, "i4 product: weights' rows start at multiples of 16 bytes");
  if (!aligned(a.y, type_bytes(type)) || !aligned(a.sx, 4) || !aligned(a.scale, type_bytes(scale_type)) ||
      !aligned(a.bias, 4))
    return ctx->fail(ZK_ERR_INVALID, "i4 product: a pointer is not aligned to its type");
  return ZK_OK;
}

static void set_sizes(I4Args& a, size_t rows, size_t n_out, size_t n_in, int group, int relu, int scale_type,
                      int type) {
  a.scale_type = scale_type, a.y_type = type;
  a.rows = (uint32_t)rows, a.n_out = (uint32_t)n_out, a.n_in = (uint32_t)n_in, a.relu = relu != 0;
  a.group = (uint32_t)group, a.groups = cdiv(n_in, group);
}

static int i4_matmul(zk_context* ctx, const I4Args& a, hipStream_t st) {
  // rows in runs of at most I8_MAX_TILES tiles of 16 x 16
  const size_t most = I8_MAX_TILES / cdiv(a.n_out, 16) * 16;
  for (size_t r = 0; r < a.rows; r += most) {
    I4Args b = a;
    b.rows = (uint32_t)(a.rows - r < most ? a.rows - r : most);
    b.x = a.x ? a.x + r * a.ld_x : a.x;
    b.sx = a.sx ? a.sx + r : a.sx;
    b.y = (uint8_t*)a.y + r * a.ld_y * type_bytes(a.y_type);
    ZK_TRY(i4_dispatch<false>(ctx, b, st));
  }
  return ZK_OK;
}

}  // namespace zk

extern "C" {

size_t zk_i4_row_bytes(size_t n_in) { return n_in > zk::I4_MAX_IN ? 0 : zk::i4_row_bytes(n_in); }

int zk_i4_quantize(zk_context* ctx, const void* d_w, int w_type, size_t ld_w, size_t rows, size_t cols, int group,
                   void* d_q, size_t ld_q, void* d_scale, int scale_type, void* stream) {
  using namespace zk;
  if (!ctx) return ZK_ERR_INVALID;
  return guard(ctx, [&]() -> int {
    ZK_TRY(check_group(ctx, cols, group));
    if (!float_type(w_type) || !float_type(scale_type))
      return ctx->fail(ZK_ERR_INVALID, "i4 quantize: weights and scales are f32, f16 or bf16");
    if (rows > 0x7fffffffu) return ctx->fail(ZK_ERR_SIZE, "i4 quantize: more than 2^31 - 1 rows");
    if (ld_w < cols || ld_q < i4_row_bytes(cols))
      return ctx->fail(ZK_ERR_INVALID, "i4 quantize: a row stride below the row's length");
    if (!aligned(d_q, 16) || ld_q % 16)
      return ctx->fail(ZK_ERR_INVALID, "i4 quantize: weights' rows start at multiples of 16 bytes");
    if (!rows || !cols) return ZK_OK;
    if (!d_w || !d_q || !d_scale) return ctx->fail(ZK_ERR_INVALID, "i4 quantize: null pointer");
    if (!aligned(d_w, type_bytes(w_type)) || !aligned(d_scale, type_bytes(scale_type)))
      return ctx->fail(ZK_ERR_INVALID, "i4 quantize: a pointer is not aligned to its type");
    OnDevice on(ctx);
    hipStream_t st = ctx->s(stream);
    const uint32_t units = cdiv(cols, group < 128 ? 128 : group);
    const size_t blocks = (rows * units + 31) / 32;
    return by_type(w_type, [&](auto wz) -> int {
      return by_type(scale_type, [&](auto sz) -> int {
        typedef decltype(wz) T;
        typedef decltype(sz) S;
        ZK_LAUNCH(ctx, st, "i4_quantize", (k_i4_quantize<T, S>), dim3(blocks < 65536 ? (uint32_t)blocks : 65536),
                  dim3(256), 0, (const T*)d_w, ld_w, (uint32_t)rows, (uint32_t)cols, (uint32_t)group,
                  cdiv(cols, group), units, (int8_t*)d_q, ld_q, (S*)d_scale);
        return ZK_OK;
      });
    });
  });
}

int zk_i4_matmul(zk_context* ctx, const int8_t* d_x, size_t ld_x, const float* d_x_scale, const void* d_w, size_t ld_w,
                 const void* d_w_scale, int scale_type, int group, const float* d_bias, size_t rows, size_t n_out,
                 size_t n_in, int relu, void* d_y, int y_type, size_t ld_y, void* stream) {
  using namespace zk;
  if (!ctx) return ZK_ERR_INVALID;
  return guard(ctx, [&]() -> int {
    I4Args a = {};
    a.x = d_x, a.w = (const int8_t*)d_w, a.sx = d_x_scale, a.scale = d_w_scale, a.bias = d_bias, a.y = d_y;
    a.ld_x = ld_x, a.ld_w = ld_w, a.ld_y = ld_y;
    ZK_TRY(check_i4(ctx, a, rows, n_out, n_in, group, scale_type, y_type));
    if (!rows || !n_out) return ZK_OK;
    set_sizes(a, rows, n_out, n_in, group, relu, scale_type, y_type);
    OnDevice on(ctx);
    return i4_matmul(ctx, a, ctx->s(stream));
  });
}

const char* zk_debug_i4_kernel(size_t rows, size_t n_out, size_t n_in, size_t ld_x, size_t address, int group,
                               int experts) {
  using namespace zk;
  if (!rows || !n_out || rows > 0x7fffffffu || n_out > 16 * I8_MAX_TILES || n_in > I4_MAX_IN || experts < 0 ||
      !group_size(group))
    return nullptr;
  I4Args a = {};
  a.x = (const int8_t*)address, a.ld_x = ld_x, a.ld_w = i4_row_bytes(n_in);
  set_sizes(a, rows, n_out, n_in, group, 0, ZK_F32, ZK_F32);
  a.experts = (uint32_t)experts, a.tokens = a.rows;
  return I4_TILES[choose_i4(a, experts > 0)].name;
}

size_t zk_i4_linear_work(size_t rows, size_t n_in) {
  if (rows > 0x7fffffffu || n_in > zk::I4_MAX_IN) return 0;
  return zk::linear_work(rows, n_in).bytes;
}

int zk_i4_linear(zk_context* ctx, const void* d_x, int x_type, size_t ld_x, const void* d_w, size_t ld_w,
                 const void* d_w_scale, int scale_type, int group, const float* d_bias, size_t rows, size_t n_out,
                 size_t n_in, int relu, void* d_y, int y_type, size_t ld_y, void* d_work, size_t work_bytes,
                 void* stream) {
  using namespace zk;
  if (!ctx) return ZK_ERR_INVALID;
  return guard(ctx, [&]() -> int {
    ZK_TRY(check_quantize(ctx, d_x, x_type, ld_x, rows, n_in));
    ZK_TRY(check_group(ctx, n_in, group));
    const LinearWork lw = linear_work(rows, n_in);
    I4Args a = {};
    a.x = (const int8_t*)d_work + lw.q, a.w = (const int8_t*)d_w, a.sx = (const float*)d_work, a.scale = d_w_scale;
    a.bias = d_bias, a.y = d_y;
    a.ld_x = lw.ld, a.ld_w = ld_w, a.ld_y = ld_y;
    ZK_TRY(check_i4(ctx, a, rows, n_out, n_in, group, scale_type, y_type));
    if (!rows || !n_out) return ZK_OK;
    if (!d_work || !aligned(d_work, 16) || work_bytes < lw.bytes)
      return ctx->fail(ZK_ERR_INVALID, "i4 linear: workspace missing, too small or not aligned to 16 bytes");
    set_sizes(a, rows, n_out, n_in, group, relu, scale_type, y_type);
    OnDevice on(ctx);
    hipStream_t st = ctx->s(stream);
    if (i4_few(rows, n_out, n_in, x_type)) {
      if (group == 32) return i4_launch_few<32>(ctx, a, d_x, x_type, ld_x, st);
      if (group == 64) return i4_launch_few<64>(ctx, a, d_x, x_type, ld_x, st);
      return i4_launch_few<128>(ctx, a, d_x, x_type, ld_x, st);
    }
    ZK_TRY(i8_quantize(ctx, d_x, x_type, ld_x, rows, n_in, (int8_t*)d_work + lw.q, lw.ld, (float*)d_work, st));
    return i4_matmul(ctx, a, st);
  });
}

int zk_i4_matmul_experts(zk_context* ctx, const int8_t* d_x, size_t ld_x, const float* d_x_scale, size_t tokens,
                         const void* d_w, size_t ld_w, const void* d_w_scale, int scale_type, int group,
                         const float* d_bias, const int32_t* d_offsets, int experts, const int32_t* d_order, int slots,
                         size_t rows, size_t n_out, size_t n_in, int relu, void* d_y, int y_type, size_t ld_y,
                         void* stream) {
  using namespace zk;
  if (!ctx) return ZK_ERR_INVALID;
  return guard(ctx, [&]() -> int {
    I4Args a = {};
    a.x = d_x, a.w = (const int8_t*)d_w, a.sx = d_x_scale, a.scale = d_w_scale, a.bias = d_bias, a.y = d_y;
    a.ld_x = ld_x, a.ld_w = ld_w, a.ld_y = ld_y;
    if (experts < 1 || experts > ZK_MAX_EXPERTS)
      return ctx->fail(ZK_ERR_SIZE, "i4 experts: between 1 and 1024 experts");
    if (slots < 1) return ctx->fail(ZK_ERR_INVALID, "i4 experts: slots is at least 1");
    ZK_TRY(check_i4(ctx, a, rows, n_out, n_in, group, scale_type, y_type, tokens > 0));
    if (rows > ZK_MAX_EXPERT_ROWS || tokens > 0x7fffffffu)
      return ctx->fail(ZK_ERR_SIZE, "i4 experts: too many rows");
    if (!rows || !n_out) return ZK_OK;
    if (!d_offsets) return ctx->fail(ZK_ERR_INVALID, "i4 experts: null pointer");
    if (!aligned(d_offsets, 4) || !aligned(d_order, 4))
      return ctx->fail(ZK_ERR_INVALID, "i4 experts: a pointer is not aligned to its type");
    set_sizes(a, rows, n_out, n_in, group, relu, scale_type, y_type);
    a.offsets = d_offsets, a.order = d_order, a.experts = (uint32_t)experts, a.slots = (uint32_t)slots;
    a.tokens = (uint32_t)tokens;
    OnDevice on(ctx);
    if (!tokens) {
      const size_t blocks = (rows * n_out + 255) / 256;
      return by_type(y_type, [&](auto zero) -> int {
        ZK_LAUNCH(ctx, ctx->s(stream), "i4_matmul_experts", k_i4_zeros<decltype(zero)>,
                  dim3(blocks < 65536 ? (uint32_t)blocks : 65536), dim3(256), 0, (decltype(zero)*)d_y, ld_y, a.rows,
                  a.n_out);
        return ZK_OK;
      });
    }
    return i4_dispatch<true>(ctx, a, ctx->s(stream));
  });
}

}  // extern "C"
