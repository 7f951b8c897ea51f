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
};

static __host__ __device__ inline size_t i4_row_bytes(size_t n_in) { return (n_in + 127) / 128 * 64; }

// Weight k of a packed row.
__device__ __forceinline__ int weight_at(const int8_t* row, uint32_t k) {
  const int b = row[(k >> 7) * 64 + (k & 63)];
  return k & 64 ? b >> 4 : (int)((uint32_t)b << 28) >> 28;
}

// sx sum + b in one rounding; what is below zero becomes zero, a NaN stays.
__device__ __forceinline__ float i4_finish(float sum, float sx, float b, int relu) {
  const float f = fmaf(sum, sx, b);
  return relu && f < 0.0f ? 0.0f : f;
}

// A thread takes one result at a time.
template <class T, class S, bool GROUPED>
__global__ __launch_bounds__(256) void k_i4_plain(I4Args a) {
  const uint64_t all = (uint64_t)a.rows * a.n_out, stride = (uint64_t)gridDim.x * 256;
  for (uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x; i < all; i += stride) {
    const uint32_t p = (uint32_t)(i / a.n_out), n = (uint32_t)(i % a.n_out);
    int64_t s = p;
    uint32_t e = 0;
    if (GROUPED) {
      uint32_t hi = a.experts;  // the last expert whose rows begin at p or before, with p among them
      while (e < hi) {
        const uint32_t mid = (e + hi) / 2;
        if (offset_of(a, mid + 1) <= p) e = mid + 1;
        else hi = mid;
      }
      s = e < a.experts ? source_row(a, p) : -1;
    }
    float v = 0.0f;
    if (s >= 0) {
      const size_t ch = (size_t)e * a.n_out + n;
      const S* scale = (const S*)a.scale + (size_t)e * a.groups * a.n_out + n;
      float sum = 0.0f;
      for (uint32_t g = 0; g < a.groups; g++) {
        const uint32_t end = (g + 1) * a.group < a.n_in ? (g + 1) * a.group : a.n_in;
        // (in parts whose sums are exact as floats)
        for (uint32_t k0 = g * a.group; k0 < end; k0 += 8192) {
          int acc = 0;
          for (uint32_t k = k0; k < end && k < k0 + 8192; k++)
            acc += (int)a.x[(size_t)s * a.ld_x + k] * weight_at(a.w + ch * a.ld_w, k);
          sum = fmaf((float)acc, (float)scale[(size_t)g * a.n_out], sum);
        }
      }
      v = i4_finish(sum, a.sx ? a.sx[s] : 1.0f, a.bias ? a.bias[ch] : 0.0f, a.relu);
    }
    ((T*)a.y)[(size_t)p * a.ld_y + n] = (T)v;
  }
}

template <bool GROUPED>
static int i4_dispatch(zk_context* ctx, const I4Args& a, int scale_type, int type, hipStream_t st) {
  const char* name = GROUPED ? "i4_matmul_experts" : "i4_matmul";
  return by_type(type, [&](auto yz) -> int {
    return by_type(scale_type, [&](auto sz) -> int {
      typedef decltype(yz) T;
      typedef decltype(sz) S;
      const size_t blocks = ((size_t)a.rows * a.n_out + 255) / 256;
      ZK_LAUNCH(ctx, st, name, (k_i4_plain<T, S, GROUPED>), dim3(blocks < 65536 ? (uint32_t)blocks : 65536), dim3(256), 0, a);
      return ZK_OK;
    });
  });
}

// ------------------------------------------------------------ weights to 4 bits
// s = a / 7 rounded to the scales' type, a = max|w| over the group; q = the integer
// nearest to w / s (ties to even), at most 7 and at least -8 (s may have been rounded
// down).  A group of zeros has s = 0 and zeros, one that holds an infinity or a NaN
// s = NaN and zeros.  Padding is zero.  A wave has one run of 128 weights (small
// groups), or a whole group of them.  Bound by memory; done once for a model.
template <class T, class S>
__global__ __launch_bounds__(256) void k_i4_quantize(const T* __restrict__ w, size_t ld_w, uint32_t rows,
                                                     uint32_t cols, uint32_t group, uint32_t groups, uint32_t units,
                                                     int8_t* __restrict__ q, size_t ld_q, S* __restrict__ scale) {
  const uint32_t lane = threadIdx.x & 63;
  const uint64_t all = (uint64_t)rows * units, stride = (uint64_t)gridDim.x * 4;
  for (uint64_t i = (uint64_t)blockIdx.x * 4 + (threadIdx.x >> 6); i < all; i += stride) {
    const uint32_t r = (uint32_t)(i / units), u = (uint32_t)(i % units);
    const T* row = w + (size_t)r * ld_w;
    const uint32_t run = group < 128 ? 128 : group, k0 = u * run, end = k0 + run < cols ? k0 + run : cols;
    auto at = [&](uint32_t k) { return k < end ? (float)row[k] : 0.0f; };
    // magnitudes as integers, in the floats' order, NaN above infinity
    uint32_t m[2] = {0, 0};
    for (uint32_t k = k0; k < end; k += 128)
#pragma unroll
      for (int h = 0; h < 2; h++) {
        const uint32_t b = __float_as_uint(at(k + 64 * h + lane)) & 0x7fffffffu;
        m[h] = b > m[h] ? b : m[h];
      }
    if (group > 64) m[0] = m[1] = m[0] > m[1] ? m[0] : m[1];
    for (uint32_t d = group < 64 ? 16 : 32; d; d >>= 1)
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
      const uint32_t g = (k0 + 64 * h + lane) / group;
      // the group's first lane writes its scale
      if (g < groups && (k0 + 64 * h + lane) % group == 0) scale[(size_t)g * rows + r] = rounded;
    }
    for (uint32_t k = k0; k < end; k += 128) {
      int v[2];
#pragma unroll
      for (int h = 0; h < 2; h++) {
        float f = s[h] > 0.0f && m[h] < 0x7f800000u ? rintf(at(k + 64 * h + lane) / s[h]) : 0.0f;
        f = f > 7.0f ? 7.0f : f < -8.0f ? -8.0f : f;
        v[h] = (int)f;
      }
      q[(size_t)r * ld_q + k / 2 + lane] = (int8_t)((v[0] & 15) | (int)((uint32_t)v[1] << 4));
    }
  }
}

// ------------------------------------------------------------ arguments
static int check_group(zk_context* ctx, size_t n_in, int group) {
  if (group != 32 && group != 64 && (group < 128 || group % 128))
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

static void set_sizes(I4Args& a, size_t rows, size_t n_out, size_t n_in, int group, int relu) {
  a.rows = (uint32_t)rows, a.n_out = (uint32_t)n_out, a.n_in = (uint32_t)n_in, a.relu = relu != 0;
  a.group = (uint32_t)group, a.groups = cdiv(n_in, group);
}

static int i4_matmul(zk_context* ctx, const I4Args& a, int scale_type, int type, hipStream_t st) {
  // rows in runs of at most I8_MAX_TILES tiles of 16 x 16
  const size_t most = I8_MAX_TILES / cdiv(a.n_out, 16) * 16;
  for (size_t r = 0; r < a.rows; r += most) {
    I4Args b = a;
    b.rows = (uint32_t)(a.rows - r < most ? a.rows - r : most);
    b.x = a.x ? a.x + r * a.ld_x : a.x;
    b.sx = a.sx ? a.sx + r : a.sx;
    b.y = (uint8_t*)a.y + r * a.ld_y * type_bytes(type);
    ZK_TRY(i4_dispatch<false>(ctx, b, scale_type, type, st));
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
    const size_t blocks = (rows * units + 3) / 4;
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
    set_sizes(a, rows, n_out, n_in, group, relu);
    OnDevice on(ctx);
    return i4_matmul(ctx, a, scale_type, y_type, ctx->s(stream));
  });
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
    set_sizes(a, rows, n_out, n_in, group, relu);
    OnDevice on(ctx);
    hipStream_t st = ctx->s(stream);
    ZK_TRY(i8_quantize(ctx, d_x, x_type, ld_x, rows, n_in, (int8_t*)d_work + lw.q, lw.ld, (float*)d_work, st));
    return i4_matmul(ctx, a, scale_type, y_type, st);
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
    set_sizes(a, rows, n_out, n_in, group, relu);
    a.offsets = d_offsets, a.order = d_order, a.experts = (uint32_t)experts, a.slots = (uint32_t)slots;
    a.tokens = (uint32_t)tokens;
    OnDevice on(ctx);
    return i4_dispatch<true>(ctx, a, scale_type, y_type, ctx->s(stream));
  });
}

}  // extern "C"
