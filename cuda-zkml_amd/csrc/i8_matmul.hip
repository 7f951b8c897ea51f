// 8-bit integer layers for gfx950: the linear layer a quantized model's
// statement proves (weights out x in, row major), over whole batches on the
// matrix cores, with the scales that tie its integers to the real-valued model.
//
//   acc[t,n] = sum_k x[t,k] w[n,k]                 int32, exact
//   y[t,n]   = act(float(acc) (sx[t] sw[n]) + b[n])  or acc itself
//
// A product of two int8 is at most 2^14, so acc is exact for n_in <= 131071.
// The grouped form takes its weights by expert: rows offsets[e] to
// offsets[e+1] of y use w[e].
#include "zk_internal.hpp"

namespace zk {

typedef int v4i __attribute__((ext_vector_type(4)));
typedef int v16i __attribute__((ext_vector_type(16)));

constexpr size_t I8_MAX_IN = 131071;

// What every kernel of this file is given.
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

// 16 bytes of a row from byte k on, zeros from n_in on.  The row's address may
// be odd: gfx950 loads 16 bytes from any address.
__device__ __forceinline__ v4i load16(const int8_t* __restrict__ row, uint32_t k, uint32_t n_in) {
  v4i v = {0, 0, 0, 0};
  if (k + 16 <= n_in) {
    __builtin_memcpy(&v, row + k, 16);
  } else if (k < n_in) {
    uint32_t b[4] = {0, 0, 0, 0};
    for (uint32_t i = 0; i < n_in - k; i++) b[i / 4] |= (uint32_t)(uint8_t)row[k + i] << (8 * (i % 4));
    v = v4i{(int)b[0], (int)b[1], (int)b[2], (int)b[3]};
  }
  return v;
}

template <class T>
__device__ __forceinline__ T finish(int acc, float s, float b, int relu) {
  float f = (float)acc * s + b;
  if (relu && f < 0.0f) f = 0.0f;  // a NaN stays
  return (T)f;
}
template <>
__device__ __forceinline__ int finish<int>(int acc, float, float, int relu) {
  return relu && acc < 0 ? 0 : acc;
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

template <class T, bool GROUPED>
__global__ __launch_bounds__(256) void k_i8_tile(I8Args a) {
  constexpr int B = 64, LD = 80;
  __shared__ __align__(16) int8_t X[B * LD], W[B * LD];
  const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const uint32_t n0 = blockIdx.x * B;
  uint32_t r0 = blockIdx.y * B, r1 = a.rows, e = 0;
  if (GROUPED) {
    // the tile's expert: tiles are counted expert by expert, the rows that
    // belong to none last
    uint32_t tile = blockIdx.y;
    bool found = false;
    for (; e < a.experts; e++) {
      const uint32_t lo = offset_of(a, e), hi = offset_of(a, e + 1);
      const uint32_t n = hi > lo ? (hi - lo + B - 1) / B : 0;
      if (tile < n) {
        r0 = lo + tile * B;
        r1 = hi;
        found = true;
        break;
      }
      tile -= n;
    }
    if (!found) {
      r0 = offset_of(a, a.experts) + tile * B;
      r1 = a.rows;
    }
  }
  if (r0 >= r1) return;
  const bool none = GROUPED && e >= a.experts;
  const int8_t* w = a.w + (size_t)e * a.n_out * a.ld_w;
  // a thread moves 16 bytes of one row of each tile
  const uint32_t lr = tid >> 2, lk = (tid & 3) * 16;
  int64_t xr = -1;
  if (r0 + lr < r1 && !none) xr = GROUPED ? source_row(a, r0 + lr) : (int64_t)(r0 + lr);
  const bool wr = n0 + lr < a.n_out && !none;
  v16i acc = {0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0};
  const uint32_t wn = (wave & 1) * 32, wt = (wave >> 1) * 32;
  for (uint32_t k = 0; k < a.n_in && !none; k += 64) {
    const v4i zero = {0, 0, 0, 0};
    const v4i xv = xr >= 0 ? load16(a.x + (size_t)xr * a.ld_x, k + lk, a.n_in) : zero;
    const v4i wv = wr ? load16(w + (size_t)(n0 + lr) * a.ld_w, k + lk, a.n_in) : zero;
    *(v4i*)&X[lr * LD + lk] = xv;
    *(v4i*)&W[lr * LD + lk] = wv;
    __syncthreads();
#pragma unroll
    for (int s = 0; s < 2; s++) {
      const uint32_t o = s * 32 + (lane >> 5) * 16;
      const v4i fw = *(const v4i*)&W[(wn + (lane & 31)) * LD + o];
      const v4i fx = *(const v4i*)&X[(wt + (lane & 31)) * LD + o];
      acc = __builtin_amdgcn_mfma_i32_32x32x32_i8(fw, fx, acc, 0, 0, 0);
    }
    __syncthreads();
  }
  const uint32_t t = r0 + wt + (lane & 31);
  if (t >= r1) return;
  int64_t src = GROUPED ? (none ? -1 : source_row(a, t)) : (int64_t)t;
  const float sx = src >= 0 && a.sx ? a.sx[src] : 1.0f;
  const size_t ch = (size_t)e * a.n_out;
#pragma unroll
  for (int i = 0; i < 16; i++) {
    const uint32_t n = n0 + wn + 8 * (i >> 2) + 4 * (lane >> 5) + (i & 3);
    if (n >= a.n_out) continue;
    T v = (T)0;
    if (!GROUPED || src >= 0)
      v = finish<T>(acc[i], sx * (a.sw ? a.sw[ch + n] : 1.0f), a.bias ? a.bias[ch + n] : 0.0f, a.relu);
    ((T*)a.y)[(size_t)t * a.ld_y + n] = v;
  }
}

template <class T>
static int launch_tile(zk_context* ctx, const I8Args& a, bool grouped, hipStream_t st) {
  const size_t by = grouped ? (size_t)(a.rows + 63) / 64 + (a.experts < a.rows ? a.experts : a.rows) + 1
                            : ((size_t)a.rows + 63) / 64;
  const dim3 grid(cdiv(a.n_out, 64), (uint32_t)by);
  if (grouped)
    ZK_LAUNCH(ctx, st, "i8_matmul_experts", (k_i8_tile<T, true>), grid, dim3(256), 0, a);
  else
    ZK_LAUNCH(ctx, st, "i8_matmul", (k_i8_tile<T, false>), grid, dim3(256), 0, a);
  return ZK_OK;
}

static int i8_dispatch(zk_context* ctx, const I8Args& a, int type, bool grouped, hipStream_t st) {
  switch (type) {
    case ZK_I32: return launch_tile<int>(ctx, a, grouped, st);
    case ZK_F32: return launch_tile<float>(ctx, a, grouped, st);
    case ZK_F16: return launch_tile<_Float16>(ctx, a, grouped, st);
    default: return launch_tile<__bf16>(ctx, a, grouped, st);
  }
}

// ------------------------------------------------------------ rows to 8 bits
// s = max|x| / 127, q = rint(127 x / max|x|).  The quotient is taken by a
// division, not by a product with the reciprocal, so that it has one rounding
// and a half-way quotient goes to the even number.  Rows far from 1 are first
// multiplied by a power of two, so that neither 127 x nor the quotient leaves
// the type.  A row of zeros gives s = 0 and zeros; a row with an infinity or a
// NaN gives s = NaN and zeros, so that its products show it.
template <class T>
__global__ __launch_bounds__(256) void k_i8_quantize(const T* __restrict__ x, size_t ld_x, uint32_t cols,
                                                     int8_t* __restrict__ q, size_t ld_q,
                                                     float* __restrict__ scale) {
  __shared__ float part[4];
  const uint32_t tid = threadIdx.x;
  const T* row = x + (size_t)blockIdx.x * ld_x;
  int8_t* out = q + (size_t)blockIdx.x * ld_q;
  // magnitudes as integers: their order is the floats', NaN above infinity
  uint32_t m = 0;
  for (uint32_t i = tid; i < cols; i += 256) {
    const uint32_t u = __float_as_uint((float)row[i]) & 0x7fffffffu;
    m = u > m ? u : m;
  }
  for (int d = 32; d; d >>= 1) {
    const uint32_t o = __shfl_xor((int)m, d);
    m = o > m ? o : m;
  }
  if ((tid & 63) == 0) part[tid >> 6] = __uint_as_float(m);
  __syncthreads();
  for (int i = 0; i < 4; i++) {
    const uint32_t o = __float_as_uint(part[i]);
    m = o > m ? o : m;
  }
  const bool finite = m < 0x7f800000u;
  float a = __uint_as_float(m);
  if (tid == 0) scale[blockIdx.x] = finite ? a / 127.0f : __uint_as_float(0x7fc00000u);
  const float c = a >= 0x1p64f ? 0x1p-32f : a < 0x1p-64f ? 0x1p64f : 1.0f;
  a *= c;
  for (uint32_t i = tid; i < cols; i += 256) {
    const float f = (float)row[i] * c;
    out[i] = finite && m ? (int8_t)rintf(f * 127.0f / a) : (int8_t)0;
  }
}

template <class T>
static int launch_quantize(zk_context* ctx, const void* x, size_t ld_x, size_t rows, size_t cols, int8_t* q,
                           size_t ld_q, float* scale, hipStream_t st) {
  ZK_LAUNCH(ctx, st, "i8_quantize", k_i8_quantize<T>, dim3((uint32_t)rows), dim3(256), 0, (const T*)x, ld_x,
            (uint32_t)cols, q, ld_q, scale);
  return ZK_OK;
}

static int i8_quantize(zk_context* ctx, const void* x, int type, size_t ld_x, size_t rows, size_t cols, int8_t* q,
                       size_t ld_q, float* scale, hipStream_t st) {
  if (rows == 0) return ZK_OK;
  switch (type) {
    case ZK_F32: return launch_quantize<float>(ctx, x, ld_x, rows, cols, q, ld_q, scale, st);
    case ZK_F16: return launch_quantize<_Float16>(ctx, x, ld_x, rows, cols, q, ld_q, scale, st);
    default: return launch_quantize<__bf16>(ctx, x, ld_x, rows, cols, q, ld_q, scale, st);
  }
}

// ------------------------------------------------------------ arguments
static size_t type_bytes(int type) { return type == ZK_F32 || type == ZK_I32 ? 4 : 2; }
static bool float_type(int type) { return type == ZK_F32 || type == ZK_F16 || type == ZK_BF16; }
static bool aligned(const void* p, size_t n) { return (uintptr_t)p % n == 0; }

// Checks that the two forms of the product share.
static int check_product(zk_context* ctx, const I8Args& a, size_t rows, size_t n_out, size_t n_in, int type) {
  if (type != ZK_I32 && !float_type(type)) return ctx->fail(ZK_ERR_INVALID, "i8 product: unknown type of y");
  if (type == ZK_I32 && (a.sx || a.sw || a.bias))
    return ctx->fail(ZK_ERR_INVALID, "i8 product: integer sums take no scales and no bias");
  if (n_in > I8_MAX_IN) return ctx->fail(ZK_ERR_SIZE, "i8 product: n_in above 131071 can pass 32 bits");
  if (rows > 0x7fffffffu || n_out > 0x7fffffffu) return ctx->fail(ZK_ERR_SIZE, "i8 product: sizes above 2^31 - 1");
  if (a.ld_x < n_in || a.ld_w < n_in || a.ld_y < n_out)
    return ctx->fail(ZK_ERR_INVALID, "i8 product: a row stride below the row's length");
  if (rows && n_out && (!a.y || (n_in && (!a.x || !a.w))))
    return ctx->fail(ZK_ERR_INVALID, "i8 product: null pointer");
  if (!aligned(a.y, type_bytes(type)) || !aligned(a.sx, 4) || !aligned(a.sw, 4) || !aligned(a.bias, 4))
    return ctx->fail(ZK_ERR_INVALID, "i8 product: a pointer is not aligned to its type");
  return ZK_OK;
}

static int check_quantize(zk_context* ctx, const void* x, int type, size_t ld_x, size_t rows, size_t cols) {
  if (!float_type(type)) return ctx->fail(ZK_ERR_INVALID, "i8 quantize: x is f32, f16 or bf16");
  if (rows > 0x7fffffffu || cols > 0x7fffffffu) return ctx->fail(ZK_ERR_SIZE, "i8 quantize: sizes above 2^31 - 1");
  if (ld_x < cols) return ctx->fail(ZK_ERR_INVALID, "i8 quantize: a row stride below the row's length");
  if (rows && cols && !x) return ctx->fail(ZK_ERR_INVALID, "i8 quantize: null pointer");
  if (!aligned(x, type_bytes(type))) return ctx->fail(ZK_ERR_INVALID, "i8 quantize: x is not aligned to its type");
  return ZK_OK;
}

// Layout of zk_i8_linear's workspace: the rows' scales, then the rows' bytes.
struct LinearWork {
  size_t ld, q, bytes;
};
static LinearWork linear_work(size_t rows, size_t n_in) {
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
  // a launch has at most 65535 row tiles
  const size_t most = (size_t)65535 * 64;
  for (size_t r = 0; r < rows; r += most) {
    I8Args b = a;
    b.rows = (uint32_t)(rows - r < most ? rows - r : most);
    b.x = x ? x + r * ld_x : x;
    b.sx = sx ? sx + r : sx;
    b.y = (uint8_t*)y + r * ld_y * type_bytes(type);
    ZK_TRY(i8_dispatch(ctx, b, type, false, st));
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
    ZK_TRY(check_product(ctx, a, rows, n_out, n_in, y_type));
    if (rows > ZK_MAX_EXPERT_ROWS || tokens > 0x7fffffffu)
      return ctx->fail(ZK_ERR_SIZE, "i8 experts: too many rows");
    if (!rows || !n_out) return ZK_OK;
    if (!d_offsets) return ctx->fail(ZK_ERR_INVALID, "i8 experts: null pointer");
    if (!aligned(d_offsets, 4) || !aligned(d_order, 4))
      return ctx->fail(ZK_ERR_INVALID, "i8 experts: a pointer is not aligned to its type");
    a.rows = (uint32_t)rows, a.n_out = (uint32_t)n_out, a.n_in = (uint32_t)n_in, a.relu = relu != 0;
    a.offsets = d_offsets, a.order = d_order, a.experts = (uint32_t)experts, a.slots = (uint32_t)slots;
    a.tokens = (uint32_t)tokens;
    return i8_dispatch(ctx, a, y_type, true, ctx->s(stream));
  });
}

}  // extern "C"
