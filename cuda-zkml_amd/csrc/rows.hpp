// Rows of f32, f16 or bf16 moved 16 bytes a lane at any address (gfx950 loads
// and stores 16 bytes from any address).  A row's last, shorter piece is taken
// 16 bytes back from its end, so that two lanes may hold, and write, the same
// elements there; rows under 16 bytes go element by element.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/zkml_gpu.h"

namespace zk {

template <class T>
struct Vec {
  static constexpr uint32_t N = 16 / sizeof(T);
  T v[N];
};

typedef int row16 __attribute__((ext_vector_type(4), aligned(1)));

// ONCE: the bytes are used once, so the caches need not keep them.
template <class T, bool ONCE = false>
__device__ __forceinline__ Vec<T> row_load(const T* p, uint32_t left) {
  Vec<T> r;
  if (left >= Vec<T>::N) {
    const row16 v = ONCE ? __builtin_nontemporal_load((const row16*)p) : *(const row16*)p;
    __builtin_memcpy(&r, &v, 16);
  } else {
#pragma unroll
    for (uint32_t i = 0; i < Vec<T>::N; i++) r.v[i] = i < left ? p[i] : (T)0.0f;
  }
  return r;
}

template <class T, bool ONCE = false>
__device__ __forceinline__ void row_store(T* p, uint32_t left, const Vec<T>& r) {
  if (left >= Vec<T>::N) {
    row16 v;
    __builtin_memcpy(&v, &r, 16);
    if (ONCE) __builtin_nontemporal_store(v, (row16*)p);
    else *(row16*)p = v;
  } else {
#pragma unroll
    for (uint32_t i = 0; i < Vec<T>::N; i++)
      if (i < left) p[i] = r.v[i];
  }
}

// First element of a row's c-th piece.
template <class T>
__device__ __forceinline__ uint32_t piece(uint32_t c, uint32_t cols) {
  const uint32_t at = c * Vec<T>::N;
  return at + Vec<T>::N <= cols || cols < Vec<T>::N ? at : cols - Vec<T>::N;
}

template <class T>
__host__ __device__ inline uint32_t pieces_of(uint32_t cols) {
  return (cols + Vec<T>::N - 1) / Vec<T>::N;
}

// ---- argument checks of the entry points
inline size_t type_bytes(int type) { return type == ZK_F32 || type == ZK_I32 ? 4 : 2; }
inline bool float_type(int type) { return type == ZK_F32 || type == ZK_F16 || type == ZK_BF16; }
inline bool aligned(const void* p, size_t n) { return (uintptr_t)p % n == 0; }

// Calls f with a value of the type.
template <class Fn>
int by_type(int type, Fn&& f) {
  if (type == ZK_F32) return f(0.0f);
  if (type == ZK_F16) return f((_Float16)0.0f);
  return f((__bf16)0.0f);
}

}  // namespace zk
