// 16 bytes of a row at any element alignment, as fp32 (layer_norm.hip, linear.hip).
#pragma once
#include "common.hpp"

namespace moy {

template <typename T>
struct Chunk {
  static constexpr int VEC = DT<T>::KPB;
  // n elements of the row are left at p: none are read past them (zeros there)
  static __device__ __forceinline__ void load(const T* p, int n, float (&v)[VEC]) {
    if (n >= VEC) {
      u32x4 t;
      __builtin_memcpy(&t, __builtin_assume_aligned(p, sizeof(T)), 16);
      unpack(t, v);
    } else {
#pragma unroll
      for (int e = 0; e < VEC; ++e) v[e] = e < n ? DT<T>::load1(p + e) : 0.f;
    }
  }
  static __device__ __forceinline__ void unpack(const u32x4& t, float (&v)[VEC]) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint32_t u = t[k];             // (a value: a bit cast of the vector's element itself reads element 0)
      if constexpr (VEC == 4) {
        v[k] = __builtin_bit_cast(float, u);
      } else {
        v[2 * k] = DT<T>::lo(u);
        v[2 * k + 1] = DT<T>::hi(u);
      }
    }
  }
  static __device__ __forceinline__ void store(T* p, int n, const float (&v)[VEC]) {
    if (n >= VEC) {
      u32x4 t;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if constexpr (VEC == 4) t[k] = __builtin_bit_cast(uint32_t, v[k]);
        else t[k] = DT<T>::pack2(v[2 * k], v[2 * k + 1]);
      }
      __builtin_memcpy(__builtin_assume_aligned(p, sizeof(T)), &t, 16);
    } else {
#pragma unroll
      for (int e = 0; e < VEC; ++e)
        if (e < n) DT<T>::store1(p + e, v[e]);
    }
  }
};

// a vector of weights or biases in its own type, one element
__device__ __forceinline__ float typed_load(const void* p, int dtype, int64_t i) {
  return dtype == MOY_F32 ? static_cast<const float*>(p)[i]
                          : dtype == MOY_BF16 ? DT<bf16_t>::load1(static_cast<const bf16_t*>(p) + i) : DT<f16_t>::load1(static_cast<const f16_t*>(p) + i);
}
__device__ __forceinline__ void typed_store(void* p, int dtype, int64_t i, float v) {
  if (dtype == MOY_F32) static_cast<float*>(p)[i] = v;
  else if (dtype == MOY_BF16) DT<bf16_t>::store1(static_cast<bf16_t*>(p) + i, v);
  else DT<f16_t>::store1(static_cast<f16_t*>(p) + i, v);
}

inline bool aligned_as(const void* p, int dtype) { return reinterpret_cast<uintptr_t>(p) % (dtype == MOY_F32 ? 4 : 2) == 0; }

// one | two [n each] = `rows` partial rows [n one | n two] added in row order: a block takes 32 columns, 32 threads to a column take every 32nd row, and the
// 32 sums are added in order.  n_two = 0: one alone.
__global__ __launch_bounds__(1024) static void column_sums_kernel(const float* __restrict__ part, int rows, int n, int n_two, void* one, void* two, int dtype) {
  __shared__ float s[32][33];
  const int c = threadIdx.x & 31, k = threadIdx.x >> 5, width = n + n_two;
  const int col = blockIdx.x * 32 + c;
  float v = 0.f;
  if (col < width) {
#pragma unroll 8
    for (int b = k; b < rows; b += 32) v += part[(int64_t)b * width + col];
  }
  s[k][c] = v;
  __syncthreads();
  if (k == 0 && col < width) {
    v = 0.f;
#pragma unroll
    for (int i = 0; i < 32; ++i) v += s[i][c];
    void* out = col < n ? one : two;
    if (out) typed_store(out, dtype, col < n ? col : col - n, v);
  }
}

}  // namespace moy
