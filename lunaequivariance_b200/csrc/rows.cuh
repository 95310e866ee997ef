// What the kernels over rows (layer norm, bias by buckets, softmax over in-edges) share: element types, packets of
// elements, and sums over the threads that work on one row.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.h"

namespace luna {
namespace rows {

using bf16 = __nv_bfloat16;
using f16 = __half;

// Sums and statistics are held in 32 bits for the 16-bit types; a value is rounded to its type once, when it is stored.
template <typename T>
struct AccOf {
  using type = float;
};
template <>
struct AccOf<double> {
  using type = double;
};
template <typename T>
using Acc = typename AccOf<T>::type;

__device__ __forceinline__ float widen(float v) { return v; }
__device__ __forceinline__ double widen(double v) { return v; }
__device__ __forceinline__ float widen(bf16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float widen(f16 v) { return __half2float(v); }
__device__ __forceinline__ void narrow(float v, float& to) { to = v; }
__device__ __forceinline__ void narrow(double v, double& to) { to = v; }
__device__ __forceinline__ void narrow(float v, bf16& to) { to = __float2bfloat16_rn(v); }
__device__ __forceinline__ void narrow(float v, f16& to) { to = __float2half_rn(v); }

template <typename T, int N>
struct alignas(sizeof(T) * N < 16 ? sizeof(T) * N : 16) Pack {
  T a[N];
};

template <typename T, int N>
__device__ __forceinline__ void load(const T* __restrict__ from, Acc<T> (&to)[N]) {
  const Pack<T, N> p = *reinterpret_cast<const Pack<T, N>*>(from);
#pragma unroll
  for (int c = 0; c < N; ++c) to[c] = widen(p.a[c]);
}
template <typename T, int N>
__device__ __forceinline__ void store(T* __restrict__ to, const Acc<T> (&from)[N]) {
  Pack<T, N> p;
#pragma unroll
  for (int c = 0; c < N; ++c) narrow(from[c], p.a[c]);
  *reinterpret_cast<Pack<T, N>*>(to) = p;
}

// Calls `f` with a value of the element type that `dtype` names; false if it names none.
template <typename F>
inline bool with_type(int dtype, F&& f) {
  switch (dtype) {
    case LUNA_F32: f(float()); return true;
    case LUNA_F64: f(double()); return true;
    case LUNA_BF16: f(bf16()); return true;
    case LUNA_F16: f(f16()); return true;
    default: return false;
  }
}
inline int64_t size_of(int dtype) { return dtype == LUNA_F64 ? 8 : dtype == LUNA_F32 ? 4 : 2; }
inline int64_t acc_size_of(int dtype) { return dtype == LUNA_F64 ? 8 : 4; }

inline int next_power_of_two(int64_t v) {
  int p = 1;
  while (p < v) p <<= 1;
  return p;
}

// Multiprocessors of the current device; 0 if it cannot be asked.
inline int processors() {
  int device = 0, count = 0;
  if (cudaGetDevice(&device) != cudaSuccess) return 0;
  if (cudaDeviceGetAttribute(&count, cudaDevAttrMultiProcessorCount, device) != cudaSuccess) return 0;
  return count;
}

}  // namespace rows
}  // namespace luna
