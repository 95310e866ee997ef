// What the kernels over rows (layer norm, bias by buckets, softmax over in-edges) share: element types, packets of
// elements, and sums over the threads that work on one row.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <atomic>

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

constexpr int kMostDevices = 64;
// The current device; -1 if it cannot be asked, or is beyond those that things are remembered for.
inline int current_device() {
  int device = -1;
  return cudaGetDevice(&device) == cudaSuccess && device < kMostDevices ? device : -1;
}
// Multiprocessors of the current device; 0 if it cannot be asked.
inline int processors() {
  static std::atomic<int> known[kMostDevices];
  const int device = current_device();
  if (device < 0) return 0;
  int count = known[device].load(std::memory_order_relaxed);
  if (count) return count;
  if (cudaDeviceGetAttribute(&count, cudaDevAttrMultiProcessorCount, device) != cudaSuccess) return 0;
  known[device].store(count, std::memory_order_relaxed);
  return count;
}

// What is known of a kernel, so that a launch does not ask the runtime again: on which devices it may use as much shared memory
// as there is (always all of it, so that calls of other shapes on other threads change nothing), and how many CTAs are resident
// with the shared memory of the last call.
struct Kernel {
  std::atomic<uint64_t> allowed{0}, last{0};

  template <typename... P>
  int allow(void (*kernel)(P...), size_t shared) {
    if (shared <= 32 * 1024) return LUNA_OK;  // with what it has at compile time within the 48 KB that every kernel may use
    const int device = current_device();
    if (device < 0) return fail(LUNA_ERR_CUDA, "the current device is unknown");
    if (shared > kMostShared) return fail(LUNA_ERR_UNSUPPORTED, "%zu bytes of shared memory", shared);
    if (!(allowed.load(std::memory_order_acquire) >> device & 1)) {
      LUNA_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kMostShared)));
      allowed.fetch_or(1ull << device, std::memory_order_release);
    }
    return LUNA_OK;
  }
  // CTAs on the whole device, or less than one (a status).
  template <typename... P>
  int resident(void (*kernel)(P...), int threads, size_t shared) {
    if (const int status = allow(kernel, shared)) return status;
    const uint64_t key = (static_cast<uint64_t>(shared) << 6 | current_device()) << 16;
    const uint64_t known = last.load(std::memory_order_relaxed);
    if (known && (known >> 16 << 16) == key) return static_cast<int>(known & 0xffff);
    int count = 0;
    LUNA_CUDA_CHECK(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&count, kernel, threads, shared));
    count *= processors();
    if (count < 1 || count > 0xffff) return fail(LUNA_ERR_CUDA, "a kernel does not fit the current device");
    last.store(key | static_cast<uint64_t>(count), std::memory_order_relaxed);
    return count;
  }
  static constexpr size_t kMostShared = 216 * 1024;  // beside what the kernels have at compile time
};

}  // namespace rows
}  // namespace luna
