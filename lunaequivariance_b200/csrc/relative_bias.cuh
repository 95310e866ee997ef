// A learned bias by buckets: out[e] = table[bucket[e]], and the gradient of the table, gtable[b] = sum of g[e] over the
// edges of bucket b.  Edges whose bucket is no row of the table take zeros and give nothing.
#pragma once

#include "rows.cuh"

namespace luna {
namespace bias {

using rows::Acc;

// ---- values ------------------------------------------------------------------------------------------------------------------
// `lanes` threads (a power of two) take an edge's packets.  Bound by the output's way to memory; the table stays in cache.
template <typename T, int VEC>
__global__ void __launch_bounds__(256)
gather_kernel(const T* __restrict__ table, const int32_t* __restrict__ buckets, T* __restrict__ out, int64_t edges, int num_buckets,
              int heads, int lanes) {
  const int lane = threadIdx.x & (lanes - 1);
  const int64_t step = static_cast<int64_t>(gridDim.x) * (blockDim.x / lanes);
  for (int64_t e = static_cast<int64_t>(blockIdx.x) * (blockDim.x / lanes) + threadIdx.x / lanes; e < edges; e += step) {
    const int b = buckets[e];
    const bool inside = b >= 0 && b < num_buckets;
    for (int h = lane * VEC; h < heads; h += lanes * VEC) {
      rows::Pack<T, VEC> p{};
      if (inside) p = *reinterpret_cast<const rows::Pack<T, VEC>*>(table + static_cast<int64_t>(b) * heads + h);
      *reinterpret_cast<rows::Pack<T, VEC>*>(out + e * heads + h) = p;
    }
  }
}

// ---- gradient of the table ------------------------------------------------------------------------------------------------------
// A CTA holds several copies of its part of the table in shared memory.  The `lanes` threads of a copy take every copies-th
// edge of the CTA's and add its row to the copy, each thread to columns of its own: no two threads add to one number, so
// there are no atomics, and the order of the sums depends on the sizes alone.  The copies are summed at the end, the CTAs'
// sums in a second launch.  What bounds it is HBM where the copies are many; the additions to one copy follow one another.
struct Cut {
  int lanes, copies, threads;  // threads per copy; copies and threads of a CTA
  int buckets;                 // rows of the table that a CTA has
  int parts_of_edges, parts_of_heads, parts_of_buckets;
  int64_t shared;              // bytes
};

template <typename T, int VEC>
__global__ void __launch_bounds__(256)
table_kernel(const T* __restrict__ g, const int32_t* __restrict__ buckets, Acc<T>* __restrict__ partial, int64_t edges,
             int num_buckets, int heads, Cut cut) {
  using A = Acc<T>;
  extern __shared__ __align__(16) unsigned char raw[];
  A* tables = reinterpret_cast<A*>(raw);
  const int width = cut.lanes * VEC, copy_size = cut.buckets * width;
  for (int i = threadIdx.x; i < cut.copies * copy_size; i += blockDim.x) tables[i] = A(0);
  __syncthreads();
  const int first_bucket = blockIdx.z * cut.buckets, first_head = blockIdx.y * width;
  const int lane = threadIdx.x & (cut.lanes - 1), copy = threadIdx.x / cut.lanes;
  const int head = first_head + lane * VEC;
  const int64_t begin = edges * blockIdx.x / gridDim.x, end = edges * (blockIdx.x + 1) / gridDim.x;
  if (copy < cut.copies && head < heads) {
    A* mine = tables + static_cast<int64_t>(copy) * copy_size + lane * VEC;
    constexpr int kAhead = 4;
    for (int64_t e = begin + copy; e < end; e += static_cast<int64_t>(cut.copies) * kAhead) {
      A v[kAhead][VEC];
      int b[kAhead];
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        const int64_t at = e + static_cast<int64_t>(j) * cut.copies;
        b[j] = -1;
        if (at < end) {
          b[j] = buckets[at];
          rows::load<T, VEC>(g + at * heads + head, v[j]);
        }
      }
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        const int row = b[j] - first_bucket;
        if (b[j] >= 0 && b[j] < num_buckets && row >= 0 && row < cut.buckets) {
          auto* to = reinterpret_cast<rows::Pack<A, VEC>*>(mine + row * width);
          rows::Pack<A, VEC> sum = *to;
#pragma unroll
          for (int c = 0; c < VEC; ++c) sum.a[c] += v[j][c];
          *to = sum;
        }
      }
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < copy_size; i += blockDim.x) {
    const int bucket = first_bucket + i / width, h = first_head + i % width;
    if (bucket >= num_buckets || h >= heads) continue;
    A sum = tables[i];
    for (int c = 1; c < cut.copies; ++c) sum += tables[c * copy_size + i];
    partial[(static_cast<int64_t>(blockIdx.x) * num_buckets + bucket) * heads + h] = sum;
  }
}

// The sums of all CTAs: 32 numbers of the table by one CTA, 16 threads for each.
constexpr int kFinalSlices = 16;
template <typename T>
__global__ void __launch_bounds__(32 * kFinalSlices)
table_final_kernel(const Acc<T>* __restrict__ partial, T* __restrict__ gtable, int64_t numbers, int parts) {
  using A = Acc<T>;
  __shared__ A tile[kFinalSlices][32];
  wait_for_previous();
  const int lane = threadIdx.x & 31, slice = threadIdx.x >> 5;
  const int64_t at = static_cast<int64_t>(blockIdx.x) * 32 + lane;
  A sum = A(0);
  if (at < numbers)
    for (int j = slice; j < parts; j += kFinalSlices) sum += partial[j * numbers + at];
  tile[slice][lane] = sum;
  __syncthreads();
  if (slice || at >= numbers) return;
#pragma unroll
  for (int j = 1; j < kFinalSlices; ++j) sum += tile[j][lane];
  rows::narrow(sum, gtable[at]);
}

// The largest packet that divides a row of `heads` and is aligned in every array.
inline int packet_of(int64_t size, int64_t heads, std::initializer_list<const void*> arrays) {
  int vec = static_cast<int>(16 / size);
  auto fits = [&](int v) {
    if (heads % v) return false;
    for (const void* p : arrays)
      if (!aligned_to(p, static_cast<size_t>(v * size))) return false;
    return true;
  };
  while (vec > 1 && !fits(vec)) vec >>= 1;
  return vec;
}

// How the table's gradient is cut up for packets of `vec`.  Shared memory of half a multiprocessor per CTA, or of a whole one
// where that would leave only a few copies.
inline Cut cut_of(int64_t acc_size, int vec, int64_t edges, int64_t num_buckets, int64_t heads) {
  constexpr int64_t kHalf = 100 * 1024, kWhole = 200 * 1024;
  Cut cut{};
  const int64_t packets = ceil_div(heads, vec);
  cut.lanes = packets >= 32 ? 32 : rows::next_power_of_two(packets);
  auto copy_bytes = [&] { return num_buckets * cut.lanes * vec * acc_size; };
  while (cut.lanes > 1 && copy_bytes() > kWhole) cut.lanes >>= 1;
  const int64_t row_bytes = cut.lanes * vec * acc_size;
  cut.buckets = static_cast<int>(copy_bytes() > kWhole ? kWhole / row_bytes : num_buckets);
  const int64_t copy = cut.buckets * row_bytes;
  const int64_t most = 256 / cut.lanes;
  int64_t copies = kHalf / copy;
  if (copies < 4) copies = kWhole / copy;
  copies = copies < 1 ? 1 : (copies > most ? most : copies);
  cut.copies = static_cast<int>(copies);
  cut.threads = static_cast<int>(ceil_div(copies * cut.lanes, 32) * 32);
  cut.shared = copies * copy;
  cut.parts_of_heads = static_cast<int>(ceil_div(packets, cut.lanes));
  cut.parts_of_buckets = static_cast<int>(ceil_div(num_buckets, cut.buckets));
  const int64_t per_processor = 220 * 1024 / (cut.shared + 1024);
  int64_t resident = rows::processors() * (per_processor < 1 ? 1 : (per_processor > 8 ? 8 : per_processor));
  int64_t parts = resident / (cut.parts_of_heads * static_cast<int64_t>(cut.parts_of_buckets));
  const int64_t wanted = ceil_div(edges, copies * 16);  // sixteen edges per copy at least
  parts = parts < wanted ? parts : wanted;
  cut.parts_of_edges = static_cast<int>(parts < 1 ? 1 : parts);
  return cut;
}
// For any packet: they differ in how many edges a CTA takes.
inline int64_t partial_numbers(int64_t size, int64_t acc_size, int64_t edges, int64_t num_buckets, int64_t heads) {
  int64_t parts = 1;
  for (int vec = 1; vec * size <= 16; vec <<= 1) {
    const Cut cut = cut_of(acc_size, vec, edges, num_buckets, heads);
    parts = parts > cut.parts_of_edges ? parts : cut.parts_of_edges;
  }
  return parts * num_buckets * heads;
}

template <typename T, int VEC>
int table_gradient(const T* g, const int32_t* buckets, T* gtable, void* scratch, int64_t edges, int64_t num_buckets, int64_t heads,
                   cudaStream_t stream) {
  using A = Acc<T>;
  const Cut cut = cut_of(sizeof(A), VEC, edges, num_buckets, heads);
  if (cut.parts_of_heads > 65535 || cut.parts_of_buckets > 65535)
    return fail(LUNA_ERR_UNSUPPORTED, "gradient of a table of %lld buckets and %lld heads", static_cast<long long>(num_buckets),
                static_cast<long long>(heads));
  LUNA_CUDA_CHECK(cudaFuncSetAttribute(table_kernel<T, VEC>, cudaFuncAttributeMaxDynamicSharedMemorySize, 200 * 1024));
  A* partial = static_cast<A*>(scratch);
  table_kernel<T, VEC><<<dim3(cut.parts_of_edges, cut.parts_of_heads, cut.parts_of_buckets), cut.threads, cut.shared, stream>>>(
      g, buckets, partial, edges, static_cast<int>(num_buckets), static_cast<int>(heads), cut);
  LUNA_LAUNCH_CHECK("gradient of the bias table");
  const int64_t numbers = num_buckets * heads;
  launch_early(table_final_kernel<T>, dim3(static_cast<unsigned>(ceil_div(numbers, 32))), 32 * kFinalSlices, 0, stream,
               static_cast<const A*>(partial), gtable, numbers, cut.parts_of_edges);
  LUNA_LAUNCH_CHECK("sums of the bias table");
  return LUNA_OK;
}

template <typename T>
int table_gradient(const void* g_, const int32_t* buckets, void* gtable_, void* scratch, int64_t edges, int64_t num_buckets,
                   int64_t heads, cudaStream_t stream) {
  const T* g = static_cast<const T*>(g_);
  T* gtable = static_cast<T*>(gtable_);
  switch (packet_of(sizeof(T), heads, {g})) {
    case 1: return table_gradient<T, 1>(g, buckets, gtable, scratch, edges, num_buckets, heads, stream);
    case 2: return table_gradient<T, 2>(g, buckets, gtable, scratch, edges, num_buckets, heads, stream);
    case 4:
      if constexpr (sizeof(T) <= 4) return table_gradient<T, 4>(g, buckets, gtable, scratch, edges, num_buckets, heads, stream);
      break;
    case 8:
      if constexpr (sizeof(T) <= 2) return table_gradient<T, 8>(g, buckets, gtable, scratch, edges, num_buckets, heads, stream);
      break;
  }
  return LUNA_ERR_UNSUPPORTED;
}

}  // namespace bias
}  // namespace luna
