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
// run of AHEAD edges of the CTA's and add their rows to the copy, each thread to columns of its own: no two threads add to one
// number, so there are no atomics, and the order of the sums depends on the sizes, on how g is aligned (its packets) and on the
// number of multiprocessors.  The copies are summed at the end,
// the CTAs' sums in a second launch.
//
// Large tables leave room for few copies, so few warps, and what counts is how long an addition takes one of them: a run is
// under way while the one before is added, its addresses are one base and its buckets one or a few wide loads, and two edges
// are added at a time: their sums are read together, and the second takes over the first's where both are of one bucket.
// (Four edges at a time and nothing under way: 2.6 M edges of 16 heads and 128 buckets 171 us.)
struct Cut {
  int lanes, copies, threads;  // threads per copy; copies and threads of a CTA
  int buckets;                 // rows of the table that a CTA has; each copy has one more, for what belongs to none
  int parts_of_edges, parts_of_heads, parts_of_buckets;
  int64_t shared;              // bytes
};

template <typename T, int VEC, int AHEAD>
__global__ void __launch_bounds__(256)
table_kernel(const T* __restrict__ g, const int32_t* __restrict__ buckets, Acc<T>* __restrict__ partial, int64_t edges,
             int num_buckets, int heads, Cut cut, bool wide_buckets) {
  using A = Acc<T>;
  extern __shared__ __align__(16) unsigned char raw[];
  A* tables = reinterpret_cast<A*>(raw);
  const int width = cut.lanes * VEC, copy_size = (cut.buckets + 1) * width;
  const int first_bucket = blockIdx.z * cut.buckets, first_head = blockIdx.y * width;
  const int last_bucket = num_buckets - first_bucket < cut.buckets ? num_buckets - first_bucket : cut.buckets;
  const int lane = threadIdx.x & (cut.lanes - 1), copy = threadIdx.x / cut.lanes;
  const int head = first_head + lane * VEC;
  const int64_t runs = (edges + AHEAD - 1) / AHEAD, first_run = runs * blockIdx.x / gridDim.x, last_run = runs * (blockIdx.x + 1) / gridDim.x;
  const bool works = copy < cut.copies && head < heads;
  // this copy's runs, and the edges behind the beginning of its next one
  const int count = works && last_run - first_run > copy ? static_cast<int>((last_run - first_run - copy + cut.copies - 1) / cut.copies) : 0;
  int64_t at = (first_run + copy) * AHEAD;
  const int32_t* bucket_at = buckets + at;
  const T* g_at = g + at * heads + head;
  const int run_step = cut.copies * AHEAD;
  const int64_t g_step = static_cast<int64_t>(run_step) * heads;
  using In = rows::Pack<T, VEC>;
  using Sum = rows::Pack<A, VEC>;
  struct Run {
    In v[AHEAD];
    int row[AHEAD];
  };
  auto fetch = [&](Run& to, int number) {
    // The run after the next one is called into L2: registers hold one run under way, which does not cover the way to memory.
    if (number + 2 < count && at + 2 * static_cast<int64_t>(run_step) + AHEAD <= edges) {
      const char* line = reinterpret_cast<const char*>(g_at + 2 * g_step - lane * VEC);
      for (int i = lane * 128; i < (AHEAD * heads - first_head) * static_cast<int>(sizeof(T)); i += cut.lanes * 128)
        asm volatile("prefetch.global.L2 [%0];" ::"l"(line + i));
      if (lane == 0) asm volatile("prefetch.global.L2 [%0];" ::"l"(bucket_at + 2 * run_step));
    }
    if (number < count && at + AHEAD <= edges) {
      if (wide_buckets) {
#pragma unroll
        for (int j = 0; j < AHEAD; j += 4) {
          const int4 four = *reinterpret_cast<const int4*>(bucket_at + j);
          to.row[j] = four.x, to.row[j + 1] = four.y, to.row[j + 2] = four.z, to.row[j + 3] = four.w;
        }
      } else {
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) to.row[j] = bucket_at[j];
      }
#pragma unroll
      for (int j = 0; j < AHEAD; ++j) to.v[j] = *reinterpret_cast<const In*>(g_at + j * heads);
    } else {  // the last run of all may be shorter
#pragma unroll
      for (int j = 0; j < AHEAD; ++j) {
        to.row[j] = -1;
        if (number < count && at + j < edges) {
          to.row[j] = bucket_at[j];
          to.v[j] = *reinterpret_cast<const In*>(g_at + j * heads);
        }
      }
    }
    at += run_step;
    bucket_at += run_step;
    g_at += g_step;
  };
  A* mine = tables + copy * copy_size + lane * VEC;
  auto place = [&](int row) {  // a row of another part, or none at all, goes to the row behind the last
    return static_cast<int>(min(static_cast<unsigned>(row) - static_cast<unsigned>(first_bucket), static_cast<unsigned>(last_bucket))) * width;
  };
  auto add = [&](const Run& from) {
#pragma unroll
    for (int j = 0; j < AHEAD; j += 2) {
      const int p = place(from.row[j]), q = place(from.row[j + 1]);
      Sum s = *reinterpret_cast<const Sum*>(mine + p), t = *reinterpret_cast<const Sum*>(mine + q);
#pragma unroll
      for (int c = 0; c < VEC; ++c) {
        s.a[c] += rows::widen(from.v[j].a[c]);
        t.a[c] = (p == q ? s.a[c] : t.a[c]) + rows::widen(from.v[j + 1].a[c]);
      }
      *reinterpret_cast<Sum*>(mine + p) = s;
      *reinterpret_cast<Sum*>(mine + q) = t;
    }
  };
  Run one, other;
  fetch(one, 0);
  {
    const Sum zeros{};
    for (int i = threadIdx.x * VEC; i < cut.copies * copy_size; i += blockDim.x * VEC) *reinterpret_cast<Sum*>(tables + i) = zeros;
  }
  __syncthreads();
  for (int i = 0; i < count; i += 2) {
    fetch(other, i + 1);
    add(one);
    if (i + 1 >= count) break;
    fetch(one, i + 2);
    add(other);
  }
  __syncthreads();
  for (int i = threadIdx.x * VEC; i < last_bucket * width; i += blockDim.x * VEC) {
    const int bucket = first_bucket + i / width, h = first_head + i % width;
    if (h >= heads) continue;  // whole packets: VEC divides the heads
    Sum sum = *reinterpret_cast<const Sum*>(tables + i);
    for (int other_copy = 1; other_copy < cut.copies; ++other_copy) {
      const Sum more = *reinterpret_cast<const Sum*>(tables + other_copy * copy_size + i);
#pragma unroll
      for (int c = 0; c < VEC; ++c) sum.a[c] += more.a[c];
    }
    *reinterpret_cast<Sum*>(partial + (static_cast<int64_t>(blockIdx.x) * num_buckets + bucket) * heads + h) = sum;
  }
}

// The sums of all CTAs: 32 numbers of the table by one CTA, 32 threads for each.
constexpr int kFinalSlices = 32;
template <typename T>
__global__ void __launch_bounds__(32 * kFinalSlices)
table_final_kernel(const Acc<T>* __restrict__ partial, T* __restrict__ gtable, int64_t numbers, int parts) {
  using A = Acc<T>;
  __shared__ A tile[kFinalSlices][33];
  wait_for_previous();
  const int lane = threadIdx.x & 31, slice = threadIdx.x >> 5;
  const int64_t first = static_cast<int64_t>(blockIdx.x) * 32;
  A sum = A(0);
  if (first + lane < numbers) {
#pragma unroll 8
    for (int j = slice; j < parts; j += kFinalSlices) sum += partial[j * numbers + first + lane];
  }
  tile[slice][lane] = sum;
  __syncthreads();
  A total = tile[lane][slice];  // a warp's threads have the slices of one number
  for (int off = 16; off; off >>= 1) total += __shfl_xor_sync(0xffffffffu, total, off);
  if (lane == 0 && first + slice < numbers) rows::narrow(total, gtable[first + slice]);
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

// How the table's gradient is cut up for packets of `vec`.
inline Cut cut_of(int64_t acc_size, int vec, int64_t edges, int64_t num_buckets, int64_t heads) {
  constexpr int64_t kRoom = 208 * 1024;  // of a multiprocessor's shared memory
  Cut cut{};
  const int64_t packets = ceil_div(heads, vec);
  cut.lanes = packets >= 32 ? 32 : rows::next_power_of_two(packets);
  auto copy_bytes = [&] { return (num_buckets + 1) * cut.lanes * vec * acc_size; };
  while (cut.lanes > 1 && copy_bytes() > kRoom) cut.lanes >>= 1;
  const int64_t row_bytes = cut.lanes * vec * acc_size;
  cut.buckets = static_cast<int>(copy_bytes() > kRoom ? kRoom / row_bytes - 1 : num_buckets);
  const int64_t copy = (cut.buckets + 1) * row_bytes;
  const int64_t most = 256 / cut.lanes;
  int64_t copies = kRoom / copy;
  copies = copies < 1 ? 1 : (copies > most ? most : copies);
  cut.parts_of_heads = static_cast<int>(ceil_div(packets, cut.lanes));
  cut.parts_of_buckets = static_cast<int>(ceil_div(num_buckets, cut.buckets));
  const int64_t others = cut.parts_of_heads * static_cast<int64_t>(cut.parts_of_buckets);
  // fewer copies where there are not eight edges (a run) for each of a GPU full of them
  const int64_t each = ceil_div(edges, (rows::processors() > 0 ? rows::processors() : 1) * 8);
  copies = copies < each ? copies : (each < 1 ? 1 : each);
  cut.copies = static_cast<int>(copies);
  cut.threads = static_cast<int>(ceil_div(copies * cut.lanes, 32) * 32);
  cut.shared = copies * copy;
  const int64_t together = kRoom / cut.shared;
  const int64_t resident = rows::processors() * (together < 1 ? 1 : (together > 4 ? 4 : together));
  int64_t parts = resident / others;
  const int64_t wanted = ceil_div(edges, copies * 8);  // eight edges per copy at least
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

// TO: the type of the table, if it is narrower than its gradient's parts.
template <typename T, typename TO, int VEC>
int table_gradient(const T* g, const int32_t* buckets, TO* gtable, void* scratch, int64_t edges, int64_t num_buckets, int64_t heads,
                   cudaStream_t stream) {
  using A = Acc<T>;
  const Cut cut = cut_of(sizeof(A), VEC, edges, num_buckets, heads);
  if (cut.parts_of_heads > 65535 || cut.parts_of_buckets > 65535)
    return fail(LUNA_ERR_UNSUPPORTED, "gradient of a table of %lld buckets and %lld heads", static_cast<long long>(num_buckets),
                static_cast<long long>(heads));
  A* partial = static_cast<A*>(scratch);
  // more edges under way where a multiprocessor has few threads
  constexpr int kMany = VEC * sizeof(A) > 16 ? 8 : 16;  // packets of eight: the registers of eight edges are all
  const auto kernel = cut.threads > 128 ? table_kernel<T, VEC, 8> : table_kernel<T, VEC, kMany>;
  static rows::Kernel known[2];
  if (const int status = known[cut.threads > 128].allow(kernel, static_cast<size_t>(cut.shared))) return status;
  kernel<<<dim3(cut.parts_of_edges, cut.parts_of_heads, cut.parts_of_buckets), cut.threads, cut.shared, stream>>>(
      g, buckets, partial, edges, static_cast<int>(num_buckets), static_cast<int>(heads), cut, aligned_to(buckets, 16));
  LUNA_LAUNCH_CHECK("gradient of the bias table");
  const int64_t numbers = num_buckets * heads;
  launch_early(table_final_kernel<TO>, dim3(static_cast<unsigned>(ceil_div(numbers, 32))), 32 * kFinalSlices, 0, stream,
               static_cast<const A*>(partial), gtable, numbers, cut.parts_of_edges);
  LUNA_LAUNCH_CHECK("sums of the bias table");
  return LUNA_OK;
}

template <typename T, typename TO>
int table_gradient(const void* g_, const int32_t* buckets, void* gtable_, void* scratch, int64_t edges, int64_t num_buckets,
                   int64_t heads, cudaStream_t stream) {
  const T* g = static_cast<const T*>(g_);
  TO* gtable = static_cast<TO*>(gtable_);
  switch (packet_of(sizeof(T), heads, {g})) {
    case 1: return table_gradient<T, TO, 1>(g, buckets, gtable, scratch, edges, num_buckets, heads, stream);
    case 2: return table_gradient<T, TO, 2>(g, buckets, gtable, scratch, edges, num_buckets, heads, stream);
    case 4:
      if constexpr (sizeof(T) <= 4) return table_gradient<T, TO, 4>(g, buckets, gtable, scratch, edges, num_buckets, heads, stream);
      break;
    case 8:
      if constexpr (sizeof(T) <= 2) return table_gradient<T, TO, 8>(g, buckets, gtable, scratch, edges, num_buckets, heads, stream);
      break;
  }
  return LUNA_ERR_UNSUPPORTED;
}

}  // namespace bias
}  // namespace luna
