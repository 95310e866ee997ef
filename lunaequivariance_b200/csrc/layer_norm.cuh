// Layer norm over irreps: forward, backward and second order, for rows of blocks `mul x l`.
//
// Of a block with elements x (d = 2l + 1 components for each of mul channels, n = mul d): mu = mean(x) for scalars and 0
// otherwise, s = (share |x - mu|^2 + eps)^(-1/2) with share = 1/n ("component") or 1/mul ("norm"), h = (x - mu) s, and
// y = w_u h + b_u.  With P t = t - mean(t) - share h <h, t> (the mean for scalars only; P is symmetric) and c = w g:
//   backward   gx = s P c,   gw_u = sum over rows and components of g h,   gb_u = sum of g
//   second     the cotangents r of gx, rw of gw and rb of gb, q = rw g, a = <r, h>, b = <c, h>, dot = <r, c> - n mean(r) mean(c):
//              hg = w s P r + rw h + rb,   hw_u = sum of s (P r) g,
//              hx = s P q - s^2 share ((dot - share a b) h + b P r + a P c)
//
// What bounds all of them is HBM: every row is read once and held in registers between its sums and its outputs.  Each block
// is normalised alone, so a CTA works on one block's columns of many rows: `lanes` threads (a power of two; up to a whole
// CTA) share a row, each with up to K packets of VEC elements, always the same columns, so that it keeps their weights and
// the sums of the weights' gradients in registers from row to row.  Those sums meet once per CTA and once more in a second
// launch, in an order that only the sizes decide: no atomics, the same bits every time.
#pragma once

#include <atomic>

#include "rows.cuh"

namespace luna {
namespace norm {

using rows::Acc;
using rows::Pack;

constexpr int kMaxBlocks = 32;
constexpr int kMaxLength = 16384;  // elements of a block

struct Block {
  int offset, length, components, scalar, weight_offset, bias_offset;
  int lanes;             // threads that share a row
  int first_cta, ctas;
  int64_t partial;       // first element of its CTAs' sums in the scratch buffer
  double share;
};

struct Params {
  int blocks, dim;
  int64_t rows;
  double eps;
  Block block[kMaxBlocks];
};

__device__ __forceinline__ const Block& block_of(const Params& P) {
  int i = 0;
  while (i + 1 < P.blocks && static_cast<int>(blockIdx.x) >= P.block[i + 1].first_cta) ++i;
  return P.block[i];
}

// The threads that share a row, and their sums.
template <typename A>
struct Team {
  int lanes, lane, index, teams;  // lane within the team, team within the CTA
  A* exchange;                    // [2][warps of the CTA][kMaxSums]
  int turn = 0;
  static constexpr int kMaxSums = 8;

  __device__ Team(int lanes_, A* exchange_) : lanes(lanes_), exchange(exchange_) {
    lane = threadIdx.x & (lanes - 1);
    index = threadIdx.x / lanes;
    teams = blockDim.x / lanes;
  }
  // The first of the team's warp's rows decides when a warp leaves its loop: lanes of a warp stay together.
  __device__ __forceinline__ int teams_before_warp() const { return lanes < 32 ? index - index % (32 / lanes) : index; }

  template <int V>
  __device__ __forceinline__ void sum(A (&v)[V]) {
    for (int off = (lanes < 32 ? lanes : 32) >> 1; off; off >>= 1)
#pragma unroll
      for (int i = 0; i < V; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], off);
    if (lanes <= 32) return;
    // Two buffers by turns: who writes the first one again has passed the barrier after which nobody reads it.
    const int warps = lanes >> 5, warp = threadIdx.x >> 5;
    A* at = exchange + turn * (blockDim.x >> 5) * kMaxSums;
    turn ^= 1;
    if ((threadIdx.x & 31) == 0)
#pragma unroll
      for (int i = 0; i < V; ++i) at[warp * kMaxSums + i] = v[i];
    asm volatile("bar.sync %0, %1;" ::"r"(index + 1), "r"(lanes) : "memory");
    const A* from = at + index * warps * kMaxSums;
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = from[i];
    for (int other = 1; other < warps; ++other)
#pragma unroll
      for (int i = 0; i < V; ++i) v[i] += from[other * kMaxSums + i];
  }
};

// One thread's columns of a block: which they are, and their parameters.
template <typename T, int VEC, int K>
struct Columns {
  using A = Acc<T>;
  int first, step, length;
  __device__ Columns(const Block& B, int lane) : first(lane * VEC), step(B.lanes * VEC), length(B.length) {}
  __device__ __forceinline__ int at(int k) const { return first + k * step; }
  __device__ __forceinline__ bool in(int k) const { return at(k) < length; }

  __device__ __forceinline__ void parameters(const T* __restrict__ p, int offset, int components, A otherwise, A (&to)[K][VEC]) const {
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int c = 0; c < VEC; ++c) to[k][c] = p && in(k) ? rows::widen(p[offset + (at(k) + c) / components]) : otherwise;
  }
  __device__ __forceinline__ void load(const T* __restrict__ row, bool active, A (&to)[K][VEC]) const {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      if (active && in(k)) {
        rows::load<T, VEC>(row + at(k), to[k]);
      } else {
#pragma unroll
        for (int c = 0; c < VEC; ++c) to[k][c] = A(0);
      }
    }
  }
};

template <typename A>
struct Moments {
  A mean, scale;
};

template <typename T, int VEC, int K, int THREADS>
__global__ void __launch_bounds__(THREADS)
forward_kernel(const __grid_constant__ Params P, const T* __restrict__ x, const T* __restrict__ weight,
               const T* __restrict__ bias, T* __restrict__ y, Moments<Acc<T>>* __restrict__ stats) {
  using A = Acc<T>;
  __shared__ A exchange[2 * (THREADS / 32) * Team<A>::kMaxSums];
  const Block& B = block_of(P);
  Team<A> team(B.lanes, exchange);
  const Columns<T, VEC, K> columns(B, team.lane);
  A w[K][VEC], b[K][VEC];
  columns.parameters(weight, B.weight_offset, B.components, A(1), w);
  columns.parameters(B.scalar ? bias : nullptr, B.bias_offset, B.components, A(0), b);
  const A share = static_cast<A>(B.share), eps = static_cast<A>(P.eps);
  const int64_t step = static_cast<int64_t>(B.ctas) * team.teams;
  const int64_t first = static_cast<int64_t>(blockIdx.x - B.first_cta) * team.teams;
  const int64_t block_index = &B - P.block;
  for (int64_t base = first; base + team.teams_before_warp() < P.rows; base += step) {
    const int64_t row = base + team.index;
    const bool active = row < P.rows;
    A v[K][VEC];
    columns.load(x + row * P.dim + B.offset, active, v);
    A mean = A(0);
    if (B.scalar) {
      A sums[1] = {A(0)};
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int c = 0; c < VEC; ++c) sums[0] += v[k][c];
      team.sum(sums);
      mean = sums[0] / static_cast<A>(B.length);
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int c = 0; c < VEC; ++c) v[k][c] = columns.in(k) ? v[k][c] - mean : A(0);
    }
    A sums[1] = {A(0)};
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int c = 0; c < VEC; ++c) sums[0] += v[k][c] * v[k][c];
    team.sum(sums);
    const A scale = A(1) / sqrt(sums[0] * share + eps);
    if (active) {
      T* to = y + row * P.dim + B.offset;
#pragma unroll
      for (int k = 0; k < K; ++k)
        if (columns.in(k)) {
#pragma unroll
          for (int c = 0; c < VEC; ++c) v[k][c] = v[k][c] * scale * w[k][c] + b[k][c];
          rows::store<T, VEC>(to + columns.at(k), v[k]);
        }
      if (stats && team.lane == 0) stats[block_index * P.rows + row] = Moments<A>{mean, scale};
    }
  }
}

// The sums of a CTA's teams for one array, written as one row of partial sums.
template <typename A, int VEC, int K>
__device__ __forceinline__ void store_partial(const Block& B, Team<A>& team, A (&sums)[K][VEC], A* tile, A* __restrict__ to) {
  for (int off = team.lanes; off < 32; off <<= 1)
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int c = 0; c < VEC; ++c) sums[k][c] += __shfl_xor_sync(0xffffffffu, sums[k][c], off);
  const int groups = team.lanes < 32 ? blockDim.x >> 5 : team.teams;
  const int group = team.lanes < 32 ? threadIdx.x >> 5 : team.index;
  if ((threadIdx.x & 31) < team.lanes) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int at = (k * team.lanes + team.lane) * VEC;
      if (at < B.length)
#pragma unroll
        for (int c = 0; c < VEC; ++c) tile[group * B.length + at + c] = sums[k][c];
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < B.length; i += blockDim.x) {
    A sum = tile[i];
    for (int other = 1; other < groups; ++other) sum += tile[other * B.length + i];
    to[i] = sum;
  }
  __syncthreads();
}

template <typename T, int VEC, int K, int THREADS>
__global__ void __launch_bounds__(THREADS)
backward_kernel(const __grid_constant__ Params P, const T* __restrict__ x, const T* __restrict__ weight,
                const Moments<Acc<T>>* __restrict__ stats, const T* __restrict__ g, T* __restrict__ gx,
                Acc<T>* __restrict__ partial) {
  using A = Acc<T>;
  extern __shared__ __align__(16) unsigned char raw[];
  __shared__ A exchange[2 * (THREADS / 32) * Team<A>::kMaxSums];
  const Block& B = block_of(P);
  Team<A> team(B.lanes, exchange);
  const Columns<T, VEC, K> columns(B, team.lane);
  A w[K][VEC], gw[K][VEC], gb[K][VEC];
  columns.parameters(weight, B.weight_offset, B.components, A(1), w);
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int c = 0; c < VEC; ++c) gw[k][c] = gb[k][c] = A(0);
  const A share = static_cast<A>(B.share);
  const int64_t step = static_cast<int64_t>(B.ctas) * team.teams;
  const int64_t first = static_cast<int64_t>(blockIdx.x - B.first_cta) * team.teams;
  const int64_t block_index = &B - P.block;
  for (int64_t base = first; base + team.teams_before_warp() < P.rows; base += step) {
    const int64_t row = base + team.index;
    const bool active = row < P.rows;
    A h[K][VEC], e[K][VEC];
    columns.load(x + row * P.dim + B.offset, active, h);
    columns.load(g + row * P.dim + B.offset, active, e);
    Moments<A> m{A(0), A(0)};
    if (active) m = stats[block_index * P.rows + row];
    A sums[2] = {A(0), A(0)};
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int c = 0; c < VEC; ++c) {
        h[k][c] = active && columns.in(k) ? (h[k][c] - m.mean) * m.scale : A(0);
        gw[k][c] += e[k][c] * h[k][c];
        gb[k][c] += e[k][c];
        e[k][c] *= w[k][c];
        sums[0] += e[k][c] * h[k][c];
        sums[1] += e[k][c];
      }
    if (gx) {
      team.sum(sums);
      const A along = sums[0] * share, mean = B.scalar ? sums[1] / static_cast<A>(B.length) : A(0);
      if (active) {
        T* to = gx + row * P.dim + B.offset;
#pragma unroll
        for (int k = 0; k < K; ++k)
          if (columns.in(k)) {
#pragma unroll
            for (int c = 0; c < VEC; ++c) e[k][c] = m.scale * (e[k][c] - mean - h[k][c] * along);
            rows::store<T, VEC>(to + columns.at(k), e[k]);
          }
      }
    }
  }
  if (!partial) return;
  A* to = partial + B.partial + static_cast<int64_t>(blockIdx.x - B.first_cta) * 2 * B.length;
  A* tile = reinterpret_cast<A*>(raw);
  store_partial(B, team, gw, tile, to);
  if (B.scalar) store_partial(B, team, gb, tile, to + B.length);
}

template <typename T, int VEC, int K, int THREADS>
__global__ void __launch_bounds__(THREADS)
second_kernel(const __grid_constant__ Params P, const T* __restrict__ x, const T* __restrict__ weight,
              const Moments<Acc<T>>* __restrict__ stats, const T* __restrict__ g, const T* __restrict__ rx,
              const T* __restrict__ rw, const T* __restrict__ rb, T* __restrict__ hx, T* __restrict__ hg,
              Acc<T>* __restrict__ partial) {
  using A = Acc<T>;
  extern __shared__ __align__(16) unsigned char raw[];
  __shared__ A exchange[2 * (THREADS / 32) * Team<A>::kMaxSums];
  const Block& B = block_of(P);
  Team<A> team(B.lanes, exchange);
  const Columns<T, VEC, K> columns(B, team.lane);
  A w[K][VEC], hw[K][VEC];
  columns.parameters(weight, B.weight_offset, B.components, A(1), w);
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int c = 0; c < VEC; ++c) hw[k][c] = A(0);
  const A share = static_cast<A>(B.share);
  const int64_t step = static_cast<int64_t>(B.ctas) * team.teams;
  const int64_t first = static_cast<int64_t>(blockIdx.x - B.first_cta) * team.teams;
  const int64_t block_index = &B - P.block;
  // rw and rb are as short as a row and the same for all of them: read again from cache instead of kept
  auto other = [&](const T* __restrict__ p, int offset, int k, int c) {
    return p ? rows::widen(p[offset + (columns.at(k) + c) / B.components]) : A(0);
  };
  for (int64_t base = first; base + team.teams_before_warp() < P.rows; base += step) {
    const int64_t row = base + team.index;
    const bool active = row < P.rows;
    A h[K][VEC], e[K][VEC], r[K][VEC];
    columns.load(x + row * P.dim + B.offset, active, h);
    columns.load(g + row * P.dim + B.offset, active, e);
    columns.load(rx ? rx + row * P.dim + B.offset : nullptr, active && rx, r);
    Moments<A> m{A(0), A(0)};
    if (active) m = stats[block_index * P.rows + row];
    A sums[5] = {A(0), A(0), A(0), A(0), A(0)}, more[2] = {A(0), A(0)};  // rh, ch, rc, r, c; q, qh
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int c = 0; c < VEC; ++c) {
        h[k][c] = active && columns.in(k) ? (h[k][c] - m.mean) * m.scale : A(0);
        const A scaled = e[k][c] * w[k][c];
        sums[0] += r[k][c] * h[k][c];
        sums[1] += scaled * h[k][c];
        sums[2] += r[k][c] * scaled;
        sums[3] += r[k][c];
        sums[4] += scaled;
        if (rw && columns.in(k)) {
          const A q = other(rw, B.weight_offset, k, c) * e[k][c];
          more[0] += q;
          more[1] += q * h[k][c];
        }
      }
    team.sum(sums);
    if (rw) team.sum(more);
    const A length = static_cast<A>(B.length);
    const A mean_r = B.scalar ? sums[3] / length : A(0), mean_c = B.scalar ? sums[4] / length : A(0);
    const A mean_q = B.scalar ? more[0] / length : A(0);
    const A dot = sums[2] - length * mean_r * mean_c;
    const A along_r = share * sums[0], along_c = share * sums[1], along_q = share * more[1];
    const A outer = m.scale * m.scale * share, on_h = dot - share * sums[0] * sums[1];
    if (active) {
      const int64_t at = row * P.dim + B.offset;
#pragma unroll
      for (int k = 0; k < K; ++k)
        if (columns.in(k)) {
#pragma unroll
          for (int c = 0; c < VEC; ++c) {
            const A p = r[k][c] - mean_r - h[k][c] * along_r;
            const A scaled = e[k][c] * w[k][c] - mean_c - h[k][c] * along_c;
            const A tangent = rw ? other(rw, B.weight_offset, k, c) : A(0);
            const A q = rw ? tangent * e[k][c] - mean_q - h[k][c] * along_q : A(0);
            hw[k][c] += m.scale * p * e[k][c];
            e[k][c] = w[k][c] * m.scale * p + tangent * h[k][c] + (B.scalar ? other(rb, B.bias_offset, k, c) : A(0));
            r[k][c] = m.scale * q - outer * (on_h * h[k][c] + sums[1] * p + sums[0] * scaled);
          }
          if (hg) rows::store<T, VEC>(hg + at + columns.at(k), e[k]);
          if (hx) rows::store<T, VEC>(hx + at + columns.at(k), r[k]);
        }
    }
  }
  if (!partial) return;
  store_partial(B, team, hw, reinterpret_cast<A*>(raw), partial + B.partial + static_cast<int64_t>(blockIdx.x - B.first_cta) * 2 * B.length);
}

// The sums of all CTAs, for 32 channels of a block by one CTA: 16 threads take every sixteenth CTA's sums of a channel each.
constexpr int kFinalSlices = 16;
template <typename T>
__global__ void __launch_bounds__(32 * kFinalSlices)
final_kernel(const __grid_constant__ Params P, const Acc<T>* __restrict__ partial, T* __restrict__ gw, T* __restrict__ gb) {
  using A = Acc<T>;
  __shared__ A tile[2][kFinalSlices][32];
  wait_for_previous();
  int i = 0, cta = blockIdx.x;  // which block, and which 32 of its channels
  auto channels = [&](int j) { return P.block[j].length / P.block[j].components; };
  while (cta >= (channels(i) + 31) / 32) cta -= (channels(i++) + 31) / 32;
  const Block& B = P.block[i];
  const int lane = threadIdx.x & 31, slice = threadIdx.x >> 5, u = cta * 32 + lane, count = channels(i);
  A sum[2] = {A(0), A(0)};
  if (u < count) {
    const A* from = partial + B.partial + static_cast<int64_t>(u) * B.components;
    for (int j = slice; j < B.ctas; j += kFinalSlices) {
      const A* row = from + static_cast<int64_t>(j) * 2 * B.length;
      if (gw)
        for (int m = 0; m < B.components; ++m) sum[0] += row[m];
      if (gb && B.scalar) sum[1] += row[B.length];
    }
  }
  tile[0][slice][lane] = sum[0];
  tile[1][slice][lane] = sum[1];
  __syncthreads();
  if (slice >= 2 || u >= count) return;
  A total = A(0);
#pragma unroll
  for (int j = 0; j < kFinalSlices; ++j) total += tile[slice][j][lane];
  if (slice == 0 && gw) rows::narrow(total, gw[B.weight_offset + u]);
  if (slice == 1 && gb && B.scalar) rows::narrow(total, gb[B.bias_offset + u]);
}

// ---- launches --------------------------------------------------------------------------------------------------------------

struct Operands {
  const void *x, *weight, *bias, *stats_in, *g, *rx, *rw, *rb;
  void *y, *stats_out, *gx, *gw, *gb, *hx, *hg;
  void* scratch;
  int64_t scratch_bytes;
};
enum Order { kForward, kBackward, kSecond };

inline int blocks_on_device(const void* kernel, int threads, size_t shared) {
  int resident = 0;
  if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&resident, kernel, threads, shared) != cudaSuccess || resident < 1) resident = 1;
  return resident * rows::processors();
}

// Gives every block its threads per row and its CTAs: as many as its rows want, or its share of the resident ones.
inline int assign(Params& P, int vec, int packets, int threads, int resident) {
  int64_t wanted = 0;
  for (int i = 0; i < P.blocks; ++i) {
    Block& B = P.block[i];
    B.lanes = rows::next_power_of_two(ceil_div(ceil_div(B.length, vec), packets));
    if (B.lanes > 32 && threads / B.lanes > 15) B.lanes = threads / 8;  // a CTA has fifteen barriers beside its own
    wanted += ceil_div(P.rows, threads / B.lanes);
  }
  int ctas = 0;
  int64_t partial = 0;
  for (int i = 0; i < P.blocks; ++i) {
    Block& B = P.block[i];
    int64_t count = ceil_div(P.rows, threads / B.lanes);
    if (wanted > resident) {
      const int64_t part = static_cast<int64_t>(resident) * B.length / P.dim;
      count = count < part ? count : (part < 1 ? 1 : part);
    }
    B.first_cta = ctas;
    B.ctas = static_cast<int>(count);
    B.partial = partial;
    ctas += B.ctas;
    partial += count * 2 * B.length;
  }
  return ctas;
}
constexpr int kThreads = 256, kWideThreads = 1024;
// At most this many CTAs of kThreads are resident on a multiprocessor, whatever a kernel needs.
constexpr int kMostResident = 2048 / kThreads;

inline int64_t scratch_elements(const Params& P) {
  const int64_t resident = static_cast<int64_t>(kMostResident) * rows::processors();
  return (P.rows < resident ? P.rows : resident) * 2 * P.dim + 2;  // never zero: a buffer of no bytes has no address
}

template <typename T, int VEC, int K, int THREADS>
int launch(Order order, Params P, const Operands& o, cudaStream_t stream) {
  using A = Acc<T>;
  auto in = [](const void* p) { return static_cast<const T*>(p); };
  auto out = [](void* p) { return static_cast<T*>(p); };
  const Moments<A>* stats = static_cast<const Moments<A>*>(o.stats_in);
  // Room for the sums of the CTA's threads: at most all of them
  const size_t shared = order == kForward ? 0 : static_cast<size_t>(THREADS) * K * VEC * sizeof(A);
  const bool sums = order != kForward && (o.gw || o.gb);
  const void* kernel = order == kForward    ? reinterpret_cast<const void*>(forward_kernel<T, VEC, K, THREADS>)
                       : order == kBackward ? reinterpret_cast<const void*>(backward_kernel<T, VEC, K, THREADS>)
                                            : reinterpret_cast<const void*>(second_kernel<T, VEC, K, THREADS>);
  if (shared > 48 * 1024) LUNA_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(shared)));
  static std::atomic<int> known[3];
  int resident = known[order].load(std::memory_order_relaxed);
  if (!resident) {
    resident = blocks_on_device(kernel, THREADS, shared);
    if (resident < 1) return fail(LUNA_ERR_CUDA, "the current device's multiprocessors are unknown");
    known[order].store(resident, std::memory_order_relaxed);
  }
  const int ctas = assign(P, VEC, K, THREADS, resident);
  A* partial = sums ? static_cast<A*>(o.scratch) : nullptr;
  if (ctas > 0) {
    if (order == kForward)
      forward_kernel<T, VEC, K, THREADS><<<ctas, THREADS, 0, stream>>>(P, in(o.x), in(o.weight), in(o.bias), out(o.y),
                                                                       static_cast<Moments<A>*>(o.stats_out));
    else if (order == kBackward)
      backward_kernel<T, VEC, K, THREADS><<<ctas, THREADS, shared, stream>>>(P, in(o.x), in(o.weight), stats, in(o.g), out(o.gx), partial);
    else
      second_kernel<T, VEC, K, THREADS><<<ctas, THREADS, shared, stream>>>(P, in(o.x), in(o.weight), stats, in(o.g), in(o.rx), in(o.rw),
                                                                           in(o.rb), out(o.hx), out(o.hg), partial);
    LUNA_LAUNCH_CHECK("layer norm");
  }
  if (sums) {
    int tasks = 0;
    for (int i = 0; i < P.blocks; ++i) tasks += static_cast<int>(ceil_div(P.block[i].length / P.block[i].components, 32));
    launch_early(final_kernel<T>, dim3(tasks), 32 * kFinalSlices, 0, stream, P, static_cast<const A*>(partial), out(o.gw), out(o.gb));
    LUNA_LAUNCH_CHECK("sums of the layer norm");
  }
  return LUNA_OK;
}

template <typename T>
int run(Order order, const Params& P, const Operands& o, cudaStream_t stream) {
  constexpr int kPacket = 16 / static_cast<int>(sizeof(T));
  bool packets = P.dim % kPacket == 0;
  int64_t longest = 0;
  for (int i = 0; i < P.blocks; ++i) {
    packets = packets && P.block[i].offset % kPacket == 0 && P.block[i].length % kPacket == 0;
    longest = P.block[i].length > longest ? P.block[i].length : longest;
  }
  for (const void* p : {o.x, o.g, o.rx, static_cast<const void*>(o.y), static_cast<const void*>(o.gx), static_cast<const void*>(o.hx),
                        static_cast<const void*>(o.hg)})
    packets = packets && aligned_to(p, 16);
  if (packets) {
    const int64_t n = longest / kPacket;
    if (n <= 32) return launch<T, kPacket, 1, kThreads>(order, P, o, stream);
    if (n <= 64) return launch<T, kPacket, 2, kThreads>(order, P, o, stream);
    if (n <= kThreads * 4) return launch<T, kPacket, 4, kThreads>(order, P, o, stream);
    if (n <= kWideThreads * 4) return launch<T, kPacket, 4, kWideThreads>(order, P, o, stream);
  }
  if (longest <= 32) return launch<T, 1, 1, kThreads>(order, P, o, stream);
  if (longest <= kThreads * 4) return launch<T, 1, 4, kThreads>(order, P, o, stream);
  if (longest <= kThreads * 16) return launch<T, 1, 16, kThreads>(order, P, o, stream);
  return launch<T, 1, 16, kWideThreads>(order, P, o, stream);
}

extern template int run<float>(Order, const Params&, const Operands&, cudaStream_t);
extern template int run<double>(Order, const Params&, const Operands&, cudaStream_t);
extern template int run<rows::bf16>(Order, const Params&, const Operands&, cudaStream_t);
extern template int run<rows::f16>(Order, const Params&, const Operands&, cudaStream_t);

}  // namespace norm
}  // namespace luna
