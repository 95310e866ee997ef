// Layer norm over irreps: forward, backward and second order, for rows of blocks `mul x l`.
//
// Of a block with elements x (d = 2l + 1 components for each of mul channels, n = mul d): mu = mean(x) for scalars and 0
// otherwise, s = (share |x - mu|^2 + eps)^(-1/2) with share = 1/n ("component") or 1/mul ("norm"), h = (x - mu) s, and
// y = w_u h + b_u.  With P t = t - mean(t) - share h <h, t> (the mean for scalars only; P is symmetric) and c = w g:
//   backward   gx = s P c,   gw_u = sum over rows and components of g h,   gb_u = sum of g
//   second     the cotangents r of gx, rw of gw and rb of gb, q = rw g, a = <r, h>, b = <c, h>, dot = <r - mean(r), c - mean(c)>:
//              hg = w s P r + rw h + rb,   hw_u = sum of s (P r) g,
//              hx = s P q - s^2 share ((dot - share a b) h + b P r + a P c)
//
// What bounds all of them is HBM: every row is read once and held in registers between its sums and its outputs.  Each block
// is normalised alone, so a CTA works on one block's columns of many rows: `lanes` threads (a power of two; up to a whole
// CTA) share a row, each with up to K packets of VEC elements, always the same columns, so that it keeps their weights and
// the sums of the weights' gradients in registers from row to row.  Those sums meet once per CTA and once more in a second
// launch, without atomics, in an order that the sizes, the alignment of the arrays and the device decide: the same call gives the same bits.
//
// Rows arrive in shared memory by asynchronous copies, one round ahead of their use, so that the memory is busy while sums
// are made.  Each thread copies what it will read itself, in the widest packets that the rows allow, and waits for nobody.  16-bit
// rows of an odd length, which no asynchronous copy can begin at, are moved a CTA's round of rows at a time, one contiguous chunk
// in aligned pieces, and read and written number by number in shared memory (20,011 rows of 1001 BF16: forward 77 -> 50 us, backward 75
// -> 59).  Rows wider than a CTA of 256 holds, and such rows of several blocks, are read when they are wanted.
#pragma once

#include <algorithm>
#include <type_traits>

#include "rows.cuh"

namespace luna {
namespace norm {

using rows::Acc;
using rows::Pack;

constexpr int kMaxBlocks = 32;
constexpr int kMaxLength = 16384;  // elements of a block
constexpr int kThreads = 256, kWideThreads = 1024;

struct Block {
  int offset, length, channels, components, scalar, weight_offset, bias_offset;
  unsigned inverse;      // 2^32 / components, rounded up: i / components is the upper half of i * inverse for i <= kMaxLength
  int lanes;             // threads that share a row
  int chunk;             // bytes of shared memory for a CTA's round of rows
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

__device__ __forceinline__ int block_index_of(const Params& P) {
  int i = 0;
  while (i + 1 < P.blocks && static_cast<int>(blockIdx.x) >= P.block[i + 1].first_cta) ++i;
  return i;
}

template <typename A>
struct Moments {
  A mean, scale;
};

template <int BYTES>
__device__ __forceinline__ void copy_async(void* to, const void* from) {
  const unsigned address = static_cast<unsigned>(__cvta_generic_to_shared(to));
  if constexpr (BYTES == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(address), "l"(from) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(address), "l"(from), "n"(BYTES) : "memory");
}
__device__ __forceinline__ void commit_copies() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int LEFT>
__device__ __forceinline__ void wait_copies() {
  asm volatile("cp.async.wait_group %0;" ::"n"(LEFT) : "memory");
}

constexpr int kMaxSums = 8;

enum Mode { kPackets, kChunks, kDirect };
constexpr int kStages = 2;  // rounds of rows on their way

// A thread's place: which columns of the CTA's block it has, and of which rows.  LANES: threads of a warp that share a row;
// where they are all of a warp, several warps may share it.  IN arrays are read, and chunks keep room for OUT.
template <typename T, int VEC, int K, int LANES, int MODE, int IN, int OUT>
struct Place {
  using A = Acc<T>;
  static constexpr int kBytes = MODE == kPackets ? VEC * static_cast<int>(sizeof(T)) : 16;  // of a copy: 4, 8 or 16
  static constexpr int kStep = LANES * VEC;   // from one of a thread's packets to the next
  static constexpr int kPiece = kStep * K;    // columns of a warp
  const Block& B;
  int lane, warps, warp, team, teams;         // in the row's part of this warp; warps per row; of the row; row of the CTA
  int begin, left;                            // first column of the warp's piece; columns from the thread's first one on
  A* exchange;
  unsigned char* shared;
  int turn = 0, stage = 0;
  const T* coming[IN];                        // chunks: where the next round to be asked for begins, and
  int64_t rest;                               // the rows from there on

  __device__ __forceinline__ Place(const Params& P, const Block& B_, const T* const (&arrays)[IN], unsigned char* shared_, A* exchange_)
      : B(B_), exchange(exchange_), shared(shared_) {
    const int in_cta = threadIdx.x >> 5;
    lane = threadIdx.x & (LANES - 1);
    warps = LANES == 32 ? B.lanes >> 5 : 1;
    warp = LANES == 32 ? in_cta & (warps - 1) : 0;
    team = LANES == 32 ? in_cta / warps : threadIdx.x / LANES;
    teams = LANES == 32 ? (blockDim.x >> 5) / warps : blockDim.x / LANES;
    begin = warp * kPiece;
    left = B.length - begin - lane * VEC;
    if (MODE == kChunks) {
      const int64_t first = static_cast<int64_t>(blockIdx.x - B.first_cta) * teams;
      rest = P.rows - first;
#pragma unroll
      for (int a = 0; a < IN; ++a) coming[a] = arrays[a] ? arrays[a] + first * B.length : nullptr;
    }
  }
  // Teams before this one whose loop this team shares: those of a warp, or of the CTA where it moves rows together.
  __device__ __forceinline__ int ahead() const { return MODE == kChunks ? team : LANES == 32 ? 0 : (threadIdx.x & 31) / LANES; }
  __device__ __forceinline__ bool in(int k) const { return k * kStep < left; }
  __device__ __forceinline__ int column(int k) const { return begin + lane * VEC + k * kStep; }
  __device__ __forceinline__ int channel(int i) const { return B.components == 1 ? i : static_cast<int>(__umulhi(i, B.inverse)); }
  // Packets: a thread's own, those of a warp's threads side by side.  Chunks: one array's after the other's.
  __device__ __forceinline__ unsigned char* packet(int array, int k) const { return shared + ((array * K + k) * blockDim.x + threadIdx.x) * kBytes; }
  __device__ __forceinline__ unsigned char* chunk(int array) const { return shared + array * B.chunk; }
  static __device__ __forceinline__ int shift_of(const T* p) { return static_cast<int>(reinterpret_cast<uintptr_t>(p) & 15); }

  __device__ __forceinline__ void parameters(const T* __restrict__ p, int offset, A otherwise, A (&to)[K][VEC]) const {
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int c = 0; c < VEC; ++c) to[k][c] = p && in(k) ? rows::widen(p[offset + channel(column(k) + c)]) : otherwise;
  }

  // Starts the copies of a round of rows, of which `row` is this team's, from arrays of P.rows rows.  Rounds are asked for in order.
  // They refill what has been read before.  A copy is ordered with the thread's own reads by a barrier, not by standing behind
  // them: that of the warp for packets, which costs nothing that could be measured, that of the CTA, which is there, for chunks.
  __device__ __forceinline__ void request(const Params& P, const T* const (&arrays)[IN], int64_t row) {
    if (MODE == kDirect) return;
    if (MODE == kPackets) {
      __syncwarp();
#pragma unroll
      for (int a = 0; a < IN; ++a) {
        if (!arrays[a]) continue;
        const T* from = arrays[a] + row * P.dim + B.offset + column(0);
#pragma unroll
        for (int k = 0; k < K; ++k)
          if (row < P.rows && in(k)) copy_async<kBytes>(packet(stage * IN + a, k), from + k * kStep);
      }
    } else if (rest > 0) {
      const int bytes = (rest < teams ? static_cast<int>(rest) : teams) * B.length * static_cast<int>(sizeof(T));
      const bool inner = rest >= 2 * teams;  // another round behind this one: more than 16 bytes
      const int64_t next = static_cast<int64_t>(B.ctas) * teams;
#pragma unroll
      for (int a = 0; a < IN; ++a) {
        if (!coming[a]) continue;
        const int shift = shift_of(coming[a]), pieces = (shift + bytes + 15) >> 4;
        const unsigned char* base = reinterpret_cast<const unsigned char*>(coming[a]) - shift;
        unsigned char* to = chunk(stage * IN + a);
        // the first piece may begin before the array, and the last one end after it: then what is inside of them, at once
        const int low = shift == 0 || coming[a] != arrays[a] ? 0 : 1, high = inner ? pieces : pieces - 1;
        for (int i = threadIdx.x; i < high; i += blockDim.x)
          if (i >= low) copy_async<16>(to + i * 16, base + i * 16);
        if (low > 0 || !inner) {
          for (int j = threadIdx.x * static_cast<int>(sizeof(T)); j < 32; j += blockDim.x * static_cast<int>(sizeof(T))) {
            const int at = j < 16 ? j : high * 16 + j - 16;
            if ((j < 16 ? low > 0 || high == 0 : !inner && high > 0) && at >= shift && at < shift + bytes)
              *reinterpret_cast<T*>(to + at) = *reinterpret_cast<const T*>(base + at);
          }
        }
        coming[a] += next * B.length;
      }
      rest -= next;
    }
    commit_copies();
    stage ^= 1;
  }
  // The oldest round of rows has come.
  __device__ __forceinline__ void wait() {
    if (MODE == kDirect) return;
    wait_copies<kStages - 1>();
    if (MODE == kChunks) __syncthreads();
  }
  // The thread's numbers of the oldest round; zeros where it has none.
  __device__ __forceinline__ void take(const Params& P, int a, const T* array, int64_t row, A (&to)[K][VEC]) const {
    const bool active = row < P.rows && array;
    const T* from = array + row * P.dim + B.offset + column(0);
    if (MODE == kChunks)
      from = reinterpret_cast<const T*>(chunk(stage * IN + a) + shift_of(array + (row - team) * B.length)) + team * B.length + column(0);
#pragma unroll
    for (int k = 0; k < K; ++k) {
      if (active && in(k)) {
        rows::load<T, VEC>(MODE == kPackets ? reinterpret_cast<const T*>(packet(stage * IN + a, k)) : from + k * kStep, to[k]);
      } else {
#pragma unroll
        for (int c = 0; c < VEC; ++c) to[k][c] = A(0);
      }
    }
  }
  // Writes the thread's numbers of a row of output `a`; a chunk still has to be sent.
  __device__ __forceinline__ void put(const Params& P, int a, T* array, int64_t row, const A (&from)[K][VEC]) const {
    if (!array || row >= P.rows) return;
    T* to = array + row * P.dim + B.offset + column(0);
    if (MODE == kChunks)
      to = reinterpret_cast<T*>(chunk(kStages * IN + a) + shift_of(array + (row - team) * B.length)) + team * B.length + column(0);
#pragma unroll
    for (int k = 0; k < K; ++k)
      if (in(k)) rows::store<T, VEC>(to + k * kStep, from[k]);
  }
  // All threads have put their numbers of a round of rows: writes a chunk of output `a` to memory.
  __device__ __forceinline__ void send(const Params& P, int a, T* array, int64_t row) const {
    const int64_t first = row - team, rows_left = P.rows - first;
    T* to = array + first * B.length;
    const int shift = shift_of(to), end = shift + (rows_left < teams ? static_cast<int>(rows_left) : teams) * B.length * static_cast<int>(sizeof(T));
    unsigned char* base = reinterpret_cast<unsigned char*>(to) - shift;
    const unsigned char* from = chunk(kStages * IN + a);
    const int low = shift == 0 ? 0 : 16, high = end & ~15;  // whole pieces; the others number by number
    for (int i = threadIdx.x * 16; i < high; i += blockDim.x * 16)
      if (i >= low) *reinterpret_cast<uint4*>(base + i) = *reinterpret_cast<const uint4*>(from + i);
    if (low > 0 || high < end)
      for (int j = threadIdx.x * static_cast<int>(sizeof(T)); j < 32; j += blockDim.x * static_cast<int>(sizeof(T))) {
        const int at = j < 16 ? j : high + j - 16;
        if ((j < 16 ? low > 0 || high == 0 : high > 0) && at >= shift && at < end)
          *reinterpret_cast<T*>(base + at) = *reinterpret_cast<const T*>(from + at);
      }
  }

  // Sums over the threads of a row.
  template <int V>
  __device__ __forceinline__ void sum(A (&v)[V]) {
#pragma unroll
    for (int off = LANES >> 1; off; off >>= 1)
#pragma unroll
      for (int i = 0; i < V; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], off);
    if (LANES < 32 || warps == 1) return;
    // Two buffers by turns: who writes the first one again has passed the barrier after which nobody reads it.
    A* at = exchange + turn * (blockDim.x >> 5) * kMaxSums + team * warps * kMaxSums;
    turn ^= 1;
    if (lane == 0)
#pragma unroll
      for (int i = 0; i < V; ++i) at[warp * kMaxSums + i] = v[i];
    asm volatile("bar.sync %0, %1;" ::"r"(team + 1), "r"(B.lanes) : "memory");
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = at[i];
    for (int other = 1; other < warps; ++other)
#pragma unroll
      for (int i = 0; i < V; ++i) v[i] += at[other * kMaxSums + i];
  }

  // The sums of the CTA's rows for one array, a number for each channel, written as one row of partial sums.  All threads have left their rows.
  __device__ __forceinline__ void store_partial(A (&sums)[K][VEC], A* tile, A* __restrict__ to) const {
#pragma unroll
    for (int off = LANES; off < 32; off <<= 1)
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int c = 0; c < VEC; ++c) sums[k][c] += __shfl_xor_sync(0xffffffffu, sums[k][c], off);
    const int groups = LANES < 32 ? blockDim.x >> 5 : teams, group = LANES < 32 ? threadIdx.x >> 5 : team;
    __syncthreads();
    if ((threadIdx.x & 31) < LANES) {
#pragma unroll
      for (int k = 0; k < K; ++k)
        if (in(k))
#pragma unroll
          for (int c = 0; c < VEC; ++c) tile[group * B.length + column(k) + c] = sums[k][c];
    }
    __syncthreads();
    for (int u = threadIdx.x; u < B.channels; u += blockDim.x) {
      A sum = A(0);
      if (B.components == 1) {
#pragma unroll 4
        for (int other = 0; other < groups; ++other) sum += tile[other * B.length + u];
      } else {
        for (int m = 0; m < B.components; ++m)
#pragma unroll 4
          for (int other = 0; other < groups; ++other) sum += tile[other * B.length + u * B.components + m];
      }
      to[u] = sum;
    }
  }
};

// Calls `f` with the number of a warp's threads that share a row of `B`, as a constant.
template <int THREADS, typename F>
__device__ __forceinline__ void with_lanes(const Block& B, F&& f) {
  if constexpr (THREADS > kThreads) {
    f(std::integral_constant<int, 32>());
  } else {
    switch (B.lanes) {
      case 1: f(std::integral_constant<int, 1>()); break;
      case 2: f(std::integral_constant<int, 2>()); break;
      case 4: f(std::integral_constant<int, 4>()); break;
      case 8: f(std::integral_constant<int, 8>()); break;
      case 16: f(std::integral_constant<int, 16>()); break;
      default: f(std::integral_constant<int, 32>()); break;
    }
  }
}

template <typename T>
struct Operands {
  const T *x, *weight, *bias, *g, *rx, *rw, *rb;
  const Moments<Acc<T>>* stats_in;
  T *y, *gx, *hx, *hg;
  Moments<Acc<T>>* stats_out;
  Acc<T>* partial;
};

template <typename T, int VEC, int K, int LANES, int MODE>
__device__ __forceinline__ void forward(const Params& P, const Block& B, int index, const Operands<T>& o, unsigned char* raw, Acc<T>* exchange) {
  using A = Acc<T>;
  const T* const arrays[1] = {o.x};
  Place<T, VEC, K, LANES, MODE, 1, 1> place(P, B, arrays, raw, exchange);
  const int64_t step = static_cast<int64_t>(B.ctas) * place.teams;
  auto request = [&](int64_t row) { place.request(P, arrays, row); };
  int64_t row = static_cast<int64_t>(blockIdx.x - B.first_cta) * place.teams + place.team;
  for (int j = 0; j < kStages; ++j) request(row + j * step);
  A w[K][VEC], b[K][VEC];
  place.parameters(o.weight, B.weight_offset, A(1), w);
  place.parameters(B.scalar ? o.bias : nullptr, B.bias_offset, A(0), b);
  const A share = static_cast<A>(B.share), eps = static_cast<A>(P.eps), per_mean = A(1) / static_cast<A>(B.length);
  for (; row - place.ahead() < P.rows; row += step) {
    A v[K][VEC];
    place.wait();
    place.take(P, 0, o.x, row, v);
    A mean = A(0);
    if (B.scalar) {
      A sums[1] = {A(0)};
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int c = 0; c < VEC; ++c) sums[0] += v[k][c];
      place.sum(sums);
      mean = sums[0] * per_mean;
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int c = 0; c < VEC; ++c) v[k][c] = place.in(k) ? v[k][c] - mean : A(0);
    }
    A sums[1] = {A(0)};
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int c = 0; c < VEC; ++c) sums[0] += v[k][c] * v[k][c];
    place.sum(sums);
    if (MODE == kPackets) request(row + kStages * step);  // the thread's numbers of this row are in registers
    const A scale = rsqrt(sums[0] * share + eps);
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int c = 0; c < VEC; ++c) v[k][c] = v[k][c] * scale * w[k][c] + b[k][c];
    place.put(P, 0, o.y, row, v);
    if (MODE == kChunks) {
      __syncthreads();
      place.send(P, 0, o.y, row);
      request(row + kStages * step);
    }
    if (row < P.rows && o.stats_out && place.lane == 0 && place.warp == 0) o.stats_out[index * P.rows + row] = Moments<A>{mean, scale};
  }
}

template <typename T, int VEC, int K, int LANES, int MODE>
__device__ __forceinline__ void backward(const Params& P, const Block& B, int index, const Operands<T>& o, unsigned char* raw, Acc<T>* exchange) {
  using A = Acc<T>;
  const T* const arrays[2] = {o.x, o.g};
  Place<T, VEC, K, LANES, MODE, 2, 1> place(P, B, arrays, raw, exchange);
  const int64_t step = static_cast<int64_t>(B.ctas) * place.teams;
  auto request = [&](int64_t row) { place.request(P, arrays, row); };
  auto moments = [&](int64_t row) { return row < P.rows ? o.stats_in[index * P.rows + row] : Moments<A>{A(0), A(0)}; };
  int64_t row = static_cast<int64_t>(blockIdx.x - B.first_cta) * place.teams + place.team;
  for (int j = 0; j < kStages; ++j) request(row + j * step);
  Moments<A> next = moments(row);  // a row ahead
  A w[K][VEC], gw[K][VEC], gb[K][VEC];
  place.parameters(o.weight, B.weight_offset, A(1), w);
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int c = 0; c < VEC; ++c) gw[k][c] = gb[k][c] = A(0);
  const A share = static_cast<A>(B.share), per_mean = B.scalar ? A(1) / static_cast<A>(B.length) : A(0);
  for (; row - place.ahead() < P.rows; row += step) {
    A h[K][VEC], e[K][VEC];
    const Moments<A> m = next;
    next = moments(row + step);
    place.wait();
    place.take(P, 0, o.x, row, h);
    place.take(P, 1, o.g, row, e);
    A sums[2] = {A(0), A(0)};
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int c = 0; c < VEC; ++c) {
        // columns that are not there have e = 0: whatever h is, they add nothing, unless the mean is no number
        h[k][c] = place.in(k) ? (h[k][c] - m.mean) * m.scale : A(0);
        gw[k][c] += e[k][c] * h[k][c];
        gb[k][c] += e[k][c];
        e[k][c] *= w[k][c];
        sums[0] += e[k][c] * h[k][c];
        sums[1] += e[k][c];
      }
    if (o.gx) place.sum(sums);
    if (MODE == kPackets) request(row + kStages * step);
    if (o.gx) {
      const A along = sums[0] * share, mean = sums[1] * per_mean;
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int c = 0; c < VEC; ++c) e[k][c] = m.scale * (e[k][c] - mean - h[k][c] * along);
      place.put(P, 0, o.gx, row, e);
    }
    if (MODE == kChunks) {
      __syncthreads();
      if (o.gx) place.send(P, 0, o.gx, row);
      request(row + kStages * step);
    }
  }
  if (!o.partial) return;
  A* to = o.partial + B.partial + static_cast<int64_t>(blockIdx.x - B.first_cta) * 2 * B.channels;
  A* tile = reinterpret_cast<A*>(raw);
  wait_copies<0>();
  place.store_partial(gw, tile, to);
  if (B.scalar) place.store_partial(gb, tile, to + B.channels);
}

template <typename T, int VEC, int K, int LANES, int MODE>
__device__ __forceinline__ void second(const Params& P, const Block& B, int index, const Operands<T>& o, unsigned char* raw, Acc<T>* exchange) {
  using A = Acc<T>;
  const T* const arrays[3] = {o.x, o.g, o.rx};
  Place<T, VEC, K, LANES, MODE, 3, 2> place(P, B, arrays, raw, exchange);
  const int64_t step = static_cast<int64_t>(B.ctas) * place.teams;
  auto request = [&](int64_t row) { place.request(P, arrays, row); };
  auto moments = [&](int64_t row) { return row < P.rows ? o.stats_in[index * P.rows + row] : Moments<A>{A(0), A(0)}; };
  int64_t row = static_cast<int64_t>(blockIdx.x - B.first_cta) * place.teams + place.team;
  for (int j = 0; j < kStages; ++j) request(row + j * step);
  Moments<A> next = moments(row);
  A w[K][VEC], hw[K][VEC];
  place.parameters(o.weight, B.weight_offset, A(1), w);
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int c = 0; c < VEC; ++c) hw[k][c] = A(0);
  // rw and rb are as short as a row and the same for all of them: read again from cache instead of kept
  auto other = [&](const T* __restrict__ p, int offset, int k, int c) {
    return p && place.in(k) ? rows::widen(p[offset + place.channel(place.column(k) + c)]) : A(0);
  };
  const A share = static_cast<A>(B.share), per_mean = B.scalar ? A(1) / static_cast<A>(B.length) : A(0);
  for (; row - place.ahead() < P.rows; row += step) {
    A h[K][VEC], e[K][VEC], r[K][VEC];
    const Moments<A> m = next;
    next = moments(row + step);
    place.wait();
    place.take(P, 0, o.x, row, h);
    place.take(P, 1, o.g, row, e);
    place.take(P, 2, o.rx, row, r);
    // Scalars: the means come first.  Of r and c far from zero, dot is what is left of n mean(r) mean(c), so it is made of distances
    // (64 scalars, r and c with a spread of one about 1000, FP32: hx was off by half of its largest).  One more sum over the row, us
    // without and with it: 1.0 M rows of 64, FP64, 458 and 461; 40,000 of 1024, FP32 142 and 154, BF16 180 and 208.  Distances from
    // the row's first numbers need no such sum, but registers: BF16 209, three blocks of 128 270 in place of 257.
    A mean_r = A(0), mean_c = A(0);
    if (B.scalar) {
      A means[2] = {A(0), A(0)};
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int c = 0; c < VEC; ++c) {
          means[0] += r[k][c];
          means[1] += e[k][c] * w[k][c];
        }
      place.sum(means);
      mean_r = means[0] * per_mean;
      mean_c = means[1] * per_mean;
    }
    A sums[3] = {A(0), A(0), A(0)}, more[2] = {A(0), A(0)};  // rh, ch, rc; q, qh
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int c = 0; c < VEC; ++c) {
        h[k][c] = place.in(k) ? (h[k][c] - m.mean) * m.scale : A(0);
        r[k][c] -= mean_r;
        const A scaled = place.in(k) ? e[k][c] * w[k][c] - mean_c : A(0);  // with h zero, too, no column that is not there adds to a sum
        sums[0] += r[k][c] * h[k][c];
        sums[1] += scaled * h[k][c];
        sums[2] += r[k][c] * scaled;
        if (o.rw) {
          const A q = other(o.rw, B.weight_offset, k, c) * e[k][c];
          more[0] += q;
          more[1] += q * h[k][c];
        }
      }
    place.sum(sums);
    if (o.rw) place.sum(more);
    if (MODE == kPackets) request(row + kStages * step);
    const A mean_q = more[0] * per_mean, dot = sums[2];
    const A along_r = share * sums[0], along_c = share * sums[1], along_q = share * more[1];
    const A outer = m.scale * m.scale * share, on_h = dot - share * sums[0] * sums[1];
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int c = 0; c < VEC; ++c) {
        const A p = r[k][c] - h[k][c] * along_r;
        const A scaled = e[k][c] * w[k][c] - mean_c - h[k][c] * along_c;
        const A from_q = on_h * h[k][c] + sums[1] * p + sums[0] * scaled;
        hw[k][c] += m.scale * p * e[k][c];  // nothing where there is no column: e is zero
        A hx = -outer * from_q, hg = w[k][c] * m.scale * p;
        if (o.rw) {
          const A tangent = other(o.rw, B.weight_offset, k, c);
          hx += m.scale * (tangent * e[k][c] - mean_q - h[k][c] * along_q);
          hg += tangent * h[k][c];
        }
        if (o.rb && B.scalar) hg += other(o.rb, B.bias_offset, k, c);
        r[k][c] = hx;
        e[k][c] = hg;
      }
    place.put(P, 0, o.hx, row, r);
    place.put(P, 1, o.hg, row, e);
    if (MODE == kChunks) {
      __syncthreads();
      if (o.hx) place.send(P, 0, o.hx, row);
      if (o.hg) place.send(P, 1, o.hg, row);
      request(row + kStages * step);
    }
  }
  if (!o.partial) return;
  wait_copies<0>();
  place.store_partial(hw, reinterpret_cast<A*>(raw), o.partial + B.partial + static_cast<int64_t>(blockIdx.x - B.first_cta) * 2 * B.channels);
}

enum Order { kForward, kBackward, kSecond };

template <typename T, int VEC, int K, int THREADS, int MODE, int ORDER>
__global__ void __launch_bounds__(THREADS)
norm_kernel(const __grid_constant__ Params P, const __grid_constant__ Operands<T> o) {
  extern __shared__ __align__(16) unsigned char raw[];
  __shared__ Acc<T> exchange[2 * (THREADS / 32) * kMaxSums];
  const int index = block_index_of(P);
  const Block& B = P.block[index];
  with_lanes<THREADS>(B, [&](auto lanes) {
    constexpr int LANES = decltype(lanes)::value;
    if constexpr (ORDER == kForward) forward<T, VEC, K, LANES, MODE>(P, B, index, o, raw, exchange);
    if constexpr (ORDER == kBackward) backward<T, VEC, K, LANES, MODE>(P, B, index, o, raw, exchange);
    if constexpr (ORDER == kSecond) second<T, VEC, K, LANES, MODE>(P, B, index, o, raw, exchange);
  });
}

// The sums of all CTAs: 32 channels of a block, for the weights or for the biases, by one CTA, 32 threads for each channel.
constexpr int kFinalSlices = 32;
template <typename T>
__global__ void __launch_bounds__(32 * kFinalSlices)
final_kernel(const __grid_constant__ Params P, const Acc<T>* __restrict__ partial, T* __restrict__ gw, T* __restrict__ gb) {
  using A = Acc<T>;
  __shared__ A tile[kFinalSlices][33];
  wait_for_previous();
  int i = 0, task = blockIdx.x;  // which block, and which 32 of its channels
  while (task >= (P.block[i].channels + 31) / 32) task -= (P.block[i++].channels + 31) / 32;
  const Block& B = P.block[i];
  const bool biases = blockIdx.y;
  T* to = biases ? gb : gw;
  if (!to || (biases && !B.scalar)) return;
  const int lane = threadIdx.x & 31, slice = threadIdx.x >> 5, first = task * 32;
  A sum = A(0);
  if (first + lane < B.channels) {
    const A* column = partial + B.partial + (biases ? B.channels : 0) + first + lane;
    const int64_t stride = 2 * static_cast<int64_t>(B.channels);
#pragma unroll 8
    for (int j = slice; j < B.ctas; j += kFinalSlices) sum += column[j * stride];
  }
  tile[slice][lane] = sum;
  __syncthreads();
  A total = tile[lane][slice];  // a warp's threads have the slices of one channel
  for (int off = 16; off; off >>= 1) total += __shfl_xor_sync(0xffffffffu, total, off);
  if (lane == 0 && first + slice < B.channels) rows::narrow(total, to[(biases ? B.bias_offset : B.weight_offset) + first + slice]);
}

// ---- launches --------------------------------------------------------------------------------------------------------------

struct Call {
  const void *x, *weight, *bias, *stats_in, *g, *rx, *rw, *rb;
  void *y, *stats_out, *gx, *gw, *gb, *hx, *hg;
  void* scratch;
  int64_t scratch_bytes;
};

// Gives every block its threads per row; returns the largest chunk.
template <typename T>
int lay_out(Params& P, int vec, int packets, int threads) {
  int most = 0;
  for (int i = 0; i < P.blocks; ++i) {
    Block& B = P.block[i];
    B.lanes = rows::next_power_of_two(ceil_div(ceil_div(B.length, vec), packets));
    if (threads > kThreads && B.lanes < 128) B.lanes = 128;  // a CTA has fifteen barriers beside its own
    B.chunk = (threads / B.lanes * B.length * static_cast<int>(sizeof(T)) + 15) / 16 * 16 + 16;  // beginning anywhere in a piece
    most = most < B.chunk ? B.chunk : most;
  }
  return most;
}

// Gives every block its CTAs: as many as its rows want, or its share of the resident ones.
inline int assign(Params& P, int threads, int resident) {
  int64_t wanted = 0;
  for (int i = 0; i < P.blocks; ++i) wanted += ceil_div(P.rows, threads / P.block[i].lanes);
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
    partial += count * 2 * B.channels;
  }
  return ctas;
}
// At most this many CTAs of kThreads are resident on a multiprocessor, whatever a kernel needs.
constexpr int kMostResident = 2048 / kThreads;
inline int64_t scratch_elements(const Params& P) {
  const int64_t resident = static_cast<int64_t>(kMostResident) * rows::processors();
  return (P.rows < resident ? P.rows : resident) * 2 * P.dim + 2;  // never zero: a buffer of no bytes has no address
}

template <typename T, int VEC, int K, int THREADS, int MODE, int ORDER>
int launch(Params P, const Call& c, cudaStream_t stream) {
  using A = Acc<T>;
  auto in = [](const void* p) { return static_cast<const T*>(p); };
  auto out = [](void* p) { return static_cast<T*>(p); };
  const bool sums = ORDER != kForward && (c.gw || c.gb);
  // Room for the rows on their way and on their way out, and later for the sums of the CTA's threads
  constexpr int in_arrays = ORDER == kForward ? 1 : ORDER == kBackward ? 2 : 3, out_arrays = ORDER == kSecond ? 2 : 1;
  const size_t chunk = lay_out<T>(P, VEC, K, THREADS);
  const size_t rows_bytes = MODE == kDirect ? 0 : MODE == kPackets ? kStages * in_arrays * K * VEC * sizeof(T) * THREADS : (kStages * in_arrays + out_arrays) * chunk;
  const size_t sums_bytes = sums ? static_cast<size_t>(THREADS) * K * VEC * sizeof(A) : 0;
  const size_t shared = std::max(rows_bytes, sums_bytes);
  const auto kernel = norm_kernel<T, VEC, K, THREADS, MODE, ORDER>;
  static rows::Kernel known;
  const int resident = known.resident(kernel, THREADS, shared);
  if (resident < 1) return resident;
  const int ctas = assign(P, THREADS, resident);
  const Operands<T> o{in(c.x), in(c.weight), in(c.bias), in(c.g), in(c.rx), in(c.rw), in(c.rb), static_cast<const Moments<A>*>(c.stats_in),
                      out(c.y), out(c.gx), out(c.hx), out(c.hg), static_cast<Moments<A>*>(c.stats_out),
                      sums ? static_cast<A*>(c.scratch) : nullptr};
  if (ctas > 0) {
    kernel<<<ctas, THREADS, shared, stream>>>(P, o);
    LUNA_LAUNCH_CHECK("layer norm");
  }
  if (sums) {
    int tasks = 0;
    for (int i = 0; i < P.blocks; ++i) tasks += (P.block[i].channels + 31) / 32;
    launch_early(final_kernel<T>, dim3(tasks, c.gb ? 2 : 1), 32 * kFinalSlices, 0, stream, P, static_cast<const A*>(o.partial), out(c.gw), out(c.gb));
    LUNA_LAUNCH_CHECK("sums of the layer norm");
  }
  return LUNA_OK;
}

// Packets narrower than sixteen bytes.  Numbers of a thread, measured, forward / backward in us for four, eight or sixteen: 600,000 rows
// of 50x0e, FP32 (packets of two) 55 / 78, 43 / 72, 46 / 76, BF16 56 / 80, 41 / 67, 37 / 59; 20,000 of 1001x0e, FP32 (single numbers)
// 55 / 64, 39 / 67, 44 / 72; 300,000 of 51x0e, FP64, four or eight 44 / 69 / 112 (second order) and 48 / 75 / 180.
template <typename T, int VEC, int ORDER>
int with_packets(const Params& P, int64_t longest, bool few, const Call& c, cudaStream_t stream) {
  constexpr int kFew = VEC < 4 ? 4 / VEC : 1, kMany = (sizeof(T) == 2 && ORDER != kSecond ? 16 : 8) / VEC;
  const int64_t n = longest / VEC;
  if ((few || sizeof(T) > 4 || longest <= 16) && n <= kThreads * kFew) return launch<T, VEC, kFew, kThreads, kPackets, ORDER>(P, c, stream);
  if (n <= kThreads * kMany) return launch<T, VEC, kMany, kThreads, kPackets, ORDER>(P, c, stream);
  return launch<T, VEC, 16 / VEC, kWideThreads, kDirect, ORDER>(P, c, stream);
}

template <typename T, int ORDER>
int choose(const Params& P, const Call& c, cudaStream_t stream) {
  constexpr int kWidest = 16 / static_cast<int>(sizeof(T));
  int64_t longest = 0;
  int vec = kWidest;  // numbers of a packet: at most 16 bytes, at least the four of an asynchronous copy
  for (int i = 0; i < P.blocks; ++i) {
    while (vec > 1 && (P.dim % vec || P.block[i].offset % vec || P.block[i].length % vec)) vec >>= 1;
    longest = P.block[i].length > longest ? P.block[i].length : longest;
  }
  for (const void* p : {c.x, c.g, c.rx, static_cast<const void*>(c.y), static_cast<const void*>(c.gx), static_cast<const void*>(c.hx),
                        static_cast<const void*>(c.hg)})
    while (vec > 1 && !aligned_to(p, vec * sizeof(T))) vec >>= 1;
  // Packets of a thread.  More of them mean fewer threads per row, so fewer steps for its sums and no barrier, as long as the
  // registers allow it.  Measured, forward / backward / second order in us: 50,000 rows of 128x0e+128x1o+128x2e, FP32, one, two
  // or four packets 139 / 199, 87 / 168, 84 / 123; 100,000 of 64x0e+64x1o+64x2e 139 / 180 / 316, 86 / 163 / 244, 82 / 123 / 308;
  // 86,000 of 64x0e 10.9 / 13.0, 8.9 / 14.9, 9.7 / 15.4; 40,000 of 1024x0e, BF16, 58 / 76, 55 / 63, 54 / 79.  Where there are not
  // enough rows to fill the GPU, the threads are: 24 rows 2.6, 2.8 and 3.6 us, 500 rows of 64x0e 2.6 / 3.1, 3.1 / 4.2, 4.0 / 5.7.
  const bool few = P.rows * P.dim <= static_cast<int64_t>(rows::processors()) * 1024 * (vec == kWidest ? kWidest : 1);
  if (vec == kWidest) {
    const int64_t n = longest / kWidest;
    const int64_t most_of_two = ORDER == kSecond || sizeof(T) == 2 ? kThreads * 2 : 64;
    if (few && n <= kThreads) return launch<T, kWidest, 1, kThreads, kPackets, ORDER>(P, c, stream);
    if (n <= most_of_two) return launch<T, kWidest, 2, kThreads, kPackets, ORDER>(P, c, stream);
    if (n <= kThreads * 4) return launch<T, kWidest, 4, kThreads, kPackets, ORDER>(P, c, stream);
    if (n <= kWideThreads * 4) return launch<T, kWidest, 4, kWideThreads, kDirect, ORDER>(P, c, stream);
    return launch<T, 1, 16, kWideThreads, kDirect, ORDER>(P, c, stream);
  }
  if constexpr (sizeof(T) == 2) {
    if (vec == 4) return with_packets<T, 4, ORDER>(P, longest, few, c, stream);
    if (vec == 2) return with_packets<T, 2, ORDER>(P, longest, few, c, stream);
    if (longest <= kThreads * 16) {
      if (P.blocks > 1) return launch<T, 1, 16, kThreads, kDirect, ORDER>(P, c, stream);
      if (few && longest <= kThreads * 4) return launch<T, 1, 4, kThreads, kChunks, ORDER>(P, c, stream);
      return launch<T, 1, 16, kThreads, kChunks, ORDER>(P, c, stream);
    }
    return launch<T, 1, 16, kWideThreads, kDirect, ORDER>(P, c, stream);
  } else {
    if constexpr (sizeof(T) == 4) {
      if (vec == 2) return with_packets<T, 2, ORDER>(P, longest, few, c, stream);
    }
    return with_packets<T, 1, ORDER>(P, longest, few, c, stream);
  }
}

template <typename T>
int run(Order order, const Params& P, const Call& c, cudaStream_t stream) {
  return order == kForward ? choose<T, kForward>(P, c, stream) : order == kBackward ? choose<T, kBackward>(P, c, stream) : choose<T, kSecond>(P, c, stream);
}

extern template int run<float>(Order, const Params&, const Call&, cudaStream_t);
extern template int run<double>(Order, const Params&, const Call&, cudaStream_t);
extern template int run<rows::bf16>(Order, const Params&, const Call&, cudaStream_t);
extern template int run<rows::f16>(Order, const Params&, const Call&, cudaStream_t);

}  // namespace norm
}  // namespace luna
