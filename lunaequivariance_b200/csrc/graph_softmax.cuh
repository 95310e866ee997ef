// Softmax over the in-edges of every node, head by head, with a learned bias by buckets added to the logits.
//
// Edges are sorted by destination, so a row is a contiguous piece of the [edges, heads] arrays.  With z = logit + table[bucket]
// (masked edges: -inf), m = max z and l = sum exp(z - m) over the row: alpha = exp(z - m) / l, zeros where nothing is left.
//   backward   with D = sum alpha g:   dz = alpha (g - D)
//   second     the cotangent r of dz, R = sum alpha r:   d/dg = alpha (r - R),   d/dalpha = (g - D) (r - R)
// Where alpha is zero nothing flows, whatever stands in g or r there.  d/dalpha is meant for an alpha whose rows sum to one: it is
// r (g - D) - g R and the row's constant D R, which the backward takes out with D.  Made of the distances from the means: the
// products of g and r themselves are as large as their squares, and what is left of them behind the constant may be nothing but
// rounding: of g and r with a spread of one about 1000, FP32, dz was off by 17 % of its largest (0.01 % like this).
//
// Bound by HBM: a row's values are read once and held in registers between its sums and its outputs, as far as they fit (K packets
// of a thread); the rest of a longer row passes twice, the second time from cache.  All loads of a batch are under way before
// the first is waited for: with the mask and the table looked up edge by edge, 2.6 M edges with 8 heads took 94 us forward.
// `lanes` threads of a warp share a row, or a whole CTA where rows are long; of them `across` (a power of two) lie side by side
// over an edge's heads.  Very long rows come cut into pieces: the first launch makes the outputs of whole rows and the sums of
// pieces, one joins those of each cut node, and one makes the pieces' outputs.
#pragma once

#include <type_traits>

#include "rows.cuh"

namespace luna {
namespace softmax {

using rows::Acc;

constexpr int kThreads = 256;

struct Rows {  // as luna_row_table
  const int32_t* rowptr;
  int64_t count, pieces, cut;
  const int32_t *piece_of_row, *row_of_piece, *cut_of_piece, *cut_first;
};

struct Shape {
  int heads, across, lanes;  // lanes: threads per row; more than 32 means the whole CTA
  int num_buckets;
};

enum Order { kForward, kBackward, kSecond, kBackwardWide };  // the last: kBackward with `gwide` in place of `g`, for the 16-bit types
constexpr bool is_backward(int order) { return order == kBackward || order == kBackwardWide; }
enum Phase { kWhole, kMixed, kApply };  // no pieces; whole rows and the pieces' sums; the pieces' outputs

template <typename T>
struct Operands {
  const T *logits, *table;
  const Acc<T>* alpha;  // as the sums are held: rounded to 16 bits, the sums by bucket of alpha (g - D) are off by more than their own rounding
  const T *g, *r, *rtable;
  const Acc<T>* gwide;
  const int32_t* buckets;
  const uint8_t* mask;
  T *out, *out2;
  Acc<T>* wide;  // 16-bit types: the output (of the second order, d/dalpha) as it was before it was rounded
};

template <typename A>
struct Pair {
  A a, b;
};

// Sums or maxima over the threads that hold the same heads of one row.
template <typename A, int VEC, int LANES>
struct Together {
  const Shape& S;
  A* exchange;  // [2][warps][32][VEC]
  int turn = 0;
  __device__ Together(const Shape& S_, A* exchange_) : S(S_), exchange(exchange_) {}

  template <typename F>
  __device__ __forceinline__ void all(A (&v)[VEC], F&& join) {
    if constexpr (LANES) {
#pragma unroll
      for (int off = LANES >> 1; off; off >>= 1)
        if (off >= S.across)
#pragma unroll
          for (int c = 0; c < VEC; ++c) v[c] = join(v[c], __shfl_xor_sync(0xffffffffu, v[c], off));
      return;
    }
    const int within = S.lanes < 32 ? S.lanes : 32;
    for (int off = within >> 1; off >= S.across; off >>= 1)
#pragma unroll
      for (int c = 0; c < VEC; ++c) v[c] = join(v[c], __shfl_xor_sync(0xffffffffu, v[c], off));
    if (S.lanes <= 32) return;
    // two buffers by turns, so that one barrier is enough
    constexpr int kWarps = kThreads / 32;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    A* at = exchange + turn * kWarps * 32 * VEC;
    turn ^= 1;
    if (lane < S.across)
#pragma unroll
      for (int c = 0; c < VEC; ++c) at[(warp * 32 + lane) * VEC + c] = v[c];
    __syncthreads();
    const int mine = lane & (S.across - 1);
#pragma unroll
    for (int c = 0; c < VEC; ++c) v[c] = at[mine * VEC + c];
    for (int other = 1; other < kWarps; ++other)
#pragma unroll
      for (int c = 0; c < VEC; ++c) v[c] = join(v[c], at[(other * 32 + mine) * VEC + c]);
  }
  __device__ __forceinline__ void sum(A (&v)[VEC]) {
    all(v, [](A p, A q) { return p + q; });
  }
  __device__ __forceinline__ void max(A (&v)[VEC]) {
    all(v, [](A p, A q) { return fmax(p, q); });
  }
};

// exp(z - m), in single precision as 2^((z - m) log2 e): a product, rounded once, and an instruction that is off by two units in
// the last place.  So the result is off by |z - m| roundings of 2^-24 and a few (a millionth at 20 below the largest), and below 1.2e-38
// it is zero.  The difference is made first: z and m may be the lowest numbers of their type.
__device__ __forceinline__ float exponential(float z, float m) {
  float v;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(v) : "f"((z - m) * 1.4426950408889634f));
  return v;
}
__device__ __forceinline__ double exponential(double z, double m) { return exp(z - m); }
// Of a sum of exponentials: at least one (the largest logit's), or zero, or no number.
__device__ __forceinline__ float reciprocal(float v) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return v == 0.0f ? 0.0f : r;
}
__device__ __forceinline__ double reciprocal(double v) { return v == 0.0 ? 0.0 : 1.0 / v; }

template <typename A>
__device__ __forceinline__ A lowest() {
  return -static_cast<A>(INFINITY);
}
// What is taken out of the logits: the largest one, or nothing where there is none (nothing left, or nothing but NaN).
template <typename A>
__device__ __forceinline__ A taken(A largest) {
  return largest == lowest<A>() ? A(0) : largest;
}

// LANES: as S.lanes, where an edge's heads fill their `across` packets, so that a row is one stretch of packets; 0: neither is known.
template <typename T, int VEC, int K, int ORDER, int PHASE, int LANES>
__global__ void __launch_bounds__(kThreads, is_backward(ORDER) ? 4 : ORDER == kForward && sizeof(T) <= 4 ? 3 : 2)
rows_kernel(const Rows R, const Shape S, const Operands<T> o, Pair<Acc<T>>* __restrict__ stats) {
  using A = Acc<T>;
  using In = rows::Pack<T, VEC>;
  __shared__ A exchange[2 * kThreads * VEC];
  Together<A, VEC, LANES> together(S, exchange);
  const int lanes = LANES ? LANES : S.lanes;
  const int lane = threadIdx.x & (lanes - 1);
  const int slot = lane / S.across, slots = lanes / S.across;
  const int head = (blockIdx.y * S.across + (lane & (S.across - 1))) * VEC;
  const bool here = LANES || head < S.heads;
  const int teams = kThreads / lanes, team = threadIdx.x / lanes;
  const int ahead = lanes < 32 ? team % (32 / lanes) : 0;  // teams of this warp before this one: they leave together
  const int stride = LANES ? LANES * VEC : slots * S.heads;  // from one of a thread's edges to the next

  // K edges of a thread: z (forward), or alpha and g and the cotangent r
  A u[K][VEC], g[K][VEC], r[K][VEC];
  const T* const table = ORDER == kForward ? o.table : ORDER == kSecond ? o.rtable : nullptr;
  // `first`: the thread's first edge of the batch; `left`: edges of the row from there on
  auto fetch = [&](int first, int left) {
    const int64_t at = static_cast<int64_t>(first) * S.heads + head;
    auto there = [&](int k) { return k * slots < left; };
    auto bring = [&](const auto* __restrict__ array, A (&to)[K][VEC], A otherwise) {
      const auto* from = array + at;
#pragma unroll
      for (int k = 0; k < K; ++k) {
        if (there(k)) {
          rows::load<std::remove_const_t<std::remove_pointer_t<decltype(from)>>, VEC>(from + k * stride, to[k]);
        } else {
#pragma unroll
          for (int c = 0; c < VEC; ++c) to[k][c] = otherwise;
        }
      }
    };
    int bucket[K];
    bool keep[K];
    if (table) {
      const int32_t* from = o.buckets + first;
#pragma unroll
      for (int k = 0; k < K; ++k) bucket[k] = there(k) ? from[k * slots] : -1;
    }
    if constexpr (ORDER == kForward) {
      if (o.mask) {
        const uint8_t* from = o.mask + first;
#pragma unroll
        for (int k = 0; k < K; ++k) keep[k] = there(k) && from[k * slots];
      }
      bring(o.logits, u, lowest<A>());
    } else {
      bring(o.alpha, u, A(0));
      if constexpr (ORDER == kBackwardWide)
        bring(o.gwide, g, A(0));
      else
        bring(o.g, g, A(0));
      if constexpr (ORDER == kSecond) {
        if (o.r) {
          bring(o.r, r, A(0));
        } else {
#pragma unroll
          for (int k = 0; k < K; ++k)
#pragma unroll
            for (int c = 0; c < VEC; ++c) r[k][c] = A(0);
        }
      }
    }
    if (table) {
      const T* const from = table + head;
      In t[K];
#pragma unroll
      for (int k = 0; k < K; ++k) {
        t[k] = In{};
        if (static_cast<unsigned>(bucket[k]) < static_cast<unsigned>(S.num_buckets))
          t[k] = *reinterpret_cast<const In*>(from + static_cast<int64_t>(bucket[k]) * S.heads);
      }
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int c = 0; c < VEC; ++c) (ORDER == kForward ? u : r)[k][c] += rows::widen(t[k].a[c]);
    }
    if constexpr (ORDER == kForward) {
      if (o.mask) {
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
          for (int c = 0; c < VEC; ++c) u[k][c] = keep[k] ? u[k][c] : lowest<A>();
      }
    }
  };
  // The outputs of a batch, from alpha times `factor` (forward), or from alpha, D and R
  auto put = [&](int first, int left, const A (&a)[VEC], const A (&b)[VEC]) {
    const int64_t at = static_cast<int64_t>(first) * S.heads + head;
    T *const out = o.out + at, *const out2 = o.out2 + at;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      if (k * slots >= left) continue;
      A v[VEC], w[VEC];
#pragma unroll
      for (int c = 0; c < VEC; ++c) {
        const A alpha = u[k][c];
        if constexpr (ORDER == kForward) {
          v[c] = alpha * b[c];
        } else if constexpr (is_backward(ORDER)) {
          v[c] = alpha != A(0) ? alpha * (g[k][c] - a[c]) : A(0);
        } else {
          v[c] = alpha != A(0) ? alpha * (r[k][c] - b[c]) : A(0);
          w[c] = alpha != A(0) ? (g[k][c] - a[c]) * (r[k][c] - b[c]) : A(0);
        }
      }
      if (ORDER != kSecond || o.out) rows::store<T, VEC>(out + k * stride, v);
      if constexpr (sizeof(T) == 2 && ORDER != kSecond)
        if (o.wide) rows::store<A, VEC>(o.wide + at + k * stride, v);
      if constexpr (ORDER == kSecond) {
        if (o.out2) rows::store<T, VEC>(out2 + k * stride, w);
        if constexpr (sizeof(T) == 2)
          if (o.wide) rows::store<A, VEC>(o.wide + at + k * stride, w);
      }
    }
    if constexpr (ORDER == kForward) {
      // Zero times a sum that is no number is none either: what is masked beside one is put right, a walk that no other row takes.
      // (A bit for each masked number in a register instead: 2.6 M edges with one head, mask and table 33 us, 27 like this.)
      bool lost = false;
#pragma unroll
      for (int c = 0; c < VEC; ++c) lost |= b[c] != b[c];
      if (lost && o.mask) {
        const A zeros[VEC] = {};
#pragma unroll 1
        for (int k = 0; k < K; ++k) {
          if (k * slots >= left || o.mask[first + k * slots]) continue;
          rows::store<T, VEC>(out + k * stride, zeros);
          if constexpr (sizeof(T) == 2)
            if (o.wide) rows::store<A, VEC>(o.wide + at + k * stride, zeros);
        }
      }
    }
  };
  auto exponentials = [&](const A (&m)[VEC]) {
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int c = 0; c < VEC; ++c) u[k][c] = exponential(u[k][c], m[c]);
  };
  auto largest = [&](A (&a)[VEC]) {
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int c = 0; c < VEC; ++c) a[c] = fmax(a[c], u[k][c]);
  };
  auto add_up = [&](A (&b)[VEC]) {
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int c = 0; c < VEC; ++c) b[c] += u[k][c];
  };

  const int batch = K * slots;
  const int64_t step = static_cast<int64_t>(gridDim.x) * teams;
  const int64_t count = PHASE == kApply ? R.pieces : R.count;
  // Where a row is, one row ahead of its use: of three trips to memory that follow one another the first
  int next_first = 0, next_length = 0, next_piece = -1;
  auto find = [&](int64_t number) {
    next_first = next_length = 0;
    next_piece = -1;
    if (number < count && here) {
      const int64_t row = PHASE == kApply ? R.row_of_piece[number] : number;
      if constexpr (PHASE == kMixed) next_piece = R.piece_of_row[row];
      next_first = R.rowptr[row];
      next_length = R.rowptr[row + 1];
    }
  };
  int64_t number = static_cast<int64_t>(blockIdx.x) * teams + team;
  find(number);
  for (; number - ahead < count; number += step) {
    int first = next_first;
    const int length = next_length - next_first, piece = next_piece;
    find(number + step);
    first += slot;
    const int left = length - slot;
    const int behind = length > 0 ? (length - 1) / batch * batch : 0;  // where the last batch begins
    A a[VEC], b[VEC];  // forward: the largest logit and the sum; else D and R
#pragma unroll
    for (int c = 0; c < VEC; ++c) {
      a[c] = ORDER == kForward ? lowest<A>() : A(0);
      b[c] = A(0);
    }
    if constexpr (PHASE != kApply) {
      if constexpr (ORDER == kForward) {
        // Batches behind the first one: each thread has a largest logit and a sum of its own, which grow together.
        for (int at = behind; at > 0; at -= batch) {
          fetch(first + at, left - at);
          A before[VEC], m[VEC];
#pragma unroll
          for (int c = 0; c < VEC; ++c) before[c] = a[c];
          largest(a);
#pragma unroll
          for (int c = 0; c < VEC; ++c) {
            m[c] = taken(a[c]);
            if (b[c] != A(0)) b[c] *= before[c] == lowest<A>() ? A(1) : exponential(before[c], m[c]);
          }
          exponentials(m);
          add_up(b);
        }
        A own[VEC], m[VEC];
#pragma unroll
        for (int c = 0; c < VEC; ++c) own[c] = a[c];
        fetch(first, left);
        largest(a);
        together.max(a);
#pragma unroll
        for (int c = 0; c < VEC; ++c) {
          m[c] = taken(a[c]);
          if (b[c] != A(0)) b[c] *= own[c] == lowest<A>() ? A(1) : exponential(own[c], m[c]);
        }
        exponentials(m);
        add_up(b);
        together.sum(b);
      } else {
        // From the last batch to the first, which stays in registers
        for (int at = behind; at >= 0; at -= batch) {
          fetch(first + at, left - at);
#pragma unroll
          for (int k = 0; k < K; ++k)
#pragma unroll
            for (int c = 0; c < VEC; ++c) {
              a[c] += u[k][c] != A(0) ? u[k][c] * g[k][c] : A(0);
              if constexpr (ORDER == kSecond) b[c] += u[k][c] != A(0) ? u[k][c] * r[k][c] : A(0);
            }
        }
        together.sum(a);
        if constexpr (ORDER == kSecond) together.sum(b);
      }
    }
    if (PHASE == kMixed && piece >= 0) {
      if (slot == 0)
#pragma unroll
        for (int c = 0; c < VEC; ++c) stats[static_cast<int64_t>(piece) * S.heads + head + c] = Pair<A>{a[c], b[c]};
      continue;
    }
    if constexpr (PHASE == kApply) {
      if (number < count && here) {
        const int64_t at = static_cast<int64_t>(R.cut_first[R.cut_of_piece[number]]) * S.heads + head;
#pragma unroll
        for (int c = 0; c < VEC; ++c) {
          const Pair<A> known = stats[at + c];
          a[c] = known.a;
          b[c] = known.b;
        }
      }
    }
    if constexpr (ORDER == kForward) {
#pragma unroll
      for (int c = 0; c < VEC; ++c) {
        a[c] = taken(a[c]);
        b[c] = reciprocal(b[c]);
      }
    }
    if constexpr (PHASE != kApply) put(first, left, a, b);
    for (int at = PHASE != kApply ? batch : 0; at <= behind; at += batch) {
      fetch(first + at, left - at);
      if constexpr (ORDER == kForward) exponentials(a);
      put(first + at, left - at, a, b);
    }
  }
}

// Joins the sums of the pieces of every cut node, in its first piece's place: a CTA per node, `across` of its threads (a power
// of two, at most a warp) side by side over the heads.
template <typename A, bool FORWARD>
__global__ void __launch_bounds__(kThreads)
join_kernel(const Rows R, int heads, int across, Pair<A>* __restrict__ stats) {
  __shared__ Pair<A> tile[kThreads];
  const int64_t first = R.cut_first[blockIdx.x], pieces = R.cut_first[blockIdx.x + 1] - first;
  // one pair after the other; a pair without a largest logit has nothing (a sum of zero), or nothing but NaN, in its sum too
  auto join = [](Pair<A> p, Pair<A> q) {
    if (!FORWARD) return Pair<A>{p.a + q.a, p.b + q.b};
    const A top = fmax(p.a, q.a), m = taken(top);
    return Pair<A>{top, (p.a == lowest<A>() ? p.b : p.b * exponential(p.a, m)) + (q.a == lowest<A>() ? q.b : q.b * exponential(q.a, m))};
  };
  for (int base = 0; base < heads; base += across) {
    const int h = base + (threadIdx.x & (across - 1));
    Pair<A> sum{FORWARD ? lowest<A>() : A(0), A(0)};
    if (h < heads) {
#pragma unroll 4
      for (int64_t p = threadIdx.x / across; p < pieces; p += kThreads / across) sum = join(sum, stats[(first + p) * heads + h]);
    }
    __syncthreads();
    tile[threadIdx.x] = sum;
    for (int off = kThreads / 2; off >= across; off >>= 1) {
      __syncthreads();
      if (static_cast<int>(threadIdx.x) < off) tile[threadIdx.x] = join(tile[threadIdx.x], tile[threadIdx.x + off]);
    }
    if (static_cast<int>(threadIdx.x) < across && h < heads) stats[first * heads + h] = tile[threadIdx.x];  // all have read the first piece
  }
}

template <typename T, int VEC, int K, int ORDER, int PHASE, int LANES = 0>
int start(const Rows& R, const Shape& S, const Operands<T>& o, Pair<Acc<T>>* stats, cudaStream_t stream) {
  // As many CTAs as are resident, which go from row to row: 2.6 M edges with 8 heads, forward 59 -> 46 us.  Rows of very different
  // length are handed out by the hardware instead: 1.0 M edges of hubs with 3 heads, FP64, 33 us, and 43 from row to row.
  const auto kernel = rows_kernel<T, VEC, K, ORDER, PHASE, LANES>;
  static rows::Kernel known;
  const int resident = known.resident(kernel, kThreads, 0);
  if (resident < 1) return resident;
  const int64_t parts = ceil_div(S.heads, S.across * VEC);
  const int64_t ctas = ceil_div(PHASE == kApply ? R.pieces : R.count, kThreads / S.lanes), most = PHASE == kMixed ? ctas : resident > parts ? resident / parts : 1;
  kernel<<<dim3(static_cast<unsigned>(ctas < most ? ctas : most), static_cast<unsigned>(parts)), kThreads, 0, stream>>>(R, S, o, stats);
  LUNA_LAUNCH_CHECK("softmax over in-edges");
  return LUNA_OK;
}

template <typename T, int VEC, int ORDER>
int launch(const Rows& R, int64_t edges, int64_t heads, int64_t num_buckets, const Operands<T>& o, void* scratch, cudaStream_t stream) {
  // Sixteen numbers of a thread in registers; single ones, with their exponentials and addresses, spill (forward, 2.6 M edges
  // with one head: 23 us, with eight 14; the backward has room: 8.3 and 9.8).  Pairs spill, too (90 to 130 bytes), and of
  // sixteen and eight either is faster somewhere: FP32, us, forward without and with bias and mask, second order: two heads 23 / 41 / 32
  // and 27 / 38 / 34, six 47 / 77 / 66 and 50 / 64 / 80.
  constexpr int K = sizeof(T) > 4 ? 8 / VEC : VEC == 1 && !is_backward(ORDER) ? 8 : 16 / VEC;
  Shape S{};
  S.heads = static_cast<int>(heads);
  S.num_buckets = static_cast<int>(num_buckets);
  const int64_t packets = heads / VEC;
  S.across = packets >= 32 ? 32 : rows::next_power_of_two(packets);
  // As many threads as hold a row (of the pieces, one) somewhat longer than the mean; a CTA where a warp would read most of a row twice:
  // four times what it holds.  2.6 M edges of 8 heads, FP32, in rows of 200, 250, 300, 400 and 500, by a warp or a CTA, us: forward 40,
  // 38, 41, 41, 45 or 88, 74, 65, 54, 49; backward 52, 57, 57, 60, 68 or 64, 56, 52, 48, 47.  It is the backward that changes sides where
  // the rule does (at 205 edges).
  const int64_t mean = ceil_div(edges, R.count);
  const int64_t wanted = ceil_div(mean + mean / 4, K) * S.across;
  S.lanes = wanted > 128 ? kThreads : wanted >= 32 ? 32 : rows::next_power_of_two(wanted);
  auto* stats = static_cast<Pair<Acc<T>>*>(scratch);
  if (!R.pieces) {
    if (S.across * VEC == S.heads && S.lanes == 32) return start<T, VEC, K, ORDER, kWhole, 32>(R, S, o, stats, stream);
    if (S.across * VEC == S.heads && S.lanes == 16) return start<T, VEC, K, ORDER, kWhole, 16>(R, S, o, stats, stream);
    if (S.across * VEC == S.heads && S.lanes == 8) return start<T, VEC, K, ORDER, kWhole, 8>(R, S, o, stats, stream);
    return start<T, VEC, K, ORDER, kWhole>(R, S, o, stats, stream);
  }
  if (const int status = start<T, VEC, K, ORDER, kMixed>(R, S, o, stats, stream)) return status;
  join_kernel<Acc<T>, ORDER == kForward><<<static_cast<unsigned>(R.cut), kThreads, 0, stream>>>(R, S.heads, S.across, stats);
  LUNA_LAUNCH_CHECK("softmax over in-edges: pieces");
  return start<T, VEC, K, ORDER, kApply>(R, S, o, stats, stream);
}

template <typename T, int ORDER>
int with_packets(int vec, const Rows& R, int64_t edges, int64_t heads, int64_t num_buckets, const Operands<T>& o, void* scratch,
                 cudaStream_t stream) {
  if constexpr (sizeof(T) <= 2) {
    if (vec == 8) return launch<T, 8, ORDER>(R, edges, heads, num_buckets, o, scratch, stream);
  }
  if constexpr (sizeof(T) <= 4) {
    if (vec == 4) return launch<T, 4, ORDER>(R, edges, heads, num_buckets, o, scratch, stream);
  }
  if (vec == 2) return launch<T, 2, ORDER>(R, edges, heads, num_buckets, o, scratch, stream);
  return launch<T, 1, ORDER>(R, edges, heads, num_buckets, o, scratch, stream);
}

template <typename T>
int run(Order order, int vec, const Rows& R, int64_t edges, int64_t heads, int64_t num_buckets, const Operands<T>& o, void* scratch,
        cudaStream_t stream) {
  if (order == kForward) return with_packets<T, kForward>(vec, R, edges, heads, num_buckets, o, scratch, stream);
  if (order == kBackward) return with_packets<T, kBackward>(vec, R, edges, heads, num_buckets, o, scratch, stream);
  if constexpr (sizeof(T) == 2) {
    if (order == kBackwardWide) return with_packets<T, kBackwardWide>(vec, R, edges, heads, num_buckets, o, scratch, stream);
  }
  return with_packets<T, kSecond>(vec, R, edges, heads, num_buckets, o, scratch, stream);
}

#define LUNA_SOFTMAX_RUN(T) \
  int run<T>(Order, int, const Rows&, int64_t, int64_t, int64_t, const Operands<T>&, void*, cudaStream_t)
extern template LUNA_SOFTMAX_RUN(float);
extern template LUNA_SOFTMAX_RUN(double);
extern template LUNA_SOFTMAX_RUN(rows::bf16);
extern template LUNA_SOFTMAX_RUN(rows::f16);

}  // namespace softmax
}  // namespace luna
