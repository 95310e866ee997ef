// Buckets of edge vectors by their length, the bias that a table gives to them, and the table's gradient.
#include "relative_bias.cuh"

namespace luna {
namespace bias {
namespace {

// bucket = number of boundaries b with b <= |v|, compared as b |b| <= |v|^2 in double precision: for single precision the
// squares are exact, so only the two additions round.  Boundaries ascend.  Bound by HBM: 12 (24) bytes in, 4 out.
// Four edges of a thread are searched for together, in as many steps for all of them.
constexpr int kSharedBoundaries = 2047;
template <typename T>
__global__ void __launch_bounds__(256)
buckets_kernel(const T* __restrict__ vec, const T* __restrict__ boundaries, int count, int32_t* __restrict__ out, int64_t edges,
               bool aligned) {
  __shared__ double squares[kSharedBoundaries];
  auto square = [&](int i) {
    const double b = static_cast<double>(boundaries[i]);
    return __dmul_rn(b, fabs(b));
  };
  int steps = 1;  // a power of two above the count
  while (steps <= count) steps <<= 1;
  const bool shared = count <= kSharedBoundaries;
  if (shared)
    for (int i = threadIdx.x; i < steps - 1; i += blockDim.x) squares[i] = i < count ? square(i) : __longlong_as_double(-1);  // no number
  __syncthreads();
  const int64_t step = static_cast<int64_t>(gridDim.x) * blockDim.x * 4;
  for (int64_t first = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) * 4; first < edges; first += step) {
    T v[12];
    if (aligned && first + 4 <= edges) {
      constexpr int per = 16 / static_cast<int>(sizeof(T));
#pragma unroll
      for (int i = 0; i < 12 / per; ++i) {
        const rows::Pack<T, per> p = reinterpret_cast<const rows::Pack<T, per>*>(vec + first * 3)[i];
#pragma unroll
        for (int c = 0; c < per; ++c) v[i * per + c] = p.a[c];
      }
    } else {
#pragma unroll
      for (int i = 0; i < 12; ++i) v[i] = first * 3 + i < edges * 3 ? vec[first * 3 + i] : T(0);
    }
    double length[4];
    int low[4] = {0, 0, 0, 0};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const double x = v[j * 3], y = v[j * 3 + 1], z = v[j * 3 + 2];
      length[j] = __dadd_rn(__dadd_rn(__dmul_rn(x, x), __dmul_rn(y, y)), __dmul_rn(z, z));
    }
    for (int half = steps >> 1; half; half >>= 1)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int next = low[j] + half;
        const double border = shared ? squares[next - 1] : next <= count ? square(next - 1) : __longlong_as_double(-1);
        low[j] = border <= length[j] ? next : low[j];
      }
    if (aligned && first + 4 <= edges) {
      *reinterpret_cast<int4*>(out + first) = make_int4(low[0], low[1], low[2], low[3]);
    } else {
      for (int j = 0; j < 4 && first + j < edges; ++j) out[first + j] = low[j];
    }
  }
}

template <typename T, int VEC>
void gather(const T* table, const int32_t* buckets, T* out, int64_t edges, int64_t num_buckets, int64_t heads, cudaStream_t stream) {
  const int64_t packets = heads / VEC;
  const int lanes = packets >= 32 ? 32 : rows::next_power_of_two(packets);
  // Short rows: the CTAs that are resident go from edge to edge (2 M edges of 8 floats, 8 or 128 CTAs a multiprocessor, 12 and 17 us);
  // long ones are handed out by the hardware (209,000 of 704 floats 100 and 84).
  const int64_t ctas = ceil_div(edges, 256 / lanes), most = static_cast<int64_t>(rows::processors()) * (lanes < 32 ? 8 : 128);
  gather_kernel<T, VEC><<<static_cast<unsigned>(ctas < most ? ctas : most), 256, 0, stream>>>(
      table, buckets, out, edges, static_cast<int>(num_buckets), static_cast<int>(heads), lanes);
}

int check(int dtype, int64_t edges, int64_t num_buckets, int64_t heads) {
  if (dtype < LUNA_F32 || dtype > LUNA_F16) return fail(LUNA_ERR_INVALID_ARGUMENT, "unknown dtype %d", dtype);
  if (edges < 0 || num_buckets < 1 || heads < 1) return fail(LUNA_ERR_INVALID_ARGUMENT, "a bias needs buckets and heads");
  if (num_buckets >= (1 << 30) || heads >= (1 << 20) || num_buckets * heads >= (1ll << 31))
    return fail(LUNA_ERR_UNSUPPORTED, "a table of %lld buckets and %lld heads", static_cast<long long>(num_buckets), static_cast<long long>(heads));
  return LUNA_OK;
}

int check_pointer(int64_t size, const void* p, const char* name, bool required) {
  if (!p) return required ? fail(LUNA_ERR_INVALID_ARGUMENT, "%s is null", name) : LUNA_OK;
  return aligned_to(p, size) ? LUNA_OK : fail(LUNA_ERR_MISALIGNED, "%s is not aligned to its element size", name);
}

}  // namespace
}  // namespace bias
}  // namespace luna

extern "C" int luna_distance_buckets(int dtype, const void* vec, const void* boundaries, int64_t num_boundaries, int32_t* out,
                                     int64_t n, void* stream) {
  using namespace luna;
  clear_error();
  if (dtype != LUNA_F32 && dtype != LUNA_F64) return fail(LUNA_ERR_INVALID_ARGUMENT, "vectors are float32 or float64");
  if (n < 0 || num_boundaries < 0) return fail(LUNA_ERR_INVALID_ARGUMENT, "negative size");
  if (num_boundaries >= (1 << 30)) return fail(LUNA_ERR_UNSUPPORTED, "too many boundaries");
  const int64_t size = rows::size_of(dtype);
  int status = bias::check_pointer(size, vec, "vec", n > 0);
  if (!status) status = bias::check_pointer(size, boundaries, "boundaries", num_boundaries > 0);
  if (!status) status = bias::check_pointer(4, out, "out", n > 0);
  if (status || n == 0) return status;
  const int64_t ctas = ceil_div(n, 1024), most = static_cast<int64_t>(rows::processors()) * 8;
  const bool aligned = aligned_to(vec, 16) && aligned_to(out, 16);
  const unsigned grid = static_cast<unsigned>(ctas < most ? ctas : most);
  const int count = static_cast<int>(num_boundaries);
  const auto s = static_cast<cudaStream_t>(stream);
  if (dtype == LUNA_F64)
    bias::buckets_kernel<double><<<grid, 256, 0, s>>>(static_cast<const double*>(vec), static_cast<const double*>(boundaries), count, out, n, aligned);
  else
    bias::buckets_kernel<float><<<grid, 256, 0, s>>>(static_cast<const float*>(vec), static_cast<const float*>(boundaries), count, out, n, aligned);
  LUNA_LAUNCH_CHECK("distance buckets");
  return LUNA_OK;
}

extern "C" int luna_relative_bias_fwd(int dtype, const void* table, const int32_t* buckets, void* out, int64_t edges,
                                      int64_t num_buckets, int64_t heads, void* stream) {
  using namespace luna;
  clear_error();
  int status = bias::check(dtype, edges, num_buckets, heads);
  const int64_t size = status ? 1 : rows::size_of(dtype);
  if (!status) status = bias::check_pointer(size, table, "table", edges > 0);
  if (!status) status = bias::check_pointer(4, buckets, "buckets", edges > 0);
  if (!status) status = bias::check_pointer(size, out, "out", edges > 0);
  if (status || edges == 0) return status;
  const auto s = static_cast<cudaStream_t>(stream);
  // moved as bits: the type's size is all that matters
  auto move = [&](auto unit) {
    using U = decltype(unit);
    const U* from = static_cast<const U*>(table);
    U* to = static_cast<U*>(out);
    switch (bias::packet_of(sizeof(U), heads, {table, out})) {
      case 1: bias::gather<U, 1>(from, buckets, to, edges, num_buckets, heads, s); break;
      case 2: bias::gather<U, 2>(from, buckets, to, edges, num_buckets, heads, s); break;
      case 4: if constexpr (sizeof(U) <= 4) bias::gather<U, 4>(from, buckets, to, edges, num_buckets, heads, s); break;
      case 8: if constexpr (sizeof(U) <= 2) bias::gather<U, 8>(from, buckets, to, edges, num_buckets, heads, s); break;
    }
  };
  if (size == 8) move(uint64_t());
  else if (size == 4) move(uint32_t());
  else move(uint16_t());
  LUNA_LAUNCH_CHECK("relative bias");
  return LUNA_OK;
}

extern "C" int64_t luna_relative_bias_scratch_bytes(int dtype, int64_t edges, int64_t num_buckets, int64_t heads) {
  using namespace luna;
  clear_error();
  if (const int status = bias::check(dtype, edges, num_buckets, heads)) return status;
  return bias::partial_numbers(rows::size_of(dtype), rows::acc_size_of(dtype), edges, num_buckets, heads) * rows::acc_size_of(dtype);
}

extern "C" int luna_relative_bias_bwd(int dtype, const void* g, const int32_t* buckets, void* gtable, void* scratch,
                                      int64_t scratch_bytes, int64_t edges, int64_t num_buckets, int64_t heads, void* stream) {
  using namespace luna;
  const int64_t needed = luna_relative_bias_scratch_bytes(dtype, edges, num_buckets, heads);
  if (needed < 0) return static_cast<int>(needed);
  const int64_t size = rows::size_of(dtype);
  int status = bias::check_pointer(size, g, "g", edges > 0);
  if (!status) status = bias::check_pointer(4, buckets, "buckets", edges > 0);
  if (!status) status = bias::check_pointer(size, gtable, "gtable", true);
  if (status) return status;
  if (!scratch || scratch_bytes < needed)
    return fail(LUNA_ERR_SCRATCH, "the gradient of a bias table needs %lld bytes of scratch, got %lld", static_cast<long long>(needed),
                static_cast<long long>(scratch ? scratch_bytes : 0));
  if (!aligned_to(scratch, 16)) return fail(LUNA_ERR_MISALIGNED, "scratch is not aligned to 16 bytes");
  rows::with_type(dtype, [&](auto zero) {
    status = bias::table_gradient<decltype(zero), decltype(zero)>(g, buckets, gtable, scratch, edges, num_buckets, heads, static_cast<cudaStream_t>(stream));
  });
  return status;
}
