// C entry points of the layer norm over irreps; the kernels are in layer_norm.cuh.
#include <cmath>

#include "layer_norm.cuh"

namespace luna {
namespace norm {
namespace {

int describe(const luna_norm_desc* desc, int64_t rows, Params* P) {
  if (!desc) return fail(LUNA_ERR_INVALID_ARGUMENT, "null description");
  if (desc->dtype < LUNA_F32 || desc->dtype > LUNA_F16) return fail(LUNA_ERR_INVALID_ARGUMENT, "unknown dtype %d", desc->dtype);
  if (desc->num_blocks < 1) return fail(LUNA_ERR_INVALID_ARGUMENT, "layer norm needs a block at least");
  if (desc->num_blocks > kMaxBlocks) return fail(LUNA_ERR_UNSUPPORTED, "layer norm of more than %d blocks", kMaxBlocks);
  if (desc->normalization != 0 && desc->normalization != 1) return fail(LUNA_ERR_INVALID_ARGUMENT, "unknown normalization %d", desc->normalization);
  if (!(desc->eps >= 0.0) || !std::isfinite(desc->eps)) return fail(LUNA_ERR_INVALID_ARGUMENT, "eps must be finite and not negative");
  if (rows < 0) return fail(LUNA_ERR_INVALID_ARGUMENT, "negative number of rows");
  *P = Params{};
  P->blocks = desc->num_blocks;
  P->rows = rows;
  P->eps = desc->eps;
  int weights = 0, biases = 0;
  for (int i = 0; i < desc->num_blocks; ++i) {
    const int mul = desc->mul[i], components = desc->components[i];
    if (mul < 1 || components < 1 || components % 2 == 0 || (desc->scalar[i] && components != 1))
      return fail(LUNA_ERR_INVALID_ARGUMENT, "block %d has %d channels of %d components", i, mul, components);
    if (static_cast<int64_t>(mul) * components > kMaxLength)
      return fail(LUNA_ERR_UNSUPPORTED, "layer norm of a block with more than %d elements", kMaxLength);
    Block& B = P->block[i];
    B.offset = P->dim;
    B.length = mul * components;
    B.channels = mul;
    B.components = components;
    B.scalar = desc->scalar[i] != 0;
    B.weight_offset = weights;
    B.bias_offset = biases;
    B.inverse = static_cast<unsigned>(((1ull << 32) + components - 1) / components);
    B.share = 1.0 / (desc->normalization == 0 ? B.length : mul);
    P->dim += B.length;
    weights += mul;
    biases += B.scalar ? mul : 0;
  }
  return LUNA_OK;
}

int checked(const luna_norm_desc* desc, const void* p, const char* name, bool required) {
  if (!p) return required ? fail(LUNA_ERR_INVALID_ARGUMENT, "%s is null", name) : LUNA_OK;
  return aligned_to(p, rows::size_of(desc->dtype)) ? LUNA_OK : fail(LUNA_ERR_MISALIGNED, "%s is not aligned to its element size", name);
}

int checked_stats(const luna_norm_desc* desc, const void* stats, bool required) {
  if (!stats) return required ? fail(LUNA_ERR_INVALID_ARGUMENT, "stats is null") : LUNA_OK;
  return aligned_to(stats, 2 * rows::acc_size_of(desc->dtype)) ? LUNA_OK : fail(LUNA_ERR_MISALIGNED, "stats is not aligned to a pair");
}

int dispatch(Order order, const luna_norm_desc* desc, const Params& P, const Call& o, void* stream) {
  int status = LUNA_OK;
  rows::with_type(desc->dtype, [&](auto zero) { status = run<decltype(zero)>(order, P, o, static_cast<cudaStream_t>(stream)); });
  return status;
}

int check_scratch(const luna_norm_desc* desc, const Params& P, const Call& o) {
  if (!o.gw && !o.gb) return LUNA_OK;
  const int64_t needed = scratch_elements(P) * rows::acc_size_of(desc->dtype);
  if (!o.scratch || o.scratch_bytes < needed)
    return fail(LUNA_ERR_SCRATCH, "layer norm needs %lld bytes of scratch, got %lld", static_cast<long long>(needed),
                static_cast<long long>(o.scratch ? o.scratch_bytes : 0));
  return aligned_to(o.scratch, 16) ? LUNA_OK : fail(LUNA_ERR_MISALIGNED, "scratch is not aligned to 16 bytes");
}

}  // namespace
}  // namespace norm
}  // namespace luna

#define LUNA_TRY(expr)                   \
  do {                                   \
    const int luna_status_ = (expr);     \
    if (luna_status_) return luna_status_; \
  } while (0)

extern "C" int64_t luna_layer_norm_scratch_bytes(const luna_norm_desc* desc, int64_t rows) {
  luna::clear_error();
  luna::norm::Params P;
  LUNA_TRY(luna::norm::describe(desc, rows, &P));
  return luna::norm::scratch_elements(P) * luna::rows::acc_size_of(desc->dtype);
}

extern "C" int luna_layer_norm_fwd(const luna_norm_desc* desc, const void* x, const void* weight, const void* bias, void* y,
                                   void* stats, int64_t rows, void* stream) {
  using namespace luna::norm;
  luna::clear_error();
  Params P;
  LUNA_TRY(describe(desc, rows, &P));
  LUNA_TRY(checked(desc, x, "x", rows > 0));
  LUNA_TRY(checked(desc, y, "y", rows > 0));
  LUNA_TRY(checked(desc, weight, "weight", false));
  LUNA_TRY(checked(desc, bias, "bias", false));
  LUNA_TRY(checked_stats(desc, stats, false));
  if (rows == 0) return LUNA_OK;
  Call o{};
  o.x = x, o.weight = weight, o.bias = bias, o.y = y, o.stats_out = stats;
  return dispatch(kForward, desc, P, o, stream);
}

extern "C" int luna_layer_norm_bwd(const luna_norm_desc* desc, const void* x, const void* weight, const void* stats, const void* g,
                                   void* gx, void* gw, void* gb, void* scratch, int64_t scratch_bytes, int64_t rows, void* stream) {
  using namespace luna::norm;
  luna::clear_error();
  Params P;
  LUNA_TRY(describe(desc, rows, &P));
  LUNA_TRY(checked(desc, x, "x", rows > 0));
  LUNA_TRY(checked(desc, g, "g", rows > 0));
  LUNA_TRY(checked(desc, weight, "weight", false));
  LUNA_TRY(checked(desc, gx, "gx", false));
  LUNA_TRY(checked(desc, gw, "gw", false));
  LUNA_TRY(checked(desc, gb, "gb", false));
  LUNA_TRY(checked_stats(desc, stats, rows > 0));
  if (!gw && !gb && (!gx || rows == 0)) return LUNA_OK;
  Call o{};
  o.x = x, o.weight = weight, o.stats_in = stats, o.g = g, o.gx = gx, o.gw = gw, o.gb = gb, o.scratch = scratch,
  o.scratch_bytes = scratch_bytes;
  LUNA_TRY(check_scratch(desc, P, o));
  return dispatch(kBackward, desc, P, o, stream);
}

extern "C" int luna_layer_norm_dbl_bwd(const luna_norm_desc* desc, const void* x, const void* weight, const void* stats, const void* g,
                                       const void* rx, const void* rw, const void* rb, void* hx, void* hw, void* hg, void* scratch,
                                       int64_t scratch_bytes, int64_t rows, void* stream) {
  using namespace luna::norm;
  luna::clear_error();
  Params P;
  LUNA_TRY(describe(desc, rows, &P));
  LUNA_TRY(checked(desc, x, "x", rows > 0));
  LUNA_TRY(checked(desc, g, "g", rows > 0));
  LUNA_TRY(checked(desc, weight, "weight", false));
  LUNA_TRY(checked(desc, rx, "rx", false));
  LUNA_TRY(checked(desc, rw, "rw", false));
  LUNA_TRY(checked(desc, rb, "rb", false));
  LUNA_TRY(checked(desc, hx, "hx", false));
  LUNA_TRY(checked(desc, hw, "hw", false));
  LUNA_TRY(checked(desc, hg, "hg", false));
  LUNA_TRY(checked_stats(desc, stats, rows > 0));
  if (!hw && ((!hx && !hg) || rows == 0)) return LUNA_OK;
  Call o{};
  o.x = x, o.weight = weight, o.stats_in = stats, o.g = g, o.rx = rx, o.rw = rw, o.rb = rb, o.hx = hx, o.gw = hw, o.hg = hg,
  o.scratch = scratch, o.scratch_bytes = scratch_bytes;
  LUNA_TRY(check_scratch(desc, P, o));
  return dispatch(kSecond, desc, P, o, stream);
}
