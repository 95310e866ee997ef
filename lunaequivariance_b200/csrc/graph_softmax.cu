// C entry points of the softmax over in-edges; the kernels are in graph_softmax.cuh.
#include "graph_softmax.cuh"
#include "relative_bias.cuh"

namespace luna {
namespace softmax {
namespace {

struct Call {
  int dtype;
  const luna_row_table* table;
  int64_t heads, num_buckets;
  const int32_t* buckets;
};

int describe(const Call& c, Rows* R) {
  if (c.dtype < LUNA_F32 || c.dtype > LUNA_F16) return fail(LUNA_ERR_INVALID_ARGUMENT, "unknown dtype %d", c.dtype);
  if (!c.table) return fail(LUNA_ERR_INVALID_ARGUMENT, "null row table");
  const luna_row_table& t = *c.table;
  if (t.num_rows < 0 || t.num_edges < 0 || t.num_pieces < 0 || t.num_cut < 0 || c.num_buckets < 0)
    return fail(LUNA_ERR_INVALID_ARGUMENT, "negative size");
  if (c.heads < 1) return fail(LUNA_ERR_INVALID_ARGUMENT, "softmax needs a head at least");
  if (c.heads >= (1 << 20)) return fail(LUNA_ERR_UNSUPPORTED, "softmax of %lld heads", static_cast<long long>(c.heads));
  if (c.num_buckets >= (1 << 30)) return fail(LUNA_ERR_UNSUPPORTED, "softmax with %lld buckets", static_cast<long long>(c.num_buckets));
  if (t.num_rows >= (1ll << 31) || t.num_edges >= (1ll << 31) - 1024)
    return fail(LUNA_ERR_OVERFLOW, "graph exceeds the 32-bit index range of this build");
  if (t.num_edges > 0 && (t.num_rows == 0 || !t.rowptr)) return fail(LUNA_ERR_INVALID_ARGUMENT, "row pointers missing");
  if (t.num_pieces > t.num_rows || t.num_cut > t.num_pieces || (t.num_pieces > 0) != (t.num_cut > 0))
    return fail(LUNA_ERR_INVALID_ARGUMENT, "pieces that no rows have");
  if (t.num_pieces > 0 && (!t.piece_of_row || !t.row_of_piece || !t.cut_of_piece || !t.cut_first))
    return fail(LUNA_ERR_INVALID_ARGUMENT, "tables of the pieces missing");
  for (const int32_t* p : {t.rowptr, t.piece_of_row, t.row_of_piece, t.cut_of_piece, t.cut_first, c.buckets})
    if (!aligned_to(p, 4)) return fail(LUNA_ERR_MISALIGNED, "a table of 32-bit indices is not aligned to them");
  *R = Rows{t.rowptr, t.num_rows, t.num_pieces, t.num_cut, t.piece_of_row, t.row_of_piece, t.cut_of_piece, t.cut_first};
  return LUNA_OK;
}

int pointer(const Call& c, const void* p, const char* name, bool required) {
  if (!p) return required ? fail(LUNA_ERR_INVALID_ARGUMENT, "%s is null", name) : LUNA_OK;
  return aligned_to(p, rows::size_of(c.dtype)) ? LUNA_OK : fail(LUNA_ERR_MISALIGNED, "%s is not aligned to its element size", name);
}

// In the type that sums are held in, whole packets of 16 bytes.
int wide_pointer(const Call& c, const void* p, const char* name, bool required) {
  if (!p) return required ? fail(LUNA_ERR_INVALID_ARGUMENT, "%s is null", name) : LUNA_OK;
  return aligned_to(p, c.dtype == LUNA_BF16 || c.dtype == LUNA_F16 ? 16 : rows::acc_size_of(c.dtype))
             ? LUNA_OK : fail(LUNA_ERR_MISALIGNED, "%s is not aligned to 16 bytes", name);
}

// Room for the sums of the pieces, rounded up, so that what follows it is aligned.
int64_t pieces_bytes(const Call& c) {
  return ceil_div(c.table->num_pieces * c.heads * 2 * rows::acc_size_of(c.dtype), 16) * 16;
}

// 16-bit types: room for the logits' gradient as it is before it is rounded, of which the table's is made.
int64_t unrounded_bytes(const Call& c) {
  return c.dtype == LUNA_BF16 || c.dtype == LUNA_F16 ? ceil_div(c.table->num_edges * c.heads * 4, 16) * 16 : 0;
}
// The type that the table's gradient is summed from.
int summed_dtype(int dtype) { return dtype == LUNA_BF16 || dtype == LUNA_F16 ? LUNA_F32 : dtype; }

int scratch_fits(int64_t needed, const void* scratch, int64_t bytes) {
  if (!needed) return LUNA_OK;
  if (!scratch || bytes < needed)
    return fail(LUNA_ERR_SCRATCH, "softmax over in-edges needs %lld bytes of scratch, got %lld", static_cast<long long>(needed),
                static_cast<long long>(scratch ? bytes : 0));
  return aligned_to(scratch, 16) ? LUNA_OK : fail(LUNA_ERR_MISALIGNED, "scratch is not aligned to 16 bytes");
}

}  // namespace
}  // namespace softmax
}  // namespace luna

using luna::softmax::Call;

extern "C" int64_t luna_graph_softmax_scratch_bytes(int dtype, const luna_row_table* rows, int64_t heads, int64_t num_buckets) {
  luna::clear_error();
  const Call call{dtype, rows, heads, num_buckets, nullptr};
  luna::softmax::Rows R;
  if (const int status = luna::softmax::describe(call, &R)) return status;
  int64_t bytes = luna::softmax::pieces_bytes(call);
  if (num_buckets > 0) {
    const int64_t more = luna_relative_bias_scratch_bytes(luna::softmax::summed_dtype(dtype), rows->num_edges, num_buckets, heads);
    if (more < 0) return more;
    bytes += more + luna::softmax::unrounded_bytes(call);
  }
  return bytes;
}

extern "C" int luna_graph_softmax_fwd(int dtype, const luna_row_table* rows, const void* logits, const void* table,
                                      const int32_t* buckets, const uint8_t* mask, void* alpha, void* wide, int64_t heads,
                                      int64_t num_buckets, void* scratch, int64_t scratch_bytes, void* stream) {
  using namespace luna;
  clear_error();
  const Call call{dtype, rows, heads, num_buckets, buckets};
  softmax::Rows R;
  int status = softmax::describe(call, &R);
  if (status) return status;
  const bool any = rows->num_edges > 0;
  if ((status = softmax::pointer(call, logits, "logits", any))) return status;
  if ((status = softmax::pointer(call, alpha, "alpha", any))) return status;
  if ((status = softmax::pointer(call, table, "table", false))) return status;
  if ((status = softmax::wide_pointer(call, wide, "wide", false))) return status;
  if (table && any && (!buckets || num_buckets < 1)) return fail(LUNA_ERR_INVALID_ARGUMENT, "a table needs buckets");
  if ((status = softmax::scratch_fits(softmax::pieces_bytes(call), scratch, scratch_bytes))) return status;
  if (!any) return LUNA_OK;
  rows::with_type(dtype, [&](auto zero) {
    using T = decltype(zero);
    softmax::Operands<T> o{};
    o.logits = static_cast<const T*>(logits);
    o.table = static_cast<const T*>(table);
    o.buckets = buckets;
    o.mask = mask;
    o.out = static_cast<T*>(alpha);
    o.wide = sizeof(T) == 2 ? static_cast<rows::Acc<T>*>(wide) : nullptr;
    status = softmax::run<T>(softmax::kForward, bias::packet_of(sizeof(T), heads, {logits, table, alpha}), R, rows->num_edges, heads,
                             num_buckets, o, scratch, static_cast<cudaStream_t>(stream));
  });
  return status;
}

namespace {

// wide: g in float for the 16-bit types
int backward(int dtype, const luna_row_table* rows, const void* alpha, const void* g, bool wide_g, const int32_t* buckets, void* glogits,
             void* gtable, int64_t heads, int64_t num_buckets, void* scratch, int64_t scratch_bytes, void* stream) {
  using namespace luna;
  clear_error();
  const Call call{dtype, rows, heads, num_buckets, buckets};
  softmax::Rows R;
  int status = softmax::describe(call, &R);
  if (status) return status;
  const bool any = rows->num_edges > 0;
  if ((status = softmax::wide_pointer(call, alpha, "alpha", any))) return status;
  if ((status = wide_g ? softmax::wide_pointer(call, g, "g", any) : softmax::pointer(call, g, "g", any))) return status;
  if ((status = softmax::pointer(call, glogits, "glogits", any))) return status;
  if ((status = softmax::pointer(call, gtable, "gtable", false))) return status;
  if (gtable && ((any && !buckets) || num_buckets < 1)) return fail(LUNA_ERR_INVALID_ARGUMENT, "a table needs buckets");
  const int64_t pieces = softmax::pieces_bytes(call), unrounded = gtable ? softmax::unrounded_bytes(call) : 0;
  int64_t sums = 0;
  if (gtable) {
    sums = luna_relative_bias_scratch_bytes(softmax::summed_dtype(dtype), rows->num_edges, num_buckets, heads);
    if (sums < 0) return static_cast<int>(sums);
  }
  if ((status = softmax::scratch_fits(pieces + unrounded + sums, scratch, scratch_bytes))) return status;
  auto* const room = static_cast<unsigned char*>(scratch);
  void* const wide = unrounded ? room + pieces : nullptr;
  if (any)
    rows::with_type(dtype, [&](auto zero) {
      using T = decltype(zero);
      softmax::Operands<T> o{};
      const bool widened = wide_g && sizeof(T) == 2;
      o.alpha = static_cast<const rows::Acc<T>*>(alpha);
      o.g = static_cast<const T*>(g);
      o.gwide = static_cast<const rows::Acc<T>*>(g);
      o.out = static_cast<T*>(glogits);
      o.wide = static_cast<rows::Acc<T>*>(wide);
      const int vec = widened          ? bias::packet_of(sizeof(T), heads, {glogits})
                      : sizeof(T) == 2 ? bias::packet_of(sizeof(T), heads, {g, glogits})
                                       : bias::packet_of(sizeof(T), heads, {alpha, g, glogits});
      status = softmax::run<T>(widened ? softmax::kBackwardWide : softmax::kBackward, vec, R, rows->num_edges, heads, num_buckets, o, scratch,
                               static_cast<cudaStream_t>(stream));
    });
  if (status || !gtable) return status;
  rows::with_type(dtype, [&](auto zero) {
    using T = decltype(zero);
    const auto on = static_cast<cudaStream_t>(stream);
    void* const parts = room + pieces + unrounded;
    if constexpr (sizeof(T) == 2)
      status = bias::table_gradient<float, T>(wide, buckets, gtable, parts, rows->num_edges, num_buckets, heads, on);
    else
      status = bias::table_gradient<T, T>(glogits, buckets, gtable, parts, rows->num_edges, num_buckets, heads, on);
  });
  return status;
}

// wide: halpha in float for the 16-bit types
int second_order(int dtype, const luna_row_table* rows, const void* alpha, const void* g, const void* r, const void* rtable,
                 const int32_t* buckets, void* halpha, bool wide_halpha, void* hg, int64_t heads, int64_t num_buckets, void* scratch,
                 int64_t scratch_bytes, void* stream) {
  using namespace luna;
  clear_error();
  const Call call{dtype, rows, heads, num_buckets, buckets};
  softmax::Rows R;
  int status = softmax::describe(call, &R);
  if (status) return status;
  const bool any = rows->num_edges > 0;
  if ((status = softmax::wide_pointer(call, alpha, "alpha", any))) return status;
  if ((status = softmax::pointer(call, g, "g", any))) return status;
  if ((status = softmax::pointer(call, r, "r", false))) return status;
  if ((status = softmax::pointer(call, rtable, "rtable", false))) return status;
  if ((status = wide_halpha ? softmax::wide_pointer(call, halpha, "halpha", false) : softmax::pointer(call, halpha, "halpha", false))) return status;
  if ((status = softmax::pointer(call, hg, "hg", false))) return status;
  if (rtable && any && (!buckets || num_buckets < 1)) return fail(LUNA_ERR_INVALID_ARGUMENT, "a table needs buckets");
  if ((status = softmax::scratch_fits(softmax::pieces_bytes(call), scratch, scratch_bytes))) return status;
  if (!any || (!halpha && !hg)) return LUNA_OK;
  rows::with_type(dtype, [&](auto zero) {
    using T = decltype(zero);
    softmax::Operands<T> o{};
    o.alpha = static_cast<const rows::Acc<T>*>(alpha);
    o.g = static_cast<const T*>(g);
    o.r = static_cast<const T*>(r);
    o.rtable = static_cast<const T*>(rtable);
    o.buckets = buckets;
    o.out = static_cast<T*>(hg);
    if (wide_halpha && sizeof(T) == 2)
      o.wide = static_cast<rows::Acc<T>*>(halpha);  // aligned to 16 bytes: to whole packets of T, whatever they are
    else
      o.out2 = static_cast<T*>(halpha);
    const int vec = sizeof(T) == 2 ? bias::packet_of(sizeof(T), heads, {g, r, rtable, halpha, hg})
                                   : bias::packet_of(sizeof(T), heads, {alpha, g, r, rtable, halpha, hg});
    status = softmax::run<T>(softmax::kSecond, vec, R, rows->num_edges, heads, num_buckets, o, scratch, static_cast<cudaStream_t>(stream));
  });
  return status;
}

}  // namespace

extern "C" int luna_graph_softmax_bwd(int dtype, const luna_row_table* rows, const void* alpha, const void* g, const int32_t* buckets,
                                      void* glogits, void* gtable, int64_t heads, int64_t num_buckets, void* scratch,
                                      int64_t scratch_bytes, void* stream) {
  return backward(dtype, rows, alpha, g, false, buckets, glogits, gtable, heads, num_buckets, scratch, scratch_bytes, stream);
}
extern "C" int luna_graph_softmax_bwd_wide(int dtype, const luna_row_table* rows, const void* alpha, const void* g, const int32_t* buckets,
                                           void* glogits, void* gtable, int64_t heads, int64_t num_buckets, void* scratch,
                                           int64_t scratch_bytes, void* stream) {
  return backward(dtype, rows, alpha, g, true, buckets, glogits, gtable, heads, num_buckets, scratch, scratch_bytes, stream);
}
extern "C" int luna_graph_softmax_dbl_bwd(int dtype, const luna_row_table* rows, const void* alpha, const void* g, const void* r,
                                          const void* rtable, const int32_t* buckets, void* halpha, void* hg, int64_t heads,
                                          int64_t num_buckets, void* scratch, int64_t scratch_bytes, void* stream) {
  return second_order(dtype, rows, alpha, g, r, rtable, buckets, halpha, false, hg, heads, num_buckets, scratch, scratch_bytes, stream);
}
extern "C" int luna_graph_softmax_dbl_bwd_wide(int dtype, const luna_row_table* rows, const void* alpha, const void* g, const void* r,
                                               const void* rtable, const int32_t* buckets, void* halpha, void* hg, int64_t heads,
                                               int64_t num_buckets, void* scratch, int64_t scratch_bytes, void* stream) {
  return second_order(dtype, rows, alpha, g, r, rtable, buckets, halpha, true, hg, heads, num_buckets, scratch, scratch_bytes, stream);
}
