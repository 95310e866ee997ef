// PyTorch side of the launch path in C++: argument checks, output allocation, the stream lookup and the autograd chain of
// the convolution and of the spherical harmonics.  A small convolution takes a few microseconds on the GPU; the same
// chain in Python costs some two hundred per forward and backward.
//
// The C-ABI library stays the product: this module only calls its entry points (resolved at load time from the path
// Python passes, so that both use the same build) and has no kernels of its own.
//
// Autograd.  F(x, y, w, g) is linear in every operand; ConvForward is dF/dg, ConvBackward the other three first
// derivatives, ConvDouble the derivatives of ConvBackward, and everything beyond is made of ConvPartial, the derivative
// of F with respect to one operand, whose own derivatives are again ConvPartial.  Which gradients are worth computing is
// asked from the running graph task (needs_input_grad).
#include <dlfcn.h>

#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/extension.h>

#include <algorithm>
#include <array>
#include <memory>
#include <mutex>
#include <optional>
#include <utility>

#include "../../include/luna_b200.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::Function;
using torch::autograd::Variable;
using torch::autograd::variable_list;

// ---- the library ------------------------------------------------------------------------------------------------------
struct Api {
  decltype(&luna_last_error) last_error = nullptr;
  decltype(&luna_uvu_plan_destroy) plan_destroy = nullptr;
  decltype(&luna_uvu_plan_query) plan_query = nullptr;
  decltype(&luna_uvu_conv_scratch_bytes) scratch_bytes = nullptr;
  decltype(&luna_uvu_conv_fwd) fwd = nullptr;
  decltype(&luna_uvu_conv_bwd) bwd = nullptr, bwd_add_gw = nullptr;
  decltype(&luna_uvu_conv_dbl_bwd) dbl_bwd = nullptr;
  decltype(&luna_graph_scratch_bytes) graph_scratch_bytes = nullptr;
  decltype(&luna_graph_build_all) graph_build_all = nullptr;
  decltype(&luna_sh_fwd) sh_fwd = nullptr;
  decltype(&luna_sh_bwd) sh_bwd = nullptr;
  decltype(&luna_sh_dbl_bwd) sh_dbl_bwd = nullptr;
  decltype(&luna_layer_norm_scratch_bytes) norm_scratch_bytes = nullptr;
  decltype(&luna_layer_norm_fwd) norm_fwd = nullptr;
  decltype(&luna_layer_norm_bwd) norm_bwd = nullptr;
  decltype(&luna_layer_norm_dbl_bwd) norm_dbl_bwd = nullptr;
  decltype(&luna_distance_buckets) distance_buckets = nullptr;
  decltype(&luna_relative_bias_fwd) bias_fwd = nullptr;
  decltype(&luna_relative_bias_scratch_bytes) bias_scratch_bytes = nullptr;
  decltype(&luna_relative_bias_bwd) bias_bwd = nullptr;
  decltype(&luna_graph_softmax_scratch_bytes) softmax_scratch_bytes = nullptr;
  decltype(&luna_graph_softmax_fwd) softmax_fwd = nullptr;
  decltype(&luna_graph_softmax_bwd) softmax_bwd = nullptr, softmax_bwd_wide = nullptr;
  decltype(&luna_graph_softmax_dbl_bwd_wide) softmax_dbl_bwd_wide = nullptr;
} api;

template <typename F>
void resolve(void* library, const char* name, F& function) {
  function = reinterpret_cast<F>(dlsym(library, name));
  TORCH_CHECK(function != nullptr, "symbol ", name, " is missing from the library");
}

void load(const std::string& path) {
  void* library = dlopen(path.c_str(), RTLD_NOW | RTLD_LOCAL);
  TORCH_CHECK(library != nullptr, "cannot load ", path, ": ", dlerror());
  resolve(library, "luna_last_error", api.last_error);
  resolve(library, "luna_uvu_plan_destroy", api.plan_destroy);
  resolve(library, "luna_uvu_plan_query", api.plan_query);
  resolve(library, "luna_uvu_conv_scratch_bytes", api.scratch_bytes);
  resolve(library, "luna_uvu_conv_fwd", api.fwd);
  resolve(library, "luna_uvu_conv_bwd", api.bwd);
  resolve(library, "luna_uvu_conv_bwd_add_gw", api.bwd_add_gw);
  resolve(library, "luna_uvu_conv_dbl_bwd", api.dbl_bwd);
  resolve(library, "luna_graph_scratch_bytes", api.graph_scratch_bytes);
  resolve(library, "luna_graph_build_all", api.graph_build_all);
  resolve(library, "luna_sh_fwd", api.sh_fwd);
  resolve(library, "luna_sh_bwd", api.sh_bwd);
  resolve(library, "luna_sh_dbl_bwd", api.sh_dbl_bwd);
  resolve(library, "luna_layer_norm_scratch_bytes", api.norm_scratch_bytes);
  resolve(library, "luna_layer_norm_fwd", api.norm_fwd);
  resolve(library, "luna_layer_norm_bwd", api.norm_bwd);
  resolve(library, "luna_layer_norm_dbl_bwd", api.norm_dbl_bwd);
  resolve(library, "luna_distance_buckets", api.distance_buckets);
  resolve(library, "luna_relative_bias_fwd", api.bias_fwd);
  resolve(library, "luna_relative_bias_scratch_bytes", api.bias_scratch_bytes);
  resolve(library, "luna_relative_bias_bwd", api.bias_bwd);
  resolve(library, "luna_graph_softmax_scratch_bytes", api.softmax_scratch_bytes);
  resolve(library, "luna_graph_softmax_fwd", api.softmax_fwd);
  resolve(library, "luna_graph_softmax_bwd", api.softmax_bwd);
  resolve(library, "luna_graph_softmax_bwd_wide", api.softmax_bwd_wide);
  resolve(library, "luna_graph_softmax_dbl_bwd_wide", api.softmax_dbl_bwd_wide);
}

// A failed status as the exception Python raises for it.
void check(int status) {
  if (C10_LIKELY(status == LUNA_OK)) return;
  const char* text = api.last_error();
  switch (status) {
    case LUNA_ERR_INVALID_ARGUMENT:
    case LUNA_ERR_MISALIGNED:
      TORCH_CHECK_VALUE(false, text);
    case LUNA_ERR_UNSUPPORTED:
      TORCH_CHECK_NOT_IMPLEMENTED(false, text);
    default:
      TORCH_CHECK(false, text, " (status ", status, ")");
  }
}

// ---- handles kept by Python and by autograd nodes -----------------------------------------------------------------------
struct Op : torch::CustomClassHolder {
  luna_uvu_plan* plan;
  int64_t X, Y, O, W;
  at::ScalarType dtype;
  Op(int64_t handle, int64_t x, int64_t y, int64_t o, int64_t w, bool f64)
      : plan(reinterpret_cast<luna_uvu_plan*>(handle)), X(x), Y(y), O(o), W(w), dtype(f64 ? at::kDouble : at::kFloat) {}
  ~Op() override { api.plan_destroy(plan); }
};

struct Graph : torch::CustomClassHolder {
  std::array<Tensor, 5> tables;  // src, dst, dst_rowptr, src_rowptr, edge_ids_by_src
  luna_graph native{};
  Graph(std::array<Tensor, 5> t, int64_t nodes, int64_t source_rows) : tables(std::move(t)) {
    native.num_nodes = nodes;
    native.num_src_nodes = source_rows;
    native.num_edges = tables[0].numel();
    native.src = tables[0].data_ptr<int32_t>();
    native.dst = tables[1].data_ptr<int32_t>();
    native.dst_rowptr = tables[2].data_ptr<int32_t>();
    native.src_rowptr = tables[3].data_ptr<int32_t>();
    native.edge_ids_by_src = tables[4].data_ptr<int32_t>();
  }
};

using OpPtr = c10::intrusive_ptr<Op>;
using GraphPtr = c10::intrusive_ptr<Graph>;

template <typename H>
void keep(AutogradContext* ctx, const char* name, const c10::intrusive_ptr<H>& holder) {
  ctx->saved_data[name] = c10::IValue::make_capsule(holder);
}
template <typename H>
c10::intrusive_ptr<H> kept(AutogradContext* ctx, const char* name) {
  return c10::static_intrusive_pointer_cast<H>(ctx->saved_data[name].toCapsule());
}

// ---- launch wrappers ----------------------------------------------------------------------------------------------------
// Contiguous and 16-byte aligned (the staged kernels move 16-byte pieces of rows).
Tensor prepared(const Tensor& t) {
  if (!t.defined()) return t;
  Tensor c = t.contiguous();
  return reinterpret_cast<uintptr_t>(c.data_ptr()) % 16 ? c.clone() : c;
}

// The kernels compute values only.  An operand of forward-mode AD does not have to require grad, so it can reach a launch
// without passing an autograd function; its tangent would be dropped, which reads as a derivative of zero.
void refuse_tangents(std::initializer_list<const Tensor*> tensors) {
  for (const Tensor* t : tensors)
    TORCH_CHECK_NOT_IMPLEMENTED(!t->defined() || !t->_fw_grad(0).defined(),
                                "forward-mode automatic differentiation is not provided");
}

void check_operand(const Op& op, const Tensor& x, const Tensor& t, const char* name, int64_t rows, int64_t columns) {
  if (!t.defined()) return;
  TORCH_CHECK_TYPE(t.scalar_type() == op.dtype, name, " must be ", op.dtype == at::kDouble ? "torch.float64" : "torch.float32",
                   ", got ", t.scalar_type());
  TORCH_CHECK_VALUE(t.device() == x.device(), "features, weights and graph must share one CUDA device");
  TORCH_CHECK_VALUE(t.dim() == 2 && t.size(0) == rows && t.size(1) == columns, name, " must have shape (", rows, ", ",
                    columns, "), got ", t.sizes());
}

void check_operands(const Op& op, const Graph& graph, const Tensor& x, const Tensor& y, const Tensor& w, const Tensor& g) {
  refuse_tangents({&x, &y, &w, &g});
  TORCH_CHECK(x.is_cuda(), "CUDA is required for SO3 LunaTP.");
  check_operand(op, x, x, "x", graph.native.num_src_nodes, op.X);
  check_operand(op, x, y, "edge_attr", graph.native.num_edges, op.Y);
  check_operand(op, x, w, "weight", graph.native.num_edges, op.W);
  check_operand(op, x, g, "grad_out", graph.native.num_nodes, op.O);
}

void* stream_of(const Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.device().index()).stream(); }
void* pointer(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

Tensor scratch_for(const Op& op, const Graph& graph, const Tensor& like, int64_t* bytes) {
  *bytes = 0;
  if (!api.plan_query(op.plan, LUNA_PLAN_NEEDS_SCRATCH)) return Tensor();
  *bytes = api.scratch_bytes(op.plan, graph.native.num_nodes, graph.native.num_edges);
  return *bytes > 0 ? at::empty({*bytes}, like.options().dtype(at::kByte)) : Tensor();
}

Tensor run_forward(const Op& op, const Graph& graph, const Tensor& x_, const Tensor& y_, const Tensor& w_) {
  check_operands(op, graph, x_, y_, w_, Tensor());
  const c10::cuda::CUDAGuard guard(x_.device());
  const Tensor x = prepared(x_), y = prepared(y_), w = prepared(w_);
  Tensor out = at::empty({graph.native.num_nodes, op.O}, x.options());
  check(api.fwd(op.plan, &graph.native, x.data_ptr(), y.data_ptr(), w.data_ptr(), out.data_ptr(), stream_of(x)));
  return out;
}

enum : int { kX = 1, kY = 2, kW = 4, kG = 8 };

// The first derivatives named in `mask`; the others stay undefined.  gw, if given, is added to and becomes the third.
std::array<Tensor, 3> run_backward(const Op& op, const Graph& graph, const Tensor& x_, const Tensor& y_, const Tensor& w_,
                                   const Tensor& g_, int mask, const Tensor& gw = Tensor()) {
  std::array<Tensor, 3> out;
  if (!mask) return out;
  check_operands(op, graph, x_, y_, w_, g_);
  const c10::cuda::CUDAGuard guard(x_.device());
  const Tensor x = prepared(x_), y = prepared(y_), w = prepared(w_), g = prepared(g_);
  const Tensor* like[3] = {&x, &y, &w};
  const bool empty = graph.native.num_edges == 0 || graph.native.num_nodes == 0;
  for (int s = 0; s < 3; ++s)
    if (mask >> s & 1) out[s] = s == 2 && gw.defined() ? gw : (empty ? at::zeros_like(*like[s]) : at::empty_like(*like[s]));
  if (empty) return out;
  int64_t bytes = 0;
  const Tensor scratch = scratch_for(op, graph, x, &bytes);
  const auto entry = gw.defined() ? api.bwd_add_gw : api.bwd;
  check(entry(op.plan, &graph.native, x.data_ptr(), y.data_ptr(), w.data_ptr(), g.data_ptr(), pointer(out[0]),
                pointer(out[1]), pointer(out[2]), pointer(scratch), bytes, stream_of(x)));
  return out;
}

// The second derivatives named in `mask` (x, y, w, g) for the cotangents rx, ry, rw, each of which may be undefined.
std::array<Tensor, 4> run_double(const Op& op, const Graph& graph, const Tensor& x_, const Tensor& y_, const Tensor& w_,
                                 const Tensor& g_, const Tensor& rx_, const Tensor& ry_, const Tensor& rw_, int mask) {
  std::array<Tensor, 4> out;
  if (!mask) return out;
  refuse_tangents({&rx_, &ry_, &rw_});
  check_operands(op, graph, x_, y_, w_, g_);
  check_operand(op, x_, rx_, "rx", graph.native.num_src_nodes, op.X);
  check_operand(op, x_, ry_, "ry", graph.native.num_edges, op.Y);
  check_operand(op, x_, rw_, "rw", graph.native.num_edges, op.W);
  const c10::cuda::CUDAGuard guard(x_.device());
  const Tensor x = prepared(x_), y = prepared(y_), w = prepared(w_), g = prepared(g_), rx = prepared(rx_),
               ry = prepared(ry_), rw = prepared(rw_);
  const Tensor* like[4] = {&x, &y, &w, &g};
  const bool empty = graph.native.num_edges == 0 || graph.native.num_nodes == 0;
  for (int s = 0; s < 4; ++s)
    if (mask >> s & 1) out[s] = empty ? at::zeros_like(*like[s]) : at::empty_like(*like[s]);
  if (empty) return out;
  int64_t bytes = 0;
  const Tensor scratch = scratch_for(op, graph, x, &bytes);
  check(api.dbl_bwd(op.plan, &graph.native, x.data_ptr(), y.data_ptr(), w.data_ptr(), g.data_ptr(), pointer(rx), pointer(ry),
                    pointer(rw), pointer(out[0]), pointer(out[1]), pointer(out[2]), pointer(out[3]), pointer(scratch), bytes,
                    stream_of(x)));
  return out;
}

// ---- the autograd chain of the convolution --------------------------------------------------------------------------------
template <size_t N>
variable_list only(const std::array<Tensor, N>& tensors, int mask) {
  variable_list list;
  for (size_t s = 0; s < N; ++s)
    if (mask >> s & 1) list.push_back(tensors[s]);
  return list;
}
// The reverse: a list that holds the entries of `mask` only.
template <size_t N>
std::array<Tensor, N> spread(const variable_list& list, int mask) {
  std::array<Tensor, N> tensors;
  size_t next = 0;
  for (size_t s = 0; s < N; ++s)
    if (mask >> s & 1) tensors[s] = list[next++];
  return tensors;
}
Tensor contiguous(const Tensor& t) { return t.defined() ? t.contiguous() : t; }

// Energy training differentiates the weights once, force training twice: the gradients of both orders meet at the weights, and
// the engine adds two tensors of the weights' size, three more passes over memory beside the two that wrote them.  So the second
// order's graph names the weights through a node of its own (SecondOrderWeights), and if both that one and the first order's node,
// ConvForward, run in a task, the first order's kernel adds to the second order's gradient in place.  Which of the two comes first is
// the engine's choice unless the energy is nonlinear in the output: the second order leaves its gradient for the first, or the first
// leaves its operands for the second.  Neither node sees anything else of the other: ConvForward has one output, and runs when
// something reaches that.
// FP64 force step, degrees (2, 3, 3), 128 channels, 1.05 M edges (18 GB of weights): 33.6 -> 27.4 ms; FP32, (2, 2, 2),
// 32 channels, 0.2 M edges (295 MB): 936 -> 818 us.  Energy and forces in one loss, the energy linear in the output: FP64, 0.4 M edges
// 11.5 -> 8.9 ms; FP32, 0.2 M edges 610 -> 514 us.
//
// Not where a hook sees what one of the nodes returns, or where a graph of the gradient is wanted: there the engine adds them.
using NodePtr = std::shared_ptr<torch::autograd::Node>;

// Whether the running task runs a node, or has.
bool in_running_task(const NodePtr& node) {
  const auto* reached = torch::autograd::get_current_graph_task_nodes_in_graph();
  const auto* wanted = torch::autograd::get_current_graph_task_exec_info();
  if (!node || !reached || !wanted || reached->count(node.get()) == 0) return false;
  if (wanted->empty()) return true;
  const auto info = wanted->find(node.get());
  return info != wanted->end() && info->second.should_execute();
}

// The last tasks that something was done in.  Their numbers rise; of those before the ones kept anything may be true.
struct RecentTasks {
  std::array<int64_t, 8> tasks{-1, -1, -1, -1, -1, -1, -1, -1};
  size_t next = 0;
  int64_t forgotten = -1;
  void add(int64_t task) {
    forgotten = std::max(forgotten, tasks[next]);
    tasks[next] = task;
    next = (next + 1) % tasks.size();
  }
  bool may_have(int64_t task) const {
    return task <= forgotten || std::find(tasks.begin(), tasks.end(), task) != tasks.end();
  }
};

// Where the two nodes leave things for each other.  What a task that failed has left stays until the graph goes, and later tasks
// leave nothing.
struct WeightGradient : torch::CustomClassHolder {
  struct Operands {
    Tensor x, y, w, g;
    OpPtr op;
    GraphPtr graph;
  };

  explicit WeightGradient(const NodePtr& node) : first(node) {}
  void second_order_is(const NodePtr& node) {
    const std::lock_guard<std::mutex> lock(mutex);
    second = node;
  }

  // By the first order's node when it runs: what the second order has left for it in this task, if anything.
  Tensor first_runs() {
    const int64_t running = torch::autograd::get_current_graph_task_id();
    const std::lock_guard<std::mutex> lock(mutex);
    first_ran.add(running);
    return gradient_task == running ? std::exchange(gradient, Tensor()) : Tensor();
  }
  // Whether its operands were left for the second order's node, which runs later in this task.
  bool leave_operands(const Operands& all) {
    const std::lock_guard<std::mutex> lock(mutex);
    const NodePtr node = second.lock();
    const int64_t running = torch::autograd::get_current_graph_task_id();
    if (running < 0 || operands || second_ran.may_have(running) || !quiet(node) || !in_running_task(node)) return false;
    operands = all;
    operands_task = running;
    operands_for = node;
    return true;
  }
  // By a second order's node when it runs.
  std::optional<Operands> second_runs() {
    const int64_t running = torch::autograd::get_current_graph_task_id();
    const std::lock_guard<std::mutex> lock(mutex);
    second_ran.add(running);
    if (!operands || operands_task != running || operands_for.lock() != torch::autograd::get_current_node()) return std::nullopt;
    return std::exchange(operands, std::nullopt);
  }
  bool leave_gradient(const Tensor& w_gradient) {
    const std::lock_guard<std::mutex> lock(mutex);
    const int64_t running = torch::autograd::get_current_graph_task_id();
    const NodePtr node = first.lock();
    if (running < 0 || gradient.defined() || first_ran.may_have(running) || !quiet(node) || !in_running_task(node)) return false;
    gradient = w_gradient;
    gradient_task = running;
    return true;
  }

 private:
  // Whether no hook sees what the running node returns, nor what the other one does.
  static bool quiet(const NodePtr& other) {
    const NodePtr running = torch::autograd::get_current_node();
    return running && other && running->post_hooks().empty() && other->post_hooks().empty();
  }

  std::mutex mutex;  // tasks of several threads may run through one graph
  const std::weak_ptr<torch::autograd::Node> first;
  std::weak_ptr<torch::autograd::Node> second;  // the last one made
  std::weak_ptr<torch::autograd::Node> operands_for;
  RecentTasks first_ran, second_ran;
  Tensor gradient;
  std::optional<Operands> operands;
  int64_t gradient_task = -1, operands_task = -1;
};

// Whether nobody else can see the second order's gradient, so that a kernel may add to it.
bool only_ours(const Tensor& t) {
  return t.defined() && t.use_count() == 1 && t.has_storage() && t.storage().use_count() == 1 && !t.requires_grad() &&
         t.layout() == at::kStrided && t.is_contiguous() && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
}
// The first order's gradients, that of the weights added to the second order's if there is one.
std::array<Tensor, 3> first_on_second(const WeightGradient::Operands& all, int mask, const Tensor& second) {
  const bool ours = mask & kW && only_ours(second);
  auto d = run_backward(*all.op, *all.graph, all.x, all.y, all.w, all.g, mask, ours ? second : Tensor());
  if (second.defined() && !ours) d[2] = d[2].defined() ? d[2] + second : second;
  return d;
}

struct SecondOrderWeights : Function<SecondOrderWeights> {
  static Tensor forward(AutogradContext* ctx, const Tensor& w, const c10::intrusive_ptr<WeightGradient>& sum) {
    ctx->set_materialize_grads(false);
    keep(ctx, "sum", sum);
    return w.detach();
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    if (at::GradMode::is_enabled()) return {grads[0], Tensor()};
    const auto sum = kept<WeightGradient>(ctx, "sum");
    if (const auto operands = sum->second_runs()) return {first_on_second(*operands, kW, grads[0])[2], Tensor()};
    if (grads[0].defined() && sum->leave_gradient(grads[0])) return {Tensor(), Tensor()};
    return {grads[0], Tensor()};
  }
};

// dF/d(operand `slot`), slots 0..3 = x, y, w, g; a, b, c: the other three operands in that order.  The kernels take all four
// operands and look at the shape of the free slot's only: `free` lends it (none for g).
struct ConvPartial : Function<ConvPartial> {
  static Tensor forward(AutogradContext* ctx, const Tensor& a, const Tensor& b, const Tensor& c,
                        const std::optional<Tensor>& free, int64_t slot, const OpPtr& op, const GraphPtr& graph) {
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({a, b, c});
    ctx->saved_data["slot"] = slot;
    keep(ctx, "op", op);
    keep(ctx, "graph", graph);
    const auto all = operands({a, b, c}, slot, free ? *free : Tensor());
    if (slot == 3) return run_forward(*op, *graph, all[0], all[1], all[2]);
    return run_backward(*op, *graph, all[0], all[1], all[2], all[3], 1 << slot)[slot];
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    variable_list out(7);
    if (!grads[0].defined()) return out;
    const auto saved = ctx->get_saved_variables();
    const int64_t slot = ctx->saved_data["slot"].toInt();
    const auto op = kept<Op>(ctx, "op");
    const auto graph = kept<Graph>(ctx, "graph");
    // <r, dF/ds(a, b, c)> = F with r in slot s: the gradient of another operand is its partial at the rest
    const auto full = operands({saved[0], saved[1], saved[2]}, slot, grads[0].contiguous());
    for (int64_t other = 0, position = 0; other < 4; ++other) {
      if (other == slot) continue;
      if (ctx->needs_input_grad(position)) out[position] = of(full, other, op, graph);
      ++position;
    }
    return out;
  }
  static std::array<Tensor, 4> operands(const std::array<Tensor, 3>& others, int64_t slot, const Tensor& free) {
    std::array<Tensor, 4> full;
    for (int64_t s = 0, next = 0; s < 4; ++s) full[s] = s == slot ? free : others[next++];
    return full;
  }
  static Tensor of(const std::array<Tensor, 4>& full, int64_t slot, const OpPtr& op, const GraphPtr& graph) {
    std::array<Tensor, 3> others;
    for (int64_t s = 0, next = 0; s < 4; ++s)
      if (s != slot) others[next++] = full[s];
    // without history: nothing depends on its values
    const std::optional<Tensor> free = slot == 3 ? std::nullopt : std::optional<Tensor>(full[slot].detach());
    return apply(others[0], others[1], others[2], free, slot, op, graph);
  }
};

struct ConvDouble : Function<ConvDouble> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& y, const Tensor& w, const Tensor& g,
                               const std::optional<Tensor>& rx, const std::optional<Tensor>& ry,
                               const std::optional<Tensor>& rw, int64_t mask, const OpPtr& op, const GraphPtr& graph) {
    const Tensor none;
    const Tensor &tx = rx ? *rx : none, &ty = ry ? *ry : none, &tw = rw ? *rw : none;
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({x, y, w, g, tx, ty, tw});
    ctx->saved_data["mask"] = mask;
    keep(ctx, "op", op);
    keep(ctx, "graph", graph);
    return only(run_double(*op, *graph, x, y, w, g, tx, ty, tw, static_cast<int>(mask)), static_cast<int>(mask));
  }
  // The outputs contracted with their cotangents b are a sum of F with three of its operands replaced; the gradient of
  // a tensor is the sum of the partials over the terms it appears in.
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    variable_list out(10);
    const auto saved = ctx->get_saved_variables();
    const auto op = kept<Op>(ctx, "op");
    const auto graph = kept<Graph>(ctx, "graph");
    const auto b = spread<4>(grads, static_cast<int>(ctx->saved_data["mask"].toInt()));
    // tensors by number: 0..6 = x, y, w, g, rx, ry, rw (saved), 7..10 = bx, by, bw, bg
    std::array<Tensor, 11> t;
    for (int s = 0; s < 7; ++s) t[s] = saved[s];
    for (int s = 0; s < 4; ++s) t[7 + s] = contiguous(b[s]);
    static constexpr int terms[9][4] = {{7, 5, 2, 3}, {7, 1, 6, 3}, {4, 8, 2, 3}, {0, 8, 6, 3}, {4, 1, 9, 3},
                                        {0, 5, 9, 3}, {4, 1, 2, 10}, {0, 5, 2, 10}, {0, 1, 6, 10}};
    for (int v = 0, edge = 0; v < 7; ++v) {
      if (!t[v].defined()) continue;  // a missing tangent has no edge
      if (!ctx->needs_input_grad(edge++)) continue;
      Tensor sum;
      for (const auto& term : terms) {
        bool whole = true;
        int slot = -1;
        for (int s = 0; s < 4; ++s) {
          whole = whole && t[term[s]].defined();
          if (term[s] == v) slot = s;
        }
        if (!whole || slot < 0) continue;
        const Tensor part = ConvPartial::of({t[term[0]], t[term[1]], t[term[2]], t[term[3]]}, slot, op, graph);
        sum = sum.defined() ? sum + part : part;
      }
      out[v] = sum;
    }
    return out;
  }
};

struct ConvBackward : Function<ConvBackward> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& y, const Tensor& w, const Tensor& g,
                               int64_t mask, const OpPtr& op, const GraphPtr& graph) {
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({x, y, w, g});
    ctx->saved_data["mask"] = mask;
    keep(ctx, "op", op);
    keep(ctx, "graph", graph);
    return only(run_backward(*op, *graph, x, y, w, g, static_cast<int>(mask)), static_cast<int>(mask));
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    variable_list out(7);
    const auto r = spread<3>(grads, static_cast<int>(ctx->saved_data["mask"].toInt()));
    if (!r[0].defined() && !r[1].defined() && !r[2].defined()) return out;
    int mask = 0;
    for (int s = 0; s < 4; ++s) mask |= ctx->needs_input_grad(s) ? 1 << s : 0;
    if (!mask) return out;
    const auto saved = ctx->get_saved_variables();
    const auto op = kept<Op>(ctx, "op");
    const auto graph = kept<Graph>(ctx, "graph");
    std::array<Tensor, 4> h;
    if (at::GradMode::is_enabled()) {
      auto optional = [](const Tensor& t) { return t.defined() ? std::optional<Tensor>(t.contiguous()) : std::nullopt; };
      h = spread<4>(ConvDouble::apply(saved[0], saved[1], saved[2], saved[3], optional(r[0]), optional(r[1]),
                                      optional(r[2]), static_cast<int64_t>(mask), op, graph),
                    mask);
    } else {
      h = run_double(*op, *graph, saved[0], saved[1], saved[2], saved[3], r[0], r[1], r[2], mask);
    }
    for (int s = 0; s < 4; ++s) out[s] = h[s];
    return out;
  }
};

// Below this size of the weights the engine's sum, 15 us for 32 MiB, is not worth a node.
constexpr int64_t kSecondOrderBytes = 32 << 20;

struct ConvForward : Function<ConvForward> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& y, const Tensor& w, const OpPtr& op,
                        const GraphPtr& graph) {
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({x, y, w});
    keep(ctx, "op", op);
    keep(ctx, "graph", graph);
    return run_forward(*op, *graph, x, y, w);
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    variable_list out(5);
    auto sum = ctx->saved_data.count("sum") ? kept<WeightGradient>(ctx, "sum") : c10::intrusive_ptr<WeightGradient>();
    const Tensor second = sum ? sum->first_runs() : Tensor();
    int mask = 0;
    for (int s = 0; s < 3; ++s) mask |= ctx->needs_input_grad(s) ? 1 << s : 0;
    if (!grads[0].defined() || !mask) {
      out[2] = second;
      return out;
    }
    const auto saved = ctx->get_saved_variables();
    const auto op = kept<Op>(ctx, "op");
    const auto graph = kept<Graph>(ctx, "graph");
    const Tensor g = grads[0].contiguous();
    std::array<Tensor, 3> d;
    if (at::GradMode::is_enabled()) {
      Tensor w = saved[2];
      if (w.requires_grad() && static_cast<int64_t>(w.nbytes()) >= kSecondOrderBytes) {
        if (!sum) {
          sum = c10::make_intrusive<WeightGradient>(torch::autograd::get_current_node());
          keep(ctx, "sum", sum);
        }
        w = SecondOrderWeights::apply(w, sum);
        sum->second_order_is(w.grad_fn());
      }
      d = spread<3>(ConvBackward::apply(saved[0], saved[1], w, g, static_cast<int64_t>(mask), op, graph), mask);
    } else {
      const WeightGradient::Operands all{saved[0], saved[1], saved[2], g, op, graph};
      if (sum && mask & kW && !second.defined() && sum->leave_operands(all)) mask &= ~kW;
      d = first_on_second(all, mask, second);
    }
    for (int s = 0; s < 3; ++s) out[s] = d[s];
    return out;
  }
};

bool tracked(std::initializer_list<const Tensor*> tensors) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor* t : tensors)
    if (t->requires_grad()) return true;
  return false;
}

Tensor conv(const OpPtr& op, const GraphPtr& graph, const Tensor& x, const Tensor& y, const Tensor& w) {
  pybind11::gil_scoped_release release;
  return tracked({&x, &y, &w}) ? ConvForward::apply(x, y, w, op, graph) : run_forward(*op, *graph, x, y, w);
}

// ---- graph tables ---------------------------------------------------------------------------------------------------------
// Every table of a graph with nodes and edges: src, dst, dst_rowptr, src_rowptr, edge_ids_by_src, edge_ids_by_dst,
// node_order, source_node_order, node_tiers and the five of the segments; nothing if an index is out of range or dst is
// not ascending.  src, dst: contiguous, int32 or int64, on one CUDA device, of one length.
std::vector<Tensor> graph_tables(const Tensor& src, const Tensor& dst, int64_t nodes, int64_t source_rows) {
  pybind11::gil_scoped_release release;
  const c10::cuda::CUDAGuard guard(src.device());
  const int64_t edges = src.numel();
  const auto options = src.options().dtype(at::kInt);
  auto table = [&](int64_t entries) { return at::empty({entries}, options); };
  const int64_t room = source_rows + edges / 32;  // a segment per row at least, and one per 32 edges at most beyond that
  Tensor by_src = table(edges), by_dst = table(edges), src_out = table(edges), dst_out = table(edges);
  Tensor dst_rowptr = table(nodes + 1), src_rowptr = table(source_rows + 1), order = table(nodes);
  Tensor source_order = table(source_rows), tiers = table(3), seg_rowptr = table(source_rows + 1);
  Tensor seg_nodes = table(room), seg_begin = table(room), seg_end = table(room), seg_order = table(room);
  const int64_t bytes = api.graph_scratch_bytes(std::max(nodes, source_rows), edges);
  const Tensor scratch = at::empty({bytes}, options.dtype(at::kByte));
  auto ints = [](const Tensor& t) { return t.data_ptr<int32_t>(); };
  const luna_graph_out out{ints(src_out), ints(dst_out), ints(dst_rowptr), ints(src_rowptr),
                           ints(by_src),  ints(order),   ints(source_order)};
  const luna_graph_pieces pieces{ints(by_dst),  ints(tiers),      ints(seg_nodes), ints(seg_begin),
                                 ints(seg_end), ints(seg_rowptr), ints(seg_order)};
  int bad = 0;
  int64_t segments = 0;
  check(api.graph_build_all(src.data_ptr(), dst.data_ptr(), src.scalar_type() == at::kLong ? 64 : 32, nodes, source_rows,
                            edges, &out, &pieces, &bad, &segments, scratch.data_ptr(), bytes, stream_of(src)));
  if (bad) return {};
  auto cut = [&](const Tensor& t) { return t.narrow(0, 0, segments); };
  return {src_out, dst_out, dst_rowptr, src_rowptr, by_src, by_dst, order, source_order, tiers,
          cut(seg_nodes), cut(seg_begin), cut(seg_end), seg_rowptr, cut(seg_order)};
}

// ---- spherical harmonics --------------------------------------------------------------------------------------------------
struct Harmonics : torch::CustomClassHolder {
  luna_sh_desc desc{};
  int64_t columns;
  bool constant;
  Harmonics(const std::vector<int64_t>& degrees, bool normalize, int64_t normalization, int64_t out_dim, bool f64)
      : columns(out_dim), constant(true) {
    TORCH_CHECK_NOT_IMPLEMENTED(degrees.size() <= 32, "at most 32 degree entries are supported");
    desc.dtype = f64 ? LUNA_F64 : LUNA_F32;
    desc.num_degrees = static_cast<int32_t>(degrees.size());
    for (size_t i = 0; i < degrees.size(); ++i) {
      desc.degrees[i] = static_cast<int32_t>(degrees[i]);
      constant = constant && degrees[i] == 0;
    }
    desc.normalize = normalize;
    desc.normalization = static_cast<int32_t>(normalization);
  }
};
using HarmonicsPtr = c10::intrusive_ptr<Harmonics>;

Tensor rows_of(const Tensor& t) { return t.reshape({-1, t.size(-1)}).contiguous(); }

void check_vectors(const Harmonics& h, const Tensor& v) {
  TORCH_CHECK(v.is_cuda(), "CUDA is required for spherical harmonics in this library");
  TORCH_CHECK_TYPE(v.scalar_type() == (h.desc.dtype == LUNA_F64 ? at::kDouble : at::kFloat),
                   "spherical harmonics require float32 or float64 input");
  TORCH_CHECK_VALUE(v.dim() > 0 && v.size(-1) == 3, "SphericalHarmonics input must have shape (...,3)");
}

Tensor sh_forward(const Harmonics& h, const Tensor& v) {
  if (!h.constant) refuse_tangents({&v});  // the values of degree 0 alone have no derivative
  check_vectors(h, v);
  const c10::cuda::CUDAGuard guard(v.device());
  const Tensor flat = rows_of(v);
  auto shape = v.sizes().vec();
  shape.back() = h.columns;
  Tensor out = at::empty(shape, v.options());
  check(api.sh_fwd(&h.desc, flat.data_ptr(), out.data_ptr(), flat.size(0), stream_of(v)));
  return out;
}

Tensor sh_backward(const Harmonics& h, const Tensor& v, const Tensor& g) {
  refuse_tangents({&v, &g});
  check_vectors(h, v);
  const c10::cuda::CUDAGuard guard(v.device());
  const Tensor flat = rows_of(v), cotangents = rows_of(g);
  Tensor dv = at::empty(v.sizes(), v.options());
  check(api.sh_bwd(&h.desc, flat.data_ptr(), cotangents.data_ptr(), dv.data_ptr(), flat.size(0), stream_of(v)));
  return dv;
}

std::array<Tensor, 2> sh_double(const Harmonics& h, const Tensor& v, const Tensor& g, const Tensor& r, int mask) {
  refuse_tangents({&v, &g, &r});
  check_vectors(h, v);
  const c10::cuda::CUDAGuard guard(v.device());
  const Tensor flat = rows_of(v), cotangents = rows_of(g), tangents = rows_of(r);
  std::array<Tensor, 2> out;
  if (mask & 1) out[0] = at::empty(v.sizes(), v.options());
  if (mask & 2) out[1] = at::empty(g.sizes(), g.options());
  check(api.sh_dbl_bwd(&h.desc, flat.data_ptr(), cotangents.data_ptr(), tangents.data_ptr(), pointer(out[0]),
                       pointer(out[1]), flat.size(0), stream_of(v)));
  return out;
}

struct ShDouble : Function<ShDouble> {
  static variable_list forward(AutogradContext* ctx, const Tensor& v, const Tensor& g, const Tensor& r,
                               const HarmonicsPtr& h) {
    ctx->set_materialize_grads(false);
    return only(sh_double(*h, v, g, r, 3), 3);
  }
  static variable_list backward(AutogradContext*, const variable_list& grads) {
    TORCH_CHECK_NOT_IMPLEMENTED(!grads[0].defined() && !grads[1].defined(),
                                "third-order derivatives of the spherical harmonics are not provided");
    return variable_list(4);
  }
};

struct ShBackward : Function<ShBackward> {
  static Tensor forward(AutogradContext* ctx, const Tensor& v, const Tensor& g, const HarmonicsPtr& h) {
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({v, g});
    keep(ctx, "op", h);
    return sh_backward(*h, v, g);
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    variable_list out(3);
    if (!grads[0].defined()) return out;
    const auto saved = ctx->get_saved_variables();
    const auto h = kept<Harmonics>(ctx, "op");
    const int mask = (ctx->needs_input_grad(0) ? 1 : 0) | (ctx->needs_input_grad(1) ? 2 : 0);
    if (!mask) return out;
    if (at::GradMode::is_enabled()) {
      const auto d = ShDouble::apply(saved[0], saved[1], grads[0], h);
      if (mask & 1) out[0] = d[0];
      if (mask & 2) out[1] = d[1];
    } else {
      const auto d = sh_double(*h, saved[0], saved[1], grads[0], mask);
      out[0] = d[0];
      out[1] = d[1];
    }
    return out;
  }
};

struct ShForward : Function<ShForward> {
  static Tensor forward(AutogradContext* ctx, const Tensor& v, const HarmonicsPtr& h) {
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({v});
    keep(ctx, "op", h);
    return sh_forward(*h, v);
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    variable_list out(2);
    const auto h = kept<Harmonics>(ctx, "op");
    if (!grads[0].defined() || h->constant || !ctx->needs_input_grad(0)) return out;
    const auto saved = ctx->get_saved_variables();
    out[0] = at::GradMode::is_enabled() ? ShBackward::apply(saved[0], grads[0], h) : sh_backward(*h, saved[0], grads[0]);
    return out;
  }
};

Tensor harmonics(const HarmonicsPtr& h, const Tensor& v) {
  pybind11::gil_scoped_release release;
  return !h->constant && tracked({&v}) ? ShForward::apply(v, h) : sh_forward(*h, v);
}

// ---- operators over rows: what they share ------------------------------------------------------------------------------------
using Maybe = std::optional<Tensor>;
const Tensor& of(const Maybe& t) {
  static const Tensor none;
  return t ? *t : none;
}
Maybe maybe(const Tensor& t) { return t.defined() ? Maybe(t) : std::nullopt; }

int row_dtype(const Tensor& t, const char* what) {
  switch (t.scalar_type()) {
    case at::kFloat: return LUNA_F32;
    case at::kDouble: return LUNA_F64;
    case at::kBFloat16: return LUNA_BF16;
    case at::kHalf: return LUNA_F16;
    default: break;
  }
  TORCH_CHECK_TYPE(false, what, " requires float32, float64, bfloat16 or float16, got ", t.scalar_type());
  return -1;
}
// `t` is an operand beside `x`: of its type unless another is named, on its device, of this shape.
void check_beside(const Tensor& x, const Tensor& t, const char* name, at::IntArrayRef shape, std::optional<at::ScalarType> type = {}) {
  if (!t.defined()) return;
  TORCH_CHECK_TYPE(t.scalar_type() == type.value_or(x.scalar_type()), name, " must be ", type.value_or(x.scalar_type()), ", got ",
                   t.scalar_type());
  TORCH_CHECK_VALUE(t.device() == x.device(), name, " must be on ", x.device(), ", got ", t.device());
  TORCH_CHECK_VALUE(t.sizes() == shape, name, " must have shape ", shape, ", got ", t.sizes());
}
Tensor scratch_of(int64_t bytes, const Tensor& like) {
  if (bytes < 0) check(static_cast<int>(bytes));
  return bytes > 0 ? at::empty({bytes}, like.options().dtype(at::kByte)) : Tensor();
}
int64_t bytes_of(const Tensor& t) { return t.defined() ? t.numel() : 0; }

// ---- layer norm ----------------------------------------------------------------------------------------------------------------
struct Norm : torch::CustomClassHolder {
  static constexpr int64_t kMostElements = 16384;  // of a block
  luna_norm_desc desc{};                           // the type comes with each call
  int64_t dim = 0, weights = 0, biases = 0;
  Norm(const std::vector<std::array<int64_t, 3>>& blocks, int64_t normalization, double eps) {
    TORCH_CHECK_NOT_IMPLEMENTED(blocks.size() <= 32, "layer norm of more than 32 blocks");
    desc.num_blocks = static_cast<int32_t>(blocks.size());
    desc.normalization = static_cast<int32_t>(normalization);
    desc.eps = eps;
    for (size_t i = 0; i < blocks.size(); ++i) {
      const auto& [mul, components, scalar] = blocks[i];
      TORCH_CHECK_NOT_IMPLEMENTED(mul <= kMostElements && components <= kMostElements, "layer norm of a block with more than ", kMostElements,
                                  " elements");  // also beyond what the description holds
      desc.mul[i] = static_cast<int32_t>(mul);
      desc.components[i] = static_cast<int32_t>(components);
      desc.scalar[i] = static_cast<int32_t>(scalar);
      dim += mul * components;
      weights += mul;
      biases += scalar ? mul : 0;
    }
  }
  luna_norm_desc as(const Tensor& x) const {
    luna_norm_desc d = desc;
    d.dtype = row_dtype(x, "layer norm");
    return d;
  }
};
using NormPtr = c10::intrusive_ptr<Norm>;

Tensor norm_rows(const Tensor& t, const Norm& n) { return t.defined() ? t.reshape({-1, n.dim}).contiguous() : t; }

luna_norm_desc check_norm(const Norm& n, const Tensor& x, const Tensor& weight, const Tensor& bias) {
  refuse_tangents({&x, &weight, &bias});
  TORCH_CHECK(x.is_cuda(), "CUDA is required for layer norm in this library");
  const luna_norm_desc desc = n.as(x);
  TORCH_CHECK_VALUE(x.dim() > 0 && x.size(-1) == n.dim, "layer norm input must have shape (..., ", n.dim, "), got ", x.sizes());
  check_beside(x, weight, "weight", {n.weights});
  check_beside(x, bias, "bias", {n.biases});
  return desc;
}

// The statistics as a forward leaves them: the launches follow them by the sizes of x.
Tensor check_stats(const Norm& n, const Tensor& x, const Tensor& stats) {
  TORCH_CHECK_VALUE(stats.defined(), "layer norm needs the forward's statistics");
  check_beside(x, stats, "stats", {n.desc.num_blocks, x.numel() / n.dim, 2}, x.scalar_type() == at::kDouble ? at::kDouble : at::kFloat);
  return prepared(stats);
}

std::array<Tensor, 2> norm_forward(const Norm& n, const Tensor& x, const Tensor& weight, const Tensor& bias, bool keep_stats) {
  const luna_norm_desc desc = check_norm(n, x, weight, bias);
  const c10::cuda::CUDAGuard guard(x.device());
  const Tensor rows = norm_rows(x, n), w = contiguous(weight), b = contiguous(bias);
  Tensor y = at::empty(x.sizes(), rows.options()), stats;
  if (keep_stats)
    stats = at::empty({desc.num_blocks, rows.size(0), 2}, rows.options().dtype(x.scalar_type() == at::kDouble ? at::kDouble : at::kFloat));
  check(api.norm_fwd(&desc, rows.data_ptr(), pointer(w), pointer(b), y.data_ptr(), pointer(stats), rows.size(0), stream_of(x)));
  return {y, stats};
}

// The gradients of x, weight and bias named in `mask`.
std::array<Tensor, 3> norm_backward(const Norm& n, const Tensor& x, const Tensor& weight, const Tensor& stats, const Tensor& g, int mask) {
  std::array<Tensor, 3> out;
  if (!mask) return out;
  const luna_norm_desc desc = check_norm(n, x, weight, Tensor());
  refuse_tangents({&g});
  check_beside(x, g, "grad_out", x.sizes());
  const c10::cuda::CUDAGuard guard(x.device());
  const Tensor rows = norm_rows(x, n), w = contiguous(weight), cotangents = norm_rows(g, n), moments = check_stats(n, x, stats);
  if (mask & 1) out[0] = at::empty(x.sizes(), rows.options());
  if (mask & 2) out[1] = at::empty({n.weights}, rows.options());
  if (mask & 4) out[2] = at::empty({n.biases}, rows.options());
  const Tensor scratch = mask & 6 ? scratch_of(api.norm_scratch_bytes(&desc, rows.size(0)), x) : Tensor();
  check(api.norm_bwd(&desc, rows.data_ptr(), pointer(w), moments.data_ptr(), cotangents.data_ptr(), pointer(out[0]), pointer(out[1]),
                     n.biases ? pointer(out[2]) : nullptr, pointer(scratch), bytes_of(scratch), rows.size(0), stream_of(x)));
  return out;
}

// The second derivatives of x, weight and g named in `mask`, for the cotangents of the three gradients.
std::array<Tensor, 3> norm_double(const Norm& n, const Tensor& x, const Tensor& weight, const Tensor& stats, const Tensor& g,
                                  const Tensor& rx, const Tensor& rw, const Tensor& rb, int mask) {
  std::array<Tensor, 3> out;
  if (!mask) return out;
  const luna_norm_desc desc = check_norm(n, x, weight, Tensor());
  refuse_tangents({&g, &rx, &rw, &rb});
  check_beside(x, g, "grad_out", x.sizes());
  check_beside(x, rx, "rx", x.sizes());
  check_beside(x, rw, "rw", {n.weights});
  check_beside(x, rb, "rb", {n.biases});
  const c10::cuda::CUDAGuard guard(x.device());
  const Tensor rows = norm_rows(x, n), w = contiguous(weight), cotangents = norm_rows(g, n), tx = norm_rows(rx, n), tw = contiguous(rw),
               tb = contiguous(rb), moments = check_stats(n, x, stats);
  if (mask & 1) out[0] = at::empty(x.sizes(), rows.options());
  if (mask & 2) out[1] = at::empty({n.weights}, rows.options());
  if (mask & 4) out[2] = at::empty(x.sizes(), rows.options());
  const Tensor scratch = mask & 2 ? scratch_of(api.norm_scratch_bytes(&desc, rows.size(0)), x) : Tensor();
  check(api.norm_dbl_bwd(&desc, rows.data_ptr(), pointer(w), moments.data_ptr(), cotangents.data_ptr(), pointer(tx), pointer(tw),
                         n.biases ? pointer(tb) : nullptr, pointer(out[0]), pointer(out[1]), pointer(out[2]), pointer(scratch),
                         bytes_of(scratch), rows.size(0), stream_of(x)));
  return out;
}

// Which of these tensors' gradients the running task wants: an edge belongs to each tensor that is there.
int wanted(AutogradContext* ctx, std::initializer_list<const Tensor*> tensors) {
  int mask = 0, bit = 0, edge = 0;
  for (const Tensor* t : tensors) {
    if (t->defined() && ctx->needs_input_grad(edge++)) mask |= 1 << bit;
    ++bit;
  }
  return mask;
}

struct NormDouble : Function<NormDouble> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Maybe& weight, const Tensor& g, const Tensor& stats,
                               const Maybe& rx, const Maybe& rw, const Maybe& rb, int64_t mask, const NormPtr& n) {
    ctx->set_materialize_grads(false);
    return only(norm_double(*n, x, of(weight), stats, g, of(rx), of(rw), of(rb), static_cast<int>(mask)), static_cast<int>(mask));
  }
  static variable_list backward(AutogradContext*, const variable_list& grads) {
    for (const Tensor& t : grads)
      TORCH_CHECK_NOT_IMPLEMENTED(!t.defined(), "third-order derivatives of the layer norm are not provided");
    return variable_list(9);
  }
};

struct NormBackward : Function<NormBackward> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Maybe& weight, const Tensor& g, const Tensor& stats,
                               int64_t mask, const NormPtr& n) {
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({x, of(weight), g, stats});
    ctx->saved_data["mask"] = mask;
    keep(ctx, "norm", n);
    return only(norm_backward(*n, x, of(weight), stats, g, static_cast<int>(mask)), static_cast<int>(mask));
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    variable_list out(6);
    const auto r = spread<3>(grads, static_cast<int>(ctx->saved_data["mask"].toInt()));
    if (!r[0].defined() && !r[1].defined() && !r[2].defined()) return out;
    const auto saved = ctx->get_saved_variables();
    const int mask = wanted(ctx, {&saved[0], &saved[1], &saved[2]});
    if (!mask) return out;
    const auto n = kept<Norm>(ctx, "norm");
    const auto h = at::GradMode::is_enabled()
                       ? spread<3>(NormDouble::apply(saved[0], maybe(saved[1]), saved[2], saved[3], maybe(r[0]), maybe(r[1]), maybe(r[2]),
                                                     static_cast<int64_t>(mask), n), mask)
                       : norm_double(*n, saved[0], saved[1], saved[3], saved[2], r[0], r[1], r[2], mask);
    for (int s = 0; s < 3; ++s) out[s] = h[s];
    return out;
  }
};

struct NormForward : Function<NormForward> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Maybe& weight, const Maybe& bias, const NormPtr& n) {
    const auto found = norm_forward(*n, x, of(weight), of(bias), true);
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({x, of(weight), found[1]});
    ctx->saved_data["bias"] = bias.has_value();
    keep(ctx, "norm", n);
    return found[0];
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    variable_list out(4);
    if (!grads[0].defined()) return out;
    const auto saved = ctx->get_saved_variables();
    const auto n = kept<Norm>(ctx, "norm");
    int mask = wanted(ctx, {&saved[0], &saved[1]});
    if (ctx->saved_data["bias"].toBool() && ctx->needs_input_grad(saved[1].defined() ? 2 : 1)) mask |= 4;
    if (!mask) return out;
    const auto d = at::GradMode::is_enabled()
                       ? spread<3>(NormBackward::apply(saved[0], maybe(saved[1]), grads[0], saved[2], static_cast<int64_t>(mask), n), mask)
                       : norm_backward(*n, saved[0], saved[1], saved[2], grads[0], mask);
    for (int s = 0; s < 3; ++s) out[s] = d[s];
    return out;
  }
};

Tensor layer_norm(const NormPtr& n, const Tensor& x, const Maybe& weight, const Maybe& bias) {
  pybind11::gil_scoped_release release;
  return tracked({&x, &of(weight), &of(bias)}) ? NormForward::apply(x, weight, bias, n)
                                               : norm_forward(*n, x, of(weight), of(bias), false)[0];
}

// ---- bias by buckets -------------------------------------------------------------------------------------------------------------
Tensor distance_buckets(const Tensor& v, const Tensor& boundaries) {
  pybind11::gil_scoped_release release;
  TORCH_CHECK(v.is_cuda(), "CUDA is required for distance buckets in this library");
  TORCH_CHECK_TYPE(v.scalar_type() == at::kFloat || v.scalar_type() == at::kDouble, "distance buckets require float32 or float64 vectors, got ",
                   v.scalar_type());
  TORCH_CHECK_VALUE(v.dim() > 0 && v.size(-1) == 3, "distance buckets require vectors of shape (...,3), got ", v.sizes());
  TORCH_CHECK_VALUE(boundaries.dim() == 1, "boundaries must be one-dimensional, got ", boundaries.sizes());
  check_beside(v, boundaries, "boundaries", boundaries.sizes());
  const c10::cuda::CUDAGuard guard(v.device());
  const Tensor flat = rows_of(v), borders = boundaries.contiguous();
  Tensor out = at::empty(v.sizes().slice(0, v.dim() - 1), v.options().dtype(at::kInt));
  check(api.distance_buckets(v.scalar_type() == at::kDouble ? LUNA_F64 : LUNA_F32, flat.data_ptr(), borders.data_ptr(), borders.numel(),
                             out.data_ptr<int32_t>(), flat.size(0), stream_of(v)));
  return out;
}

void check_buckets(const Tensor& beside, const Tensor& buckets) {
  TORCH_CHECK(beside.is_cuda(), "CUDA is required for the relative bias in this library");
  TORCH_CHECK_TYPE(buckets.scalar_type() == at::kInt, "buckets must be Int, got ", buckets.scalar_type());
  TORCH_CHECK_VALUE(buckets.device() == beside.device(), "buckets must be on ", beside.device(), ", got ", buckets.device());
}

Tensor bias_forward(const Tensor& table, const Tensor& buckets) {
  refuse_tangents({&table});
  check_buckets(table, buckets);
  const int dtype = row_dtype(table, "relative bias");
  TORCH_CHECK_VALUE(table.dim() == 2 && table.size(0) > 0 && table.size(1) > 0, "the bias table must have shape (buckets, heads), got ",
                    table.sizes());
  const c10::cuda::CUDAGuard guard(table.device());
  const Tensor t = table.contiguous(), b = buckets.contiguous();
  auto shape = buckets.sizes().vec();
  shape.push_back(table.size(1));
  Tensor out = at::empty(shape, table.options());
  check(api.bias_fwd(dtype, t.data_ptr(), b.data_ptr<int32_t>(), out.data_ptr(), b.numel(), t.size(0), t.size(1), stream_of(t)));
  return out;
}

Tensor bias_backward(const Tensor& g, const Tensor& buckets, int64_t num_buckets) {
  refuse_tangents({&g});
  check_buckets(g, buckets);
  const int dtype = row_dtype(g, "relative bias");
  TORCH_CHECK_VALUE(g.dim() == buckets.dim() + 1 && g.sizes().slice(0, buckets.dim()) == buckets.sizes() && g.size(-1) > 0,
                    "the gradient of a bias must have shape (*buckets, heads), got ", g.sizes());
  const c10::cuda::CUDAGuard guard(g.device());
  const Tensor e = g.contiguous(), b = buckets.contiguous();
  Tensor out = at::empty({num_buckets, g.size(-1)}, g.options());
  const Tensor scratch = scratch_of(api.bias_scratch_bytes(dtype, b.numel(), num_buckets, g.size(-1)), g);
  check(api.bias_bwd(dtype, e.data_ptr(), b.data_ptr<int32_t>(), out.data_ptr(), pointer(scratch), bytes_of(scratch), b.numel(), num_buckets,
                     g.size(-1), stream_of(g)));
  return out;
}

// Linear, and each the other's derivative: every order is there.
struct BiasBackward;
struct BiasForward : Function<BiasForward> {
  static Tensor forward(AutogradContext* ctx, const Tensor& table, const Tensor& buckets);
  static variable_list backward(AutogradContext* ctx, const variable_list& grads);
};
struct BiasBackward : Function<BiasBackward> {
  static Tensor forward(AutogradContext* ctx, const Tensor& g, const Tensor& buckets, int64_t num_buckets);
  static variable_list backward(AutogradContext* ctx, const variable_list& grads);
};
Tensor BiasForward::forward(AutogradContext* ctx, const Tensor& table, const Tensor& buckets) {
  ctx->set_materialize_grads(false);
  ctx->save_for_backward({buckets});
  ctx->saved_data["buckets"] = table.dim() ? table.size(0) : 0;
  return bias_forward(table, buckets);
}
variable_list BiasForward::backward(AutogradContext* ctx, const variable_list& grads) {
  if (!grads[0].defined()) return variable_list(2);
  const Tensor buckets = ctx->get_saved_variables()[0];
  const int64_t count = ctx->saved_data["buckets"].toInt();
  return {tracked({&grads[0]}) ? BiasBackward::apply(grads[0], buckets, count) : bias_backward(grads[0], buckets, count), Tensor()};
}
Tensor BiasBackward::forward(AutogradContext* ctx, const Tensor& g, const Tensor& buckets, int64_t num_buckets) {
  ctx->set_materialize_grads(false);
  ctx->save_for_backward({buckets});
  return bias_backward(g, buckets, num_buckets);
}
variable_list BiasBackward::backward(AutogradContext* ctx, const variable_list& grads) {
  if (!grads[0].defined()) return variable_list(3);
  const Tensor buckets = ctx->get_saved_variables()[0];
  return {tracked({&grads[0]}) ? BiasForward::apply(grads[0], buckets) : bias_forward(grads[0], buckets), Tensor(), Tensor()};
}

Tensor relative_bias(const Tensor& table, const Tensor& buckets) {
  pybind11::gil_scoped_release release;
  return tracked({&table}) ? BiasForward::apply(table, buckets) : bias_forward(table, buckets);
}

// ---- softmax over in-edges ----------------------------------------------------------------------------------------------------------
struct Rows : torch::CustomClassHolder {
  std::array<Tensor, 5> tables;  // rowptr, and of the pieces of cut rows: those of the rows, their rows, their nodes, the nodes' first ones
  luna_row_table native{};
  Rows(const Tensor& rowptr, int64_t edges, const Maybe& piece_of_row, const Maybe& row_of_piece, const Maybe& cut_of_piece,
       const Maybe& cut_first)
      : tables{rowptr, of(piece_of_row), of(row_of_piece), of(cut_of_piece), of(cut_first)} {
    for (const Tensor& t : tables)
      TORCH_CHECK_VALUE(!t.defined() || (t.dim() == 1 && t.is_contiguous()), "tables of rows must be one-dimensional and contiguous, got ", t.sizes());
    TORCH_CHECK_VALUE(rowptr.numel() > 0, "row pointers must not be empty");
    native.num_rows = rowptr.numel() - 1;
    native.num_edges = edges;
    native.rowptr = rowptr.data_ptr<int32_t>();
    if (!piece_of_row) return;
    native.num_pieces = row_of_piece->numel();
    native.num_cut = cut_first->numel() - 1;
    native.piece_of_row = piece_of_row->data_ptr<int32_t>();
    native.row_of_piece = row_of_piece->data_ptr<int32_t>();
    native.cut_of_piece = cut_of_piece->data_ptr<int32_t>();
    native.cut_first = cut_first->data_ptr<int32_t>();
  }
};
using RowsPtr = c10::intrusive_ptr<Rows>;

int check_softmax(const Rows& rows, const Tensor& x, const char* name) {
  refuse_tangents({&x});
  TORCH_CHECK(x.is_cuda(), "CUDA is required for the softmax over in-edges in this library");
  const int dtype = row_dtype(x, "the softmax over in-edges");
  TORCH_CHECK_VALUE((x.dim() == 1 || x.dim() == 2) && x.size(0) == rows.native.num_edges && (x.dim() == 1 || x.size(1) > 0), name,
                    " must have shape (", rows.native.num_edges, ") or (", rows.native.num_edges, ", heads), got ", x.sizes());
  TORCH_CHECK_VALUE(rows.tables[0].device() == x.device() || !rows.native.num_edges, "logits and graph must share one CUDA device");
  return dtype;
}
int64_t heads_of(const Tensor& x) { return x.dim() == 2 ? x.size(1) : 1; }
void check_table(const Tensor& x, const Tensor& table, const Tensor& buckets) {
  if (table.defined())
    TORCH_CHECK_VALUE(table.dim() == 2 && table.size(0) > 0, "the bias table must have shape (buckets, heads), got ", table.sizes());
  check_beside(x, table, "table", {table.defined() ? table.size(0) : 0, heads_of(x)});
  check_beside(x, buckets, "buckets", {x.size(0)}, at::kInt);
}

bool narrow(at::ScalarType t) { return t == at::kBFloat16 || t == at::kHalf; }
bool narrow(const Tensor& t) { return narrow(t.scalar_type()); }

// alpha, and what the backward makes gradients of: alpha itself, or for the 16-bit types alpha before it was rounded.
std::array<Tensor, 2> softmax_forward(const Rows& rows, const Tensor& logits, const Tensor& table, const Tensor& buckets, const Tensor& mask,
                                      bool differentiated) {
  const int dtype = check_softmax(rows, logits, "logits");
  refuse_tangents({&table});
  TORCH_CHECK_VALUE(table.defined() == buckets.defined(), "a bias table and the edges' buckets come together");
  check_table(logits, table, buckets);
  check_beside(logits, mask, "mask", {logits.size(0)}, at::kBool);
  const c10::cuda::CUDAGuard guard(logits.device());
  const Tensor z = logits.contiguous(), t = contiguous(table), b = contiguous(buckets), m = contiguous(mask);
  Tensor alpha = at::empty(z.sizes(), z.options()), wide;
  if (differentiated && narrow(z)) wide = at::empty(z.sizes(), z.options().dtype(at::kFloat));
  const Tensor scratch = scratch_of(api.softmax_scratch_bytes(dtype, &rows.native, heads_of(z), 0), z);
  check(api.softmax_fwd(dtype, &rows.native, z.data_ptr(), pointer(t), static_cast<const int32_t*>(pointer(b)),
                        static_cast<const uint8_t*>(pointer(m)), alpha.data_ptr(), pointer(wide), heads_of(z), t.defined() ? t.size(0) : 0,
                        pointer(scratch), bytes_of(scratch), stream_of(z)));
  return {alpha, wide};
}

// In what follows `alpha` is as the launches read it, in float for the 16-bit types, and `type` is the operator's type.  Its cotangent is
// of either: of `type` from a loss, and as wide as alpha from the second order, whose differences 16 bits may not hold.
void check_alpha(const Rows& rows, const Tensor& alpha, at::ScalarType type, const Tensor& g) {
  check_softmax(rows, alpha, "alpha");
  refuse_tangents({&g});
  TORCH_CHECK_TYPE(alpha.scalar_type() == (narrow(type) ? at::kFloat : type), "alpha must be ", narrow(type) ? at::kFloat : type, ", got ",
                   alpha.scalar_type());
  check_beside(alpha, g, "grad_out", alpha.sizes(), g.scalar_type() == alpha.scalar_type() ? alpha.scalar_type() : type);
}
int code_of(at::ScalarType type) { return type == at::kDouble ? LUNA_F64 : type == at::kFloat ? LUNA_F32 : type == at::kHalf ? LUNA_F16 : LUNA_BF16; }

// The gradients of the logits and of the table, as far as `mask` names them.
std::array<Tensor, 2> softmax_backward(const Rows& rows, const Tensor& alpha, at::ScalarType type, const Tensor& g, const Tensor& buckets,
                                       int64_t num_buckets, int mask) {
  std::array<Tensor, 2> out;
  if (!mask) return out;
  check_alpha(rows, alpha, type, g);
  check_table(alpha, Tensor(), buckets);
  const c10::cuda::CUDAGuard guard(alpha.device());
  const Tensor a = prepared(alpha), e = prepared(g), b = contiguous(buckets);
  const auto options = a.options().dtype(type);
  out[0] = at::empty(e.sizes(), options);  // the table's gradient is made of it
  if (mask & 2) out[1] = at::empty({num_buckets, heads_of(e)}, options);
  const int dtype = code_of(type);
  const Tensor scratch = scratch_of(api.softmax_scratch_bytes(dtype, &rows.native, heads_of(e), mask & 2 ? num_buckets : 0), e);
  const auto entry = e.scalar_type() == type ? api.softmax_bwd : api.softmax_bwd_wide;
  check(entry(dtype, &rows.native, a.data_ptr(), e.data_ptr(), static_cast<const int32_t*>(pointer(b)), out[0].data_ptr(), pointer(out[1]),
              heads_of(e), num_buckets, pointer(scratch), bytes_of(scratch), stream_of(e)));
  if (!(mask & 1)) out[0] = Tensor();
  return out;
}

// The derivatives with respect to alpha, as wide as it is, and g named in `mask`.
std::array<Tensor, 2> softmax_double(const Rows& rows, const Tensor& alpha, at::ScalarType type, const Tensor& g, const Tensor& buckets,
                                     const Tensor& r, const Tensor& rtable, int mask) {
  std::array<Tensor, 2> out;
  if (!mask) return out;
  check_alpha(rows, alpha, type, g);
  refuse_tangents({&r, &rtable});
  check_beside(alpha, r, "r", alpha.sizes(), type);
  check_table(alpha, Tensor(), buckets);
  if (rtable.defined()) check_beside(alpha, rtable, "table", {rtable.size(0), heads_of(alpha)}, type);
  const c10::cuda::CUDAGuard guard(alpha.device());
  auto widened = [&](const Tensor& t) { return t.defined() ? t.to(alpha.scalar_type()) : t; };
  if (g.scalar_type() != type)  // the backward of a second order's cotangent: in the type of the sums altogether
    return softmax_double(rows, alpha, alpha.scalar_type(), g, buckets, widened(r), widened(rtable), mask);
  const Tensor a = prepared(alpha), e = g.contiguous(), b = contiguous(buckets), t = contiguous(r), tt = contiguous(rtable);
  if (mask & 1) out[0] = at::empty(a.sizes(), a.options());
  if (mask & 2) out[1] = at::empty(e.sizes(), e.options());
  const int dtype = code_of(type);
  const Tensor scratch = scratch_of(api.softmax_scratch_bytes(dtype, &rows.native, heads_of(e), 0), e);
  check(api.softmax_dbl_bwd_wide(dtype, &rows.native, a.data_ptr(), e.data_ptr(), pointer(t), pointer(tt),
                                 static_cast<const int32_t*>(pointer(b)), pointer(out[0]), pointer(out[1]), heads_of(e),
                                 tt.defined() ? tt.size(0) : 0, pointer(scratch), bytes_of(scratch), stream_of(e)));
  return out;
}

struct SoftmaxDouble : Function<SoftmaxDouble> {
  static variable_list forward(AutogradContext* ctx, const Tensor& alpha, const Tensor& g, const Maybe& buckets, const Maybe& r,
                               const Maybe& rtable, int64_t type, int64_t mask, const RowsPtr& rows) {
    ctx->set_materialize_grads(false);
    return only(softmax_double(*rows, alpha, static_cast<at::ScalarType>(type), g, of(buckets), of(r), of(rtable), static_cast<int>(mask)),
                static_cast<int>(mask));
  }
  static variable_list backward(AutogradContext*, const variable_list& grads) {
    for (const Tensor& t : grads)
      TORCH_CHECK_NOT_IMPLEMENTED(!t.defined(), "third-order derivatives of the softmax over in-edges are not provided");
    return variable_list(8);
  }
};

struct SoftmaxBackward : Function<SoftmaxBackward> {
  static variable_list forward(AutogradContext* ctx, const Tensor& alpha, const Tensor& g, const Maybe& buckets, int64_t num_buckets,
                               int64_t type, int64_t mask, const RowsPtr& rows) {
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({alpha, g, of(buckets)});
    ctx->saved_data["type"] = type;
    ctx->saved_data["mask"] = mask;
    keep(ctx, "rows", rows);
    return only(softmax_backward(*rows, alpha, static_cast<at::ScalarType>(type), g, of(buckets), num_buckets, static_cast<int>(mask)),
                static_cast<int>(mask));
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    variable_list out(7);
    const auto r = spread<2>(grads, static_cast<int>(ctx->saved_data["mask"].toInt()));
    if (!r[0].defined() && !r[1].defined()) return out;
    const auto saved = ctx->get_saved_variables();
    const int mask = wanted(ctx, {&saved[0], &saved[1]});
    if (!mask) return out;
    const auto rows = kept<Rows>(ctx, "rows");
    const int64_t type = ctx->saved_data["type"].toInt();
    const auto h = at::GradMode::is_enabled()
                       ? spread<2>(SoftmaxDouble::apply(saved[0], saved[1], maybe(saved[2]), maybe(r[0]), maybe(r[1]), type,
                                                        static_cast<int64_t>(mask), rows), mask)
                       : softmax_double(*rows, saved[0], static_cast<at::ScalarType>(type), saved[1], saved[2], r[0], r[1], mask);
    for (int s = 0; s < 2; ++s) out[s] = h[s];
    return out;
  }
};

// For the 16-bit types alpha as it was before it was rounded is an output of its own, which no caller sees: the second order's cotangent
// of alpha comes back through it, as wide as it was made.
struct SoftmaxForward : Function<SoftmaxForward> {
  static variable_list forward(AutogradContext* ctx, const Tensor& logits, const Maybe& table, const Maybe& buckets, const Maybe& mask,
                               const RowsPtr& rows) {
    const auto found = softmax_forward(*rows, logits, of(table), of(buckets), of(mask), true);
    ctx->set_materialize_grads(false);
    const bool rounded = found[1].defined();
    ctx->save_for_backward({found[rounded ? 1 : 0], of(buckets)});  // alpha says all about the logits, the table and the mask
    ctx->saved_data["buckets"] = table ? table->size(0) : 0;
    ctx->saved_data["type"] = static_cast<int64_t>(logits.scalar_type());
    keep(ctx, "rows", rows);
    return rounded ? variable_list{found[0], found[1]} : variable_list{found[0]};
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    variable_list out(5);
    Tensor g = grads[0];
    if (grads.size() > 1 && grads[1].defined()) g = g.defined() ? grads[1] + g : grads[1];
    if (!g.defined()) return out;
    const auto saved = ctx->get_saved_variables();
    const int64_t num_buckets = ctx->saved_data["buckets"].toInt(), type = ctx->saved_data["type"].toInt();
    int mask = ctx->needs_input_grad(0) ? 1 : 0;
    if (num_buckets && ctx->needs_input_grad(1)) mask |= 2;
    if (!mask) return out;
    const auto rows = kept<Rows>(ctx, "rows");
    const auto d = at::GradMode::is_enabled()
                       ? spread<2>(SoftmaxBackward::apply(saved[0], g, maybe(saved[1]), num_buckets, type, static_cast<int64_t>(mask), rows), mask)
                       : softmax_backward(*rows, saved[0], static_cast<at::ScalarType>(type), g, saved[1], num_buckets, mask);
    for (int s = 0; s < 2; ++s) out[s] = d[s];
    return out;
  }
};

// What the launches read alpha from, for a caller of the operators: `wide` where there is one.
Tensor exact_alpha(const Tensor& alpha, const Tensor& wide) {
  if (!narrow(alpha)) return alpha;
  if (!wide.defined() || !wide.numel()) return alpha.to(at::kFloat);
  check_beside(alpha, wide, "wide", alpha.sizes(), at::kFloat);
  return wide;
}

Tensor graph_softmax(const RowsPtr& rows, const Tensor& logits, const Maybe& table, const Maybe& buckets, const Maybe& mask) {
  pybind11::gil_scoped_release release;
  return tracked({&logits, &of(table)}) ? SoftmaxForward::apply(logits, table, buckets, mask, rows)[0]
                                        : softmax_forward(*rows, logits, of(table), of(buckets), of(mask), false)[0];
}

// The launches alone, for the operators that a traced program names.
template <size_t N>
std::vector<Maybe> listed(const std::array<Tensor, N>& tensors) {
  std::vector<Maybe> list;
  for (const Tensor& t : tensors) list.push_back(maybe(t));
  return list;
}

}  // namespace

PYBIND11_MODULE(luna_torch, m) {
  m.def("load", torch::wrap_pybind_function(load));
  py::class_<Op, OpPtr>(m, "Op").def(py::init<int64_t, int64_t, int64_t, int64_t, int64_t, bool>());
  py::class_<Graph, GraphPtr>(m, "Graph").def(py::init<std::array<Tensor, 5>, int64_t, int64_t>());
  py::class_<Harmonics, HarmonicsPtr>(m, "Harmonics")
      .def(py::init<const std::vector<int64_t>&, bool, int64_t, int64_t, bool>());
  m.def("graph_tables", torch::wrap_pybind_function(graph_tables));
  m.def("conv", torch::wrap_pybind_function(conv));
  m.def("harmonics", torch::wrap_pybind_function(harmonics));
  py::class_<Norm, NormPtr>(m, "Norm").def(py::init<const std::vector<std::array<int64_t, 3>>&, int64_t, double>());
  py::class_<Rows, RowsPtr>(m, "Rows").def(py::init<const Tensor&, int64_t, const Maybe&, const Maybe&, const Maybe&, const Maybe&>());
  m.def("layer_norm", torch::wrap_pybind_function(layer_norm));
  m.def("distance_buckets", torch::wrap_pybind_function(distance_buckets));
  m.def("relative_bias", torch::wrap_pybind_function(relative_bias));
  m.def("graph_softmax", torch::wrap_pybind_function(graph_softmax));
  m.def("layer_norm_forward", torch::wrap_pybind_function([](const NormPtr& n, const Tensor& x, const Maybe& weight, const Maybe& bias) {
    return listed(norm_forward(*n, x, of(weight), of(bias), true));
  }));
  m.def("layer_norm_backward", torch::wrap_pybind_function([](const NormPtr& n, const Tensor& x, const Maybe& weight, const Tensor& stats, const Tensor& g, int mask) {
    return listed(norm_backward(*n, x, of(weight), stats, g, mask));
  }));
  m.def("layer_norm_double", torch::wrap_pybind_function([](const NormPtr& n, const Tensor& x, const Maybe& weight, const Tensor& stats, const Tensor& g,
                                const Maybe& rx, const Maybe& rw, const Maybe& rb, int mask) {
    return listed(norm_double(*n, x, of(weight), stats, g, of(rx), of(rw), of(rb), mask));
  }));
  m.def("relative_bias_forward", torch::wrap_pybind_function(bias_forward));
  m.def("relative_bias_backward", torch::wrap_pybind_function(bias_backward));
  m.def("graph_softmax_forward", torch::wrap_pybind_function([](const RowsPtr& rows, const Tensor& logits, const Maybe& table,
                                                                const Maybe& buckets, const Maybe& mask) {
    return listed(softmax_forward(*rows, logits, of(table), of(buckets), of(mask), true));
  }));
  m.def("graph_softmax_backward", torch::wrap_pybind_function([](const RowsPtr& rows, const Tensor& alpha, const Maybe& wide, const Tensor& g,
                                                                 const Maybe& buckets, int64_t num_buckets, int mask) {
    return listed(softmax_backward(*rows, exact_alpha(alpha, of(wide)), alpha.scalar_type(), g, of(buckets), num_buckets, mask));
  }));
  m.def("graph_softmax_double", torch::wrap_pybind_function([](const RowsPtr& rows, const Tensor& alpha, const Maybe& wide, const Tensor& g,
                                                               const Maybe& buckets, const Maybe& r, const Maybe& rtable, int mask) {
    return listed(softmax_double(*rows, exact_alpha(alpha, of(wide)), alpha.scalar_type(), g, of(buckets), of(r), of(rtable), mask));
  }));
}
