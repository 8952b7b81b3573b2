// Autograd nodes of the experts' operators for torch tensors, over the C ABI.
//
// A node written in Python runs in Python on the engine's thread in a backward pass, which for small calls takes several
// times what their kernels do: a gather of 333 rows of 768 fp32 with its gradient 78 us, with the nodes here 45 (torch's own
// x[index] with its gradient 70, index_select 48), of which the way to the engine's thread and back is 25.
// Arguments are checked by experts.py; tensors arrive contiguous, on one GPU and in types that the kernels take.
//
// What a backward pass reads is saved by the graph, which refuses tensors that were written to since.  A backward pass is
// made of operators that can be differentiated themselves: where a graph of the gradient is asked for they record one, else
// they are plain launches; the gradient has the same bits either way.  There is no forward mode: a tensor with a tangent is
// refused, as a launch would lose the tangent without a word.
#include <torch/extension.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include "../../include/gptq_hip.h"

namespace {

using at::Tensor;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;

// the C entry points, from the library that the package has loaded
struct Entries {
  decltype(&gptq_hip_error_string) error_string;
  decltype(&gptq_hip_expert_sort_workspace_bytes) sort_bytes;
  decltype(&gptq_hip_expert_sort) sort;
  decltype(&gptq_hip_expert_gather) gather;
  decltype(&gptq_hip_expert_combine) combine;
  decltype(&gptq_hip_expert_combine_grad) combine_grad;
  decltype(&gptq_hip_expert_qmatmul_workspace_bytes) matmul_bytes;
  decltype(&gptq_hip_expert_qmatmul) matmul;
} entry;

void check(int code, const char *what) {
  if (code == GPTQ_HIP_OK) return;
  const std::string text = std::string(what) + ": " + entry.error_string(code);
  TORCH_CHECK_VALUE(code != GPTQ_HIP_EINVAL, text);
  TORCH_CHECK_TYPE(code != GPTQ_HIP_EDTYPE, text);
  TORCH_CHECK(false, text);
}

int type_of(at::ScalarType t) {
  if (t == at::kFloat) return GPTQ_HIP_F32;
  return t == at::kHalf ? GPTQ_HIP_F16 : GPTQ_HIP_BF16;
}
int type_of(const Tensor &t) { return type_of(t.scalar_type()); }
const int32_t *ints(const Tensor &t) { return static_cast<const int32_t *>(t.const_data_ptr()); }
int experts_of(const Tensor &offsets) { return (int)offsets.numel() - 1; }
// the stream and the device of a launch
struct Launch {
  c10::DeviceGuard guard;
  void *stream;
  explicit Launch(const Tensor &t)
      : guard(t.device()), stream(c10::hip::getCurrentHIPStream(t.device().index()).stream()) {}
};
Tensor workspace(size_t bytes, const Tensor &like) {
  return bytes ? at::empty({(int64_t)bytes}, like.options().dtype(at::kByte)) : Tensor();
}
void *address(const Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; }
// Where autograd follows an input, a node of type N whose edges lead to the inputs; an undefined input has an empty edge.
template <typename N, typename... T> std::shared_ptr<N> node_of(const T &...inputs) {
  TORCH_CHECK_NOT_IMPLEMENTED(!((inputs.defined() && inputs._fw_grad(0).defined()) || ...),
                              "the experts' operators have no forward-mode derivative");
  if (!torch::autograd::compute_requires_grad(inputs...)) return nullptr;
  std::shared_ptr<N> node(new N(), torch::autograd::deleteNode);
  node->set_next_edges(torch::autograd::collect_next_edges(inputs...));
  return node;
}
SavedVariable saved(const Tensor &t) { return SavedVariable(t, false); }
// A plan's or a stack's tensor, saved.  One that was made in inference mode cannot be: nothing counts what is written to
// it.  It is kept as it is, so that a stack that was quantised in inference mode can be trained through.
class Kept {
 public:
  void keep(const Tensor &t) {
    if (t.is_inference()) plain = t;
    else counted = saved(t);
  }
  Tensor unpack() const {
    const Tensor t = plain.defined() ? plain : counted.unpack();
    TORCH_CHECK(t.defined(), "a second backward pass through a graph that the first has released");
    return t;
  }
  void release() {
    plain.reset();
    counted.reset_data();
  }

 private:
  SavedVariable counted;
  Tensor plain;
};
Tensor dense(const Tensor &t) { return t.is_contiguous() ? t : t.contiguous(); }

std::tuple<Tensor, Tensor, Tensor> sort(const Tensor &ids, int64_t n_experts) {
  const Launch here(ids);
  const int64_t pairs = ids.numel();
  const Tensor all = at::empty({2 * pairs + n_experts + 1}, ids.options().dtype(at::kInt));
  const Tensor order = all.narrow(0, 0, pairs), position = all.narrow(0, pairs, pairs),
               offsets = all.narrow(0, 2 * pairs, n_experts + 1);
  const size_t bytes = entry.sort_bytes(pairs, (int)n_experts);
  const Tensor ws = workspace(bytes, ids);
  check(entry.sort(here.stream, ids.data_ptr(), (int)ids.element_size(), pairs, (int)n_experts,
                   order.data_ptr<int32_t>(), position.data_ptr<int32_t>(), offsets.data_ptr<int32_t>(), address(ws),
                   bytes),
        "expert_sort");
  return {order, position, offsets};
}

Tensor gather_raw(const Tensor &x, const Tensor &position, const Tensor &offsets, int64_t top_k) {
  const Launch here(x);
  const int64_t tokens = x.size(0), width = x.size(1);
  const Tensor out = at::empty({tokens * top_k, width}, x.options());
  check(entry.gather(here.stream, x.const_data_ptr(), type_of(x), tokens, (int)top_k, width, ints(position), ints(offsets),
                     experts_of(offsets), out.data_ptr()),
        "expert_gather");
  return out;
}

// `weights` may be undefined: ones
Tensor combine_raw(const Tensor &y, const Tensor &weights, const Tensor &position, const Tensor &offsets, int64_t top_k,
                   at::ScalarType type) {
  const Launch here(y);
  const int64_t tokens = position.numel() / top_k, width = y.size(1);
  const Tensor out = at::empty({tokens, width}, y.options().dtype(type));
  check(entry.combine(here.stream, y.const_data_ptr(), type_of(y), tokens, (int)top_k, width, ints(position), ints(offsets),
                      experts_of(offsets), weights.defined() ? weights.const_data_ptr() : nullptr,
                      weights.defined() ? type_of(weights) : GPTQ_HIP_F32, out.data_ptr(), type_of(type)),
        "expert_combine");
  return out;
}

// gradients of the rows and of the weights, those that are wanted
std::pair<Tensor, Tensor> combine_grad_raw(const Tensor &y, const Tensor &weights, const Tensor &g, const Tensor &position,
                                           const Tensor &offsets, int64_t top_k, bool want_y, bool want_weights) {
  const Launch here(y);
  const Tensor dy = want_y ? at::empty_like(y) : Tensor(), dw = want_weights ? at::empty_like(weights) : Tensor();
  check(entry.combine_grad(here.stream, y.const_data_ptr(), g.const_data_ptr(), type_of(y), g.size(0), (int)top_k,
                           y.size(1), ints(position), ints(offsets), experts_of(offsets), weights.const_data_ptr(),
                           type_of(weights), address(dy), address(dw)),
        "expert_combine_grad");
  return {dy, dw};
}

// the packed stack, and which product
struct Product {
  Tensor packed, zero, scale, order, position, offsets;
  int64_t top_k, bits, group;
  bool sorted_rows, transpose;
};

Tensor matmul_raw(Tensor x, const Product &p, at::ScalarType type) {
  const Launch here(x);
  const int64_t E = p.packed.size(0), R = p.packed.size(1), C = p.packed.size(2), rows = p.order.numel();
  const Tensor out = at::empty({rows, p.transpose ? R * (8 / p.bits) : C}, x.options().dtype(type));
  if (p.transpose && (uintptr_t)x.const_data_ptr() % 16) {   // (those kernels load 16 bytes at a time)
    const at::NoGradGuard plain;
    x = x.clone();
  }
  const size_t bytes = entry.matmul_bytes(x.size(0), rows, R, C, (int)p.bits, p.group, (int)E, type_of(x), type_of(p.zero),
                                          p.transpose);
  const Tensor ws = workspace(bytes, x);
  check(entry.matmul(here.stream, x.const_data_ptr(), type_of(x), x.size(0), p.sorted_rows ? nullptr : ints(p.order),
                     (int)p.top_k, rows, ints(p.offsets), (int)E, p.packed.const_data_ptr<uint8_t>(), R, C,
                     p.zero.const_data_ptr(), p.scale.const_data_ptr(), type_of(p.zero), p.group, (int)p.bits, p.transpose,
                     out.data_ptr(), type_of(type), address(ws), bytes),
        "expert_qmatmul");
  return out;
}

Tensor gather(const Tensor &x, const Tensor &position, const Tensor &offsets, int64_t top_k);
Tensor combine(const Tensor &y, const Tensor &weights, const Tensor &position, const Tensor &offsets, int64_t top_k,
               at::ScalarType type);
std::pair<Tensor, Tensor> combine_grad(const Tensor &y, const Tensor &weights, const Tensor &g, const Tensor &position,
                                       const Tensor &offsets, int64_t top_k);
Tensor matmul(const Tensor &x, const Product &p, at::ScalarType type);

// A node that reads a plan.  apply() holds the lock: another thread may release what is saved.
struct PlanNode : torch::autograd::Node {
  Kept position, offsets;
  int64_t top_k;
  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    position.release();
    offsets.release();
    release();
  }
  virtual void release() {}
  void keep(const Tensor &position_, const Tensor &offsets_, int64_t top_k_) {
    position.keep(position_);
    offsets.keep(offsets_);
    top_k = top_k_;
  }
};

struct GatherNode : PlanNode {
  std::string name() const override { return "ExpertGatherBackward"; }
  variable_list apply(variable_list &&grads) override {
    std::lock_guard<std::mutex> lock(mutex_);
    if (!grads[0].defined()) return {Tensor()};
    return {combine(dense(grads[0]), Tensor(), position.unpack(), offsets.unpack(), top_k, grads[0].scalar_type())};
  }
};

struct CombineNode : PlanNode {
  SavedVariable y, weights;
  bool weighted;
  at::ScalarType type;                 // of y
  std::string name() const override { return "ExpertCombineBackward"; }
  void release() override {
    y.reset_data();
    weights.reset_data();
  }
  variable_list apply(variable_list &&grads) override {
    std::lock_guard<std::mutex> lock(mutex_);
    if (!grads[0].defined()) return {Tensor(), Tensor()};
    const Tensor g = dense(grads[0].to(type)), p = position.unpack(), o = offsets.unpack();
    if (!weighted) return {gather(g, p, o, top_k), Tensor()};
    const Tensor rows = y.unpack(), w = weights.unpack();
    const auto both = at::GradMode::is_enabled() || g._fw_grad(0).defined()
                          ? combine_grad(rows, w, g, p, o, top_k)
                          : combine_grad_raw(rows, w, g, p, o, top_k, task_should_compute_output(0),
                                             task_should_compute_output(1));
    return {both.first, both.second};
  }
};

// dy[p] = w[t, j] g[t] and dw[t, j] = <g[t], y[p]> for the pair (t, j) of row p, to be differentiated again: with ey, ew in
// the places of their gradients, y gets ew g and w gets <g, ey>, which is the same operator, and g the sum of w ey + ew y
// over the pairs of a token.
struct CombineGradNode : PlanNode {
  SavedVariable y, weights, g;
  std::string name() const override { return "ExpertCombineGradBackward"; }
  void release() override {
    y.reset_data();
    weights.reset_data();
    g.reset_data();
  }
  variable_list apply(variable_list &&grads) override {
    std::lock_guard<std::mutex> lock(mutex_);
    const Tensor rows = y.unpack(), w = weights.unpack(), h = g.unpack(), p = position.unpack(), o = offsets.unpack();
    const Tensor ey = grads[0].defined() ? dense(grads[0]) : at::zeros_like(rows);
    const Tensor ew = grads[1].defined() ? dense(grads[1]) : at::zeros_like(w);
    const auto both = combine_grad(ey, ew, h, p, o, top_k);
    return {both.first, both.second,
            combine(ey, w, p, o, top_k, h.scalar_type()) + combine(rows, ew, p, o, top_k, h.scalar_type())};
  }
};

struct MatmulNode : PlanNode {
  Kept packed, zero, scale, order;
  int64_t bits, group;
  bool sorted_rows, transpose;
  at::ScalarType type;                 // of x
  std::string name() const override { return "ExpertMatmulBackward"; }
  void release() override {
    packed.release();
    zero.release();
    scale.release();
    order.release();
  }
  variable_list apply(variable_list &&grads) override {
    std::lock_guard<std::mutex> lock(mutex_);
    if (!grads[0].defined()) return {Tensor()};
    const Tensor g = dense(grads[0]);
    const Product p = {packed.unpack(), zero.unpack(), scale.unpack(), order.unpack(), position.unpack(),
                       offsets.unpack(), top_k, bits, group, true, !transpose};
    // a token's copies are added up before the one rounding: their gradients travel in fp32
    const Tensor dx = matmul(g, p, sorted_rows ? g.scalar_type() : at::kFloat);
    return {sorted_rows ? dx.to(type) : combine(dx, Tensor(), p.position, p.offsets, p.top_k, type)};
  }
};

Tensor gather(const Tensor &x, const Tensor &position, const Tensor &offsets, int64_t top_k) {
  const auto node = node_of<GatherNode>(x);
  const Tensor out = gather_raw(x, position, offsets, top_k);
  if (node) {
    node->keep(position, offsets, top_k);
    torch::autograd::set_history(out, node);
  }
  return out;
}

Tensor combine(const Tensor &y, const Tensor &weights, const Tensor &position, const Tensor &offsets, int64_t top_k,
               at::ScalarType type) {
  const auto node = node_of<CombineNode>(y, weights);
  const Tensor out = combine_raw(y, weights, position, offsets, top_k, type);
  if (node) {
    node->keep(position, offsets, top_k);
    node->weighted = weights.defined();
    if (node->weighted) {
      node->y = saved(y);
      node->weights = saved(weights);
    }
    node->type = y.scalar_type();
    torch::autograd::set_history(out, node);
  }
  return out;
}

std::pair<Tensor, Tensor> combine_grad(const Tensor &y, const Tensor &weights, const Tensor &g, const Tensor &position,
                                       const Tensor &offsets, int64_t top_k) {
  const auto node = node_of<CombineGradNode>(y, weights, g);
  const auto both = combine_grad_raw(y, weights, g, position, offsets, top_k, true, true);
  if (node) {
    node->keep(position, offsets, top_k);
    node->y = saved(y);
    node->weights = saved(weights);
    node->g = saved(g);
    torch::autograd::set_history({both.first, both.second}, node);
  }
  return both;
}

Tensor matmul(const Tensor &x, const Product &p, at::ScalarType type) {
  const auto node = node_of<MatmulNode>(x);
  const Tensor out = matmul_raw(x, p, type);
  if (node) {
    node->keep(p.position, p.offsets, p.top_k);
    node->packed.keep(p.packed);
    node->zero.keep(p.zero);
    node->scale.keep(p.scale);
    node->order.keep(p.order);
    node->bits = p.bits;
    node->group = p.group;
    node->sorted_rows = p.sorted_rows;
    node->transpose = p.transpose;
    node->type = x.scalar_type();
    torch::autograd::set_history(out, node);
  }
  return out;
}

template <typename F> void take(F &f, const std::map<std::string, uintptr_t> &addresses, const char *name) {
  f = reinterpret_cast<F>(addresses.at(name));
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("bind", [](const std::map<std::string, uintptr_t> &addresses) {
    take(entry.error_string, addresses, "gptq_hip_error_string");
    take(entry.sort_bytes, addresses, "gptq_hip_expert_sort_workspace_bytes");
    take(entry.sort, addresses, "gptq_hip_expert_sort");
    take(entry.gather, addresses, "gptq_hip_expert_gather");
    take(entry.combine, addresses, "gptq_hip_expert_combine");
    take(entry.combine_grad, addresses, "gptq_hip_expert_combine_grad");
    take(entry.matmul_bytes, addresses, "gptq_hip_expert_qmatmul_workspace_bytes");
    take(entry.matmul, addresses, "gptq_hip_expert_qmatmul");
  });
  m.def("sort", &sort);
  m.def("gather", &gather);
  m.def("combine", [](const Tensor &y, const std::optional<Tensor> &weights, const Tensor &position,
                      const Tensor &offsets, int64_t top_k) {
    return combine(y, weights ? *weights : Tensor(), position, offsets, top_k, y.scalar_type());
  });
  m.def("matmul", [](const Tensor &x, const Tensor &packed, const Tensor &zero, const Tensor &scale, const Tensor &order,
                     const Tensor &position, const Tensor &offsets, int64_t top_k, int64_t bits, int64_t group,
                     bool sorted_rows, bool transpose) {
    return matmul(x, Product{packed, zero, scale, order, position, offsets, top_k, bits, group, sorted_rows, transpose},
                  x.scalar_type());
  });
}
