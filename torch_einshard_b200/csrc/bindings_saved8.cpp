// Contractions whose first operand backward keeps in 8 bits, as autograd nodes
// on the native products (the same nodes for other tensors: ops/saved8.py):
//
//   z = x y     dx = dz y^T     dy = x^^T dz     with x^ from its codes, or silu of what they stand for
//
// A contraction is planned as [batch, rows, red] x [batch, red, cols]: orders
// that bring the operands' axes there and the product's to the result's.
//
// Several contractions of one operand meet in a ReadersNode: their backward
// passes leave dz and y there, and sum_i dz_i y_i^T is one product with one
// rounding, where autograd would add rounded gradients.
#include "bindings_train.h"

#include <ATen/core/LegacyTypeDispatch.h>
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/CUDAEvent.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/engine.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>

#include <map>
#include <memory>
#include <mutex>

#include "gemm.h"
#include "quant8.h"

namespace es {
namespace {

using torch::autograd::Node;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;
using Order = std::vector<int64_t>;  // empty: as they are
using Opt = c10::optional<at::Tensor>;

GemmOps g_ops;

Order inverse(const Order& order) {
  Order back(order.size());
  for (size_t i = 0; i < order.size(); ++i) back[order[i]] = static_cast<int64_t>(i);
  return back;
}

at::Tensor moved(const at::Tensor& t, const Order& order) { return order.empty() ? t : t.permute(order); }

struct ContractPlan {
  int64_t batch, rows, cols, red;
  Order x_order, y_order, z_order, x_back, y_back, z_back;
  Order x_shape, y_shape, z_shape;

  ContractPlan(const Order& gemm, const Order& xo, const Order& yo, const Order& zo, const Order& xs, const Order& ys,
               const Order& zs)
      : batch(gemm.at(0)), rows(gemm.at(1)), cols(gemm.at(2)), red(gemm.at(3)), x_order(xo), y_order(yo), z_order(zo),
        x_back(inverse(xo)), y_back(inverse(yo)), z_back(inverse(zo)), x_shape(xs), y_shape(ys), z_shape(zs) {}

  at::Tensor operand_x(const at::Tensor& x) const { return moved(x, x_order).reshape({batch, rows, red}); }
  at::Tensor operand_y(const at::Tensor& y) const { return moved(y, y_order).reshape({batch, red, cols}); }
  at::Tensor result(const at::Tensor& z) const { return moved(z.view(z_shape), z_order); }
  at::Tensor product_of(const at::Tensor& z) const { return moved(z, z_back).reshape({batch, rows, cols}); }
  // whether the operands' matrices are the same
  bool reads_like(const ContractPlan& p) const {
    return x_order == p.x_order && batch == p.batch && rows == p.rows;
  }
  at::Tensor x_of(const at::Tensor& t) const { return moved(t.view(x_shape), x_back); }
};

// Whether the products read the matrix as it is, contiguous along `dim`.
bool readable(const at::Tensor& t, int64_t dim) {
  const int64_t other = 3 - dim, size = t.element_size();
  if (t.stride(dim) != 1 && t.size(dim) > 1) return false;
  if (reinterpret_cast<uintptr_t>(t.data_ptr()) % 16) return false;
  const int64_t row = t.size(other) > 1 ? t.stride(other) : t.size(dim);
  return row * size % 16 == 0 && (t.size(0) == 1 || t.stride(0) * size % 16 == 0);
}

// The matrix in a layout that the products read; a copy has rows (columns, where these are in a row) that are a
// multiple of 16 bytes apart.
at::Tensor prepared(const at::Tensor& t) {
  if (readable(t, 2) || readable(t, 1)) return t;
  if (t.stride(1) == 1 && t.stride(2) != 1) return prepared(t.transpose(1, 2)).transpose(1, 2);
  const int64_t unit = 16 / t.element_size(), pitch = (t.size(2) + unit - 1) / unit * unit;
  at::Tensor copy = at::empty({t.size(0), t.size(1), pitch}, t.options()).narrow(2, 0, t.size(2));
  copy.copy_(t);
  return copy;
}

int64_t code_of(at::ScalarType t) { return t == at::kHalf ? kDtypeF16 : kDtypeBF16; }

at::Tensor place_of(const at::Tensor& t) { return at::empty({}, t.options()).expand(t.sizes()); }

// The products of operand pairs, added in 32 bits.
at::Tensor product_sum(const std::vector<at::Tensor>& a, const std::vector<at::Tensor>& b, const at::Tensor& err) {
  if (a.size() == 1) return g_ops.product(a[0], b[0], err);
  const Opt sum = g_ops.sum(a, b, err);
  if (sum.has_value()) return *sum;
  // more than it takes, or of different layouts: one product over all their columns
  return g_ops.product(prepared(at::cat(a, 2)), prepared(at::cat(b, 1)), err);
}

// What a contraction's backward pass leaves for the gradient of the operand that it shares.
struct Part {
  std::shared_ptr<const ContractPlan> plan;
  at::Tensor dz, yt;
  c10::cuda::CUDAStream stream;
  std::vector<at::Tensor> sources;  // what its gradient depends on
};

// One backward pass's: the parts, and the operand restored by the first contraction, for those on its stream that
// read it in the same order.
struct Pass {
  std::vector<Part> parts;
  at::Tensor operand;
  std::shared_ptr<const ContractPlan> plan;
  c10::optional<c10::cuda::CUDAStream> stream;
};

// The place where the gradients of an operand's contractions meet.  A backward pass is known by its number: passes
// over one graph (again, or from two threads) do not meet.  What a pass has brought when it raises stays until the
// graph goes.
struct ReadersNode : public Node {
  std::mutex lock;
  std::map<int, Pass> passes;
  at::Tensor err;

  void add(Part part) {
    const std::lock_guard<std::mutex> held(lock);
    passes[torch::autograd::get_current_graph_task_id()].parts.push_back(std::move(part));
  }

  template <class Restore>
  at::Tensor operand(const std::shared_ptr<const ContractPlan>& plan, const Restore& restore) {
    const auto stream = at::cuda::getCurrentCUDAStream();
    const std::lock_guard<std::mutex> held(lock);
    Pass& pass = passes[torch::autograd::get_current_graph_task_id()];
    if (pass.stream.has_value() && *pass.stream == stream && pass.plan->reads_like(*plan)) return pass.operand;
    const at::Tensor x = restore();
    if (!pass.stream.has_value()) {
      pass.operand = x;
      pass.plan = plan;
      pass.stream = stream;
    }
    return x;
  }

  variable_list apply(variable_list&&) override {
    std::vector<Part> parts;
    {
      const std::lock_guard<std::mutex> held(lock);
      const auto found = passes.find(torch::autograd::get_current_graph_task_id());
      if (found != passes.end()) {
        parts = std::move(found->second.parts);
        passes.erase(found);
      }
    }
    if (parts.empty()) return {at::Tensor()};
    const c10::cuda::CUDAGuard guard(parts[0].dz.device());
    const auto here = at::cuda::getCurrentCUDAStream();
    std::vector<at::Tensor> total(1), from;
    {
      const at::AutoDispatchBelowAutograd below;
      for (const Part& p : parts) {
        if (p.stream == here) continue;
        at::cuda::CUDAEvent done;
        done.record(p.stream);
        done.block(here);
        for (const at::Tensor& t : {p.dz, p.yt}) c10::cuda::CUDACachingAllocator::recordStream(t.storage().data_ptr(), here);
      }
      std::vector<bool> used(parts.size());
      for (size_t i = 0; i < parts.size(); ++i) {
        if (used[i]) continue;
        const ContractPlan& plan = *parts[i].plan;
        std::vector<at::Tensor> dz, yt;
        for (size_t j = i; j < parts.size(); ++j) {
          const ContractPlan& p = *parts[j].plan;
          if (used[j] || !p.reads_like(plan)) continue;
          used[j] = true;
          dz.push_back(parts[j].dz);
          yt.push_back(prepared(parts[j].yt));
        }
        const at::Tensor dx = plan.x_of(product_sum(dz, yt, err));
        total[0] = total[0].defined() ? total[0] + dx : dx;
      }
    }
    for (const Part& p : parts) from.insert(from.end(), p.sources.begin(), p.sources.end());
    finalise(total, from);
    return total;
  }

  void release_variables() override {}
};

// What is kept of an operand: its codes, whether they are a silu's pre-activation, the shape that was quantised and
// the order of axes that leads from there to the operand.
struct Kept {
  bool act;
  Order base, order;
};

struct ContractNode : public Node {
  std::mutex lock;
  std::shared_ptr<const ContractPlan> plan;
  SavedVariable y, codes, exps, h_codes, h_exps;
  Kept kept;
  bool silu = false;
  at::ScalarType dtype;
  at::Tensor err;

  at::Tensor restored(const at::Tensor& c, const at::Tensor& e) const {
    const at::Tensor x = restore8_op(c.contiguous(), e, c10::nullopt, code_of(dtype), kept.act ? kRestoreSilu : kRestoreValue);
    return moved(x.view(kept.base), kept.order);
  }

  // grad times silu' of what the codes stand for, in grad's axes
  static at::Tensor through_silu(const at::Tensor& grad, const at::Tensor& c, const at::Tensor& e, const Order& order) {
    const at::Tensor g = moved(grad, inverse(order));
    const at::Tensor d = restore8_op(c.contiguous(), e, g.reshape(c.sizes()).contiguous(),
                                     code_of(grad.scalar_type()), kRestoreSiluGrad);
    return moved(d.view(g.sizes()), order);
  }

  // whether the pre-activation was quantised in the very rows this product reads
  bool same_rows(const at::Tensor& c) const {
    for (size_t i = 0; i < kept.order.size(); ++i)
      if (kept.order[i] != static_cast<int64_t>(i)) return false;
    return plan->x_order.empty() && c.size(0) == plan->batch * plan->rows && c.size(1) == plan->red;
  }

  variable_list apply(variable_list&& grads) override {
    const std::lock_guard<std::mutex> held(lock);
    variable_list out(2);  // of the place, of y
    const bool any = grads[0].defined() || (silu && grads[1].defined());
    if (!any) return out;
    const at::Tensor yv = y.unpack(), c = codes.unpack(), e = exps.unpack();
    const c10::cuda::CUDAGuard guard(yv.device());
    ReadersNode* readers = nullptr;
    const bool want_place = task_should_compute_output(0);
    if (want_place) readers = dynamic_cast<ReadersNode*>(next_edge(0).function.get());
    std::vector<at::Tensor> found(2);
    {
      const at::AutoDispatchBelowAutograd below;
      at::Tensor grad = plain(grads[0]);
      if (grad.defined() && silu) grad = through_silu(grad, h_codes.unpack(), h_exps.unpack(), plan->z_order);
      if (silu && grads[1].defined()) grad = grad.defined() ? grad + grads[1] : plain(grads[1]);
      const at::Tensor gz = prepared(plan->product_of(grad));
      const at::Tensor y3 = plan->operand_y(yv), yt = y3.transpose(1, 2);
      at::Tensor x;  // the operand, for dy
      if (readers != nullptr) {
        std::vector<at::Tensor> sources(grads);
        sources.push_back(yv);
        readers->add({plan, gz, yt, at::cuda::getCurrentCUDAStream(), sources});
      } else if (want_place && same_rows(c)) {
        // (dz y^T) silu'(h^) and silu(h^) from one product
        const auto both = g_ops.silu_grad(gz, prepared(yt), c, e, err);
        found[0] = plan->x_of(both[0]);
        x = both[1];
      } else if (want_place) {
        found[0] = through_silu(plan->x_of(g_ops.product(gz, prepared(yt), err)), c, e, kept.order);
      }
      if (task_should_compute_output(1)) {
        if (!x.defined()) {
          const auto restore = [&] { return prepared(plan->operand_x(restored(c, e))); };
          x = readers == nullptr ? restore() : readers->operand(plan, restore);
        }
        // a transposed y (an [out, in] weight) gets its gradient in its own memory order
        const bool turned = y3.stride(1) == 1 && y3.size(1) > 1;
        at::Tensor dy = turned ? g_ops.product(prepared(gz.transpose(1, 2)), x, err).transpose(1, 2)
                               : g_ops.product(prepared(x.transpose(1, 2)), gz, err);
        found[1] = moved(dy.reshape(plan->y_shape), plan->y_back);
      }
    }
    finalise(found, grads);
    finalise(found, {yv});
    for (size_t i = 0; i < 2; ++i) out[i] = found[i];
    return out;
  }

  void release_variables() override {
    const std::lock_guard<std::mutex> held(lock);
    for (SavedVariable* v : {&y, &codes, &exps, &h_codes, &h_exps}) v->reset_data();
  }
};

// The place where the gradients of x's contractions meet: x's shape, without values.
at::Tensor readers_of(const at::Tensor& x, const at::Tensor& err) {
  at::Tensor place;
  {
    const at::AutoDispatchBelowADInplaceOrView below;
    place = place_of(x.detach());
  }
  auto node = std::shared_ptr<ReadersNode>(new ReadersNode(), torch::autograd::deleteNode);
  node->err = err;
  node->set_next_edges(torch::autograd::collect_next_edges(x));
  torch::autograd::set_history(place, node);
  return place;
}

// The contraction of x, whose gradient goes to `place` (a pre-activation's place, or readers_of; none: it has none),
// with y: (z), or with `silu` (silu(z), its pre-activation's place, codes and exponents).  `ready` is x's matrix as an
// earlier contraction read it; where that takes a copy, the matrix is the last result.
std::vector<at::Tensor> contract8(const at::Tensor& x, const Opt& place, const at::Tensor& y,
                                  const std::shared_ptr<ContractPlan>& plan, const at::Tensor& codes,
                                  const at::Tensor& exps, bool act, const Order& base, const Order& order, bool silu,
                                  const at::Tensor& err, const Opt& ready) {
  TORCH_CHECK(x.is_cuda() && y.device() == x.device() && codes.device() == x.device() && exps.device() == x.device(),
              "einshard: operands of an 8-bit contraction on one CUDA device");
  const c10::cuda::CUDAGuard guard(x.device());
  std::vector<at::Tensor> out;
  at::Tensor copied;
  const auto results = [&]() -> std::vector<at::Tensor>& {
    if (copied.defined()) out.push_back(copied);
    return out;
  };
  {
    const at::AutoDispatchBelowADInplaceOrView below;
    const at::Tensor own = ready.has_value() ? *ready : plan->operand_x(x.detach());
    const at::Tensor xv = prepared(own), yv = prepared(plan->operand_y(y.detach()));
    if (!xv.is_same(own)) copied = xv;
    if (silu) {
      out = g_ops.silu(xv, yv, err);
      out[0] = plan->result(out[0]);
      out.insert(out.begin() + 1, place_of(out[0]));
    } else {
      out = {plan->result(g_ops.product(xv, yv, err).contiguous())};
    }
  }
  const at::Tensor at = place.has_value() ? *place : at::Tensor();
  if (!torch::autograd::compute_requires_grad(at, y)) return results();
  auto node = std::shared_ptr<ContractNode>(new ContractNode(), torch::autograd::deleteNode);
  node->set_next_edges(torch::autograd::collect_next_edges(at, y));
  node->plan = plan;
  node->y = SavedVariable(y, false);
  node->codes = SavedVariable(codes, false);
  node->exps = SavedVariable(exps, false);
  node->kept = {act, base, order};
  node->silu = silu;
  node->dtype = x.scalar_type();
  node->err = err;
  if (silu) {
    node->h_codes = SavedVariable(out[2], false);
    node->h_exps = SavedVariable(out[3], false);
  }
  torch::autograd::set_history(out[0], node);
  if (silu) torch::autograd::set_history(out[1], node);
  return results();
}

}  // namespace

void bind_saved8_ops(pybind11::module_& m, const GemmOps& ops) {
  namespace py = pybind11;
  g_ops = ops;
  py::class_<ContractPlan, std::shared_ptr<ContractPlan>>(m, "ContractPlan")
      .def(py::init<const Order&, const Order&, const Order&, const Order&, const Order&, const Order&, const Order&>());
  m.def("readers8", &readers_of, "the place where the gradients of an operand's contractions meet",
        py::call_guard<py::gil_scoped_release>());
  m.def("contract8", &contract8, "a contraction whose first operand is kept in 8 bits, with gradients",
        py::call_guard<py::gil_scoped_release>());
}

}  // namespace es
