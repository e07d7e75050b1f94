// Torch bindings of the training-step operators around the contractions:
// activations kept in 8 bits (quant8.h), norms with gate and residual (norm.h),
// the policy loss (policy.h).
#include "bindings_train.h"

#include <ATen/cuda/CUDAContext.h>
#include <ATen/core/LegacyTypeDispatch.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/custom_function.h>

#include "gemm.h"
#include "norm.h"
#include "policy.h"
#include "quant8.h"

namespace es {
namespace {

std::atomic<long long>* g_count = nullptr;

void counted(int rc, const char* what, int launches = 1) {
  TORCH_CHECK(rc == 0, "einshard ", what, ": launch failed (", rc, ")");
  g_count->fetch_add(launches, std::memory_order_relaxed);
}

int code_of(at::ScalarType t, const char* what) {
  switch (t) {
    case at::kBFloat16:
      return kDtypeBF16;
    case at::kHalf:
      return kDtypeF16;
    case at::kFloat:
      return kDtypeF32;
    default:
      TORCH_CHECK(false, "einshard ", what, ": bf16, fp16 or fp32, not ", t);
  }
}

int sms_of(const at::Tensor& t) { return at::cuda::getDeviceProperties(t.get_device())->multiProcessorCount; }

int64_t blocks_of(int64_t d) { return (d + kQuantBlock - 1) / kQuantBlock; }

// (codes [rows, d], exps [rows, ceil(d / 32)]) of a contiguous [rows, d] tensor
std::vector<at::Tensor> quant8_op(const at::Tensor& x) {
  TORCH_CHECK(x.is_cuda() && x.dim() == 2 && x.is_contiguous(), "einshard checkpoint8: contiguous 2-D CUDA tensor");
  const c10::cuda::CUDAGuard guard(x.device());
  const int64_t rows = x.size(0), d = x.size(1);
  at::Tensor codes = at::empty({rows, d}, x.options().dtype(at::kChar));
  at::Tensor exps = at::empty({rows, blocks_of(d)}, x.options().dtype(at::kByte));
  if (x.numel() == 0) return {codes, exps};
  counted(quant8(x.data_ptr(), code_of(x.scalar_type(), "checkpoint8"), codes.data_ptr<int8_t>(),
                 exps.data_ptr<uint8_t>(), rows, d, sms_of(x), at::cuda::getCurrentCUDAStream()),
          "checkpoint8");
  return {codes, exps};
}

at::ScalarType type_of(int64_t dtype) {
  return dtype == kDtypeF32 ? at::kFloat : (dtype == kDtypeF16 ? at::kHalf : at::kBFloat16);
}

// (silu(h), codes, exps) of a contiguous fp32 [rows, d] pre-activation
std::vector<at::Tensor> quant8_silu_op(const at::Tensor& h, int64_t out_dtype) {
  TORCH_CHECK(h.is_cuda() && h.dim() == 2 && h.is_contiguous() && h.scalar_type() == at::kFloat,
              "einshard checkpoint8 silu: contiguous 2-D fp32 CUDA tensor");
  const c10::cuda::CUDAGuard guard(h.device());
  const int64_t rows = h.size(0), d = h.size(1);
  at::Tensor out = at::empty({rows, d}, h.options().dtype(type_of(out_dtype)));
  at::Tensor codes = at::empty({rows, d}, h.options().dtype(at::kChar));
  at::Tensor exps = at::empty({rows, blocks_of(d)}, h.options().dtype(at::kByte));
  if (h.numel() == 0) return {out, codes, exps};
  counted(quant8_silu(h.data_ptr<float>(), out.data_ptr(), static_cast<int>(out_dtype), codes.data_ptr<int8_t>(),
                      exps.data_ptr<uint8_t>(), rows, d, sms_of(h), at::cuda::getCurrentCUDAStream()),
          "checkpoint8 silu");
  return {out, codes, exps};
}

}  // namespace

at::Tensor restore8_op(const at::Tensor& codes, const at::Tensor& exps, const c10::optional<at::Tensor>& grad,
                       int64_t dtype, int64_t mode) {
  TORCH_CHECK(codes.is_cuda() && codes.dim() == 2 && codes.is_contiguous() && codes.scalar_type() == at::kChar,
              "einshard restore8: contiguous 2-D int8 codes");
  TORCH_CHECK(exps.device() == codes.device() && exps.is_contiguous() && exps.scalar_type() == at::kByte &&
                  exps.dim() == 2 && exps.size(0) == codes.size(0) && exps.size(1) == blocks_of(codes.size(1)),
              "einshard restore8: exponents [rows, ceil(d / 32)]");
  TORCH_CHECK((mode == kRestoreSiluGrad) == grad.has_value(), "einshard restore8: a gradient goes with mode 2 alone");
  const c10::cuda::CUDAGuard guard(codes.device());
  at::Tensor out = at::empty(codes.sizes(), codes.options().dtype(type_of(dtype)));
  const void* g = nullptr;
  if (grad.has_value()) {
    TORCH_CHECK(grad->device() == codes.device() && grad->is_contiguous() && grad->sizes() == codes.sizes() &&
                    grad->scalar_type() == out.scalar_type(),
                "einshard restore8: gradient of the codes' shape, contiguous");
    g = grad->data_ptr();
  }
  if (codes.numel() == 0) return out;
  counted(restore8(codes.data_ptr<int8_t>(), exps.data_ptr<uint8_t>(), g, out.data_ptr(), static_cast<int>(dtype),
                   static_cast<int>(mode), codes.size(0), codes.size(1), sms_of(codes),
                   at::cuda::getCurrentCUDAStream()),
          "restore8");
  return out;
}

namespace {

// ------------------------------------------------------------------ norms

using Opt = c10::optional<at::Tensor>;

void norm_param(NormParam& q, const Opt& t, const at::Tensor& x, int64_t count, const char* name) {
  if (!t.has_value()) return;
  TORCH_CHECK(t->device() == x.device() && t->is_contiguous() && t->numel() == count &&
                  (t->scalar_type() == x.scalar_type() || t->scalar_type() == at::kFloat),
              "einshard norm: ", name, " of ", count, " elements, contiguous, of the stream's type or fp32");
  q.p = t->data_ptr();
  q.f32 = t->scalar_type() == at::kFloat ? 1 : 0;
}

NormArgs norm_args(const at::Tensor& x, const Opt& y, const Opt& w, const Opt& b, const Opt& pw, const Opt& pb,
                   const Opt& gate, int64_t gate_inner, int64_t gate_count, bool post, bool center, double scale,
                   double eps) {
  TORCH_CHECK(x.is_cuda() && x.dim() == 2 && x.size(1) > 0 && (x.stride(1) == 1 || x.size(1) == 1),
              "einshard norm: [rows, d] CUDA tensor");
  NormArgs a;
  a.dtype = code_of(x.scalar_type(), "norm");
  a.rows = x.size(0);
  a.d = x.size(1);
  a.x = x.data_ptr();
  a.ldx = x.stride(0);
  if (y.has_value()) {
    TORCH_CHECK(y->device() == x.device() && y->sizes() == x.sizes() && y->scalar_type() == x.scalar_type() &&
                    (y->stride(1) == 1 || y->size(1) == 1),
                "einshard norm: block output of the stream's shape and type");
    a.y = y->data_ptr();
    a.ldy = y->stride(0);
  }
  TORCH_CHECK(y.has_value() || (!post && !gate.has_value()), "einshard norm: a norm or gate of an absent block");
  norm_param(a.w, w, x, a.d, "weight");
  norm_param(a.b, b, x, a.d, "bias");
  norm_param(a.pw, pw, x, a.d, "post weight");
  norm_param(a.pb, pb, x, a.d, "post bias");
  TORCH_CHECK(post || (!pw.has_value() && !pb.has_value()), "einshard norm: post parameters without post");
  if (gate.has_value()) {
    TORCH_CHECK(gate_inner > 0 && gate_count > 0 && a.rows % (gate_inner * gate_count) == 0,
                "einshard norm: gate rows");
    norm_param(a.gate, gate, x, gate_count * a.d, "gate");
    a.gate_inner = gate_inner;
    a.gate_count = gate_count;
  }
  a.post = post;
  a.center = center;
  a.scale = static_cast<float>(scale);
  a.eps = static_cast<float>(eps);
  a.sms = sms_of(x);
  return a;
}

// (h, n, stats); h is undefined without a block output, stats unless kept
std::vector<Opt> norm_forward_op(const at::Tensor& x, const Opt& y, const Opt& w, const Opt& b, const Opt& pw,
                                 const Opt& pb, const Opt& gate, int64_t gate_inner, int64_t gate_count, bool post,
                                 bool center, double scale, double eps, bool keep) {
  const c10::cuda::CUDAGuard guard(x.device());
  const NormArgs a = norm_args(x, y, w, b, pw, pb, gate, gate_inner, gate_count, post, center, scale, eps);
  NormForward f;
  Opt h, stats;
  at::Tensor n = at::empty(x.sizes(), x.options());
  f.n = n.data_ptr();
  if (y.has_value()) {
    h = at::empty(x.sizes(), x.options());
    f.h = h->data_ptr();
  }
  if (keep) {
    stats = at::empty({x.size(0), 4}, x.options().dtype(at::kFloat));
    f.stats = stats->data_ptr<float>();
  }
  if (x.numel() > 0) counted(norm_forward(a, f, at::cuda::getCurrentCUDAStream()), "norm");
  return {h, n, stats};
}

// Gradients of x, y, w, b, pw, pb, gate (as `want` says) for those of h and n
std::vector<Opt> norm_backward_op(const Opt& dh, const Opt& dn, const at::Tensor& x, const Opt& y, const Opt& w,
                                  const Opt& b, const Opt& pw, const Opt& pb, const Opt& gate, int64_t gate_inner,
                                  int64_t gate_count, bool post, bool center, double scale, double eps,
                                  const at::Tensor& stats, const std::vector<bool>& want) {
  const c10::cuda::CUDAGuard guard(x.device());
  const NormArgs a = norm_args(x, y, w, b, pw, pb, gate, gate_inner, gate_count, post, center, scale, eps);
  TORCH_CHECK(want.size() == 7, "einshard norm: seven gradients");
  TORCH_CHECK(stats.device() == x.device() && stats.is_contiguous() && stats.scalar_type() == at::kFloat &&
                  stats.numel() == 4 * a.rows,
              "einshard norm: statistics of the forward pass");
  std::vector<Opt> out(7);
  const Opt given[7] = {x, y, w, b, pw, pb, gate};
  for (int i = 0; i < 7; ++i) {
    if (!want[i] || !given[i].has_value()) continue;
    out[i] = a.rows == 0 ? at::zeros(given[i]->sizes(), given[i]->options())
                         : at::empty(given[i]->sizes(), given[i]->options());
  }
  if (a.rows == 0) return out;
  for (const Opt& g : {dh, dn})
    TORCH_CHECK(!g.has_value() || (g->device() == x.device() && g->sizes() == x.sizes() && g->is_contiguous() &&
                                   g->scalar_type() == x.scalar_type()),
                "einshard norm: gradients of the stream's shape and type, contiguous");
  NormPlan plan = norm_plan(a);
  NormBackward g;
  NormSums s;
  g.dh = dh.has_value() ? dh->data_ptr() : nullptr;
  g.dn = dn.has_value() ? dn->data_ptr() : nullptr;
  g.stats = stats.data_ptr<float>();
  g.dx = out[0].has_value() ? out[0]->data_ptr() : nullptr;
  g.dy = out[1].has_value() ? out[1]->data_ptr() : nullptr;
  s.dw = out[2].has_value() ? out[2]->data_ptr() : nullptr;
  s.db = out[3].has_value() ? out[3]->data_ptr() : nullptr;
  s.dpw = out[4].has_value() ? out[4]->data_ptr() : nullptr;
  s.dpb = out[5].has_value() ? out[5]->data_ptr() : nullptr;
  at::Tensor products, ws, coef;
  if (out[6].has_value()) {
    if (plan.grouped) {
      s.dgate = out[6]->data_ptr();
    } else if (gate_count == a.rows) {
      g.dgate_rows = out[6]->data_ptr();
      g.dgate_f32 = a.gate.f32;
    } else {
      products = at::empty({a.rows, a.d}, x.options().dtype(at::kFloat));
      g.dgate_rows = products.data_ptr();
      g.dgate_f32 = 1;
    }
  }
  if (s.dw || s.db || s.dpw || s.dpb || s.dgate) {
    ws = at::empty({plan.units(), plan.sums(), plan.pitch(a.d)}, x.options().dtype(at::kFloat));
    g.ws = ws.data_ptr<float>();
  }
  if (!norm_in_registers(a)) {
    coef = at::empty({a.rows, 4}, x.options().dtype(at::kFloat));
    g.coef = coef.data_ptr<float>();
  }
  int launches = 0;
  const int rc = norm_backward(a, plan, g, s, at::cuda::getCurrentCUDAStream(), &launches);
  counted(rc, "norm backward", launches);
  if (products.defined()) {
    const int64_t outer = a.rows / (gate_inner * gate_count);
    out[6]->copy_(products.view({outer, gate_count, gate_inner, a.d}).sum(c10::IntArrayRef{0, 2}).view(out[6]->sizes()));
  }
  return out;
}

// A gradient that has no derivative of its own: under create_graph, using it further raises.
struct Final : public torch::autograd::Function<Final> {
  static at::Tensor forward(torch::autograd::AutogradContext*, const at::Tensor& t, const at::Tensor&) {
    return t.view_as(t);
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext*, torch::autograd::variable_list) {
    TORCH_CHECK(false, "einshard: trying to differentiate twice a function that was marked with once_differentiable");
  }
};

}  // namespace

int64_t capture_of(c10::DeviceIndex device) {
  cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
  unsigned long long id = 0;
  C10_CUDA_CHECK(cudaStreamGetCaptureInfo(at::cuda::getCurrentCUDAStream(device), &status, &id));
  return status == cudaStreamCaptureStatusNone ? 0 : static_cast<int64_t>(id);
}

at::Tensor plain(const at::Tensor& t) { return t.defined() && t.is_neg() ? t.resolve_neg() : t; }

void finalise(std::vector<at::Tensor>& grads, const std::vector<at::Tensor>& from) {
  if (!at::GradMode::is_enabled()) return;
  for (const at::Tensor& input : from) {
    if (!input.defined() || !input.requires_grad()) continue;
    for (at::Tensor& g : grads)
      if (g.defined()) g = Final::apply(g, input);
  }
}

namespace {

Opt some(const at::Tensor& t) { return t.defined() ? Opt(t) : Opt(); }
at::Tensor none(const Opt& t) { return t.has_value() ? *t : at::Tensor(); }

Opt plain_opt(const Opt& t) { return t.has_value() ? Opt(plain(*t)) : t; }

// [rows, d] of a tensor whose last axis is the row, with a unit stride.
at::Tensor rows_of(const at::Tensor& t) {
  if (!t.defined()) return t;
  const int64_t d = t.size(-1);
  at::Tensor r = t.dim() == 2 ? t : t.reshape({t.numel() / d, d});
  return r.stride(1) == 1 || d == 1 ? r : r.contiguous();
}

struct NormFunction : public torch::autograd::Function<NormFunction> {
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const at::Tensor& x,
                                                const Opt& y, const Opt& w, const Opt& b, const Opt& pw, const Opt& pb,
                                                const Opt& gate, int64_t inner, int64_t count, bool post, bool center, double scale,
                                                double eps) {
    const at::Tensor xr = rows_of(x), yr = rows_of(none(y));
    auto out = norm_forward_op(xr, some(yr), w, b, pw, pb, gate, inner, count, post, center, scale, eps, true);
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({x, none(y), none(w), none(b), none(pw), none(pb), none(gate), *out[2]});
    ctx->saved_data["conf"] = c10::ivalue::Tuple::create({inner, count, post, center, scale, eps});
    at::AutoDispatchBelowADInplaceOrView own;  // results of their own, not views
    if (!y.has_value()) return {out[1]->view(x.sizes())};
    return {out[0]->view(x.sizes()), out[1]->view(x.sizes())};
  }

  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list grads) {
    const auto s = ctx->get_saved_variables();
    const auto conf = ctx->saved_data["conf"].toTuple()->elements();
    at::Tensor dh = grads.size() == 2 ? grads[0] : at::Tensor(), dn = grads.back();
    torch::autograd::variable_list out(13);
    if (!dh.defined() && !dn.defined()) return out;
    std::vector<bool> want(7);
    size_t edge = 0;  // absent inputs have none
    for (size_t i = 0; i < 7; ++i) want[i] = s[i].defined() && ctx->needs_input_grad(edge++);
    std::vector<at::Tensor> found(7);
    {
      at::AutoDispatchBelowAutograd below;
      const at::Tensor xr = rows_of(s[0]), yr = rows_of(s[1]);
      auto whole = [&](const at::Tensor& g) {
        return g.defined() ? Opt(plain(g).reshape(xr.sizes()).contiguous()) : Opt();
      };
      auto got = norm_backward_op(whole(dh), whole(dn), xr, some(yr), some(s[2]), some(s[3]), some(s[4]),
                                  some(s[5]), some(s[6]), conf[0].toInt(), conf[1].toInt(), conf[2].toBool(),
                                  conf[3].toBool(), conf[4].toDouble(), conf[5].toDouble(), s[7], want);
      for (size_t i = 0; i < 7; ++i) {
        found[i] = none(got[i]);
        if (i < 2 && found[i].defined()) found[i] = found[i].view(s[0].sizes());
      }
    }
    finalise(found, grads);
    finalise(found, s);
    for (size_t i = 0; i < 7; ++i) out[i] = found[i];
    return out;
  }
};

// norm_forward on tensors whose last axis is normalised, with gradients: (h, n) or (n)
std::vector<at::Tensor> norm_op(const at::Tensor& x, const Opt& y, const Opt& w, const Opt& b, const Opt& pw,
                                const Opt& pb, const Opt& gate, int64_t inner, int64_t count, bool post, bool center,
                                double scale, double eps) {
  return NormFunction::apply(plain(x), plain_opt(y), plain_opt(w), plain_opt(b), plain_opt(pw), plain_opt(pb),
                             plain_opt(gate), inner, count, post, center, scale, eps);
}

// ------------------------------------------------------------------ policy loss

void per_token(const Opt& t, const at::Tensor& logits, int64_t count, at::ScalarType type, const char* name) {
  if (!t.has_value()) return;
  TORCH_CHECK(t->device() == logits.device() && t->is_contiguous() && t->numel() == count && t->scalar_type() == type,
              "einshard policy loss: ", name, " of ", count, " elements, contiguous, ", type);
}

PolicyArgs policy_args(const at::Tensor& logits, const at::Tensor& ids, const Opt& mask, const Opt& old,
                       const Opt& ref, const at::Tensor& adv, int64_t length, double lo, double hi, double kl,
                       double temperature, int64_t reduction, double weight) {
  TORCH_CHECK(logits.is_cuda() && logits.dim() == 2 && logits.size(1) > 0 &&
                  (logits.stride(1) == 1 || logits.size(1) == 1),
              "einshard policy loss: [tokens, vocabulary] CUDA logits");
  PolicyArgs a;
  a.dtype = code_of(logits.scalar_type(), "policy loss");
  a.logits = logits.data_ptr();
  a.tokens = logits.size(0);
  a.vocab = logits.size(1);
  a.ld = logits.stride(0);
  TORCH_CHECK(length > 0 && a.tokens % length == 0, "einshard policy loss: sequence length");
  a.length = length;
  per_token(ids, logits, a.tokens, at::kLong, "ids");
  per_token(mask, logits, a.tokens, at::kBool, "mask");
  per_token(old, logits, a.tokens, at::kFloat, "old log-probabilities");
  per_token(ref, logits, a.tokens, at::kFloat, "reference log-probabilities");
  const bool per_sequence = adv.numel() != a.tokens;
  per_token(adv, logits, per_sequence ? a.tokens / length : a.tokens, at::kFloat, "advantages");
  a.ids = ids.data_ptr<int64_t>();
  a.mask = mask.has_value() ? mask->data_ptr<bool>() : nullptr;
  a.old = old.has_value() ? old->data_ptr<float>() : nullptr;
  a.ref = ref.has_value() ? ref->data_ptr<float>() : nullptr;
  a.adv = adv.data_ptr<float>();
  a.adv_per_sequence = per_sequence;
  a.least = 1.0 - lo;
  a.most = 1.0 + hi;
  a.kl = kl;
  a.inv_temp = 1.0 / temperature;
  a.reduction = static_cast<int>(reduction);
  a.weight = static_cast<float>(weight);
  a.sms = sms_of(logits);
  return a;
}

PolicyState policy_state(const at::Tensor& terms, const at::Tensor& share) {
  PolicyState s;
  s.terms = reinterpret_cast<float4*>(terms.data_ptr<float>());
  s.share = share.data_ptr<float>();
  return s;
}

// (loss, KL, clipped share, logp, terms, token shares) and, with `gradient`, that of the logits and its factors
std::vector<at::Tensor> policy_forward_op(const at::Tensor& logits, const at::Tensor& ids, const Opt& mask,
                                          const Opt& old, const Opt& ref, const at::Tensor& adv, int64_t length,
                                          double lo, double hi, double kl, double temperature, int64_t reduction,
                                          double weight, bool gradient) {
  const c10::cuda::CUDAGuard guard(logits.device());
  const PolicyArgs a = policy_args(logits, ids, mask, old, ref, adv, length, lo, hi, kl, temperature, reduction, weight);
  const auto f32 = logits.options().dtype(at::kFloat);
  const int64_t sequences = a.tokens / length;
  TORCH_CHECK(a.tokens > 0, "einshard policy loss: no tokens");
  at::Tensor loss = at::empty({}, f32), kl_out = at::empty({}, f32), clipped = at::empty({}, f32);
  at::Tensor logp = at::empty({a.tokens}, f32), terms = at::empty({a.tokens, 4}, f32);
  at::Tensor shares = at::empty({sequences}, f32);
  at::Tensor sums = at::empty({3 * policy_sum_blocks(a.tokens) + 1}, f32.dtype(at::kDouble));
  PolicyState s = policy_state(terms, shares);
  s.logp = logp.data_ptr<float>();
  s.sums = reinterpret_cast<PolicySums*>(sums.data_ptr<double>());
  s.done = reinterpret_cast<unsigned*>(sums.data_ptr<double>() + 3 * policy_sum_blocks(a.tokens));
  s.loss = loss.data_ptr<float>();
  s.kl = kl_out.data_ptr<float>();
  s.clipped = clipped.data_ptr<float>();
  std::vector<at::Tensor> out{loss, kl_out, clipped, logp, terms, shares};
  if (gradient) {
    out.push_back(at::empty(logits.sizes(), logits.options()));
    out.push_back(at::empty({a.tokens}, f32));
    s.dlogits = out[6].data_ptr();
    s.factors = out[7].data_ptr<float>();
  }
  int launches = 0;
  const int rc = policy_forward(a, s, at::cuda::getCurrentCUDAStream(), &launches);
  counted(rc, "policy loss", launches);
  return out;
}

// The gradient of the logits; in `kept` (with its factors), which the forward pass wrote, or a new tensor.
at::Tensor policy_backward_op(const at::Tensor& grad, const at::Tensor& logits, const at::Tensor& ids,
                              const Opt& mask, const Opt& old, const Opt& ref, const at::Tensor& adv, int64_t length,
                              double lo, double hi, double kl, double temperature, int64_t reduction, double weight,
                              const at::Tensor& terms, const at::Tensor& shares,
                              const Opt& kept, const Opt& factors) {
  const c10::cuda::CUDAGuard guard(logits.device());
  const PolicyArgs a = policy_args(logits, ids, mask, old, ref, adv, length, lo, hi, kl, temperature, reduction, weight);
  TORCH_CHECK(grad.device() == logits.device() && grad.numel() == 1 && grad.scalar_type() == at::kFloat,
              "einshard policy loss: fp32 gradient of the loss");
  TORCH_CHECK(a.tokens > 0, "einshard policy loss: no tokens");
  per_token(terms, logits, 4 * a.tokens, at::kFloat, "terms");
  per_token(shares, logits, a.tokens / length, at::kFloat, "token shares");
  TORCH_CHECK(kept.has_value() == factors.has_value(), "einshard policy loss: a kept gradient has factors");
  per_token(kept, logits, a.tokens * a.vocab, logits.scalar_type(), "kept gradient");
  per_token(factors, logits, a.tokens, at::kFloat, "factors");
  at::Tensor out = kept.has_value() ? *kept : at::empty(logits.sizes(), logits.options());
  PolicyState s = policy_state(terms, shares);
  s.dlogits = out.data_ptr();
  s.factors = factors.has_value() ? factors->data_ptr<float>() : nullptr;
  counted(policy_backward(a, s, grad.data_ptr<float>(), at::cuda::getCurrentCUDAStream()), "policy loss backward");
  return out;
}

// The forward pass writes the gradient for an upstream gradient of 1 while it has the logits at hand; the first
// backward pass hands it out (formed again in place where the upstream gradient is another), later ones form their
// own.  A backward pass captured apart from its forward pass (in another graph, or one of the two eager) has its own
// too: a replay of the one would write under the other's result.  The buffer is no saved tensor: hooks that recompute
// or offload saved tensors do not see it.
struct PolicyFunction : public torch::autograd::Function<PolicyFunction> {
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const at::Tensor& logits,
                                                const at::Tensor& ids, const Opt& mask, const Opt& old, const Opt& ref,
                                                const at::Tensor& adv, int64_t length, double lo, double hi, double kl, double temperature, int64_t reduction,
                                                double weight) {
    const at::Tensor rows = rows_of(logits);
    auto r = policy_forward_op(rows, ids, mask, old, ref, adv, length, lo, hi, kl, temperature, reduction, weight, true);
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({logits, ids, none(mask), none(old), none(ref), adv, r[4], r[5]});
    ctx->saved_data["conf"] = c10::ivalue::Tuple::create({length, lo, hi, kl, temperature, reduction, weight});
    ctx->saved_data["kept"] = r[6];
    ctx->saved_data["factors"] = r[7];
    ctx->saved_data["capture"] = capture_of(logits.get_device());
    ctx->mark_non_differentiable({r[1], r[2], r[3]});
    return {r[0], r[1], r[2], r[3]};
  }

  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list grads) {
    torch::autograd::variable_list out(13);
    if (!grads[0].defined()) return out;
    const auto s = ctx->get_saved_variables();
    const auto conf = ctx->saved_data["conf"].toTuple()->elements();
    Opt kept, factors;
    if (ctx->saved_data.count("kept")) {
      if (ctx->saved_data["capture"].toInt() == capture_of(s[0].get_device())) {
        kept = ctx->saved_data["kept"].toTensor();
        factors = ctx->saved_data["factors"].toTensor();
      }
      ctx->saved_data.erase("kept");
      ctx->saved_data.erase("factors");
    }
    std::vector<at::Tensor> found(1);
    {
      at::AutoDispatchBelowAutograd below;
      found[0] = policy_backward_op(plain(grads[0]).contiguous(), rows_of(s[0]), s[1], some(s[2]), some(s[3]), some(s[4]), s[5],
                                    conf[0].toInt(), conf[1].toDouble(), conf[2].toDouble(), conf[3].toDouble(),
                                    conf[4].toDouble(), conf[5].toInt(), conf[6].toDouble(), s[6], s[7], kept,
                                    factors)
                     .view(s[0].sizes());
    }
    finalise(found, grads);
    finalise(found, s);
    out[0] = found[0];
    return out;
  }
};

// policy_forward on logits whose last axis is the vocabulary, with gradients: (loss, KL, clipped share, logp)
std::vector<at::Tensor> policy_op(const at::Tensor& logits, const at::Tensor& ids, const Opt& mask, const Opt& old,
                                  const Opt& ref, const at::Tensor& adv, int64_t length, double lo, double hi,
                                  double kl, double temperature, int64_t reduction, double weight) {
  return PolicyFunction::apply(logits, ids, mask, old, ref, adv, length, lo, hi, kl, temperature, reduction, weight);
}

}  // namespace

void bind_training_ops(pybind11::module_& m, std::atomic<long long>& launches) {
  g_count = &launches;
  m.def("quant8", &quant8_op, "(codes, exponents) of a [rows, d] tensor kept in 8 bits");
  m.def("quant8_silu", &quant8_silu_op, "(silu(h), codes, exponents) of an fp32 pre-activation");
  m.def("norm_forward", &norm_forward_op, "(h, n, statistics) of the norms around a block's residual");
  m.def("norm", &norm_op, "norm_forward with gradients", pybind11::call_guard<pybind11::gil_scoped_release>());
  m.def("policy", &policy_op, "policy_forward with gradients", pybind11::call_guard<pybind11::gil_scoped_release>());
  m.def("policy_forward", &policy_forward_op, "clipped policy loss of token logits, with what its gradient needs");
  m.def("capture_of", &capture_of, "number of the capture on the device's current stream, or 0");
  m.def("restore8", &restore8_op, "what 8-bit codes stand for, its silu, or grad * silu'");
}

}  // namespace es
