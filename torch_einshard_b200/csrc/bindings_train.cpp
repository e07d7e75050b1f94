// Torch bindings of the training-step operators around the contractions:
// activations kept in 8 bits (quant8.h).
#include "bindings_train.h"

#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include "gemm.h"
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

// What the codes stand for, its silu, or grad times its silu' (mode 0, 1, 2)
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

}  // namespace

void bind_training_ops(pybind11::module_& m, std::atomic<long long>& launches) {
  g_count = &launches;
  m.def("quant8", &quant8_op, "(codes, exponents) of a [rows, d] tensor kept in 8 bits");
  m.def("quant8_silu", &quant8_silu_op, "(silu(h), codes, exponents) of an fp32 pre-activation");
  m.def("restore8", &restore8_op, "what 8-bit codes stand for, its silu, or grad * silu'");
}

}  // namespace es
