// Bindings of the kernels on logits (logit_kernels.hip), with the autograd
// node of the distillation loss.  The Python side (logit_ops.py) checks the
// arguments' meaning; here are the checks that the kernels rely on.

#include <torch/extension.h>

#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPException.h>
#include <c10/hip/HIPStream.h>

#include <limits>
#include <tuple>

#include "logit_kernels.h"
#include "op_bindings.h"

namespace {

using torch::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

hipStream_t cur_stream() { return c10::hip::getCurrentHIPStream().stream(); }

int type_of(const Tensor& t) {
  switch (t.scalar_type()) {
    case torch::kFloat32: return ATOMO_F32;
    case torch::kBFloat16: return ATOMO_BF16;
    case torch::kFloat16: return ATOMO_F16;
    default: TORCH_CHECK(false, "logits must be fp32, bf16 or fp16");
  }
}

void check_logits(const Tensor& z) {
  TORCH_CHECK(z.is_cuda(), "logits must be a CUDA (ROCm) tensor");
  TORCH_CHECK(z.dim() == 2 && z.size(1) >= 1, "logits must be (rows, classes)");
  TORCH_CHECK(z.size(1) == 1 || z.stride(1) == 1,
              "the classes of a row must be contiguous");
  TORCH_CHECK(z.size(1) < std::numeric_limits<int32_t>::max(),
              "too many classes");
  TORCH_CHECK(z.stride(0) >= 0, "logits must not have a negative stride");
}

void check_rows(const Tensor& t, const Tensor& z, torch::ScalarType type,
                const char* name) {
  TORCH_CHECK(t.device() == z.device(), name, " must be on the logits' device");
  TORCH_CHECK(t.scalar_type() == type, name, " has a wrong type");
  TORCH_CHECK(t.is_contiguous(), name, " must be contiguous");
  TORCH_CHECK(t.dim() >= 1 && t.size(0) == z.size(0), name,
              " must have one row for each row of logits");
}

const int64_t* labels_of(const Tensor& labels, const Tensor& z) {
  if (!labels.defined()) return nullptr;
  check_rows(labels, z, torch::kInt64, "labels");
  TORCH_CHECK(labels.dim() == 1, "labels must be (rows)");
  return labels.data_ptr<int64_t>();
}

std::tuple<Tensor, Tensor, Tensor, Tensor> label_logprobs(
    const Tensor& z, const c10::optional<Tensor>& labels_opt, int64_t top,
    int64_t ignore) {
  check_logits(z);
  const Tensor labels = labels_opt.value_or(Tensor());
  const c10::DeviceGuard guard(z.device());
  const int64_t* y = labels_of(labels, z);
  const int64_t rows = z.size(0), classes = z.size(1);
  TORCH_CHECK(top >= 0 && top <= ATOMO_LOGIT_TOP_MAX && top <= classes,
              "top must lie in 0..min(classes, ", ATOMO_LOGIT_TOP_MAX, ")");
  const auto f32 = z.options().dtype(torch::kFloat32);
  Tensor logprob = y ? torch::empty({rows}, f32) : Tensor();
  Tensor entropy = torch::empty({rows}, f32);
  Tensor top_logprob = torch::empty({rows, top}, f32);
  Tensor top_index = torch::empty({rows, top}, f32.dtype(torch::kInt64));
  if (rows > 0) {
    atomo_label_logprobs_launch(
        z.data_ptr(), type_of(z), z.stride(0), rows, (int)classes, y, ignore,
        (int)top, y ? logprob.data_ptr<float>() : nullptr,
        entropy.data_ptr<float>(), top_logprob.data_ptr<float>(),
        top_index.data_ptr<int64_t>(), cur_stream());
    C10_HIP_KERNEL_LAUNCH_CHECK();
  }
  return {logprob, entropy, top_logprob, top_index};
}

enum Reduction { kNone = 0, kMean = 1, kSum = 2 };

struct DistillLoss : public torch::autograd::Function<DistillLoss> {
  static Tensor forward(AutogradContext* ctx, const Tensor& z,
                        const Tensor& values, const Tensor& index,
                        const c10::optional<Tensor>& labels_opt, double tau,
                        double weight, int64_t ignore, int64_t reduction) {
    const Tensor labels = labels_opt.value_or(Tensor());
    check_logits(z);
    check_rows(values, z, torch::kFloat32, "teacher_value");
    check_rows(index, z, torch::kInt64, "teacher_index");
    TORCH_CHECK(values.dim() == 2 && index.sizes() == values.sizes() &&
                    values.size(1) <= ATOMO_LOGIT_TOP_MAX,
                "teacher_value and teacher_index must be (rows, k) with k <= ",
                ATOMO_LOGIT_TOP_MAX);
    const c10::DeviceGuard guard(z.device());
    const int64_t* y = labels_of(labels, z);
    const int64_t rows = z.size(0);
    // without the teacher's weight its entries are not looked at
    const int k = weight == 0.0 ? 0 : (int)values.size(1);
    const auto f32 = z.options().dtype(torch::kFloat32);
    Tensor row_loss = torch::empty({rows}, f32);
    Tensor stats = torch::empty({rows, 3}, f32);
    Tensor inverse;  // one over the counted rows, where labels decide them
    double factor = 1.0;
    if (reduction == kMean) {
      if (y)
        inverse = torch::empty({1}, f32);
      else
        factor = 1.0 / (double)std::max<int64_t>(rows, 1);
    }
    Tensor loss = reduction == kNone ? row_loss : torch::empty({}, f32);
    const hipStream_t stream = cur_stream();
    float* inv = inverse.defined() ? inverse.data_ptr<float>() : nullptr;
    if (inv) {
      atomo_distill_count_launch(y, rows, ignore, inv, stream);
      C10_HIP_KERNEL_LAUNCH_CHECK();
    }
    if (rows > 0) {
      atomo_distill_loss_launch(
          z.data_ptr(), type_of(z), z.stride(0), rows, (int)z.size(1),
          values.data_ptr<float>(), index.data_ptr<int64_t>(), k, y, ignore,
          (float)tau, (float)weight, row_loss.data_ptr<float>(),
          stats.data_ptr<float>(), stream);
      C10_HIP_KERNEL_LAUNCH_CHECK();
    }
    if (reduction != kNone) {
      atomo_distill_sum_launch(row_loss.data_ptr<float>(), rows, inv,
                               (float)factor, loss.data_ptr<float>(), stream);
      C10_HIP_KERNEL_LAUNCH_CHECK();
    }
    ctx->save_for_backward({z, values, index, labels, stats, inverse});
    ctx->saved_data["tau"] = tau;
    ctx->saved_data["weight"] = weight;
    ctx->saved_data["ignore"] = ignore;
    ctx->saved_data["k"] = (int64_t)k;
    ctx->saved_data["factor"] = factor;
    ctx->saved_data["per_row"] = reduction == kNone;
    return loss;
  }

  static variable_list backward(AutogradContext* ctx, variable_list up_list) {
    TORCH_CHECK(!c10::GradMode::is_enabled(),
                "distill_loss has no second derivative (create_graph)");
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &z = saved[0], &labels = saved[3], &inverse = saved[5];
    const c10::DeviceGuard guard(z.device());
    const int64_t rows = z.size(0);
    const bool per_row = ctx->saved_data["per_row"].toBool();
    const Tensor up = up_list[0].to(torch::kFloat32).contiguous();
    Tensor grad = torch::empty({rows, z.size(1)}, z.options());
    if (rows > 0) {
      atomo_distill_grad_launch(
          z.data_ptr(), type_of(z), z.stride(0), rows, (int)z.size(1),
          saved[1].data_ptr<float>(), saved[2].data_ptr<int64_t>(),
          (int)ctx->saved_data["k"].toInt(), labels_of(labels, z),
          ctx->saved_data["ignore"].toInt(),
          (float)ctx->saved_data["tau"].toDouble(),
          (float)ctx->saved_data["weight"].toDouble(),
          saved[4].data_ptr<float>(), up.data_ptr<float>(), per_row,
          inverse.defined() ? inverse.data_ptr<float>() : nullptr,
          (float)ctx->saved_data["factor"].toDouble(), grad.data_ptr(),
          cur_stream());
      C10_HIP_KERNEL_LAUNCH_CHECK();
    }
    return {grad, Tensor(), Tensor(), Tensor(), Tensor(),
            Tensor(), Tensor(), Tensor()};
  }
};

Tensor distill_loss(const Tensor& z, const Tensor& values, const Tensor& index,
                    const c10::optional<Tensor>& labels, double tau,
                    double weight, int64_t ignore, int64_t reduction) {
  return DistillLoss::apply(z, values, index, labels, tau, weight, ignore,
                            reduction);
}

}  // namespace

void register_logit_ops(pybind11::module& m) {
  namespace py = pybind11;
  m.attr("LOGIT_TOP_MAX") = ATOMO_LOGIT_TOP_MAX;
  m.def("label_logprobs", &label_logprobs,
        py::call_guard<py::gil_scoped_release>(),
        "log probability of a class, entropy and top alternatives of each row");
  m.def("distill_loss", &distill_loss,
        py::call_guard<py::gil_scoped_release>(),
        "distillation from a teacher's top logits (differentiable)");
}
