// Bindings of the kernels on logits (logit_kernels.hip), with the autograd
// node of the distillation loss.  The Python side (logit_ops.py) checks the
// arguments' meaning; here are the checks that the kernels rely on.

#include <torch/extension.h>

#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPException.h>
#include <c10/hip/HIPStream.h>

#include <algorithm>
#include <limits>
#include <tuple>

#include "logit_kernels.h"
#include "op_bindings.h"

namespace {

using torch::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

hipStream_t cur_stream() { return c10::hip::getCurrentHIPStream().stream(); }

// the capture that a stream's work goes to, 0 for none
int64_t capture_of(hipStream_t stream) {
  hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
  unsigned long long id = 0;
  C10_HIP_CHECK(hipStreamGetCaptureInfo(stream, &status, &id));
  return status == hipStreamCaptureStatusNone ? 0 : (int64_t)id;
}

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
  TORCH_CHECK(z.size(1) <= (int64_t)1 << 30, "more than 2^30 classes");
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
    AtomoLogprobs a{};
    a.logits = z.data_ptr();
    a.labels = y;
    a.logprob = y ? logprob.data_ptr<float>() : nullptr;
    a.entropy = entropy.data_ptr<float>();
    a.top_logprob = top_logprob.data_ptr<float>();
    a.top_index = top_index.data_ptr<int64_t>();
    a.row_stride = z.stride(0);
    a.rows = rows;
    a.ignore = ignore;
    a.type = type_of(z);
    a.classes = (int)classes;
    a.top = (int)top;
    a.splits = atomo_logit_splits(rows, a.classes, a.type, &a.part_size);
    Tensor part_stat, part_keys;
    if (a.splits > 1) {
      part_stat = torch::empty({rows, a.splits, 3}, f32);
      part_keys = torch::empty({rows, a.splits, top}, top_index.options());
      a.part_stat = part_stat.data_ptr<float>();
      a.part_keys = part_keys.data_ptr<int64_t>();
    }
    atomo_label_logprobs_launch(&a, cur_stream());
    C10_HIP_KERNEL_LAUNCH_CHECK();
  }
  return {logprob, entropy, top_logprob, top_index};
}

enum Reduction { kNone = 0, kMean = 1, kSum = 2 };

struct DistillLoss : public torch::autograd::Function<DistillLoss> {
  // `wanted`: a gradient may be asked for
  static Tensor forward(AutogradContext* ctx, const Tensor& z,
                        const Tensor& values, const Tensor& index,
                        const c10::optional<Tensor>& labels_opt, double tau,
                        double weight, int64_t ignore, int64_t reduction,
                        bool wanted) {
    const Tensor labels = labels_opt.value_or(Tensor());
    check_logits(z);
    check_rows(values, z, torch::kFloat32, "teacher_value");
    check_rows(index, z, torch::kInt64, "teacher_index");
    TORCH_CHECK(values.dim() == 2 && index.sizes() == values.sizes() &&
                    values.size(1) <= ATOMO_LOGIT_TOP_MAX,
                "teacher_value and teacher_index must be (rows, k) with k <= ",
                ATOMO_LOGIT_TOP_MAX);
    const c10::DeviceGuard guard(z.device());
    const hipStream_t stream = cur_stream();
    const int64_t rows = z.size(0);
    const auto f32 = z.options().dtype(torch::kFloat32);

    AtomoDistill a{};
    a.labels = labels_of(labels, z);
    share(a, weight);
    // without the teacher's weight its entries are not looked at
    a.k = weight == 0.0 ? 0 : (int)values.size(1);
    a.tau = weight == 0.0 ? 1.f : (float)tau;
    a.inv_tau = 1.f / a.tau;
    a.ignore = ignore;
    a.factor = 1.f;
    if (a.labels == nullptr || weight == 1.0)
      a.mode = ATOMO_DISTILL_SOFT;
    else if (a.tau == 1.f)
      a.mode = ATOMO_DISTILL_TAU1;
    else if (a.tau == 2.f)
      a.mode = ATOMO_DISTILL_TAU2;
    else if (a.tau == 4.f)
      a.mode = ATOMO_DISTILL_TAU4;
    else
      a.mode = ATOMO_DISTILL_ANY;
    Tensor inverse;  // one over the counted rows
    if (reduction == kMean && a.labels) {
      a.count = rows <= ATOMO_LOGIT_COUNT_ROWS;
      if (!a.count) {
        inverse = torch::empty({1}, f32);
        atomo_distill_count_launch(a.labels, rows, ignore,
                                   inverse.data_ptr<float>(), stream);
        C10_HIP_KERNEL_LAUNCH_CHECK();
      }
    } else if (reduction == kMean) {
      a.factor = 1.f / (float)std::max<int64_t>(rows, 1);
    }
    describe(a, z, values, index, inverse);

    const bool fits = atomo_distill_fits(rows, a.classes, a.type);
    // The gradient of a mean or a sum is written along with the loss, for an
    // upstream gradient of 1; the backward pass writes it anew where that is
    // not so.  Not in fp16: a scaled loss is the rule there, as its smallest
    // steps lose most of an unscaled gradient.
    const bool fused = wanted && fits && reduction != kNone &&
                       z.scalar_type() != torch::kFloat16;
    // one read of a short row by one wave; long ones are swept
    const bool in_registers = fused || atomo_distill_short(a.classes, a.type);
    if (in_registers) {
      a.splits = 1;
    } else {
      a.splits = atomo_logit_splits(rows, a.classes, a.type, &a.part_size);
    }
    Tensor row_loss = torch::empty({rows}, f32);
    Tensor stats = torch::empty({rows, a.splits, 3}, f32);
    Tensor loss = reduction == kNone ? row_loss : torch::empty({}, f32);
    Tensor grad;
    a.row_loss = row_loss.data_ptr<float>();
    a.stats = stats.data_ptr<float>();
    if (fused) {
      grad = torch::empty({rows, z.size(1)}, z.options());
      a.grad = grad.data_ptr();
    }
    if (rows > 0) {
      if (in_registers)
        atomo_distill_fused_launch(&a, stream);
      else
        atomo_distill_loss_launch(&a, stream);
      C10_HIP_KERNEL_LAUNCH_CHECK();
    }
    if (reduction != kNone) {
      atomo_distill_sum_launch(&a, loss.data_ptr<float>(), stream);
      C10_HIP_KERNEL_LAUNCH_CHECK();
    }
    if (wanted) {
      ctx->save_for_backward({z, values, index, labels, stats, inverse});
      auto& d = ctx->saved_data;
      d["tau"] = (double)a.tau;
      d["weight"] = weight;
      d["ignore"] = ignore;
      d["factor"] = (double)a.factor;
      d["k"] = (int64_t)a.k;
      d["mode"] = (int64_t)a.mode;
      d["splits"] = (int64_t)a.splits;
      d["count"] = a.count != 0;
      d["per_row"] = reduction == kNone;
      if (fused) {
        d["grad"] = grad;
        d["capture"] = capture_of(stream);
      }
    }
    return loss;
  }

  // The shares of teacher and labels, each rounded by itself: 1 minus a rounded
  // weight would be off by 2^-25, however little is left.  Neither becomes 0.
  static void share(AtomoDistill& a, double weight) {
    a.weight = weight > 0.0 ? std::max((float)weight,
                                       std::numeric_limits<float>::min())
                            : 0.f;
    a.rest = (float)(1.0 - weight);
  }

  static void describe(AtomoDistill& a, const Tensor& z, const Tensor& values,
                       const Tensor& index, const Tensor& inverse) {
    a.logits = z.data_ptr();
    a.values = values.data_ptr<float>();
    a.index = index.data_ptr<int64_t>();
    a.inverse = inverse.defined() ? inverse.data_ptr<float>() : nullptr;
    a.row_stride = z.stride(0);
    a.rows = z.size(0);
    a.type = type_of(z);
    a.classes = (int)z.size(1);
  }

  static variable_list backward(AutogradContext* ctx, variable_list up_list) {
    TORCH_CHECK(!c10::GradMode::is_enabled(),
                "distill_loss has no second derivative (create_graph)");
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &z = saved[0], &labels = saved[3], &stats = saved[4];
    const c10::DeviceGuard guard(z.device());
    auto& d = ctx->saved_data;
    const Tensor up = up_list[0].to(torch::kFloat32).contiguous();
    AtomoDistill a{};
    a.labels = labels_of(labels, z);
    share(a, d["weight"].toDouble());
    a.k = (int)d["k"].toInt();
    a.tau = (float)d["tau"].toDouble();
    a.inv_tau = 1.f / a.tau;
    a.ignore = d["ignore"].toInt();
    a.factor = (float)d["factor"].toDouble();
    a.mode = (int)d["mode"].toInt();
    a.splits = (int)d["splits"].toInt();
    a.count = d["count"].toBool();
    describe(a, z, saved[1], saved[2], saved[5]);
    a.stats = stats.data_ptr<float>();
    a.up = up.data_ptr<float>();
    a.up_per_row = d["per_row"].toBool();
    const hipStream_t stream = cur_stream();
    // The gradient that the forward pass wrote is given away once; a further
    // backward pass makes its own.  So does one that is captured apart from
    // the forward pass: its graph may be replayed more than once for each.
    Tensor grad;
    const auto found = d.find("grad");
    if (found != d.end() && d["capture"].toInt() == capture_of(stream)) {
      grad = found->second.toTensor();
      d.erase(found);
      a.skip_one = 1;
    } else {
      grad = torch::empty({z.size(0), z.size(1)}, z.options());
    }
    a.grad = grad.data_ptr();
    a.grad_splits =
        atomo_logit_splits(z.size(0), a.classes, a.type, &a.grad_part);
    if (z.size(0) > 0) {
      atomo_distill_grad_launch(&a, stream);
      C10_HIP_KERNEL_LAUNCH_CHECK();
    }
    return {grad,     Tensor(), Tensor(), Tensor(), Tensor(),
            Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

Tensor distill_loss(const Tensor& z, const Tensor& values, const Tensor& index,
                    const c10::optional<Tensor>& labels, double tau,
                    double weight, int64_t ignore, int64_t reduction) {
  const bool wanted = c10::GradMode::is_enabled() && z.requires_grad();
  return DistillLoss::apply(z, values, index, labels, tau, weight, ignore,
                            reduction, wanted);
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
