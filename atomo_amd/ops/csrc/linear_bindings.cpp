// Binding of the fused linear layer (linear_kernels.hip) with its autograd
// node.

#include <torch/extension.h>

#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPException.h>
#include <c10/hip/HIPStream.h>

#include <algorithm>

#include "linear_kernels.h"
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
    default: TORCH_CHECK(false, "x must be fp32, bf16 or fp16");
  }
}

void check_matrix(const Tensor& t, const Tensor& x, int64_t rows,
                  int64_t columns, const char* name) {
  TORCH_CHECK(t.device() == x.device(), name, " must be on x's device");
  TORCH_CHECK(t.scalar_type() == x.scalar_type(), name, " must have x's type");
  TORCH_CHECK(t.dim() == 2 && t.size(0) == rows && t.size(1) == columns, name,
              " must be (", rows, ", ", columns, ")");
  TORCH_CHECK(columns == 1 || t.stride(1) == 1, name,
              " must have contiguous rows");
}

// a row's stride means nothing where there is one row
int64_t row_stride(const Tensor& t) {
  return t.size(0) > 1 ? t.stride(0) : t.size(1);
}

// fp32 numbers that a planned product needs to put its parts
int64_t parts_of(const AtomoProduct& a) {
  return a.splits > 1 ? a.splits * a.nj * a.ld_part : 0;
}

Tensor floats(int64_t n, const Tensor& like) {
  return n ? torch::empty({n}, like.options().dtype(torch::kFloat32)) : Tensor();
}

void product(const AtomoProduct& a) {
  atomo_product_launch(&a, cur_stream());
  C10_HIP_KERNEL_LAUNCH_CHECK();
}

struct LinearAct : public torch::autograd::Function<LinearAct> {
  // `train`: a gradient may be asked for, so the slope is kept
  static Tensor forward(AutogradContext* ctx, const Tensor& x,
                        const Tensor& weight,
                        const c10::optional<Tensor>& bias_opt,
                        const c10::optional<Tensor>& residual_opt, int64_t act,
                        bool train) {
    const Tensor bias = bias_opt.value_or(Tensor());
    const Tensor residual = residual_opt.value_or(Tensor());
    TORCH_CHECK(x.is_cuda(), "x must be a CUDA (ROCm) tensor");
    TORCH_CHECK(x.dim() == 2 && weight.dim() == 2, "x and weight must be 2-d");
    const int64_t m = x.size(0), k = x.size(1), n = weight.size(0);
    const int64_t most = (int64_t)1 << 30;
    TORCH_CHECK(m <= most && k <= most && n <= most && k >= 1 && n >= 1,
                "x and weight have a size that is not supported");
    check_matrix(x, x, m, k, "x");
    check_matrix(weight, x, n, k, "weight");
    if (bias.defined()) check_matrix(bias.unsqueeze(0), x, 1, n, "bias");
    if (residual.defined()) check_matrix(residual, x, m, n, "residual");
    const c10::DeviceGuard guard(x.device());
    Tensor y = torch::empty({m, n}, x.options());
    // relu's slope can be seen from its output, unless a residual is added
    const bool by_output = act == ATOMO_ACT_RELU && !residual.defined();
    Tensor slope;
    if (train && act != ATOMO_ACT_NONE && !by_output)
      slope = torch::empty({m, n}, x.options().dtype(torch::kFloat32));
    if (m > 0) {
      AtomoProduct a{};
      a.p = weight.data_ptr();
      a.q = x.data_ptr();
      a.out = y.data_ptr();
      a.bias = bias.defined() ? bias.data_ptr() : nullptr;
      a.residual = residual.defined() ? residual.data_ptr() : nullptr;
      a.slope = slope.defined() ? slope.data_ptr() : nullptr;
      a.ldp = row_stride(weight);
      a.ldq = row_stride(x);
      a.ldo = n;
      a.ldr = residual.defined() ? row_stride(residual) : 0;
      a.ni = (int)n;
      a.nj = (int)m;
      a.nk = (int)k;
      a.type = type_of(x);
      a.form = ATOMO_FORWARD;
      a.act = (int)act;
      atomo_product_plan(&a);
      const Tensor partial = floats(parts_of(a), x);
      a.partial = partial.defined() ? partial.data_ptr<float>() : nullptr;
      product(a);
    }
    ctx->saved_data["train"] = train;
    ctx->saved_data["bias"] = bias.defined();
    ctx->saved_data["residual"] = residual.defined();
    if (train) {
      ctx->save_for_backward({x, weight, by_output ? y : slope});
      ctx->saved_data["by_output"] = by_output;
    }
    return y;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    TORCH_CHECK(!c10::GradMode::is_enabled(),
                "linear_act has no second derivative (create_graph)");
    // tensors that were not given have no edge: the others move up
    const bool has_bias = ctx->saved_data["bias"].toBool();
    const Tensor dr =
        ctx->saved_data["residual"].toBool() ? grads[0] : Tensor();
    if (!ctx->saved_data["train"].toBool())  // the residual alone asks
      return {Tensor(), Tensor(), Tensor(), dr, Tensor(), Tensor()};
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &weight = saved[1], &slope = saved[2];
    const c10::DeviceGuard guard(x.device());
    const int64_t m = x.size(0), k = x.size(1), n = weight.size(0);
    const int type = type_of(x);
    Tensor dy = grads[0];
    if (n > 1 && dy.stride(1) != 1) dy = dy.contiguous();
    const bool want_x = ctx->needs_input_grad(0);
    const bool want_w = ctx->needs_input_grad(1);
    const bool want_b = has_bias && ctx->needs_input_grad(2);
    Tensor dx, dw, db;
    if (m == 0) {
      if (want_x) dx = torch::empty_like(x);
      if (want_w) dw = torch::zeros({n, k}, x.options());
      if (want_b) db = torch::zeros({n}, x.options());
      return {dx, dw, db, dr, Tensor(), Tensor()};
    }
    // What the three steps need in between lies in one piece of memory, in
    // turn: the products' parts and db's block sums.
    const bool make_dp = slope.defined() && (want_x || want_w);
    Tensor dp = make_dp ? torch::empty({m, n}, x.options()) : dy;
    AtomoProduct px{}, pw{};
    int64_t work = 0;
    if (want_x) {
      dx = torch::empty({m, k}, x.options());
      px.p = weight.data_ptr();
      px.ldp = row_stride(weight);
      px.q = dp.data_ptr();
      px.ldq = row_stride(dp);
      px.out = dx.data_ptr();
      px.ldo = k;
      px.form = ATOMO_GRAD_X;
      px.type = type;
      px.ni = (int)k;
      px.nj = (int)m;
      px.nk = (int)n;
      atomo_product_plan(&px);
      work = std::max(work, parts_of(px));
    }
    if (want_w) {
      dw = torch::empty({n, k}, x.options());
      pw.p = x.data_ptr();
      pw.ldp = row_stride(x);
      pw.q = dp.data_ptr();
      pw.ldq = row_stride(dp);
      pw.out = dw.data_ptr();
      pw.ldo = k;
      pw.form = ATOMO_GRAD_W;
      pw.type = type;
      pw.ni = (int)k;
      pw.nj = (int)n;
      pw.nk = (int)m;
      atomo_product_plan(&pw);
      work = std::max(work, parts_of(pw));
    }
    AtomoLinearDp d{};
    // blocks of 128 rows (8 for each of 16 waves) or more, 1024 at most
    d.block_rows = (int)std::max<int64_t>(128, (m + 1023) / 1024);
    d.row_blocks = (int)((m + d.block_rows - 1) / d.block_rows);
    if (want_b && d.row_blocks > 1) work = std::max(work, d.row_blocks * n);
    const Tensor between = floats(work, x);
    float* partial = between.defined() ? between.data_ptr<float>() : nullptr;

    if (make_dp || want_b) {
      if (want_b) db = torch::empty({n}, x.options());
      d.dy = dy.data_ptr();
      d.ld_dy = row_stride(dy);
      d.slope = slope.defined() ? slope.data_ptr() : nullptr;
      d.by_output = ctx->saved_data["by_output"].toBool();
      d.dp = make_dp ? dp.data_ptr() : nullptr;
      d.db = want_b ? db.data_ptr() : nullptr;
      d.partial = partial;
      d.rows = (int)m;
      d.columns = (int)n;
      d.type = type;
      atomo_linear_dp_launch(&d, cur_stream());
      C10_HIP_KERNEL_LAUNCH_CHECK();
    }
    if (want_x) {
      px.partial = partial;
      product(px);
    }
    if (want_w) {
      pw.partial = partial;
      product(pw);
    }
    return {dx, dw, db, dr, Tensor(), Tensor()};
  }
};

Tensor linear_act(const Tensor& x, const Tensor& weight,
                  const c10::optional<Tensor>& bias,
                  const c10::optional<Tensor>& residual, int64_t act) {
  const auto wants = [](const c10::optional<Tensor>& t) {
    return t.has_value() && t->defined() && t->requires_grad();
  };
  const bool train =
      c10::GradMode::is_enabled() &&
      (x.requires_grad() || weight.requires_grad() || wants(bias));
  return LinearAct::apply(x, weight, bias, residual, act, train);
}

}  // namespace

void register_linear_ops(pybind11::module& m) {
  namespace py = pybind11;
  m.def("linear_act", &linear_act, py::call_guard<py::gil_scoped_release>(),
        "act(x W^T + b) + residual (differentiable)");
}
