// Python bindings for the atomo_amd gfx950 kernels (atomo_kernels.hip).
// Compiled as C++ with the torch extension glue; kernel launches are the
// extern "C" functions in the .hip translation unit.

#include <torch/extension.h>

#include <c10/hip/HIPStream.h>
#include <hip/hip_runtime_api.h>
#include <rocblas/rocblas.h>
#include <rocsolver/rocsolver.h>

#include <cstdint>

#include "op_bindings.h"

extern "C" {
void atomo_qsgd_pack_launch(const float*, float*, uint32_t*, int64_t, int, int,
                            bool, uint64_t, int, int, hipStream_t);
void atomo_qsgd_unpack_acc_launch(const float*, const uint32_t*, float*,
                                  int64_t, int, int, int, int, hipStream_t);
void atomo_svd_decode_acc_launch(const float*, float*, int, int64_t, int, int,
                                 int, hipStream_t);
void atomo_fused_sgd_launch(float*, const float*, float*, int64_t, float,
                            float, float, bool, float, float, const float*,
                            hipStream_t);
void atomo_fused_adam_launch(float*, const float*, float*, float*, float*,
                             int64_t, float, float, float, float, float,
                             float, float, float, hipStream_t);
void atomo_svd_decode_batched_launch(const float*, int64_t, int, float*,
                                     const int64_t*, const int32_t*, int,
                                     hipStream_t);
void atomo_qsgd_pack_batched_launch(const float*, float*, const int64_t*,
                                    const int32_t*, int, int, int, bool,
                                    const unsigned long long*, hipStream_t);
void atomo_qsgd_unpack_batched_launch(const float*, float*, const int64_t*,
                                      const int32_t*, int, int, int,
                                      hipStream_t);
void atomo_batched_gram_launch(const float*, float*, const int64_t*,
                               const int32_t*, int, hipStream_t);
void atomo_batched_sel_launch(const float*, float*, const float*,
                              const int64_t*, const int32_t*, int, int,
                              hipStream_t);
void atomo_jacobi_dense_launch(float*, float*, int, int, int, hipStream_t);
void atomo_jacobi_eigh_launch(float*, float*, const int64_t*, const int64_t*,
                              const int32_t*, int, int, float*,
                              const int64_t*, int, int, hipStream_t);
void atomo_jacobi_eigh_big_launch(float*, float*, float*, const int64_t*,
                                  const int64_t*, const int32_t*,
                                  const int64_t*, int, hipStream_t);
void atomo_build_stage_launch(const float*, const float*, const float*,
                              float*, const int64_t*, const int64_t*, int,
                              hipStream_t);
void atomo_sample_stage_launch(const float*, const float*, float*,
                               const int64_t*, const int64_t*, int, int, int,
                               const unsigned long long*,
                               unsigned long long*, hipStream_t);
}

namespace {

void check_f32_cuda(const torch::Tensor& t, const char* name) {
  TORCH_CHECK(t.is_cuda(), name, " must be a CUDA (ROCm) tensor");
  TORCH_CHECK(t.scalar_type() == torch::kFloat32, name, " must be fp32");
  TORCH_CHECK(t.is_contiguous(), name, " must be contiguous");
}

hipStream_t cur_stream() {
  return c10::hip::getCurrentHIPStream().stream();
}

void qsgd_pack(torch::Tensor grad, torch::Tensor region, int64_t bucket_size,
               int64_t qlevel, bool terngrad, int64_t seed) {
  check_f32_cuda(grad, "grad");
  check_f32_cuda(region, "region");
  const int64_t numel = grad.numel();
  const int bits = 1 + (int)qlevel;
  const int epw = 32 / bits;
  const int nb = (int)((numel + bucket_size - 1) / bucket_size);
  const int wpb = (int)((bucket_size + epw - 1) / epw);
  TORCH_CHECK(region.numel() >= nb + (int64_t)nb * wpb, "region too small");
  TORCH_CHECK(bucket_size <= 8192, "bucket_size too large for LDS staging");
  float* norms = region.data_ptr<float>();
  uint32_t* packed = reinterpret_cast<uint32_t*>(norms + nb);
  atomo_qsgd_pack_launch(grad.data_ptr<float>(), norms, packed, numel,
                         (int)bucket_size, (int)qlevel, terngrad,
                         (uint64_t)seed, nb, wpb, cur_stream());
}

void qsgd_unpack_acc(torch::Tensor region, torch::Tensor out, int64_t numel,
                     int64_t bucket_size, int64_t qlevel) {
  check_f32_cuda(region, "region");
  check_f32_cuda(out, "out");
  const int bits = 1 + (int)qlevel;
  const int epw = 32 / bits;
  const int nb = (int)((numel + bucket_size - 1) / bucket_size);
  const int wpb = (int)((bucket_size + epw - 1) / epw);
  TORCH_CHECK(out.numel() >= numel, "out too small");
  TORCH_CHECK(region.numel() >= nb + (int64_t)nb * wpb, "region too small");
  const float* norms = region.data_ptr<float>();
  const uint32_t* packed = reinterpret_cast<const uint32_t*>(norms + nb);
  atomo_qsgd_unpack_acc_launch(norms, packed, out.data_ptr<float>(), numel,
                               (int)bucket_size, (int)qlevel, nb, wpb,
                               cur_stream());
}

void svd_decode_acc(torch::Tensor regions, torch::Tensor out2d, int64_t m,
                    int64_t n, int64_t r_max) {
  // regions may be a narrow() view of the stacked (W, total_wire) gather
  // buffer: row-contiguous with an arbitrary row stride.
  TORCH_CHECK(regions.is_cuda(), "regions must be a CUDA (ROCm) tensor");
  TORCH_CHECK(regions.scalar_type() == torch::kFloat32, "regions must be fp32");
  check_f32_cuda(out2d, "out2d");
  TORCH_CHECK(regions.dim() == 2, "regions must be (W, wire_words)");
  TORCH_CHECK(regions.stride(1) == 1, "regions rows must be contiguous");
  const int W = (int)regions.size(0);
  const int64_t stride = regions.stride(0);
  TORCH_CHECK(regions.size(1) >= 1 + r_max * (m + n + 1), "region too small");
  TORCH_CHECK(out2d.numel() == m * n, "out2d shape mismatch");
  atomo_svd_decode_acc_launch(regions.data_ptr<float>(),
                              out2d.data_ptr<float>(), W, stride, (int)m,
                              (int)n, (int)r_max, cur_stream());
}

void fused_sgd(torch::Tensor p, torch::Tensor g, torch::Tensor buf, double lr,
               double momentum, double weight_decay, bool nesterov,
               double dampening, double grad_scale, torch::Tensor lr_dev) {
  check_f32_cuda(p, "p");
  check_f32_cuda(g, "g");
  const int64_t n = p.numel();
  TORCH_CHECK(g.numel() == n, "grad size mismatch");
  if (momentum != 0.0)
    TORCH_CHECK(buf.numel() == n, "momentum buffer size mismatch");
  if (lr_dev.numel())
    TORCH_CHECK(lr_dev.is_cuda() && lr_dev.scalar_type() == torch::kFloat32,
                "lr_dev must be cuda fp32");
  atomo_fused_sgd_launch(p.data_ptr<float>(), g.data_ptr<float>(),
                         buf.numel() ? buf.data_ptr<float>() : nullptr, n,
                         (float)lr, (float)momentum, (float)weight_decay,
                         nesterov, (float)dampening, (float)grad_scale,
                         lr_dev.numel() ? lr_dev.data_ptr<float>() : nullptr,
                         cur_stream());
}

// Batched Jacobi eigensolver via rocSOLVER (syevj_strided_batched): solves
// B symmetric fp32 matrices in one call.  A is overwritten with the
// eigenvectors in rocBLAS column-major (transpose before use); W ascending.
// Measured on MI355X: 5-10x SLOWER than hipSOLVER syevd through
// torch.linalg.eigh (e.g. 34 vs 6.8 ms for 36x256^2), so the encoder keeps
// syevd; this binding stays for benchmarking alternatives.
void rocsolver_eigh_batched(torch::Tensor a, torch::Tensor w,
                            int64_t max_sweeps, double abstol) {
  check_f32_cuda(a, "a");
  check_f32_cuda(w, "w");
  TORCH_CHECK(a.dim() == 3 && a.size(1) == a.size(2), "a must be (B, n, n)");
  const int B = (int)a.size(0);
  const int n = (int)a.size(1);
  TORCH_CHECK(w.numel() == (int64_t)B * n, "w must be (B, n)");
  static rocblas_handle handle = nullptr;
  if (handle == nullptr) {
    TORCH_CHECK(rocblas_create_handle(&handle) == rocblas_status_success,
                "rocblas_create_handle failed");
  }
  rocblas_set_stream(handle, cur_stream());
  auto opts = torch::TensorOptions()
                  .device(a.device())
                  .dtype(torch::kInt32);
  auto info = torch::zeros({B}, opts);
  auto n_sweeps = torch::zeros({B}, opts);
  auto residual = torch::zeros({B}, a.options());
  auto st = rocsolver_ssyevj_strided_batched(
      handle, rocblas_esort_ascending, rocblas_evect_original,
      rocblas_fill_upper, n, a.data_ptr<float>(), n,
      (rocblas_stride)((int64_t)n * n), (float)abstol,
      residual.data_ptr<float>(), (rocblas_int)max_sweeps,
      (rocblas_int*)n_sweeps.data_ptr<int32_t>(), w.data_ptr<float>(),
      (rocblas_stride)n, (rocblas_int*)info.data_ptr<int32_t>(), B);
  TORCH_CHECK(st == rocblas_status_success, "rocsolver syevj failed: ",
              (int)st);
}

void fused_adam(torch::Tensor p, torch::Tensor g, torch::Tensor exp_avg,
                torch::Tensor exp_avg_sq, torch::Tensor max_exp_avg_sq,
                double lr, double beta1, double beta2, double eps,
                double weight_decay, double bias1, double bias2,
                double grad_scale) {
  check_f32_cuda(p, "p");
  check_f32_cuda(g, "g");
  check_f32_cuda(exp_avg, "exp_avg");
  check_f32_cuda(exp_avg_sq, "exp_avg_sq");
  const int64_t n = p.numel();
  TORCH_CHECK(g.numel() == n && exp_avg.numel() == n &&
                  exp_avg_sq.numel() == n,
              "adam buffer size mismatch");
  atomo_fused_adam_launch(
      p.data_ptr<float>(), g.data_ptr<float>(), exp_avg.data_ptr<float>(),
      exp_avg_sq.data_ptr<float>(),
      max_exp_avg_sq.numel() ? max_exp_avg_sq.data_ptr<float>() : nullptr, n,
      (float)lr, (float)beta1, (float)beta2, (float)eps, (float)weight_decay,
      (float)bias1, (float)bias2, (float)grad_scale, cur_stream());
}

void svd_decode_batched(torch::Tensor stacked, torch::Tensor agg,
                        torch::Tensor desc, torch::Tensor work,
                        int64_t n_tiles) {
  TORCH_CHECK(stacked.is_cuda() && stacked.scalar_type() == torch::kFloat32 &&
                  stacked.dim() == 2 && stacked.stride(1) == 1,
              "stacked must be cuda fp32 (W, words) row-contiguous");
  check_f32_cuda(agg, "agg");
  if (n_tiles == 0) return;
  atomo_svd_decode_batched_launch(
      stacked.data_ptr<float>(), stacked.stride(0), (int)stacked.size(0),
      agg.data_ptr<float>(), desc.data_ptr<int64_t>(),
      work.data_ptr<int32_t>(), (int)n_tiles, cur_stream());
}

void qsgd_pack_batched(torch::Tensor flat, torch::Tensor wire,
                       torch::Tensor desc, torch::Tensor work,
                       int64_t n_tiles, int64_t bucket_size, int64_t qlevel,
                       bool terngrad, torch::Tensor seed_dev) {
  check_f32_cuda(flat, "flat");
  check_f32_cuda(wire, "wire");
  TORCH_CHECK(seed_dev.is_cuda() && seed_dev.scalar_type() == torch::kInt64,
              "seed_dev must be cuda int64");
  TORCH_CHECK(bucket_size <= 8192, "bucket_size too large for LDS staging");
  if (n_tiles == 0) return;
  atomo_qsgd_pack_batched_launch(
      flat.data_ptr<float>(), wire.data_ptr<float>(),
      desc.data_ptr<int64_t>(), work.data_ptr<int32_t>(), (int)n_tiles,
      (int)bucket_size, (int)qlevel, terngrad,
      reinterpret_cast<const unsigned long long*>(
          seed_dev.data_ptr<int64_t>()),
      cur_stream());
}

void qsgd_unpack_batched(torch::Tensor wire, torch::Tensor agg,
                         torch::Tensor desc, torch::Tensor work,
                         int64_t n_tiles, int64_t bucket_size,
                         int64_t qlevel) {
  TORCH_CHECK(wire.is_cuda() && wire.scalar_type() == torch::kFloat32,
              "wire must be cuda fp32");
  check_f32_cuda(agg, "agg");
  if (n_tiles == 0) return;
  atomo_qsgd_unpack_batched_launch(
      wire.data_ptr<float>(), agg.data_ptr<float>(), desc.data_ptr<int64_t>(),
      work.data_ptr<int32_t>(), (int)n_tiles, (int)bucket_size, (int)qlevel,
      cur_stream());
}

void batched_gram(torch::Tensor flat, torch::Tensor grams, torch::Tensor desc,
                  torch::Tensor work, int64_t n_tiles) {
  check_f32_cuda(flat, "flat");
  check_f32_cuda(grams, "grams");
  TORCH_CHECK(desc.is_cuda() && desc.scalar_type() == torch::kInt64 &&
                  desc.is_contiguous(),
              "desc must be contiguous cuda int64");
  TORCH_CHECK(work.is_cuda() && work.scalar_type() == torch::kInt32 &&
                  work.is_contiguous(),
              "work must be contiguous cuda int32");
  atomo_batched_gram_launch(flat.data_ptr<float>(), grams.data_ptr<float>(),
                            desc.data_ptr<int64_t>(), work.data_ptr<int32_t>(),
                            (int)n_tiles, cur_stream());
}

void batched_sel(torch::Tensor flat, torch::Tensor wire, torch::Tensor stage,
                 torch::Tensor desc, torch::Tensor work, int64_t n_tiles,
                 int64_t sel_elems) {
  check_f32_cuda(flat, "flat");
  check_f32_cuda(wire, "wire");
  check_f32_cuda(stage, "stage");
  TORCH_CHECK(desc.is_cuda() && desc.scalar_type() == torch::kInt64 &&
                  desc.is_contiguous(),
              "desc must be contiguous cuda int64");
  TORCH_CHECK(work.is_cuda() && work.scalar_type() == torch::kInt32 &&
                  work.is_contiguous(),
              "work must be contiguous cuda int32");
  atomo_batched_sel_launch(flat.data_ptr<float>(), wire.data_ptr<float>(),
                           stage.data_ptr<float>(), desc.data_ptr<int64_t>(),
                           work.data_ptr<int32_t>(), (int)n_tiles,
                           (int)sel_elems, cur_stream());
}

void jacobi_eigh(torch::Tensor grams, torch::Tensor evals, torch::Tensor desc,
                 torch::Tensor eval_offs, torch::Tensor rows, int64_t n_mats,
                 int64_t jmax, torch::Tensor vwarm, torch::Tensor vwarm_offs,
                 int64_t warm, int64_t max_sweeps) {
  check_f32_cuda(grams, "grams");
  check_f32_cuda(evals, "evals");
  TORCH_CHECK(desc.is_cuda() && desc.scalar_type() == torch::kInt64 &&
                  desc.is_contiguous(),
              "desc must be contiguous cuda int64");
  TORCH_CHECK(eval_offs.is_cuda() && eval_offs.scalar_type() == torch::kInt64,
              "eval_offs must be cuda int64");
  TORCH_CHECK(rows.is_cuda() && rows.scalar_type() == torch::kInt32,
              "rows must be cuda int32");
  if (n_mats == 0) return;
  atomo_jacobi_eigh_launch(
      grams.data_ptr<float>(), evals.data_ptr<float>(),
      desc.data_ptr<int64_t>(), eval_offs.data_ptr<int64_t>(),
      rows.data_ptr<int32_t>(), (int)n_mats, (int)jmax,
      vwarm.numel() > 1 ? vwarm.data_ptr<float>() : nullptr,
      vwarm_offs.numel() ? vwarm_offs.data_ptr<int64_t>() : nullptr,
      (int)warm, (int)max_sweeps, cur_stream());
}

void jacobi_dense(torch::Tensor a, torch::Tensor evals, int64_t n_mats,
                  int64_t nb, int64_t max_sweeps) {
  check_f32_cuda(a, "a");
  check_f32_cuda(evals, "evals");
  TORCH_CHECK(nb <= 64 && nb % 2 == 0, "nb must be even and <= 64");
  TORCH_CHECK(a.numel() >= n_mats * nb * nb && evals.numel() >= n_mats * nb,
              "jacobi_dense: buffer too small");
  if (n_mats == 0) return;
  atomo_jacobi_dense_launch(a.data_ptr<float>(), evals.data_ptr<float>(),
                            (int)n_mats, (int)nb, (int)max_sweeps,
                            cur_stream());
}

void jacobi_eigh_big(torch::Tensor grams, torch::Tensor vbuf,
                     torch::Tensor evals, torch::Tensor desc,
                     torch::Tensor eval_offs, torch::Tensor rows,
                     torch::Tensor v_offs, int64_t n_mats) {
  check_f32_cuda(grams, "grams");
  check_f32_cuda(vbuf, "vbuf");
  check_f32_cuda(evals, "evals");
  if (n_mats == 0) return;
  atomo_jacobi_eigh_big_launch(
      grams.data_ptr<float>(), vbuf.data_ptr<float>(),
      evals.data_ptr<float>(), desc.data_ptr<int64_t>(),
      eval_offs.data_ptr<int64_t>(), rows.data_ptr<int32_t>(),
      v_offs.data_ptr<int64_t>(), (int)n_mats, cur_stream());
}

void build_stage(torch::Tensor evecs, torch::Tensor evals,
                 torch::Tensor sel_table, torch::Tensor stage,
                 torch::Tensor desc, torch::Tensor eval_offs,
                 int64_t n_layers) {
  check_f32_cuda(evecs, "evecs");
  check_f32_cuda(evals, "evals");
  check_f32_cuda(sel_table, "sel_table");
  check_f32_cuda(stage, "stage");
  atomo_build_stage_launch(
      evecs.data_ptr<float>(), evals.data_ptr<float>(),
      sel_table.data_ptr<float>(), stage.data_ptr<float>(),
      desc.data_ptr<int64_t>(), eval_offs.data_ptr<int64_t>(), (int)n_layers,
      cur_stream());
}

void sample_stage(torch::Tensor evecs, torch::Tensor evals,
                  torch::Tensor stage, torch::Tensor desc,
                  torch::Tensor eval_offs, int64_t n_layers, int64_t rank,
                  bool truncate, torch::Tensor seed_dev,
                  torch::Tensor used_words) {
  check_f32_cuda(evecs, "evecs");
  check_f32_cuda(evals, "evals");
  check_f32_cuda(stage, "stage");
  TORCH_CHECK(seed_dev.is_cuda() && seed_dev.scalar_type() == torch::kInt64,
              "seed_dev must be cuda int64");
  TORCH_CHECK(used_words.is_cuda() &&
                  used_words.scalar_type() == torch::kInt64,
              "used_words must be cuda int64");
  if (n_layers == 0) return;
  atomo_sample_stage_launch(
      evecs.data_ptr<float>(), evals.data_ptr<float>(),
      stage.data_ptr<float>(), desc.data_ptr<int64_t>(),
      eval_offs.data_ptr<int64_t>(), (int)n_layers, (int)rank,
      truncate ? 1 : 0,
      reinterpret_cast<const unsigned long long*>(
          seed_dev.data_ptr<int64_t>()),
      reinterpret_cast<unsigned long long*>(used_words.data_ptr<int64_t>()),
      cur_stream());
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  register_linear_ops(m);
  register_logit_ops(m);
  m.def("sample_stage", &sample_stage,
        "fused on-device Bernoulli atom sampler + stage builder");
  m.def("jacobi_eigh", &jacobi_eigh, py::arg("grams"), py::arg("evals"),
        py::arg("desc"), py::arg("eval_offs"), py::arg("rows"),
        py::arg("n_mats"), py::arg("jmax"), py::arg("vwarm"),
        py::arg("vwarm_offs"), py::arg("warm"), py::arg("max_sweeps") = 10,
        "batched parallel-Jacobi symmetric eigensolver (sm <= 64, LDS)");
  m.def("jacobi_eigh_big", &jacobi_eigh_big,
        "batched parallel-Jacobi eigensolver (64 < sm <= 512, L2-resident)");
  m.def("jacobi_dense", &jacobi_dense, py::arg("a"), py::arg("evals"),
        py::arg("n_mats"), py::arg("nb"), py::arg("max_sweeps") = 10,
        "batched dense small (nb<=64) symmetric eigh, one wave per matrix; "
        "eigenvalues descending, eigenvectors overwrite the input");
  m.def("build_stage", &build_stage,
        "gather sampled atoms into the staged wire factors");
  m.def("batched_gram", &batched_gram,
        "batched per-layer Gram matrices (small-dim <= 64)");
  m.def("batched_sel", &batched_sel,
        "batched selection GEMM + packet scatter into the wire");
  m.def("qsgd_pack", &qsgd_pack, "QSGD bucket quantize+pack (gfx950)");
  m.def("svd_decode_batched", &svd_decode_batched,
        "one-launch SVD decode+accumulate over all layers and workers");
  m.def("qsgd_pack_batched", &qsgd_pack_batched,
        "one-launch QSGD pack over all layers");
  m.def("qsgd_unpack_batched", &qsgd_unpack_batched,
        "one-launch QSGD unpack+accumulate over all layers");
  m.def("qsgd_unpack_acc", &qsgd_unpack_acc, "QSGD unpack+accumulate");
  m.def("svd_decode_acc", &svd_decode_acc,
        "fused rank-k SVD decode+accumulate over W packets");
  m.def("fused_sgd", &fused_sgd, py::arg("p"), py::arg("g"), py::arg("buf"),
        py::arg("lr"), py::arg("momentum"), py::arg("weight_decay"),
        py::arg("nesterov"), py::arg("dampening"), py::arg("grad_scale"),
        py::arg("lr_dev") = torch::Tensor(), "fused flat SGD apply");
  m.def("fused_adam", &fused_adam, "fused flat Adam apply");
  m.def("rocsolver_eigh_batched", &rocsolver_eigh_batched,
        "rocSOLVER batched Jacobi eigensolver (fp32, in-place)");
}
