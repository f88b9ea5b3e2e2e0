// pybind surface: submodule ``_C.xentropy_cuda`` (reference apex/contrib/csrc/xentropy/
// interface.cpp:5-52: forward(input, labels, smoothing, half_to_float) -> [losses,
// max_log_sum_exp]; backward(grad_loss, logits, max_log_sum_exp, labels, smoothing)).
// The padding-index masking the reference does in python is folded into the kernels here.
#include "common.h"
#include "apex_amd/topk_distill_api.h"

namespace apex_amd {

void xentropy_fwd(const void* logits, int dt, const int64_t* labels, float* losses, float* lse, int64_t rows,
                  int classes, float smoothing, int64_t padding_idx, bool use_pad, hipStream_t s);
void xentropy_bwd(const float* grad_loss, const void* logits, int dt, const float* lse, const int64_t* labels,
                  void* grad, int64_t rows, int classes, float smoothing, int64_t padding_idx, bool use_pad,
                  hipStream_t s);

namespace {

std::vector<at::Tensor> fwd(const at::Tensor& input, const at::Tensor& labels_, double smoothing, bool half_to_float,
                            c10::optional<int64_t> padding_idx) {
  TORCH_CHECK(input.is_cuda() && input.dim() == 2, "xentropy: [rows, classes] GPU logits expected");
  const c10::hip::HIPGuard g(input.get_device());
  at::Tensor x = input.contiguous();
  at::Tensor labels = labels_.contiguous().to(at::kLong);
  TORCH_CHECK(labels.numel() == x.size(0), "xentropy: one label per row");
  auto fo = x.options().dtype(at::kFloat);
  auto losses = at::empty({x.size(0)}, fo), lse = at::empty({x.size(0)}, fo);
  xentropy_fwd(x.data_ptr(), dtype_code(x.scalar_type()), labels.data_ptr<int64_t>(), losses.data_ptr<float>(),
               lse.data_ptr<float>(), x.size(0), (int)x.size(1), (float)smoothing, padding_idx.value_or(0),
               padding_idx.has_value(), cur_stream());
  if (!half_to_float && x.scalar_type() != at::kFloat) losses = losses.to(x.scalar_type());
  return {losses, lse};
}

at::Tensor bwd(const at::Tensor& grad_loss, const at::Tensor& logits, const at::Tensor& lse, const at::Tensor& labels_,
               double smoothing, c10::optional<int64_t> padding_idx) {
  const c10::hip::HIPGuard g(logits.get_device());
  at::Tensor x = logits.contiguous();
  at::Tensor gl = grad_loss.contiguous().to(at::kFloat);
  at::Tensor ls = lse.contiguous().to(at::kFloat);
  at::Tensor labels = labels_.contiguous().to(at::kLong);
  auto grad = at::empty_like(x);
  xentropy_bwd(gl.data_ptr<float>(), x.data_ptr(), dtype_code(x.scalar_type()), ls.data_ptr<float>(),
               labels.data_ptr<int64_t>(), grad.data_ptr(), x.size(0), (int)x.size(1), (float)smoothing,
               padding_idx.value_or(0), padding_idx.has_value(), cur_stream());
  return grad;
}

// ---- distillation from a teacher's top logits (csrc/xentropy/topk_distill.hip) ----
struct DistillHold {
  TopkDistillArgs a{};
  at::Tensor x, tz, ti;
};

void distill_setup(DistillHold& h, const at::Tensor& logits, const at::Tensor& tz, const at::Tensor& ti, double temperature) {
  TORCH_CHECK(logits.is_cuda() && logits.dim() == 2 && logits.size(1) > 0,
              "topk_distill: [rows, classes] GPU logits expected");
  TORCH_CHECK(tz.is_cuda() && ti.is_cuda() && tz.get_device() == logits.get_device() &&
                  ti.get_device() == logits.get_device() && tz.dim() == 2 && tz.sizes() == ti.sizes() &&
                  tz.size(0) == logits.size(0) && tz.size(1) <= kDistillMaxTop,
              "topk_distill: teacher logits and indices must be [rows, top <= ", kDistillMaxTop, "] on the logits' device");
  TORCH_CHECK(ti.scalar_type() == at::kLong || ti.scalar_type() == at::kInt,
              "topk_distill: teacher indices must be int64 or int32");
  TORCH_CHECK(logits.size(1) < (int64_t(1) << 30), "topk_distill: too many classes");
  TORCH_CHECK(temperature > 0, "topk_distill: the temperature must be positive");
  // rows of any pitch are read in place; other layouts are copied
  h.x = logits.stride(1) == 1 || logits.size(1) == 1 ? logits : logits.contiguous();
  h.tz = tz.contiguous().to(at::kFloat);
  h.ti = ti.contiguous();
  TopkDistillArgs& a = h.a;
  a.logits = h.x.data_ptr();
  a.pitch = h.x.stride(0);
  a.rows = h.x.size(0);
  a.classes = (int)h.x.size(1);
  a.top = (int)tz.size(1);
  a.teacher_logits = h.tz.data_ptr<float>();
  a.teacher_indices = h.ti.data_ptr();
  a.index64 = h.ti.scalar_type() == at::kLong;
  a.temperature = (float)temperature;
  a.dtype = dtype_code(h.x.scalar_type());
}

std::vector<at::Tensor> distill_fwd(const at::Tensor& logits, const at::Tensor& tz, const at::Tensor& ti,
                                    double temperature) {
  TORCH_CHECK(logits.is_cuda(), "topk_distill: GPU logits expected");
  const c10::hip::HIPGuard g(logits.get_device());
  DistillHold h;
  distill_setup(h, logits, tz, ti, temperature);
  auto fo = logits.options().dtype(at::kFloat);
  auto losses = at::empty({h.a.rows}, fo), stats = at::empty({h.a.rows, 2}, fo);
  const int cus = device_cus(logits.get_device());
  auto parts = at::empty({topk_distill_part_floats(h.a, cus)}, fo);
  topk_distill_fwd(h.a, losses.data_ptr<float>(), stats.data_ptr<float>(), parts.data_ptr<float>(), cus, cur_stream());
  return {losses, stats};
}

at::Tensor distill_bwd(const at::Tensor& grad_loss, const at::Tensor& logits, const at::Tensor& stats,
                       const at::Tensor& tz, const at::Tensor& ti, double temperature) {
  TORCH_CHECK(logits.is_cuda(), "topk_distill: GPU logits expected");
  const c10::hip::HIPGuard g(logits.get_device());
  DistillHold h;
  distill_setup(h, logits, tz, ti, temperature);
  auto on_rows = [&](const at::Tensor& t) {
    return t.is_cuda() && t.get_device() == logits.get_device() && t.dim() >= 1 && t.size(0) == h.a.rows;
  };
  TORCH_CHECK(on_rows(grad_loss) && grad_loss.dim() == 1 && on_rows(stats) && stats.numel() == 2 * h.a.rows &&
                  stats.scalar_type() == at::kFloat && stats.is_contiguous(),
              "topk_distill: [rows] grad_loss and [rows, 2] statistics on the logits' device expected");
  at::Tensor gl = grad_loss.to(at::kFloat);  // any stride (a broadcast gradient has stride 0)
  auto grad = at::empty(logits.sizes(), logits.options());
  topk_distill_bwd(h.a, gl.data_ptr<float>(), gl.stride(0), stats.data_ptr<float>(), grad.data_ptr(),
                   device_cus(logits.get_device()), cur_stream());
  return grad;
}

// The autograd node lives in C++ (a python one costs 10-20 us more host time a step)
struct TopkDistillFn : torch::autograd::Function<TopkDistillFn> {
  static at::Tensor forward(torch::autograd::AutogradContext* ctx, const at::Tensor& logits, const at::Tensor& tz,
                            const at::Tensor& ti, double temperature, bool half_to_float) {
    auto r = distill_fwd(logits, tz, ti, temperature);
    ctx->save_for_backward({logits, tz, ti, r[1]});
    ctx->saved_data["temperature"] = temperature;
    return half_to_float ? r[0] : r[0].to(logits.scalar_type());
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list g) {
    TORCH_CHECK(!at::GradMode::is_enabled(),
                "SoftmaxTopKDistillationLoss is differentiable once (create_graph is not supported)");
    const auto s = ctx->get_saved_variables();
    const at::Tensor none;
    return {distill_bwd(g[0], s[0], s[3], s[1], s[2], ctx->saved_data["temperature"].toDouble()), none, none, none, none};
  }
};

at::Tensor topk_distill(const at::Tensor& logits, const at::Tensor& tz, const at::Tensor& ti, double temperature,
                        bool half_to_float) {
  return TopkDistillFn::apply(logits, tz, ti, temperature, half_to_float);
}

}  // namespace

void bind_xentropy(pybind11::module_& root) {
  namespace py = pybind11;
  auto m = root.def_submodule("xentropy_cuda", "gfx950 softmax cross-entropy with label smoothing");
  m.def("forward", &fwd, py::arg("input"), py::arg("labels"), py::arg("smoothing"), py::arg("half_to_float"),
        py::arg("padding_idx") = c10::nullopt);
  m.def("backward", &bwd, py::arg("grad_loss"), py::arg("logits"), py::arg("max_log_sum_exp"), py::arg("labels"),
        py::arg("smoothing"), py::arg("padding_idx") = c10::nullopt);
  m.def("topk_distill", &topk_distill, py::arg("logits"), py::arg("teacher_logits"), py::arg("teacher_indices"),
        py::arg("temperature"), py::arg("half_to_float"));
}

}  // namespace apex_amd
