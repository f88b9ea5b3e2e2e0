// pybind surface of the MFMA GEMM:
//   _C.gemm.matmul(...)          generic C = op(A) op(B) (+ epilogue), any of the 4 major-ness combos
//   _C.gemm.column_sum(x)        bias gradients
//   _C.fused_dense_cuda.*        the reference's module (csrc/fused_dense.cpp:20-190):
//       linear_bias_forward / linear_bias_backward / linear_gelu_linear_forward / _backward
// Every GEMM of a Linear layer (forward, input gradient, weight gradient) is one launch of the
// same kernel family; no operand is transposed in memory.
#include "common.h"
#include "apex_amd/gated_ffn_api.h"
#include "apex_amd/gemm_api.h"

namespace apex_amd {

namespace {

using OT = c10::optional<at::Tensor>;
bool has(const OT& t) { return t.has_value() && t->defined(); }

// C[M][N] = A(M x K) B(K x N); see gemm_api.h for the major-ness conventions.
at::Tensor run_gemm(const at::Tensor& a, bool a_kmajor, const at::Tensor& b, bool b_kmajor, int64_t m, int64_t n,
                    int64_t k, int epilogue, const OT& bias, const OT& aux_in, at::Tensor* aux_out,
                    at::Tensor* colsum_out = nullptr, at::ScalarType colsum_t = at::kFloat) {
  TORCH_CHECK(a.is_cuda() && b.is_cuda(), "gemm: GPU tensors expected");
  TORCH_CHECK(a.is_contiguous() && b.is_contiguous(), "gemm: contiguous operands expected");
  TORCH_CHECK(a.scalar_type() == b.scalar_type(), "gemm: operand dtype mismatch");
  auto c = at::empty({m, n}, a.options());
  GemmArgs g{};
  g.a = a.data_ptr();
  g.b = b.data_ptr();
  g.c = c.data_ptr();
  g.m = (int)m;
  g.n = (int)n;
  g.k = (int)k;
  g.a_kmajor = a_kmajor;
  g.b_kmajor = b_kmajor;
  g.lda = a_kmajor ? k : m;
  g.ldb = b_kmajor ? k : n;
  g.ldc = n;
  g.dtype = dtype_code(a.scalar_type());
  g.epilogue = epilogue;
  at::Tensor bias_c, aux_c;
  if (has(bias)) {
    bias_c = bias->contiguous().to(a.scalar_type());
    TORCH_CHECK(bias_c.numel() == n, "gemm: bias size mismatch");
    g.bias = bias_c.data_ptr();
  }
  if (has(aux_in)) {
    aux_c = aux_in->contiguous();
    TORCH_CHECK(aux_c.numel() == m * n && aux_c.scalar_type() == a.scalar_type(), "gemm: aux_in mismatch");
    g.aux_in = aux_c.data_ptr();
  }
  if (aux_out != nullptr) {
    *aux_out = at::empty({m, n}, a.options());
    g.aux_out = aux_out->data_ptr();
  }
  TORCH_CHECK(gemm_supported(g), "gemm: unsupported shape/alignment/dtype (need fp16/bf16, K, N multiples of 8, "
              "16-byte aligned operands)");
  const int cus = device_cus(a.get_device());
  at::Tensor ws;  // split-K partials (weight gradients with few output tiles); caching allocator
  const int64_t wsf = gemm_splitk_workspace_floats(g, cus);
  const char* sk = std::getenv("APEX_AMD_SPLITK");  // =off disables (A/B timing)
  if (wsf > 0 && !(sk != nullptr && sk[0] == 'o')) {
    ws = at::empty({wsf}, a.options().dtype(at::kFloat));
    g.splitk_ws = ws.data_ptr<float>();
  }
  at::Tensor cpart;
  const bool fused_cs = colsum_out != nullptr && gemm_colsum_fusable(g, cus);
  if (fused_cs) {
    // column sums of C in the epilogue: one fp32 row per 256-row tile, then a fixed-order fold
    cpart = at::empty({(m + 255) / 256, n}, a.options().dtype(at::kFloat));
    g.colpart = cpart.data_ptr<float>();
  }
  gemm_mfma(g, cus, cur_stream());
  if (colsum_out != nullptr) {
    *colsum_out = at::empty({n}, a.options().dtype(colsum_t));
    if (fused_cs) {
      column_sum_finalize(cpart.data_ptr<float>(), (int)cpart.size(0), (int)n, colsum_out->data_ptr(),
                          dtype_code(colsum_t), cur_stream());
    } else {
      auto cws = at::empty({column_sum_workspace_floats(m, (int)n, cus)}, a.options().dtype(at::kFloat));
      column_sum(c.data_ptr(), dtype_code(c.scalar_type()), m, (int)n, n, colsum_out->data_ptr(), dtype_code(colsum_t),
                 cws.data_ptr<float>(), cus, cur_stream());
    }
  }
  return c;
}

at::Tensor colsum(const at::Tensor& x2d, at::ScalarType out_t) {
  const c10::hip::HIPGuard g(x2d.get_device());
  at::Tensor x = x2d.contiguous();
  const int64_t m = x.size(0), n = x.size(1);
  auto out = at::empty({n}, x.options().dtype(out_t));
  const int cus = device_cus(x.get_device());
  auto ws = at::empty({column_sum_workspace_floats(m, n, cus)}, x.options().dtype(at::kFloat));
  column_sum(x.data_ptr(), dtype_code(x.scalar_type()), m, (int)n, n, out.data_ptr(), dtype_code(out_t),
             ws.data_ptr<float>(), cus, cur_stream());
  return out;
}

at::Tensor as2d(const at::Tensor& t) {
  at::Tensor c = t.contiguous();
  return c.view({-1, c.size(-1)});
}

// ---- Linear building blocks (x [M, K], W [N, K]) ----
at::Tensor linear_fwd(const at::Tensor& x2, const at::Tensor& w, const OT& bias, int epi, at::Tensor* aux) {
  return run_gemm(x2, true, w.contiguous(), true, x2.size(0), w.size(0), x2.size(1), epi, bias, c10::nullopt, aux);
}
// dx[M, K] = dy[M, N] W[N, K]   (epilogue may multiply by an activation derivative of aux_in)
at::Tensor linear_dgrad(const at::Tensor& dy2, const at::Tensor& w, int epi, const OT& aux_in) {
  return run_gemm(dy2, true, w.contiguous(), false, dy2.size(0), w.size(1), dy2.size(1), epi, c10::nullopt, aux_in,
                  nullptr);
}
// dW[N, K] = dy[M, N]^T x[M, K]
at::Tensor linear_wgrad(const at::Tensor& dy2, const at::Tensor& x2) {
  return run_gemm(dy2, false, x2, false, dy2.size(1), x2.size(1), dy2.size(0), kEpiNone, c10::nullopt, c10::nullopt,
                  nullptr);
}

// ---- gated feed-forward block (csrc/gemm/gated_ffn.hip) ----
// contiguous, and 16-byte aligned even where a contiguous view starts inside a vector
at::Tensor vec16(const at::Tensor& t) {
  at::Tensor c = t.contiguous();
  return ((uintptr_t)c.data_ptr() & 15u) ? c.clone() : c;
}

void ffn_run(int op, const at::Tensor& a, bool a_kmajor, const at::Tensor& b, bool b_kmajor, int64_t m, int64_t n,
             int64_t k, const at::Tensor& c, int act, const at::Tensor& bias, const at::Tensor& hi,
             const at::Tensor& lo) {
  TORCH_CHECK(m < (int64_t(1) << 31) && n < (int64_t(1) << 30) && k < (int64_t(1) << 31), "gated_ffn: sizes too large");
  FfnArgs g{};
  g.a = a.data_ptr();
  g.b = b.data_ptr();
  g.c = c.data_ptr();
  g.m = (int)m;
  g.n = (int)n;
  g.k = (int)k;
  g.a_kmajor = a_kmajor;
  g.b_kmajor = b_kmajor;
  g.lda = a.size(1);
  g.ldb = b.size(1);
  g.ldc = c.size(1);
  g.dtype = dtype_code(a.scalar_type());
  g.op = op;
  g.act = act;
  g.bias = bias.defined() ? bias.data_ptr() : nullptr;
  g.au_hi = hi.defined() ? (uint16_t*)hi.data_ptr<int16_t>() : nullptr;
  g.au_lo = lo.defined() ? lo.data_ptr<uint8_t>() : nullptr;
  TORCH_CHECK(ffn_supported(g), "gated_ffn: unsupported sizes or alignment (fp16 / bf16, widths multiples of 8)");
  const int cus = device_cus(a.get_device());
  at::Tensor ws;
  const int64_t wsf = ffn_workspace_floats(g, cus);
  if (wsf > 0) {
    ws = at::empty({wsf}, a.options().dtype(at::kFloat));
    g.ws = ws.data_ptr<float>();
  }
  ffn_gemm(g, cus, cur_stream());
}

void ffn_check(const at::Tensor& x, const at::Tensor& w1, const at::Tensor& w2, int64_t act) {
  auto ok = [&](const at::Tensor& t) {
    return t.is_cuda() && t.get_device() == x.get_device() && t.scalar_type() == x.scalar_type() && t.dim() == 2;
  };
  TORCH_CHECK(ok(x) && ok(w1) && ok(w2) && w1.size(1) == x.size(1) && w1.size(0) == 2 * w2.size(1),
              "gated_ffn: [m, k] input, [2f, k] weight1 and [n, f] weight2 of one dtype and device expected");
  TORCH_CHECK(act == kGateSilu || act == kGateGelu, "gated_ffn: unknown activation");
}

at::Tensor ffn_bias(const OT& b, int64_t n, const at::Tensor& x) {
  if (!has(b)) return at::Tensor();
  TORCH_CHECK(b->is_cuda() && b->get_device() == x.get_device() && b->scalar_type() == x.scalar_type() &&
                  b->numel() == n,
              "gated_ffn: bias size, dtype or device mismatch");
  return vec16(*b);
}

// (y, h, au's planes); the last three (the backward's inputs) are undefined unless save
std::vector<at::Tensor> ffn_forward(const at::Tensor& x_, const at::Tensor& w1_, const OT& b1_, const at::Tensor& w2_,
                                    const OT& b2_, int64_t act, bool save) {
  TORCH_CHECK(x_.is_cuda(), "gated_ffn: GPU tensors expected");
  const c10::hip::HIPGuard guard(x_.get_device());
  ffn_check(x_, w1_, w2_, act);
  at::Tensor x = vec16(x_), w1 = vec16(w1_), w2 = vec16(w2_);
  const int64_t m = x.size(0), k = x.size(1), f = w2.size(1), n = w2.size(0);
  at::Tensor b1 = ffn_bias(b1_, 2 * f, x), b2 = ffn_bias(b2_, n, x);
  at::Tensor h = at::empty({m, f}, x.options()), y = at::empty({m, n}, x.options()), hi, lo;
  if (save) {
    hi = at::empty({m, 2 * f}, x.options().dtype(at::kShort));
    lo = at::empty({m, 2 * f}, x.options().dtype(at::kByte));
  }
  if (m > 0) {
    ffn_run(kFfnGated, x, true, w1, true, m, f, k, h, (int)act, b1, hi, lo);
    ffn_run(kFfnPlain, h, true, w2, true, m, n, f, y, 0, b2, at::Tensor(), at::Tensor());
  }
  return {y, save ? h : at::Tensor(), hi, lo};
}

// (dx, dw1, db1, dw2, db2), undefined where not needed
std::vector<at::Tensor> ffn_backward(const at::Tensor& dy_, const at::Tensor& x_, const at::Tensor& w1_,
                                     const at::Tensor& w2_, const at::Tensor& h, const at::Tensor& hi,
                                     const at::Tensor& lo, int64_t act, bool need_dx, bool need_dw1, bool need_db1, bool need_dw2, bool need_db2) {
  TORCH_CHECK(x_.is_cuda(), "gated_ffn: GPU tensors expected");
  const c10::hip::HIPGuard guard(x_.get_device());
  ffn_check(x_, w1_, w2_, act);
  at::Tensor dy = vec16(dy_), x = vec16(x_), w1 = vec16(w1_), w2 = vec16(w2_);
  const int64_t m = x.size(0), k = x.size(1), f = w2.size(1), n = w2.size(0);
  auto is = [&](const at::Tensor& t, int64_t c, at::ScalarType type) {
    return t.is_cuda() && t.get_device() == x.get_device() && t.scalar_type() == type && t.dim() == 2 &&
           t.size(0) == m && t.size(1) == c && t.is_contiguous();
  };
  TORCH_CHECK(is(dy, n, x.scalar_type()) && is(h, f, x.scalar_type()) && is(hi, 2 * f, at::kShort) &&
                  is(lo, 2 * f, at::kByte),
              "gated_ffn: backward operands do not fit");
  const at::Tensor none;
  at::Tensor dx, dw1, db1, dw2, db2;
  if (m == 0) {
    if (need_dx) dx = at::empty({0, k}, x.options());
    if (need_dw1) dw1 = at::zeros_like(w1);
    if (need_db1) db1 = at::zeros({2 * f}, x.options());
    if (need_dw2) dw2 = at::zeros_like(w2);
    if (need_db2) db2 = at::zeros({n}, x.options());
    return {dx, dw1, db1, dw2, db2};
  }
  if (need_dw2) {
    dw2 = at::empty({n, f}, x.options());
    ffn_run(kFfnPlain, dy, false, h, false, n, f, m, dw2, 0, none, none, none);
  }
  if (need_db2) db2 = colsum(dy, x.scalar_type());
  if (need_dx || need_dw1 || need_db1) {
    at::Tensor dau = at::empty({m, 2 * f}, x.options());
    ffn_run(kFfnDGated, dy, true, w2, false, m, f, n, dau, (int)act, none, hi, lo);
    if (need_dw1) {
      dw1 = at::empty({2 * f, k}, x.options());
      ffn_run(kFfnPlain, dau, false, x, false, 2 * f, k, m, dw1, 0, none, none, none);
    }
    if (need_db1) db1 = colsum(dau, x.scalar_type());
    if (need_dx) {
      dx = at::empty({m, k}, x.options());
      ffn_run(kFfnPlain, dau, true, w1, false, m, k, 2 * f, dx, 0, none, none, none);
    }
  }
  return {dx, dw1, db1, dw2, db2};
}

// The autograd node lives in C++ (a python one costs 10-20 us more host time a step)
struct GatedFfnFn : torch::autograd::Function<GatedFfnFn> {
  static at::Tensor forward(torch::autograd::AutogradContext* ctx, const at::Tensor& x, const at::Tensor& w1,
                            const OT& b1, const at::Tensor& w2, const OT& b2, int64_t act, bool save) {
    auto r = ffn_forward(x, w1, b1, w2, b2, act, save);
    if (save) ctx->save_for_backward({x, w1, w2, r[1], r[2], r[3]});
    ctx->saved_data["act"] = act;
    ctx->saved_data["b1"] = has(b1);
    ctx->saved_data["b2"] = has(b2);
    return r[0];
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list g) {
    TORCH_CHECK(!at::GradMode::is_enabled(),
                "fused_dense_gated_dense_function is differentiable once (create_graph is not supported)");
    const auto s = ctx->get_saved_variables();
    // the node's edges are the tensors that were given: x, weight1, [bias1], weight2, [bias2]
    const bool b1 = ctx->saved_data["b1"].toBool(), b2 = ctx->saved_data["b2"].toBool();
    auto d = ffn_backward(g[0], s[0], s[1], s[2], s[3], s[4], s[5], ctx->saved_data["act"].toInt(),
                          ctx->needs_input_grad(0), ctx->needs_input_grad(1), b1 && ctx->needs_input_grad(2),
                          ctx->needs_input_grad(2 + b1), b2 && ctx->needs_input_grad(3 + b1));
    const at::Tensor none;
    return {d[0], d[1], d[2], d[3], d[4], none, none};
  }
};

at::Tensor gated_ffn(const at::Tensor& x, const at::Tensor& w1, const OT& b1, const at::Tensor& w2, const OT& b2,
                     int64_t act) {
  auto grad = [](const OT& t) { return has(t) && t->requires_grad(); };
  const bool save = at::GradMode::is_enabled() && (grad(x) || grad(w1) || grad(w2) || grad(b1) || grad(b2));
  return GatedFfnFn::apply(x, w1, b1, w2, b2, act, save);
}

}  // namespace

void bind_lt(pybind11::module_& root);  // lt_epilogue.cpp

void bind_gemm(pybind11::module_& root) {
  bind_lt(root);
  namespace py = pybind11;
  auto g = root.def_submodule("gemm", "gfx950 MFMA GEMM with fused epilogues");
  g.attr("EPI_NONE") = (int)kEpiNone;
  g.attr("EPI_GELU") = (int)kEpiGelu;
  g.attr("EPI_RELU") = (int)kEpiRelu;
  g.attr("EPI_SIGMOID") = (int)kEpiSigmoid;
  g.attr("EPI_DGELU") = (int)kEpiDGelu;
  g.attr("EPI_DRELU") = (int)kEpiDRelu;
  g.attr("EPI_DSIGMOID") = (int)kEpiDSigmoid;
  g.def("matmul",
        [](at::Tensor a, bool a_kmajor, at::Tensor b, bool b_kmajor, int64_t m, int64_t n, int64_t k, int epilogue,
           OT bias, OT aux_in, bool want_aux) {
          const c10::hip::HIPGuard guard(a.get_device());
          at::Tensor aux;
          auto c = run_gemm(a.contiguous(), a_kmajor, b.contiguous(), b_kmajor, m, n, k, epilogue, bias, aux_in,
                            want_aux ? &aux : nullptr);
          return std::make_tuple(c, aux);
        },
        py::arg("a"), py::arg("a_kmajor"), py::arg("b"), py::arg("b_kmajor"), py::arg("m"), py::arg("n"),
        py::arg("k"), py::arg("epilogue") = (int)kEpiNone, py::arg("bias") = c10::nullopt,
        py::arg("aux_in") = c10::nullopt, py::arg("want_aux") = false);
  g.def("linear", [](at::Tensor x, at::Tensor w, OT bias, int epi, bool want_aux) {
    const c10::hip::HIPGuard guard(x.get_device());
    at::Tensor aux;
    auto y = linear_fwd(as2d(x), w, bias, epi, want_aux ? &aux : nullptr);
    return std::make_tuple(y, aux);
  });
  g.def("linear_dgrad", [](at::Tensor dy, at::Tensor w, int epi, OT aux_in) {
    const c10::hip::HIPGuard guard(dy.get_device());
    return linear_dgrad(as2d(dy), w, epi, aux_in);
  });
  g.def("linear_wgrad", [](at::Tensor dy, at::Tensor x) {
    const c10::hip::HIPGuard guard(dy.get_device());
    return linear_wgrad(as2d(dy), as2d(x));
  });
  g.def("linear_dgrad_bgrad", [](at::Tensor dy, at::Tensor w, int epi, at::Tensor aux_in,
                                 c10::optional<at::ScalarType> out_dtype) {
    // (dz, db): dz = (dy W) * act'(aux_in) with db = column sums of the stored dz in the GEMM's
    // epilogue (the reference's DGELU_BGRAD, csrc/fused_dense_cuda.cu:977) — no pass over dz
    const c10::hip::HIPGuard guard(dy.get_device());
    at::Tensor d = as2d(dy), db;
    auto dz = run_gemm(d, true, w.contiguous(), false, d.size(0), w.size(1), d.size(1), epi, c10::nullopt, aux_in,
                       nullptr, &db, out_dtype.value_or(d.scalar_type()));
    return std::make_tuple(dz, db);
  }, py::arg("dy"), py::arg("w"), py::arg("epilogue"), py::arg("aux_in"), py::arg("out_dtype") = c10::nullopt);
  g.def("dgelu_column_sum", [](at::Tensor dy, at::Tensor aux, c10::optional<at::ScalarType> out_dtype) {
    // (dz, db): dz = dy * gelu_tanh'(aux), db = column sums of dz — one pass
    const c10::hip::HIPGuard guard(dy.get_device());
    at::Tensor d = as2d(dy), a = as2d(aux);
    TORCH_CHECK(d.sizes() == a.sizes() && d.scalar_type() == a.scalar_type(), "dgelu_column_sum: shape mismatch");
    const int64_t m = d.size(0), n = d.size(1);
    auto dz = at::empty_like(d);
    const at::ScalarType ot = out_dtype.value_or(d.scalar_type());
    auto db = at::empty({n}, d.options().dtype(ot));
    const int cus = device_cus(d.get_device());
    auto ws = at::empty({column_sum_workspace_floats(m, n, cus)}, d.options().dtype(at::kFloat));
    dgelu_column_sum(d.data_ptr(), a.data_ptr(), dz.data_ptr(), dtype_code(d.scalar_type()), m, (int)n, db.data_ptr(),
                     dtype_code(ot), ws.data_ptr<float>(), cus, cur_stream());
    return std::make_tuple(dz, db);
  }, pybind11::arg("dy"), pybind11::arg("aux"), pybind11::arg("out_dtype") = c10::nullopt);
  g.def("gelu", [](at::Tensor z) {
    // y = gelu_tanh(z) (the tanh approximation of the reference's cuBLASLt GELU epilogue)
    const c10::hip::HIPGuard guard(z.get_device());
    at::Tensor zc = z.contiguous();
    auto y = at::empty_like(zc);
    gelu_tanh_forward(zc.data_ptr(), y.data_ptr(), dtype_code(zc.scalar_type()), zc.numel(), device_cus(zc.get_device()),
                      cur_stream());
    return y;
  });
  g.def("column_sum", [](at::Tensor x, c10::optional<at::ScalarType> out_dtype) {
    return colsum(as2d(x), out_dtype.value_or(x.scalar_type()));
  }, py::arg("x"), py::arg("out_dtype") = c10::nullopt);

  auto gf = root.def_submodule("gated_ffn", "gated feed-forward block on gfx950 MFMA");
  gf.attr("ACT_SILU") = (int)kGateSilu;
  gf.attr("ACT_GELU") = (int)kGateGelu;
  gf.def("gated_ffn", &gated_ffn);
  // (tile width, splits of K) of the six products, in order: gated, down, dW2, [da | du], dW1, dx
  gf.def("plans", [](int64_t m, int64_t k, int64_t f, int64_t n, int64_t cus) {
    for (int64_t v : {m, k, f, n, cus}) TORCH_CHECK(v > 0 && v < (int64_t(1) << 30), "gated_ffn.plans: sizes out of range");
    struct Product { int op; bool a, b; int64_t m, n, k; };
    const Product ps[] = {{kFfnGated, true, true, m, f, k},  {kFfnPlain, true, true, m, n, f},
                          {kFfnPlain, false, false, n, f, m}, {kFfnDGated, true, false, m, f, n},
                          {kFfnPlain, false, false, 2 * f, k, m}, {kFfnPlain, true, false, m, k, 2 * f}};
    std::vector<std::pair<int, int>> out;
    for (const Product& p : ps) {
      FfnArgs g{};
      g.op = p.op;
      g.a_kmajor = p.a;
      g.b_kmajor = p.b;
      g.m = (int)p.m;
      g.n = (int)p.n;
      g.k = (int)p.k;
      const FfnPlan r = ffn_plan(g, (int)cus);
      out.emplace_back(r.bn, r.splits);
    }
    return out;
  });

  auto fd = root.def_submodule("fused_dense_cuda", "fused dense (GEMM + bias [+ GeLU]) on gfx950 MFMA");
  fd.def("linear_bias_forward", [](at::Tensor input, at::Tensor weight, OT bias) {
    const c10::hip::HIPGuard guard(input.get_device());
    return linear_fwd(as2d(input), weight, bias, kEpiNone, nullptr);
  });
  fd.def("linear_bias_backward", [](at::Tensor input, at::Tensor weight, at::Tensor grad_output) {
    const c10::hip::HIPGuard guard(input.get_device());
    auto x2 = as2d(input), dy2 = as2d(grad_output);
    auto dx = linear_dgrad(dy2, weight, kEpiNone, c10::nullopt);
    auto dw = linear_wgrad(dy2, x2);
    auto db = colsum(dy2, weight.scalar_type());
    return std::vector<at::Tensor>{dx, dw, db};
  });
  fd.def("linear_gelu_linear_forward",
         [](at::Tensor input, at::Tensor w1, at::Tensor b1, at::Tensor w2, at::Tensor b2) {
           const c10::hip::HIPGuard guard(input.get_device());
           at::Tensor gelu_in;
           auto out1 = linear_fwd(as2d(input), w1, b1, kEpiGelu, &gelu_in);
           auto out2 = linear_fwd(out1, w2, b2, kEpiNone, nullptr);
           return std::vector<at::Tensor>{out1, out2, gelu_in};
         });
  fd.def("linear_gelu_linear_backward", [](at::Tensor input, at::Tensor gelu_in, at::Tensor output1, at::Tensor w1,
                                           at::Tensor w2, at::Tensor grad_output) {
    const c10::hip::HIPGuard guard(input.get_device());
    auto x2 = as2d(input), dy2 = as2d(grad_output);
    auto dw2 = linear_wgrad(dy2, output1);
    auto db2 = colsum(dy2, w2.scalar_type());
    // (dy W2) * gelu'(pre-activation), its column sums (db1) in the same epilogue
    at::Tensor db1;
    auto dh = run_gemm(dy2, true, w2.contiguous(), false, dy2.size(0), w2.size(1), dy2.size(1), kEpiDGelu,
                       c10::nullopt, gelu_in, nullptr, &db1, w1.scalar_type());
    auto dw1 = linear_wgrad(dh, x2);
    auto dx = linear_dgrad(dh, w1, kEpiNone, c10::nullopt);
    return std::vector<at::Tensor>{dx, dw1, db1, dw2, db2};
  });
}

}  // namespace apex_amd
