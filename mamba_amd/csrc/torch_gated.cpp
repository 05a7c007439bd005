// The gated linear recurrence, its single-token step and the norm between two blocks on at::Tensor: argument checks,
// allocation, launch through the C ABI, and the autograd nodes.
#include "torch_common.h"

#include <torch/csrc/autograd/functions/basic_ops.h>

#include <cmath>

namespace mamba_ext {
namespace {

// Gradients of a node whose backward pass has no gradient of its own: with create_graph a second derivative through
// them is an error, not a zero.
variable_list once(variable_list g, const char *what) {
  if (!at::GradMode::is_enabled()) return g;
  for (at::Tensor &t : g)
    if (t.defined()) t = t.detach().requires_grad_();
  torch::autograd::DelayedError fn(std::string(what) + " has no second derivatives", (int64_t)g.size());
  return fn.apply(std::move(g));
}

bool unit(const at::Tensor &t) { return t.stride(-1) == 1 || t.size(-1) == 1; }
bool rate_ok(double rate) { return rate >= 0.0 && rate <= 3e38; }
bool decay_ok(const at::Tensor &decay, int64_t dim, const c10::Device &dev) {
  return on_device(decay, dev) && dtype_code(decay) >= 0 && decay.dim() == 1 && decay.size(0) == dim && decay.is_contiguous();
}

// ------------------------------------------------------------------ scan
struct Scan {
  double rate;
  bool final_states;
};

void fill(GatedScanParams &p, const at::Tensor &x, const at::Tensor &ga, const at::Tensor &gx, const at::Tensor &decay,
          const OptTensor &initial, const OptTensor &cu, double rate) {
  p.batch = (int32_t)x.size(0), p.seqlen = (int32_t)x.size(1), p.dim = (int32_t)x.size(2);
  p.nseq = cu ? (int32_t)cu->size(0) - 1 : 0;
  p.dtype = dtype_code(x), p.decay_dtype = dtype_code(decay), p.rate = (float)rate;
  p.x = x.data_ptr(), p.gate_a = ga.data_ptr(), p.gate_x = gx.data_ptr(), p.decay = decay.data_ptr();
  p.initial_states = initial ? initial->data_ptr<float>() : nullptr, p.cu_seqlens = cu ? cu->data_ptr<int32_t>() : nullptr;
  p.x_bs = x.stride(0), p.x_ls = x.stride(1), p.gate_a_bs = ga.stride(0), p.gate_a_ls = ga.stride(1);
  p.gate_x_bs = gx.stride(0), p.gate_x_ls = gx.stride(1);
}
at::Tensor bytes(int64_t n, const char *what, const at::Tensor &like) {
  if (n < 0) check_rc((int)n, what);
  return at::empty({n}, like.options().dtype(at::kByte));
}

// out, final states (undefined unless wanted), checkpoints
std::tuple<at::Tensor, at::Tensor, at::Tensor> scan_fwd(const at::Tensor &x, const at::Tensor &ga, const at::Tensor &gx,
                                                        const at::Tensor &decay, const OptTensor &initial, const OptTensor &cu,
                                                        const Scan &o) {
  GatedScanParams p{};
  fill(p, x, ga, gx, decay, initial, cu, o.rate);
  c10::DeviceGuard guard(x.device());
  at::Tensor out = at::empty(x.sizes(), x.options()), final;
  if (o.final_states) final = at::empty({p.nseq ? p.nseq : p.batch, p.dim}, x.options().dtype(at::kFloat));
  at::Tensor ckpt = bytes(gated_scan_ckpt_bytes(&p), "gated_scan_ckpt_bytes", x);
  p.out = out.data_ptr(), p.out_bs = out.stride(0), p.out_ls = out.stride(1), p.ckpt = ckpt.data_ptr();
  p.final_states = final.defined() ? final.data_ptr<float>() : nullptr;
  check_rc(gated_scan_fwd(&p, stream_of(x.device())), "gated_scan_fwd");
  return {out, final, ckpt};
}

struct GatedScanFn : torch::autograd::Function<GatedScanFn> {
  static variable_list forward(AutogradContext *ctx, const at::Tensor &x, const at::Tensor &ga, const at::Tensor &gx,
                               const at::Tensor &decay, const OptTensor &initial, const OptTensor &cu, const Scan &o) {
    auto [out, final, ckpt] = scan_fwd(x, ga, gx, decay, initial, cu, o);
    ctx->save_for_backward({x, ga, gx, decay, tensor_or_none(initial), tensor_or_none(cu), ckpt});
    ctx->set_materialize_grads(false);
    ctx->saved_data["rate"] = o.rate;
    variable_list r = {out};
    if (o.final_states) r.push_back(final);
    return r;
  }
  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    const variable_list s = ctx->get_saved_variables();
    const at::Tensor &x = s[0], &decay = s[3], &ckpt = s[6];
    const OptTensor initial = opt(s[4]), cu = opt(s[5]);
    variable_list g(7);
    const bool has_final = grads.size() > 1 && grads[1].defined();
    if (!grads[0].defined() && !has_final) return g;
    GatedScanParams p{};
    fill(p, x, s[1], s[2], decay, initial, cu, ctx->saved_data["rate"].toDouble());
    c10::DeviceGuard guard(x.device());
    at::Tensor dout = grads[0].defined() ? grads[0] : at::zeros(x.sizes(), x.options()), dfinal;
    if (!unit(dout)) dout = dout.contiguous();
    if (has_final) dfinal = grads[1].contiguous();
    for (int i = 0; i < 3; ++i) g[i] = at::empty(x.sizes(), x.options());
    g[3] = at::empty(decay.sizes(), decay.options());
    if (initial) g[4] = at::empty(initial->sizes(), initial->options());
    at::Tensor ws = bytes(gated_scan_bwd_ws_bytes(&p), "gated_scan_bwd_ws_bytes", x);
    p.ckpt = ckpt.data_ptr(), p.ws = ws.data_ptr();
    p.dout = dout.data_ptr(), p.dout_bs = dout.stride(0), p.dout_ls = dout.stride(1);
    p.dfinal_states = has_final ? dfinal.data_ptr<float>() : nullptr;
    p.dx = g[0].data_ptr(), p.dgate_a = g[1].data_ptr(), p.dgate_x = g[2].data_ptr(), p.ddecay = g[3].data_ptr();
    p.dinitial_states = initial ? g[4].data_ptr<float>() : nullptr;
    p.dx_bs = p.dgate_a_bs = p.dgate_x_bs = g[0].stride(0), p.dx_ls = p.dgate_a_ls = p.dgate_x_ls = g[0].stride(1);
    check_rc(gated_scan_bwd(&p, stream_of(x.device())), "gated_scan_bwd");
    return once(std::move(g), "gated_linear_scan");
  }
};

// gated_linear_scan_fn: out, or (out, final states); None = declined
pybind11::object gated_scan(const at::Tensor &x, const at::Tensor &ga, const at::Tensor &gx, const at::Tensor &decay, double rate,
                            const OptTensor &initial, const OptTensor &cu, bool final_states) {
  const pybind11::object no = pybind11::none();
  if (!x.is_cuda() || x.dim() != 3 || dtype_code(x) < 0 || x.numel() == 0 || python_call(x, ga, gx, decay, initial)) return no;
  const c10::Device dev = x.device();
  for (const at::Tensor *t : {&x, &ga, &gx})
    if (!on_device(*t, dev) || t->scalar_type() != x.scalar_type() || t->sizes() != x.sizes() || !unit(*t)) return no;
  const int64_t batch = x.size(0), L = x.size(1), dim = x.size(2);
  if (batch > INT32_MAX || L > INT32_MAX || dim > INT32_MAX || !decay_ok(decay, dim, dev) || !rate_ok(rate)) return no;
  int64_t seqs = batch;
  if (cu) {
    if (!on_device(cu, dev) || cu->scalar_type() != at::kInt || cu->dim() != 1 || cu->size(0) < 2 || cu->size(0) > INT32_MAX ||
        !cu->is_contiguous() || batch != 1)
      return no;
    seqs = cu->size(0) - 1;
  }
  if (initial && (!on_device(initial, dev) || initial->scalar_type() != at::kFloat || !initial->is_contiguous() ||
                  initial->dim() != 2 || initial->size(0) != seqs || initial->size(1) != dim))
    return no;
  const Scan o{rate, final_states};
  if (!records(x, ga, gx, decay, initial)) {
    auto [out, final, ckpt] = scan_fwd(x, ga, gx, decay, initial, cu, o);
    return final_states ? pybind11::object(pybind11::make_tuple(out, final)) : pybind11::cast(out);
  }
  variable_list r = GatedScanFn::apply(x, ga, gx, decay, initial, cu, o);
  return final_states ? pybind11::object(pybind11::make_tuple(r[0], r[1])) : pybind11::cast(r[0]);
}

// ------------------------------------------------------------------ one token
at::Tensor step(const at::Tensor &state, const at::Tensor &x, const at::Tensor &ga, const at::Tensor &gx, const at::Tensor &decay,
                double rate, const OptTensor &indices) {
  GatedStepParams p{};
  p.batch = (int32_t)x.size(0), p.dim = (int32_t)x.size(1), p.state_rows = (int32_t)state.size(0);
  p.dtype = dtype_code(x), p.state_dtype = dtype_code(state), p.decay_dtype = dtype_code(decay), p.rate = (float)rate;
  c10::DeviceGuard guard(x.device());
  at::Tensor out = at::empty({p.batch, p.dim}, x.options());
  p.state = state.data_ptr(), p.x = x.data_ptr(), p.gate_a = ga.data_ptr(), p.gate_x = gx.data_ptr(), p.decay = decay.data_ptr();
  p.state_batch_indices = indices ? indices->data_ptr<int32_t>() : nullptr, p.out = out.data_ptr();
  p.state_rs = state.stride(0), p.x_rs = x.stride(0), p.gate_a_rs = ga.stride(0), p.gate_x_rs = gx.stride(0), p.out_rs = p.dim;
  check_rc(gated_state_update(&p, stream_of(x.device())), "gated_state_update");
  if (!state.is_inference()) state.unsafeGetTensorImpl()->bump_version();  // a graph that has saved it has to notice
  return out;
}

// A call that autograd would record: there are no gradients, and a backward pass that comes to it raises.
struct GatedStepFn : torch::autograd::Function<GatedStepFn> {
  static at::Tensor forward(AutogradContext *, const at::Tensor &state, const at::Tensor &x, const at::Tensor &ga, const at::Tensor &gx,
                            const at::Tensor &decay, double rate, const OptTensor &indices) {
    return step(state, x, ga, gx, decay, rate, indices);
  }
  static variable_list backward(AutogradContext *, variable_list) {
    TORCH_CHECK(false, "gated_linear_state_update has no gradients; gated_linear_scan_fn over one position has");
    return {};
  }
};

OptTensor gated_step(const at::Tensor &state, const at::Tensor &x, const at::Tensor &ga, const at::Tensor &gx, const at::Tensor &decay,
                     double rate, const OptTensor &indices) {
  if (!x.is_cuda() || x.dim() != 2 || state.dim() != 2 || dtype_code(x) < 0 || dtype_code(state) < 0 || x.numel() == 0 ||
      state.size(0) == 0 || python_call(state, x, ga, gx, decay) || records(state))
    return std::nullopt;
  const c10::Device dev = x.device();
  for (const at::Tensor *t : {&x, &ga, &gx})
    if (!on_device(*t, dev) || t->scalar_type() != x.scalar_type() || t->sizes() != x.sizes() || !unit(*t)) return std::nullopt;
  const int64_t batch = x.size(0), dim = x.size(1), rows = state.size(0);
  if (!on_device(state, dev) || state.size(1) != dim || !unit(state) || !decay_ok(decay, dim, dev) || !rate_ok(rate)) return std::nullopt;
  if (batch > INT32_MAX || dim > (1 << 30) || rows > INT32_MAX || (!indices && rows < batch) || (rows > 1 && state.stride(0) < dim))
    return std::nullopt;
  if (indices && (!on_device(indices, dev) || indices->scalar_type() != at::kInt || indices->dim() != 1 || indices->size(0) != batch ||
                  !indices->is_contiguous()))
    return std::nullopt;
  if (records(x, ga, gx, decay)) return GatedStepFn::apply(state, x, ga, gx, decay, rate, indices);
  return step(state, x, ga, gx, decay, rate, indices);
}

// ------------------------------------------------------------------ the norm between two blocks
struct Block {
  double eps, scale;
  bool is_rms;
};
at::Tensor rows_of(const at::Tensor &t) {
  const at::Tensor r = t.dim() == 2 ? t : t.reshape({-1, t.size(-1)});
  return unit(r) ? r : r.contiguous();
}

void fill(NormBlockParams &p, const at::Tensor &x, const at::Tensor &residual, const at::Tensor &norm_w, const at::Tensor &next_w,
          const OptTensor &z, const OptTensor &scale, const OptTensor &norm_b, const OptTensor &next_b, const Block &o) {
  p.rows = (int32_t)x.size(0), p.dim = (int32_t)x.size(1);
  p.dtype = dtype_code(x), p.res_dtype = dtype_code(residual), p.weight_dtype = dtype_code(norm_w);
  p.is_rms = o.is_rms, p.eps = (float)o.eps, p.scale_value = (float)o.scale;
  p.x = x.data_ptr(), p.z = ptr(z), p.residual = residual.data_ptr(), p.norm_weight = norm_w.data_ptr();
  p.next_weight = next_w.data_ptr(), p.norm_bias = ptr(norm_b), p.next_bias = ptr(next_b), p.scale = ptr(scale);
  p.x_rs = x.stride(0), p.z_rs = z ? z->stride(0) : 0, p.residual_rs = residual.stride(0);
}

// out and residual_out in `sizes` (no views of rows: an output of several that is a view takes no in-place writes), the rows'
// statistics (undefined unless they are to be kept)
std::tuple<at::Tensor, at::Tensor, at::Tensor> block_fwd(at::IntArrayRef sizes, const at::Tensor &x, const at::Tensor &residual,
                                                         const at::Tensor &norm_w, const at::Tensor &next_w, const OptTensor &z,
                                                         const OptTensor &scale, const OptTensor &norm_b, const OptTensor &next_b,
                                                         const Block &o, bool keep) {
  NormBlockParams p{};
  fill(p, x, residual, norm_w, next_w, z, scale, norm_b, next_b, o);
  c10::DeviceGuard guard(x.device());
  at::Tensor out = at::empty(sizes, x.options()), total = at::empty(sizes, residual.options()), stats;
  if (keep) stats = at::empty({p.rows, 4}, x.options().dtype(at::kFloat)), p.stats = stats.data_ptr<float>();
  p.out = out.data_ptr(), p.residual_out = total.data_ptr(), p.out_rs = p.residual_out_rs = p.dim;
  check_rc(norm_block_fwd(&p, stream_of(x.device())), "norm_block_fwd");
  return {out, total, stats};
}

struct BlockNormFn : torch::autograd::Function<BlockNormFn> {
  static variable_list forward(AutogradContext *ctx, const at::Tensor &x, const at::Tensor &residual, const at::Tensor &norm_w,
                               const at::Tensor &next_w, const OptTensor &z, const OptTensor &scale, const OptTensor &norm_b,
                               const OptTensor &next_b, const Block &o) {
    const at::Tensor x2 = rows_of(x), r2 = rows_of(residual);
    const OptTensor z2 = z ? OptTensor(rows_of(*z)) : std::nullopt;
    auto [out, total, stats] = block_fwd(x.sizes(), x2, r2, norm_w, next_w, z2, scale, norm_b, next_b, o, true);
    ctx->save_for_backward({x2, r2, norm_w, next_w, tensor_or_none(z2), tensor_or_none(scale), tensor_or_none(norm_b),
                            tensor_or_none(next_b), stats});
    ctx->set_materialize_grads(false);
    ctx->saved_data["o"] = std::vector<double>{o.eps, o.scale, (double)o.is_rms};
    ctx->saved_data["shape"] = x.sizes().vec();
    return {out, total};
  }
  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    variable_list g(9);
    if (!grads[0].defined() && !grads[1].defined()) return g;
    const variable_list s = ctx->get_saved_variables();
    const at::Tensor &x = s[0], &residual = s[1], &norm_w = s[2];
    const OptTensor z = opt(s[4]), scale = opt(s[5]), norm_b = opt(s[6]), next_b = opt(s[7]);
    const std::vector<double> v = ctx->saved_data["o"].toDoubleVector();
    const Block o{v[0], v[1], v[2] != 0.0};
    const std::vector<int64_t> shape = ctx->saved_data["shape"].toIntVector();
    NormBlockParams p{};
    fill(p, x, residual, norm_w, s[3], z, scale, norm_b, next_b, o);
    c10::DeviceGuard guard(x.device());
    const at::Tensor dout = grads[0].defined() ? rows_of(grads[0]) : at::zeros(x.sizes(), x.options());
    const at::Tensor dsum = grads[1].defined() ? rows_of(grads[1]) : at::Tensor();
    const at::Tensor dx = at::empty(shape, x.options()), dres = at::empty(shape, residual.options());
    const at::Tensor dz = z ? at::empty(shape, x.options()) : at::Tensor();
    const int nsums = 2 + (scale ? 1 : 0) + (norm_b ? 1 : 0) + (next_b ? 1 : 0);
    const std::vector<at::Tensor> sums = at::empty({nsums, p.dim}, norm_w.options()).unbind(0);
    p.stats = s[8].data_ptr<float>();
    p.dout = dout.data_ptr(), p.dout_rs = dout.stride(0);
    if (dsum.defined()) p.dsum = dsum.data_ptr(), p.dsum_rs = dsum.stride(0);
    p.dx = dx.data_ptr(), p.dresidual = dres.data_ptr(), p.dx_rs = p.dresidual_rs = p.dz_rs = p.dim;
    if (z) p.dz = dz.data_ptr();
    int n = 0;
    auto sum = [&](at::Tensor &grad) -> void * {
      grad = sums[n++];
      return grad.data_ptr();
    };
    p.dnorm_weight = sum(g[2]), p.dnext_weight = sum(g[3]);
    if (scale) p.dscale = sum(g[5]);
    if (norm_b) p.dnorm_bias = sum(g[6]);
    if (next_b) p.dnext_bias = sum(g[7]);
    p.nparts = norm_block_bwd_nparts(&p);
    const int64_t carried = 2 + (norm_b ? 1 : 0) + (next_b ? 1 : 0);
    const at::Tensor parts = at::empty({carried * p.nparts * p.dim}, x.options().dtype(at::kFloat));
    p.parts = parts.data_ptr<float>();
    check_rc(norm_block_bwd(&p, stream_of(x.device())), "norm_block_bwd");
    g[0] = dx, g[1] = dres;
    if (z) g[4] = dz;
    return once(std::move(g), "block_norm");
  }
};

// block_norm_fn: (out, residual_out); None = declined
pybind11::object block_norm(const at::Tensor &x, const at::Tensor &residual, const at::Tensor &norm_w, const at::Tensor &next_w,
                            const OptTensor &z, const OptTensor &scale, double scale_value, const OptTensor &norm_b,
                            const OptTensor &next_b, double eps, bool is_rms) {
  const pybind11::object no = pybind11::none();
  if (!x.is_cuda() || x.dim() < 1 || dtype_code(x) < 0 || x.numel() == 0 ||
      python_call(x, residual, norm_w, next_w, z, scale, norm_b, next_b))
    return no;
  const c10::Device dev = x.device();
  const int64_t dim = x.size(-1);
  if (dim > 32768 || x.numel() / dim > INT32_MAX) return no;
  if (!on_device(residual, dev) || residual.sizes() != x.sizes() ||
      (residual.scalar_type() != x.scalar_type() && residual.scalar_type() != at::kFloat))
    return no;
  if (z && (!on_device(*z, dev) || z->sizes() != x.sizes() || z->scalar_type() != x.scalar_type())) return no;
  if (dtype_code(norm_w) < 0) return no;
  auto param = [&](const at::Tensor &t) {
    return on_device(t, dev) && t.scalar_type() == norm_w.scalar_type() && t.dim() == 1 && t.size(0) == dim && t.is_contiguous();
  };
  if (!param(norm_w) || !param(next_w)) return no;
  for (const OptTensor *t : {&scale, &norm_b, &next_b})
    if (*t && !param(**t)) return no;
  const Block o{eps, scale_value, is_rms};
  if (!records(x, residual, norm_w, next_w, z, scale, norm_b, next_b)) {
    auto [out, total, stats] = block_fwd(x.sizes(), rows_of(x), rows_of(residual), norm_w, next_w,
                                         z ? OptTensor(rows_of(*z)) : std::nullopt, scale, norm_b, next_b, o, false);
    return pybind11::make_tuple(out, total);
  }
  variable_list r = BlockNormFn::apply(x, residual, norm_w, next_w, z, scale, norm_b, next_b, o);
  return pybind11::make_tuple(r[0], r[1]);
}

}  // namespace

void bind_gated(pybind11::module_ &m) {
  namespace py = pybind11;
  m.def("gated_linear_scan", &gated_scan, py::arg("x"), py::arg("gate_a"), py::arg("gate_x"), py::arg("decay"), py::arg("rate"),
        py::arg("initial_states"), py::arg("cu_seqlens"), py::arg("return_final_states"),
        "Gated linear recurrence with autograd: out, or (out, final_states); None when the arguments need the Python path.");
  m.def("gated_linear_state_update", &gated_step, py::arg("state"), py::arg("x"), py::arg("gate_a"), py::arg("gate_x"), py::arg("decay"),
        py::arg("rate"), py::arg("state_batch_indices"), "One token: out, or None when the arguments need the Python path.");
  m.def("block_norm", &block_norm, py::arg("x"), py::arg("residual"), py::arg("norm_weight"), py::arg("next_weight"), py::arg("z"),
        py::arg("scale"), py::arg("scale_value"), py::arg("norm_bias"), py::arg("next_bias"), py::arg("eps"), py::arg("is_rms"),
        "(out, residual_out) with autograd; None when the arguments need the Python path.");
}

}  // namespace mamba_ext
