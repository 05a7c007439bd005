// Linear attention, its single-token step and the attention of one token over a paged cache on at::Tensor: argument checks,
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
at::Tensor bytes(int64_t n, const char *what, const at::Tensor &like) {  // undefined for none
  if (n < 0) check_rc((int)n, what);
  return n > 0 ? at::empty({n}, like.options().dtype(at::kByte)) : at::Tensor();
}
void *at_or_null(const at::Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; }

// q (.., nheads, headdim_k), k and v (.., nkvheads, ..) as the kernels take them
bool heads_ok(const at::Tensor &q, const at::Tensor &k, const at::Tensor &v, const c10::Device &dev) {
  for (const at::Tensor *t : {&k, &v}) {
    if (!on_device(*t, dev) || t->scalar_type() != q.scalar_type() || t->dim() != q.dim() || !unit(*t)) return false;
    for (int64_t i = 0; i < q.dim() - 2; ++i)
      if (t->size(i) != q.size(i)) return false;
  }
  const int64_t H = q.size(-2), G = k.size(-2), dk = q.size(-1), dv = v.size(-1);
  return G > 0 && H % G == 0 && v.size(-2) == G && k.size(-1) == dk && dk >= 1 && dv >= 1 && dk <= 256 && dv <= 256 && H <= INT32_MAX && unit(q);
}
bool decay_ok(const at::Tensor &l, int64_t heads, const c10::Device &dev) {
  return on_device(l, dev) && l.scalar_type() == at::kFloat && l.dim() == 1 && l.size(0) == heads && l.is_contiguous() && !records(l);
}
double scale_of(std::optional<double> scale, int64_t headdim) { return scale ? *scale : 1.0 / std::sqrt((double)headdim); }
bool scale_ok(double scale, double most = 3.4e38) { return std::fabs(scale) <= most; }

// ------------------------------------------------------------------ whole sequences
struct Linear {
  double scale;
  bool final_states;
};

#define MAMBA_ROWS(p, name, t) (p).name##_bs = (t).stride(0), (p).name##_ls = (t).stride(1), (p).name##_hs = (t).stride(2)

void fill(LinearAttnParams &p, const at::Tensor &q, const at::Tensor &k, const at::Tensor &v, const at::Tensor &log_decay,
          const OptTensor &initial, const OptTensor &cu, double scale) {
  p.batch = (int32_t)q.size(0), p.seqlen = (int32_t)q.size(1), p.nheads = (int32_t)q.size(2), p.nkvheads = (int32_t)k.size(2);
  p.headdim_k = (int32_t)q.size(3), p.headdim_v = (int32_t)v.size(3), p.nseq = cu ? (int32_t)cu->size(0) - 1 : 0;
  p.dtype = dtype_code(q), p.scale = (float)scale;
  p.q = q.data_ptr(), p.k = k.data_ptr(), p.v = v.data_ptr(), p.log_decay = log_decay.data_ptr<float>();
  p.initial_states = initial ? initial->data_ptr<float>() : nullptr, p.cu_seqlens = cu ? cu->data_ptr<int32_t>() : nullptr;
  MAMBA_ROWS(p, q, q), MAMBA_ROWS(p, k, k), MAMBA_ROWS(p, v, v);
}

// out, final states (undefined unless wanted)
std::tuple<at::Tensor, at::Tensor> linear_fwd(const at::Tensor &q, const at::Tensor &k, const at::Tensor &v, const at::Tensor &log_decay,
                                              const OptTensor &initial, const OptTensor &cu, const Linear &o) {
  LinearAttnParams p{};
  fill(p, q, k, v, log_decay, initial, cu, o.scale);
  c10::DeviceGuard guard(q.device());
  at::Tensor out = at::empty({p.batch, p.seqlen, p.nheads, p.headdim_v}, q.options()), final;
  if (o.final_states) final = at::empty({p.nseq ? p.nseq : p.batch, p.nheads, p.headdim_k, p.headdim_v}, q.options().dtype(at::kFloat));
  p.out = out.data_ptr(), p.final_states = static_cast<float *>(at_or_null(final));
  MAMBA_ROWS(p, out, out);
  const at::Tensor ws = bytes(linear_attn_fwd_ws_bytes(&p), "linear_attn_fwd_ws_bytes", q);
  p.ws = at_or_null(ws);
  check_rc(linear_attn_fwd(&p, stream_of(q.device())), "linear_attn_fwd");
  return {out, final};
}

struct LinearAttnFn : torch::autograd::Function<LinearAttnFn> {
  static variable_list forward(AutogradContext *ctx, const at::Tensor &q, const at::Tensor &k, const at::Tensor &v,
                               const at::Tensor &log_decay, const OptTensor &initial, const OptTensor &cu, const Linear &o) {
    auto [out, final] = linear_fwd(q, k, v, log_decay, initial, cu, o);
    ctx->save_for_backward({q, k, v, log_decay, tensor_or_none(initial), tensor_or_none(cu)});
    ctx->set_materialize_grads(false);
    ctx->saved_data["scale"] = o.scale;
    variable_list r = {out};
    if (o.final_states) r.push_back(final);
    return r;
  }
  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    const variable_list s = ctx->get_saved_variables();
    const at::Tensor &q = s[0], &k = s[1], &v = s[2];
    const OptTensor initial = opt(s[4]), cu = opt(s[5]);
    variable_list g(7);
    const bool has_final = grads.size() > 1 && grads[1].defined();
    if (!grads[0].defined() && !has_final) return g;
    LinearAttnParams p{};
    fill(p, q, k, v, s[3], initial, cu, ctx->saved_data["scale"].toDouble());
    c10::DeviceGuard guard(q.device());
    at::Tensor dout = grads[0].defined() ? grads[0] : at::zeros({p.batch, p.seqlen, p.nheads, p.headdim_v}, q.options()), dfinal;
    if (!unit(dout)) dout = dout.contiguous();
    if (has_final) dfinal = grads[1].contiguous();
    for (int i = 0; i < 3; ++i) g[i] = at::empty(s[i].sizes(), s[i].options());
    if (initial) g[4] = at::empty(initial->sizes(), initial->options());
    p.dout = dout.data_ptr(), p.dfinal_states = static_cast<float *>(at_or_null(dfinal));
    p.dq = g[0].data_ptr(), p.dk = g[1].data_ptr(), p.dv = g[2].data_ptr();
    p.dinitial_states = initial ? g[4].data_ptr<float>() : nullptr;
    MAMBA_ROWS(p, dout, dout), MAMBA_ROWS(p, dq, g[0]), MAMBA_ROWS(p, dk, g[1]), MAMBA_ROWS(p, dv, g[2]);
    const at::Tensor ws = bytes(linear_attn_bwd_ws_bytes(&p), "linear_attn_bwd_ws_bytes", q);
    p.ws = at_or_null(ws);
    check_rc(linear_attn_bwd(&p, stream_of(q.device())), "linear_attn_bwd");
    return once(std::move(g), "linear_attention");
  }
};

// linear_attention_fn: out, or (out, final states); None = declined
pybind11::object linear_attention(const at::Tensor &q, const at::Tensor &k, const at::Tensor &v, const at::Tensor &log_decay,
                                  std::optional<double> scale, const OptTensor &initial, const OptTensor &cu, bool final_states) {
  const pybind11::object no = pybind11::none();
  if (!q.is_cuda() || q.dim() != 4 || dtype_code(q) < 0 || q.numel() == 0 || python_call(q, k, v, log_decay, initial)) return no;
  const c10::Device dev = q.device();
  if (!heads_ok(q, k, v, dev) || !decay_ok(log_decay, q.size(2), dev)) return no;
  const Linear o{scale_of(scale, q.size(3)), final_states};
  if (!scale_ok(o.scale) || q.size(0) > INT32_MAX || q.size(1) > (1 << 30) || q.size(2) > (1 << 22)) return no;
  int64_t seqs = q.size(0);
  if (cu) {
    if (!on_device(cu, dev) || cu->scalar_type() != at::kInt || cu->dim() != 1 || cu->size(0) < 2 || cu->size(0) > (1 << 30) ||
        !cu->is_contiguous() || q.size(0) != 1)
      return no;
    seqs = cu->size(0) - 1;
  }
  if (initial && (!on_device(initial, dev) || initial->scalar_type() != at::kFloat || !initial->is_contiguous() ||
                  initial->sizes() != at::IntArrayRef({seqs, q.size(2), q.size(3), v.size(3)})))
    return no;
  if (!records(q, k, v, initial)) {
    auto [out, final] = linear_fwd(q, k, v, log_decay, initial, cu, o);
    return final_states ? pybind11::object(pybind11::make_tuple(out, final)) : pybind11::cast(out);
  }
  variable_list r = LinearAttnFn::apply(q, k, v, log_decay, initial, cu, o);
  return final_states ? pybind11::object(pybind11::make_tuple(r[0], r[1])) : pybind11::cast(r[0]);
}

// ------------------------------------------------------------------ one token
at::Tensor step(const at::Tensor &state, const at::Tensor &q, const at::Tensor &k, const at::Tensor &v, const at::Tensor &log_decay,
                double scale, const OptTensor &indices) {
  LinearAttnStepParams p{};
  p.batch = (int32_t)q.size(0), p.nheads = (int32_t)q.size(1), p.nkvheads = (int32_t)k.size(1), p.headdim_k = (int32_t)q.size(2);
  p.headdim_v = (int32_t)v.size(2), p.state_rows = (int32_t)state.size(0), p.dtype = dtype_code(q), p.state_dtype = dtype_code(state);
  p.scale = (float)scale;
  c10::DeviceGuard guard(q.device());
  at::Tensor out = at::empty({p.batch, p.nheads, p.headdim_v}, q.options());
  p.state = state.data_ptr(), p.q = q.data_ptr(), p.k = k.data_ptr(), p.v = v.data_ptr(), p.log_decay = log_decay.data_ptr<float>();
  p.state_batch_indices = indices ? indices->data_ptr<int32_t>() : nullptr, p.out = out.data_ptr();
  p.state_rs = state.stride(0), p.q_bs = q.stride(0), p.q_hs = q.stride(1), p.k_bs = k.stride(0), p.k_hs = k.stride(1);
  p.v_bs = v.stride(0), p.v_hs = v.stride(1), p.out_bs = out.stride(0), p.out_hs = out.stride(1);
  check_rc(linear_attn_state_update(&p, stream_of(q.device())), "linear_attn_state_update");
  if (!state.is_inference()) state.unsafeGetTensorImpl()->bump_version();  // a graph that has saved it has to notice
  return out;
}

// A call that autograd would record: there are no gradients, and a backward pass that comes to it raises.
struct LinearStepFn : torch::autograd::Function<LinearStepFn> {
  static at::Tensor forward(AutogradContext *, const at::Tensor &state, const at::Tensor &q, const at::Tensor &k, const at::Tensor &v,
                            const at::Tensor &log_decay, double scale, const OptTensor &indices) {
    return step(state, q, k, v, log_decay, scale, indices);
  }
  static variable_list backward(AutogradContext *, variable_list) {
    TORCH_CHECK(false, "linear_attention_state_update has no gradients; linear_attention_fn over one position has");
    return {};
  }
};

OptTensor linear_step(const at::Tensor &state, const at::Tensor &q, const at::Tensor &k, const at::Tensor &v, const at::Tensor &log_decay,
                      std::optional<double> scale, const OptTensor &indices) {
  if (!q.is_cuda() || q.dim() != 3 || state.dim() != 4 || dtype_code(q) < 0 || dtype_code(state) < 0 || q.numel() == 0 ||
      state.size(0) == 0 || python_call(state, q, k, v, log_decay) || records(state))
    return std::nullopt;
  const c10::Device dev = q.device();
  if (!heads_ok(q, k, v, dev) || !decay_ok(log_decay, q.size(1), dev) || !on_device(state, dev)) return std::nullopt;
  const int64_t batch = q.size(0), H = q.size(1), dk = q.size(2), dv = v.size(2), rows = state.size(0);
  const double s = scale_of(scale, dk);
  if (!scale_ok(s) || state.size(1) != H || state.size(2) != dk || state.size(3) != dv) return std::nullopt;
  if ((dv > 1 && state.stride(3) != 1) || (dk > 1 && state.stride(2) != dv) || (H > 1 && state.stride(1) != dk * dv) ||
      (rows > 1 && state.stride(0) < H * dk * dv))
    return std::nullopt;
  if (batch > INT32_MAX || rows > INT32_MAX || H > 65535 || (!indices && rows < batch)) return std::nullopt;
  if (indices && (!on_device(indices, dev) || indices->scalar_type() != at::kInt || indices->dim() != 1 || indices->size(0) != batch ||
                  !indices->is_contiguous()))
    return std::nullopt;
  if (records(q, k, v)) return LinearStepFn::apply(state, q, k, v, log_decay, s, indices);
  return step(state, q, k, v, log_decay, s, indices);
}

// ------------------------------------------------------------------ one token over a paged cache
struct Paged {
  double scale;
  int64_t window;
};

at::Tensor paged(const at::Tensor &q, const OptTensor &k, const OptTensor &v, const at::Tensor &k_cache, const at::Tensor &v_cache,
                 const at::Tensor &table, const at::Tensor &lens, const Paged &o) {
  PagedAttnParams p{};
  p.batch = (int32_t)q.size(0), p.nheads = (int32_t)q.size(1), p.nkvheads = (int32_t)k_cache.size(2), p.headdim_k = (int32_t)q.size(2);
  p.headdim_v = (int32_t)v_cache.size(3), p.num_pages = (int32_t)k_cache.size(0), p.page_size = (int32_t)k_cache.size(1);
  p.max_pages = (int32_t)table.size(1), p.window = (int32_t)o.window, p.dtype = dtype_code(q), p.scale = (float)o.scale;
  c10::DeviceGuard guard(q.device());
  at::Tensor out = at::empty({p.batch, p.nheads, p.headdim_v}, q.options());
  p.q = q.data_ptr(), p.k_cache = k_cache.data_ptr(), p.v_cache = v_cache.data_ptr(), p.block_table = table.data_ptr<int32_t>();
  p.cache_seqlens = lens.data_ptr<int32_t>(), p.out = out.data_ptr();
  p.q_bs = q.stride(0), p.q_hs = q.stride(1), p.out_bs = out.stride(0), p.out_hs = out.stride(1), p.table_bs = table.stride(0);
  if (k) {
    p.k = k->data_ptr(), p.v = v->data_ptr();
    p.k_bs = k->stride(0), p.k_hs = k->stride(1), p.v_bs = v->stride(0), p.v_hs = v->stride(1);
  }
  p.kc_ps = k_cache.stride(0), p.kc_ls = k_cache.stride(1), p.kc_hs = k_cache.stride(2);
  p.vc_ps = v_cache.stride(0), p.vc_ls = v_cache.stride(1), p.vc_hs = v_cache.stride(2);
  p.nsplit = paged_attn_parts(&p);
  if (p.nsplit < 0) check_rc(p.nsplit, "paged_attn_parts");
  const at::Tensor ws = bytes(paged_attn_ws_bytes(&p), "paged_attn_ws_bytes", q);
  p.ws = static_cast<float *>(at_or_null(ws));
  check_rc(paged_attn_update(&p, stream_of(q.device())), "paged_attn_update");
  if (k)
    for (const at::Tensor *t : {&k_cache, &v_cache})
      if (!t->is_inference()) t->unsafeGetTensorImpl()->bump_version();  // a graph that has saved it has to notice
  return out;
}

struct PagedFn : torch::autograd::Function<PagedFn> {
  static at::Tensor forward(AutogradContext *, const at::Tensor &q, const OptTensor &k, const OptTensor &v, const at::Tensor &k_cache,
                            const at::Tensor &v_cache, const at::Tensor &table, const at::Tensor &lens, const Paged &o) {
    return paged(q, k, v, k_cache, v_cache, table, lens, o);
  }
  static variable_list backward(AutogradContext *, variable_list) {
    TORCH_CHECK(false, "paged_attention_update has no gradients: it is made for generating");
    return {};
  }
};

// The ordinary layouts, dense or (pages, heads, positions, head size) by strides; anything else is looked at in Python.
bool cache_ok(const at::Tensor &t, const at::Tensor &q, const c10::Device &dev) {
  if (!on_device(t, dev) || t.dim() != 4 || t.scalar_type() != q.scalar_type() || t.numel() == 0 || t.size(0) > INT32_MAX ||
      (t.stride(3) != 1 && t.size(3) > 1))
    return false;
  const int64_t d = t.size(3), in = t.stride(1) < t.stride(2) ? 1 : 2, out = 3 - in;
  return t.stride(in) >= d && t.stride(out) >= t.stride(in) * t.size(in) && t.stride(0) >= t.stride(out) * t.size(out);
}
bool counts_ok(const at::Tensor &t, const c10::Device &dev) { return on_device(t, dev) && t.scalar_type() == at::kInt && t.is_contiguous(); }

OptTensor paged_attention(const at::Tensor &q, const OptTensor &k, const OptTensor &v, const at::Tensor &k_cache, const at::Tensor &v_cache,
                          const at::Tensor &table, const at::Tensor &lens, std::optional<double> scale, std::optional<int64_t> window) {
  if (!q.is_cuda() || q.dim() != 3 || dtype_code(q) < 0 || q.numel() == 0 || k.has_value() != v.has_value() ||
      python_call(q, k, v, k_cache, v_cache) || (k && records(k_cache, v_cache)))
    return std::nullopt;
  const c10::Device dev = q.device();
  if (!unit(q) || !cache_ok(k_cache, q, dev) || !cache_ok(v_cache, q, dev)) return std::nullopt;
  for (int i = 0; i < 3; ++i)
    if (k_cache.size(i) != v_cache.size(i)) return std::nullopt;
  const int64_t batch = q.size(0), H = q.size(1), G = k_cache.size(2), dk = q.size(2), dv = v_cache.size(3);
  if (k) {
    if (!heads_ok(q, *k, *v, dev) || k->size(1) != G || v->size(2) != dv) return std::nullopt;
  } else if (H % G != 0) {
    return std::nullopt;
  }
  if (k_cache.size(3) != dk || dk > 256 || dv > 256 || H > INT32_MAX || batch > 65535) return std::nullopt;
  if (!counts_ok(table, dev) || table.dim() != 2 || table.size(0) != batch || table.size(1) < 1) return std::nullopt;
  if (!counts_ok(lens, dev) || lens.dim() != 1 || lens.size(0) != batch) return std::nullopt;
  if (k_cache.size(1) > (1 << 30) || table.size(1) > (1 << 30) || table.size(1) * k_cache.size(1) > (1 << 30)) return std::nullopt;
  const Paged o{scale_of(scale, dk), window.value_or(0)};
  if (!scale_ok(o.scale, 2e38) || (window && (*window < 1 || *window > INT32_MAX))) return std::nullopt;
  if (records(q, k, v, k_cache, v_cache)) return PagedFn::apply(q, k, v, k_cache, v_cache, table, lens, o);
  return paged(q, k, v, k_cache, v_cache, table, lens, o);
}

#undef MAMBA_ROWS

}  // namespace

void bind_attention(pybind11::module_ &m) {
  namespace py = pybind11;
  m.def("linear_attention", &linear_attention, py::arg("q"), py::arg("k"), py::arg("v"), py::arg("log_decay"), py::arg("scale"),
        py::arg("initial_states"), py::arg("cu_seqlens"), py::arg("return_final_states"),
        "Linear attention with autograd: out, or (out, final_states); None when the arguments need the Python path.");
  m.def("linear_attention_state_update", &linear_step, py::arg("state"), py::arg("q"), py::arg("k"), py::arg("v"), py::arg("log_decay"),
        py::arg("scale"), py::arg("state_batch_indices"), "One token: out, or None when the arguments need the Python path.");
  m.def("paged_attention_update", &paged_attention, py::arg("q"), py::arg("k"), py::arg("v"), py::arg("k_cache"), py::arg("v_cache"),
        py::arg("block_table"), py::arg("cache_seqlens"), py::arg("scale"), py::arg("window"),
        "One token over a paged cache: out, or None when the arguments need the Python path.");
}

}  // namespace mamba_ext
