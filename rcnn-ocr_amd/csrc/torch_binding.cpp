// torch binding of the sequence operators (crnn_layernorm_*, crnn_linear_*, crnn_gated_scan_*): torch.ops.crnn.layer_norm,
// linear and gated_scan, differentiable once. The rest of the library is driven by the engine, which makes one host call per
// kernel; these are called one by one from a user's program, whose backward torch runs on a thread of its own: as Python
// autograd functions over ctypes a small training call cost 100 us of host time (8192 x 512 layer norm: 18 us of GPU time).
//
// The C ABI stays free of torch types: this file only unpacks tensors, allocates results and workspaces on the current stream
// of the tensors' device and calls it. Its symbols are those of the libcrnn_hip.so that crnn_hip/_lib.py has loaded.
#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/variable.h>
#include <torch/library.h>

#include "crnn_hip.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
typedef std::optional<Tensor> OptTensor;

// ---------------------------------------------------------------- arguments
int dtype_code(const char* op, const Tensor& t) {
  if (t.scalar_type() == at::kBFloat16) return CRNN_BF16;
  TORCH_CHECK_VALUE(t.scalar_type() == at::kFloat, op, ": unsupported compute dtype ", t.scalar_type(), " (fp32 or bf16)");
  return CRNN_F32;
}
void require_device(const Tensor& t) {
  TORCH_CHECK(t.is_cuda(), "crnn_hip ops run only on a HIP device (no CPU fallback); got a tensor on ", t.device());
}
void check(const char* op, const char* name, const Tensor& t, at::IntArrayRef shape, const Tensor& like) {
  TORCH_CHECK_VALUE(t.sizes() == shape, op, ": ", name, " must have shape ", shape, ", got ", t.sizes());
  TORCH_CHECK_VALUE(t.device() == like.device(), op, ": ", name, " must be on ", like.device(), ", got ", t.device());
}
void check_type(const char* op, const char* name, const Tensor& t, at::ScalarType a, at::ScalarType b) {
  TORCH_CHECK_VALUE(t.scalar_type() == a || t.scalar_type() == b, op, ": ", name, " must be ", a, a == b ? "" : " or fp32", ", got ",
                    t.scalar_type());
}
bool has(const OptTensor& t) { return t.has_value() && t->defined(); }
// The kernels take addresses, so only plain tensors, run at once, will do. Tracers (torch.compile, make_fx, fake tensors), torch.func's
// derivatives and subclasses with a __torch_dispatch__ are refused: make_fx over real tensors would record the results' allocation and not
// the kernel that fills them. (torch.vmap calls the operator for each sample on plain tensors;
// a batch of upstream gradients, is_grads_batched, is refused.)
bool is_plain(const Tensor& t) {
  using c10::DispatchKey;
  static constexpr c10::DispatchKeySet wrapped(
      {DispatchKey::Python, DispatchKey::FuncTorchGradWrapper, DispatchKey::FuncTorchBatched, DispatchKey::Functionalize, DispatchKey::Batched});
  return !t.unsafeGetTensorImpl()->key_set().has_any(wrapped);
}
void check_eager(const char* op, std::initializer_list<OptTensor> ts) {
  using Mode = c10::impl::TorchDispatchModeTLS;
  using Key = c10::impl::TorchDispatchModeKey;
  bool plain = true;
  for (const OptTensor& t : ts) plain = plain && (!has(t) || is_plain(*t));
  if (Mode::any_modes_set())
    plain = plain && !Mode::get_mode(Key::FAKE) && !Mode::get_mode(Key::PROXY) && !Mode::get_mode(Key::FUNCTIONAL);
  TORCH_CHECK(plain, op, " runs eagerly, on plain tensors: no tracing (torch.compile, make_fx, fake tensors), no torch.func derivatives, no "
              "subclasses with a __torch_dispatch__; torch.compiler.disable keeps it out of a compiled region");
}
// whether autograd has to record the call. Forward-mode tangents are refused: a plain call would drop them silently
bool records(const char* op, std::initializer_list<OptTensor> ts) {
  bool grad = false;
  for (const OptTensor& t : ts) {
    if (!has(t)) continue;
    TORCH_CHECK(!t->_fw_grad(0).defined(), op, " has no forward-mode derivative");
    grad = grad || t->requires_grad();
  }
  return grad && at::GradMode::is_enabled();
}
// the values where the memory holds their negatives (views such as z.conj().imag, also as upstream gradients)
Tensor values(const Tensor& t) { return t.is_neg() ? t.resolve_neg() : t; }
Tensor contiguous(const OptTensor& t) { return has(t) ? values(*t).contiguous() : Tensor(); }
void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
float* fptr(const Tensor& t) { return (float*)ptr(t); }

// [..., N] as m rows of N contiguous elements, ld apart: the tensor itself where its strides allow, else a contiguous copy
struct Rows {
  Tensor t;
  int64_t m, ld;
};
Rows rows(const Tensor& t_) {
  const Tensor t = values(t_);
  const int64_t n = t.size(-1), m = n ? t.numel() / n : 0, d = t.dim();
  if (t.is_contiguous()) return {t, m, n};
  if (d >= 2 && (t.stride(-1) == 1 || n == 1) && t.stride(-2) >= n) {
    bool even = true;
    for (int64_t i = 0; i + 2 < d; ++i) even = even && t.stride(i) == t.stride(i + 1) * t.size(i + 1);
    if (even) return {t, m, t.stride(-2)};
  }
  return {t.contiguous(), m, n};
}
// channels contiguous
Tensor chan(const Tensor& t) { return t.stride(-1) == 1 || t.size(-1) == 1 ? values(t) : t.contiguous(); }

Tensor bytes(size_t n, const Tensor& like) {
  return n ? at::empty({(int64_t)n}, like.options().dtype(at::kByte)) : Tensor();
}
Tensor floats(at::IntArrayRef shape, const Tensor& like) { return at::empty(shape, like.options().dtype(at::kFloat)); }

void* stream(const Tensor& t) { return (void*)c10::hip::getCurrentHIPStream(t.get_device()).stream(); }
void call(int rc, const char* name) { TORCH_CHECK(rc == 0, name, " failed (hip error ", rc, "): ", crnn_last_error_string()); }

// What the backward reads goes through autograd's saved tensors, and a saved-tensor hook (offloading to the host and back,
// torch.autograd.graph.save_on_cpu) may give back another layout than it took. So nothing about a layout is kept beside them: strides are
// read from what comes back, and a tensor of another shape, type or device is refused.
void save(AutogradContext* ctx, const variable_list& ts) {
  std::vector<int64_t> meta;
  for (const Tensor& t : ts) {
    meta.push_back(t.defined() ? t.dim() : -1);
    if (!t.defined()) continue;
    meta.push_back((int64_t)t.scalar_type());
    meta.push_back(t.get_device());
    meta.insert(meta.end(), t.sizes().begin(), t.sizes().end());
  }
  ctx->save_for_backward(ts);
  ctx->saved_data["meta"] = std::move(meta);
}
variable_list saved(const char* op, AutogradContext* ctx) {
  variable_list ts = ctx->get_saved_variables();
  const auto meta = ctx->saved_data["meta"].toIntVector();
  const int64_t* p = meta.data();
  for (const Tensor& t : ts) {
    const int64_t dim = *p++;
    TORCH_CHECK(t.defined() == (dim >= 0), op, ": a saved-tensor hook gave back ", t.defined() ? "a tensor for none" : "no tensor");
    if (dim < 0) continue;
    const auto type = (at::ScalarType)p[0];
    const int64_t dev = p[1];
    const at::IntArrayRef shape(p + 2, dim);
    p += 2 + dim;
    const bool plain = is_plain(t) && t.layout() == at::kStrided;
    TORCH_CHECK(plain && t.is_cuda() && t.get_device() == dev && t.scalar_type() == type && t.sizes() == shape, op,
                ": a saved-tensor hook gave back a ", plain ? "" : "wrapped or sparse ", t.scalar_type(), " tensor of shape ", t.sizes(), " on ",
                t.device(), " for a ", type, " one of shape ", shape, " on device ", dev);
  }
  return ts;
}

// A captured backward may not hand its gradients to a node of the default stream: autograd would order that stream behind the
// captured one, which no capture allows, and torch does not survive it. Such a node is a leaf's accumulator that an eager graph,
// built on the default stream and still alive, holds on to. Refused here, before autograd does it.
void check_capture(const char* op) {
  if (!c10::hip::getCurrentHIPStream().stream() || c10::hip::currentStreamCaptureStatusMayInitCtx() == c10::hip::CaptureStatus::None) return;
  const auto node = torch::autograd::get_current_node();
  if (!node) return;
  for (size_t i = 0; i < node->num_outputs(); ++i) {
    const auto& e = node->next_edge(i);
    if (!e.is_valid() || !node->task_should_compute_output(i)) continue;
    const auto s = e.function->stream();
    TORCH_CHECK(!s || s->id() != 0, op, ": this backward is being captured into a graph, but an eager graph that was built on the default stream "
                "and is still alive holds one of its inputs: drop that graph (its outputs and losses) before the capture");
  }
}

// create_graph: the results refuse to be differentiated again
variable_list once(const char* op, variable_list grads) {
  if (!at::GradMode::is_enabled()) return grads;
  variable_list in;
  for (auto& g : grads)
    if (g.defined()) in.push_back(g.detach().requires_grad_(true));
  auto err = std::make_shared<torch::autograd::DelayedError>(std::string(op) + " is differentiable once", (int64_t)in.size());
  variable_list out = (*err)(std::move(in));
  size_t k = 0;
  for (auto& g : grads)
    if (g.defined()) g = out[k++];
  return grads;
}

// ---------------------------------------------------------------- layer norm
Tensor layer_norm_run(const Rows& x, at::IntArrayRef shape, const Tensor& w, const Tensor& b, double eps, const Tensor& stats) {
  const int dt = dtype_code("layer_norm", x.t);
  const int64_t n = shape.back();
  Tensor y = at::empty(shape, x.t.options());
  float* s = fptr(stats);
  call(crnn_layernorm_fwd(dt, ptr(x.t), x.ld, fptr(w), fptr(b), ptr(y), n, s, s ? s + x.m : nullptr, x.m, (int)n, (float)eps, stream(x.t)),
       "crnn_layernorm_fwd");
  return y;
}

struct LayerNormFn : public torch::autograd::Function<LayerNormFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const OptTensor& weight, const OptTensor& bias, double eps) {
    at::AutoDispatchBelowADInplaceOrView below;
    const Rows r = rows(x);
    const Tensor w = contiguous(weight), b = contiguous(bias);
    Tensor stats = floats({2 * r.m}, x);   // mean, then rstd of every row
    Tensor y = layer_norm_run(r, x.sizes(), w, b, eps, stats);
    save(ctx, {r.t, w, stats});
    ctx->saved_data["w"] = has(weight);
    ctx->saved_data["b"] = has(bias);
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    const auto kept = saved("layer_norm", ctx);
    const Tensor& x = kept[0];
    const bool has_w = ctx->saved_data["w"].toBool(), has_b = ctx->saved_data["b"].toBool();
    size_t e = 0;
    const bool need_x = ctx->needs_input_grad(e++);
    const bool need_w = has_w && ctx->needs_input_grad(e++), need_b = has_b && ctx->needs_input_grad(e++);
    variable_list out(4);
    {
      at::AutoDispatchBelowADInplaceOrView below;
      const c10::OptionalDeviceGuard guard(x.device());
      check_eager("layer_norm", {g[0]});
      check_capture("layer_norm");
      const Rows xr = rows(x), dy = rows(g[0]);
      const Tensor w = contiguous(kept[1]), stats = contiguous(kept[2]);
      const int64_t n = x.size(-1), m = stats.numel() / 2;
      const int dt = dtype_code("layer_norm", x);
      if (need_x) out[0] = at::empty(x.sizes(), x.options());
      if (need_w) out[1] = floats({n}, x);
      if (need_b) out[2] = floats({n}, x);
      const size_t need = need_w || need_b ? crnn_layernorm_bwd_workspace(dt, m, (int)n) : 0;
      const Tensor ws = bytes(need, x);
      float* s = fptr(stats);
      call(crnn_layernorm_bwd(dt, ptr(dy.t), dy.ld, ptr(xr.t), xr.ld, fptr(w), s, s + m, nullptr, 0, ptr(out[0]), n, fptr(out[1]), fptr(out[2]), 0,
                              fptr(ws), need, m, (int)n, stream(x)),
           "crnn_layernorm_bwd");
    }
    return once("layer_norm", std::move(out));
  }
};

Tensor layer_norm(const Tensor& x, const OptTensor& weight, const OptTensor& bias, double eps) {
  dtype_code("layer_norm", x);
  TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) >= 1, "layer_norm: x needs a last axis of at least one element, got ", x.sizes());
  const int64_t n = x.size(-1);
  TORCH_CHECK_VALUE(n <= 1 << 30, "layer_norm: the last axis must be at most 2^30, got ", n);
  for (int i = 0; i < 2; ++i) {
    const OptTensor& p = i ? bias : weight;
    if (!has(p)) continue;
    check("layer_norm", i ? "bias" : "weight", *p, {n}, x);
    check_type("layer_norm", i ? "bias" : "weight", *p, at::kFloat, at::kFloat);
  }
  TORCH_CHECK_VALUE(eps >= 0, "layer_norm: eps must be >= 0, got ", eps);
  check_eager("layer_norm", {x, weight, bias});
  require_device(x);
  const c10::OptionalDeviceGuard guard(x.device());
  if (records("layer_norm", {x, weight, bias}))
    return LayerNormFn::apply(x, weight, bias, eps);
  return layer_norm_run(rows(x), x.sizes(), contiguous(weight), contiguous(bias), eps, Tensor());
}

// ---------------------------------------------------------------- linear
Tensor linear_run(const Rows& x, at::IntArrayRef shape, const Rows& w, const Tensor& b, int act, const OptTensor& residual, const Tensor& z) {
  const int dt = dtype_code("linear", x.t);
  const int64_t n = w.t.size(0), k = w.t.size(1);
  auto out = shape.vec();
  out.back() = n;
  Tensor y = at::empty(out, x.t.options());
  Rows r{Tensor(), 0, n};
  if (has(residual)) r = rows(*residual);
  const size_t need = crnn_linear_fwd_workspace(dt, ptr(x.t), x.ld, ptr(w.t), w.ld, x.m, (int)n, (int)k);
  const Tensor ws = bytes(need, x.t);
  call(crnn_linear_fwd(dt, ptr(x.t), x.ld, ptr(w.t), w.ld, ptr(b), b.defined() && b.scalar_type() == at::kFloat, act, ptr(r.t), r.ld, ptr(y), n,
                       ptr(z), n, ptr(ws), need, x.m, (int)n, (int)k, stream(x.t)),
       "crnn_linear_fwd");
  return y;
}

struct LinearFn : public torch::autograd::Function<LinearFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, const OptTensor& bias, int64_t act,
                        const OptTensor& residual) {
    at::AutoDispatchBelowADInplaceOrView below;
    const Rows r = rows(x), w = rows(weight);
    const Tensor z = act ? at::empty({r.m, weight.size(0)}, x.options()) : Tensor();   // the pre-activation
    Tensor y = linear_run(r, x.sizes(), w, contiguous(bias), (int)act, residual, z);
    save(ctx, {r.t, w.t, z});
    ctx->saved_data["act"] = act;
    ctx->saved_data["b"] = has(bias) ? (bias->scalar_type() == at::kFloat ? 2 : 1) : 0;   // 2: fp32
    ctx->saved_data["r"] = has(residual);
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    const auto kept = saved("linear", ctx);
    const Tensor &x = kept[0], &w = kept[1];
    const int64_t bias = ctx->saved_data["b"].toInt();
    size_t e = 0;
    const bool need_x = ctx->needs_input_grad(e++), need_w = ctx->needs_input_grad(e++);
    const bool need_b = bias && ctx->needs_input_grad(e++);
    const bool need_r = ctx->saved_data["r"].toBool() && ctx->needs_input_grad(e++);
    variable_list out(5);
    {
      at::AutoDispatchBelowADInplaceOrView below;
      const c10::OptionalDeviceGuard guard(x.device());
      check_eager("linear", {g[0]});
      check_capture("linear");
      if (need_x || need_w || need_b) {
        const int dt = dtype_code("linear", x), act = (int)ctx->saved_data["act"].toInt();
        const Rows xr = rows(x), wr = rows(w), dy = rows(g[0]);
        const Tensor z = contiguous(kept[2]);
        const int64_t n = w.size(0), k = w.size(1), m = xr.m;
        if (need_x) out[0] = at::empty(x.sizes(), x.options());
        if (need_w) out[1] = at::empty({n, k}, w.options());
        if (need_b) out[2] = bias == 2 ? floats({n}, x) : at::empty({n}, x.options());
        const size_t need = crnn_linear_bwd_workspace(dt, ptr(dy.t), dy.ld, ptr(xr.t), xr.ld, ptr(wr.t), wr.ld, act, need_x, need_w, need_b, m,
                                                      (int)n, (int)k);
        const Tensor ws = bytes(need, x);
        call(crnn_linear_bwd(dt, ptr(dy.t), dy.ld, ptr(xr.t), xr.ld, ptr(wr.t), wr.ld, ptr(z), n, act, ptr(out[0]), k, ptr(out[1]),
                             w.scalar_type() == at::kFloat, ptr(out[2]), bias == 2, 0, ptr(ws), need, m, (int)n, (int)k, stream(x)),
             "crnn_linear_bwd");
      }
      if (need_r) out[4] = g[0];
    }
    return once("linear", std::move(out));
  }
};

Tensor linear(const Tensor& x, const Tensor& weight, const OptTensor& bias, int64_t act, const OptTensor& residual) {
  dtype_code("linear", x);
  TORCH_CHECK_VALUE(act >= CRNN_ACT_NONE && act <= CRNN_ACT_SILU, "linear: unknown activation ", act);
  TORCH_CHECK_VALUE(x.dim() >= 1, "linear: x needs at least one axis");
  check_type("linear", "weight", weight, x.scalar_type(), x.scalar_type());
  const int64_t k = x.size(-1);
  TORCH_CHECK_VALUE(weight.dim() == 2 && weight.size(1) == k && weight.size(0) >= 1 && k >= 1, "linear: weight must be [N, ", k,
                    "] with N, K >= 1, got ", weight.sizes());
  const int64_t n = weight.size(0);
  TORCH_CHECK_VALUE(n < 1LL << 31 && k < 1LL << 31, "linear: sizes must be below 2^31, got ", weight.sizes());
  check("linear", "weight", weight, weight.sizes(), x);
  if (has(bias)) {
    check("linear", "bias", *bias, {n}, x);
    check_type("linear", "bias", *bias, x.scalar_type(), at::kFloat);
  }
  if (has(residual)) {
    auto shape = x.sizes().vec();
    shape.back() = n;
    check("linear", "residual", *residual, shape, x);
    check_type("linear", "residual", *residual, x.scalar_type(), x.scalar_type());
  }
  check_eager("linear", {x, weight, bias, residual});
  require_device(x);
  const c10::OptionalDeviceGuard guard(x.device());
  if (records("linear", {x, weight, bias, residual}))
    return LinearFn::apply(x, weight, bias, act, residual);
  return linear_run(rows(x), x.sizes(), rows(weight), contiguous(bias), (int)act, residual, Tensor());
}

// ---------------------------------------------------------------- gated scan
Tensor scan_run(const Tensor& f, const Tensor& v, const Tensor& h0, const Tensor& lengths, int dir, const Tensor& hT, const Tensor& ckpt) {
  const int dt = dtype_code("gated_scan", f), B = (int)f.size(0), T = (int)f.size(1), D = (int)f.size(2);
  Tensor y = at::empty(f.sizes(), f.options().memory_format(at::MemoryFormat::Contiguous));
  const size_t need = crnn_gated_scan_workspace(dt, B, T, D, dir);
  const Tensor ws = bytes(need, f);
  call(crnn_gated_scan_fwd(dt, ptr(f), f.stride(0), f.stride(1), ptr(v), v.stride(0), v.stride(1), fptr(h0), (const int*)ptr(lengths), ptr(y),
                           (long)T * D, D, fptr(hT), fptr(ckpt), fptr(ws), need, B, T, D, dir, stream(f)),
       "crnn_gated_scan_fwd");
  return y;
}

struct GatedScanFn : public torch::autograd::Function<GatedScanFn> {
  static variable_list forward(AutogradContext* ctx, const Tensor& f_, const Tensor& v_, const OptTensor& h0, const OptTensor& lengths,
                               int64_t dir, bool state) {
    at::AutoDispatchBelowADInplaceOrView below;
    const Tensor f = chan(f_), v = chan(v_), len = has(lengths) ? *lengths : Tensor();
    const int B = (int)f.size(0), T = (int)f.size(1), D = (int)f.size(2);
    const Tensor ckpt = bytes(crnn_gated_scan_ckpt_bytes(dtype_code("gated_scan", f), B, T, D, (int)dir), f);   // the backward starts from it
    const Tensor hT = state ? floats({B, D}, f) : Tensor();
    Tensor y = scan_run(f, v, contiguous(h0), len, (int)dir, hT, ckpt);
    save(ctx, {f, v, len, ckpt});
    ctx->saved_data["dir"] = dir;
    ctx->saved_data["h0"] = has(h0);
    ctx->set_materialize_grads(false);
    if (state) return {y, hT};
    return {y};
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    const auto kept = saved("gated_scan", ctx);
    const int dir = (int)ctx->saved_data["dir"].toInt(), B = (int)kept[0].size(0), T = (int)kept[0].size(1), D = (int)kept[0].size(2);
    const bool need_f = ctx->needs_input_grad(0), need_v = ctx->needs_input_grad(1);
    const bool need_h = ctx->saved_data["h0"].toBool() && ctx->needs_input_grad(2);
    variable_list out(6);
    {
      at::AutoDispatchBelowADInplaceOrView below;
      const c10::OptionalDeviceGuard guard(kept[0].device());
      check_eager("gated_scan", {g[0], g.size() > 1 ? g[1] : Tensor()});
      check_capture("gated_scan");
      const Tensor f = chan(kept[0]), v = chan(kept[1]), len = contiguous(kept[2]), ckpt = contiguous(kept[3]);
      const int dt = dtype_code("gated_scan", f);
      // only the final state was used: no upstream gradient for y
      const Tensor dy = g[0].defined() ? chan(g[0]) : at::zeros(f.sizes(), f.options());
      const Tensor dhT = g.size() > 1 && g[1].defined() ? contiguous(g[1]) : Tensor();
      const auto opt = f.options().memory_format(at::MemoryFormat::Contiguous);
      Tensor df = at::empty(f.sizes(), opt), dv = at::empty(f.sizes(), opt), dh0 = need_h ? floats({B, D}, f) : Tensor();
      const size_t need = crnn_gated_scan_workspace(dt, B, T, D, dir);
      const Tensor ws = bytes(need, f);
      call(crnn_gated_scan_bwd(dt, ptr(dy), dy.stride(0), dy.stride(1), ptr(f), f.stride(0), f.stride(1), ptr(v), v.stride(0), v.stride(1),
                               (const int*)ptr(len), fptr(dhT), fptr(ckpt), ptr(df), (long)T * D, D, ptr(dv), (long)T * D, D, fptr(dh0), fptr(ws),
                               need, B, T, D, dir, stream(f)),
           "crnn_gated_scan_bwd");
      if (need_f) out[0] = df;
      if (need_v) out[1] = dv;
      out[2] = dh0;
    }
    return once("gated_scan", std::move(out));
  }
};

// no byte of a is a byte of b (taking each from its first to its last element)
bool apart(const Tensor& a, const Tensor& b) {
  if (!a.numel() || !b.numel()) return true;
  auto end = [](const Tensor& t) {
    int64_t n = 1;
    for (int64_t i = 0; i < t.dim(); ++i) n += (t.size(i) - 1) * t.stride(i);
    return (const char*)t.data_ptr() + n * t.element_size();
  };
  return end(a) <= (const char*)b.data_ptr() || end(b) <= (const char*)a.data_ptr();
}

void check_scan(const char* op, const Tensor& f, const Tensor& v, int64_t dims) {
  dtype_code(op, f);
  TORCH_CHECK_VALUE(f.dim() == dims, op, ": f must have ", dims, " axes, got ", f.sizes());
  for (int64_t s : f.sizes()) TORCH_CHECK_VALUE(s <= 1LL << 30, op, ": sizes must be at most 2^30, got ", f.sizes());
  check(op, "v", v, f.sizes(), f);
  check_type(op, "v", v, f.scalar_type(), f.scalar_type());
}

std::tuple<Tensor, Tensor> gated_scan(const Tensor& f, const Tensor& v, const OptTensor& h0, const OptTensor& lengths, int64_t dir, bool state) {
  check_scan("gated_scan", f, v, 3);
  const int64_t B = f.size(0), T = f.size(1), D = f.size(2);
  TORCH_CHECK_VALUE(dir >= 0 && dir <= 2, "gated_scan: unknown direction ", dir);
  TORCH_CHECK_VALUE(dir != 2 || D % 2 == 0, "gated_scan: direction 'both' needs an even number of channels, got ", D);
  if (has(h0)) {
    check("gated_scan", "h0", *h0, {B, D}, f);
    check_type("gated_scan", "h0", *h0, at::kFloat, at::kFloat);
  }
  if (has(lengths))
    TORCH_CHECK_VALUE(lengths->dim() == 1 && lengths->size(0) == B && (lengths->scalar_type() == at::kInt || lengths->scalar_type() == at::kLong),
                      "gated_scan: lengths must be an int32 or int64 tensor of shape [", B, "], got ", lengths->scalar_type(), " ", lengths->sizes());
  check_eager("gated_scan", {f, v, h0, lengths});
  require_device(f);
  const c10::OptionalDeviceGuard guard(f.device());
  OptTensor len;
  if (has(lengths)) {   // before the conversion: a 64-bit length must not wrap
    len = (lengths->scalar_type() == at::kLong ? lengths->clamp(0, T) : *lengths).to(f.options().dtype(at::kInt)).contiguous();
  }
  if (records("gated_scan", {f, v, h0})) {
    variable_list r = GatedScanFn::apply(f, v, h0, len, dir, state);
    return {r[0], state ? r[1] : Tensor()};
  }
  const Tensor hT = state ? floats({B, D}, f) : Tensor();
  return {scan_run(chan(f), chan(v), contiguous(h0), has(len) ? *len : Tensor(), (int)dir, hT, Tensor()), hT};
}

std::tuple<Tensor, Tensor> gated_scan_step(const Tensor& f, const Tensor& v, const Tensor& state, const OptTensor& out_state) {
  const char* op = "gated_scan_step";
  check_scan(op, f, v, 2);
  check(op, "state", state, f.sizes(), f);
  check_type(op, "state", state, at::kFloat, at::kFloat);
  check_eager(op, {f, v, state, out_state});
  TORCH_CHECK(!records(op, {f, v, state, out_state}),
              "gated_scan_step is inference only: use gated_scan(..., return_state=True) where gradients are needed");
  if (has(out_state)) {
    check(op, "out_state", *out_state, f.sizes(), f);
    check_type(op, "out_state", *out_state, at::kFloat, at::kFloat);
    TORCH_CHECK_VALUE(out_state->is_contiguous() && !out_state->is_neg(), op, ": out_state must be contiguous, and no negated view");
    TORCH_CHECK_VALUE((out_state->data_ptr() == state.data_ptr() && state.is_contiguous()) || apart(*out_state, state), op,
                      ": out_state overlaps state without being it");
    TORCH_CHECK_VALUE(apart(*out_state, f) && apart(*out_state, v), op, ": out_state overlaps f or v");
  }
  require_device(f);
  const c10::OptionalDeviceGuard guard(f.device());
  if (has(out_state)) torch::autograd::impl::bump_version(*out_state);   // a graph that saved it has to notice
  Tensor out = has(out_state) ? *out_state : floats(f.sizes(), f);
  Tensor y = scan_run(chan(f.unsqueeze(1)), chan(v.unsqueeze(1)), contiguous(state), Tensor(), 0, out, Tensor());
  return {y.squeeze(1), out};
}

TORCH_LIBRARY(crnn, m) {
  m.def("layer_norm(Tensor x, Tensor? weight, Tensor? bias, float eps) -> Tensor", &layer_norm);
  m.def("linear(Tensor x, Tensor weight, Tensor? bias, int activation, Tensor? residual) -> Tensor", &linear);
  m.def("gated_scan(Tensor f, Tensor v, Tensor? h0, Tensor? lengths, int direction, bool return_state) -> (Tensor, Tensor)", &gated_scan);
  m.def("gated_scan_step(Tensor f, Tensor v, Tensor state, Tensor(a!)? out_state) -> (Tensor, Tensor)", &gated_scan_step);
}

}  // namespace
