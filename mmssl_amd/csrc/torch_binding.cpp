// Binding of the operators that are called often on little data (embed_rows, layernorm_rows, logprobs_rows, grad_norm,
// clip_grads): argument checks, output and workspace tensors, autograd nodes and the C entry points' calls without the
// interpreter in between. What the GPU does is libmmssl_hip.so's, reached through its C ABI like every other operator; this
// file launches nothing by itself.
//
// Measured on one MI355X host, 200 rows looked up in a 500 x 64 fp32 table: forward 4.5 us (through ctypes 8.3), forward and
// gradient through torch.autograd.grad 57 us (a Python autograd.Function over ctypes 92; the engine's own share is about 40).
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <dlfcn.h>
#include <torch/extension.h>

#include <algorithm>
#include <optional>
#include <string>
#include <unordered_set>
#include <vector>

#include "../../include/mmssl_hip.h"

namespace {

using torch::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// mmssl_amd._lib.MmsslError on the Python side (a RuntimeError, also where the engine reports it)
struct Refused : std::runtime_error {
  using std::runtime_error::runtime_error;
};
PyObject* g_error = nullptr;

[[noreturn]] void refuse(const std::string& what) { throw Refused(what); }

// ---- the library's entry points, from the handle that mmssl_amd._lib has loaded ----------------------------------------
#define MMSSL_BOUND(F)                                \
  F(mmssl_strerror)                                   \
  F(mmssl_embed_rows)                                 \
  F(mmssl_embed_rows_bwd_workspace_bytes)             \
  F(mmssl_embed_rows_bwd)                             \
  F(mmssl_layernorm_rows)                             \
  F(mmssl_layernorm_rows_bwd_workspace_bytes)         \
  F(mmssl_layernorm_rows_bwd)                         \
  F(mmssl_logprobs_rows_workspace_bytes)              \
  F(mmssl_logprobs_rows)                              \
  F(mmssl_logprobs_rows_bwd)                          \
  F(mmssl_grad_norm_workspace_bytes)                  \
  F(mmssl_grad_norm)                                  \
  F(mmssl_clip_grads)
struct Lib {
#define MMSSL_MEMBER(f) decltype(&f) p_##f = nullptr;
  MMSSL_BOUND(MMSSL_MEMBER)
  hipError_t (*is_capturing)(hipStream_t, hipStreamCaptureStatus*) = nullptr;      // the runtime's that the library runs on
} lib;
#define CALL(f) lib.p_##f

void bind(uintptr_t handle, py::object error) {
  Lib l;
#define MMSSL_RESOLVE(f)                                                                        \
  l.p_##f = reinterpret_cast<decltype(l.p_##f)>(dlsym(reinterpret_cast<void*>(handle), #f));    \
  if (!l.p_##f) throw std::runtime_error("libmmssl_hip.so does not export " #f " (stale build?)");
  MMSSL_BOUND(MMSSL_RESOLVE)
  l.is_capturing = reinterpret_cast<decltype(l.is_capturing)>(dlsym(reinterpret_cast<void*>(handle), "hipStreamIsCapturing"));
  if (!l.is_capturing) throw std::runtime_error("no hipStreamIsCapturing among the libraries of libmmssl_hip.so");
  lib = l;
  Py_XDECREF(g_error);
  g_error = error.inc_ref().ptr();
}

void check(int rc, const char* what) {
  if (rc) refuse(std::string(what) + " failed: " + CALL(mmssl_strerror)(rc) + " (code " + std::to_string(rc) + ")");
}

// ---- tensors ------------------------------------------------------------------------------------------------------------
int dtype_code(at::ScalarType t) {
  return t == at::kFloat ? MMSSL_F32 : t == at::kBFloat16 ? MMSSL_BF16 : t == at::kHalf ? MMSSL_F16 : -1;
}
// A tangent of forward-mode differentiation on an operand: the operators have no such derivative, and their outputs would come
// out as if it were zero. (Undefined where the mode is off.)
void no_tangent(const Tensor& t, const char* name) {
  if (t.defined() && t._fw_grad(/*level=*/0).defined())
    refuse(std::string(name) + " carries a forward-mode tangent: only reverse-mode derivatives are there");
}
int typed(const Tensor& t, const char* name) {
  if (!t.is_cuda()) refuse(std::string(name) + " must be a CUDA (HIP) tensor: this package has no CPU path");
  no_tangent(t, name);
  const int c = dtype_code(t.scalar_type());
  if (c < 0 || t.layout() != at::kStrided)
    refuse(std::string(name) + " must be a dense float32, bfloat16 or float16 tensor, got " + toString(t.scalar_type()));
  return c;
}
void same_device(const Tensor& t, const Tensor& other, const char* name) {
  if (other.device() != t.device())
    refuse(std::string(name) + " is on " + other.device().str() + ", expected " + t.device().str());
}
void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }
bool capturing(const Tensor& t) {
  hipStreamCaptureStatus st = hipStreamCaptureStatusNone;
  return lib.is_capturing(static_cast<hipStream_t>(stream_of(t)), &st) == hipSuccess && st != hipStreamCaptureStatusNone;
}
Tensor bytes_on(const Tensor& t, size_t n) { return at::empty({(int64_t)n}, t.options().dtype(at::kByte)); }
std::string shape_of(at::IntArrayRef s) {
  std::string r = "[";
  for (size_t i = 0; i < s.size(); ++i) r += (i ? ", " : "") + std::to_string(s[i]);
  return r + "]";
}

// The kernels read memory as it is: a lazily negated view (the imaginary part of a conjugate) is written out first.
Tensor plain(const Tensor& t) { return t.defined() && t.is_neg() ? t.resolve_neg() : t; }

// t as [rows, d] with unit column stride (a view where the strides allow it) and its row pitch
struct Rows {
  Tensor t;
  int64_t rows, d, ld;
};
Rows rows_of(const Tensor& x) {
  Rows r;
  r.t = x.dim() == 2 ? x : x.reshape({-1, x.size(-1)});
  if (r.t.size(1) > 1 && r.t.stride(1) != 1) r.t = r.t.contiguous();
  r.rows = r.t.size(0);
  r.d = r.t.size(1);
  r.ld = r.rows > 1 ? r.t.stride(0) : r.d;
  return r;
}
void fits_int(int64_t d, const char* what) {
  if (d > (1 << 24)) refuse(std::string(what) + ": rows of at most 2^24 columns, got " + std::to_string(d));
}
void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
void first_order(const char* what, const variable_list& grads) {
  if (at::GradMode::is_enabled())            // the engine enables it only for create_graph=True
    refuse(std::string(what) + ": the gradient is not differentiable again");
  for (const Tensor& g : grads) no_tangent(g, what);
}
bool records(const Tensor& a) { return a.defined() && a.requires_grad(); }

// Recorded inside a capture, with an input from which the graph reaches a node of the default stream: an eager producer, or the
// accumulator that an eager graph of the same leaf keeps alive, however many nodes of the capture lie between. The engine would
// make the capture wait for that stream, which cannot be captured. The engine's threads do not come back from that, so it is
// refused here. (What the caller joins to the output afterwards is out of sight.)
void recordable(const Tensor& input, const char* what) {
  if (!records(input)) return;
  const auto none = c10::hip::getDefaultHIPStream(input.device().index()).id();
  if (c10::hip::getCurrentHIPStream(input.device().index()).id() == none || !capturing(input)) return;
  const auto root = input.is_leaf() ? torch::autograd::impl::try_get_grad_accumulator(input) : input.grad_fn();
  if (!root) return;
  std::vector<torch::autograd::Node*> todo{root.get()};
  std::unordered_set<torch::autograd::Node*> seen{root.get()};
  while (!todo.empty()) {
    torch::autograd::Node* node = todo.back();
    todo.pop_back();
    const auto s = node->stream();
    if (s && s->id() == none)
      refuse(std::string(what) + ": a captured backward pass cannot reach into an eager graph of the default stream: run the " +
             "warm-up on the capture's own stream and release its graph, or capture under torch.no_grad()");
    for (const auto& edge : node->next_edges())
      if (edge.function && seen.insert(edge.function.get()).second) todo.push_back(edge.function.get());
  }
}

// int32 / int64 numbers on t's device, contiguous; host tensors are uploaded
Tensor tokens(const Tensor& t, Tensor idx, const char* name) {
  const auto s = idx.scalar_type();
  if (s != at::kLong && s != at::kInt)
    refuse(std::string(name) + " must hold int64 or int32 numbers, got " + toString(s));
  if (idx.device() != t.device()) {
    if (idx.is_cuda()) same_device(t, idx, name);
    if (capturing(t)) refuse(std::string(name) + ": host tensors cannot be uploaded while a graph is captured");
    idx = idx.to(t.device());
  }
  return idx.contiguous();
}

// ---- embed_rows -----------------------------------------------------------------------------------------------------------
struct Pad {
  bool has;
  int64_t idx;
};

Tensor embed_forward(const Tensor& table, const Tensor& idx, double scale, Pad pad) {
  const c10::DeviceGuard guard(table.device());
  const int64_t rows = table.size(0), d = table.size(1);
  auto sizes = idx.sizes().vec();
  sizes.push_back(d);
  Tensor out = at::empty(sizes, table.options().requires_grad(false));
  check(CALL(mmssl_embed_rows)(table.data_ptr(), rows > 1 ? table.stride(0) : d, dtype_code(table.scalar_type()), rows, (int)d,
                               idx.data_ptr(), (int)idx.element_size(), idx.numel(), (float)scale, pad.has, pad.idx,
                               out.data_ptr(), d, stream_of(table)),
        "mmssl_embed_rows");
  return out;
}

struct EmbedRows : torch::autograd::Function<EmbedRows> {
  static Tensor forward(AutogradContext* ctx, const Tensor& table, const Tensor& idx, double scale, bool has_pad,
                        int64_t pad) {
    ctx->save_for_backward({idx});
    ctx->saved_data["cfg"] = c10::List<int64_t>({table.size(0), table.size(1), (int64_t)has_pad, pad});
    ctx->saved_data["scale"] = scale;
    return embed_forward(table, idx, scale, {has_pad, pad});
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    first_order("embed_rows", grads);
    const Tensor idx = ctx->get_saved_variables()[0];
    const auto cfg = ctx->saved_data["cfg"].toIntVector();
    const int64_t rows = cfg[0], d = cfg[1];
    const Rows g = rows_of(plain(grads[0]));
    const c10::DeviceGuard guard(g.t.device());
    Tensor grad = at::empty({rows, d}, g.t.options());
    const size_t nb = CALL(mmssl_embed_rows_bwd_workspace_bytes)(rows, (int)d, idx.numel());
    const Tensor ws = bytes_on(g.t, nb);
    check(CALL(mmssl_embed_rows_bwd)(g.t.data_ptr(), g.ld, dtype_code(g.t.scalar_type()), idx.data_ptr(),
                                     (int)idx.element_size(), idx.numel(), rows, (int)d,
                                     (float)ctx->saved_data["scale"].toDouble(), (int)cfg[2], cfg[3], grad.data_ptr(),
                                     ws.data_ptr(), nb, stream_of(g.t)),
          "mmssl_embed_rows_bwd");
    return {grad, Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

Tensor embed_rows(const Tensor& table_, const Tensor& idx_, double scale, std::optional<int64_t> padding_idx) {
  typed(table_, "table");
  const Tensor table = plain(table_);
  if (table.dim() != 2 || table.size(1) < 1 || (table.size(1) > 1 && table.stride(1) != 1))
    refuse("embed_rows: table must be [rows, d] with unit column stride");
  fits_int(table.size(1), "embed_rows");
  const Tensor idx = tokens(table, idx_, "idx");
  const Pad pad{padding_idx.has_value(), padding_idx.value_or(0)};
  if (at::GradMode::is_enabled() && records(table)) {
    recordable(table, "embed_rows");
    return EmbedRows::apply(table, idx, scale, pad.has, pad.idx);
  }
  return embed_forward(table, idx, scale, pad);
}

// ---- layernorm_rows ---------------------------------------------------------------------------------------------------------
Tensor layernorm_forward(const Tensor& X, const Tensor& w, const Tensor& b, double eps, Tensor* stats) {
  const c10::DeviceGuard guard(X.device());
  const Rows x = rows_of(X);
  Tensor y = at::empty(X.sizes(), X.options().requires_grad(false));
  if (stats) *stats = at::empty({x.rows, 2}, X.options().dtype(at::kFloat).requires_grad(false));
  const Tensor& p = w.defined() ? w : b;
  check(CALL(mmssl_layernorm_rows)(x.t.data_ptr(), x.ld, dtype_code(X.scalar_type()), x.rows, (int)x.d, ptr(w), ptr(b),
                                   p.defined() ? dtype_code(p.scalar_type()) : MMSSL_F32, (float)eps, y.data_ptr(),
                                   stats ? stats->data_ptr<float>() : nullptr, stream_of(X)),
        "mmssl_layernorm_rows");
  return y;
}

struct LayerNormRows : torch::autograd::Function<LayerNormRows> {
  // an absent weight or bias is no input of the node: the edges are X, then weight and bias as far as they are there
  static Tensor forward(AutogradContext* ctx, const Tensor& X, const std::optional<Tensor>& weight,
                        const std::optional<Tensor>& bias, double eps) {
    const Tensor w = weight.value_or(Tensor()), b = bias.value_or(Tensor());
    Tensor stats;
    Tensor y = layernorm_forward(X, w, b, eps, &stats);
    ctx->save_for_backward({X, w, stats});
    const auto pt = (w.defined() ? w : b.defined() ? b : X).scalar_type();
    ctx->saved_data["cfg"] = c10::List<int64_t>({(int64_t)pt, (int64_t)b.defined()});
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    first_order("layernorm_rows", grads);
    const auto saved = ctx->get_saved_variables();
    const Tensor &X = saved[0], &w = saved[1], &stats = saved[2];
    const auto cfg = ctx->saved_data["cfg"].toIntVector();
    const auto pt = (at::ScalarType)cfg[0];
    const c10::DeviceGuard guard(X.device());
    const Rows x = rows_of(X), g = rows_of(plain(grads[0]));
    Tensor gx, gw, gb, ws;
    if (ctx->needs_input_grad(0)) gx = at::empty(X.sizes(), X.options());
    const int edge_b = w.defined() ? 2 : 1;
    if (w.defined() && ctx->needs_input_grad(1)) gw = at::empty({x.d}, X.options().dtype(pt));
    if (cfg[1] && ctx->needs_input_grad(edge_b)) gb = at::empty({x.d}, X.options().dtype(pt));
    const int dt = dtype_code(X.scalar_type());
    size_t nb = 0;
    if (gw.defined() || gb.defined()) {
      nb = CALL(mmssl_layernorm_rows_bwd_workspace_bytes)(dt, x.rows, (int)x.d);
      ws = bytes_on(X, nb);
    }
    check(CALL(mmssl_layernorm_rows_bwd)(x.t.data_ptr(), x.ld, g.t.data_ptr(), g.ld, dt, x.rows, (int)x.d, ptr(w),
                                         dtype_code(pt), stats.data_ptr<float>(), ptr(gx), ptr(gw), ptr(gb), ptr(ws), nb,
                                         stream_of(X)),
          "mmssl_layernorm_rows_bwd");
    return {gx, gw, gb, Tensor()};
  }
};

Tensor layernorm_rows(const Tensor& X_, const std::optional<Tensor>& weight, const std::optional<Tensor>& bias, double eps) {
  typed(X_, "X");
  const Tensor X = plain(X_);
  if (X.dim() < 1 || X.size(-1) < 1) refuse("layernorm_rows: X must be [..., d] with d >= 1");
  fits_int(X.size(-1), "layernorm_rows");
  if (!(eps >= 0.0 && eps <= 3.0e38)) refuse("layernorm_rows: eps must be a finite number >= 0, got " + std::to_string(eps));
  auto param = [&](const std::optional<Tensor>& p, const char* name) {
    if (!p.has_value()) return Tensor();
    typed(*p, name);
    same_device(X, *p, name);
    if (p->dim() != 1 || p->size(0) != X.size(-1))
      refuse(std::string("layernorm_rows: ") + name + " must be [" + std::to_string(X.size(-1)) + "], got " + shape_of(p->sizes()));
    if (p->scalar_type() != X.scalar_type() && p->scalar_type() != at::kFloat)
      refuse(std::string("layernorm_rows: ") + name + " must be of X's type or float32");
    return plain(*p).contiguous();
  };
  const Tensor w = param(weight, "weight"), b = param(bias, "bias");
  if (w.defined() && b.defined() && w.scalar_type() != b.scalar_type())
    refuse("layernorm_rows: weight and bias must be of one type");
  if (at::GradMode::is_enabled() && (records(X) || records(w) || records(b))) {
    for (const Tensor* t : {&X, &w, &b}) recordable(*t, "layernorm_rows");
    auto there = [](const Tensor& t) { return t.defined() ? std::optional<Tensor>(t) : std::nullopt; };
    return LayerNormRows::apply(X, there(w), there(b), eps);
  }
  return layernorm_forward(X, w, b, eps, nullptr);
}

// ---- logprobs_rows ----------------------------------------------------------------------------------------------------------
// {logp, entropy, top_logp, top_idx}, the last two undefined for k = 0
variable_list logprobs_forward(const Tensor& X, const Tensor& target, int64_t k, double temperature, int64_t ignore,
                               Tensor* stats) {
  const c10::DeviceGuard guard(X.device());
  const Rows x = rows_of(X);
  const auto f32 = X.options().dtype(at::kFloat).requires_grad(false);
  const auto lead = target.sizes();
  Tensor logp = at::empty(lead, f32), entropy = at::empty(lead, f32), top_logp, top_idx;
  if (k) {
    auto with_k = lead.vec();
    with_k.push_back(k);
    top_logp = at::empty(with_k, f32);
    top_idx = at::empty(with_k, f32.dtype(at::kLong));
  }
  if (stats) *stats = at::empty({x.rows, 4}, f32);
  const int dt = dtype_code(X.scalar_type());
  const size_t nb = CALL(mmssl_logprobs_rows_workspace_bytes)(dt, x.rows, x.d, (int)k);
  const Tensor ws = bytes_on(X, nb);
  check(CALL(mmssl_logprobs_rows)(x.t.data_ptr(), x.ld, dt, x.rows, x.d, target.data_ptr(), (int)target.element_size(), ignore,
                                  (int)k, (float)temperature, logp.data_ptr<float>(), entropy.data_ptr<float>(),
                                  static_cast<float*>(ptr(top_logp)), static_cast<int64_t*>(ptr(top_idx)),
                                  stats ? stats->data_ptr<float>() : nullptr, ws.data_ptr(), nb, stream_of(X)),
        "mmssl_logprobs_rows");
  return {logp, entropy, top_logp, top_idx};
}

struct LogprobsRows : torch::autograd::Function<LogprobsRows> {
  static variable_list forward(AutogradContext* ctx, const Tensor& X, const Tensor& target, int64_t k, double temperature,
                               int64_t ignore) {
    Tensor stats;
    variable_list out = logprobs_forward(X, target, k, temperature, ignore, &stats);
    ctx->save_for_backward({X, target, stats, out[3]});
    ctx->saved_data["cfg"] = c10::List<int64_t>({k, ignore});
    ctx->saved_data["temperature"] = temperature;
    ctx->set_materialize_grads(false);
    if (k) {
      ctx->mark_non_differentiable({out[3]});
    } else {
      out.resize(2);
    }
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    first_order("logprobs_rows", grads);
    const auto saved = ctx->get_saved_variables();
    const Tensor &X = saved[0], &target = saved[1], &stats = saved[2], &top_idx = saved[3];
    const auto cfg = ctx->saved_data["cfg"].toIntVector();
    const variable_list none(5);
    Tensor gl = grads[0], ge = grads[1], gt = grads.size() > 2 ? grads[2] : Tensor();
    if (!gl.defined() && !ge.defined() && !gt.defined()) return none;
    const c10::DeviceGuard guard(X.device());
    const Rows x = rows_of(X);
    for (Tensor* g : {&gl, &ge, &gt})
      if (g->defined()) *g = plain(*g).contiguous();
    Tensor gx = at::empty(X.sizes(), X.options());
    check(CALL(mmssl_logprobs_rows_bwd)(x.t.data_ptr(), x.ld, dtype_code(X.scalar_type()), x.rows, x.d, target.data_ptr(),
                                        (int)target.element_size(), cfg[1], (int)cfg[0],
                                        (float)ctx->saved_data["temperature"].toDouble(),
                                        static_cast<const int64_t*>(ptr(top_idx)), stats.data_ptr<float>(),
                                        static_cast<const float*>(ptr(gl)), static_cast<const float*>(ptr(ge)),
                                        static_cast<const float*>(ptr(gt)), gx.data_ptr(), stream_of(X)),
          "mmssl_logprobs_rows_bwd");
    variable_list out(5);
    out[0] = gx;
    return out;
  }
};

py::tuple logprobs_rows(const Tensor& X_, const Tensor& target_, int64_t k, double temperature, int64_t ignore) {
  constexpr int64_t kMost = 128;
  typed(X_, "X");
  const Tensor X = plain(X_);
  if (X.dim() < 1 || X.size(-1) < 1) refuse("logprobs_rows: X must be [..., n] with n >= 1");
  if (k < 0 || k > kMost || k > X.size(-1))
    refuse("logprobs_rows: 0 <= k <= min(" + std::to_string(kMost) + ", n) expected, got " + std::to_string(k));
  if (!(temperature >= 1e-30 && temperature <= 1e30))
    refuse("logprobs_rows: temperature must be a positive number, got " + std::to_string(temperature));
  const Tensor target = tokens(X, target_, "target");
  const auto lead = X.sizes().slice(0, X.dim() - 1);
  if (target.sizes() != lead)
    refuse("logprobs_rows: target must be " + shape_of(lead) + ", got " + shape_of(target.sizes()));
  const bool record = at::GradMode::is_enabled() && records(X);
  if (record) recordable(X, "logprobs_rows");
  const variable_list out = record ? LogprobsRows::apply(X, target, k, temperature, ignore)
                                   : logprobs_forward(X, target, k, temperature, ignore, nullptr);
  if (!k) return py::make_tuple(out[0], out[1], py::none(), py::none());
  return py::make_tuple(out[0], out[1], out[2], out[3]);
}

// ---- gradient lists -----------------------------------------------------------------------------------------------------------
struct GradList {
  std::vector<const void*> at;
  std::vector<int64_t> numel;
  std::vector<int32_t> dtype;
};
GradList list_of(const std::vector<Tensor>& ts, const char* what, c10::Device dev) {
  GradList l;
  l.at.reserve(ts.size());
  l.numel.reserve(ts.size());
  l.dtype.reserve(ts.size());
  const bool recording = at::GradMode::is_enabled();
  for (const Tensor& t : ts) {
    if (!t.defined() || t.layout() != at::kStrided) refuse(std::string(what) + ": dense tensors expected");
    if (t.unsafeGetTensorImpl()->autograd_meta()) {      // plain data has neither
      no_tangent(t, what);
      // nothing of this is recorded: a norm would be a constant of its backward pass, a leaf be written behind autograd's back
      if (recording && t.requires_grad())
        refuse(std::string(what) + ": not differentiable; detach the tensors or call it under torch.no_grad()");
    }
    if (!t.is_cuda() || t.device() != dev)
      refuse(std::string(what) + ": gradients must be on one CUDA (HIP) device: this package has no CPU path");
    const int c = dtype_code(t.scalar_type());
    if (c < 0) refuse(std::string(what) + ": gradients must be float32, bfloat16 or float16");
    if (!t.is_contiguous()) refuse(std::string(what) + ": gradients must be contiguous");
    l.at.push_back(t.data_ptr());
    l.numel.push_back(t.numel());
    l.dtype.push_back(c);
  }
  return l;
}
c10::Device device_of_first(const std::vector<Tensor>& ts, const char* what) {
  if (ts.empty()) refuse(std::string(what) + ": no gradients");
  return ts[0].device();
}

Tensor grad_norm(const std::vector<Tensor>& grads) {
  const c10::Device dev = device_of_first(grads, "grad_norm");
  const GradList l = list_of(grads, "grad_norm", dev);
  const c10::DeviceGuard guard(dev);
  Tensor norm = at::empty({}, at::TensorOptions(dev).dtype(at::kFloat));
  const size_t nb = CALL(mmssl_grad_norm_workspace_bytes)((int)grads.size());
  const Tensor ws = bytes_on(norm, nb);
  check(CALL(mmssl_grad_norm)(l.at.data(), l.numel.data(), l.dtype.data(), (int)grads.size(), norm.data_ptr<float>(),
                              ws.data_ptr(), nb, stream_of(norm)),
        "mmssl_grad_norm");
  return norm;
}

Tensor clip_grads(const std::vector<Tensor>& grads, double max_norm, double eps,
                  const std::optional<std::vector<Tensor>>& out) {
  if (!(max_norm >= 0.0)) refuse("clip_grads: max_norm must be a number >= 0, got " + std::to_string(max_norm));
  const c10::Device dev = device_of_first(grads, "clip_grads");
  const GradList l = list_of(grads, "clip_grads", dev);
  GradList o;
  if (out.has_value()) {
    if (out->size() != grads.size())
      refuse("clip_grads: " + std::to_string(out->size()) + " outputs for " + std::to_string(grads.size()) + " gradients");
    o = list_of(*out, "clip_grads: out", dev);
    if (o.numel != l.numel || o.dtype != l.dtype) refuse("clip_grads: out must match the gradients' types and sizes");
    for (size_t i = 0; i < grads.size(); ++i)          // (in place, and for the norm, a lazy sign makes no difference)
      if ((*out)[i].is_neg() != grads[i].is_neg()) refuse("clip_grads: out and a lazily negated gradient differ in sign");
  } else {
    o = l;
  }
  // every output is written by its own blocks: no two may share memory, nor an output a gradient other than its own
  struct Span {
    uintptr_t a, b;
    size_t i;
    bool written;
  };
  std::vector<Span> spans;
  spans.reserve(2 * grads.size());
  for (size_t i = 0; i < grads.size(); ++i) {
    const uintptr_t size = (uintptr_t)l.numel[i] * (l.dtype[i] == MMSSL_F32 ? 4 : 2);
    if (!size) continue;
    const uintptr_t w = (uintptr_t)o.at[i], r = (uintptr_t)l.at[i];
    spans.push_back({w, w + size, i, true});
    if (r != w) spans.push_back({r, r + size, i, false});
  }
  std::sort(spans.begin(), spans.end(), [](const Span& x, const Span& y) { return x.a < y.a; });
  uintptr_t end_written = 0, end_any = 0;
  for (const Span& s : spans) {
    if (s.a < end_written || (s.written && s.a < end_any)) refuse("clip_grads: tensors that are written overlap others");
    end_any = std::max(end_any, s.b);
    if (s.written) end_written = std::max(end_written, s.b);
  }
  const c10::DeviceGuard guard(dev);
  Tensor norm = at::empty({}, at::TensorOptions(dev).dtype(at::kFloat));
  const size_t nb = CALL(mmssl_grad_norm_workspace_bytes)((int)grads.size());
  const Tensor ws = bytes_on(norm, nb);
  check(CALL(mmssl_clip_grads)(l.at.data(), const_cast<void* const*>(o.at.data()), l.numel.data(), l.dtype.data(),
                               (int)grads.size(), (float)max_norm, (float)eps, norm.data_ptr<float>(), ws.data_ptr(), nb,
                               stream_of(norm)),
        "mmssl_clip_grads");
  for (const Tensor& t : out.has_value() ? *out : grads)             // autograd sees that they were written
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
  return norm;
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  py::register_exception_translator([](std::exception_ptr p) {
    try {
      if (p) std::rethrow_exception(p);
    } catch (const Refused& e) {
      PyErr_SetString(g_error ? g_error : PyExc_RuntimeError, e.what());
    }
  });
  m.def("bind", &bind);
  m.def("embed_rows", &embed_rows);
  m.def("layernorm_rows", &layernorm_rows);
  m.def("logprobs_rows", &logprobs_rows);
  m.def("grad_norm", &grad_norm);
  m.def("clip_grads", &clip_grads);
}
