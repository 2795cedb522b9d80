// The torch side of the trainable block's operators (layernorm.hip, linear16.hip, gradclip.hip): argument checks, autograd and the calls
// of the C ABI, in C++.  The calls are small -- a window of 34 frames is 4 us on the device -- and a backward pass runs on a thread of
// its own: the same functions written in Python cost 13-18 us per forward and 60-90 us per backward call on the host, which is what a
// training step of 128 clips then waited for (147 us for a layer norm forward + backward of 22 us).
// The library is the one that ctypes has loaded: its path and the error class come in through init().
#include <ATen/autocast_mode.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/DeviceGuard.h>
#include <dlfcn.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/utils/pybind.h>
#include <torch/types.h>

#include <algorithm>
#include <string>

#include "hopmi.h"

namespace {

namespace py = pybind11;
using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using OptTensor = std::optional<Tensor>;

struct Refused : std::runtime_error {
  using std::runtime_error::runtime_error;
};
template <typename... A> [[noreturn]] void refuse(const A&... a) { throw Refused(std::string("hopmi: ") + std::string(c10::str(a...))); }

PyObject* g_error = nullptr;                       // _lib.HopmiError

#define HOPMI_API(X)                                                                                                       \
  X(hopmi_last_error) X(hopmi_layernorm_fwd) X(hopmi_layernorm_bwd_ws_floats) X(hopmi_layernorm_bwd) X(hopmi_gemm16_ws_floats) \
  X(hopmi_gemm16) X(hopmi_gemm16_direct) X(hopmi_pad16) X(hopmi_pad16_two) X(hopmi_act_bwd16_ws_floats) X(hopmi_act_bwd16) \
  X(hopmi_linear16_bwd_ws_floats) X(hopmi_linear16_bwd) X(hopmi_axis_sum_ws_floats) X(hopmi_axis_sum) X(hopmi_grad_clip_ws_bytes) \
  X(hopmi_grad_clip)
struct Api {
#define X(f) decltype(&::f) f = nullptr;
  HOPMI_API(X)
#undef X
} L;

void init(const std::string& path, py::object error) {
  void* h = dlopen(path.c_str(), RTLD_NOW);
  if (h == nullptr) refuse("dlopen of ", path, ": ", dlerror());
#define X(f)                                                                       \
  L.f = reinterpret_cast<decltype(L.f)>(dlsym(h, #f));                             \
  if (L.f == nullptr) refuse(path, " does not export " #f);
  HOPMI_API(X)
#undef X
  g_error = error.release().ptr();
}

void check(int rc, const char* what) {
  if (rc != 0) refuse(what, " failed (code ", rc, "): ", L.hopmi_last_error());
}
void* stream(const Tensor& t) { return c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.device().index()).stream(); }

at::ScalarType type(int code) { return code == 0 ? at::kFloat : code == 1 ? at::kBFloat16 : at::kHalf; }
int code(at::ScalarType t) { return t == at::kFloat ? 0 : t == at::kBFloat16 ? 1 : t == at::kHalf ? 2 : -1; }
const void* ptr(const OptTensor& t) { return t.has_value() && t->defined() ? t->const_data_ptr() : nullptr; }
void* out(const Tensor& t) { return t.defined() ? t.mutable_data_ptr() : nullptr; }
float* fout(const Tensor& t) { return static_cast<float*>(out(t)); }
bool has(const OptTensor& t) { return t.has_value() && t->defined(); }
Tensor unwrap(const OptTensor& t) { return has(t) ? *t : Tensor(); }
bool wants_grad(const OptTensor& t) { return has(t) && t->requires_grad(); }
OptTensor dense(const OptTensor& t) { return has(t) && !t->is_contiguous() ? OptTensor(t->contiguous()) : t; }

// What the kernels would not see: they read memory, and neither a tangent nor a pending negation is in it.
void plain_values(const char* what, const Tensor& t) {
  if (t._fw_grad(0).defined()) refuse(what, ": no forward-mode derivative");
  if (t.is_neg()) refuse(what, ": a tensor with a pending negation (.resolve_neg() makes a plain one)");
}
void plain_values(const char* what, const OptTensor& t) {
  if (has(t)) plain_values(what, *t);
}
void on_device(const Tensor& first, const char* what) {
  if (!first.is_cuda()) refuse(what, ": the operand is on ", first.device(), "; this operator only runs on a ROCm device (no CPU fallback)");
}
void same_device(const Tensor& first, const char* name, const OptTensor& t) {
  if (has(t) && t->device() != first.device()) refuse("`", name, "` is on ", t->device(), ", the first operand on ", first.device());
}

// A tensor (..., width) as rows: a view, or a dense copy where its rows do not lie at one stride.
struct Rows {
  Tensor t;
  int64_t ld = 0;
  int m = 0, n = 0;
  const void* inside = nullptr;                    // rows in a part of t
  bool copied = false;                             // t is a copy made here, not the tensor itself
  const void* data() const { return inside != nullptr ? inside : t.const_data_ptr(); }
};
Rows rows(const Tensor& x, int64_t width) {
  const int64_t m = x.numel() / width;
  if (m >= int64_t(1) << 31 || width >= int64_t(1) << 31) refuse("a tensor of shape ", x.sizes(), " has 2^31 rows or columns, or more");
  Rows r{x, width, (int)m, (int)width};
  if (x.is_contiguous()) return r;
  r.t = x.dim() == 2 ? x : x.reshape({m, width});
  if ((width > 1 && r.t.stride(1) != 1) || (m > 1 && r.t.stride(0) < width)) r.t = r.t.contiguous();
  r.ld = m > 1 ? r.t.stride(0) : width;
  r.copied = !r.t.is_alias_of(x);
  return r;
}

// What a backward pass hands out under create_graph: gradients whose own backward pass, to whatever they were made of, is an error.  They
// were made of `dy` and of the first `operands` operands of the node that is being run (by its edges, whether it saved them or not).
variable_list once(variable_list g, const Tensor& dy, size_t operands) {
  if (!at::GradMode::is_enabled()) return g;
  torch::autograd::edge_list edges;
  const auto node = torch::autograd::get_current_node();
  for (size_t i = 0; i < operands; ++i)
    if (node->next_edge(i).is_valid()) edges.push_back(node->next_edge(i));
  if (dy.requires_grad()) edges.push_back(torch::autograd::impl::gradient_edge(dy));
  if (edges.empty()) return g;
  auto e = std::make_shared<torch::autograd::Error>("hopmi: this operator is differentiable once: its backward pass has no gradient", std::move(edges));
  for (Tensor& t : g)
    if (t.defined()) {
      t = t.detach();
      torch::autograd::set_history(t, e);
    }
  return g;
}

// ------------------------------------------------------------------------------------------------------------- layer norm
constexpr int64_t MOST_WIDTH = int64_t(1) << 29;   // (a row's two sums, next to each other, count in 31 bits)

int weight_code(const Tensor& x, const OptTensor& w, const OptTensor& b) { return code((has(w) ? *w : has(b) ? *b : x).scalar_type()); }

Tensor ln_forward(const Tensor& x, const OptTensor& w, const OptTensor& b, double eps, Tensor* stat) {
  const Rows r = rows(x, x.size(-1));
  Tensor y = at::empty(x.sizes(), x.options());
  float *mean = nullptr, *rstd = nullptr;
  if (stat != nullptr) {
    *stat = at::empty({2, r.m}, x.options().dtype(at::kFloat));
    mean = fout(*stat);
    rstd = mean + r.m;
  }
  if (r.m > 0)
    check(L.hopmi_layernorm_fwd(r.t.const_data_ptr(), r.ld, ptr(w), ptr(b), weight_code(x, w, b), out(y), mean, rstd, r.m, r.n, (float)eps,
                                code(x.scalar_type()), stream(x)), "hopmi_layernorm_fwd");
  return y;
}

struct LayerNormFn : torch::autograd::Function<LayerNormFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const OptTensor& w, const OptTensor& b, double eps) {
    Tensor stat;
    Tensor y = ln_forward(x, w, b, eps, &stat);
    // what the wanted gradients read, and nothing else: x behind dx and dw, w behind dx (an operand may change where it is not read)
    ctx->save_for_backward({x.requires_grad() || wants_grad(w) ? x : Tensor(), x.requires_grad() ? unwrap(w) : Tensor(), stat});
    ctx->saved_data["call"] = weight_code(x, w, b) | (has(w) ? 4 : 0) | (has(b) ? 8 : 0);
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grad) {
    const variable_list s = ctx->get_saved_variables();
    const Tensor &x = s[0], &w = s[1], &stat = s[2];
    const int call = (int)ctx->saved_data["call"].toInt(), wt = call & 3;
    size_t edge = 0;
    const bool need_x = ctx->needs_input_grad(edge++);
    const bool need_w = (call & 4) && ctx->needs_input_grad(edge++);
    const bool need_b = (call & 8) && ctx->needs_input_grad(edge++);      // (edge: how many operands there are)
    variable_list g(4);
    if (!grad[0].defined()) return g;
    const c10::DeviceGuard guard(grad[0].device());
    {
      at::NoGradGuard no_grad;
      const Tensor dy = grad[0].resolve_neg().contiguous();   // (autograd may hand over a view with a pending negation)
      const int64_t D = dy.size(-1);
      // (where only the bias is wanted there is no x: dy is read in its place, and the sums made with it are not asked for)
      const Rows r = rows(x.defined() ? x : dy, D);
      const auto weights = stat.options().dtype(type(wt));
      if (need_x) g[0] = at::empty(x.sizes(), x.options());
      if (need_w) g[1] = r.m > 0 ? at::empty({D}, weights) : at::zeros({D}, weights);
      if (need_b) g[2] = r.m > 0 ? at::empty({D}, weights) : at::zeros({D}, weights);
      if (r.m > 0) {
        const int dt = code(dy.scalar_type());
        Tensor ws;
        if (need_w || need_b) ws = at::empty({(int64_t)L.hopmi_layernorm_bwd_ws_floats(r.m, r.n, dt)}, stat.options());
        const float* mean = static_cast<const float*>(stat.const_data_ptr());
        check(L.hopmi_layernorm_bwd(r.t.const_data_ptr(), r.ld, dy.const_data_ptr(), mean, mean + r.m, w.defined() ? w.const_data_ptr() : nullptr, wt,
                                    out(g[0]), out(g[1]), out(g[2]), fout(ws), r.m, r.n, dt, stream(dy)), "hopmi_layernorm_bwd");
      }
    }
    return once(std::move(g), grad[0], edge);
  }
};

Tensor layer_norm(const Tensor& x, const OptTensor& w0, const OptTensor& b0, double eps) {
  const int64_t d = x.dim() > 0 ? x.size(-1) : 0;
  if (d < 1 || code(x.scalar_type()) < 0)
    refuse("layer_norm: x has shape ", x.sizes(), " and type ", x.scalar_type(), " (fp32, bf16 or fp16 with a last axis of at least 1)");
  if (d > MOST_WIDTH) refuse("layer_norm: x has shape ", x.sizes(), ": a last axis of up to 2^29");
  if (!(eps >= 0.0)) refuse("layer_norm: eps=", eps);
  plain_values("layer_norm", x);
  plain_values("layer_norm", w0);
  plain_values("layer_norm", b0);
  on_device(x, "layer_norm");
  for (const auto& [name, t] : {std::pair<const char*, const OptTensor&>{"weight", w0}, {"bias", b0}}) {
    if (!has(t)) continue;
    same_device(x, name, t);
    if (t->dim() != 1 || t->size(0) != d || (t->scalar_type() != x.scalar_type() && t->scalar_type() != at::kFloat))
      refuse("layer_norm: `", name, "` has shape ", t->sizes(), " and type ", t->scalar_type(), "; x's last axis is ", d, ", its type ",
             x.scalar_type(), " (that type, or fp32)");
  }
  if (has(w0) && has(b0) && w0->scalar_type() != b0->scalar_type())
    refuse("layer_norm: weight is ", w0->scalar_type(), " and bias ", b0->scalar_type(), ": one type for both");
  const c10::DeviceGuard guard(x.device());
  const OptTensor w = dense(w0), b = dense(b0);
  if (at::GradMode::is_enabled() && (x.requires_grad() || wants_grad(w) || wants_grad(b))) return LayerNormFn::apply(x, w, b, eps);
  return ln_forward(x, w, b, eps, nullptr);
}

// ------------------------------------------------------------------------------------------------------------- linear_act
constexpr int FEW_ROWS = 64;                       // up to here layout 0 takes operands of any alignment
constexpr int64_t MOST = int64_t(1) << 22;         // longest row that the tiled products address
constexpr int64_t MOST_ROWS = int64_t(1) << 30;

bool direct(const Rows& r) { return L.hopmi_gemm16_direct(r.data(), r.ld, r.n) != 0; }
// as hopmi_gemm16 takes it: as it lies where its rows start and end on 16 bytes, else copied into rows padded with zeros
Rows padding(const Rows& r) {
  const int64_t ld = (int64_t(r.n) + 7) / 8 * 8;
  return Rows{at::empty({r.m, ld}, r.t.options()), ld, r.m, r.n, nullptr, true};
}
Rows operand(const Rows& r) {
  if (direct(r)) return r;
  Rows p = padding(r);
  check(L.hopmi_pad16(r.t.const_data_ptr(), r.ld, out(p.t), p.ld, r.m, r.n, stream(r.t)), "hopmi_pad16");
  return p;
}
void operands(Rows& a, Rows& b) {
  if (direct(a) || direct(b)) {
    a = operand(a);
    b = operand(b);
    return;
  }
  Rows p = padding(a), q = padding(b);
  check(L.hopmi_pad16_two(a.t.const_data_ptr(), a.ld, out(p.t), p.ld, a.m, a.n, b.t.const_data_ptr(), b.ld, out(q.t), q.ld, b.m, b.n, stream(a.t)),
        "hopmi_pad16_two");
  a = std::move(p);
  b = std::move(q);
}

void gemm(const Rows& a, const Rows& b, int layout, const Tensor& c, int M, int N, int K, const OptTensor& bias, const Rows& res, const Tensor& z,
          int act) {
  const size_t n = L.hopmi_gemm16_ws_floats(M, N, K, layout);
  Tensor ws;
  if (n > 0) ws = at::empty({(int64_t)n}, c.options().dtype(at::kFloat));
  check(L.hopmi_gemm16(a.data(), a.ld, b.data(), b.ld, layout, out(c), N, ptr(bias), ptr(res.t), res.ld, out(z),
                       z.defined() ? z.size(1) : 0, act, M, N, K, code(c.scalar_type()), fout(ws), stream(c)), "hopmi_gemm16");
}

// The gradient of an operand of shape `to` that was broadcast to dy's: its sums over the axes along which it was repeated, one run of
// neighbouring axes after the other, from the last on, in fp32 between them.
Tensor summed_to(const Tensor& grad, at::IntArrayRef to) {
  if (grad.numel() == 0) return at::zeros(to, grad.options());
  Tensor cur = grad.contiguous();
  struct Run { int64_t size; bool summed; };
  std::vector<Run> runs;
  const int64_t lead = cur.dim() - (int64_t)to.size();
  for (int64_t i = 0; i < cur.dim(); ++i) {
    const int64_t size = cur.size(i);
    if (size == 1) continue;
    const bool summed = i < lead || to[i - lead] == 1;
    if (!runs.empty() && runs.back().summed == summed) runs.back().size *= size;
    else runs.push_back({size, summed});
  }
  int left = 0;
  for (const Run& r : runs) left += r.summed;
  if (left == 0) return cur.view(to);                        // (axes of one element only)
  int64_t inner = 1;
  for (size_t k = runs.size(); k-- > 0;) {
    if (!runs[k].summed) {
      inner *= runs[k].size;
      continue;
    }
    int64_t outer = 1;
    for (size_t j = 0; j < k; ++j) outer *= runs[j].size;
    const bool last = --left == 0;
    const auto f32 = cur.options().dtype(at::kFloat);
    const Tensor sums = last ? at::empty(to, grad.options()) : at::empty({outer * inner}, f32);
    const size_t n = L.hopmi_axis_sum_ws_floats(outer, runs[k].size, inner);
    Tensor ws;
    if (n > 0) ws = at::empty({(int64_t)n}, f32);
    check(L.hopmi_axis_sum(cur.const_data_ptr(), code(cur.scalar_type()), out(sums), code(sums.scalar_type()), outer, runs[k].size, inner, fout(ws),
                           stream(cur)), "hopmi_axis_sum");
    cur = sums;
  }
  return cur;
}

struct Linear16 {
  Tensor y, z;
  Rows x, w;                                       // as the product took them
};
Linear16 linear_forward(const Tensor& x, const Tensor& w, const OptTensor& bias, const OptTensor& res, int act, bool keep) {
  Linear16 o{Tensor(), Tensor(), rows(x, x.size(-1)), rows(w, w.size(1))};
  const int M = o.x.m, N = o.w.m, K = o.x.n;
  at::DimVector shape(x.sizes().begin(), x.sizes().end());
  shape.back() = N;
  o.y = at::empty(shape, x.options());
  if (keep) o.z = at::empty({M, (int64_t(N) + 7) / 8 * 8}, x.options());
  if (M == 0) return o;
  const Rows r = has(res) ? rows(res->sizes() == o.y.sizes() ? *res : res->expand(o.y.sizes()), N) : Rows{};
  if (M > FEW_ROWS) {
    operands(o.x, o.w);
  }
  gemm(o.x, o.w, 0, o.y, M, N, K, bias, r, o.z, act);
  return o;
}

struct LinearActFn : torch::autograd::Function<LinearActFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, const OptTensor& bias, const OptTensor& res, int64_t act) {
    const bool need_x = x.requires_grad(), need_w = w.requires_grad(), keep = act != 0 && (need_x || need_w || wants_grad(bias));
    Linear16 o = linear_forward(x, w, bias, res, (int)act, keep);
    // dx reads w and dw reads x, no gradient anything else (an operand may change where it is not read); where the product took a copy
    // (dense or padded), that serves the backward's products too
    ctx->save_for_backward({!need_w ? Tensor() : o.x.copied ? o.x.t : x, !need_x ? Tensor() : o.w.copied ? o.w.t : w, o.z});
    ctx->saved_data["call"] = act | (has(bias) ? 4 : 0) | (has(res) ? 8 : 0);
    ctx->saved_data["k"] = w.size(1);
    if (wants_grad(res) && res->sizes() != o.y.sizes()) ctx->saved_data["residual"] = res->sizes().vec();
    return o.y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grad) {
    const variable_list s = ctx->get_saved_variables();
    const Tensor &x = s[0], &w = s[1], &z = s[2];
    const int call = (int)ctx->saved_data["call"].toInt(), act = call & 3;
    const bool bias = call & 4, res = call & 8;
    size_t edge = 0;
    const bool need_x = ctx->needs_input_grad(edge++), need_w = ctx->needs_input_grad(edge++);
    const bool need_b = bias && ctx->needs_input_grad(edge++), need_r = res && ctx->needs_input_grad(edge++);
    variable_list g(5);
    const Tensor& dy = grad[0];
    if (!dy.defined()) return g;
    const c10::DeviceGuard guard(dy.device());
    {
      at::NoGradGuard no_grad;
      const int64_t N = dy.size(-1), K = ctx->saved_data["k"].toInt();
      const auto opt = at::TensorOptions().device(dy.device()).dtype(dy.scalar_type());
      at::DimVector shape(dy.sizes().begin(), dy.sizes().end());
      shape.back() = K;
      if (need_x) g[0] = at::empty(shape, opt);
      const Rows d = rows(dy.resolve_neg(), N);    // (autograd may hand over a view with a pending negation)
      const int M = d.m;
      if (need_w) g[1] = M > 0 ? at::empty({N, K}, opt) : at::zeros({N, K}, opt);
      if (need_b) g[2] = M > 0 ? at::empty({N}, opt) : at::zeros({N}, opt);
      if (M > 0 && (need_x || need_w || need_b)) {
        const bool make = (act != 0 || !direct(d)) && (need_x || need_w);       // else dz is dy as it lies there
        const bool both = need_x && need_w;        // (with the bias gradient's last sums in the same launch)
        // one piece of scratch memory: dz, the bias gradient's partial sums, the split contractions' partial results
        const int64_t ldz = (N + 7) / 8 * 8, z_floats = make ? (M * ldz / 2 + 3) / 4 * 4 : 0;
        const int64_t part_floats = need_b ? ((int64_t)L.hopmi_act_bwd16_ws_floats(M, (int)N) + 3) / 4 * 4 : 0;
        const int64_t ws_floats = both ? (int64_t)L.hopmi_linear16_bwd_ws_floats(M, (int)N, (int)K) : 0;
        Tensor scratch;
        float* mem = nullptr;
        if (z_floats + part_floats + ws_floats > 0) {
          scratch = at::empty({z_floats + part_floats + ws_floats}, opt.dtype(at::kFloat));
          mem = fout(scratch);
        }
        Rows dz = d;
        if (make) dz = Rows{scratch, ldz, M, (int)N, mem};
        float *part = need_b ? mem + z_floats : nullptr, *ws = mem + z_floats + part_floats;
        if (make || need_b)
          check(L.hopmi_act_bwd16(d.data(), d.ld, ptr(z), z.defined() ? z.size(1) : 0, make ? mem : nullptr, dz.ld, both ? nullptr : out(g[2]),
                                  part, act, M, (int)N, code(dy.scalar_type()), stream(dy)), "hopmi_act_bwd16");
        auto kept = [](const Tensor& t) { return rows(t, t.size(-1)); };        // (a padded copy as rows of its own length)
        if (both) {
          Rows pw = kept(w), px = kept(x);
          operands(pw, px);
          check(L.hopmi_linear16_bwd(dz.data(), dz.ld, pw.data(), pw.ld, px.data(), px.ld, out(g[0]), out(g[1]), part, out(g[2]), M, (int)N,
                                     (int)K, code(dy.scalar_type()), ws_floats > 0 ? ws : nullptr, stream(dy)), "hopmi_linear16_bwd");
        } else if (need_x) gemm(dz, operand(kept(w)), 1, g[0], M, (int)K, (int)N, OptTensor(), Rows{}, Tensor(), 0);
        else if (need_w) gemm(dz, operand(kept(x)), 2, g[1], (int)N, (int)K, M, OptTensor(), Rows{}, Tensor(), 0);
      }
      // (a broadcast residual's by kernels of this library's own: see csrc/axis_sum.hip for why)
      const auto shape_r = ctx->saved_data.find("residual");
      if (need_r) g[3] = shape_r == ctx->saved_data.end() ? dy : summed_to(dy.resolve_neg(), shape_r->second.toIntVector());
    }
    return once(std::move(g), dy, 2 + (bias && act != 0));      // (the bias is in z, and z in act'(z))
  }
};

Tensor linear_act(const Tensor& x0, const Tensor& w0, const OptTensor& b0, const OptTensor& r0, int64_t act) {
  Tensor x = x0, w = w0;
  OptTensor b = b0, r = r0;
  plain_values("linear_act", x);
  plain_values("linear_act", w);
  plain_values("linear_act", b);
  plain_values("linear_act", r);
  // One type for all: the product's operands are 16-bit ones and its result is one of them (a residual in fp32 would be rounded with the
  // sum at the latest).  Cast in every call: a copy kept by the weight's identity would be stale after an in-place update.
  if (at::autocast::is_autocast_enabled(at::kCUDA)) {
    const at::ScalarType t = at::autocast::get_autocast_dtype(at::kCUDA);
    x = x.to(t);
    w = w.to(t);
    if (has(b)) b = b->to(t);
    if (has(r)) r = r->to(t);
  }
  on_device(x, "linear_act");
  same_device(x, "w", w);
  same_device(x, "bias", b);
  same_device(x, "residual", r);
  if (code(x.scalar_type()) < 1) refuse("linear_act: x is ", x.scalar_type(), ": bf16 or fp16 (fp32 products: ops.linear)");
  auto same_type = [&](const char* name, at::ScalarType t) {
    if (t != x.scalar_type()) refuse("linear_act: `", name, "` is ", t, ", x ", x.scalar_type(), ": one type for all operands");
  };
  same_type("w", w.scalar_type());
  if (has(b)) same_type("bias", b->scalar_type());
  if (has(r)) same_type("residual", r->scalar_type());
  if (x.dim() < 1 || w.dim() != 2 || w.size(1) != x.size(-1) || w.size(0) < 1 || w.size(1) < 1)
    refuse("linear_act: x ", x.sizes(), " and w ", w.sizes(), " (N, K) do not fit, or have an empty side");
  if (w.size(0) > MOST || w.size(1) > MOST) refuse("linear_act: w ", w.sizes(), ": sides of up to 2^22");
  if (x.numel() / x.size(-1) > MOST_ROWS) refuse("linear_act: x has shape ", x.sizes(), ": up to 2^30 rows");
  if (has(b) && (b->dim() != 1 || b->size(0) != w.size(0))) refuse("linear_act: bias has shape ", b->sizes(), ", w ", w.sizes());
  if (has(r)) {
    at::DimVector shape(x.sizes().begin(), x.sizes().end());
    shape.back() = w.size(0);
    if (r->sizes() != at::IntArrayRef(shape)) {
      bool fits = r->dim() <= (int64_t)shape.size();
      for (int64_t i = 1; fits && i <= r->dim(); ++i) fits = r->size(-i) == 1 || r->size(-i) == shape[shape.size() - i];
      if (!fits) refuse("linear_act: residual of shape ", r->sizes(), " does not broadcast to ", at::IntArrayRef(shape));
    }
  }
  const c10::DeviceGuard guard(x.device());
  b = dense(b);
  if (at::GradMode::is_enabled() && (x.requires_grad() || w.requires_grad() || wants_grad(b) || wants_grad(r))) return LinearActFn::apply(x, w, b, r, act);
  return linear_forward(x, w, b, r, (int)act, false).y;
}

// -------------------------------------------------------------------------------------------------------------- GradClip
// Does the tensor fill one stretch of memory, each place once (in whatever order of its axes)?
bool fills(const Tensor& t) { return t.is_contiguous() || t.is_non_overlapping_and_dense(); }

struct ClipPlan {
  std::vector<Tensor> in, to;
  std::vector<const void*> src;
  std::vector<void*> dst;
  std::vector<long long> n;
  std::vector<int> dt;
  bool into = false, separate = false;               // separate: apart() has seen these addresses

  ClipPlan(std::vector<Tensor> tensors, std::optional<std::vector<Tensor>> outs) : in(std::move(tensors)), into(outs.has_value()) {
    if (outs) to = std::move(*outs);
    if (in.empty()) refuse("GradClip: an empty list of tensors");
    if (into && to.size() != in.size()) refuse("GradClip: ", to.size(), " outputs for ", in.size(), " tensors");
    on_device(in[0], "GradClip");
    src.resize(in.size());
    dst.resize(into ? in.size() : 0);
    n.resize(in.size());
    dt.resize(in.size());
    read(true);
    apart();
  }

  // The tensors' memory as it is now (`.data = ...` changes it under a plan), checked again.
  void read(bool first) {
    const at::Device dev = in[0].device();
    if (!dev.is_cuda()) refuse("GradClip: tensors[0] is on ", dev);
    for (size_t i = 0; i < in.size(); ++i) {
      const Tensor& t = in[i];
      if (t.device() != dev) refuse("GradClip: tensors[", i, "] is on ", t.device(), ", the first on ", dev);
      if (t.layout() != at::kStrided || code(t.scalar_type()) < 0 || !fills(t))
        refuse("GradClip: tensors[", i, "] (", t.scalar_type(), ", shape ", t.sizes(), ") is not an fp32, bf16 or fp16 tensor without gaps "
               "(.contiguous() makes one)");
      if (t.is_neg()) refuse("GradClip: tensors[", i, "] has a pending negation (.resolve_neg() makes a plain tensor)");
      // (in place the tensor is written: one whose memory is a lazy copy of another's gets its own first)
      const void* p = into ? t.const_data_ptr() : t.mutable_data_ptr();
      const int c = code(t.scalar_type());
      if (!first && (n[i] != t.numel() || dt[i] != c)) refuse("GradClip: tensors[", i, "] is not the tensor that the plan was made for any more");
      if (p != src[i]) separate = false;
      src[i] = p;
      n[i] = t.numel();
      dt[i] = c;
      if (!into) continue;
      const Tensor& o = to[i];
      if (o.device() != dev) refuse("GradClip: out[", i, "] is on ", o.device(), ", the first tensor on ", dev);
      if (o.layout() != at::kStrided || o.scalar_type() != at::kFloat || o.sizes() != t.sizes() || !fills(o) || o.is_neg() ||
          (!(t.is_contiguous() && o.is_contiguous()) && o.strides() != t.strides()))
        refuse("GradClip: out[", i, "] is not an fp32 tensor of tensors[", i, "]'s shape and strides");
      void* q = o.mutable_data_ptr();
      if (q != dst[i]) separate = false;
      dst[i] = q;
    }
  }

  void apart() {
    struct Span { uintptr_t p, end; const char* list; size_t i; };
    std::vector<Span> spans;
    for (size_t i = 0; i < in.size(); ++i) {
      if (n[i] == 0) continue;
      const auto p = reinterpret_cast<uintptr_t>(src[i]);
      spans.push_back({p, p + n[i] * in[i].element_size(), "tensors", i});
      if (!into) continue;
      const auto q = reinterpret_cast<uintptr_t>(dst[i]);
      spans.push_back({q, q + n[i] * 4, "out", i});
    }
    std::sort(spans.begin(), spans.end(), [](const Span& a, const Span& b) { return a.p < b.p; });
    for (size_t k = 1; k < spans.size(); ++k)
      if (spans[k - 1].end > spans[k].p)
        refuse("GradClip: ", spans[k - 1].list, "[", spans[k - 1].i, "] and ", spans[k].list, "[", spans[k].i, "] share memory");
    separate = true;
  }

  Tensor clip(double max_norm) {
    if (!(max_norm >= 0.0)) refuse("GradClip: max_norm=", max_norm);
    read(false);
    if (!separate) apart();
    const c10::DeviceGuard guard(in[0].device());
    at::NoGradGuard no_grad;
    const auto opt = at::TensorOptions().device(in[0].device());
    const Tensor norm = at::empty({}, opt.dtype(at::kFloat)), ws = at::empty({(int64_t)L.hopmi_grad_clip_ws_bytes()}, opt.dtype(at::kByte));
    check(L.hopmi_grad_clip(src.data(), into ? dst.data() : nullptr, n.data(), dt.data(), (int)src.size(), (float)max_norm, fout(norm), out(ws),
                            stream(in[0])), "hopmi_grad_clip");
    for (const Tensor& t : into ? to : in)           // (written behind autograd's back; inference tensors keep no versions)
      if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
    return norm;
  }
};

}  // namespace

PYBIND11_MODULE(_block, m) {
  py::register_exception_translator([](std::exception_ptr p) {
    try {
      if (p) std::rethrow_exception(p);
    } catch (const Refused& e) {
      PyErr_SetString(g_error != nullptr ? g_error : PyExc_RuntimeError, e.what());
    }
  });
  m.def("init", &init);
  m.def("layer_norm", &layer_norm);
  m.def("linear_act", &linear_act);
  py::class_<ClipPlan>(m, "ClipPlan").def(py::init<std::vector<Tensor>, std::optional<std::vector<Tensor>>>()).def("clip", &ClipPlan::clip);
}
