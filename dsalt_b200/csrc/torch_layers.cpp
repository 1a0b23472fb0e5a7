// Torch's side of the operators around the attention (dsalt_b200/layers.py): checks of arguments, outputs
// and workspaces from torch's allocator, and autograd nodes, over the C entry points.
//
// Compiled, because these calls are short: from Python the checks, the outputs and the call of 23 to 33
// arguments take 15 to 20 us and a backward node some 50 us more than an empty one, several times
// the device time of a decode step (4 us for the heads of 64 tokens) and as much as that of a
// training step's head norms over 24000 tokens.
#include <torch/extension.h>

#include <limits>

#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include "../../include/dsalt_b200.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

constexpr int64_t GROUP = 32;

template <typename... Args>
std::string words(const Args&... args) { return c10::str(args...); }

// `python`: the call came from Python, not from autograd's own threads
void check(int rc, const char* fn, bool python) {
  if (rc == DSALT_OK) return;
  const std::string msg = dsalt_last_error();
  if (python) {
    const py::gil_scoped_acquire gil;
    const py::object cls = py::module_::import("dsalt_b200._lib").attr("DsaltError");
    PyErr_SetObject(cls.ptr(), cls(rc, fn, msg).ptr());
    throw py::error_already_set();
  }
  TORCH_CHECK(false, fn, " failed (status ", rc, "): ", msg);
}

int type_code(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return DSALT_F32;
    case at::kBFloat16: return DSALT_BF16;
    case at::kHalf: return DSALT_F16;
    default: throw py::type_error(words("unsupported dtype ", t.dtype()));
  }
}

// every defined tensor on one CUDA device
c10::Device one_device(std::initializer_list<const Tensor*> ts) {
  const Tensor& first = **ts.begin();
  TORCH_CHECK(first.is_cuda(), "dsalt_b200 operators need CUDA tensors (no CPU path)");
  for (const Tensor* t : ts)
    TORCH_CHECK(!t->defined() || t->device() == first.device(), "tensors on ", first.device(), " and ", t->device(),
                " in one call");
  return first.device();
}

void want(const Tensor& t, const char* name, at::ScalarType type, at::IntArrayRef shape) {
  if (t.scalar_type() != type) throw py::type_error(words(name, " must be ", type, ", got ", t.scalar_type()));
  if (t.sizes() != shape) throw py::value_error(words(name, " must have shape ", shape, ", got ", t.sizes()));
  if (!t.is_contiguous()) throw py::value_error(words(name, " must be contiguous"));
}

bool at16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }
void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
Tensor empty(at::IntArrayRef shape, at::ScalarType type, c10::Device dev) {
  return at::empty(shape, at::TensorOptions().dtype(type).device(dev));
}
Tensor workspace(size_t bytes, c10::Device dev) { return empty({(int64_t)std::max<size_t>(bytes, 256)}, at::kByte, dev); }
void no_second_derivative() {
  TORCH_CHECK(!at::GradMode::is_enabled(), "dsalt_b200 operators have no second derivative");  // create_graph=True
}

// A dual tensor need not require a gradient, so that the call would go past the node and lose its tangent
void no_forward_mode(std::initializer_list<const Tensor*> ts) {
  for (const Tensor* t : ts)
    TORCH_CHECK(!t->defined() || !t->_fw_grad(0).defined(), "dsalt_b200 operators have no forward-mode derivative");
}

// A tensor that was kept for the backward pass: hooks on saved tensors may give back one of other strides, which is
// copied; anything else is an error.
Tensor saved(const Tensor& t, const char* name, at::ScalarType type, at::IntArrayRef shape, c10::Device dev) {
  TORCH_CHECK(t.defined() && t.device() == dev && t.scalar_type() == type && t.sizes() == shape, "the saved ", name,
              " came back as another tensor");
  return t.is_contiguous() ? t : t.contiguous();
}

// The tensor's device as the current one, and its current stream, while a call is made
struct Launch {
  c10::cuda::CUDAGuard guard;
  void* stream;
  explicit Launch(c10::Device dev) : guard(dev), stream(c10::cuda::getCurrentCUDAStream(dev.index()).stream()) {}
};

// --------------------------------------------------------------------------- 8 bits
// x [..., n] as rows of consecutive values and their stride (a copy where its strides do not allow that)
std::pair<Tensor, int64_t> matrix(const Tensor& x) {
  const int64_t n = x.size(-1);
  if (x.is_contiguous()) return {x.dim() == 2 ? x : x.view({-1, n}), n};
  Tensor m = x.dim() == 2 ? x : x.reshape({-1, n});
  const bool several = m.size(0) > 1;
  if ((n > 1 && m.stride(1) != 1) || (several && m.stride(0) < n)) return {m.contiguous(), n};
  return {m, several ? m.stride(0) : n};
}

std::tuple<Tensor, Tensor> pack_rows(const Tensor& m, int64_t stride, c10::Device dev) {
  const int64_t rows = m.size(0), n = m.size(1);
  Tensor codes = empty({rows, n}, at::kChar, dev), exps = empty({rows, (n + GROUP - 1) / GROUP}, at::kByte, dev);
  const Launch launch(dev);
  check(dsalt_pack8(m.data_ptr(), type_code(m), rows, n, stride, codes.data_ptr<int8_t>(), exps.data_ptr<uint8_t>(),
                    launch.stream),
        "dsalt_pack8", true);
  return {codes, exps};
}

std::tuple<Tensor, Tensor> pack8(const Tensor& x) {
  const c10::Device dev = one_device({&x});
  if (x.dim() < 1) throw py::value_error("pack8 needs at least one axis");
  type_code(x);
  std::vector<int64_t> groups = x.sizes().vec();
  groups.back() = (groups.back() + GROUP - 1) / GROUP;
  if (x.numel() == 0) return {empty(x.sizes(), at::kChar, dev), empty(groups, at::kByte, dev)};
  const at::NoGradGuard no_grad;
  const auto [m, stride] = matrix(x);
  auto [codes, exps] = pack_rows(m, stride, dev);
  if (x.dim() == 2) return {codes, exps};
  return {codes.view(x.sizes()), exps.view(groups)};
}

Tensor unpack8(const Tensor& codes, const Tensor& exps, int dtype) {
  const c10::Device dev = one_device({&codes, &exps});
  if (codes.dim() < 1) throw py::value_error("codes need at least one axis");
  std::vector<int64_t> groups = codes.sizes().vec();
  const int64_t n = groups.back();
  groups.back() = (n + GROUP - 1) / GROUP;
  want(codes, "codes", at::kChar, codes.sizes());
  want(exps, "exps", at::kByte, groups);
  Tensor out = empty(codes.sizes(), dtype == DSALT_F32 ? at::kFloat : dtype == DSALT_BF16 ? at::kBFloat16 : at::kHalf, dev);
  const Launch launch(dev);
  check(dsalt_unpack8(codes.data_ptr<int8_t>(), exps.data_ptr<uint8_t>(), n ? codes.numel() / n : 0, n, out.data_ptr(), dtype,
                      launch.stream),
        "dsalt_unpack8", true);
  return out;
}

// --------------------------------------------------------------------------- heads
// x [T, H, D] with its token and head strides, as 16-byte loads can take its rows; else a copy
struct Heads {
  Tensor t;
  int64_t token, head;
};
Heads heads(const Tensor& x) {
  const int64_t T = x.size(0), H = x.size(1), D = x.size(2);
  if (at16(x.data_ptr())) {
    if (x.is_contiguous()) return {x, H * D, D};
    const int64_t es = x.element_size(), token = T == 1 ? H * D : x.stride(0), head = H == 1 ? D : x.stride(1);
    if (x.stride(2) == 1 && token * es % 16 == 0 && head * es % 16 == 0) return {x, token, head};
  }
  return {x.clone(at::MemoryFormat::Contiguous), H * D, D};
}

// a table of angles as fp32 with 16-byte aligned rows, and their stride
std::pair<Tensor, int64_t> table(const Tensor& t, int64_t D) {
  Tensor u = t.scalar_type() == at::kFloat ? t : t.to(at::kFloat);
  const bool several = u.size(0) > 1;
  if (u.stride(1) != 1 || !at16(u.data_ptr()) || (several && (u.stride(0) % 4 || u.stride(0) < D / 2)))
    u = u.clone(at::MemoryFormat::Contiguous);
  return {u, several ? u.stride(0) : (D + 3) / 4 * 4};
}

struct Rope {
  c10::Device dev{c10::kCPU};
  int64_t T = 0, H = 0, Hk = 0, D = 0, stride = 0;
  Tensor cos, sin, positions, q_weight, k_weight;
};

Rope rope_args(const Tensor& q, const Tensor& k, const Tensor& cos, const Tensor& sin, const Tensor& positions,
               const Tensor& q_weight, const Tensor& k_weight) {
  if (q.dim() != 3 || k.dim() != 3) throw py::value_error("q must be [T, H, D] and k [T, H_kv, D]");
  Rope a;
  a.dev = one_device({&q, &k, &cos, &sin, &positions, &q_weight, &k_weight});
  a.T = q.size(0), a.H = q.size(1), a.D = q.size(2), a.Hk = k.size(1);
  if (k.size(0) != a.T || k.size(2) != a.D)
    throw py::value_error(words("k must be [", a.T, ", H_kv, ", a.D, "], got ", k.sizes()));
  if (k.scalar_type() != q.scalar_type()) throw py::type_error("q and k must share a dtype");
  type_code(q);
  if (q_weight.defined() != k_weight.defined()) throw py::value_error("q_weight and k_weight go together");
  if (q_weight.defined()) {
    type_code(q_weight);
    want(q_weight, "q_weight", q_weight.scalar_type(), {a.D});
    want(k_weight, "k_weight", q_weight.scalar_type(), {a.D});
  }
  if (a.D % 2) throw py::value_error(words("head_dim ", a.D, " is odd"));
  if (cos.dim() != 2 || cos.sizes() != sin.sizes() || (cos.size(1) != a.D && cos.size(1) != a.D / 2))
    throw py::value_error(words("cos and sin must be [rows, ", a.D, "] or [rows, ", a.D / 2, "], both alike"));
  int64_t other;
  std::tie(a.cos, a.stride) = table(cos, a.D);
  std::tie(a.sin, other) = table(sin, a.D);
  if (other != a.stride) {
    a.cos = a.cos.contiguous(), a.sin = a.sin.contiguous();
    a.stride = a.cos.stride(0);
  }
  a.positions = positions;
  if (positions.defined()) {
    if (positions.dim() != 1 || positions.size(0) != a.T ||
        (positions.scalar_type() != at::kInt && positions.scalar_type() != at::kLong))
      throw py::value_error(words("positions must be [", a.T, "] whole numbers"));
    if (positions.scalar_type() == at::kLong)  // what 32 bits do not hold stays outside the tables
      a.positions = positions.clamp(-1, std::numeric_limits<int32_t>::max()).to(at::kInt);
    a.positions = a.positions.contiguous();
    if (cos.size(0) == 0 && a.T) throw py::value_error("empty tables");
  } else if (cos.size(0) < a.T) {
    throw py::value_error(words("tables of ", cos.size(0), " rows for ", a.T, " tokens"));
  }
  a.q_weight = q_weight, a.k_weight = k_weight;
  return a;
}

variable_list rope_forward(const Tensor& q, const Tensor& k, const Rope& a, double eps) {
  Tensor qo = empty({a.T, a.H, a.D}, q.scalar_type(), a.dev), ko = empty({a.T, a.Hk, a.D}, q.scalar_type(), a.dev);
  const Heads x = heads(q), y = heads(k);
  const Launch launch(a.dev);
  check(dsalt_qk_norm_rope(x.t.data_ptr(), y.t.data_ptr(), type_code(q), a.T, (int)a.H, (int)a.Hk, (int)a.D, x.token, x.head,
                           y.token, y.head, ptr(a.q_weight), ptr(a.k_weight), a.q_weight.defined() ? type_code(a.q_weight) : 0,
                           (float)eps, a.cos.data_ptr<float>(), a.sin.data_ptr<float>(), std::max<int64_t>(a.cos.size(0), 1),
                           a.stride, static_cast<const int32_t*>(ptr(a.positions)), qo.data_ptr(), ko.data_ptr(),
                           launch.stream),
        "dsalt_qk_norm_rope", true);
  return {qo, ko};
}

// the gradients of q, k and the weights (undefined where there are none) from those of the outputs, of which one that
// nothing used is undefined
variable_list rope_backward(const Tensor& dq_out, const Tensor& dk_out, const Tensor& q, const Tensor& k, const Rope& a,
                            double eps, bool python) {
  const int64_t T = a.T, H = a.H, D = a.D, Hk = a.Hk;
  const bool norm = a.q_weight.defined();
  Tensor dq = empty({T, H, D}, q.scalar_type(), a.dev), dk = empty({T, Hk, D}, q.scalar_type(), a.dev), dwq, dwk, ws;
  if (norm) {
    dwq = empty({D}, a.q_weight.scalar_type(), a.dev), dwk = empty({D}, a.q_weight.scalar_type(), a.dev);
    ws = workspace(dsalt_qk_norm_rope_bwd_workspace_bytes((int)D), a.dev);
  }
  const Heads x = heads(q), y = heads(k);
  const Heads gx = heads(dq_out.defined() ? dq_out : at::zeros_like(dq)), gy = heads(dk_out.defined() ? dk_out : at::zeros_like(dk));
  const Launch launch(a.dev);
  check(dsalt_qk_norm_rope_bwd(x.t.data_ptr(), y.t.data_ptr(), gx.t.data_ptr(), gy.t.data_ptr(), type_code(q), T, (int)H,
                               (int)Hk, (int)D, x.token, x.head, y.token, y.head, gx.token, gx.head, gy.token, gy.head,
                               ptr(a.q_weight), ptr(a.k_weight), norm ? type_code(a.q_weight) : 0, (float)eps,
                               a.cos.data_ptr<float>(), a.sin.data_ptr<float>(), std::max<int64_t>(a.cos.size(0), 1), a.stride,
                               static_cast<const int32_t*>(ptr(a.positions)), dq.data_ptr(), dk.data_ptr(), ptr(dwq), ptr(dwk),
                               ptr(ws), norm ? (size_t)ws.numel() : 0, launch.stream),
        "dsalt_qk_norm_rope_bwd", python);
  return {dq, dk, dwq, dwk};
}

// q and k are kept as they came; the norms are formed again in the backward pass
struct RopeNode : torch::autograd::Function<RopeNode> {
  // the weights are arguments of their own (any tensor where there are none), so that the node sees them
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor&, const Tensor&,
                               const Rope& a, double eps) {
    ctx->save_for_backward({q, k, a.q_weight, a.k_weight, a.cos, a.sin, a.positions});
    ctx->saved_data["eps"] = eps;
    return rope_forward(q, k, a, eps);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    no_second_derivative();
    const variable_list s = ctx->get_saved_variables();
    const Tensor &q = s[0], &k = s[1];
    TORCH_CHECK(q.defined() && k.defined() && s[4].defined() && s[5].defined() && q.dim() == 3 && k.dim() == 3 &&
                    (!grads[0].defined() || grads[0].sizes() == q.sizes()) &&
                    (!grads[1].defined() || grads[1].sizes() == k.sizes()),
                "the saved heads came back as other tensors");
    variable_list d = rope_backward(grads[0], grads[1], q, k, rope_args(q, k, s[4], s[5], s[6], s[2], s[3]),
                                    ctx->saved_data["eps"].toDouble(), false);
    d.resize(6);
    return d;
  }
};

bool wants_grad(std::initializer_list<const Tensor*> ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor* t : ts)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}

std::tuple<Tensor, Tensor> qk_norm_rope(const Tensor& q, const Tensor& k, const Tensor& cos, const Tensor& sin,
                                        const std::optional<Tensor>& positions, const std::optional<Tensor>& q_weight,
                                        const std::optional<Tensor>& k_weight, double eps) {
  const Tensor pos = positions.value_or(Tensor()), wq = q_weight.value_or(Tensor()), wk = k_weight.value_or(Tensor());
  no_forward_mode({&q, &k, &cos, &sin, &wq, &wk});
  const Rope a = rope_args(q, k, cos, sin, pos, wq, wk);
  const variable_list out = wants_grad({&q, &k, &wq, &wk})
                                ? RopeNode::apply(q, k, wq.defined() ? wq : cos, wk.defined() ? wk : cos, a, eps)
                                : rope_forward(q, k, a, eps);
  return {out[0], out[1]};
}

// the gradients for a registered operator, whose outputs are all tensors: empty where there is no weight
variable_list qk_norm_rope_grads(const Tensor& dq_out, const Tensor& dk_out, const Tensor& q, const Tensor& k, const Tensor& cos,
                                 const Tensor& sin, const std::optional<Tensor>& positions, const std::optional<Tensor>& q_weight,
                                 const std::optional<Tensor>& k_weight, double eps) {
  const at::NoGradGuard no_grad;
  const Rope a = rope_args(q, k, cos, sin, positions.value_or(Tensor()), q_weight.value_or(Tensor()), k_weight.value_or(Tensor()));
  one_device({&q, &dq_out, &dk_out});
  if (dq_out.sizes() != q.sizes() || dk_out.sizes() != k.sizes()) throw py::value_error("gradients must have the shapes of q and k");
  if (dq_out.scalar_type() != q.scalar_type() || dk_out.scalar_type() != q.scalar_type())
    throw py::type_error("gradients must have the dtype of q and k");
  variable_list d = rope_backward(dq_out, dk_out, q, k, a, eps, true);
  for (Tensor& t : d)
    if (!t.defined()) t = empty({0}, q.scalar_type(), a.dev);
  return d;
}

// --------------------------------------------------------------------------- feed-forward
// whether the rows are 16-byte aligned, or their length does not allow that anyway
bool rows_aligned(const Tensor& t, int64_t stride) {
  const int64_t es = t.element_size();
  return t.size(1) * es % 16 || (at16(t.data_ptr()) && stride * es % 16 == 0);
}
std::pair<Tensor, int64_t> ffn_rows(const Tensor& x) {
  auto [m, stride] = matrix(x);
  if (!rows_aligned(m, stride)) return {m.clone(at::MemoryFormat::Contiguous), m.size(1)};
  return {m, stride};
}
Tensor ffn_weight(const Tensor& w) {
  if (!w.is_contiguous()) return w.contiguous();
  return rows_aligned(w, w.size(1)) ? w : w.clone();
}

struct Ffn {
  c10::Device dev{c10::kCPU};
  int64_t d = 0, F = 0, d_out = 0;
};
Ffn ffn_args(const Tensor& x, const Tensor& w_gate, const Tensor& w_up, const Tensor& w_down) {
  Ffn a;
  a.dev = one_device({&x, &w_gate, &w_up, &w_down});
  if (w_gate.dim() != 2 || w_down.dim() != 2 || x.dim() < 1)
    throw py::value_error("x must be [..., d_model], w_gate and w_up [d_ff, d_model], w_down [d_out, d_ff]");
  a.F = w_gate.size(0), a.d = w_gate.size(1), a.d_out = w_down.size(0);
  if (x.size(-1) != a.d || w_up.sizes() != w_gate.sizes() || w_down.size(1) != a.F)
    throw py::value_error(words("x ", x.sizes(), ", w_gate ", w_gate.sizes(), ", w_up ", w_up.sizes(), " and w_down ",
                                w_down.sizes(), " do not fit together"));
  const at::ScalarType type = x.scalar_type();
  if (w_gate.scalar_type() != type || w_up.scalar_type() != type || w_down.scalar_type() != type)
    throw py::type_error("x and the weights must share a dtype");
  type_code(x);
  return a;
}

struct Kept {
  Tensor y, kept, exps;
};
// the rows of m; nothing is kept with DSALT_KEEP_NONE
Kept ffn_forward(const Tensor& x, const Tensor& m, int64_t stride, const Tensor& w_gate, const Tensor& w_up,
                 const Tensor& w_down, const Ffn& a, int act, int keep) {
  const int64_t T = m.size(0);
  std::vector<int64_t> shape = x.sizes().vec();
  shape.back() = a.d_out;
  const int dt = type_code(m);
  Kept k;
  k.y = empty(shape, m.scalar_type(), a.dev);
  if (keep != DSALT_KEEP_NONE) {
    const int64_t pitch = dsalt_gated_ffn_pitch((int)a.F);
    const bool coded = keep == DSALT_KEEP_8BIT;
    k.kept = empty({coded ? 2 : 3, T, pitch}, coded ? at::kChar : m.scalar_type(), a.dev);
    if (coded) k.exps = empty({2, pitch / GROUP, T}, at::kByte, a.dev);
  }
  const Tensor ws = workspace(dsalt_gated_ffn_keep_workspace_bytes(dt, T, (int)a.d, (int)a.F, (int)a.d_out, keep), a.dev);
  const Launch launch(a.dev);
  check(dsalt_gated_ffn(m.data_ptr(), dt, T, (int)a.d, stride, w_gate.data_ptr(), w_up.data_ptr(), w_down.data_ptr(),
                        (int)a.F, (int)a.d_out, act, keep, ptr(k.kept), static_cast<uint8_t*>(ptr(k.exps.defined() ? k.exps : k.kept)), k.y.data_ptr(),
                        ws.data_ptr(), (size_t)ws.numel(), launch.stream),
        "dsalt_gated_ffn", true);
  return k;
}

// x as the weights' gradients read it: rows, or codes and their scales
struct Rows {
  Tensor t;
  int64_t stride;
  Tensor exps;
};
// the gradients of x and the weights that are wanted
variable_list ffn_backward(const Tensor& grad, const Rows& x, const Kept& k, const Tensor& wg, const Tensor& wu, const Tensor& wd,
                           const Ffn& a, at::IntArrayRef x_shape, int act, int keep, const bool (&wanted)[4], bool python) {
  const at::ScalarType type = grad.scalar_type();
  const int dt = type_code(grad);
  const int64_t T = grad.numel() / a.d_out;
  const auto [dy, dy_stride] = ffn_rows(grad.reshape({T, a.d_out}));
  Tensor dx, dwg, dwu, dwd;
  if (wanted[0]) dx = empty(x_shape, type, a.dev);
  if (wanted[1] || wanted[2]) dwg = empty({a.F, a.d}, type, a.dev), dwu = empty({a.F, a.d}, type, a.dev);
  if (wanted[3]) dwd = empty({a.d_out, a.F}, type, a.dev);
  const Tensor ws = workspace(dsalt_gated_ffn_bwd_workspace_bytes(dt, T, (int)a.d, (int)a.F, (int)a.d_out, keep), a.dev);
  const Launch launch(a.dev);
  check(dsalt_gated_ffn_bwd(dy.data_ptr(), dt, T, (int)a.d, dy_stride, ptr(x.t), x.stride,
                            static_cast<const uint8_t*>(ptr(x.exps)), wg.data_ptr(), wu.data_ptr(), wd.data_ptr(), (int)a.F,
                            (int)a.d_out, act, keep, k.kept.data_ptr(),
                            static_cast<const uint8_t*>(ptr(k.exps.defined() ? k.exps : k.kept)), ptr(dx), ptr(dwg), ptr(dwu),
                            ptr(dwd), ws.data_ptr(), (size_t)ws.numel(), launch.stream),
        "dsalt_gated_ffn_bwd", python);
  return {dx, wanted[1] ? dwg : Tensor(), wanted[2] ? dwu : Tensor(), dwd};
}

// Kept for the backward pass: gate's and up's sums and x, in 24 bits and as it is, or in 8 bits. The rows that
// the last product read are formed again; of fp32 inputs everything is kept as it is, those rows too.
struct FfnNode : torch::autograd::Function<FfnNode> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& w_gate, const Tensor& w_up,
                               const Tensor& w_down, int64_t act, int64_t keep) {
    const Ffn a = ffn_args(x, w_gate, w_up, w_down);
    auto [m, stride] = ffn_rows(x);
    const Tensor wg = ffn_weight(w_gate), wu = ffn_weight(w_up), wd = ffn_weight(w_down);
    const Kept k = ffn_forward(x, m, stride, wg, wu, wd, a, (int)act, (int)keep);
    Tensor x_exps;
    if (!w_gate.requires_grad() && !w_up.requires_grad()) m = Tensor();  // only their gradients read it
    else if (keep == DSALT_KEEP_8BIT && m.numel()) std::tie(m, x_exps) = pack_rows(m, stride, a.dev);
    ctx->save_for_backward({m, x_exps, k.kept, k.exps, wg, wu, wd});
    ctx->saved_data["act"] = act;
    ctx->saved_data["keep"] = keep;
    ctx->saved_data["shape"] = x.sizes().vec();
    ctx->saved_data["d_ff"] = a.F;
    return {k.y};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    no_second_derivative();
    const variable_list s = ctx->get_saved_variables();
    if (!grads[0].defined()) return {Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
    const std::vector<int64_t> shape = ctx->saved_data["shape"].toIntVector();
    const int64_t F = ctx->saved_data["d_ff"].toInt(), d = shape.back(), d_out = grads[0].size(-1);
    const int64_t T = d_out ? grads[0].numel() / d_out : 0, pitch = dsalt_gated_ffn_pitch((int)F);
    const int keep = (int)ctx->saved_data["keep"].toInt();
    const bool coded = keep == DSALT_KEEP_8BIT;
    const c10::Device dev = grads[0].device();
    const at::ScalarType type = grads[0].scalar_type();
    const Tensor kept = saved(s[2], "activations", coded ? at::kChar : type, {coded ? 2 : 3, T, pitch}, dev);
    const Tensor wg = ffn_weight(saved(s[4], "gate weight", type, {F, d}, dev)),
                 wu = ffn_weight(saved(s[5], "up weight", type, {F, d}, dev)),
                 wd = ffn_weight(saved(s[6], "down weight", type, {d_out, F}, dev));
    Tensor x, x_exps, exps;
    if (coded) exps = saved(s[3], "scales", at::kByte, {2, pitch / GROUP, T}, dev);
    int64_t x_stride = d;
    if (s[0].defined()) {
      if (coded && T) {
        x = saved(s[0], "codes", at::kChar, {T, d}, dev);
        x_exps = saved(s[1], "scales", at::kByte, {T, (d + GROUP - 1) / GROUP}, dev);
      } else {
        TORCH_CHECK(s[0].device() == dev && s[0].scalar_type() == type && s[0].dim() == 2 && s[0].size(0) == T && s[0].size(1) == d,
                    "the saved input came back as another tensor");
        std::tie(x, x_stride) = ffn_rows(s[0]);
      }
    }
    const bool wanted[4] = {ctx->needs_input_grad(0), ctx->needs_input_grad(1), ctx->needs_input_grad(2), ctx->needs_input_grad(3)};
    variable_list out = ffn_backward(grads[0], {x, x_stride, x_exps}, {Tensor(), kept, exps}, wg, wu, wd, {dev, d, F, d_out},
                                     shape, (int)ctx->saved_data["act"].toInt(), keep, wanted, false);
    out.resize(6);
    return out;
  }
};

Tensor gated_ffn(const Tensor& x, const Tensor& w_gate, const Tensor& w_up, const Tensor& w_down, int act, int keep) {
  no_forward_mode({&x, &w_gate, &w_up, &w_down});
  const Ffn a = ffn_args(x, w_gate, w_up, w_down);
  if (wants_grad({&x, &w_gate, &w_up, &w_down})) return FfnNode::apply(x, w_gate, w_up, w_down, (int64_t)act, (int64_t)keep)[0];
  const at::NoGradGuard no_grad;
  const auto [m, stride] = ffn_rows(x);
  return ffn_forward(x, m, stride, ffn_weight(w_gate), ffn_weight(w_up), ffn_weight(w_down), a, act, DSALT_KEEP_NONE).y;
}

// The gradients for a registered operator, which keeps its inputs alone: what the backward pass reads is formed again.
// Empty where one is not wanted.
variable_list gated_ffn_grads(const Tensor& dy, const Tensor& x, const Tensor& w_gate, const Tensor& w_up, const Tensor& w_down,
                              int act, std::vector<bool> wanted) {
  const at::NoGradGuard no_grad;
  const Ffn a = ffn_args(x, w_gate, w_up, w_down);
  one_device({&x, &dy});
  std::vector<int64_t> shape = x.sizes().vec();
  shape.back() = a.d_out;
  if (dy.sizes() != at::IntArrayRef(shape)) throw py::value_error(words("the gradient must have shape ", shape, ", got ", dy.sizes()));
  if (dy.scalar_type() != x.scalar_type()) throw py::type_error("the gradient must have the dtype of x");
  if (wanted.size() != 4) throw py::value_error("wanted names x and three weights");
  const auto [m, stride] = ffn_rows(x);
  const Tensor wg = ffn_weight(w_gate), wu = ffn_weight(w_up), wd = ffn_weight(w_down);
  const Kept k = ffn_forward(x, m, stride, wg, wu, wd, a, act, DSALT_KEEP_INPUT);
  const bool which[4] = {wanted[0], wanted[1], wanted[2], wanted[3]};
  variable_list d = ffn_backward(dy, {m, stride, Tensor()}, k, wg, wu, wd, a, x.sizes(), act, DSALT_KEEP_INPUT, which, true);
  for (Tensor& t : d)
    if (!t.defined()) t = empty({0}, x.scalar_type(), a.dev);
  return d;
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  // without the interpreter's lock: a launch waits where the queue is full, and what it waits for may need the lock
  const py::call_guard<py::gil_scoped_release> free;
  m.def("pack8", &pack8, free);
  m.def("unpack8", &unpack8, free);
  m.def("qk_norm_rope", &qk_norm_rope, free);
  m.def("gated_ffn", &gated_ffn, free);
  m.def("qk_norm_rope_grads", &qk_norm_rope_grads, free);
  m.def("gated_ffn_grads", &gated_ffn_grads, free);
}
