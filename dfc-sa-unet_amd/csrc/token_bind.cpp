// Host side of dfcsa.token_ops: argument checks, output and workspace allocation (torch's caching
// allocator), autograd nodes, and the calls of the C entry points on the current stream.  It is C++
// because these operators are called once per layer and token.  The same steps in Python cost 17 to 22 us
// for a serving call and 124 to 147 us for a forward and backward on one host; here 7 to 11 and 60 to 75, most
// of it torch's engine (another host: 82 us for the norm, 66 for an empty node with its tensors).
//
// The entry points are handed over as addresses by the Python side (dfcsa/_lib.py has loaded the
// library), so there is one copy of it in the process, whichever file it came from.
#include <torch/extension.h>

#include <ATen/TracerMode.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPStream.h>

#include <cmath>
#include <string>
#include <vector>

#include "dfcsa.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::Function;
using torch::autograd::variable_list;

struct Api {
  decltype(&dfcsa_rms_fwd) rms_fwd;
  decltype(&dfcsa_rms_fwd_q8) rms_fwd_q8;
  decltype(&dfcsa_rms_bwd_work_floats) rms_bwd_work_floats;
  decltype(&dfcsa_rms_bwd) rms_bwd;
  decltype(&dfcsa_dequant_q8) dequant_q8;
  decltype(&dfcsa_rotary) rotary;
  decltype(&dfcsa_wattn_work_floats) wattn_work_floats;
  decltype(&dfcsa_wattn_fwd) wattn_fwd;
  decltype(&dfcsa_wattn_bwd) wattn_bwd;
} api;

template <typename F> void take(const py::dict& d, const char* name, F& f) {
  f = reinterpret_cast<F>(d[name].cast<uintptr_t>());
}
void bind(const py::dict& d) {
  take(d, "dfcsa_rms_fwd", api.rms_fwd);
  take(d, "dfcsa_rms_fwd_q8", api.rms_fwd_q8);
  take(d, "dfcsa_rms_bwd_work_floats", api.rms_bwd_work_floats);
  take(d, "dfcsa_rms_bwd", api.rms_bwd);
  take(d, "dfcsa_dequant_q8", api.dequant_q8);
  take(d, "dfcsa_rotary", api.rotary);
  take(d, "dfcsa_wattn_work_floats", api.wattn_work_floats);
  take(d, "dfcsa_wattn_fwd", api.wattn_fwd);
  take(d, "dfcsa_wattn_bwd", api.wattn_bwd);
}

// ------------------------------------------------------------------ checks
[[noreturn]] void bad_value(const std::string& s) { throw py::value_error(s); }
[[noreturn]] void bad_type(const std::string& s) { throw py::type_error(s); }
std::string shape(const Tensor& t) {
  std::string s = "(";
  for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.size(i));
  return s + ")";
}
std::string name(at::ScalarType t) { return std::string(c10::toString(t)); }

// The kernels read and write memory that torch's own operators allocated: a tracer would record the allocation and
// return uninitialised memory, a forward-mode tangent would be lost, and wrapped tensors have no memory to read.
bool traced() {
  using Modes = c10::impl::TorchDispatchModeTLS;
  using Mode = c10::impl::TorchDispatchModeKey;
  if (at::tracer::impl::is_dispatch_enabled() || c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::PreDispatch)) return true;
  if (!Modes::any_modes_set()) return false;
  return Modes::get_mode(Mode::PROXY) || Modes::get_mode(Mode::FAKE) || Modes::get_mode(Mode::FUNCTIONAL);
}
void need_plain(at::ArrayRef<Tensor> ts) {
  if (traced())
    throw std::runtime_error("dfcsa.token_ops cannot be traced (torch.jit.trace, make_fx, torch.export, fake tensors)");
  constexpr c10::DispatchKeySet wrapped({c10::DispatchKey::Python, c10::DispatchKey::FuncTorchBatched,
                                         c10::DispatchKey::FuncTorchGradWrapper, c10::DispatchKey::Functionalize,
                                         c10::DispatchKey::ZeroTensor});
  for (const Tensor& t : ts) {
    if (!t.defined()) continue;
    if (t._fw_grad(0).defined())
      throw std::runtime_error("dfcsa.token_ops has no forward-mode derivatives: detach() inputs that carry a tangent");
    if (t.key_set().has_any(wrapped) || t.layout() != at::kStrided)
      throw std::runtime_error("dfcsa.token_ops needs dense tensors, not tensors wrapped by torch.func or a subclass with a dispatch of its own");
  }
}
void need_gpu(std::initializer_list<const Tensor*> ts) {
  const Tensor* first = nullptr;
  for (const Tensor* t : ts) {
    if (!t || !t->defined()) continue;
    if (!t->is_cuda()) throw std::runtime_error("dfcsa kernels need GPU tensors (MI355X/ROCm); got a CPU tensor");
    if (!first) first = t;
    else if (t->device() != first->device())
      bad_value("tensors on " + first->device().str() + " and " + t->device().str() + ": one device is needed");
  }
}
int dtype_of(const Tensor& t, const char* what) {
  if (t.scalar_type() == at::kBFloat16) return DFCSA_DT_BF16;
  if (t.scalar_type() == at::kFloat) return DFCSA_DT_F32;
  bad_type(std::string(what) + ": bfloat16 or float32 is needed, got " + name(t.scalar_type()));
}
void done(int rc, const char* what) {
  if (rc == 0) return;
  throw std::runtime_error(std::string(what) + " failed: " +
                           (rc == DFCSA_EINVAL ? "invalid argument/shape" : "HIP error " + std::to_string(-rc)));
}
void first_order(const variable_list& g) {
  TORCH_CHECK(!at::GradMode::is_enabled(),
              "dfcsa.token_ops: gradients are first order only (create_graph=True is refused)");
  need_plain(g);
}
bool wants_grad(std::initializer_list<const Tensor*> ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor* t : ts)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}

// The current stream of the tensor's device, with that device current while it lives.
struct On {
  c10::DeviceGuard guard;
  void* stream;
  explicit On(const Tensor& t)
      : guard(t.device()), stream((void*)c10::hip::getCurrentHIPStream(t.device().index()).stream()) {}
};

// contiguous and 16-byte aligned: a copy where it is not
Tensor packed(const Tensor& t) {
  Tensor c = t.contiguous();
  return (uintptr_t)c.data_ptr() % 16 ? c.clone() : c;
}
Tensor floats(const Tensor& like, int64_t n) { return at::empty({n}, like.options().dtype(at::kFloat)); }
float* fptr(const Tensor& t) { return t.defined() ? (float*)t.data_ptr() : nullptr; }
void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

// ------------------------------------------------------------------ RMS norm of the residual stream
struct Norm {
  int ty, rt, rows, C;
};
Norm norm_args(const Tensor& x, const Tensor& res, const Tensor& w, double eps) {
  need_gpu({&x, &res, &w});
  Norm n;
  n.ty = dtype_of(x, "x");
  n.rt = dtype_of(res, "residual");
  if (x.dim() < 1 || !x.sizes().equals(res.sizes()))
    bad_value("x " + shape(x) + " and residual " + shape(res) + ": one shape [..., C] is needed");
  const int64_t C = x.size(-1);
  if (C < 8 || C % 8 || C > 16384) bad_value(std::to_string(C) + " columns: a multiple of 8 up to 16384 is needed");
  if (w.scalar_type() != at::kFloat) bad_type("weight: float32 is needed, got " + name(w.scalar_type()));
  if (w.dim() != 1 || w.size(0) != C) bad_value("weight " + shape(w) + ": (" + std::to_string(C) + ",) is needed");
  if (n.ty == DFCSA_DT_F32 && n.rt != DFCSA_DT_F32) bad_type("a float32 x needs a float32 residual");
  if (!(eps >= 0.0) || !std::isfinite((float)eps)) bad_value("eps: a finite fp32 value of at least 0 is needed");
  if (x.numel() / C > 0x7fff0000) bad_value("at most 2^31 - 2^16 rows");
  n.rows = (int)(x.numel() / C);
  n.C = (int)C;
  return n;
}

// (y, r, rstd); rstd undefined unless asked for
std::tuple<Tensor, Tensor, Tensor> norm_forward(const Tensor& x0, const Tensor& res0, const Tensor& w0, double eps,
                                                bool keep) {
  const Norm n = norm_args(x0, res0, w0, eps);
  const Tensor x = packed(x0), res = packed(res0), w = packed(w0);
  const Tensor y = at::empty(x.sizes(), x.options()), r = at::empty(res.sizes(), res.options());
  const Tensor rstd = keep ? floats(x, n.rows) : Tensor();
  if (n.rows) {
    const On on(x);
    done(api.rms_fwd(n.ty, n.rt, n.rows, n.C, ptr(x), ptr(res), fptr(w), (float)eps, ptr(y), ptr(r), fptr(rstd),
                     on.stream), "dfcsa_rms_fwd");
  }
  return {y, r, rstd};
}

struct RmsNorm : public Function<RmsNorm> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& res, const Tensor& w, double eps) {
    auto [y, r, rstd] = norm_forward(x, res, w, eps, true);
    ctx->save_for_backward({r, rstd, w});
    ctx->saved_data["x"] = (int64_t)x.scalar_type();
    ctx->set_materialize_grads(false);
    return {y, r};
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    first_order(g);
    const auto saved = ctx->get_saved_variables();
    const Tensor &r = saved[0], &rstd = saved[1], w = packed(saved[2]);
    const auto xt = (at::ScalarType)ctx->saved_data["x"].toInt();
    const bool nx = ctx->needs_input_grad(0), nr = ctx->needs_input_grad(1), nw = ctx->needs_input_grad(2);
    if (!g[0].defined() && !g[1].defined()) return {Tensor(), Tensor(), Tensor(), Tensor()};
    const Tensor dy = g[0].defined() ? packed(g[0]) : at::zeros(r.sizes(), r.options().dtype(xt));
    const Tensor dr = g[1].defined() ? packed(g[1]) : Tensor();
    const int C = (int)r.size(-1), rows = (int)(r.numel() / C);
    const bool same = xt == r.scalar_type();   // then dx and dres are one tensor
    const Tensor dx = nx || (same && nr) ? at::empty(r.sizes(), r.options().dtype(xt)) : Tensor();
    const Tensor dres = nr && !same ? at::empty(r.sizes(), r.options()) : Tensor();
    const Tensor dw = nw ? (rows ? at::empty(w.sizes(), w.options()) : at::zeros(w.sizes(), w.options())) : Tensor();
    if (rows) {
      const On on(r);
      const Tensor work = nw ? floats(r, api.rms_bwd_work_floats(rows, C)) : Tensor();
      done(api.rms_bwd(xt == at::kFloat ? DFCSA_DT_F32 : DFCSA_DT_BF16,
                       r.scalar_type() == at::kFloat ? DFCSA_DT_F32 : DFCSA_DT_BF16, rows, C, ptr(dy), ptr(dr), ptr(r),
                       fptr(rstd), fptr(w), ptr(dx), ptr(dres), fptr(dw), fptr(work), work.defined() ? work.numel() : 0,
                       on.stream), "dfcsa_rms_bwd");
    }
    return {nx ? dx : Tensor(), nr ? (same ? dx : dres) : Tensor(), dw, Tensor()};
  }
};

std::tuple<Tensor, Tensor> rms_norm_residual(const Tensor& x, const Tensor& res, const Tensor& w, double eps) {
  need_plain({x, res, w});
  if (wants_grad({&x, &res, &w})) {
    norm_args(x, res, w, eps);
    const variable_list o = RmsNorm::apply(x, res, w, eps);
    return {o[0], o[1]};
  }
  auto [y, r, rstd] = norm_forward(x, res, w, eps, false);
  return {y, r};
}

int64_t group_of(int64_t group, int64_t C) {
  if (group != 0 && group != 32 && group != 64 && group != 128)
    bad_value("group " + std::to_string(group) + ": 0 (the whole row), 32, 64 or 128");
  if (group && C % group) bad_value(std::to_string(C) + " columns are no multiple of the group, " + std::to_string(group));
  return group;
}

std::tuple<Tensor, Tensor, Tensor> rms_norm_residual_q8(const Tensor& x0, const Tensor& res0, const Tensor& w0,
                                                        double eps, int64_t group) {
  need_plain({x0, res0, w0});
  if (wants_grad({&x0, &res0, &w0}))
    throw std::runtime_error("rms_norm_residual_q8 has no gradient: call it under torch.no_grad(), or rms_norm_residual");
  const Norm n = norm_args(x0, res0, w0, eps);
  group_of(group, n.C);
  const Tensor x = packed(x0), res = packed(res0), w = packed(w0);
  const Tensor y8 = at::empty(x.sizes(), x.options().dtype(at::kFloat8_e4m3fn));
  auto sizes = x.sizes().vec();
  sizes.back() = group ? n.C / group : 1;
  const Tensor scales = at::empty(sizes, x.options().dtype(at::kFloat)), r = at::empty(res.sizes(), res.options());
  if (n.rows) {
    const On on(x);
    done(api.rms_fwd_q8(n.ty, n.rt, n.rows, n.C, (int)group, ptr(x), ptr(res), fptr(w), (float)eps, ptr(y8),
                        fptr(scales), ptr(r), on.stream), "dfcsa_rms_fwd_q8");
  }
  return {y8, scales, r};
}

Tensor dequant_q8(const Tensor& y8, const Tensor& scales, at::ScalarType out) {
  need_plain({y8, scales});
  if (wants_grad({&scales})) throw std::runtime_error("dequant_q8 has no gradient: call it under torch.no_grad()");
  need_gpu({&y8, &scales});
  if (y8.scalar_type() != at::kFloat8_e4m3fn || scales.scalar_type() != at::kFloat)
    bad_type("float8_e4m3fn values and float32 scales are needed, got " + name(y8.scalar_type()) + " and " +
             name(scales.scalar_type()));
  if (out != at::kFloat && out != at::kBFloat16) bad_type("dtype: bfloat16 or float32 is needed, got " + name(out));
  if (y8.dim() < 1 || scales.dim() != y8.dim() ||
      !scales.sizes().slice(0, y8.dim() - 1).equals(y8.sizes().slice(0, y8.dim() - 1)))
    bad_value("values " + shape(y8) + " and scales " + shape(scales) + " do not belong together");
  const int64_t C = y8.size(-1), ng = scales.size(-1);
  if (C < 8 || C % 8 || C > 16384 || ng < 1 || C % ng)
    bad_value(std::to_string(ng) + " scales for " + std::to_string(C) + " columns");
  const int64_t group = ng == 1 ? 0 : group_of(C / ng, C);
  const Tensor v = packed(y8), s = scales.contiguous();
  const Tensor o = at::empty(v.sizes(), v.options().dtype(out));
  if (v.numel()) {
    const On on(v);
    done(api.dequant_q8(out == at::kFloat ? DFCSA_DT_F32 : DFCSA_DT_BF16, v.numel() / C, (int)C, (int)group, ptr(v),
                        fptr(s), ptr(o), on.stream), "dfcsa_dequant_q8");
  }
  return o;
}

// ------------------------------------------------------------------ rotary positions
// Turns per position of each pair and its axis: constants of a shape, kept by the caller.
struct TurnTable {
  std::vector<double> turns;
  std::vector<unsigned char> axis;
  int axes;
  TurnTable(const std::vector<int64_t>& pairs, double base, bool shared) : axes((int)pairs.size()) {
    if (pairs.empty() || pairs.size() > 4) bad_value("the rotated pairs of one to four axes are needed");
    int64_t total = 0;
    for (int64_t n : pairs) {
      if (n < 1 || n > 256) bad_value("axes: between 1 and 256 rotated pairs each");
      total += n;
    }
    if (total > DFCSA_ROTARY_MAX_PAIRS) bad_value(std::to_string(total) + " rotated pairs: at most 256");
    if (!(base >= 1.0) || !std::isfinite(base)) bad_value("base: a finite value of at least 1 is needed");
    for (size_t a = 0; a < pairs.size(); ++a)
      for (int64_t i = 0; i < pairs[a]; ++i) {
        const double power = shared ? (double)turns.size() / (double)total : (double)i / (double)pairs[a];
        turns.push_back(std::pow(base, -power) / (2.0 * M_PI));
        axis.push_back((unsigned char)a);
      }
  }
};

void rotary_check(const Tensor& q, const Tensor& k, const Tensor& pos, const TurnTable& t) {
  need_gpu({&q, &k, &pos});
  dtype_of(q, "q");
  if (q.dim() != 4 || (k.defined() && k.dim() != 4)) bad_value("q and k: [batch, tokens, heads, width] is needed");
  const int64_t B = q.size(0), N = q.size(1), D = q.size(3);
  if (k.defined()) {
    if (k.scalar_type() != q.scalar_type())
      bad_type("q " + name(q.scalar_type()) + " and k " + name(k.scalar_type()) + ": one type is needed");
    if (k.size(0) != B || k.size(1) != N || k.size(3) != D)
      bad_value("q " + shape(q) + " and k " + shape(k) + " differ in more than their heads");
  }
  if (2 * (int64_t)t.turns.size() > D || D > 1024)
    bad_value(std::to_string(t.turns.size()) + " rotated pairs in a width of " + std::to_string(D) +
              ": at most half of it, and a width of 1024");
  if (pos.scalar_type() != at::kInt && pos.scalar_type() != at::kLong)
    bad_type("positions: int32 or int64 is needed, got " + name(pos.scalar_type()));
  const int64_t o = pos.dim() - 2;
  if (o < 0 || o > 1 || (o == 1 && pos.size(0) != B) || pos.size(o) != N || pos.size(o + 1) != t.axes)
    bad_value("positions " + shape(pos) + ": (" + std::to_string(B) + ", " + std::to_string(N) + ", " +
              std::to_string(t.axes) + ") or its last two are needed");
  if (B * N > INT_MAX || q.size(2) > 4096 || (k.defined() && k.size(2) > 4096))
    bad_value("at most 2^31 - 1 tokens and 4096 heads");
}

// new tensors; either of q and k may be undefined
std::pair<Tensor, Tensor> rotate(const Tensor& q, const Tensor& k, const Tensor& pos, const TurnTable& t,
                                 bool interleaved, bool inverse) {
  const Tensor& one = q.defined() ? q : k;
  dfcsa_rotary_desc d = {};
  Tensor in[2] = {q, k}, out[2];
  bool any = false;
  for (int i = 0; i < 2; ++i) {
    if (!in[i].defined()) continue;
    if (in[i].stride(3) != 1 && in[i].size(3) > 1) in[i] = in[i].contiguous();
    out[i] = at::empty(in[i].sizes(), in[i].options());
    any = any || out[i].numel() > 0;
    d.heads[i] = (int)in[i].size(2);
    d.src[i] = ptr(in[i]);
    d.dst[i] = ptr(out[i]);
    d.src_sb[i] = in[i].stride(0);
    d.src_sn[i] = in[i].stride(1);
    d.src_sh[i] = in[i].stride(2);
  }
  if (any) {
    d.dtype = dtype_of(one, "q");
    d.B = (int)one.size(0);
    d.N = (int)one.size(1);
    d.D = (int)one.size(3);
    d.npairs = (int)t.turns.size();
    d.naxes = t.axes;
    d.interleaved = interleaved;
    d.inverse = inverse;
    d.positions = ptr(pos);
    d.pos64 = pos.scalar_type() == at::kLong;
    d.pos_sb = pos.dim() == 3 ? pos.stride(0) : 0;
    d.pos_sn = pos.stride(-2);
    d.pos_sa = pos.stride(-1);
    d.turns = t.turns.data();
    d.axis = t.axis.data();
    const On on(one);
    done(api.rotary(&d, on.stream), "dfcsa_rotary");
  }
  return {out[0], out[1]};
}

using TablePtr = std::shared_ptr<TurnTable>;
struct TableHolder : public torch::CustomClassHolder {
  TablePtr t;
  explicit TableHolder(TablePtr p) : t(std::move(p)) {}
};

struct Rotary : public Function<Rotary> {
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const std::optional<Tensor>& k, const Tensor& pos,
                               const c10::intrusive_ptr<TableHolder>& table, bool interleaved) {
    ctx->save_for_backward({pos});
    ctx->saved_data["table"] = c10::IValue::make_capsule(table);
    ctx->saved_data["interleaved"] = interleaved;
    ctx->set_materialize_grads(false);
    auto [a, b] = rotate(q, k.value_or(Tensor()), pos, *table->t, interleaved, false);
    if (!k) return {a};
    return {a, b};
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    first_order(g);
    const Tensor gq = ctx->needs_input_grad(0) ? g[0] : Tensor();
    const Tensor gk = g.size() > 1 && ctx->needs_input_grad(1) ? g[1] : Tensor();
    if (!gq.defined() && !gk.defined()) return {Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
    const auto holder = c10::static_intrusive_pointer_cast<TableHolder>(ctx->saved_data["table"].toCapsule());
    auto [dq, dk] = rotate(gq, gk, ctx->get_saved_variables()[0], *holder->t, ctx->saved_data["interleaved"].toBool(), true);
    return {dq, dk, Tensor(), Tensor(), Tensor()};
  }
};

std::tuple<Tensor, std::optional<Tensor>> rotary(const Tensor& q, const std::optional<Tensor>& k0, const Tensor& pos,
                                                 const TablePtr& table, bool interleaved) {
  const Tensor k = k0.value_or(Tensor());
  need_plain({q, k, pos});
  rotary_check(q, k, pos, *table);
  Tensor a, b;
  if (wants_grad({&q, &k})) {
    const variable_list o = Rotary::apply(q, k.defined() ? std::optional<Tensor>(k) : std::nullopt, pos,
                                          c10::make_intrusive<TableHolder>(table), interleaved);
    a = o[0];
    if (o.size() > 1) b = o[1];
  } else {
    std::tie(a, b) = rotate(q, k, pos, *table, interleaved, false);
  }
  return {a, b.defined() ? std::optional<Tensor>(b) : std::nullopt};
}

// ------------------------------------------------------------------ attention
// a dimension of one has whatever stride its tensor came with; it is never multiplied by more than 0
int64_t step(const Tensor& t, int i) { return t.size(i) == 1 ? 0 : t.stride(i); }
// strides the kernels read in place, or a contiguous copy; group: heads that a tile spans (k and v: 0)
Tensor strided(const Tensor& t, int64_t group) {
  const int64_t es = t.element_size();
  if (t.stride(3) != 1 || (uintptr_t)t.data_ptr() % 16 || step(t, 0) * es % 16 || step(t, 1) * es % 16 ||
      step(t, 2) * es % 16 || step(t, 1) * es >= 1 << 23 || step(t, 2) * es * group >= 1 << 29)
    return packed(t);
  return t;
}

void attn_check(const Tensor& q, const Tensor& k, const Tensor& v, int64_t window, int64_t sinks, double scale,
                const Tensor& lengths, bool cached) {
  need_gpu({&q, &k, &v, &lengths});
  dtype_of(q, "q");
  if (k.scalar_type() != q.scalar_type() || v.scalar_type() != q.scalar_type())
    bad_type("q " + name(q.scalar_type()) + ", k " + name(k.scalar_type()) + ", v " + name(v.scalar_type()) +
             ": one type is needed");
  if (q.dim() != 4 || k.dim() != 4 || !k.sizes().equals(v.sizes()))
    bad_value("q [batch, tokens, heads, width] and k, v of one shape [batch, keys, key heads, width] are needed, got " +
              shape(q) + ", " + shape(k) + ", " + shape(v));
  const int64_t B = q.size(0), T = q.size(1), H = q.size(2), D = q.size(3), M = k.size(1), Hk = k.size(2);
  if (k.size(0) != B || k.size(3) != D) bad_value("q " + shape(q) + " and k " + shape(k) + " differ in batch or width");
  if (Hk < 1 || H < 1 || H % Hk || H > 65536)
    bad_value(std::to_string(H) + " heads over " + std::to_string(Hk) + " key heads: a multiple is needed");
  if (D < 8 || D % 8 || D > 128) bad_value("width " + std::to_string(D) + ": a multiple of 8 up to 128 is needed");
  if (window < 1) bad_value("window " + std::to_string(window) + ": at least 1");
  if (sinks < 0) bad_value("sinks " + std::to_string(sinks) + ": at least 0");
  if (!(scale > 0.0) || !((float)scale > 0.f) || !std::isfinite((float)scale))
    bad_value("scale: a finite value above 0 is needed");
  if (lengths.defined()) {
    if (lengths.scalar_type() != at::kInt) bad_type("lengths: int32 is needed, got " + name(lengths.scalar_type()));
    if (lengths.dim() != 1 || lengths.size(0) != B)
      bad_value("lengths " + shape(lengths) + ": (" + std::to_string(B) + ",) is needed");
  }
  const int64_t G = H / Hk;
  if (T > INT_MAX || M > INT_MAX || T * G > 1 << 29 || M * G > 1 << 29 || B * Hk > 1 << 24)
    bad_value("at most 2^29 tokens times heads per key head, and 2^24 sequences times key heads");
  // tiles of 128 rows or keys: what one launch of the kernels can hold (cached: the rows alone count)
  const int64_t long_side = std::max(T * G, cached ? 0 : M);
  if (B * Hk * std::max<int64_t>((long_side + 127) / 128, 1) >= (1 << 23) - 24)
    bad_value("sequences times key heads times tiles of 128 tokens: fewer than 2^23 - 24 are needed");
  if (H * D * q.element_size() >= 1 << 23) bad_value("a token of q: less than 2^23 bytes are needed");
  if (!std::isfinite((float)scale * 1.5f)) bad_value("scale: too large for float32 scores");
}

struct Attn {
  int window, sinks;
  bool causal, cached;
  float scale;
};
void set_strides(int64_t (&s)[3], const Tensor& t) {
  for (int i = 0; i < 3; ++i) s[i] = step(t, i);
}
dfcsa_wattn_desc attn_desc(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& lengths, const Attn& p,
                           const Tensor& o, const Tensor& lse, const Tensor& rest) {
  dfcsa_wattn_desc d = {};
  d.dtype = q.scalar_type() == at::kFloat ? DFCSA_DT_F32 : DFCSA_DT_BF16;
  d.B = (int)q.size(0);
  d.T = (int)q.size(1);
  d.M = (int)k.size(1);
  d.H = (int)q.size(2);
  d.Hk = (int)k.size(2);
  d.D = (int)q.size(3);
  d.window = p.window;
  d.sinks = p.sinks;
  d.causal = p.causal;
  d.cached = p.cached;
  d.scale = p.scale;
  d.q = ptr(q);
  d.k = ptr(k);
  d.v = ptr(v);
  set_strides(d.q_stride, q);
  set_strides(d.k_stride, k);
  set_strides(d.v_stride, v);
  d.lengths = lengths.defined() ? (const int*)lengths.data_ptr() : nullptr;
  d.o = ptr(o);
  d.lse = fptr(lse);
  d.o_rest = ptr(rest);
  return d;
}
Tensor workspace(dfcsa_wattn_desc& d, int backward, const Tensor& like) {
  int64_t n = 0;
  done(api.wattn_work_floats(&d, backward, &n), "dfcsa_wattn_work_floats");
  if (!n) return Tensor();
  const Tensor w = floats(like, n);
  d.work = fptr(w);
  d.work_floats = n;
  return w;
}
// q, k, v as strided() gives them, lengths contiguous
Tensor attend(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& lengths, const Attn& p, const Tensor& lse,
              const Tensor& rest) {
  const On on(q);
  const Tensor o = at::empty(q.sizes(), q.options());
  dfcsa_wattn_desc d = attn_desc(q, k, v, lengths, p, o, lse, rest);
  const Tensor work = workspace(d, 0, q);
  done(api.wattn_fwd(&d, on.stream), "dfcsa_wattn_fwd");
  return o;
}

struct WindowAttention : public Function<WindowAttention> {
  static Tensor forward(AutogradContext* ctx, const Tensor& q0, const Tensor& k0, const Tensor& v0,
                        const std::optional<Tensor>& lengths0, int64_t window, int64_t sinks, bool causal, double scale) {
    const Tensor lengths = lengths0.value_or(Tensor());
    const Tensor q = strided(q0, q0.size(2) / k0.size(2)), k = strided(k0, 0), v = strided(v0, 0);
    const Tensor lse = floats(q, q.size(0) * q.size(1) * q.size(2));
    // bf16: the backward's dO . O needs more of O than its 8 bits, so what the rounding left is kept too
    const Tensor rest = q.scalar_type() == at::kBFloat16 ? at::empty(q.sizes(), q.options()) : Tensor();
    const Tensor o = attend(q, k, v, lengths, Attn{(int)window, (int)sinks, causal, false, (float)scale}, lse, rest);
    ctx->save_for_backward({q0, k0, v0, o, lse, lengths, rest});
    ctx->saved_data["window"] = window;
    ctx->saved_data["sinks"] = sinks;
    ctx->saved_data["causal"] = causal;
    ctx->saved_data["scale"] = scale;
    return o;
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    first_order(g);
    const auto s = ctx->get_saved_variables();
    const int64_t G = s[0].size(2) / s[1].size(2);
    const Tensor q = strided(s[0], G), k = strided(s[1], 0), v = strided(s[2], 0), dout = strided(g[0], G);
    const Attn p{(int)ctx->saved_data["window"].toInt(), (int)ctx->saved_data["sinks"].toInt(),
                 ctx->saved_data["causal"].toBool(), false, (float)ctx->saved_data["scale"].toDouble()};
    const On on(q);
    const bool keys = ctx->needs_input_grad(1) || ctx->needs_input_grad(2);   // else the key-major passes are left out
    const Tensor dq = at::empty(q.sizes(), q.options()), dk = keys ? at::empty(k.sizes(), k.options()) : Tensor(),
                 dv = keys ? at::empty(v.sizes(), v.options()) : Tensor(), delta = at::empty(s[4].sizes(), s[4].options());
    dfcsa_wattn_desc d = attn_desc(q, k, v, s[5], p, s[3], s[4], s[6]);
    d.dout = ptr(dout);
    set_strides(d.dout_stride, dout);
    d.delta = fptr(delta);
    d.dq = ptr(dq);
    d.dk = ptr(dk);
    d.dv = ptr(dv);
    const Tensor work = workspace(d, 1, q);
    done(api.wattn_bwd(&d, on.stream), "dfcsa_wattn_bwd");
    const Tensor n;
    return {dq, dk, dv, n, n, n, n, n};
  }
};
// no tokens: zero gradients
struct Nothing : public Function<Nothing> {
  static Tensor forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v) {
    ctx->save_for_backward({q, k, v});
    return at::zeros(q.sizes(), q.options());
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    first_order(g);
    variable_list z;
    for (const Tensor& t : ctx->get_saved_variables()) z.push_back(at::zeros_like(t));
    return z;
  }
};

int clamp32(int64_t v) { return (int)std::min<int64_t>(v, INT_MAX); }

Tensor window_attention(const Tensor& q, const Tensor& k, const Tensor& v, int64_t window, int64_t sinks, bool causal,
                        double scale, const std::optional<Tensor>& lengths0) {
  Tensor lengths = lengths0.value_or(Tensor());
  need_plain({q, k, v, lengths});
  attn_check(q, k, v, window, sinks, scale, lengths, false);
  if (k.size(1) != q.size(1))
    bad_value(std::to_string(q.size(1)) + " queries and " + std::to_string(k.size(1)) +
              " keys: as many are needed (or window_attention_cached)");
  if (q.numel() == 0) return Nothing::apply(q, k, v);
  if (lengths.defined()) lengths = lengths.contiguous();
  if (wants_grad({&q, &k, &v}))
    return WindowAttention::apply(q, k, v, lengths.defined() ? std::optional<Tensor>(lengths) : std::nullopt, (int64_t)clamp32(window), (int64_t)clamp32(sinks), causal, scale);
  return attend(strided(q, q.size(2) / k.size(2)), strided(k, 0), strided(v, 0), lengths,
                Attn{clamp32(window), clamp32(sinks), causal, false, (float)scale}, Tensor(), Tensor());
}

Tensor window_attention_cached(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& lengths, int64_t window,
                               int64_t sinks, double scale) {
  need_plain({q, k, v, lengths});
  if (wants_grad({&q, &k, &v}))
    throw std::runtime_error("window_attention_cached has no gradient: call it under torch.no_grad(), or window_attention");
  attn_check(q, k, v, window, sinks, scale, lengths, true);
  if (q.numel() == 0 || k.size(1) == 0) return at::zeros(q.sizes(), q.options());
  return attend(strided(q, q.size(2) / k.size(2)), strided(k, 0), strided(v, 0), lengths.contiguous(),
                Attn{clamp32(window), clamp32(sinks), true, true, (float)scale}, Tensor(), Tensor());
}

}  // namespace

PYBIND11_MODULE(_tokens, m) {
  m.def("bind", &bind);
  py::class_<TurnTable, TablePtr>(m, "TurnTable").def(py::init<const std::vector<int64_t>&, double, bool>());
  m.def("rms_norm_residual", &rms_norm_residual);
  m.def("rms_norm_residual_q8", &rms_norm_residual_q8);
  m.def("dequant_q8", [](const Tensor& y8, const Tensor& s, const py::object& dtype) {
    return dequant_q8(y8, s, torch::python::detail::py_object_to_dtype(dtype));
  });
  m.def("rotary", &rotary);
  m.def("window_attention", &window_attention);
  m.def("window_attention_cached", &window_attention_cached);
}
