// The operators as torch functions: the checks of their arguments, the tensors of their results and workspaces, and
// their places in the autograd graph.  In C++ because at the sizes of one image or one token the host is what counts:
// through Python the same calls cost 22 - 24 us forward and about 190 us with a backward pass, the kernels 5 - 60.
//
// Everything runs on the tensors' own device and its current stream.  Refusals are Python's ValueError, TypeError and
// RuntimeError, raised before anything is allocated or launched.
#include <ATen/ATen.h>
#include <ATen/TensorUtils.h>
#include <ATen/autocast_mode.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/utils/pybind.h>

#include <sstream>

#include "pixelsplat_ops.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
namespace py = pybind11;

template <typename... A>
std::string text(const A&... a) {
  std::ostringstream s;
  (s << ... << a);
  return s.str();
}
template <typename... A>
void need_value(bool ok, const A&... a) {
  if (!ok) throw py::value_error(text(a...));
}
std::string shape(const Tensor& t) {
  std::ostringstream s;
  s << "(";
  for (int64_t i = 0; i < t.dim(); ++i) s << (i ? ", " : "") << t.size(i);
  s << ")";
  return s.str();
}

int dtype_code(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return PS_DTYPE_F32;
    case at::kBFloat16: return PS_DTYPE_BF16;
    case at::kHalf: return PS_DTYPE_F16;
    default: return -1;
  }
}
void check_dtype(const char* op, const Tensor& t) {
  if (dtype_code(t) < 0) throw py::type_error(text(op, ": fp32, bf16 or fp16 tensors, got ", t.scalar_type()));
}
// last of the checks: the arguments fit each other, now where they lie
void check_device(const char* op, const Tensor& first, std::initializer_list<std::pair<const char*, const Tensor*>> others) {
  if (!first.is_cuda()) throw std::runtime_error(text(op, " needs GPU tensors (no CPU fallback)"));
  for (const auto& o : others)
    if (o.second->defined() && o.second->device() != first.device())
      throw std::runtime_error(text(op, ": ", o.first, " is on ", o.second->device(), ", the input on ", first.device()));
}

// Under autocast the tensors of products take its type, as those of torch's own products do.  (The norm's and the
// attention table's parameters may be fp32 beside 16-bit tensors and stay what they are.)
Tensor cast(const Tensor& t) {
  return t.defined() && at::autocast::is_autocast_enabled(at::kCUDA)
             ? at::autocast::cached_cast(at::autocast::get_autocast_dtype(at::kCUDA), t, at::kCUDA) : t;
}

void check_status(const char* what, int rc) {
  if (rc == PS_OK) return;
  const char* why = rc == PS_ERR_BAD_ARG ? "bad argument (null or misaligned pointer, inconsistent descriptor)"
                    : rc == PS_ERR_WORKSPACE ? "workspace too small"
                    : rc == PS_ERR_LAUNCH ? "HIP launch failed" : "unsupported configuration";
  throw std::runtime_error(text(what, " failed: ", why, " (PsStatus ", rc, ")"));
}

void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }
void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
float* f32(const Tensor& t) { return t.defined() ? t.data_ptr<float>() : nullptr; }
Tensor bytes(size_t n, const Tensor& like) { return at::empty({(int64_t)n}, like.options().dtype(at::kByte)); }
bool wants_grad(std::initializer_list<const Tensor*> ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor* t : ts)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}
void once(const char* op) {
  // create_graph: the backward's own results would have to be differentiable
  if (at::GradMode::is_enabled()) throw std::runtime_error(text(op, " is differentiable once: no create_graph"));
}
Tensor plain(const Tensor& t) { return t.defined() ? t.detach().contiguous() : t; }
// Function::apply takes no undefined tensor; a missing one has no edge, and the edges behind it move up
using Maybe = std::optional<Tensor>;
Maybe maybe(const Tensor& t) { return t.defined() ? Maybe(t) : Maybe(); }
struct Edges {
  const AutogradContext* ctx;
  int next = 0;
  bool wanted(const Tensor& t) { return t.defined() && ctx->needs_input_grad(next++); }
};
bool aligned16(const Tensor& t) { return (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0; }
int64_t vec_of(const Tensor& t) { return 16 / t.element_size(); }

// ---- group norm ---------------------------------------------------------------------------------------------------
// [n, rows, c] with unit channel stride: a view where the strides allow one, a copy otherwise
Tensor rows_view(const Tensor& x) {
  const int64_t n = x.size(0), c = x.size(-1);
  Tensor v = x.dim() == 3 ? x : x.reshape({n, x.numel() / (n * c), c});
  if ((c > 1 && v.stride(2) != 1) || (v.size(1) > 1 && v.stride(1) < c)) v = v.contiguous();
  return v;
}

PsGroupNormDesc norm_desc(const Tensor& x, int64_t groups, double eps, int64_t act, const Tensor& param, const Tensor& dy) {
  PsGroupNormDesc d = {};
  const int64_t n = x.size(0), s = x.size(1), c = x.size(2);
  need_value(n <= 65535 && c <= 8192 && s * c < ((int64_t)1 << 31),
             "group_norm: at most 65535 samples, 8192 channels and 2^31 elements in a sample, got ", n, ", ", c, ", ", s * c);
  d.samples = (int32_t)n; d.rows = (int32_t)s; d.channels = (int32_t)c; d.groups = (int32_t)groups;
  d.dtype = dtype_code(x); d.activation = (int32_t)act; d.param_f32 = param.defined() && param.scalar_type() == at::kFloat;
  d.eps = (float)eps;
  d.x_sample_stride = n > 1 ? x.stride(0) : 0;
  d.x_row_stride = s > 1 ? x.stride(1) : c;
  if (dy.defined()) {
    d.dy_sample_stride = n > 1 ? dy.stride(0) : 0;
    d.dy_row_stride = s > 1 ? dy.stride(1) : c;
  }
  return d;
}

// x [n, rows, c] -> y of x's shape `sizes`; stats [2, n, groups]
Tensor norm_forward(const Tensor& x, at::IntArrayRef sizes, int64_t groups, const Tensor& w, const Tensor& b, double eps,
                    int64_t act, Tensor& stats) {
  const PsGroupNormDesc d = norm_desc(x, groups, eps, act, w.defined() ? w : b, Tensor());
  Tensor y = at::empty(sizes, x.options());
  const int64_t ng = x.size(0) * groups;
  stats = at::empty({2, x.size(0), groups}, x.options().dtype(at::kFloat));
  const size_t size = ps_group_norm_workspace_bytes(&d, 0);
  const Tensor ws = bytes(size, x);
  check_status("ps_group_norm_forward", ps_group_norm_forward(&d, ptr(x), ptr(w), ptr(b), ptr(y), f32(stats), f32(stats) + ng,
                                                              ptr(ws), size, stream_of(x)));
  return y;
}

struct GroupNorm : torch::autograd::Function<GroupNorm> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Maybe& weight, const Maybe& bias, int64_t groups,
                        double eps, int64_t act) {
    const c10::OptionalDeviceGuard guard(x.device());
    ctx->saved_data["groups"] = groups;
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["act"] = act;
    ctx->saved_data["sizes"] = x.sizes().vec();
    const Tensor w = plain(weight.value_or(Tensor())), b = plain(bias.value_or(Tensor()));
    if (x.numel() == 0) {
      ctx->save_for_backward({x, w, b, Tensor()});
      return at::empty(x.sizes(), x.options());
    }
    const Tensor v = rows_view(x.detach());             // what is saved is no view of x, but notices changes of it
    Tensor stats;
    Tensor y = norm_forward(v, x.sizes(), groups, w, b, eps, act, stats);
    ctx->save_for_backward({v, w, b, stats});
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    once("group_norm");
    const auto saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &w = saved[1], &b = saved[2], &stats = saved[3];
    const c10::OptionalDeviceGuard guard(x.device());
    const auto sizes = ctx->saved_data["sizes"].toIntVector();
    Edges edges{ctx, 1};
    const Tensor dw = edges.wanted(w) ? at::empty_like(w) : Tensor();
    const Tensor db = edges.wanted(b) ? at::empty_like(b) : Tensor();
    Tensor dx = at::empty(sizes, x.options());
    if (x.numel() == 0) {
      if (dw.defined()) dw.zero_();
      if (db.defined()) db.zero_();
      return {dx, dw, db, Tensor(), Tensor(), Tensor()};
    }
    const Tensor dy = rows_view(grads[0]);
    const int64_t groups = ctx->saved_data["groups"].toInt(), ng = x.size(0) * groups;
    const PsGroupNormDesc d = norm_desc(x, groups, ctx->saved_data["eps"].toDouble(), ctx->saved_data["act"].toInt(),
                                        w.defined() ? w : b, dy);
    const size_t size = ps_group_norm_workspace_bytes(&d, 1);
    const Tensor ws = bytes(size, x);
    check_status("ps_group_norm_backward",
                 ps_group_norm_backward(&d, ptr(x), ptr(dy), ptr(w), ptr(b), f32(stats), f32(stats) + ng, ptr(dx), ptr(dw),
                                        ptr(db), ptr(ws), size, stream_of(x)));
    return {dx, dw, db, Tensor(), Tensor(), Tensor()};
  }
};

Tensor group_norm(const Tensor& x, int64_t groups, const std::optional<Tensor>& weight, const std::optional<Tensor>& bias,
                  double eps, int64_t act) {
  const Tensor w = weight.value_or(Tensor()), b = bias.value_or(Tensor());
  check_dtype("group_norm", x);
  need_value(x.dim() >= 2, "group_norm: x is [n, ..., channels], got ", shape(x));
  const int64_t c = x.size(-1);
  need_value(groups >= 1 && c > 0 && c % groups == 0, "group_norm: ", c, " channels do not divide into ", groups, " groups");
  need_value(eps >= 0, "group_norm: eps ", eps, " is negative");
  for (const auto& p : {std::make_pair("weight", &w), std::make_pair("bias", &b)}) {
    const Tensor& t = *p.second;
    need_value(!t.defined() || (t.dim() == 1 && t.size(0) == c && (t.scalar_type() == x.scalar_type() || t.scalar_type() == at::kFloat)),
               "group_norm: ", p.first, " is [", c, "] in ", x.scalar_type(), " or Float, got ", t.defined() ? shape(t) : "",
               " ", t.defined() ? t.scalar_type() : x.scalar_type());
  }
  need_value(!w.defined() || !b.defined() || w.scalar_type() == b.scalar_type(),
             "group_norm: weight and bias have different types");
  check_device("group_norm", x, {{"weight", &w}, {"bias", &b}});
  if (wants_grad({&x, &w, &b})) return GroupNorm::apply(x, maybe(w), maybe(b), groups, eps, act);
  const c10::OptionalDeviceGuard guard(x.device());
  const at::NoGradGuard no_grad;
  if (x.numel() == 0) return at::empty(x.sizes(), x.options());
  Tensor stats;
  return norm_forward(rows_view(x), x.sizes(), groups, plain(w), plain(b), eps, act, stats);
}

// ---- gated linear -------------------------------------------------------------------------------------------------
// [rows, dim] as the kernels read it: unit column stride, rows of whole 16-byte chunks that start on one.  Read in place
// where it lies like that, copied (with `pad` zero columns) otherwise.
Tensor chunked(const Tensor& t, int64_t pad) {
  if (pad) return at::constant_pad_nd(t, {0, pad});
  const bool ok = (t.size(1) <= 1 || t.stride(1) == 1) &&
                  (t.size(0) <= 1 || (t.stride(0) % vec_of(t) == 0 && t.stride(0) >= t.size(1))) && aligned16(t);
  return ok ? t : t.clone(at::MemoryFormat::Contiguous);
}
int64_t row_stride(const Tensor& t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); }

PsGatedLinearDesc gated_desc(const Tensor& x, const Tensor& w, int64_t act, const Tensor& dh) {
  PsGatedLinearDesc d = {};
  need_value(x.size(0) <= 1 << 28 && x.size(1) <= 1 << 24 && w.size(0) <= 1 << 24,
             "gated_linear: at most 2^28 rows and 2^24 columns, got ", shape(x), ", ", shape(w));
  d.rows = (int32_t)x.size(0); d.dim = (int32_t)x.size(1); d.hidden = (int32_t)w.size(0);
  d.dtype = dtype_code(x); d.activation = (int32_t)act;
  d.x_row_stride = row_stride(x); d.w_row_stride = row_stride(w);
  d.dh_row_stride = dh.defined() ? row_stride(dh) : 0;
  return d;
}

void gated_operands(Tensor& x, Tensor& wg, Tensor& wu) {
  const int64_t vec = vec_of(x), pad = (vec - x.size(1) % vec) % vec;
  x = chunked(x, pad);
  wg = chunked(wg, pad);
  wu = chunked(wu, pad);
  if (row_stride(wg) != row_stride(wu)) {                // one row stride for both
    wg = wg.clone(at::MemoryFormat::Contiguous);
    wu = wu.clone(at::MemoryFormat::Contiguous);
  }
}

std::vector<int64_t> with_last(at::IntArrayRef sizes, int64_t last) {
  std::vector<int64_t> s = sizes.vec();
  s.back() = last;
  return s;
}

// x [rows, dim] -> h of shape `sizes`; kept [2, rows, hidden] fp32 where asked for
Tensor gated_forward(const Tensor& x, const Tensor& wg, const Tensor& wu, const Tensor& bg, const Tensor& bu, int64_t act,
                     at::IntArrayRef sizes, bool keep, Tensor& kept) {
  const PsGatedLinearDesc d = gated_desc(x, wg, act, Tensor());
  Tensor h = at::empty(sizes, x.options());
  if (keep) kept = at::empty({2, x.size(0), wg.size(0)}, x.options().dtype(at::kFloat));
  float* gate = keep ? f32(kept) : nullptr;
  check_status("ps_gated_linear_forward",
               ps_gated_linear_forward(&d, ptr(x), ptr(wg), ptr(wu), ptr(bg), ptr(bu), ptr(h), gate,
                                       keep ? gate + h.numel() : nullptr, stream_of(x)));
  return h;
}

struct GatedLinear : torch::autograd::Function<GatedLinear> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& w_gate, const Tensor& w_up, const Maybe& b_gate0,
                        const Maybe& b_up0, int64_t act) {
    const c10::OptionalDeviceGuard guard(x.device());
    const Tensor b_gate = b_gate0.value_or(Tensor()), b_up = b_up0.value_or(Tensor());
    ctx->saved_data["act"] = act;
    ctx->saved_data["sizes"] = x.sizes().vec();
    const auto out = with_last(x.sizes(), w_gate.size(0));
    if (x.numel() == 0 || w_gate.numel() == 0) {
      ctx->save_for_backward({x, w_gate, w_up, b_gate, b_up, Tensor()});
      return at::empty(out, x.options());
    }
    Tensor x2 = x.detach().reshape({-1, x.size(-1)}), wg = w_gate.detach(), wu = w_up.detach(), kept;
    gated_operands(x2, wg, wu);
    const Tensor bg = plain(b_gate), bu = plain(b_up);
    Tensor h = gated_forward(x2, wg, wu, bg, bu, act, out, x.scalar_type() == at::kFloat, kept);
    ctx->save_for_backward({x2, wg, wu, bg, bu, kept});
    return h;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    once("gated_linear");
    const auto saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &wg = saved[1], &wu = saved[2], &bg = saved[3], &bu = saved[4], &kept = saved[5];
    const c10::OptionalDeviceGuard guard(x.device());
    const auto sizes = ctx->saved_data["sizes"].toIntVector();
    const int64_t dim = sizes.back();
    Edges edges{ctx};
    auto fresh = [&](const Tensor& t) { return edges.wanted(t) ? at::empty(t.sizes(), t.options()) : Tensor(); };
    Tensor dx = fresh(x);              // in the order of the edges
    Tensor dwg = fresh(wg);
    Tensor dwu = fresh(wu);
    Tensor dbg = fresh(bg);
    Tensor dbu = fresh(bu);
    if (x.numel() == 0 || wg.numel() == 0) {
      for (Tensor* t : {&dx, &dwg, &dwu, &dbg, &dbu})
        if (t->defined()) t->zero_();
      return {dx, dwg, dwu, dbg, dbu, Tensor()};
    }
    Tensor dh = grads[0].reshape({x.size(0), wg.size(0)});
    if ((dh.size(1) > 1 && dh.stride(1) != 1) || (dh.size(0) > 1 && dh.stride(0) < dh.size(1))) dh = dh.contiguous();
    const PsGatedLinearDesc d = gated_desc(x, wg, ctx->saved_data["act"].toInt(), dh);
    const size_t size = ps_gated_linear_backward_workspace_bytes(&d);
    const Tensor ws = bytes(size, x);
    const float* gate = kept.defined() ? f32(kept) : nullptr;
    check_status("ps_gated_linear_backward",
                 ps_gated_linear_backward(&d, ptr(x), ptr(wg), ptr(wu), ptr(bg), ptr(bu), gate,
                                          gate ? gate + kept.numel() / 2 : nullptr, ptr(dh), ptr(dx), ptr(dwg), ptr(dwu),
                                          ptr(dbg), ptr(dbu), ptr(ws), size, stream_of(x)));
    for (Tensor* t : {&dx, &dwg, &dwu})
      if (t->defined() && t->size(1) != dim) *t = t->narrow(1, 0, dim);
    if (dx.defined()) dx = dx.reshape(sizes);
    return {dx, dwg, dwu, dbg, dbu, Tensor()};
  }
};

Tensor gated_linear(const Tensor& x0, const Tensor& w_gate0, const Tensor& w_up0, const std::optional<Tensor>& b_gate,
                    const std::optional<Tensor>& b_up, int64_t act) {
  const Tensor x = cast(x0), w_gate = cast(w_gate0), w_up = cast(w_up0), bg = cast(b_gate.value_or(Tensor())),
               bu = cast(b_up.value_or(Tensor()));
  check_dtype("gated_linear", x);
  need_value(x.dim() >= 1 && w_gate.dim() == 2 && w_gate.sizes() == w_up.sizes() && w_gate.size(1) == x.size(-1),
             "gated_linear: x [..., dim] and two weights [hidden, dim], got ", shape(x), ", ", shape(w_gate), ", ", shape(w_up));
  const int64_t hidden = w_gate.size(0), dim = w_gate.size(1);
  need_value(dim > 0, "gated_linear: dim is 0");
  for (const auto& p : {std::make_pair("w_gate", &w_gate), std::make_pair("w_up", &w_up), std::make_pair("b_gate", &bg),
                        std::make_pair("b_up", &bu)}) {
    const Tensor& t = *p.second;
    need_value(!t.defined() || (t.scalar_type() == x.scalar_type() && (t.dim() == 2 || (t.dim() == 1 && t.size(0) == hidden))),
               "gated_linear: ", p.first, " is [", hidden, p.first[0] == 'w' ? text(", ", dim) : "", "] in ", x.scalar_type(),
               ", got ", t.defined() ? shape(t) : "", " ", t.defined() ? t.scalar_type() : x.scalar_type());
    need_value(!t.defined() || (p.first[0] == 'w') == (t.dim() == 2), "gated_linear: ", p.first, " is [", hidden, "], got ",
               t.defined() ? shape(t) : "");
  }
  check_device("gated_linear", x, {{"w_gate", &w_gate}, {"w_up", &w_up}, {"b_gate", &bg}, {"b_up", &bu}});
  if (wants_grad({&x, &w_gate, &w_up, &bg, &bu})) return GatedLinear::apply(x, w_gate, w_up, maybe(bg), maybe(bu), act);
  const c10::OptionalDeviceGuard guard(x.device());
  const at::NoGradGuard no_grad;
  const auto out = with_last(x.sizes(), hidden);
  if (x.numel() == 0 || hidden == 0) return at::empty(out, x.options());
  Tensor x2 = x.reshape({-1, dim}), wg = w_gate, wu = w_up, kept;
  gated_operands(x2, wg, wu);
  return gated_forward(x2, wg, wu, plain(bg), plain(bu), act, out, false, kept);
}

// ---- attention with a relative position bias ------------------------------------------------------------------------
// [batch, heads, tokens, dim] as the kernels read it: rows that start on 16 bytes
Tensor token_rows(const Tensor& t, int64_t pad) {
  if (pad) return at::constant_pad_nd(t, {0, pad});
  bool ok = (t.size(3) <= 1 || t.stride(3) == 1) && aligned16(t) && t.stride(2) < 1 << 24;
  for (int i = 0; i < 3; ++i) ok = ok && (t.size(i) <= 1 || t.stride(i) % vec_of(t) == 0);
  // copied token-major, as a packed projection would lay it out
  return ok ? t : t.transpose(1, 2).clone(at::MemoryFormat::Contiguous).transpose(1, 2);
}
// The first `dim` columns of a token-major [batch, heads, tokens, like's width].  No view of another tensor: autograd would
// refuse to change a result in place that a function returns as a view.
Tensor token_major(const Tensor& like, int64_t dim) {
  const int64_t h = like.size(1), n = like.size(2), d = like.size(3);
  const std::vector<int64_t> sizes = {like.size(0), h, n, dim}, strides = {n * h * d, d, h * d, 1};
  if (dim == d) return at::empty_strided(sizes, strides, like.options());
  const Tensor room = at::empty({like.numel()}, like.options());
  return at::empty({0}, like.options()).set_(room.storage(), 0, sizes, strides);
}
Tensor token_major(const Tensor& like) { return token_major(like, like.size(3)); }
void strides_of(const Tensor& t, int64_t* s) {
  for (int i = 0; i < 3; ++i) s[i] = t.size(i) > 1 ? t.stride(i) : vec_of(t);
}

PsRelativeAttentionDesc attention_desc(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& table,
                                       const Tensor& buckets, const Tensor& mask, double scale, int64_t start,
                                       const Tensor& dout) {
  PsRelativeAttentionDesc d = {};
  d.batch = (int32_t)q.size(0); d.heads = (int32_t)q.size(1); d.queries = (int32_t)q.size(2); d.query_start = (int32_t)start;
  d.grid_h = (int32_t)(buckets.size(0) + 1) / 2; d.grid_w = (int32_t)(buckets.size(1) + 1) / 2; d.dim = (int32_t)q.size(3);
  d.dtype = dtype_code(q); d.buckets = (int32_t)table.size(0); d.table_f32 = table.scalar_type() == at::kFloat;
  d.scale = (float)scale;
  strides_of(q, d.q_strides);
  strides_of(k, d.k_strides);
  strides_of(v, d.v_strides);
  if (dout.defined()) strides_of(dout, d.do_strides);
  d.mask_stride = mask.defined() ? mask.stride(0) : 0;
  return d;
}

struct Kept { Tensor out32, stats, bias; };

// dim: of the result, whose rows are as wide as q's
Tensor attention_forward(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& table, const Tensor& buckets,
                         const Tensor& mask, double scale, int64_t start, int64_t dim, bool keep, Kept& kept) {
  const PsRelativeAttentionDesc d = attention_desc(q, k, v, table, buckets, mask, scale, start, Tensor());
  const size_t size = ps_relative_attention_workspace_bytes(&d, PS_FORWARD);
  if (size == 0) throw std::runtime_error("relative_attention: unsupported configuration (see its limits)");
  Tensor out = token_major(q, dim);
  const auto fp32 = q.options().dtype(at::kFloat);
  kept.bias = at::empty({q.size(1), buckets.numel()}, fp32);
  if (keep) {
    kept.stats = at::empty({2, q.size(0), q.size(1), (q.size(2) + 63) / 64 * 64}, fp32);
    if (q.scalar_type() != at::kFloat) kept.out32 = at::empty({q.size(0), q.size(2), q.size(1), q.size(3)}, fp32);
  }
  const Tensor ws = bytes(size, q);
  check_status("ps_relative_attention_forward",
               ps_relative_attention_forward(&d, ptr(q), ptr(k), ptr(v), (const uint8_t*)ptr(mask), (const int32_t*)ptr(buckets),
                                             ptr(table), ptr(out), f32(kept.out32), f32(kept.stats), f32(kept.bias), ptr(ws),
                                             size, stream_of(q)));
  return out;
}

struct RelativeAttention : torch::autograd::Function<RelativeAttention> {
  static Tensor forward(AutogradContext* ctx, const Tensor& q0, const Tensor& k0, const Tensor& v0, const Tensor& table0,
                        const Tensor& buckets, const Maybe& mask0, double scale, int64_t start) {
    const c10::OptionalDeviceGuard guard(q0.device());
    const Tensor mask = mask0.value_or(Tensor());
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["start"] = start;
    ctx->saved_data["dim"] = q0.size(3);
    if (q0.numel() == 0) {
      ctx->save_for_backward({q0, k0, v0, table0});
      return token_major(q0);
    }
    const int64_t vec = vec_of(q0), pad = (vec - q0.size(3) % vec) % vec;
    const Tensor q = token_rows(q0.detach(), pad), k = token_rows(k0.detach(), pad), v = token_rows(v0.detach(), pad);
    const Tensor table = plain(table0);
    Kept kept;
    Tensor out = attention_forward(q, k, v, table, buckets, mask, scale, start, q0.size(3), true, kept);
    ctx->save_for_backward({q, k, v, table, buckets, mask, kept.out32.defined() ? kept.out32 : out, kept.stats, kept.bias});
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    once("relative_attention");
    const auto saved = ctx->get_saved_variables();
    const Tensor &q = saved[0], &k = saved[1], &v = saved[2], &table = saved[3];
    const c10::OptionalDeviceGuard guard(q.device());
    const int64_t dim = ctx->saved_data["dim"].toInt();
    Tensor dq, dk, dv, dtable;
    if (ctx->needs_input_grad(0)) dq = token_major(q);
    if (ctx->needs_input_grad(1)) dk = token_major(k);
    if (ctx->needs_input_grad(2)) dv = token_major(v);
    if (ctx->needs_input_grad(3)) dtable = at::empty_like(table);
    if (q.numel() == 0) {
      for (Tensor* t : {&dq, &dk, &dv, &dtable})
        if (t->defined()) t->zero_();
      return {dq, dk, dv, dtable, Tensor(), Tensor(), Tensor(), Tensor()};
    }
    const Tensor &buckets = saved[4], &mask = saved[5], &kept = saved[6], &stats = saved[7], &bias = saved[8];
    const Tensor dout = token_rows(grads[0], q.size(3) - dim);
    const PsRelativeAttentionDesc d = attention_desc(q, k, v, table, buckets, mask, ctx->saved_data["scale"].toDouble(),
                                                     ctx->saved_data["start"].toInt(), dout);
    const size_t size = ps_relative_attention_workspace_bytes(&d, dtable.defined() ? PS_BACKWARD : PS_BACKWARD_NO_TABLE);
    const Tensor ws = bytes(size, q);
    check_status("ps_relative_attention_backward",
                 ps_relative_attention_backward(&d, ptr(q), ptr(k), ptr(v), (const uint8_t*)ptr(mask),
                                                (const int32_t*)ptr(buckets), f32(bias), f32(kept), f32(stats), ptr(dout),
                                                ptr(dq), ptr(dk), ptr(dv), ptr(dtable), ptr(ws), size, stream_of(q)));
    if (q.size(3) != dim)
      for (Tensor* t : {&dq, &dk, &dv})
        if (t->defined()) *t = t->narrow(3, 0, dim);
    return {dq, dk, dv, dtable, Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

Tensor relative_attention(const Tensor& q0, const Tensor& k0, const Tensor& v0, const Tensor& table, const Tensor& buckets0,
                          const std::optional<Tensor>& key_mask, const std::optional<double>& scale0, int64_t start) {
  const Tensor q = cast(q0), k = cast(k0), v = cast(v0);
  Tensor mask = key_mask.value_or(Tensor());
  check_dtype("relative_attention", q);
  need_value(q.dim() == 4 && k.dim() == 4 && k.sizes() == v.sizes() && k.size(0) == q.size(0) && k.size(1) == q.size(1) &&
                 k.size(3) == q.size(3),
             "relative_attention: q [batch, heads, queries, dim], k and v [batch, heads, keys, dim], got ", shape(q), ", ",
             shape(k), ", ", shape(v));
  need_value(k.scalar_type() == q.scalar_type() && v.scalar_type() == q.scalar_type() &&
                 (table.scalar_type() == q.scalar_type() || table.scalar_type() == at::kFloat),
             "relative_attention: k and v are ", q.scalar_type(), " as q, the table that or Float, got ", k.scalar_type(), ", ",
             v.scalar_type(), ", ", table.scalar_type());
  need_value(buckets0.scalar_type() == at::kInt && buckets0.dim() == 2 && buckets0.size(0) % 2 == 1 && buckets0.size(1) % 2 == 1,
             "relative_attention: buckets is [2 rows - 1, 2 columns - 1] int32, got ", shape(buckets0), " ",
             buckets0.scalar_type());
  const int64_t b = q.size(0), h = q.size(1), n = q.size(2), dim = q.size(3);
  const int64_t gh = (buckets0.size(0) + 1) / 2, gw = (buckets0.size(1) + 1) / 2;
  need_value(dim > 0 && dim <= 128 && gh <= 1 << 20 && gw <= 1 << 20 && gh * gw <= 1 << 20 && (gh == 1 || gw <= 512),
             "relative_attention: dim ", dim, " is 1 .. 128, a grid of ", gh, " x ", gw,
             " has at most 2^20 tokens and 512 columns (one row: any)");
  need_value(k.size(2) == gh * gw, "relative_attention: ", k.size(2), " keys on a grid of ", gh, " x ", gw);
  need_value(start >= 0 && start + n <= gh * gw, "relative_attention: queries ", start, " .. ", start + n - 1, " of ", gh * gw,
             " tokens");
  need_value(table.dim() == 2 && table.size(1) == h && table.size(0) > 0 && table.size(0) <= 1 << 24,
             "relative_attention: table is [buckets, ", h, "], got ", shape(table));
  need_value(!mask.defined() || (mask.scalar_type() == at::kBool && mask.dim() == 2 && mask.size(0) == b && mask.size(1) == gh * gw),
             "relative_attention: key_mask is [", b, ", ", gh * gw, "] bool, got ", mask.defined() ? shape(mask) : "", " ",
             mask.defined() ? mask.scalar_type() : at::kBool);
  need_value(h <= 65535 && b * h < 1 << 24 && b * h * ((std::max(n, gh * gw) + 63) / 64 * 2) < 1 << 26,
             "relative_attention: at most 65535 heads, and less than 2^24 heads and 2^26 tiles of 32 tokens in the batch");
  check_device("relative_attention", q, {{"k", &k}, {"v", &v}, {"table", &table}, {"buckets", &buckets0}, {"key_mask", &mask}});
  const double scale = scale0 ? *scale0 : 1.0 / std::sqrt((double)dim);
  const Tensor buckets = buckets0.contiguous();
  if (mask.defined() && mask.size(1) > 1 && mask.stride(1) != 1) mask = mask.contiguous();
  if (wants_grad({&q, &k, &v, &table})) return RelativeAttention::apply(q, k, v, table, buckets, maybe(mask), scale, start);
  const c10::OptionalDeviceGuard guard(q.device());
  const at::NoGradGuard no_grad;
  if (q.numel() == 0) return token_major(q);
  const int64_t vec = vec_of(q), pad = (vec - dim % vec) % vec;
  Kept kept;
  return attention_forward(token_rows(q, pad), token_rows(k, pad), token_rows(v, pad), table.contiguous(), buckets, mask, scale,
                           start, dim, false, kept);
}

}  // namespace

PYBIND11_MODULE(_binding, m) {
  const auto free = py::call_guard<py::gil_scoped_release>();
  m.def("group_norm", &group_norm, free);
  m.def("gated_linear", &gated_linear, free);
  m.def("relative_attention", &relative_attention, free);
}
