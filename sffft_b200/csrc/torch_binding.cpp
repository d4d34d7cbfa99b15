// torch.ops.sffft.linear_attention, linear_attention_step and block_norm over the C ABI, with their gradients.
//
// In C++ because a call's own cost decides at the sizes of single tokens and small batches: through a Python operator and a
// Python autograd function a training step of either cost 165 to 195 us of the host's time and a single call 17 to 21.
// Shapes without a GPU (for tracing) are given in torch_ops.py, where the operators are documented.
#include <ATen/ATen.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/autograd.h>
#include <torch/library.h>

#include <algorithm>
#include <cmath>

#include "../../include/sffft.h"

namespace {

using at::Tensor;
using std::optional;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// Messages are put together without streams: where a process holds two C++ runtimes, formatting a number in one can end it.
void add(std::string& s, const char* x) { s += x; }
void add(std::string& s, int64_t n) { s += std::to_string(n); }
void add(std::string& s, at::ScalarType t) { s += c10::toString(t); }
void add(std::string& s, at::IntArrayRef x) {
  s += '[';
  for (size_t i = 0; i < x.size(); i++) s += (i ? ", " : "") + std::to_string(x[i]);
  s += ']';
}
// ValueError unless ok
template <class... P>
void need(bool ok, const P&... parts) {
  if (ok) return;
  std::string s;
  (add(s, parts), ...);
  TORCH_CHECK_VALUE(false, s);
}

void status(int rc, const char* what) {
  if (rc == SFFFT_OK) return;
  std::string s = what;
  add(s, ": "), add(s, sffft_status_string(rc)), add(s, " (status "), add(s, (int64_t)rc), add(s, ")");
  if (rc == SFFFT_ERR_TIMEOUT)
    add(s, ": results of an earlier call are not valid; sffft_b200.linear_attention_check(device) reports and clears this");
  TORCH_CHECK(false, s);
}

int io_of(const Tensor& t, const char* what) {
  const auto d = t.scalar_type();
  need(d == at::kFloat || d == at::kBFloat16, what, " must be float32 or bfloat16, not ", d);
  return d == at::kBFloat16 ? SFFFT_IO_BF16 : SFFFT_IO_FP32;
}

void same_device(const Tensor& a, const Tensor& b) { need(a.device() == b.device(), "all tensors must be on one device"); }

void need_cuda(const Tensor& t, const char* what) {
  need(t.is_cuda(), what, " needs CUDA tensors (there is no CPU path)");
}

void* stream_of(const Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.get_device()).stream(); }

const void* ptr(const Tensor& t) { return t.const_data_ptr(); }
const void* ptr(const optional<Tensor>& t) { return t ? t->const_data_ptr() : nullptr; }
void* out_ptr(const optional<Tensor>& t) { return t ? t->mutable_data_ptr() : nullptr; }

Tensor unit(const Tensor& t) { return t.stride(-1) == 1 || t.size(-1) == 1 ? t : t.contiguous(); }
optional<Tensor> packed(const optional<Tensor>& t) { return t ? optional<Tensor>(t->contiguous()) : t; }

// An empty [B][H][L][D] tensor whose memory is ordered like `like`'s: [B][L][H][D] where its positions are outermost.
Tensor heads_like(const Tensor& like, int64_t B, int64_t H, int64_t L, int64_t D) {
  if (like.stride(2) > like.stride(1) && H > 1) return at::empty_strided({B, H, L, D}, {L * H * D, D, H * D, 1}, like.options());
  return at::empty({B, H, L, D}, like.options());
}

Tensor workspace(size_t bytes, const Tensor& like) {
  return bytes ? at::empty({(int64_t)bytes}, like.options().dtype(at::kByte)) : Tensor();
}

template <int N>
void strides(long long (&d)[N], const Tensor& t) {
  for (int i = 0; i < N; i++) d[i] = t.stride(i);
}

// ---------------------------------------------------------------------------------------------------------------
// linear attention
// ---------------------------------------------------------------------------------------------------------------
sffft_linear_attention_t check_attention(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& log_decay,
                                         const optional<Tensor>& s0, const optional<Tensor>& lengths, double scale,
                                         const optional<Tensor>& ds1) {
  need(q.dim() == 4 && k.dim() == 4 && v.dim() == 4,
                    "q, k and v must be [B][H][L][D], [B][Hkv][L][D] and [B][Hkv][L][Dv]");
  const int64_t B = q.size(0), H = q.size(1), L = q.size(2), D = q.size(3), Hkv = k.size(1), Dv = v.size(3);
  need(k.size(0) == B && k.size(2) == L && k.size(3) == D && v.size(0) == B && v.size(1) == Hkv && v.size(2) == L,
                    "q ", q.sizes(), ", k ", k.sizes(), " and v ", v.sizes(), " do not belong together");
  need(H > 0 && Hkv > 0 && H % Hkv == 0, H, " query heads cannot share ", Hkv, " key and value heads evenly");
  need(D > 0 && Dv > 0, "head sizes must be positive");
  need(std::max({B, H, L, D, Dv}) < (1ll << 31), "sizes must be below 2^31");
  const int io = io_of(q, "q");
  need(k.scalar_type() == q.scalar_type() && v.scalar_type() == q.scalar_type(), "q, k and v must have one type");
  need(log_decay.dim() == 1 && log_decay.size(0) == H && log_decay.scalar_type() == at::kFloat,
                    "log_decay must be a float32 [", H, "] tensor");
  need(std::isfinite(scale) && scale != 0, "scale must be finite and not 0");
  for (const auto* t : {&s0, &ds1})
    need(!*t || ((*t)->scalar_type() == at::kFloat && (*t)->sizes() == at::IntArrayRef({B, H, D, Dv})),
                      "initial_state and the final state's gradient must be float32 [", B, ", ", H, ", ", D, ", ", Dv, "] tensors");
  need(!lengths || (lengths->dim() == 1 && lengths->size(0) == B && lengths->scalar_type() == at::kInt),
                    "lengths must be an int32 [", B, "] tensor");
  same_device(q, k), same_device(q, v), same_device(q, log_decay);
  for (const auto* t : {&s0, &lengths, &ds1})
    if (*t) same_device(q, **t);
  need_cuda(q, "linear_attention");
  sffft_linear_attention_t d = {(int)B, (int)H, (int)Hkv, (int)L, (int)D, (int)Dv, io, (int)q.get_device(), (float)scale, {}, {}, {}, {}};
  return d;
}

std::tuple<Tensor, Tensor> attention(const Tensor& q_, const Tensor& k_, const Tensor& v_, const Tensor& log_decay,
                                     const optional<Tensor>& s0_, const optional<Tensor>& lengths_, double scale) {
  sffft_linear_attention_t d = check_attention(q_, k_, v_, log_decay, s0_, lengths_, scale, {});
  const Tensor q = unit(q_), k = unit(k_), v = unit(v_), ld = log_decay.contiguous();
  const auto s0 = packed(s0_), lengths = packed(lengths_);
  Tensor y = heads_like(q, d.B, d.H, d.L, d.Dv), s1 = at::empty({d.B, d.H, d.D, d.Dv}, q.options().dtype(at::kFloat));
  strides(d.q_stride, q), strides(d.k_stride, k), strides(d.v_stride, v), strides(d.y_stride, y);
  size_t bytes = 0;
  status(sffft_linear_attention_workspace_bytes(&d, 0, &bytes), "linear_attention");
  const Tensor work = workspace(bytes, q);
  status(sffft_linear_attention(&d, ptr(q), ptr(k), ptr(v), (const float*)ptr(ld), (const int*)ptr(lengths), (const float*)ptr(s0),
                                y.mutable_data_ptr(), (float*)s1.mutable_data_ptr(), bytes ? work.mutable_data_ptr() : nullptr,
                                bytes, stream_of(q)),
         "linear_attention");
  return {y, s1};
}

std::vector<Tensor> attention_backward(const Tensor& q_, const Tensor& k_, const Tensor& v_, const Tensor& log_decay,
                                       const optional<Tensor>& s0_, const optional<Tensor>& lengths_, double scale,
                                       const Tensor& dy_, const optional<Tensor>& ds1_) {
  sffft_linear_attention_t d = check_attention(q_, k_, v_, log_decay, s0_, lengths_, scale, ds1_);
  need(dy_.sizes() == at::IntArrayRef({d.B, d.H, d.L, d.Dv}) && dy_.scalar_type() == q_.scalar_type() &&
                        dy_.device() == q_.device(),
                    "dy must be like y");
  const Tensor q = unit(q_), k = unit(k_), v = unit(v_), ld = log_decay.contiguous();
  Tensor dy = dy_;
  for (int i = 0; i < 4; i++)   // a sum's gradient comes expanded
    if (i == 3 ? dy.stride(3) != 1 : dy.stride(i) == 0) dy = dy.contiguous();
  const auto s0 = packed(s0_), lengths = packed(lengths_), ds1 = packed(ds1_);
  Tensor dq = heads_like(q, d.B, d.H, d.L, d.D), dk = heads_like(k, d.B, d.Hkv, d.L, d.D), dv = heads_like(v, d.B, d.Hkv, d.L, d.Dv);
  optional<Tensor> ds0;
  if (s0) ds0 = at::empty({d.B, d.H, d.D, d.Dv}, s0->options());
  strides(d.q_stride, q), strides(d.k_stride, k), strides(d.v_stride, v);
  sffft_linear_attention_grads_t g;
  strides(g.dy_stride, dy), strides(g.dq_stride, dq), strides(g.dk_stride, dk), strides(g.dv_stride, dv);
  size_t bytes = 0;
  status(sffft_linear_attention_workspace_bytes(&d, 1, &bytes), "linear_attention_backward");
  const Tensor work = workspace(bytes, q);
  status(sffft_linear_attention_backward(&d, &g, ptr(q), ptr(k), ptr(v), (const float*)ptr(ld), (const int*)ptr(lengths),
                                         (const float*)ptr(s0), ptr(dy), (const float*)ptr(ds1), dq.mutable_data_ptr(),
                                         dk.mutable_data_ptr(), dv.mutable_data_ptr(), (float*)out_ptr(ds0),
                                         bytes ? work.mutable_data_ptr() : nullptr, bytes, stream_of(q)),
         "linear_attention_backward");
  std::vector<Tensor> out = {dq, dk, dv};
  if (ds0) out.push_back(*ds0);
  return out;
}

Tensor attention_step(const Tensor& q_, const Tensor& k_, const Tensor& v_, const Tensor& log_decay, Tensor& state,
                      const optional<Tensor>& slots_, double scale) {
  need(q_.dim() == 3 && k_.dim() == 3 && v_.dim() == 3, "q, k and v must be [B][H][D], [B][Hkv][D] and [B][Hkv][Dv]");
  const int64_t B = q_.size(0), H = q_.size(1), D = q_.size(2), Hkv = k_.size(1), Dv = v_.size(2);
  need(k_.size(0) == B && k_.size(2) == D && v_.size(0) == B && v_.size(1) == Hkv, "q ", q_.sizes(), ", k ",
                    k_.sizes(), " and v ", v_.sizes(), " do not belong together");
  need(H > 0 && Hkv > 0 && H % Hkv == 0, H, " query heads cannot share ", Hkv, " key and value heads evenly");
  need(D > 0 && Dv > 0, "head sizes must be positive");
  const int io = io_of(q_, "q");
  need(k_.scalar_type() == q_.scalar_type() && v_.scalar_type() == q_.scalar_type(), "q, k and v must have one type");
  need(log_decay.dim() == 1 && log_decay.size(0) == H && log_decay.scalar_type() == at::kFloat,
                    "log_decay must be a float32 [", H, "] tensor");
  need(std::isfinite(scale), "scale must be finite");
  need(state.dim() == 4 && state.size(1) == H && state.size(2) == D && state.size(3) == Dv &&
                        state.scalar_type() == at::kFloat,
                    "state must be a float32 [pool, ", H, ", ", D, ", ", Dv, "] tensor");
  const int64_t pool = state.size(0);
  auto axis = [&](int i, int64_t want) { return state.size(i) == 1 || state.stride(i) == want; };
  need(axis(1, D * Dv) && axis(2, Dv) && axis(3, 1) && (pool <= 1 || state.stride(0) >= H * D * Dv),
                    "a slot's state must be contiguous and slots must not overlap");
  need(!slots_ || (slots_->dim() == 1 && slots_->size(0) == B && slots_->scalar_type() == at::kInt),
                    "slots must be an int32 [", B, "] tensor");
  need(slots_ || pool >= B, B, " rows need ", B, " slots");
  need(std::max({B, H, D, Dv, pool}) < (1ll << 31), "sizes must be below 2^31");
  same_device(q_, k_), same_device(q_, v_), same_device(q_, log_decay), same_device(q_, state);
  if (slots_) same_device(q_, *slots_);
  need_cuda(q_, "linear_attention_step");
  const Tensor q = unit(q_), k = unit(k_), v = unit(v_), ld = log_decay.contiguous();
  const auto slots = packed(slots_);
  Tensor y = at::empty({B, H, Dv}, q.options());
  sffft_linear_attention_step_t d = {(int)B, (int)H, (int)Hkv, (int)D, (int)Dv, (int)pool, io, (int)q.get_device(), (float)scale,
                                     {}, {}, {}, {}, state.stride(0)};
  strides(d.q_stride, q), strides(d.k_stride, k), strides(d.v_stride, v), strides(d.y_stride, y);
  status(sffft_linear_attention_step(&d, ptr(q), ptr(k), ptr(v), (const float*)ptr(ld), (float*)state.mutable_data_ptr(),
                                     (const int*)ptr(slots), y.mutable_data_ptr(), stream_of(q)),
         "linear_attention_step");
  return y;
}

// ---------------------------------------------------------------------------------------------------------------
// norms around a block
// ---------------------------------------------------------------------------------------------------------------
struct NormCall {
  sffft_block_norm_t d;
  optional<Tensor> x, y, gate, pw, w;
  Tensor lead;
};

// The tensor with evenly spaced rows of contiguous channels (a copy where it has not), and their stride.
Tensor as_rows(const Tensor& t, int64_t C, long long* stride) {
  *stride = C;
  if (t.is_contiguous()) return t;
  if (t.size(-1) > 1 && t.stride(-1) != 1) return t.contiguous();
  int64_t step = -1, rows = 1;
  for (int64_t i = t.dim() - 2; i >= 0; i--) {
    if (t.size(i) == 1) continue;
    if (step < 0) step = t.stride(i);
    else if (t.stride(i) != step * rows) return t.contiguous();
    rows *= t.size(i);
  }
  if (step >= 0) *stride = step;
  return t;
}

NormCall norm_call(const optional<Tensor>& x, const optional<Tensor>& y, const optional<Tensor>& gate, const optional<Tensor>& pw,
                   const optional<Tensor>& w, double scale, double eps, int64_t groups, c10::string_view act, int64_t dim) {
  need(x || y, "block_norm needs x or y");
  const Tensor& lead = y ? *y : *x;
  const int64_t nd = lead.dim();
  need(dim == -1 || dim == 1 || dim == nd - 1, "dim must be -1, or 1 for [B][C][L] tensors");
  const bool first = dim == 1 && nd != 2;
  need(!first || nd == 3, "dim 1 is for [B][C][L] tensors");
  need(nd >= 1 && lead.size(dim) > 0, "there must be channels");
  const int64_t C = lead.size(dim);
  const int io = io_of(lead, "the tensors");
  if (!y) {
    need(!gate && !pw, "a gate and post_weight act on y");
    need(w.has_value(), "without y there must be a weight to norm x with");
  }
  if (x && y) {
    need(x->sizes() == y->sizes(), "x ", x->sizes(), " and y ", y->sizes(), " must have one shape");
    need(x->scalar_type() == y->scalar_type() || x->scalar_type() == at::kFloat,
                      "x must have y's type, or be float32 beside bfloat16");
    same_device(*x, *y);
  }
  int kind = SFFFT_GATE_NONE;
  if (gate) {
    kind = gate->sizes() == y->sizes() ? SFFFT_GATE_FULL : SFFFT_GATE_CHANNEL;
    need(kind == SFFFT_GATE_FULL || (gate->dim() == 1 && gate->size(0) == C), "gate must be shaped like y or [", C, "]");
    need(gate->scalar_type() == y->scalar_type(), "gate must have y's type");
    same_device(lead, *gate);
  }
  int wio = SFFFT_IO_FP32;
  for (const auto* t : {&pw, &w})
    if (*t) {
      need((*t)->dim() == 1 && (*t)->size(0) == C, "the weights must be [", C, "]");
      wio = io_of(**t, "the weights");
      same_device(lead, **t);
    }
  need(!pw || !w || pw->scalar_type() == w->scalar_type(), "the weights must have one type");
  need(groups >= 1 && C % groups == 0, C, " channels do not fall into ", groups, " groups");
  const int a = act == "none" ? SFFFT_ACT_NONE : act == "silu" ? SFFFT_ACT_SILU : act == "sigmoid" ? SFFFT_ACT_SIGMOID : -1;
  need(a >= 0, "act must be none, silu or sigmoid");
  need(std::isfinite(scale), "scale must be finite");
  need(std::isfinite(eps) && eps >= 0, "eps must be finite and not negative");
  need_cuda(lead, "block_norm");
  need(C < (1ll << 31) && (!first || lead.size(2) < (1ll << 31)), "sizes must be below 2^31");
  NormCall c;
  c.lead = lead;
  c.d = {lead.numel() / C, (int)C, first ? (int)lead.size(2) : 0, (int)groups, io,
         (x ? *x : lead).scalar_type() == at::kBFloat16 ? SFFFT_IO_BF16 : SFFFT_IO_FP32, wio, kind, a, (float)scale, (float)eps,
         (int)lead.get_device(), 0, 0, 0};
  if (first) {
    c.x = packed(x), c.y = packed(y), c.gate = packed(gate);
  } else {
    if (x) c.x = as_rows(*x, C, &c.d.x_stride);
    if (y) c.y = as_rows(*y, C, &c.d.y_stride);
    if (gate) c.gate = kind == SFFFT_GATE_FULL ? as_rows(*gate, C, &c.d.gate_stride) : gate->contiguous();
  }
  c.pw = packed(pw), c.w = packed(w);
  return c;
}

Tensor packed_like(const Tensor& t) { return at::empty(t.sizes(), t.options()); }

// h (with y), n (with weight); with stats also the rstd of y's groups (with post_weight) and of h (with weight)
std::vector<Tensor> norm(const optional<Tensor>& x, const optional<Tensor>& y, const optional<Tensor>& gate, const optional<Tensor>& pw,
                         const optional<Tensor>& w, double scale, double eps, int64_t groups, c10::string_view act, int64_t dim,
                         bool stats) {
  const NormCall c = norm_call(x, y, gate, pw, w, scale, eps, groups, act, dim);
  optional<Tensor> h, n, r1, r2;
  const auto f32 = c.lead.options().dtype(at::kFloat);
  if (y) h = packed_like(x ? *x : *y);
  if (w) n = packed_like(c.lead);
  if (stats && pw) r1 = at::empty({c.d.rows, groups}, f32);
  if (stats && w) r2 = at::empty({c.d.rows}, f32);
  if (c.d.rows)
    status(sffft_block_norm(&c.d, ptr(c.x), ptr(c.y), ptr(c.gate), ptr(c.pw), ptr(c.w), out_ptr(h), out_ptr(n), (float*)out_ptr(r1),
                            (float*)out_ptr(r2), stream_of(c.lead)),
           "block_norm");
  std::vector<Tensor> out;
  for (const auto* t : {&h, &n, &r1, &r2})
    if (*t) out.push_back(**t);
  return out;
}

std::vector<Tensor> norm_backward(const optional<Tensor>& dh, const optional<Tensor>& dn, const optional<Tensor>& x,
                                  const optional<Tensor>& y, const optional<Tensor>& gate, const optional<Tensor>& pw,
                                  const optional<Tensor>& w, const optional<Tensor>& rstd_post, const optional<Tensor>& rstd,
                                  double scale, double eps, int64_t groups, c10::string_view act, int64_t dim) {
  const NormCall c = norm_call(x, y, gate, pw, w, scale, eps, groups, act, dim);
  need(dn.has_value() == w.has_value(), "dn is needed where there is a weight, and only there");
  need(dh || w, "dh or dn is needed");
  auto like = [&](const optional<Tensor>& t, const Tensor& as, const char* what) {
    if (!t) return;
    need(t->sizes() == as.sizes() && t->scalar_type() == as.scalar_type(), what);
    same_device(c.lead, *t);
  };
  like(dn, c.lead, "dn must be like n");
  like(dh, x ? *x : c.lead, "dh must be like h");
  auto kept = [&](const optional<Tensor>& t, const optional<Tensor>& weight, int64_t n) {
    if (!weight) return;
    need(t && t->numel() == n && t->scalar_type() == at::kFloat && t->is_contiguous(), "rstd must be the forward pass's");
    same_device(c.lead, *t);
  };
  kept(rstd_post, pw, c.d.rows * groups);
  kept(rstd, w, c.d.rows);
  const auto pdh = packed(dh), pdn = packed(dn);
  optional<Tensor> g[5];
  const optional<Tensor>* from[5] = {&x, &y, &gate, &pw, &w};
  for (int i = 0; i < 5; i++)
    if (*from[i]) g[i] = packed_like(**from[i]);
  if (!c.d.rows) {   // empty buffers have no address to pass
    if (c.d.gate == SFFFT_GATE_CHANNEL) g[2]->zero_();
    for (int i = 3; i < 5; i++)
      if (g[i]) g[i]->zero_();
  } else {
    size_t bytes = 0;
    status(sffft_block_norm_workspace_bytes(&c.d, &bytes), "block_norm_backward");
    const Tensor work = workspace(bytes, c.lead);
    status(sffft_block_norm_backward(&c.d, ptr(c.x), ptr(c.y), ptr(c.gate), ptr(c.pw), ptr(c.w), (const float*)ptr(rstd_post),
                                     (const float*)ptr(rstd), ptr(pdh), ptr(pdn), out_ptr(g[0]), out_ptr(g[1]), out_ptr(g[2]),
                                     out_ptr(g[3]), out_ptr(g[4]), bytes ? work.mutable_data_ptr() : nullptr, bytes,
                                     stream_of(c.lead)),
           "block_norm_backward");
  }
  std::vector<Tensor> out;
  for (auto& t : g)
    if (t) out.push_back(*t);
  return out;
}

// ---------------------------------------------------------------------------------------------------------------
// gradients
// ---------------------------------------------------------------------------------------------------------------
template <class F>
auto op(const char* name) {
  return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<F>();
}

bool wants(std::initializer_list<const optional<Tensor>*> ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const auto* t : ts)
    if (*t && (*t)->requires_grad()) return true;
  return false;
}

// A tensor of forward-mode differentiation need not require a gradient, and would pass the autograd functions by: the result
// would have no tangent, which counts as a zero one.
template <class... T>
void need_no_tangent(const char* what, const T&... ts) {
  auto has = [](const auto& t) {
    if constexpr (std::is_same_v<std::decay_t<decltype(t)>, Tensor>) return t._fw_grad(0).defined();
    else return t && t->_fw_grad(0).defined();
  };
  need(!(has(ts) || ...), what, " has no forward-mode derivative");
}

Tensor or_none(const optional<Tensor>& t) { return t ? *t : Tensor(); }
optional<Tensor> opt(const Tensor& t) { return t.defined() ? optional<Tensor>(t) : optional<Tensor>(); }

decltype(auto) attention_op() {
  static const auto f = op<decltype(attention)>("sffft::linear_attention");
  return (f);
}
decltype(auto) attention_backward_op() {
  static const auto f = op<decltype(attention_backward)>("sffft::linear_attention_backward");
  return (f);
}
decltype(auto) step_op() {
  static const auto f = op<decltype(attention_step)>("sffft::linear_attention_step");
  return (f);
}
decltype(auto) norm_op() {
  static const auto f = op<decltype(norm)>("sffft::block_norm");
  return (f);
}
decltype(auto) norm_backward_op() {
  static const auto f = op<decltype(norm_backward)>("sffft::block_norm_backward");
  return (f);
}

struct Attention : torch::autograd::Function<Attention> {
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& log_decay,
                               const optional<Tensor>& s0, const optional<Tensor>& lengths, double scale) {
    at::AutoDispatchBelowADInplaceOrView guard;
    ctx->save_for_backward({q, k, v, log_decay, or_none(s0), or_none(lengths)});
    ctx->saved_data["scale"] = scale;
    ctx->set_materialize_grads(false);
    auto [y, s1] = attention_op().call(q, k, v, log_decay, s0, lengths, scale);
    return {y, s1};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto t = ctx->get_saved_variables();
    Tensor dy = grads[0];
    if (!dy.defined()) dy = at::zeros_symint({t[0].sym_size(0), t[0].sym_size(1), t[0].sym_size(2), t[2].sym_size(3)}, t[0].options());
    const auto g = attention_backward_op().call(t[0], t[1], t[2], t[3], opt(t[4]), opt(t[5]), ctx->saved_data["scale"].toDouble(), dy,
                                                opt(grads[1]));
    return {g[0], g[1], g[2], Tensor(), t[4].defined() ? g[3] : Tensor(), Tensor(), Tensor()};
  }
};

std::tuple<Tensor, Tensor> attention_grad(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& log_decay,
                                          const optional<Tensor>& s0, const optional<Tensor>& lengths, double scale) {
  need(!at::GradMode::is_enabled() || !log_decay.requires_grad(),
       "log_decay is a constant: it has no gradient (pass log_decay.detach())");
  need_no_tangent("linear_attention", q, k, v, log_decay, s0);
  if (wants({&s0}) || (at::GradMode::is_enabled() && (q.requires_grad() || k.requires_grad() || v.requires_grad()))) {
    auto out = Attention::apply(q, k, v, log_decay, s0, lengths, scale);
    return {out[0], out[1]};
  }
  at::AutoDispatchBelowADInplaceOrView guard;
  return attention_op().call(q, k, v, log_decay, s0, lengths, scale);
}

Tensor step_grad(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& log_decay, Tensor& state,
                 const optional<Tensor>& slots, double scale) {
  need(!at::GradMode::is_enabled() || !(q.requires_grad() || k.requires_grad() || v.requires_grad() ||
                                                     log_decay.requires_grad() || state.requires_grad()),
                    "linear_attention_step updates its state in place and has no gradient: use linear_attention, or no_grad");
  need_no_tangent("linear_attention_step", q, k, v, log_decay, state);
  {
    at::AutoDispatchBelowADInplaceOrView guard;
    Tensor y = step_op().call(q, k, v, log_decay, state, slots, scale);
    if (!state.is_inference()) state.unsafeGetTensorImpl()->bump_version();   // changed in place
    return y;
  }
}

struct Norm : torch::autograd::Function<Norm> {
  static variable_list forward(AutogradContext* ctx, const optional<Tensor>& x, const optional<Tensor>& y, const optional<Tensor>& gate,
                               const optional<Tensor>& pw, const optional<Tensor>& w, double scale, double eps, int64_t groups,
                               std::string act, int64_t dim) {
    at::AutoDispatchBelowADInplaceOrView guard;
    auto out = norm_op().call(x, y, gate, pw, w, scale, eps, groups, act, dim, true);
    Tensor r2, r1;
    if (w) r2 = out.back(), out.pop_back();
    if (pw) r1 = out.back(), out.pop_back();
    ctx->save_for_backward({or_none(x), or_none(y), or_none(gate), or_none(pw), or_none(w), r1, r2});
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["groups"] = groups;
    ctx->saved_data["act"] = act;
    ctx->saved_data["dim"] = dim;
    ctx->set_materialize_grads(false);
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto t = ctx->get_saved_variables();
    const bool has_y = t[1].defined(), has_w = t[4].defined();
    Tensor dh = has_y ? grads[0] : Tensor(), dn = has_w ? grads[has_y ? 1 : 0] : Tensor();
    const Tensor& lead = has_y ? t[1] : t[0];
    if (has_w && !dn.defined()) dn = at::zeros_like(lead);
    if (!has_w && !dh.defined()) dh = at::zeros_like(t[0].defined() ? t[0] : lead);
    auto g = norm_backward_op().call(opt(dh), opt(dn), opt(t[0]), opt(t[1]), opt(t[2]), opt(t[3]), opt(t[4]), opt(t[5]), opt(t[6]),
                                     ctx->saved_data["scale"].toDouble(), ctx->saved_data["eps"].toDouble(),
                                     ctx->saved_data["groups"].toInt(), ctx->saved_data["act"].toStringRef(),
                                     ctx->saved_data["dim"].toInt());
    variable_list out(10);
    for (int i = 0, j = 0; i < 5; i++)
      if (t[i].defined()) out[i] = g[j++];
    return out;
  }
};

std::vector<Tensor> norm_grad(const optional<Tensor>& x, const optional<Tensor>& y, const optional<Tensor>& gate,
                              const optional<Tensor>& pw, const optional<Tensor>& w, double scale, double eps, int64_t groups,
                              c10::string_view act, int64_t dim, bool stats) {
  need_no_tangent("block_norm", x, y, gate, pw, w);
  if (wants({&x, &y, &gate, &pw, &w})) {
    need(!stats, "stats are for calls without a gradient");
    return Norm::apply(x, y, gate, pw, w, scale, eps, groups, std::string(act), dim);
  }
  at::AutoDispatchBelowADInplaceOrView guard;
  return norm_op().call(x, y, gate, pw, w, scale, eps, groups, act, dim, stats);
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(sffft, m) {
  m.def("linear_attention(Tensor q, Tensor k, Tensor v, Tensor log_decay, Tensor? initial_state, Tensor? lengths, float scale) "
        "-> (Tensor, Tensor)", {at::Tag::pt2_compliant_tag});
  m.def("linear_attention_backward(Tensor q, Tensor k, Tensor v, Tensor log_decay, Tensor? initial_state, Tensor? lengths, "
        "float scale, Tensor dy, Tensor? dfinal_state) -> Tensor[]", {at::Tag::pt2_compliant_tag});
  m.def("linear_attention_step(Tensor q, Tensor k, Tensor v, Tensor log_decay, Tensor(a!) state, Tensor? slots, float scale) "
        "-> Tensor", {at::Tag::pt2_compliant_tag});
  m.def("block_norm(Tensor? x, Tensor? y, Tensor? gate, Tensor? post_weight, Tensor? weight, float scale, float eps, int groups, "
        "str act, int dim, bool stats=False) -> Tensor[]", {at::Tag::pt2_compliant_tag});
  m.def("block_norm_backward(Tensor? dh, Tensor? dn, Tensor? x, Tensor? y, Tensor? gate, Tensor? post_weight, Tensor? weight, "
        "Tensor? rstd_post, Tensor? rstd, float scale, float eps, int groups, str act, int dim) -> Tensor[]",
        {at::Tag::pt2_compliant_tag});
}

// CPU tensors come this way too, to be refused with the other checks.
#define SFFFT_IMPL(key)                                       \
  TORCH_LIBRARY_IMPL(sffft, key, m) {                         \
    m.impl("linear_attention", &attention);                   \
    m.impl("linear_attention_backward", &attention_backward); \
    m.impl("linear_attention_step", &attention_step);         \
    m.impl("block_norm", &norm);                              \
    m.impl("block_norm_backward", &norm_backward);            \
  }
SFFFT_IMPL(CUDA)
SFFFT_IMPL(CPU)

TORCH_LIBRARY_IMPL(sffft, Autograd, m) {
  m.impl("linear_attention", &attention_grad);
  m.impl("linear_attention_step", &step_grad);
  m.impl("block_norm", &norm_grad);
  m.impl("linear_attention_backward", torch::autograd::autogradNotImplementedFallback());   // first derivatives only
  m.impl("block_norm_backward", torch::autograd::autogradNotImplementedFallback());
}
