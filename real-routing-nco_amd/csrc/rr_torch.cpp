// The torch side of the decoder operators (rr_xattn.hip, rr_norm.hip, rr_draw.hip): argument checks, outputs, workspaces, autograd nodes.
// A Python autograd.Function around the C entry points took 120 - 140 us for a forward and a backward of a small batch (and 11 - 13 us for a
// forward alone), most of it interpreter time on two threads; the kernels of such a call take a tenth of that.
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/extension.h>

#include <cmath>
#include <limits>

#include "../../include/rrnco_hip.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
typedef std::optional<Tensor> MaybeTensor;

int type_code(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return 0;
    case at::kHalf: return 1;
    case at::kBFloat16: return 2;
    default: return -1;
  }
}
std::string shape_of(const Tensor& t) {
  std::string s = "(";
  for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.size(i));
  return s + ")";
}
void need_gpu(const Tensor& t) {
  TORCH_CHECK(t.is_cuda(), "rrnco_amd: the MI355X hot path needs tensors on a ROCm device (no CPU fallback)");
}
// launches go to the device that holds the tensors and to its current stream
struct OnDevice {
  c10::DeviceIndex back = -1;
  hipStream_t stream;
  explicit OnDevice(const Tensor& t) {
    const c10::DeviceIndex dev = t.get_device(), cur = c10::hip::current_device();
    if (dev != cur) {
      c10::hip::set_device(dev);
      back = cur;
    }
    stream = c10::hip::getCurrentHIPStream(dev).stream();
  }
  ~OnDevice() {
    if (back >= 0) c10::hip::set_device(back);
  }
};
void done(int rc, const char* what) {
  TORCH_CHECK(rc == 0, "rrnco_amd: ", what, " failed with status ", rc, " (-1 invalid argument, -2 HIP launch error)");
}
void* ptr(const Tensor& t) { return t.data_ptr(); }
void* ptr(const MaybeTensor& t) { return t.has_value() ? t->data_ptr() : nullptr; }
bool tracked(const Tensor& t) { return t.requires_grad(); }
bool tracked(const MaybeTensor& t) { return t.has_value() && t->requires_grad(); }
// a forward-mode tangent (a dual tensor may have one without requires_grad) would be dropped without a word
bool dual(const Tensor& t) { return t.defined() && t._fw_grad(0).defined(); }
bool dual(const MaybeTensor& t) { return t.has_value() && dual(*t); }
template <typename... Ts>
void no_tangents(const char* what, const Ts&... ts) {
  TORCH_CHECK_NOT_IMPLEMENTED(!(dual(ts) || ...), what, ": no forward-mode derivatives");
}
Tensor some(const MaybeTensor& t) { return t.has_value() ? *t : Tensor(); }
MaybeTensor maybe(const Tensor& t) { return t.defined() ? MaybeTensor(t) : MaybeTensor(); }

// gradients that cannot be differentiated again: an error node behind them where a graph of the backward is asked for
variable_list once(variable_list grads) {
  if (!at::GradMode::is_enabled()) return grads;
  variable_list real;
  for (auto& g : grads)
    if (g.defined()) real.push_back(g.detach().requires_grad_());
  auto err = std::make_shared<torch::autograd::DelayedError>("trying to differentiate twice a function whose gradient is computed by a kernel", (int64_t)real.size());
  auto out = (*err)(std::move(real));
  size_t i = 0;
  for (auto& g : grads)
    if (g.defined()) g = out[i++];
  return grads;
}

// ------------------------------------------------------------------------------------------------ cross attention
// the kernels read 16 bytes of a head at a time: a unit last stride, the base and every other stride (that is used) on 16 bytes; anything else is copied
Tensor placed(const Tensor& t) {
  const int64_t per = 16 / (int64_t)t.element_size();
  bool ok = t.stride(3) == 1 && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
  for (int i = 0; i < 3 && ok; ++i) ok = t.size(i) == 1 || t.stride(i) % per == 0;
  return ok ? t : t.clone(at::MemoryFormat::Contiguous);
}
void strides(const Tensor& t, long long (&s)[3]) {
  for (int i = 0; i < 3; ++i) s[i] = t.size(i) == 1 ? 0 : t.stride(i);
}

double attention_checked(const Tensor& q, const Tensor& k, const Tensor& v, const MaybeTensor& mask, const MaybeTensor& lens, std::optional<double> scale) {
  TORCH_CHECK_TYPE(type_code(q) >= 0 && k.scalar_type() == q.scalar_type() && v.scalar_type() == q.scalar_type(),
                   "cross_attention: query, key and value of one type out of float32, float16, bfloat16, got ", q.scalar_type(), ", ", k.scalar_type(), ", ", v.scalar_type());
  TORCH_CHECK_VALUE(q.dim() == 4 && k.dim() == 4 && k.sizes() == v.sizes() && k.size(0) == q.size(0) && k.size(3) == q.size(3),
                    "cross_attention: query [B, Lq, H, D], key and value [B, Lk, Hk, D], got ", shape_of(q), ", ", shape_of(k), ", ", shape_of(v));
  const int64_t B = q.size(0), Lq = q.size(1), H = q.size(2), D = q.size(3), Lk = k.size(1), Hk = k.size(2);
  TORCH_CHECK_VALUE(D % 8 == 0 && D >= 8 && D <= 128, "cross_attention: a head dim that is a multiple of 8 up to 128, got ", D);
  TORCH_CHECK_VALUE(Hk >= 1 && H >= 1 && H % Hk == 0, "cross_attention: the query's heads are a multiple of the key's, got ", H, " and ", Hk);
  TORCH_CHECK_VALUE(k.device() == q.device() && v.device() == q.device(), "cross_attention: query, key and value are on one device");
  if (mask.has_value()) {
    TORCH_CHECK_VALUE(mask->scalar_type() == at::kBool && mask->dim() == 4 && mask->device() == q.device(),
                      "cross_attention: mask is a bool tensor of four axes (batch, head, query, key) on the query's device, True where a key may be seen");
    const int64_t full[4] = {B, H, Lq, Lk};
    for (int i = 0; i < 4; ++i)
      TORCH_CHECK_VALUE(mask->size(i) == 1 || mask->size(i) == full[i], "cross_attention: mask ", shape_of(*mask), " does not broadcast to (", B, ", ", H, ", ", Lq, ", ", Lk, ")");
  }
  if (lens.has_value())
    TORCH_CHECK_VALUE((lens->scalar_type() == at::kInt || lens->scalar_type() == at::kLong) && lens->dim() == 1 && lens->size(0) == B && lens->device() == q.device(),
                      "cross_attention: kv_lens is [B], int32 or int64, on the query's device");
  const double s = scale.has_value() ? *scale : 1.0 / std::sqrt((double)D);
  TORCH_CHECK_VALUE(s >= 1e-37 && s < 3e38, "cross_attention: scale > 0, got ", s);
  const int64_t lim = std::numeric_limits<int32_t>::max();
  TORCH_CHECK_VALUE(B <= lim && Lq <= lim && Lk <= lim && H <= lim, "cross_attention: more rows, keys or heads than 32-bit counts hold");
  need_gpu(q);
  return s;
}

void attention_call(const Tensor& q_, const Tensor& k_, const Tensor& v_, const MaybeTensor& mask_, const MaybeTensor& lens_, double scale, const Tensor& out, const Tensor& lse,
                    const Tensor& dout_, const Tensor& dq, const Tensor& dk, const Tensor& dv) {
  const bool back = dout_.defined();
  const Tensor q = placed(q_), k = placed(k_), v = placed(v_);
  Tensor mask, lens, dout, delta, ws;
  XAttnIO io = {};
  io.q = ptr(q);
  io.k = ptr(k);
  io.v = ptr(v);
  io.out = ptr(out);
  io.lse = lse.defined() ? (float*)ptr(lse) : nullptr;
  strides(q, io.q_stride);
  strides(k, io.k_stride);
  strides(v, io.v_stride);
  io.dtype = type_code(q);
  io.B = (int)q.size(0);
  io.Lq = (int)q.size(1);
  io.Lk = (int)k.size(1);
  io.Hk = (int)k.size(2);
  io.G = (int)(q.size(2) / k.size(2));
  io.D = (int)q.size(3);
  io.scale = (float)scale;
  if (mask_.has_value()) {
    mask = *mask_;
    if (mask.size(3) != io.Lk || (io.Lk > 1 && mask.stride(3) != 1)) mask = mask.expand({mask.size(0), mask.size(1), mask.size(2), io.Lk}).contiguous();
    io.mask = (const uint8_t*)ptr(mask);
    strides(mask, io.mask_stride);
  }
  if (lens_.has_value()) {
    lens = lens_->contiguous();
    io.kv_lens = ptr(lens);
    io.lens_int64 = lens.scalar_type() == at::kLong;
  }
  if (back) {
    dout = placed(dout_);
    delta = at::empty_like(lse);
    io.dout = ptr(dout);
    strides(dout, io.dout_stride);
    io.delta = (float*)ptr(delta);
    io.dq = ptr(dq);
    io.dk = ptr(dk);
    io.dv = ptr(dv);
  }
  const long long n = rr_cross_attn_workspace(io.dtype, io.B, io.Lq, io.Lk, io.Hk, io.G, io.D, back);
  TORCH_CHECK_VALUE(n >= 0, "cross_attention: more than 2^31 - 1 queries of all heads, or an instance of more than 2^29 queries or keys of its key heads");
  if (n > 0) {
    ws = at::empty({(int64_t)n}, q.options().dtype(at::kByte));
    io.workspace = ptr(ws);
    io.workspace_bytes = n;
  }
  const OnDevice on(q);
  if (back) done(rr_cross_attn_bwd(&io, on.stream), "rr_cross_attn_bwd");
  else done(rr_cross_attn(&io, on.stream), "rr_cross_attn");
}

std::pair<Tensor, Tensor> attention_forward(const Tensor& q, const Tensor& k, const Tensor& v, const MaybeTensor& mask, const MaybeTensor& lens, double scale, bool want_lse) {
  Tensor out = at::empty(q.sizes(), q.options()), lse;
  if (want_lse) lse = at::empty({q.size(0), q.size(2), q.size(1)}, q.options().dtype(at::kFloat));
  if (q.numel() == 0) return {out, lse};
  if (k.numel() == 0) {                                 // nothing to see
    out.zero_();
    if (want_lse) lse.fill_(-std::numeric_limits<double>::infinity());
    return {out, lse};
  }
  attention_call(q, k, v, mask, lens, scale, out, lse, Tensor(), Tensor(), Tensor(), Tensor());
  return {out, lse};
}

struct CrossAttention : torch::autograd::Function<CrossAttention> {
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v, const MaybeTensor& mask, const MaybeTensor& lens, double scale) {
    auto [out, lse] = attention_forward(q, k, v, mask, lens, scale, true);
    ctx->save_for_backward({q, k, v, some(mask), some(lens), out, lse});
    ctx->saved_data["scale"] = scale;
    ctx->mark_non_differentiable({lse});
    ctx->set_materialize_grads(false);
    return {out, lse};
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    const auto s = ctx->get_saved_variables();
    variable_list out(6);
    if (!g[0].defined()) return out;
    no_tangents("cross_attention", g[0]);
    const Tensor &q = s[0], &k = s[1], &v = s[2];
    const bool create = at::GradMode::is_enabled();
    {
      at::NoGradGuard guard;
      Tensor grads[3];
      for (int i = 0; i < 3; ++i) grads[i] = at::empty(s[i].sizes(), s[i].options());
      if (q.numel() == 0 || k.numel() == 0) {
        for (auto& t : grads) t.zero_();
      } else {
        attention_call(q, k, v, maybe(s[3]), maybe(s[4]), ctx->saved_data["scale"].toDouble(), s[5], s[6], g[0], grads[0], grads[1], grads[2]);
      }
      for (int i = 0; i < 3; ++i)
        if (ctx->needs_input_grad(i)) out[i] = grads[i];
    }
    return create ? once(std::move(out)) : out;
  }
};

std::tuple<Tensor, MaybeTensor> cross_attention(const Tensor& q, const Tensor& k, const Tensor& v, const MaybeTensor& mask, const MaybeTensor& lens, std::optional<double> scale,
                                                bool want_lse) {
  no_tangents("cross_attention", q, k, v);
  const double s = attention_checked(q, k, v, mask, lens, scale);
  if (at::GradMode::is_enabled() && (tracked(q) || tracked(k) || tracked(v))) {
    auto out = CrossAttention::apply(q, k, v, mask, lens, s);
    return {out[0], maybe(out[1])};
  }
  auto [out, lse] = attention_forward(q, k, v, mask, lens, s, want_lse);
  return {out, maybe(lse)};
}

// ------------------------------------------------------------------------------------------------ residual + RMS norm
// [..., E] as rows of unit column stride; a view where the strides allow it
Tensor rows_of(const Tensor& t, int64_t E) {
  Tensor x = t.dim() == 2 ? t : t.reshape({-1, E});
  return x.stride(1) == 1 || E == 1 ? x : x.contiguous();
}
long long pitch(const Tensor& t) { return t.size(0) > 1 ? t.stride(0) : 0; }

void norm_checked(const Tensor& x, const MaybeTensor& r, const MaybeTensor& w, double eps) {
  TORCH_CHECK_TYPE(type_code(x) >= 0, "add_rms_norm: float32, float16 or bfloat16, got ", x.scalar_type());
  TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) >= 1 && x.size(-1) <= 16384, "add_rms_norm: a last axis of 1 .. 16384, got shape ", shape_of(x));
  if (r.has_value())
    TORCH_CHECK_VALUE(r->sizes() == x.sizes() && r->scalar_type() == x.scalar_type() && r->device() == x.device(), "add_rms_norm: the residual has the input's shape, type and device");
  if (w.has_value())
    TORCH_CHECK_VALUE(w->dim() == 1 && w->size(0) == x.size(-1) && (w->scalar_type() == x.scalar_type() || w->scalar_type() == at::kFloat) && w->device() == x.device(),
                      "add_rms_norm: the weight is [width], of the input's type or float32, on its device");
  TORCH_CHECK_VALUE(eps >= 0.0 && eps < 1e30, "add_rms_norm: eps >= 0, got ", eps);
  TORCH_CHECK_VALUE(x.numel() / x.size(-1) <= std::numeric_limits<int32_t>::max(), "add_rms_norm: at most 2^31 - 1 rows");
  need_gpu(x);
}

struct NormOut { Tensor y, h, rstd, q, scale; };
NormOut norm_forward(const Tensor& x, const MaybeTensor& r, const MaybeTensor& w, double eps, bool want_rstd, bool eight) {
  const int64_t E = x.size(-1);
  const Tensor x2 = rows_of(x, E), r2 = r.has_value() ? rows_of(*r, E) : Tensor(), wc = w.has_value() ? w->contiguous() : Tensor();
  const int64_t rows = x2.size(0);
  NormOut o;
  if (r.has_value()) o.h = at::empty(x.sizes(), x.options());
  if (want_rstd) o.rstd = at::empty({rows}, x.options().dtype(at::kFloat));
  if (eight) {
    o.q = at::empty(x.sizes(), x.options().dtype(at::kFloat8_e4m3fn));
    auto s = x.sizes().vec();
    s.back() = (E + 127) / 128;
    o.scale = at::empty(s, x.options().dtype(at::kFloat));
  } else {
    o.y = at::empty(x.sizes(), x.options());
  }
  if (rows > 0) {
    auto opt = [](const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; };
    const OnDevice on(x);
    done(rr_add_rms_norm(type_code(x), ptr(x2), pitch(x2), opt(r2), r2.defined() ? pitch(r2) : 0, opt(wc), wc.defined() && wc.scalar_type() == at::kFloat, opt(o.y), opt(o.h),
                         (float*)opt(o.rstd), (uint8_t*)opt(o.q), (float*)opt(o.scale), rows, (int)E, (float)eps, on.stream),
         "rr_add_rms_norm");
  }
  return o;
}

struct AddRMSNorm : torch::autograd::Function<AddRMSNorm> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const MaybeTensor& r, const MaybeTensor& w, double eps) {
    NormOut o = norm_forward(x, r, w, eps, true, false);
    ctx->save_for_backward({x, some(r), some(w), o.rstd});
    ctx->set_materialize_grads(false);
    if (o.h.defined()) return {o.y, o.h};
    return {o.y};
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    const auto s = ctx->get_saved_variables();
    const Tensor &x = s[0], &r = s[1], &w = s[2], &rstd = s[3];
    const bool create = at::GradMode::is_enabled(), nx = ctx->needs_input_grad(0), nr = r.defined() && ctx->needs_input_grad(1),
               nw = w.defined() && ctx->needs_input_grad(r.defined() ? 2 : 1);      // (an input that was not given has no place in the count)
    variable_list out(4);
    const Tensor dy = g[0], dh = g.size() > 1 ? g[1] : Tensor();
    if (!dy.defined()) {                                // only the sum was used, or nothing
      if (dh.defined() && nx) out[0] = dh;
      if (dh.defined() && nr) out[1] = dh;
      return out;
    }
    no_tangents("add_rms_norm", dy, dh);
    {
      at::NoGradGuard guard;
      const int64_t E = x.size(-1), rows = rstd.size(0);
      const Tensor dx = at::empty(x.sizes(), x.options());
      Tensor dw, ws;
      if (nw) dw = rows ? at::empty(w.sizes(), w.options()) : at::zeros(w.sizes(), w.options());
      if (rows > 0) {
        const Tensor x2 = rows_of(x, E), r2 = r.defined() ? rows_of(r, E) : Tensor(), wc = w.defined() ? w.contiguous() : Tensor(), dy2 = rows_of(dy, E),
                     dh2 = dh.defined() ? rows_of(dh, E) : Tensor();
        const int parts = rr_add_rms_norm_parts(rows, (int)E);
        if (nw) ws = at::empty({parts * E}, x.options().dtype(at::kFloat));
        auto opt = [](const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; };
        const OnDevice on(x);
        done(rr_add_rms_norm_bwd(type_code(x), ptr(x2), pitch(x2), opt(r2), r2.defined() ? pitch(r2) : 0, opt(wc), wc.defined() && wc.scalar_type() == at::kFloat, ptr(dy2), pitch(dy2),
                                 opt(dh2), dh2.defined() ? pitch(dh2) : 0, (const float*)ptr(rstd), ptr(dx), opt(dw), (float*)opt(ws), parts, rows, (int)E, on.stream),
             "rr_add_rms_norm_bwd");
      }
      if (nx) out[0] = dx;
      if (nr) out[1] = dx;
      if (nw) out[2] = dw;
    }
    return create ? once(std::move(out)) : out;
  }
};

std::tuple<Tensor, Tensor> add_rms_norm(const Tensor& x, const MaybeTensor& r, const MaybeTensor& w, double eps) {
  no_tangents("add_rms_norm", x, r, w);
  norm_checked(x, r, w, eps);
  if (at::GradMode::is_enabled() && (tracked(x) || tracked(r) || tracked(w))) {
    auto o = AddRMSNorm::apply(x, r, w, eps);
    return {o[0], o.size() > 1 ? o[1] : x};
  }
  NormOut o = norm_forward(x, r, w, eps, false, false);
  return {o.y, o.h.defined() ? o.h : x};
}

std::tuple<Tensor, Tensor, Tensor> add_rms_norm_fp8(const Tensor& x, const MaybeTensor& r, const MaybeTensor& w, double eps) {
  no_tangents("add_rms_norm_fp8", x, r, w);
  norm_checked(x, r, w, eps);
  TORCH_CHECK(!(at::GradMode::is_enabled() && (tracked(x) || tracked(r) || tracked(w))), "add_rms_norm_fp8 has no gradient: call it under torch.no_grad()");
  NormOut o = norm_forward(x, r, w, eps, false, true);
  return {o.q, o.scale, o.h.defined() ? o.h : x};
}

// ------------------------------------------------------------------------------------------------ sampling
// a number for all rows, or a tensor with one for each in the kernel's type
struct Setting {
  double all = 0.0;
  Tensor row;
  void* ptr() const { return row.defined() ? row.data_ptr() : nullptr; }
};
Setting setting(const char* name, const py::object& v, int64_t R, const at::Device& dev, double low, double high, at::ScalarType type) {
  Setting s;
  if (THPVariable_Check(v.ptr())) {
    const Tensor& t = THPVariable_Unpack(v.ptr());
    no_tangents("sample", t);
    TORCH_CHECK_VALUE(t.numel() == R && t.device() == dev && !t.is_complex() && t.scalar_type() != at::kBool, "sample: ", name,
                      " is a number or a tensor of one number for each of the ", R, " rows on the logits' device");
    s.row = t.detach().reshape({R});
    if (type == at::kInt && s.row.scalar_type() == at::kLong) s.row = s.row.clamp(-1, 1 << 30);      // (a wide count narrowed would wrap)
    s.row = s.row.to(type).contiguous();
  } else {
    TORCH_CHECK_TYPE(PyFloat_Check(v.ptr()) || PyLong_Check(v.ptr()) || PyIndex_Check(v.ptr()), "sample: ", name, " is a number or a tensor");
    s.all = v.cast<double>();
    TORCH_CHECK_VALUE(s.all >= low && s.all <= high, "sample: ", name, " in ", low, " .. ", high, ", got ", s.all);
    TORCH_CHECK_VALUE(type != at::kInt || s.all == std::floor(s.all), "sample: ", name, " is a whole number, got ", s.all);
  }
  return s;
}

std::tuple<Tensor, Tensor> sample(const Tensor& logits, const Tensor& uniforms, const py::object& temperature, const py::object& top_k, const py::object& top_p, const py::object& min_p,
                                  const MaybeTensor& mask_) {
  no_tangents("sample", logits);
  TORCH_CHECK_TYPE(type_code(logits) >= 0, "sample: logits float32, float16 or bfloat16, got ", logits.scalar_type());
  TORCH_CHECK_VALUE(logits.dim() >= 1 && logits.size(-1) >= 1 && logits.size(-1) <= (1 << 24), "sample: logits [..., V] with V in 1 .. ", 1 << 24, ", got shape ", shape_of(logits));
  const int64_t V = logits.size(-1), R = logits.numel() / V;
  const auto lead = logits.sizes().slice(0, logits.dim() - 1);
  const at::Device dev = logits.device();
  TORCH_CHECK_VALUE(uniforms.sizes() == lead && uniforms.scalar_type() == at::kFloat && uniforms.device() == dev,
                    "sample: uniforms float32 of the logits' shape without the last axis, on their device, got ", uniforms.scalar_type(), " ", shape_of(uniforms));
  if (mask_.has_value()) {
    TORCH_CHECK_VALUE(mask_->scalar_type() == at::kBool && mask_->device() == dev, "sample: mask is a bool tensor on the logits' device, True where a key may be drawn");
    bool ok = mask_->dim() <= logits.dim();
    for (int64_t i = 1; ok && i <= mask_->dim(); ++i) ok = mask_->size(-i) == 1 || mask_->size(-i) == logits.size(-i);
    TORCH_CHECK_VALUE(ok, "sample: mask ", shape_of(*mask_), " does not broadcast to the logits' ", shape_of(logits));
  }
  TORCH_CHECK_VALUE(R <= std::numeric_limits<int32_t>::max(), "sample: at most 2^31 - 1 rows");
  const Setting t = setting("temperature", temperature, R, dev, 0.0, 1e29, at::kFloat), k = setting("top_k", top_k, R, dev, 0.0, 1e15, at::kInt),
                p = setting("top_p", top_p, R, dev, 0.0, 1.0, at::kFloat), mp = setting("min_p", min_p, R, dev, 0.0, 1.0, at::kFloat);
  need_gpu(logits);
  at::NoGradGuard guard;
  const Tensor x = rows_of(logits, V), u = uniforms.contiguous();
  Tensor mask, ws;
  if (mask_.has_value()) {
    mask = mask_->sizes() == x.sizes() ? *mask_ : mask_->expand(logits.sizes()).reshape({-1, V});
    if (V > 1 && mask.stride(1) != 1) mask = mask.contiguous();
  }
  const Tensor index = at::empty(lead, logits.options().dtype(at::kLong)), logp = at::empty(lead, logits.options().dtype(at::kFloat));
  if (R > 0) {
    const long long n = rr_draw_workspace((int)R, (int)V);
    if (n > 0) ws = at::empty({(int64_t)n}, logits.options().dtype(at::kByte));
    const OnDevice on(logits);
    done(rr_draw(type_code(x), ptr(x), pitch(x), mask.defined() ? (const uint8_t*)ptr(mask) : nullptr, mask.defined() ? pitch(mask) : 0, (const float*)ptr(u), (int64_t*)ptr(index),
                 (float*)ptr(logp), (int)R, (int)V, t.all, (int)std::min<double>(k.all, (double)V), p.all, mp.all, (const float*)t.ptr(), (const int*)k.ptr(), (const float*)p.ptr(),
                 (const float*)mp.ptr(), ws.defined() ? ptr(ws) : nullptr, n, on.stream),
         "rr_draw");
  }
  return {index, logp};
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("cross_attention", &cross_attention);
  m.def("add_rms_norm", &add_rms_norm);
  m.def("add_rms_norm_fp8", &add_rms_norm_fp8);
  m.def("sample", &sample);
}
