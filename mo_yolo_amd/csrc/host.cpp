// The host side of the transformer-layer operators (layer norm, linear, attention): layouts, outputs, workspaces and autograd nodes, in C++ because a training
// step calls them from autograd's own thread, where each Python operation costs several times its usual price (forward and gradient of a small layer
// norm: 118 us through Python functions, 67 us here, of which autograd itself takes 51).  Arguments have been checked by mo_yolo_amd.ops; the entry points of
// the C ABI (include/moyolo.h) are handed over as addresses, so that whichever build of the library is loaded is the one that is called.
#include <c10/core/AutogradState.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/extension.h>

#include "../../include/moyolo.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using MaybeTensor = std::optional<Tensor>;

struct Entries {
  decltype(&moy_strerror) strerror_ = nullptr;
  decltype(&moy_layer_norm) norm = nullptr;
  decltype(&moy_layer_norm_bwd) norm_bwd = nullptr;
  decltype(&moy_layer_norm_bwd_ws) norm_bwd_ws = nullptr;
  decltype(&moy_linear) linear = nullptr;
  decltype(&moy_linear_ws) linear_ws = nullptr;
  decltype(&moy_linear_bwd) linear_bwd = nullptr;
  decltype(&moy_linear_bwd_ws) linear_bwd_ws = nullptr;
  decltype(&moy_attention) attention = nullptr;
  decltype(&moy_attention_ws) attention_ws = nullptr;
  decltype(&moy_attention_bwd) attention_bwd = nullptr;
  decltype(&moy_attention_bwd_ws) attention_bwd_ws = nullptr;
} lib;

struct MoyError : std::runtime_error {
  using std::runtime_error::runtime_error;
};

int64_t check(int64_t rc, const char* what) {
  if (rc < 0) throw MoyError(std::string(what) + " failed: " + lib.strerror_((int)rc) + " (code " + std::to_string(rc) + ")");
  return rc;
}

int code_of(at::ScalarType t) { return t == at::kFloat ? MOY_F32 : t == at::kBFloat16 ? MOY_BF16 : MOY_F16; }

// What records torch's operations (torch.jit.trace, make_fx) sees the outputs made and not the launches that fill them: a replay would return memory that nothing wrote.
bool not_recorded() {
  TORCH_CHECK(!torch::jit::tracer::isTracing() && !c10::impl::TorchDispatchModeTLS::get_mode(c10::impl::TorchDispatchModeKey::PROXY).has_value() &&
                  !c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::PreDispatch),
              "the transformer-layer operators launch kernels of their own and cannot be recorded by torch.jit.trace or make_fx");
  return true;
}

// the tensor's device as the current one, and its current stream
struct On {
  bool live = not_recorded();
  at::AutoGradMode plain{false};           // (layout copies are no part of a graph)
  c10::OptionalDeviceGuard guard;
  void* stream;
  explicit On(const Tensor& x) : guard(x.device()), stream(c10::hip::getCurrentHIPStream(x.device().index()).stream()) {}
};

void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
Tensor tensor_of(const MaybeTensor& t) { return t.has_value() ? *t : Tensor(); }
Tensor made(bool wanted, at::IntArrayRef shape, const Tensor& like, at::ScalarType type) {
  return wanted ? at::empty(shape, like.options().dtype(type)) : Tensor();
}
Tensor floats(int64_t n, const Tensor& like) { return n ? at::empty({n}, like.options().dtype(at::kFloat)) : Tensor(); }

// [..., C] -> a 2-D view [rows, C] with unit column stride (a copy where the strides allow none)
Tensor as_rows(const Tensor& t) {
  if (!t.defined()) return t;
  Tensor r = t.dim() == 2 ? t : t.reshape({t.numel() / t.size(-1), t.size(-1)});
  return r.stride(1) == 1 || r.size(1) == 1 ? r : r.contiguous();
}
int64_t row_stride(const Tensor& t) { return !t.defined() ? 0 : t.size(0) == 1 ? t.size(1) : t.stride(0); }   // (of a single row: its length, whatever it says)
Tensor dense(const Tensor& t) { return t.defined() ? t.contiguous() : t; }

// The gradients of a node whose backward has none of its own: where a graph of them is asked for (create_graph), they hang by a node that raises on what they
// were computed from, so that differentiating them is an error and never takes them for constants.
variable_list once(variable_list grads, std::initializer_list<const Tensor*> from) {
  if (!at::GradMode::is_enabled()) return grads;
  const size_t n = grads.size();
  variable_list all = std::move(grads);
  bool any = false;
  for (const Tensor* t : from)
    if (t->defined() && t->requires_grad()) {
      all.push_back(*t);
      any = true;
    }
  if (!any) return all;
  const size_t count = all.size();
  auto node = std::make_shared<torch::autograd::DelayedError>("the gradients of this operator cannot be differentiated again", (int64_t)count);
  all = (*node)(std::move(all));
  all.resize(n);
  return all;
}

// What a backward pass is given comes out of autograd's hands: a saved tensor's hooks or a `.data` that was set in between may have made another type or size of it, and the
// kernels would read past its end.
bool like(const Tensor& t, const Tensor& x, at::IntArrayRef sizes) {
  return t.defined() && t.scalar_type() == x.scalar_type() && t.device() == x.device() && t.sizes() == sizes;
}
bool maybe_like(const Tensor& t, const Tensor& x, at::IntArrayRef sizes) { return !t.defined() || like(t, x, sizes); }
bool block_of(const Tensor& t, const Tensor& x, at::ScalarType type, int64_t n) {
  return t.defined() && t.scalar_type() == type && t.device() == x.device() && t.numel() == n && t.is_contiguous();
}
void as_saved(bool ok, const char* what) {
  TORCH_CHECK(ok, what, ": a saved tensor or the incoming gradient does not have the forward's size, type or device");
}

// Which inputs of a Function want a gradient: AutogradContext counts the tensors that were given, this counts all of them.
struct Wants {
  AutogradContext* ctx;
  size_t next = 0;
  bool operator()(bool given) { return given && ctx->needs_input_grad(next++); }
};

// Forward-mode derivatives: no operator here has one, and a tangent that is dropped would be taken for zero by whatever comes after.
void no_tangents(std::initializer_list<const Tensor*> ts) {
  if (!c10::AutogradState::get_tls_state().get_fw_grad_mode()) return;
  for (const Tensor* t : ts)
    TORCH_CHECK_NOT_IMPLEMENTED(!t->defined() || !t->_fw_grad(/*level=*/0).defined(), "this operator has no forward-mode derivative (a tensor given to it has a tangent)");
}

bool wants_grad(std::initializer_list<const Tensor*> ts) {
  no_tangents(ts);
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor* t : ts)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}

// ----------------------------------------------------------------------------------------------------------------- layer norm
std::tuple<Tensor, Tensor> norm_forward(const Tensor& x, const Tensor& w, const Tensor& b, double eps, const Tensor& r, bool stats) {
  const On on(x);
  const Tensor x2 = as_rows(x), r2 = as_rows(r), wc = dense(w), bc = dense(b);
  const int64_t rows = x2.size(0), c = x2.size(1);
  Tensor y = at::empty(x.sizes(), x.options()), stat = made(stats, {2, rows}, x, at::kFloat);
  if (rows) {
    float* at = stats ? stat.data_ptr<float>() : nullptr;
    const int wcode = wc.defined() ? code_of(wc.scalar_type()) : bc.defined() ? code_of(bc.scalar_type()) : MOY_F32;
    check(lib.norm(x2.data_ptr(), row_stride(x2), ptr(r2), row_stride(r2), ptr(wc), ptr(bc), wcode, rows, (int)c, (float)eps, y.data_ptr(), c, at,
                   at ? at + rows : nullptr, code_of(x.scalar_type()), on.stream),
          "moy_layer_norm");
  }
  return {y, stat};
}

std::tuple<Tensor, Tensor, Tensor> norm_backward(const Tensor& dy, const Tensor& x, const Tensor& w, const Tensor& stat, const Tensor& r, bool need_x, bool need_w,
                                                 bool need_b, at::ScalarType wtype) {
  as_saved(x.dim() > 0 && x.size(-1) > 0 && like(dy, x, x.sizes()) && maybe_like(r, x, x.sizes()) && block_of(stat, x, at::kFloat, 2 * (x.numel() / x.size(-1))) &&
               (!w.defined() || (w.scalar_type() == wtype && w.device() == x.device() && w.sizes() == x.sizes().slice(x.dim() - 1))) && (wtype == at::kFloat || wtype == x.scalar_type()),
           "layer_norm");
  const On on(x);
  const Tensor x2 = as_rows(x), g2 = as_rows(dy), r2 = as_rows(r), wc = dense(w);
  const int64_t rows = x2.size(0), c = x2.size(1);
  const int code = code_of(x.scalar_type());
  Tensor dx = made(need_x, x.sizes(), x, x.scalar_type()), dw = made(need_w, {c}, x, wtype), db = made(need_b, {c}, x, wtype);
  if (rows == 0) {
    if (need_w) dw.zero_();
    if (need_b) db.zero_();
  } else if (need_x || need_w || need_b) {
    const int64_t n = need_w || need_b ? check(lib.norm_bwd_ws(rows, (int)c, code), "moy_layer_norm_bwd_ws") : 0;
    Tensor ws = floats(n, x);
    float* at = stat.data_ptr<float>();
    check(lib.norm_bwd(g2.data_ptr(), row_stride(g2), x2.data_ptr(), row_stride(x2), ptr(r2), row_stride(r2), ptr(wc), code_of(wtype), at, at + rows, rows, (int)c,
                       ptr(dx), c, ptr(dw), ptr(db), (float*)ptr(ws), n, code, on.stream),
          "moy_layer_norm_bwd");
  }
  return {dx, dw, db};
}

struct NormNode : torch::autograd::Function<NormNode> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const MaybeTensor& w, const MaybeTensor& b, double eps, const MaybeTensor& r) {
    const Tensor wt = tensor_of(w), bt = tensor_of(b), rt = tensor_of(r);
    auto [y, stat] = norm_forward(x, wt, bt, eps, rt, true);
    ctx->save_for_backward({x, wt, rt, stat});
    const auto type = wt.defined() ? wt.scalar_type() : bt.defined() ? bt.scalar_type() : at::kFloat;
    ctx->saved_data["how"] = (int64_t)type * 2 + (bt.defined() ? 1 : 0);
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    no_tangents({&grads[0]});
    const auto s = ctx->get_saved_variables();
    const int64_t how = ctx->saved_data["how"].toInt();
    Wants wants{ctx};
    const bool nx = wants(true), nw = wants(s[1].defined()), nb = wants(how & 1), nr = wants(s[2].defined());
    auto [dx, dw, db] = norm_backward(grads[0], s[0], s[1], s[3], s[2], nx || nr, nw, nb, (at::ScalarType)(how / 2));
    return once({nx ? dx : Tensor(), dw, db, Tensor(), nr ? dx : Tensor()}, {&grads[0], &s[0], &s[1], &s[2]});
  }
};

// ---------------------------------------------------------------------------------------------------------------------- linear
// The rows of x, w, r and dy may lie at any distance.  The entry points take the strides of a view where their kernels' offsets reach (4 MiB from row to row, and any
// stride of a single row or of a few rows going forward) and refuse others as MOY_ENOSYS: those operands are copied to dense rows, and the call is made again.
struct LinearCall {
  moy_linear_args a{};
  Tensor x, w, b, r, dy;
  LinearCall(const Tensor& x_, const Tensor& w_, const Tensor& b_, int64_t act, const Tensor& r_, const Tensor& dy_ = Tensor())
      : x(as_rows(x_)), w(as_rows(w_)), b(dense(b_)), r(as_rows(r_)), dy(as_rows(dy_)) {
    a.act = (int)act; a.dtype = code_of(x.scalar_type());
    a.M = (int)x.size(0); a.N = (int)w.size(0); a.K = (int)w.size(1);
    a.b = ptr(b); a.b_dtype = b.defined() ? code_of(b.scalar_type()) : MOY_F32;
    place();
  }
  void place() {
    a.x = x.data_ptr(); a.ldx = row_stride(x); a.w = w.data_ptr(); a.ldw = row_stride(w);
    a.r = ptr(r); a.ldr = row_stride(r); a.dy = ptr(dy); a.ldd = row_stride(dy);
  }
  bool compact() {                         // (what lies further apart than that, if anything)
    bool any = false;
    for (Tensor* t : {&x, &w, &r, &dy})
      if (t->defined() && t->size(0) > 1 && t->stride(0) * t->element_size() > (1 << 22)) {
        *t = t->contiguous();
        any = true;
      }
    place();
    return any;
  }
  template <typename Query, typename Launch>
  void run(Query query, Launch launch, const char* what, void* stream) {
    int64_t n = query(&a);
    if (n == MOY_ENOSYS && compact()) n = query(&a);
    check(n, what);
    Tensor ws = n ? at::empty({n}, x.options().dtype(at::kByte)) : Tensor();
    a.ws = ptr(ws); a.ws_len = n;
    check(launch(&a, stream), what);
  }
};

std::tuple<Tensor, Tensor> linear_forward(const Tensor& x, const Tensor& w, const Tensor& b, int64_t act, const Tensor& r, bool keep_pre) {
  const On on(x);
  LinearCall c(x, w, b, act, r);
  auto shape = x.sizes().vec();
  shape.back() = c.a.N;
  Tensor y = at::empty(shape, x.options()), z = made(keep_pre && act != MOY_ACT_NONE, {c.a.M, c.a.N}, x, x.scalar_type());
  if (c.a.M) {
    c.a.y = y.data_ptr(); c.a.ldy = c.a.N; c.a.z = ptr(z);
    c.run(lib.linear_ws, lib.linear, "moy_linear", on.stream);
  }
  return {y, z};
}

std::tuple<Tensor, Tensor, Tensor> linear_backward(const Tensor& dy, const Tensor& x, const Tensor& w, const Tensor& z, int64_t act, bool need_x, bool need_w,
                                                   bool need_b, at::ScalarType btype) {
  bool ok = x.dim() > 0 && w.dim() == 2 && w.numel() > 0 && like(w, x, {w.size(0), x.size(-1)}) && (btype == at::kFloat || btype == x.scalar_type());
  if (ok) {
    auto shape = x.sizes().vec();
    shape.back() = w.size(0);
    ok = like(dy, x, shape) && (act == MOY_ACT_NONE || block_of(z, x, x.scalar_type(), x.numel() / x.size(-1) * w.size(0)));
  }
  as_saved(ok, "linear");
  const On on(x);
  LinearCall c(x, w, Tensor(), act, Tensor(), dy);
  c.a.b_dtype = code_of(btype);
  Tensor dx = made(need_x, x.sizes(), x, x.scalar_type()), dw = made(need_w, w.sizes(), x, x.scalar_type()), db = made(need_b, {c.a.N}, x, btype);
  if (c.a.M == 0) {
    if (need_w) dw.zero_();
    if (need_b) db.zero_();
  } else if (need_x || need_w || need_b) {
    c.a.z = ptr(z); c.a.dx = ptr(dx); c.a.dw = ptr(dw); c.a.db = ptr(db);
    c.run(lib.linear_bwd_ws, lib.linear_bwd, "moy_linear_bwd", on.stream);
  }
  return {dx, dw, db};
}

struct LinearNode : torch::autograd::Function<LinearNode> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, const MaybeTensor& b, int64_t act, const MaybeTensor& r) {
    const Tensor bt = tensor_of(b);
    auto [y, z] = linear_forward(x, w, bt, act, tensor_of(r), true);
    ctx->save_for_backward({x, w, z});
    ctx->saved_data["how"] = (((int64_t)(bt.defined() ? bt.scalar_type() : at::kFloat) * 16 + act) * 2 + (bt.defined() ? 1 : 0)) * 2 + (r.has_value() ? 1 : 0);
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    no_tangents({&grads[0]});
    const auto s = ctx->get_saved_variables();
    const int64_t how = ctx->saved_data["how"].toInt();
    Wants wants{ctx};
    const bool nx = wants(true), nw = wants(true), nb = wants(how & 2), nr = wants(how & 1);
    auto [dx, dw, db] = linear_backward(grads[0], s[0], s[1], s[2], how / 4 % 16, nx, nw, nb, (at::ScalarType)(how / 64));
    auto all = once({dx, dw, db, Tensor(), Tensor()}, {&grads[0], &s[0], &s[1]});
    if (nr) all[4] = grads[0];
    return all;
  }
};

// ------------------------------------------------------------------------------------------------------------------- attention
// a view that the kernels address: unit stride within a head, 16-byte steps and base (a copy where the strides allow none); its strides, 0 for an axis of 1
Tensor strided(const Tensor& t, int64_t* sb, int64_t* sl, int64_t* sh) {
  const int64_t step = 16 / t.element_size();
  auto off = [&](int i) { return t.size(i) > 1 && t.stride(i) % step; };
  Tensor r = t;
  if (t.stride(3) != 1 || reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 || off(0) || off(1) || off(2)) {
    r = t.contiguous();
    if (reinterpret_cast<uintptr_t>(r.data_ptr()) % 16) r = r.clone();
  }
  *sb = r.size(0) == 1 ? 0 : r.stride(0);
  *sl = r.size(1) == 1 ? 0 : r.stride(1);
  *sh = r.size(2) == 1 ? 0 : r.stride(2);
  return r;
}

struct AttentionHow {
  bool causal, from_end;
  int64_t q_start;
  double scale;
};

struct AttentionCall {
  moy_attention_args a{};
  Tensor q, k, v, table, lut, k_len, mask;
  AttentionCall(const Tensor& q_, const Tensor& k_, const Tensor& v_, const Tensor& table_, const Tensor& lut_, const Tensor& k_len_, const Tensor& mask_,
                const AttentionHow& how)
      : table(dense(table_)), lut(dense(lut_)), k_len(dense(k_len_)), mask(mask_) {
    q = strided(q_, &a.q_sb, &a.q_sl, &a.q_sh);
    k = strided(k_, &a.k_sb, &a.k_sl, &a.k_sh);
    v = strided(v_, &a.v_sb, &a.v_sl, &a.v_sh);
    a.q = q.data_ptr(); a.k = k.data_ptr(); a.v = v.data_ptr(); a.dtype = code_of(q.scalar_type());
    a.B = (int)q.size(0); a.Lq = (int)q.size(1); a.H = (int)q.size(2); a.D = (int)q.size(3); a.Lk = (int)k.size(1); a.Hk = (int)k.size(2);
    a.scale = (float)how.scale; a.causal = how.causal; a.q_from_end = how.from_end; a.q_start = (int)how.q_start;
    if (table.defined()) {
      a.table = table.data_ptr(); a.lut = lut.data_ptr<uint8_t>(); a.num_buckets = (int)table.size(0); a.max_distance = (int)(lut.size(0) / 2);
    }
    if (k_len.defined()) a.k_len = k_len.data_ptr<int32_t>();
    if (mask.defined()) {
      const int64_t d = mask.dim();
      if (mask.stride(d - 1) != 1 && mask.size(d - 1) > 1) mask = mask.contiguous();
      a.mask = static_cast<const uint8_t*>(mask.data_ptr());
      a.m_sq = mask.size(d - 2) == 1 ? 0 : mask.stride(d - 2);
      if (d == 4) {
        a.m_sb = mask.size(0) == 1 ? 0 : mask.stride(0);
        a.m_sh = mask.size(1) == 1 ? 0 : mask.stride(1);
      }
    }
  }
};

std::tuple<Tensor, Tensor, Tensor> attention_forward(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& table, const Tensor& lut, const Tensor& k_len,
                                                     const Tensor& mask, const AttentionHow& how, bool stats) {
  const On on(q);
  Tensor o = at::empty(q.sizes(), q.options()), lse = made(stats, {q.size(0), q.size(2), q.size(1)}, q, at::kFloat);
  Tensor rest = made(stats && q.scalar_type() != at::kFloat, q.sizes(), q, q.scalar_type());
  if (o.numel() && k.size(1) == 0) {
    o.zero_();
    if (rest.defined()) rest.zero_();
    if (stats) lse.fill_(-std::numeric_limits<double>::infinity());
  } else if (o.numel()) {
    AttentionCall c(q, k, v, table, lut, k_len, mask, how);
    c.a.o = o.data_ptr(); c.a.o_rest = ptr(rest); c.a.lse = (float*)ptr(lse);
    const int64_t n = check(lib.attention_ws(&c.a), "moy_attention_ws");
    Tensor ws = floats(n, q);
    c.a.ws = (float*)ptr(ws); c.a.ws_len = n;
    check(lib.attention(&c.a, on.stream), "moy_attention");
  }
  return {o, lse, rest};
}

std::tuple<Tensor, Tensor, Tensor, Tensor> attention_backward(const Tensor& dout, const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& o, const Tensor& lse,
                                                              const Tensor& rest, const Tensor& table, const Tensor& lut, const Tensor& k_len, const Tensor& mask,
                                                              const AttentionHow& how, bool nq, bool nk, bool nv, bool nt) {
  bool ok = q.dim() == 4 && k.dim() == 4 && k.size(2) > 0 && q.size(2) % k.size(2) == 0 && like(k, q, {q.size(0), k.size(1), k.size(2), q.size(3)}) && like(v, q, k.sizes()) &&
            like(dout, q, q.sizes()) && like(o, q, q.sizes()) && o.is_contiguous() && maybe_like(rest, q, q.sizes()) && (!rest.defined() || rest.is_contiguous()) &&
            block_of(lse, q, at::kFloat, q.size(0) * q.size(1) * q.size(2)) && table.defined() == lut.defined();
  if (ok && table.defined())
    ok = table.dim() == 2 && like(table, q, {table.size(0), q.size(2)}) && lut.dim() == 1 && lut.size(0) % 2 == 1 && lut.scalar_type() == at::kByte && lut.device() == q.device();
  if (ok && k_len.defined()) ok = k_len.dim() == 1 && k_len.size(0) == q.size(0) && k_len.scalar_type() == at::kInt && k_len.device() == q.device();
  if (ok && mask.defined()) {
    const int64_t d = mask.dim(), want[4] = {q.size(0), q.size(2), q.size(1), k.size(1)};
    ok = (d == 2 || d == 4) && mask.element_size() == 1 && mask.device() == q.device() && mask.size(d - 1) == want[3];
    for (int64_t i = 0; ok && i < d - 1; ++i) ok = mask.size(i) == 1 || mask.size(i) == want[4 - d + i];
  }
  as_saved(ok, "attention");
  const On on(q);
  const auto type = q.scalar_type();
  nt = nt && table.defined();
  Tensor dq = made(nq, q.sizes(), q, type), dk = made(nk, k.sizes(), q, type), dv = made(nv, k.sizes(), q, type);
  Tensor dt = nt ? made(true, table.sizes(), q, type) : Tensor();
  if (q.numel() == 0 || k.numel() == 0) {
    for (Tensor* t : {&dq, &dk, &dv, &dt})
      if (t->defined()) t->zero_();
  } else if (nq || nk || nv || nt) {
    AttentionCall c(q, k, v, table, lut, k_len, mask, how);
    const Tensor g = strided(dout, &c.a.g_sb, &c.a.g_sl, &c.a.g_sh);
    c.a.dout = g.data_ptr(); c.a.o = o.data_ptr(); c.a.o_rest = ptr(rest); c.a.lse = lse.data_ptr<float>();
    c.a.dq = ptr(dq); c.a.dk = ptr(dk); c.a.dv = ptr(dv); c.a.dtable = ptr(dt);
    const int64_t n = check(lib.attention_bwd_ws(&c.a), "moy_attention_bwd_ws");
    Tensor ws = floats(n, q);
    c.a.ws = (float*)ptr(ws); c.a.ws_len = n;
    check(lib.attention_bwd(&c.a, on.stream), "moy_attention_bwd");
  }
  return {dq, dk, dv, dt};
}

struct AttentionNode : torch::autograd::Function<AttentionNode> {
  static Tensor forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v, const MaybeTensor& table, const MaybeTensor& lut,
                        const MaybeTensor& k_len, const MaybeTensor& mask, bool causal, bool from_end, int64_t q_start, double scale) {
    const Tensor t = tensor_of(table), l = tensor_of(lut), n = tensor_of(k_len), m = tensor_of(mask);
    auto [o, lse, rest] = attention_forward(q, k, v, t, l, n, m, {causal, from_end, q_start, scale}, true);
    ctx->save_for_backward({q, k, v, o, lse, rest, t, l, n, m});
    ctx->saved_data["how"] = q_start * 4 + (causal ? 2 : 0) + (from_end ? 1 : 0);
    ctx->saved_data["scale"] = scale;
    return o;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    no_tangents({&grads[0]});
    const auto s = ctx->get_saved_variables();
    const int64_t how = ctx->saved_data["how"].toInt();
    Wants wants{ctx};
    const bool nq = wants(true), nk = wants(true), nv = wants(true), nt = wants(s[6].defined());
    auto [dq, dk, dv, dt] = attention_backward(grads[0], s[0], s[1], s[2], s[3], s[4], s[5], s[6], s[7], s[8], s[9],
                                               {(how & 2) != 0, (how & 1) != 0, how >> 2, ctx->saved_data["scale"].toDouble()}, nq, nk, nv, nt);
    return once({dq, dk, dv, dt, Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor()}, {&grads[0], &s[0], &s[1], &s[2], &s[6]});
  }
};

MaybeTensor maybe(const Tensor& t) { return t.defined() ? MaybeTensor(t) : MaybeTensor(); }

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.doc() = "Host side of the transformer-layer operators (csrc/host.cpp); use mo_yolo_amd.ops / mo_yolo_amd.modules.";
  m.def("bind", [](std::map<std::string, uintptr_t> at, py::object error) {
    auto set = [&](auto& f, const char* name) { f = reinterpret_cast<std::decay_t<decltype(f)>>(at.at(name)); };
    set(lib.strerror_, "moy_strerror");
    set(lib.norm, "moy_layer_norm"); set(lib.norm_bwd, "moy_layer_norm_bwd"); set(lib.norm_bwd_ws, "moy_layer_norm_bwd_ws");
    set(lib.linear, "moy_linear"); set(lib.linear_ws, "moy_linear_ws"); set(lib.linear_bwd, "moy_linear_bwd"); set(lib.linear_bwd_ws, "moy_linear_bwd_ws");
    set(lib.attention, "moy_attention"); set(lib.attention_ws, "moy_attention_ws"); set(lib.attention_bwd, "moy_attention_bwd");
    set(lib.attention_bwd_ws, "moy_attention_bwd_ws");
    static PyObject* type = nullptr;
    if (!type) {
      type = error.release().ptr();
      py::register_exception_translator([](std::exception_ptr p) {
        try {
          if (p) std::rethrow_exception(p);
        } catch (const MoyError& e) {
          PyErr_SetString(type, e.what());
        }
      });
    }
  });
  m.def("layer_norm_forward", [](const Tensor& x, const MaybeTensor& w, const MaybeTensor& b, double eps, const MaybeTensor& r, bool stats) {
    return norm_forward(x, tensor_of(w), tensor_of(b), eps, tensor_of(r), stats);
  });
  m.def("layer_norm_backward", [](const Tensor& dy, const Tensor& x, const MaybeTensor& w, const Tensor& stat, const MaybeTensor& r, bool nx, bool nw, bool nb,
                                  at::ScalarType type) {
    return norm_backward(dy, x, tensor_of(w), stat, tensor_of(r), nx, nw, nb, type);
  });
  m.def("layer_norm", [](const Tensor& x, const MaybeTensor& w, const MaybeTensor& b, double eps, const MaybeTensor& r) {
    const Tensor wt = tensor_of(w), bt = tensor_of(b), rt = tensor_of(r);
    if (wants_grad({&x, &wt, &bt, &rt})) return NormNode::apply(x, maybe(wt), maybe(bt), eps, maybe(rt));
    return std::get<0>(norm_forward(x, wt, bt, eps, rt, false));
  });
  m.def("linear_forward", [](const Tensor& x, const Tensor& w, const MaybeTensor& b, int64_t act, const MaybeTensor& r, bool keep_pre) {
    return linear_forward(x, w, tensor_of(b), act, tensor_of(r), keep_pre);
  });
  m.def("linear_backward", [](const Tensor& dy, const Tensor& x, const Tensor& w, const MaybeTensor& z, int64_t act, bool nx, bool nw, bool nb, at::ScalarType type) {
    return linear_backward(dy, x, w, tensor_of(z), act, nx, nw, nb, type);
  });
  m.def("linear", [](const Tensor& x, const Tensor& w, const MaybeTensor& b, int64_t act, const MaybeTensor& r) {
    const Tensor bt = tensor_of(b), rt = tensor_of(r);
    if (wants_grad({&x, &w, &bt, &rt})) return LinearNode::apply(x, w, maybe(bt), act, maybe(rt));
    return std::get<0>(linear_forward(x, w, bt, act, rt, false));
  });
  m.def("attention_forward", [](const Tensor& q, const Tensor& k, const Tensor& v, const MaybeTensor& table, const MaybeTensor& lut, const MaybeTensor& k_len,
                                const MaybeTensor& mask, bool causal, bool from_end, int64_t q_start, double scale, bool stats) {
    return attention_forward(q, k, v, tensor_of(table), tensor_of(lut), tensor_of(k_len), tensor_of(mask), {causal, from_end, q_start, scale}, stats);
  });
  m.def("attention_backward", [](const Tensor& dout, const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& o, const Tensor& lse, const MaybeTensor& rest,
                                 const MaybeTensor& table, const MaybeTensor& lut, const MaybeTensor& k_len, const MaybeTensor& mask, bool causal, bool from_end,
                                 int64_t q_start, double scale, bool nq, bool nk, bool nv, bool nt) {
    return attention_backward(dout, q, k, v, o, lse, tensor_of(rest), tensor_of(table), tensor_of(lut), tensor_of(k_len), tensor_of(mask),
                              {causal, from_end, q_start, scale}, nq, nk, nv, nt);
  });
  m.def("attention", [](const Tensor& q, const Tensor& k, const Tensor& v, const MaybeTensor& table, const MaybeTensor& lut, const MaybeTensor& k_len,
                        const MaybeTensor& mask, bool causal, bool from_end, int64_t q_start, double scale) {
    const Tensor t = tensor_of(table), l = tensor_of(lut), n = tensor_of(k_len), mk = tensor_of(mask);
    if (wants_grad({&q, &k, &v, &t})) return AttentionNode::apply(q, k, v, maybe(t), maybe(l), maybe(n), maybe(mk), causal, from_end, q_start, scale);
    return std::get<0>(attention_forward(q, k, v, t, l, n, mk, {causal, from_end, q_start, scale}, false));
  });
}
