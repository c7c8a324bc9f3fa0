// Attention over packed sequences and the rotation by several axes on torch's C++
// side: checks, autograd nodes, and the launches through the C ABI.
#include "nodes.h"

namespace {

void no_tangents(const char* who, std::initializer_list<const Tensor*> tensors) {
  for (const Tensor* t : tensors)
    if (is_dual(*t)) throw std::runtime_error(std::string(who) + " has no forward-mode derivative");
}

bool wants_gradient(std::initializer_list<const Tensor*> tensors) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor* t : tensors)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}

// What a backward pass gives under create_graph: gradients that say so when they
// are differentiated once more.
variable_list once(const char* who, variable_list out) {
  if (!at::GradMode::is_enabled()) return out;
  for (Tensor& t : out)
    if (t.defined()) t.requires_grad_(true);
  return torch::autograd::DelayedError(std::string(who) + " can be differentiated once",
                                       static_cast<int>(out.size()))(std::move(out));
}

// A tensor that is written has no element twice.
void writable(const char* name, const Tensor& t) {
  for (int64_t i = 0; i < t.dim(); ++i)
    if (t.stride(i) == 0 && t.size(i) > 1)
      bad(std::string(name) + " overlaps itself (an expanded tensor)");
}

// Outputs share no memory with what is read or written beside them (views of one
// buffer that lie between each other's elements are the caller's to keep apart).
void apart(const char* name, const Tensor& out, std::initializer_list<const Tensor*> others) {
  for (const Tensor* t : others) {
    if (!t->defined() || t->numel() == 0 || out.numel() == 0) continue;
    const at::MemOverlapStatus s = at::get_overlap_status(out, *t);
    if (s == at::MemOverlapStatus::Full || s == at::MemOverlapStatus::Partial ||
        out.data_ptr() == t->data_ptr())
      bad(std::string(name) + " overlaps another tensor of the call");
  }
}

// ------------------------------------------------------- packed attention ---
// plan: the int32 words of zk_packed_plan; positions may be undefined.
void packed_plan(const Tensor& offsets, int64_t tokens, const Tensor& plan, const MaybeTensor& given_pos) {
  const Tensor pos = given(given_pos);
  one_gpu({&offsets, &plan, &pos});
  if (offsets.dim() != 1 || offsets.numel() == 0 || !offsets.is_contiguous() ||
      (offsets.scalar_type() != at::kInt && offsets.scalar_type() != at::kLong))
    bad("offsets must be a contiguous int32 or int64 [sequences + 1] tensor");
  const int64_t bytes = zk_packed_plan_bytes(tokens);
  if (bytes < 0) bad(zk_last_error());
  if (plan.scalar_type() != at::kInt || !plan.is_contiguous() || plan.numel() * 4 < bytes)
    bad(c10::str("the plan of ", tokens, " tokens is a contiguous int32 tensor of ", bytes / 4, " words"));
  if (pos.defined() && (pos.scalar_type() != at::kLong || pos.dim() != 1 || pos.size(0) != tokens ||
                        !pos.is_contiguous()))
    bad("positions must be a contiguous int64 [tokens] tensor");
  const c10::DeviceGuard on(offsets.device());
  check(zk_packed_plan(offsets.data_ptr(), offsets.scalar_type() == at::kLong, offsets.numel() - 1, tokens,
                       plan.data_ptr(), plan.numel() * 4, static_cast<int64_t*>(address(pos)),
                       stream_of(offsets)),
        "zk_packed_plan");
}

void heads_like(const char* name, const Tensor& x, const Tensor& t, bool out) {
  if (x.sizes() != t.sizes() || x.scalar_type() != t.scalar_type())
    bad(std::string(name) + " must have the shape and type of its heads");
  if (x.stride(2) != 1 && x.numel() != 0) bad(std::string(name) + " needs unit stride along d");
  if (out) writable(name, x);
}

zk_packed_desc packed_checked(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& plan,
                              bool causal, int64_t window, std::optional<double> scale) {
  if (q.dim() != 3 || k.dim() != 3 || v.dim() != 3)
    bad("packed attention: q must be [tokens, Hq, d], k and v [tokens, Hkv, d]");
  one_gpu({&q, &k, &v, &plan});
  zk_packed_desc D{};
  D.T = q.size(0), D.Hq = q.size(1), D.d = q.size(2), D.Hkv = k.size(1);
  D.dtype = float_code("q", q.scalar_type());
  if (k.size(0) != D.T || k.size(2) != D.d || k.scalar_type() != q.scalar_type() ||
      v.sizes() != k.sizes() || v.scalar_type() != k.scalar_type())
    bad(c10::str("packed attention: k and v must be [", D.T, ", Hkv, ", D.d, "] of q's dtype"));
  if (D.Hq == 0 || D.Hkv == 0 || D.Hq % D.Hkv != 0)
    bad(c10::str("packed attention: ", D.Hq, " query heads are no multiple of ", D.Hkv, " key heads"));
  if (D.d == 0 || D.d > 128 || (D.dtype != ZK_F32 && D.d % 2 != 0))
    bad(c10::str("packed attention: head dims are up to 128, even for 2-byte types (got ", D.d, ")"));
  heads_like("q", q, q, false);
  heads_like("k", k, k, false);
  heads_like("v", v, v, false);
  const int64_t bytes = zk_packed_plan_bytes(D.T);
  if (bytes < 0) bad(zk_last_error());
  if (plan.scalar_type() != at::kInt || !plan.is_contiguous() || plan.numel() * 4 != bytes)
    bad(c10::str("packed attention: the plan is not one of ", D.T, " tokens"));
  if (window < 0 || (window > 0 && !causal))
    bad(c10::str("packed attention: a window (", window, ") needs causal attention and is positive"));
  D.scale = static_cast<float>(scale.value_or(1.0 / std::sqrt(static_cast<double>(D.d))));
  if (!(D.scale > 0.f && D.scale < INFINITY)) bad("packed attention: scale must be positive");
  D.causal = causal;
  D.window = window;
  D.q_s = q.stride(0), D.q_h = q.stride(1);
  D.k_s = k.stride(0), D.k_h = k.stride(1);
  D.v_s = v.stride(0), D.v_h = v.stride(1);
  return D;
}

// The launches, for checked arguments; outputs that are undefined are made, with
// zeros behind the last sequence, where given ones are left as they are.
std::pair<Tensor, Tensor> packed_fwd_launch(zk_packed_desc D, const Tensor& q, const Tensor& k,
                                            const Tensor& v, const Tensor& plan, Tensor o) {
  const c10::DeviceGuard on(q.device());
  D.keep_tail = o.defined();
  if (!o.defined()) o = at::empty(q.sizes(), q.options());
  D.o_s = o.stride(0), D.o_h = o.stride(1);
  const Tensor lse = at::empty({D.Hq, D.T}, q.options().dtype(at::kFloat));
  check(zk_attn_packed_fwd(&D, q.data_ptr(), k.data_ptr(), v.data_ptr(), plan.data_ptr(), o.data_ptr(),
                           static_cast<float*>(lse.data_ptr()), stream_of(q)),
        "zk_attn_packed_fwd");
  return {o, lse};
}

variable_list packed_bwd_launch(zk_packed_desc D, const Tensor& q, const Tensor& k, const Tensor& v,
                                const Tensor& plan, const Tensor& o, const Tensor& dout,
                                const Tensor& lse, Tensor dq, Tensor dk, Tensor dv) {
  const c10::DeviceGuard on(q.device());
  D.keep_tail = dq.defined();
  if (!dq.defined()) {
    dq = at::empty(q.sizes(), q.options());
    dk = at::empty(k.sizes(), k.options());
    dv = at::empty(v.sizes(), v.options());
  }
  D.o_s = o.stride(0), D.o_h = o.stride(1);
  D.do_s = dout.stride(0), D.do_h = dout.stride(1);
  D.dq_s = dq.stride(0), D.dq_h = dq.stride(1);
  D.dk_s = dk.stride(0), D.dk_h = dk.stride(1);
  D.dv_s = dv.stride(0), D.dv_h = dv.stride(1);
  const int64_t bytes = zk_attn_packed_bwd_workspace(&D);
  const Tensor ws = workspace(bytes, q);
  check(zk_attn_packed_bwd(&D, q.data_ptr(), k.data_ptr(), v.data_ptr(), plan.data_ptr(), o.data_ptr(),
                           dout.data_ptr(), static_cast<const float*>(lse.data_ptr()), dq.data_ptr(),
                           dk.data_ptr(), dv.data_ptr(), address(ws), bytes, stream_of(q)),
        "zk_attn_packed_bwd");
  return {dq, dk, dv};
}

// Heads that the 2-byte kernels can read: unit stride along d and rows at
// multiples of 4 bytes; others (an odd view) are copied.
Tensor readable(const Tensor& t) {
  if (t.dim() != 3 || t.numel() == 0) return t;
  bool ok = t.stride(2) == 1;
  if (t.element_size() == 2 && t.is_cuda())
    ok = ok && reinterpret_cast<uintptr_t>(t.data_ptr()) % 4 == 0 && t.stride(0) % 2 == 0 &&
         t.stride(1) % 2 == 0;
  return ok ? t : t.contiguous();
}

struct PackedAttention : torch::autograd::Function<PackedAttention> {
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v,
                               const Tensor& plan, const zk_packed_desc& D) {
    const auto [o, lse] = packed_fwd_launch(D, q, k, v, plan, Tensor());
    ctx->save_for_backward({q, k, v, plan, o, lse});
    ctx->saved_data["desc"] = std::string(reinterpret_cast<const char*>(&D), sizeof(D));
    return {o};
  }
  static variable_list backward(AutogradContext* ctx, variable_list dy) {
    const variable_list s = ctx->get_saved_variables();
    zk_packed_desc D;
    std::memcpy(&D, ctx->saved_data["desc"].toStringRef().data(), sizeof(D));
    no_tangents("packed_attention", {&dy[0]});
    variable_list out = packed_bwd_launch(D, s[0], s[1], s[2], s[3], s[4], readable(dy[0]), s[5],
                                          Tensor(), Tensor(), Tensor());
    out.resize(5);
    return once("packed_attention", std::move(out));
  }
};

// functional.packed_attention
Tensor packed_attention(const Tensor& q_, const Tensor& k_, const Tensor& v_, const Tensor& plan,
                        bool causal, int64_t window, std::optional<double> scale) {
  const Tensor q = readable(q_), k = readable(k_), v = readable(v_);
  const zk_packed_desc D = packed_checked(q, k, v, plan, causal, window, scale);
  no_tangents("packed_attention", {&q, &k, &v});
  if (!wants_gradient({&q, &k, &v})) return packed_fwd_launch(D, q, k, v, plan, Tensor()).first;
  return PackedAttention::apply(q, k, v, plan, D)[0];
}

std::pair<Tensor, Tensor> attn_packed_fwd(const Tensor& q, const Tensor& k, const Tensor& v,
                                          const Tensor& plan, bool causal, int64_t window,
                                          std::optional<double> scale, const MaybeTensor& out) {
  const zk_packed_desc D = packed_checked(q, k, v, plan, causal, window, scale);
  const Tensor o = given(out);
  if (o.defined()) {
    one_gpu({&q, &o});
    heads_like("out", o, q, true);
    apart("out", o, {&q, &k, &v});
  }
  return packed_fwd_launch(D, q, k, v, plan, o);
}

variable_list attn_packed_bwd(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& o,
                              const Tensor& dout, const Tensor& lse, const Tensor& plan, bool causal,
                              int64_t window, std::optional<double> scale, const MaybeTensor& dq,
                              const MaybeTensor& dk, const MaybeTensor& dv) {
  const zk_packed_desc D = packed_checked(q, k, v, plan, causal, window, scale);
  one_gpu({&q, &o, &dout, &lse});
  heads_like("o", o, q, false);
  heads_like("dout", dout, q, false);
  if (lse.scalar_type() != at::kFloat || lse.dim() != 2 || lse.size(0) != D.Hq || lse.size(1) != D.T ||
      !lse.is_contiguous())
    bad("lse must be the forward's contiguous fp32 [Hq, tokens]");
  if (dq.has_value() != dk.has_value() || dq.has_value() != dv.has_value())
    bad("an output for each of dq, dk and dv is needed");
  if (dq.has_value()) {
    one_gpu({&q, &*dq, &*dk, &*dv});
    heads_like("dq", *dq, q, true);
    heads_like("dk", *dk, k, true);
    heads_like("dv", *dv, v, true);
    apart("dq", *dq, {&q, &k, &v, &o, &dout, &*dk, &*dv});
    apart("dk", *dk, {&q, &k, &v, &o, &dout, &*dv});
    apart("dv", *dv, {&q, &k, &v, &o, &dout});
  }
  return packed_bwd_launch(D, q, k, v, plan, o, dout, lse, given(dq), given(dk), given(dv));
}

// ------------------------------------------------- rotation by several axes ---
struct AxesStrides {
  int64_t b = 0, s = 0, h = 0;
};
// Heads [tokens, H, d] or [B, S, H, d].
AxesStrides axes_strides(const Tensor& t) {
  if (t.dim() == 3) return {0, t.stride(0), t.stride(1)};
  return {t.stride(0), t.stride(1), t.stride(2)};
}

zk_axes_desc axes_checked(const Tensor& q, const Tensor& k, const Tensor& cos, const Tensor& sin,
                          const Tensor& positions, const std::string& pair_axes, bool interleaved,
                          bool inverse) {
  if (q.dim() != 3 && q.dim() != 4) bad("rope_axes: q must be [tokens, H, d] or [B, S, H, d]");
  one_gpu({&q, &k, &cos, &sin, &positions});
  const int n = static_cast<int>(q.dim());
  zk_axes_desc D{};
  D.B = n == 4 ? q.size(0) : 1;
  D.S = q.size(n - 3), D.Hq = q.size(n - 2), D.d = q.size(n - 1);
  D.dtype = float_code("q", q.scalar_type());
  if (D.Hq == 0) bad("rope_axes: q has no heads");
  if (D.d == 0 || D.d % 2 != 0 || D.d > 512)
    bad(c10::str("rope_axes: head dims are even and up to 512 (got ", D.d, ")"));
  if (q.stride(n - 1) != 1 && q.numel() != 0) bad("rope_axes: q needs unit stride along d");
  if (k.defined()) {
    if (k.dim() != n || k.size(n - 1) != D.d || k.size(n - 3) != D.S || (n == 4 && k.size(0) != D.B) ||
        k.scalar_type() != q.scalar_type())
      bad("rope_axes: k must match q in all but its heads");
    if (k.stride(n - 1) != 1 && k.numel() != 0) bad("rope_axes: k needs unit stride along d");
    D.Hkv = k.size(n - 2);
  }
  const int64_t half = D.d / 2;
  if (cos.scalar_type() != at::kFloat || sin.scalar_type() != at::kFloat || cos.dim() != 2 ||
      cos.size(1) != half || sin.sizes() != cos.sizes() || !cos.is_contiguous() || !sin.is_contiguous())
    bad(c10::str("cos and sin must be contiguous fp32 [n_pos, ", half, "] tables of as many positions"));
  D.n_pos = cos.size(0);
  if (D.n_pos == 0) bad("the tables hold no positions");
  if (positions.scalar_type() != at::kLong || positions.dim() != n - 1 || !positions.is_contiguous() ||
      positions.size(n - 2) != D.S || (n == 4 && positions.size(1) != D.B))
    bad("rope_axes: positions must be contiguous int64 [axes, tokens] or [axes, B, S]");
  D.n_axes = positions.size(0);
  if (D.n_axes == 0 || D.n_axes > 256) bad(c10::str("rope_axes: 1 to 256 axes (got ", D.n_axes, ")"));
  if (static_cast<int64_t>(pair_axes.size()) != half)
    bad(c10::str("rope_axes: an axis for each of ", half, " pairs is needed (got ", pair_axes.size(), ")"));
  for (const char c : pair_axes)
    if (static_cast<unsigned char>(c) >= D.n_axes)
      bad(c10::str("rope_axes: axis ", static_cast<int>(static_cast<unsigned char>(c)), " of ", D.n_axes));
  D.pairing = interleaved ? ZK_ROPE_INTERLEAVED : ZK_ROPE_HALF;
  D.inverse = inverse;
  return D;
}

std::pair<Tensor, Tensor> axes_launch(zk_axes_desc D, const Tensor& q, const Tensor& k, const Tensor& cos,
                                      const Tensor& sin, const Tensor& positions,
                                      const std::string& pair_axes, Tensor qo, Tensor ko) {
  const c10::DeviceGuard on(q.device());
  if (!qo.defined()) {
    qo = at::empty(q.sizes(), q.options());
    if (k.defined()) ko = at::empty(k.sizes(), k.options());
  }
  AxesStrides s = axes_strides(q);
  D.q_sb = s.b, D.q_ss = s.s, D.q_sh = s.h;
  s = axes_strides(qo);
  D.oq_sb = s.b, D.oq_ss = s.s, D.oq_sh = s.h;
  if (k.defined()) {
    s = axes_strides(k);
    D.k_sb = s.b, D.k_ss = s.s, D.k_sh = s.h;
    s = axes_strides(ko);
    D.ok_sb = s.b, D.ok_ss = s.s, D.ok_sh = s.h;
  }
  check(zk_rope_axes(&D, q.data_ptr(), address(k), qo.data_ptr(), address(ko),
                     static_cast<const float*>(cos.data_ptr()), static_cast<const float*>(sin.data_ptr()),
                     static_cast<const int64_t*>(positions.data_ptr()),
                     reinterpret_cast<const unsigned char*>(pair_axes.data()), stream_of(q)),
        "zk_rope_axes");
  return {qo, ko};
}

struct RopeAxes : torch::autograd::Function<RopeAxes> {
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const MaybeTensor& k,
                               const Tensor& cos, const Tensor& sin, const Tensor& positions,
                               const std::string& pair_axes, const zk_axes_desc& D) {
    const auto [qo, ko] = axes_launch(D, q, given(k), cos, sin, positions, pair_axes, Tensor(), Tensor());
    ctx->save_for_backward({cos, sin, positions});
    ctx->saved_data["desc"] = std::string(reinterpret_cast<const char*>(&D), sizeof(D));
    ctx->saved_data["axes"] = pair_axes;
    return k.has_value() ? variable_list{qo, ko} : variable_list{qo};
  }
  static variable_list backward(AutogradContext* ctx, variable_list dy);
};

// Linear in q and k: a backward pass is the rotation by the opposite angle, and
// differentiates as it does.
variable_list rotated(const Tensor& q, const Tensor& k, const Tensor& cos, const Tensor& sin,
                      const Tensor& positions, const std::string& pair_axes, const zk_axes_desc& D) {
  no_tangents("rope_axes", {&q, &k});
  if (wants_gradient({&q, &k})) {
    variable_list out = RopeAxes::apply(q, maybe(k), cos, sin, positions, pair_axes, D);
    out.resize(2);
    return out;
  }
  const auto [qo, ko] = axes_launch(D, q, k, cos, sin, positions, pair_axes, Tensor(), Tensor());
  return {qo, ko};
}

variable_list RopeAxes::backward(AutogradContext* ctx, variable_list dy) {
  const variable_list s = ctx->get_saved_variables();
  zk_axes_desc D;
  std::memcpy(&D, ctx->saved_data["desc"].toStringRef().data(), sizeof(D));
  D.inverse = !D.inverse;
  const Tensor gk = dy.size() > 1 ? rows_of(dy[1]) : Tensor();
  variable_list out = rotated(rows_of(dy[0]), gk, s[0], s[1], s[2],
                              ctx->saved_data["axes"].toStringRef(), D);
  out.resize(7);
  return out;
}

typedef std::pair<Tensor, MaybeTensor> Heads;

// functional.rope_axes
Heads rope_axes(const Tensor& q_, const MaybeTensor& k_, const Tensor& cos, const Tensor& sin,
                const Tensor& positions, const py::bytes& pair_axes, bool interleaved) {
  const std::string axes = pair_axes;
  const Tensor q = rows_of(q_), k = rows_of(given(k_));
  const zk_axes_desc D = axes_checked(q, k, cos, sin, positions, axes, interleaved, false);
  if (is_dual(cos) || is_dual(sin) || wants_gradient({&cos, &sin}))
    bad("rope_axes: the tables have no gradient");
  const py::gil_scoped_release free_gil;
  const variable_list out = rotated(q, k, cos, sin, positions, axes, D);
  return {out[0], maybe(out[1])};
}

// kernels.rope_axes: either direction; outputs may be the inputs
Heads rope_axes_to(const Tensor& q, const MaybeTensor& k_, const Tensor& cos, const Tensor& sin,
                   const Tensor& positions, const py::bytes& pair_axes, bool interleaved, bool inverse,
                   const MaybeTensor& q_out, const MaybeTensor& k_out) {
  const std::string axes = pair_axes;
  const Tensor k = given(k_), qo = given(q_out), ko = given(k_out);
  const zk_axes_desc D = axes_checked(q, k, cos, sin, positions, axes, interleaved, inverse);
  if ((qo.defined() || ko.defined()) && !(qo.defined() && ko.defined() == k.defined()))
    bad("rope_axes: an output for each of q and k is needed");
  for (const auto& [name, out, in] : {std::tuple{"q output", qo, q}, std::tuple{"k output", ko, k}}) {
    if (!out.defined()) continue;
    one_gpu({&q, &out});
    if (out.sizes() != in.sizes() || out.scalar_type() != in.scalar_type() ||
        (out.stride(-1) != 1 && out.numel() != 0))
      bad(std::string("rope_axes: ") + name + " must have the shape and type of its heads, unit stride along d");
    writable(name, out);
    // in place, or apart
    if (out.data_ptr() != in.data_ptr() || out.strides() != in.strides()) apart(name, out, {&in});
    apart(name, out, {out.is_same(qo) ? &k : &q, out.is_same(qo) ? &ko : &qo});
  }
  const py::gil_scoped_release free_gil;
  const auto out = axes_launch(D, q, k, cos, sin, positions, axes, qo, ko);
  return {out.first, maybe(out.second)};
}

}  // namespace

void bind_packed(py::module_& m) {
  const py::call_guard<py::gil_scoped_release> free_gil;
  m.def("packed_plan", &packed_plan, free_gil);
  m.def("packed_attention", &packed_attention, free_gil);
  m.def("attn_packed_fwd", &attn_packed_fwd, free_gil);
  m.def("attn_packed_bwd", &attn_packed_bwd, free_gil);
  m.def("rope_axes", &rope_axes);
  m.def("rope_axes_to", &rope_axes_to);
}
