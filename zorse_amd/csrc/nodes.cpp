// The token embedding, the norm of query and key heads and the tables of the
// steps over lists of tensors on torch's C++ side: checks, autograd nodes, and
// the launches through the C ABI.
//
// Small calls are bound by the host.  torch runs a backward pass in a thread of
// its own, which finds every Python object of a node written in Python in
// another core's caches: a training pass of few tokens took 85 us where torch's
// own lookup takes 54, of which the kernels are 10.  A node in C++ touches no
// Python object.  The tables of 150 tensors are 750 checks and 1500 numbers,
// 350 us of Python and 20 us here.
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>
#include <pybind11/stl.h>
#include <torch/csrc/utils/pybind.h>

#include <algorithm>
#include <cstring>
#include <optional>
#include <string>
#include <utility>
#include <vector>

#include "../../include/zorse_amd.h"

namespace py = pybind11;
using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
typedef std::optional<Tensor> MaybeTensor;

namespace {

[[noreturn]] void bad(const std::string& what) { throw py::value_error(what); }

void check(int status, const char* who) {
  if (status == 0) return;
  static const char* const names[] = {"ZK_EINVAL", "ZK_EDTYPE", "ZK_EALIGN", "ZK_EUNSUPPORTED",
                                      "ZK_EWORKSPACE"};
  throw std::runtime_error(std::string(who) + " failed with " +
                           (status < 0 && status >= -5 ? names[-1 - status]
                                                       : "hipError " + std::to_string(status)) +
                           ": " + zk_last_error());
}

zk_stream_t stream_of(const Tensor& t) {
  return c10::hip::getCurrentHIPStream(t.get_device()).stream();
}

at::ScalarType type_of(int64_t code) {
  return code == ZK_F32 ? at::kFloat : code == ZK_F16 ? at::kHalf : at::kBFloat16;
}
int code_of(at::ScalarType t) {
  return t == at::kFloat ? ZK_F32 : t == at::kHalf ? ZK_F16 : t == at::kBFloat16 ? ZK_BF16 : -1;
}
int float_code(const char* name, at::ScalarType t) {
  const int code = code_of(t);
  if (code < 0) bad(c10::str("unsupported ", name, " dtype ", t));
  return code;
}

constexpr const char* kNeedGpu = "zorse_amd kernels need GPU tensors (got a CPU tensor)";

void one_gpu(std::initializer_list<const Tensor*> tensors) {
  const Tensor& first = **tensors.begin();
  for (const Tensor* t : tensors) {
    if (!t->defined()) continue;
    if (!t->is_cuda()) bad(kNeedGpu);
    if (t->get_device() != first.get_device()) bad("tensors are on different devices");
  }
}

void* address(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

Tensor given(const MaybeTensor& t) { return t.has_value() ? *t : Tensor(); }

Tensor workspace(int64_t bytes, const Tensor& like) {
  return bytes > 0 ? at::empty({bytes}, like.options().dtype(at::kByte)) : Tensor();
}

// Forward-mode derivatives: a dual tensor carries its tangent beside its values.
bool is_dual(const Tensor& t) { return t.defined() && t._fw_grad(/*level=*/0).defined(); }

// f(t) for a linear f and a dual t, a dual tensor too.
template <typename F>
Tensor linear_of_dual(const Tensor& t, const F& f) {
  const auto [values, tangent] = at::_unpack_dual(t, /*level=*/0);
  // torch's own zeros may have no memory
  const Tensor held = tangent._is_zerotensor() ? at::zeros(tangent.sizes(), values.options()) : tangent;
  return at::_make_dual(f(values), f(held), /*level=*/0);
}

// -------------------------------------------------------- token embedding ---
void check_ids(const Tensor& ids) {
  if (ids.scalar_type() != at::kInt && ids.scalar_type() != at::kLong)
    bad(c10::str("token ids must be int32 or int64 (got ", ids.scalar_type(), ")"));
  if (!ids.is_contiguous()) bad("ids must be contiguous");
}

Tensor embedding_fwd(const Tensor& ids, const Tensor& weight, double scale,
                     std::optional<at::ScalarType> dtype, const MaybeTensor& given_out) {
  Tensor out = given(given_out);
  one_gpu({&ids, &weight, &out});
  check_ids(ids);
  if (weight.dim() != 2 || weight.numel() == 0)
    bad(c10::str("weight must be a [vocab, hidden] table, got ", weight.sizes()));
  if (!weight.is_contiguous()) bad("weight must be contiguous");
  const at::ScalarType type =
      dtype ? *dtype : out.defined() ? out.scalar_type() : weight.scalar_type();
  const int w_code = float_code("weight", weight.scalar_type()), y_code = float_code("output", type);
  std::vector<int64_t> shape = ids.sizes().vec();
  shape.push_back(weight.size(1));
  const c10::DeviceGuard on(weight.device());
  if (!out.defined())
    out = at::empty(shape, weight.options().dtype(type));
  else if (out.sizes() != shape || !out.is_contiguous() || out.scalar_type() != type)
    bad(c10::str("out must be contiguous ", shape, " of the output's dtype"));
  check(zk_embedding_fwd(ids.data_ptr(), ids.scalar_type() == at::kLong, ids.numel(),
                         weight.data_ptr(), weight.size(0), weight.size(1), out.data_ptr(),
                         static_cast<float>(scale), w_code, y_code, stream_of(weight)),
        "zk_embedding_fwd");
  return out;
}

// The launches of the gradient, for checked arguments; pad -1: none.
void embedding_grad(const Tensor& ids, const Tensor& dy, const Tensor& dw, double scale, int64_t pad,
                    bool accumulate) {
  const c10::DeviceGuard on(dy.device());
  const int64_t vocab = dw.size(0), h = dw.size(1);
  const int64_t bytes = zk_embedding_bwd_workspace(ids.numel(), vocab, h);
  if (bytes < 0)
    bad(c10::str("embedding_bwd: ", ids.numel(), " tokens of a ", dw.sizes(), " table are out of range"));
  const Tensor ws = workspace(bytes, dy);
  check(zk_embedding_bwd(ids.data_ptr(), ids.scalar_type() == at::kLong, ids.numel(), dy.data_ptr(),
                         code_of(dy.scalar_type()), dw.data_ptr(), code_of(dw.scalar_type()), vocab, h,
                         static_cast<float>(scale), pad, accumulate, address(ws), bytes, stream_of(dy)),
        "zk_embedding_bwd");
}

Tensor embedding_bwd(const Tensor& ids, const Tensor& dy, int64_t vocab, double scale,
                     std::optional<int64_t> pad, const MaybeTensor& given_dw, bool accumulate,
                     std::optional<at::ScalarType> dw_dtype) {
  Tensor dw = given(given_dw);
  one_gpu({&ids, &dy, &dw});
  check_ids(ids);
  if (!dy.is_contiguous()) bad("dy must be contiguous");
  if (dy.dim() < 1 || dy.sizes().slice(0, dy.dim() - 1) != ids.sizes() || dy.size(-1) == 0)
    bad(c10::str("dy must be [*ids.shape, hidden], got ", dy.sizes(), " for ids ", ids.sizes()));
  const int64_t h = dy.size(-1);
  if (vocab <= 0) bad(c10::str("a table has rows (got vocab ", vocab, ")"));
  if (pad && !(*pad >= 0 && *pad < vocab))
    bad(c10::str("padding_idx ", *pad, " outside [0, ", vocab, ")"));
  float_code("dy", dy.scalar_type());
  const at::ScalarType type =
      dw_dtype ? *dw_dtype : dw.defined() ? dw.scalar_type() : dy.scalar_type();
  float_code("dw", type);
  if (!dw.defined()) {
    if (accumulate) bad("accumulate needs the dw to add to");
    dw = at::empty({vocab, h}, dy.options().dtype(type));
  } else if (dw.dim() != 2 || dw.size(0) != vocab || dw.size(1) != h || !dw.is_contiguous() ||
             dw.scalar_type() != type) {
    bad(c10::str("dw must be contiguous [", vocab, ", ", h, "] of dw_dtype"));
  }
  embedding_grad(ids, dy, dw, scale, pad.value_or(-1), accumulate);
  return dw;
}

// Both nodes know no tangents: apply() is for tensors without one, and
// embedding_of and table_gradient for all.
struct Embedding : torch::autograd::Function<Embedding> {
  static Tensor forward(AutogradContext* ctx, const Tensor& ids, const Tensor& weight, double scale,
                        int64_t pad, int64_t y_code);
  static variable_list backward(AutogradContext* ctx, variable_list dy);
};

Tensor embedding_of(const Tensor& ids, const Tensor& weight, double scale, int64_t pad, int64_t y_code) {
  if (is_dual(weight))
    return linear_of_dual(weight, [&](const Tensor& w) {
      return embedding_of(ids, w.contiguous(), scale, pad, y_code);
    });
  return Embedding::apply(ids, weight, scale, pad, y_code);
}

// The table's gradient as a function of dy (a second differentiation): linear
// in it, and its gradient is the lookup, without the tokens that have none.
struct EmbeddingGrad : torch::autograd::Function<EmbeddingGrad> {
  static Tensor forward(AutogradContext* ctx, const Tensor& ids, const Tensor& dy, int64_t vocab,
                        double scale, int64_t pad, int64_t w_code) {
    ctx->save_for_backward({ids});
    ctx->saved_data["cfg"] = std::vector<int64_t>{vocab, pad, code_of(dy.scalar_type())};
    ctx->saved_data["scale"] = scale;
    const Tensor dw = at::empty({vocab, dy.size(-1)}, dy.options().dtype(type_of(w_code)));
    embedding_grad(ids, dy, dw, scale, pad, false);
    return dw;
  }
  static variable_list backward(AutogradContext* ctx, variable_list ddw) {
    const Tensor ids = ctx->get_saved_variables()[0];
    const auto cfg = ctx->saved_data["cfg"].toIntVector();
    const double scale = ctx->saved_data["scale"].toDouble();
    Tensor none = ids.lt(0).logical_or_(ids.ge(cfg[0]));
    if (cfg[1] >= 0) none.logical_or_(ids.eq(cfg[1]));
    const Tensor ddy = embedding_of(ids, ddw[0].contiguous(), scale, cfg[1], cfg[2]);
    return {Tensor(), ddy.masked_fill(none.unsqueeze(-1), 0), Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

Tensor table_gradient(const Tensor& ids, const Tensor& dy, int64_t vocab, double scale, int64_t pad,
                      int64_t w_code) {
  if (is_dual(dy))
    return linear_of_dual(dy, [&](const Tensor& g) {
      return table_gradient(ids, g.contiguous(), vocab, scale, pad, w_code);
    });
  if (at::GradMode::is_enabled() && dy.requires_grad())  // create_graph
    return EmbeddingGrad::apply(ids, dy, vocab, scale, pad, w_code);
  const Tensor dw = at::empty({vocab, dy.size(-1)}, dy.options().dtype(type_of(w_code)));
  embedding_grad(ids, dy, dw, scale, pad, false);
  return dw;
}

Tensor Embedding::forward(AutogradContext* ctx, const Tensor& ids, const Tensor& weight, double scale,
                          int64_t pad, int64_t y_code) {
  ctx->save_for_backward({ids});
  ctx->saved_data["cfg"] = std::vector<int64_t>{weight.size(0), pad, code_of(weight.scalar_type())};
  ctx->saved_data["scale"] = scale;
  return embedding_fwd(ids, weight, scale, type_of(y_code), MaybeTensor());
}

variable_list Embedding::backward(AutogradContext* ctx, variable_list dy) {
  const Tensor ids = ctx->get_saved_variables()[0];
  const auto cfg = ctx->saved_data["cfg"].toIntVector();
  const double scale = ctx->saved_data["scale"].toDouble();
  const Tensor g = dy[0].contiguous();
  return {Tensor(), table_gradient(ids, g, cfg[0], scale, cfg[1], cfg[2]), Tensor(), Tensor(), Tensor()};
}

// functional.embedding
Tensor embedding(const Tensor& ids, const Tensor& weight, double scale, std::optional<int64_t> padding,
                 std::optional<at::ScalarType> dtype) {
  int64_t pad = -1;
  if (padding) {
    const int64_t rows = weight.dim() > 0 ? weight.size(0) : 0;
    if (*padding < -rows || *padding >= rows)
      bad(c10::str("padding_idx ", *padding, " outside a table of ", rows, " rows"));
    pad = *padding < 0 ? *padding + rows : *padding;
  }
  const Tensor i = ids.contiguous(), w = weight.contiguous();
  if (!is_dual(w) && (!at::GradMode::is_enabled() || !w.requires_grad()))
    return embedding_fwd(i, w, scale, dtype, MaybeTensor());
  return embedding_of(i, w, scale, pad, float_code("output", dtype.value_or(w.scalar_type())));
}

// ---------------------------------------- norm of q and k heads, rotation ---
struct Qk {  // operands; k, wk and positions may be undefined
  Tensor q, k, wq, wk, cos, sin, positions;
};

// Unit stride along d (expanded heads and gradients have none).
Tensor rows_of(const Tensor& t) {
  return !t.defined() || t.dim() == 0 || t.stride(-1) == 1 ? t : t.contiguous();
}

struct Strides {
  int64_t b = 0, s = 0, h = 0;
};
Strides contiguous_strides(const Tensor& t) {
  return Strides{t.size(1) * t.size(2) * t.size(3), t.size(2) * t.size(3), t.size(3)};
}
// Of x, which lies over the heads t; `out`: and is written.
Strides strides_over(const char* name, const Tensor& x, const Tensor& t, bool out) {
  if (x.sizes() != t.sizes() || x.scalar_type() != t.scalar_type())
    bad(std::string(name) + " must have the shape and type of its heads");
  if (x.stride(3) != 1 && x.numel() != 0) bad(std::string(name) + " needs unit stride along d");
  for (int i = 0; out && i < 3; ++i)
    if (x.stride(i) == 0 && x.size(i) > 1)
      bad(std::string(name) + " overlaps itself (an expanded tensor)");
  return Strides{x.stride(0), x.stride(1), x.stride(2)};
}

// Neither direction has a forward-mode derivative.
void no_tangents(std::initializer_list<const Tensor*> tensors) {
  for (const Tensor* t : tensors)
    if (is_dual(*t)) throw std::runtime_error("qk_norm_rope has no forward-mode derivative");
}

// The checks of both directions.  qo, ko: y or dx (undefined: new contiguous
// tensors); gq, gk: dy, of the backward.
zk_qk_desc qk_checked(const Qk& A, double eps, bool interleaved, const Tensor& qo, const Tensor& ko,
                      const Tensor& gq, const Tensor& gk) {
  const Tensor &q = A.q, &k = A.k;
  if (q.dim() != 4) bad("q must be [B, S, H, d]");
  if (k.defined() != A.wk.defined()) bad("k and k_weight belong together");
  // both or none: a missing one would be made new and contiguous, and written
  // with the given one's strides
  if ((qo.defined() || ko.defined()) && !(qo.defined() && ko.defined() == k.defined()))
    bad("an output for each of q and k is needed");
  one_gpu({&q, &k, &A.wq, &A.wk, &A.cos, &A.sin, &A.positions, &qo, &ko, &gq, &gk});
  zk_qk_desc D{};
  D.B = q.size(0), D.S = q.size(1), D.Hq = q.size(2), D.d = q.size(3);
  D.dtype = float_code("q", q.scalar_type());
  D.w_dtype = float_code("q_weight", A.wq.scalar_type());
  if (D.Hq == 0) bad("q has no heads");
  if (D.d % 2 != 0 || D.d <= 0 || D.d > 1024)
    bad(c10::str("head dims are even and up to 1024 (got ", D.d, ")"));
  if (A.wq.dim() != 1 || A.wq.size(0) != D.d || !A.wq.is_contiguous())
    bad(c10::str("q_weight must be contiguous [", D.d, "]"));
  if (k.defined()) {
    if (k.dim() != 4 || k.size(0) != D.B || k.size(1) != D.S || k.size(3) != D.d ||
        k.scalar_type() != q.scalar_type())
      bad("k must be [B, S, H, d] matching q");
    if (A.wk.dim() != 1 || A.wk.size(0) != D.d || A.wk.scalar_type() != A.wq.scalar_type() ||
        !A.wk.is_contiguous())
      bad(c10::str("k_weight must be contiguous [", D.d, "] of q_weight's dtype"));
    D.Hkv = k.size(2);
  }
  Strides s = strides_over("q", q, q, false);
  D.q_sb = s.b, D.q_ss = s.s, D.q_sh = s.h;
  s = qo.defined() ? strides_over("q output", qo, q, true) : contiguous_strides(q);
  D.oq_sb = s.b, D.oq_ss = s.s, D.oq_sh = s.h;
  if (gq.defined()) s = strides_over("q gradient", gq, q, false);
  D.dyq_sb = s.b, D.dyq_ss = s.s, D.dyq_sh = s.h;
  if (k.defined()) {
    s = strides_over("k", k, k, false);
    D.k_sb = s.b, D.k_ss = s.s, D.k_sh = s.h;
    s = ko.defined() ? strides_over("k output", ko, k, true) : contiguous_strides(k);
    D.ok_sb = s.b, D.ok_ss = s.s, D.ok_sh = s.h;
    if (gk.defined()) s = strides_over("k gradient", gk, k, false);
    D.dyk_sb = s.b, D.dyk_ss = s.s, D.dyk_sh = s.h;
  }
  const int64_t half = D.d / 2;
  if (A.cos.scalar_type() != at::kFloat || A.sin.scalar_type() != at::kFloat || A.cos.dim() != 2 ||
      A.cos.size(1) != half || A.sin.sizes() != A.cos.sizes() || !A.cos.is_contiguous() ||
      !A.sin.is_contiguous())
    bad(c10::str("cos and sin must be contiguous fp32 [n_pos, ", half,
                 "] tables of as many positions"));
  D.n_pos = A.cos.size(0);
  if (A.positions.defined()) {
    const Tensor& p = A.positions;
    const bool shared = p.dim() == 1 && p.size(0) == D.S;
    const bool own = p.dim() == 2 && p.size(0) == D.B && p.size(1) == D.S;
    if (p.scalar_type() != at::kLong || !(shared || own) || !p.is_contiguous())
      bad("positions must be a contiguous int64 [S] or [B, S] tensor");
    D.pos_sb = own ? D.S : 0;
  } else if (D.n_pos < D.S) {
    bad(c10::str("table holds ", D.n_pos, " positions < S=", D.S));
  }
  if (D.n_pos == 0) bad("the tables hold no positions");
  D.eps = static_cast<float>(eps);
  D.pairing = interleaved ? ZK_ROPE_INTERLEAVED : ZK_ROPE_HALF;
  return D;
}

// The launches, for checked arguments; outputs that are undefined are made.
void qk_fwd(const Qk& A, const zk_qk_desc& D, Tensor& qo, Tensor& ko) {
  const c10::DeviceGuard on(A.q.device());
  if (!qo.defined()) {
    qo = at::empty(A.q.sizes(), A.q.options());
    if (A.k.defined()) ko = at::empty(A.k.sizes(), A.k.options());
  }
  check(zk_qk_norm_rope_fwd(&D, A.q.data_ptr(), address(A.k), A.wq.data_ptr(), address(A.wk),
                            qo.data_ptr(), address(ko), static_cast<const float*>(A.cos.data_ptr()),
                            static_cast<const float*>(A.sin.data_ptr()),
                            static_cast<const int64_t*>(address(A.positions)), stream_of(A.q)),
        "zk_qk_norm_rope_fwd");
}

variable_list qk_bwd(const Qk& A, const zk_qk_desc& D, const Tensor& gq, const Tensor& gk, Tensor dq,
                     Tensor dk) {
  const c10::DeviceGuard on(A.q.device());
  if (!dq.defined()) {
    dq = at::empty(A.q.sizes(), A.q.options());
    if (A.k.defined()) dk = at::empty(A.k.sizes(), A.k.options());
  }
  const Tensor dwq = at::empty({D.d}, A.wq.options());
  const Tensor dwk = A.k.defined() ? at::empty({D.d}, A.wk.options()) : Tensor();
  const int64_t bytes = zk_qk_norm_rope_bwd_workspace(D.d);
  const Tensor ws = workspace(bytes, A.q);
  check(zk_qk_norm_rope_bwd(&D, A.q.data_ptr(), address(A.k), A.wq.data_ptr(), address(A.wk),
                            gq.data_ptr(), address(gk), dq.data_ptr(), address(dk), dwq.data_ptr(),
                            address(dwk), static_cast<const float*>(A.cos.data_ptr()),
                            static_cast<const float*>(A.sin.data_ptr()),
                            static_cast<const int64_t*>(address(A.positions)), address(ws), bytes,
                            stream_of(A.q)),
        "zk_qk_norm_rope_bwd");
  return {dq, dk, dwq, dwk};
}

// Saves its inputs only, and takes the norm from them again.
struct QkNormRope : torch::autograd::Function<QkNormRope> {
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const MaybeTensor& k,
                               const Tensor& wq, const MaybeTensor& wk, const Tensor& cos,
                               const Tensor& sin, const MaybeTensor& positions,
                               const zk_qk_desc& desc) {
    const Qk A{q, given(k), wq, given(wk), cos, sin, given(positions)};
    ctx->save_for_backward({A.q, A.k, A.wq, A.wk, A.cos, A.sin, A.positions});
    ctx->saved_data["desc"] = std::string(reinterpret_cast<const char*>(&desc), sizeof(desc));
    Tensor qo, ko;
    qk_fwd(A, desc, qo, ko);
    return A.k.defined() ? variable_list{qo, ko} : variable_list{qo};
  }

  static variable_list backward(AutogradContext* ctx, variable_list dy) {
    const variable_list s = ctx->get_saved_variables();
    const Qk A{s[0], s[1], s[2], s[3], s[4], s[5], s[6]};
    zk_qk_desc D;
    std::memcpy(&D, ctx->saved_data["desc"].toStringRef().data(), sizeof(D));
    const Tensor gq = rows_of(dy[0]), gk = A.k.defined() ? rows_of(dy[1]) : Tensor();
    no_tangents({&gq, &gk});
    D.dyq_sb = gq.stride(0), D.dyq_ss = gq.stride(1), D.dyq_sh = gq.stride(2);
    if (gk.defined()) D.dyk_sb = gk.stride(0), D.dyk_ss = gk.stride(1), D.dyk_sh = gk.stride(2);
    variable_list out = qk_bwd(A, D, gq, gk, Tensor(), Tensor());
    out.resize(8);
    // dx and dw depend on the saved inputs as well as on dy, one of which
    // requires a gradient
    if (!at::GradMode::is_enabled()) return out;
    // create_graph: what is differentiated once more says so
    for (Tensor& t : out)
      if (t.defined()) t.requires_grad_(true);
    return torch::autograd::DelayedError("qk_norm_rope can be differentiated once", 8)(std::move(out));
  }
};

typedef std::pair<Tensor, MaybeTensor> QkPair;
MaybeTensor maybe(const Tensor& t) { return t.defined() ? MaybeTensor(t) : MaybeTensor(); }

// functional.qk_norm_rope
QkPair qk_norm_rope(const Tensor& q, const MaybeTensor& k, const Tensor& wq, const MaybeTensor& wk,
                    const Tensor& cos, const Tensor& sin, const MaybeTensor& positions, double eps,
                    bool interleaved) {
  const Qk A{rows_of(q), rows_of(given(k)), wq, given(wk), cos, sin, given(positions)};
  const zk_qk_desc D = qk_checked(A, eps, interleaved, Tensor(), Tensor(), Tensor(), Tensor());
  no_tangents({&A.q, &A.k, &A.wq, &A.wk, &A.cos, &A.sin});
  bool grad = false;
  for (const Tensor* t : {&A.q, &A.k, &A.wq, &A.wk}) grad = grad || (t->defined() && t->requires_grad());
  if (!grad || !at::GradMode::is_enabled()) {
    Tensor qo, ko;
    qk_fwd(A, D, qo, ko);
    return {qo, maybe(ko)};
  }
  const variable_list out = QkNormRope::apply(A.q, maybe(A.k), wq, wk, cos, sin, positions, D);
  return {out[0], A.k.defined() ? MaybeTensor(out[1]) : MaybeTensor()};
}

QkPair qk_norm_rope_fwd(const Tensor& q, const MaybeTensor& k, const Tensor& wq, const MaybeTensor& wk,
                        const Tensor& cos, const Tensor& sin, const MaybeTensor& positions, double eps,
                        bool interleaved, const MaybeTensor& q_out, const MaybeTensor& k_out) {
  const Qk A{q, given(k), wq, given(wk), cos, sin, given(positions)};
  Tensor qo = given(q_out), ko = given(k_out);
  const zk_qk_desc D = qk_checked(A, eps, interleaved, qo, ko, Tensor(), Tensor());
  qk_fwd(A, D, qo, ko);
  return {qo, maybe(ko)};
}

std::vector<MaybeTensor> qk_norm_rope_bwd(const MaybeTensor& dq_out, const MaybeTensor& dk_out,
                                          const Tensor& q, const MaybeTensor& k, const Tensor& wq,
                                          const MaybeTensor& wk, const Tensor& cos, const Tensor& sin,
                                          const MaybeTensor& positions, double eps, bool interleaved,
                                          const MaybeTensor& dq, const MaybeTensor& dk) {
  const Qk A{q, given(k), wq, given(wk), cos, sin, given(positions)};
  if (!dq_out || dk_out.has_value() != k.has_value()) bad("a gradient for each of q and k is needed");
  const zk_qk_desc D =
      qk_checked(A, eps, interleaved, given(dq), given(dk), given(dq_out), given(dk_out));
  std::vector<MaybeTensor> out;
  for (const Tensor& t : qk_bwd(A, D, given(dq_out), given(dk_out), given(dq), given(dk)))
    out.push_back(maybe(t));
  return out;
}

// ------------------------------------------------- lists of tensors: tables ---
constexpr int kByteBit = 3, kShortBit = 4;  // beside the three types' codes
constexpr int64_t kBlock = 256;             // elements that share a base of 8-bit codes

int bit_of(at::ScalarType t) {
  return t == at::kByte ? kByteBit : t == at::kShort ? kShortBit : code_of(t);
}

struct Sequence {  // a list or tuple (or what can be made one), held while it is read
  py::object held;
  Py_ssize_t size;
  PyObject** items;
  explicit Sequence(py::handle h)
      : held(py::reinterpret_steal<py::object>(PySequence_Fast(h.ptr(), "a list is needed"))) {
    if (!held) throw py::error_already_set();
    size = PySequence_Fast_GET_SIZE(held.ptr());
    items = PySequence_Fast_ITEMS(held.ptr());
  }
};

int64_t integer(PyObject* o) {
  if (PyLong_Check(o)) {
    const int64_t v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) throw py::error_already_set();
    return v;
  }
  const py::object i = py::reinterpret_steal<py::object>(PyNumber_Long(o));  // a tensor's count
  if (!i) throw py::error_already_set();
  return integer(i.ptr());
}

// Memory of a list's tensor `owner`.
struct Span {
  int64_t begin, end;
  int owner;
  bool written;
  bool operator<(const Span& o) const { return begin < o.begin; }
};

// Sorts what mostly is a few ascending runs.
void sort_runs(std::vector<Span>& spans) {
  const auto begin = spans.begin();
  auto mid = std::is_sorted_until(begin, spans.end());
  for (int run = 1; mid != spans.end(); ++run) {
    if (run == 8) return std::sort(begin, spans.end());
    const auto end = std::is_sorted_until(mid, spans.end());
    std::inplace_merge(begin, mid, end);
    mid = end;
  }
}

// Whether one that is written meets another: workgroups would write it from two
// places, or read it before or after at random.  A tensor's own columns may be
// one (a copy that is the parameter): the same thread has the same element of
// both.
bool spans_clash(std::vector<Span>& spans) {
  sort_runs(spans);
  struct {
    Span last{0, 0, -1, false};  // owner -1: several
    bool is(const Span& s) const {
      return s.owner == last.owner && s.begin == last.begin && s.end == last.end;
    }
    bool meets(const Span& s) const { return s.begin < last.end && !is(s); }
    void add(const Span& s) {
      if (s.begin >= last.end) last = s;
      else if (!is(s)) last = {last.begin, std::max(last.end, s.end), -1, s.written};
    }
  } read, written;
  for (const Span& s : spans) {
    if (written.meets(s) || (s.written && read.meets(s))) return true;
    (s.written ? written : read).add(s);
  }
  return false;
}

// The memory of a column's tensors, one after another unless `mixed`.
struct Reach {
  int64_t begin = INT64_MAX, end = 0;
  bool written = false, mixed = false;
  void add(int64_t from, int64_t to) {
    mixed = mixed || from < end;
    begin = std::min(begin, from);
    end = std::max(end, to);
  }
  // nothing of the two can clash
  bool apart(const Reach& o) const {
    return (!written && !o.written) || begin >= o.end || o.begin >= end;
  }
};

// The columns that the reaches alone do not clear.
std::vector<size_t> unclear(const std::vector<Reach>& columns) {
  std::vector<size_t> out;
  for (size_t c = 0; c < columns.size(); ++c) {
    bool clear = !(columns[c].written && columns[c].mixed);
    for (size_t d = 0; d < columns.size(); ++d) clear = clear && (d == c || columns[c].apart(columns[d]));
    if (!clear) out.push_back(c);
  }
  return out;
}

// (device index, rows of 64-bit fields) of a list of tensors: for each the
// addresses of the columns, the elements of the first column's, the integers,
// and the type codes of the columns in `codes`.  A column is (name, tensors,
// mask of type bits, kind, written): contiguous tensors on one GPU, as large as
// the first column's (kind 0; 1: None is allowed too) or two for each block of
// them (2).  Those that are written share no memory with others.
py::tuple rows(const std::string& who, const py::tuple& columns, const py::tuple& integers,
               const py::tuple& codes) {
  const size_t nc = columns.size(), ni = integers.size(), fields = nc + 1 + ni + codes.size();
  std::vector<Sequence> lists;
  for (const auto& c : columns) lists.emplace_back(py::tuple(c.cast<py::tuple>())[1]);
  for (const auto& c : integers) lists.emplace_back(c);
  const Py_ssize_t n = lists[0].size;
  for (const Sequence& l : lists)
    if (l.size != n) throw py::value_error(who + ": the lists differ in length");
  py::bytes table = py::reinterpret_steal<py::bytes>(
      PyBytes_FromStringAndSize(nullptr, n * static_cast<Py_ssize_t>(fields) * 8));
  if (!table) throw py::error_already_set();
  int64_t* out = reinterpret_cast<int64_t*>(PyBytes_AS_STRING(table.ptr()));
  int64_t index = -1;
  std::vector<int64_t> numel(n), code(n * nc);
  std::vector<int64_t> ends(n * nc, 0);  // 0: no memory
  std::vector<Reach> reaches(nc);
  for (size_t c = 0; c < nc; ++c) {
    const py::tuple column = columns[c].cast<py::tuple>();
    const int64_t mask = column[2].cast<int64_t>(), kind = column[3].cast<int64_t>();
    reaches[c].written = column[4].cast<bool>();
    for (Py_ssize_t i = 0; i < n; ++i) {
      PyObject* o = lists[c].items[i];
      int64_t& field = out[i * fields + c];
      if (kind == 1 && o == Py_None) {
        field = 0;
        continue;
      }
      if (!THPVariable_Check(o)) throw py::type_error(who + ": lists of tensors are needed");
      const Tensor& t = THPVariable_Unpack(o);
      if (!t.is_cuda()) throw py::value_error(kNeedGpu);
      if (c == 0) numel[i] = t.numel();
      if (index < 0) index = t.get_device();
      const int64_t want = kind == 2 ? (numel[i] + kBlock - 1) / kBlock * 2 : numel[i];
      const int bit = bit_of(t.scalar_type());
      if (bit < 0 || !(mask >> bit & 1) || t.numel() != want || t.get_device() != index ||
          !t.is_contiguous()) {
        static const char* const names[] = {"fp32", "fp16", "bf16", "uint8", "int16"};
        static const int bits[] = {ZK_F32, ZK_F16, ZK_BF16, kByteBit, kShortBit};
        std::string types;
        for (int k = 0; k < 5; ++k)
          if (mask >> bits[k] & 1) types += (types.empty() ? "" : " / ") + std::string(names[k]);
        throw py::value_error(who + ": " + column[0].cast<std::string>() + " " + std::to_string(i) +
                              " must be contiguous " + types + " with " + std::to_string(want) +
                              " elements on cuda:" + std::to_string(index));
      }
      field = reinterpret_cast<int64_t>(t.data_ptr());
      code[c * n + i] = bit;
      if (want > 0) {
        const int64_t end = field + want * static_cast<int64_t>(t.element_size());
        ends[i * nc + c] = end;
        reaches[c].add(field, end);
      }
    }
  }
  std::vector<Span> spans;
  if (const std::vector<size_t> left = unclear(reaches); !left.empty()) {
    spans.reserve(n * left.size());
    for (Py_ssize_t i = 0; i < n; ++i)  // a tensor's columns in turn, as states are allocated
      for (const size_t c : left)
        if (ends[i * nc + c] != 0)
          spans.push_back({out[i * fields + c], ends[i * nc + c], static_cast<int>(i), reaches[c].written});
  }
  if (spans_clash(spans))
    throw py::value_error(who + ": a tensor that is written is in the lists twice, or overlaps another");
  for (Py_ssize_t i = 0; i < n; ++i) {
    int64_t* row = out + i * fields + nc;
    *row++ = numel[i];
    for (size_t c = 0; c < ni; ++c) *row++ = integer(lists[nc + c].items[i]);
    for (const auto& c : codes) *row++ = code[c.cast<size_t>() * n + i];
  }
  return py::make_tuple(index, std::move(table));
}

}  // namespace

PYBIND11_MODULE(_nodes, m) {
  const py::call_guard<py::gil_scoped_release> free_gil;
  m.def("embedding", &embedding, free_gil);
  m.def("embedding_fwd", &embedding_fwd, free_gil);
  m.def("embedding_bwd", &embedding_bwd, free_gil);
  m.def("qk_norm_rope", &qk_norm_rope, free_gil);
  m.def("qk_norm_rope_fwd", &qk_norm_rope_fwd, free_gil);
  m.def("qk_norm_rope_bwd", &qk_norm_rope_bwd, free_gil);
  m.def("rows", &rows);
}
