// Autograd nodes of the token embedding and of the norm of query and key heads,
// and the tables of the steps over lists of tensors, for torch's C++ side.
//
// torch runs a backward pass in a thread of its own, which finds every Python
// object of a node written in Python in another core's caches: a training pass
// of few tokens took 85 us where torch's own lookup takes 54, of which the
// kernels are 10.  A node in C++ touches no Python object.  The tables of 150
// tensors are 750 checks and 1500 numbers, 350 us of Python and 20 us here.
//
// The arguments of the nodes are checked by the Python functions that call
// them; the kernels are called through the C ABI, as from Python.
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

void check(int status, const char* who) {
  TORCH_CHECK(status == 0, who, " failed with status ", status, ": ", zk_last_error());
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

void* address(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

Tensor workspace(int64_t bytes, const Tensor& like) {
  return bytes > 0 ? at::empty({bytes}, like.options().dtype(at::kByte)) : Tensor();
}

// -------------------------------------------------------- token embedding ---
Tensor embedding_grad(const Tensor& ids, const Tensor& dy, int64_t vocab, double scale, int64_t pad,
                      int64_t w_code) {
  const c10::DeviceGuard on(dy.device());
  const int64_t h = dy.size(-1), bytes = zk_embedding_bwd_workspace(ids.numel(), vocab, h);
  TORCH_CHECK_VALUE(bytes >= 0, "embedding: ", ids.numel(), " tokens of a [", vocab, ", ", h,
                    "] table are out of range");
  Tensor dw = at::empty({vocab, h}, dy.options().dtype(type_of(w_code)));
  const Tensor ws = workspace(bytes, dy);
  check(zk_embedding_bwd(ids.data_ptr(), ids.scalar_type() == at::kLong, ids.numel(), dy.data_ptr(),
                         code_of(dy.scalar_type()), dw.data_ptr(), static_cast<int>(w_code), vocab, h,
                         static_cast<float>(scale), pad, 0, address(ws), bytes, stream_of(dy)),
        "zk_embedding_bwd");
  return dw;
}

struct Embedding : torch::autograd::Function<Embedding> {
  static Tensor forward(AutogradContext* ctx, const Tensor& ids, const Tensor& weight, double scale,
                        int64_t pad, int64_t y_code);
  static variable_list backward(AutogradContext* ctx, variable_list dy);
};

// The table's gradient as a function of dy (a second differentiation): linear
// in it, and its gradient is the lookup, without the tokens that have none.
struct EmbeddingGrad : torch::autograd::Function<EmbeddingGrad> {
  static Tensor forward(AutogradContext* ctx, const Tensor& ids, const Tensor& dy, int64_t vocab,
                        double scale, int64_t pad, int64_t w_code) {
    ctx->save_for_backward({ids});
    ctx->saved_data["cfg"] = std::vector<int64_t>{vocab, pad, code_of(dy.scalar_type())};
    ctx->saved_data["scale"] = scale;
    return embedding_grad(ids, dy, vocab, scale, pad, w_code);
  }
  static variable_list backward(AutogradContext* ctx, variable_list ddw) {
    const Tensor ids = ctx->get_saved_variables()[0];
    const auto cfg = ctx->saved_data["cfg"].toIntVector();
    const double scale = ctx->saved_data["scale"].toDouble();
    Tensor none = ids.lt(0).logical_or_(ids.ge(cfg[0]));
    if (cfg[1] >= 0) none.logical_or_(ids.eq(cfg[1]));
    const Tensor ddy = Embedding::apply(ids, ddw[0].contiguous(), scale, cfg[1], cfg[2]);
    return {Tensor(), ddy.masked_fill(none.unsqueeze(-1), 0), Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

Tensor Embedding::forward(AutogradContext* ctx, const Tensor& ids, const Tensor& weight, double scale,
                          int64_t pad, int64_t y_code) {
  const c10::DeviceGuard on(weight.device());
  const int64_t vocab = weight.size(0), h = weight.size(1), w_code = code_of(weight.scalar_type());
  ctx->save_for_backward({ids});
  ctx->saved_data["cfg"] = std::vector<int64_t>{vocab, pad, w_code};
  ctx->saved_data["scale"] = scale;
  std::vector<int64_t> shape = ids.sizes().vec();
  shape.push_back(h);
  Tensor y = at::empty(shape, weight.options().dtype(type_of(y_code)));
  check(zk_embedding_fwd(ids.data_ptr(), ids.scalar_type() == at::kLong, ids.numel(),
                         weight.data_ptr(), vocab, h, y.data_ptr(), static_cast<float>(scale),
                         static_cast<int>(w_code), static_cast<int>(y_code), stream_of(weight)),
        "zk_embedding_fwd");
  return y;
}

variable_list Embedding::backward(AutogradContext* ctx, variable_list dy) {
  const Tensor ids = ctx->get_saved_variables()[0];
  const auto cfg = ctx->saved_data["cfg"].toIntVector();
  const double scale = ctx->saved_data["scale"].toDouble();
  const Tensor g = dy[0].contiguous();
  const Tensor dw = at::GradMode::is_enabled() && g.requires_grad()
                        ? EmbeddingGrad::apply(ids, g, cfg[0], scale, cfg[1], cfg[2])
                        : embedding_grad(ids, g, cfg[0], scale, cfg[1], cfg[2]);
  return {Tensor(), dw, Tensor(), Tensor(), Tensor()};
}

// ---------------------------------------- norm of q and k heads, rotation ---
Tensor rows_of(const Tensor& t) {  // unit stride along d (an expanded gradient has none)
  return !t.defined() || t.stride(-1) == 1 ? t : t.contiguous();
}

struct QkNormRope : torch::autograd::Function<QkNormRope> {
  // desc: of contiguous outputs, whose gradients' strides backward() fills in
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const MaybeTensor& k,
                               const Tensor& wq, const MaybeTensor& wk, const Tensor& cos,
                               const Tensor& sin, const MaybeTensor& positions,
                               const zk_qk_desc& desc) {
    const c10::DeviceGuard on(q.device());
    const Tensor key = k.value_or(Tensor()), key_w = wk.value_or(Tensor()),
                 pos = positions.value_or(Tensor());
    ctx->save_for_backward({q, key, wq, key_w, cos, sin, pos});
    ctx->saved_data["desc"] = std::string(reinterpret_cast<const char*>(&desc), sizeof(desc));
    variable_list out = {at::empty(q.sizes(), q.options())};
    if (key.defined()) out.push_back(at::empty(key.sizes(), q.options()));
    check(zk_qk_norm_rope_fwd(&desc, q.data_ptr(), address(key), wq.data_ptr(), address(key_w),
                              out[0].data_ptr(), key.defined() ? out[1].data_ptr() : nullptr,
                              static_cast<const float*>(cos.data_ptr()),
                              static_cast<const float*>(sin.data_ptr()),
                              static_cast<const int64_t*>(address(pos)), stream_of(q)),
          "zk_qk_norm_rope_fwd");
    return out;
  }

  static variable_list backward(AutogradContext* ctx, variable_list dy) {
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &q = saved[0], &k = saved[1], &wq = saved[2], &wk = saved[3], &cos = saved[4],
                 &sin = saved[5], &pos = saved[6];
    const c10::DeviceGuard on(q.device());
    zk_qk_desc desc;
    std::memcpy(&desc, ctx->saved_data["desc"].toStringRef().data(), sizeof(desc));
    const Tensor gq = rows_of(dy[0]), gk = k.defined() ? rows_of(dy[1]) : Tensor();
    desc.dyq_sb = gq.stride(0), desc.dyq_ss = gq.stride(1), desc.dyq_sh = gq.stride(2);
    if (k.defined()) desc.dyk_sb = gk.stride(0), desc.dyk_ss = gk.stride(1), desc.dyk_sh = gk.stride(2);
    const int64_t bytes = zk_qk_norm_rope_bwd_workspace(desc.d);
    const Tensor dq = at::empty(q.sizes(), q.options()), dwq = at::empty({desc.d}, wq.options());
    const Tensor dk = k.defined() ? at::empty(k.sizes(), k.options()) : Tensor();
    const Tensor dwk = k.defined() ? at::empty({desc.d}, wk.options()) : Tensor();
    const Tensor ws = workspace(bytes, q);
    check(zk_qk_norm_rope_bwd(&desc, q.data_ptr(), address(k), wq.data_ptr(), address(wk),
                              gq.data_ptr(), address(gk), dq.data_ptr(), address(dk), dwq.data_ptr(),
                              address(dwk), static_cast<const float*>(cos.data_ptr()),
                              static_cast<const float*>(sin.data_ptr()),
                              static_cast<const int64_t*>(address(pos)), address(ws), bytes,
                              stream_of(q)),
          "zk_qk_norm_rope_bwd");
    variable_list out = {dq, dk, dwq, dwk, Tensor(), Tensor(), Tensor(), Tensor()};
    if (!at::GradMode::is_enabled() || !(gq.requires_grad() || (gk.defined() && gk.requires_grad())))
      return out;
    // create_graph: what is differentiated once more says so
    for (Tensor& t : out)
      if (t.defined()) t.requires_grad_(true);
    return torch::autograd::DelayedError("qk_norm_rope can be differentiated once", 8)(std::move(out));
  }
};

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

// (device index, rows of 64-bit fields) of a list of tensors: for each the
// addresses of the columns, the elements of the first column's, the integers,
// and the type codes of the columns in `codes`.  A column is (name, tensors,
// mask of type bits, kind): contiguous tensors on one GPU, as large as the first
// column's (kind 0; 1: None is allowed too) or two for each block of them (2).
// `apart`: refuse a first column whose tensors share memory.
py::tuple rows(const std::string& who, const py::tuple& columns, const py::tuple& integers,
               const py::tuple& codes, bool apart) {
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
  std::vector<std::pair<int64_t, int64_t>> spans;
  for (size_t c = 0; c < nc; ++c) {
    const py::tuple column = columns[c].cast<py::tuple>();
    const int64_t mask = column[2].cast<int64_t>(), kind = column[3].cast<int64_t>();
    for (Py_ssize_t i = 0; i < n; ++i) {
      PyObject* o = lists[c].items[i];
      int64_t& field = out[i * fields + c];
      if (kind == 1 && o == Py_None) {
        field = 0;
        continue;
      }
      if (!THPVariable_Check(o)) throw py::type_error(who + ": lists of tensors are needed");
      const Tensor& t = THPVariable_Unpack(o);
      if (!t.is_cuda()) throw py::value_error("zorse_amd kernels need GPU tensors (got a CPU tensor)");
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
      if (c == 0 && apart && want > 0)
        spans.emplace_back(field, field + want * static_cast<int64_t>(t.element_size()));
    }
  }
  std::sort(spans.begin(), spans.end());
  for (size_t i = 1; i < spans.size(); ++i)
    if (spans[i].first < spans[i - 1].second)
      throw py::value_error(who + ": a parameter is in the list twice, or parameters overlap");
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
  m.def("embedding",
        [](const Tensor& ids, const Tensor& weight, double scale, int64_t pad, int64_t y_code) {
          return Embedding::apply(ids, weight, scale, pad, y_code);
        },
        py::call_guard<py::gil_scoped_release>());
  m.def("qk_norm_rope",
        [](const Tensor& q, const MaybeTensor& k, const Tensor& wq, const MaybeTensor& wk,
           const Tensor& cos, const Tensor& sin, const MaybeTensor& positions, int64_t desc) {
          return QkNormRope::apply(q, k, wq, wk, cos, sin, positions,
                                   *reinterpret_cast<const zk_qk_desc*>(desc));
        },
        py::call_guard<py::gil_scoped_release>());
  m.def("rows", &rows);
}
