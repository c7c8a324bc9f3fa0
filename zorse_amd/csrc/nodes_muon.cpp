// The lists of the orthogonal updates on torch's C++ side: checks, tables and the
// launches through the C ABI.
#include <array>

#include "nodes.h"

namespace {

std::vector<MaybeTensor> list_of(const std::string& who, const py::object& o) {
  std::vector<MaybeTensor> out;
  for (const py::handle h : o) {
    if (h.is_none()) {
      out.emplace_back();
      continue;
    }
    if (!THPVariable_Check(h.ptr())) throw py::type_error(who + ": lists of tensors are needed");
    out.emplace_back(THPVariable_Unpack(h.ptr()));
  }
  return out;
}

struct Span {  // of a matrix: bytes, and those of a row and between rows
  uintptr_t begin, end, width, pitch;
  bool written;
};

// A matrix of a list: its row stride, after the checks.
int64_t matrix(const std::string& who, const char* name, size_t i, const Tensor& t, const Tensor& like,
               int types, bool written, std::vector<Span>& spans) {
  if (!t.is_cuda()) bad(kNeedGpu);
  const std::string at = who + ": " + name + " " + std::to_string(i);
  if (t.dim() != 2) bad(at + " must be a matrix");
  if (t.sizes() != like.sizes() || t.get_device() != like.get_device())
    bad(at + " must have its matrix' shape and device");
  const int code = code_of(t.scalar_type());
  if (code < 0 || !(types >> code & 1)) bad(at + (types == 1 << ZK_F32 ? " must be fp32" : " must be fp32, fp16 or bf16"));
  const int64_t rows = t.size(0), cols = t.size(1);
  const int64_t ld = rows > 1 ? t.stride(0) : cols;
  if ((cols > 1 && t.stride(1) != 1) || ld < cols)
    bad(at + " needs unit column stride and rows that do not overlap");
  if (rows > 0 && cols > 0) {
    const uintptr_t p = reinterpret_cast<uintptr_t>(t.data_ptr());
    const uintptr_t e = t.element_size();
    spans.push_back({p, p + ((rows - 1) * ld + cols) * e, cols * e, rows > 1 ? ld * e : 0, written});
  }
  return ld;
}

// Whether matrices whose spans meet, b's beginning in a's, share bytes: columns of one
// buffer, rows equally far apart, lie beside each other.
bool share(const Span& a, const Span& b) {
  const uintptr_t pitch = a.pitch ? a.pitch : b.pitch;
  if (pitch == 0 || (a.pitch && b.pitch && a.pitch != b.pitch)) return true;
  const uintptr_t at = (b.begin - a.begin) % pitch;
  return at < a.width || at + b.width > pitch;
}

void no_overlaps(const std::string& who, std::vector<Span>& spans) {
  std::sort(spans.begin(), spans.end(), [](const Span& a, const Span& b) { return a.begin < b.begin; });
  std::vector<Span> open;  // that end behind the current one's beginning
  for (const Span& s : spans) {
    open.erase(std::remove_if(open.begin(), open.end(), [&](const Span& o) { return o.end <= s.begin; }),
               open.end());
    for (const Span& o : open)
      if ((s.written || o.written) && share(o, s))
        bad(who + ": a tensor that is written is in the lists twice, or overlaps another");
    open.push_back(s);
  }
}

void one_device(const std::string& who, const Tensor& t, const Tensor& first) {
  if (!t.is_cuda()) bad(kNeedGpu);
  if (t.get_device() != first.get_device()) bad(who + ": tensors are on different devices");
}

constexpr int kAnyFloat = 1 << ZK_F32 | 1 << ZK_F16 | 1 << ZK_BF16;

// kernels.orthogonalize
std::vector<Tensor> orthogonalize(const py::object& matrices, const py::object& given_outs,
                                  std::optional<at::ScalarType> dtype, int steps, double a, double b,
                                  double c, double eps) {
  const std::string who = "orthogonalize";
  const std::vector<MaybeTensor> xs = list_of(who, matrices);
  std::vector<MaybeTensor> outs;
  if (!given_outs.is_none()) {
    outs = list_of(who, given_outs);
    if (outs.size() != xs.size()) bad(who + ": the lists differ in length");
  }
  std::vector<Tensor> result;
  std::vector<zk_muon_matrix> table;
  std::vector<Span> spans;
  for (size_t i = 0; i < xs.size(); ++i) {
    if (!xs[i]) bad(who + ": matrix " + std::to_string(i) + " is None");
    const Tensor& x = *xs[i];
    zk_muon_matrix m{};
    m.ld_grad = matrix(who, "matrix", i, x, x, kAnyFloat, false, spans);
    one_device(who, x, *xs[0]);
    m.grad = x.data_ptr();
    m.rows = x.size(0), m.cols = x.size(1);
    m.grad_dtype = code_of(x.scalar_type());
    Tensor out;
    if (!outs.empty()) {
      if (!outs[i]) bad(who + ": out " + std::to_string(i) + " is None");
      out = *outs[i];
      if (dtype && out.scalar_type() != *dtype) bad(who + ": outs are not of dtype");
    } else {
      const at::ScalarType type = dtype.value_or(x.scalar_type());
      float_code("output", type);
      const c10::DeviceGuard on(x.device());
      out = at::empty(x.sizes(), x.options().dtype(type));
    }
    m.ld_out = matrix(who, "out", i, out, x, kAnyFloat, true, spans);
    m.out = out.data_ptr();
    m.out_dtype = code_of(out.scalar_type());
    result.push_back(out);
    if (x.numel() > 0) table.push_back(m);
  }
  no_overlaps(who, spans);
  const int64_t n = static_cast<int64_t>(table.size());
  const py::gil_scoped_release free_gil;
  std::optional<c10::DeviceGuard> on;
  Tensor ws;
  zk_stream_t stream = nullptr;
  int64_t bytes = 0;
  if (n > 0) {
    on.emplace(result[0].device());
    bytes = zk_muon_workspace(table.data(), n);  // it goes by the device's CUs
    ws = workspace(bytes, result[0]);
    stream = stream_of(result[0]);
  }
  check(zk_orthogonalize(table.data(), n, steps, a, b, c, eps, address(ws), bytes, stream), "zk_orthogonalize");
  return result;
}

// kernels.muon_step: a step whose arguments are checked and whose workspace is there,
// so that run() refuses nothing.
class MuonStep {
 public:
  MuonStep(const py::object& params_, const py::object& grads_, const py::object& momenta_, const py::object& lows_,
           int steps, double a, double b, double c, double eps, double lr, double momentum, double weight_decay,
           bool nesterov, bool match_rms)
      : steps_(steps), nesterov_(nesterov), adjust_(match_rms ? ZK_MUON_MATCH_RMS : ZK_MUON_ORIGINAL),
        hyper_{a, b, c, eps, lr, momentum, weight_decay} {
    const std::string who = "muon_multi";
    std::vector<MaybeTensor> params = list_of(who, params_), grads = list_of(who, grads_),
                             momenta = list_of(who, momenta_), lows(params.size());
    if (!lows_.is_none()) lows = list_of(who, lows_);
    if (grads.size() != params.size() || momenta.size() != params.size() || lows.size() != params.size())
      bad(who + ": the lists differ in length");
    std::vector<Span> spans;
    for (size_t i = 0; i < params.size(); ++i) {
      if (!params[i] || !grads[i] || !momenta[i]) bad(who + ": tensor " + std::to_string(i) + " is None");
      const Tensor& p = *params[i];
      zk_muon_matrix m{};
      m.ld_param = matrix(who, "param", i, p, p, 1 << ZK_F32, true, spans);
      one_device(who, p, *params[0]);
      m.ld_grad = matrix(who, "grad", i, *grads[i], p, kAnyFloat, false, spans);
      m.ld_momentum = matrix(who, "momentum", i, *momenta[i], p, 1 << ZK_F32, true, spans);
      m.param = static_cast<float*>(p.data_ptr());
      m.grad = grads[i]->data_ptr();
      m.momentum = static_cast<float*>(momenta[i]->data_ptr());
      m.rows = p.size(0), m.cols = p.size(1);
      m.grad_dtype = code_of(grads[i]->scalar_type());
      if (lows[i]) {
        m.ld_out = matrix(who, "lowp_out", i, *lows[i], p, kAnyFloat, true, spans);
        m.out = lows[i]->data_ptr();
        m.out_dtype = code_of(lows[i]->scalar_type());
      }
      if (p.numel() > 0) table_.push_back(m);
    }
    no_overlaps(who, spans);
    for (std::vector<MaybeTensor>* list : {&params, &grads, &momenta, &lows})
      for (const MaybeTensor& t : *list)
        if (t) kept_.push_back(*t);
    const py::gil_scoped_release free_gil;
    std::optional<c10::DeviceGuard> on;
    if (!table_.empty()) on.emplace(kept_[0].device());
    const int status = call(nullptr, 0, nullptr);  // with no workspace: all other checks
    if (status != ZK_EWORKSPACE) check(status, "zk_muon_multi");
    if (table_.empty()) return;
    bytes_ = zk_muon_workspace(table_.data(), static_cast<int64_t>(table_.size()));
    ws_ = workspace(bytes_, kept_[0]);
  }

  void run() {
    if (table_.empty()) return;
    const py::gil_scoped_release free_gil;
    const c10::DeviceGuard on(ws_.device());
    check(call(ws_.data_ptr(), bytes_, stream_of(ws_)), "zk_muon_multi");
  }

 private:
  int call(void* ws, int64_t bytes, zk_stream_t stream) const {
    const auto& [a, b, c, eps, lr, momentum, weight_decay] = hyper_;
    return zk_muon_multi(table_.data(), static_cast<int64_t>(table_.size()), steps_, a, b, c, eps, lr, momentum,
                         weight_decay, nesterov_, adjust_, ws, bytes, stream);
  }

  int steps_, nesterov_, adjust_;
  std::array<double, 7> hyper_;
  std::vector<zk_muon_matrix> table_;
  std::vector<Tensor> kept_;
  Tensor ws_;
  int64_t bytes_ = 0;
};

}  // namespace

void bind_muon(py::module_& m) {
  m.def("orthogonalize", &orthogonalize);
  py::class_<MuonStep>(m, "MuonStep")
      .def(py::init<const py::object&, const py::object&, const py::object&, const py::object&, int, double, double,
                    double, double, double, double, double, bool, bool>())
      .def("run", &MuonStep::run);
}
