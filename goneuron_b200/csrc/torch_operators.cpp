// torch_operators.cpp -- the operators on device memory for torch tensors: checks of the arguments, outputs and workspaces from torch's allocator, the current stream, one call of the C ABI.
//
// Only goneuron_b200/operators.py calls this module.  It is compiled because a decoding step's kernel takes less time than the same checks in Python: norm of queries and keys for five
// tokens, 21 us a call with ctypes.  Wrong arguments are ValueError, a status of the library is raised as the class that operators.py registers.
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/pybind.h>
#include <torch/types.h>

#include <optional>
#include <string>
#include <tuple>

#include "../../include/goneuron_cuda.h"

namespace py = pybind11;
using at::Tensor;
using OptTensor = std::optional<Tensor>;

namespace {

py::object* error_class = nullptr;      // GoNeuronCudaError(code, message); lives until the process ends

[[noreturn]] void wrong(const std::string& what) { throw py::value_error(what); }
void check(int rc) {
  if (rc == GN_OK) return;
  py::object e = (*error_class)(rc, std::string(gn_last_error()));
  PyErr_SetObject(error_class->ptr(), e.ptr());
  throw py::error_already_set();
}
std::string shape_of(const Tensor& t) { std::string s = "("; for (auto n : t.sizes()) s += std::to_string(n) + ", "; return s + ")"; }

// A context and its GPU, as a Python Device holds them.
struct Dev { gn_ctx* ctx; int index; void* stream() const { return c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)index).stream(); } };
Dev dev_of(uint64_t handle, int index) { return Dev{reinterpret_cast<gn_ctx*>(handle), index}; }
void here(const Dev& d, const char* name, const Tensor& t) {
  if (!t.is_cuda() || t.get_device() != d.index) wrong(std::string(name) + " is on " + t.device().str() + ", the operator runs on cuda:" + std::to_string(d.index));
}
int dtype_of(const char* name, const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return GN_F32;
    case at::kHalf: return GN_F16;
    case at::kBFloat16: return GN_BF16;
    default: wrong(std::string(name) + " is " + c10::toString(t.scalar_type()) + ": float32, float16 or bfloat16 is needed");
  }
}
// of a floating type (of that of `like`, and its shape), with a contiguous last dimension
void floating(const char* name, const Tensor& t, const Tensor* like = nullptr) {
  dtype_of(name, t);
  if (like && t.scalar_type() != like->scalar_type()) wrong(std::string(name) + " is " + c10::toString(t.scalar_type()) + ", " + c10::toString(like->scalar_type()) + " is needed");
  if (like && !t.sizes().equals(like->sizes())) wrong(std::string(name) + " has shape " + shape_of(t) + ", " + shape_of(*like) + " is needed");
  if (t.dim() == 0 || (t.stride(-1) != 1 && t.size(-1) > 1 && t.numel())) wrong("the last dimension of " + std::string(name) + " is not contiguous");
}
// contiguous, of this type and shape (-1: any)
void dense(const char* name, const Tensor& t, at::ScalarType type, std::initializer_list<int64_t> shape) {
  bool ok = t.scalar_type() == type && t.is_contiguous() && t.dim() == (int64_t)shape.size();
  if (ok) { int64_t i = 0; for (int64_t n : shape) { if (n >= 0 && t.size(i) != n) ok = false; i++; } }
  if (ok) return;
  std::string s = "("; for (int64_t n : shape) s += n < 0 ? "any, " : std::to_string(n) + ", ";
  wrong(std::string(name) + " is " + c10::toString(t.scalar_type()) + " of shape " + shape_of(t) + (t.is_contiguous() ? "" : ", not contiguous") + "; contiguous " + c10::toString(type) + " of shape " + s + ") is needed");
}
int index_type(const char* name, const Tensor& t) {
  if (t.scalar_type() != at::kInt && t.scalar_type() != at::kLong) wrong(std::string(name) + " is " + c10::toString(t.scalar_type()) + ": int32 or int64 is needed");
  if (!t.is_contiguous()) wrong(std::string(name) + " is not contiguous");
  return t.scalar_type() == at::kLong ? GN_I64 : GN_I32;
}
void* ptr(const Tensor& t) { return t.numel() ? t.data_ptr() : nullptr; }
void* ptr(const OptTensor& t) { return t ? ptr(*t) : nullptr; }
// [tokens, dim] of a tensor [..., dim]: the distance of its rows
struct Rows { int64_t n, dim, stride; };
Rows rows(const char* name, const Tensor& t, const Tensor* like = nullptr) {
  floating(name, t, like);
  const int64_t d = t.dim(), dim = t.size(-1); int64_t n = 1, stride = dim, expect = -1;
  if (t.numel() == 0) { for (int64_t i = 0; i + 1 < d; i++) n *= t.size(i); return Rows{dim ? n : 0, dim, dim}; }
  for (int64_t i = d - 2; i >= 0; i--) {                             // dimensions of one element do not count; each other one has to continue the ones behind it
    if (t.size(i) == 1) continue;
    if (expect < 0) stride = t.stride(i); else if (t.stride(i) != expect) wrong(std::string(name) + ": the strides of its first dimensions do not make one of tokens");
    n *= t.size(i); expect = stride * n;
  }
  return Rows{n, dim, stride};
}
// A tensor of the caller's that is written.  What autograd knows of it would not be true any more; what kept it for a backward pass notices by its version.
void writable(const char* name, const Tensor& t) {
  if (at::GradMode::is_enabled() && t.requires_grad()) wrong(std::string(name) + " requires a gradient and would be overwritten: call under torch.no_grad(), or give another tensor");
  if (t.is_inference() && !c10::InferenceMode::is_enabled()) wrong(std::string(name) + " was made in inference mode and can only be written there");
}
void written(const Tensor& t) { t.unsafeGetTensorImpl()->bump_version(); }
Tensor empty(const Tensor& like, at::IntArrayRef shape) { return at::empty(shape, like.options()); }
Tensor empty(const Tensor& like, at::IntArrayRef shape, at::ScalarType type) { return at::empty(shape, like.options().dtype(type)); }
Tensor bytes(const Tensor& like, int64_t n) { return at::empty({n}, like.options().dtype(at::kByte)); }

// ------------------------------------------------------------------ norm of queries and keys with the rotation
// [tokens, heads, size] or [batch, tokens, heads, size] as tokens, without copying
int64_t heads_of(const char* name, const Tensor& t, gn_heads* h, const Tensor* like = nullptr) {
  floating(name, t, like);
  const int64_t d = t.dim();
  if (d != 3 && d != 4) wrong(std::string(name) + " has shape " + shape_of(t) + ": [tokens, heads, size] or [batch, tokens, heads, size] is needed");
  int64_t n = t.size(d - 3), stride = t.stride(d - 3);
  if (d == 4) {
    if (t.size(0) != 1 && t.numel()) {
      if (n == 1) stride = t.stride(0); else if (t.stride(0) != stride * n) wrong(std::string(name) + ": the strides of its first two dimensions do not make one of tokens");
    }
    n *= t.size(0);
  }
  if (t.size(d - 2) > INT32_MAX || t.size(d - 1) > INT32_MAX) wrong(std::string(name) + " has too many heads");
  *h = gn_heads{ptr(t), stride, t.stride(d - 2), (int32_t)t.size(d - 2), 0};
  return n;
}
struct Qk {
  Dev d; int dtype, rotated = 0, wide = 0; int64_t n, size; gn_heads q{}, k{}; bool keys; float *gain_q, *gain_k; void* positions = nullptr; double* frequencies = nullptr;
  Qk(const Dev& dev, const Tensor& qt, const OptTensor& kt, const OptTensor& gq, const OptTensor& gk, const OptTensor& pos, const OptTensor& freq) : d(dev), keys(kt.has_value()) {
    n = heads_of("q", qt, &q); size = qt.size(-1); dtype = dtype_of("q", qt);
    if (keys && (heads_of("k", *kt, &k) != n || kt->scalar_type() != qt.scalar_type() || kt->size(-1) != size)) wrong("q and k differ in type, tokens or head size");
    if (gq) dense("gain_q", *gq, at::kFloat, {size});
    if (gk) dense("gain_k", *gk, at::kFloat, {size});
    if (freq) {
      dense("frequencies", *freq, at::kDouble, {-1});
      if (!pos) wrong("positions are needed for a rotation");
      wide = index_type("positions", *pos);
      if (pos->numel() != n) wrong("positions: one for each token is needed");
      if (freq->size(0) > INT32_MAX / 2) wrong("frequencies: more than half a head");
      rotated = (int)(2 * freq->size(0)); positions = ptr(*pos); frequencies = (double*)ptr(*freq);
      here(d, "positions", *pos); here(d, "frequencies", *freq);
    }
    gain_q = (float*)ptr(gq); gain_k = (float*)ptr(gk);
    here(d, "q", qt);
    if (kt) here(d, "k", *kt);
    if (gq) here(d, "gain_q", *gq);
    if (gk) here(d, "gain_k", *gk);
  }
  const gn_heads* key(const gn_heads& h) const { return keys ? &h : nullptr; }
};

std::tuple<Tensor, OptTensor> qk_norm_rope(uint64_t handle, int index, const Tensor& q, const OptTensor& k, const OptTensor& gain_q, const OptTensor& gain_k, const OptTensor& positions, const OptTensor& frequencies,
                                           double eps, bool interleaved, const OptTensor& q_out, const OptTensor& k_out) {
  const Qk a(dev_of(handle, index), q, k, gain_q, gain_k, positions, frequencies);
  if (q_out && k && !k_out) wrong("out: a pair of tensors is needed");
  gn_heads qo{}, ko{};
  Tensor qt = q_out ? *q_out : empty(q, q.sizes()); OptTensor kt;
  heads_of("out[0]", qt, &qo, &q); writable("out[0]", qt); here(a.d, "out[0]", qt);
  if (k) { kt = k_out ? *k_out : empty(*k, k->sizes()); heads_of("out[1]", *kt, &ko, &*k); writable("out[1]", *kt); here(a.d, "out[1]", *kt); }
  check(gn_op_qk_norm_rope(a.d.ctx, a.dtype, a.n, (int)a.size, a.rotated, interleaved, (float)eps, &a.q, a.key(a.k), a.gain_q, a.gain_k, a.positions, a.wide, a.frequencies, &qo, a.key(ko), a.d.stream()));
  if (q_out) written(*q_out);
  if (k && k_out) written(*k_out);
  return {qt, kt};
}

std::tuple<Tensor, OptTensor, OptTensor, OptTensor> qk_norm_rope_backward(uint64_t handle, int index, const Tensor& dq_out, const OptTensor& dk_out, const Tensor& q, const OptTensor& k, const OptTensor& gain_q,
                                                                          const OptTensor& gain_k, const OptTensor& positions, const OptTensor& frequencies, double eps, bool interleaved) {
  const Qk a(dev_of(handle, index), q, k, gain_q, gain_k, positions, frequencies);
  gn_heads dqo{}, dko{}, dqh{}, dkh{};
  heads_of("dq_out", dq_out, &dqo, &q); here(a.d, "dq_out", dq_out);
  if (k) { if (!dk_out) wrong("dk_out is needed"); heads_of("dk_out", *dk_out, &dko, &*k); here(a.d, "dk_out", *dk_out); }
  Tensor dq = empty(q, q.sizes()), ws; OptTensor dk, dgq, dgk;
  heads_of("dq", dq, &dqh);
  if (k) { dk = empty(*k, k->sizes()); heads_of("dk", *dk, &dkh); }
  if (gain_q) dgq = empty(*gain_q, {a.size});
  if (gain_k && k) dgk = empty(*gain_k, {a.size});
  int64_t n = 0;
  if (dgq || dgk) { check(gn_op_qk_norm_rope_workspace(a.d.ctx, a.n, a.q.heads, a.k.heads, (int)a.size, &n)); ws = bytes(q, n); }
  check(gn_op_qk_norm_rope_backward(a.d.ctx, a.dtype, a.n, (int)a.size, a.rotated, interleaved, (float)eps, &a.q, a.key(a.k), a.gain_q, a.gain_k, a.positions, a.wide, a.frequencies, &dqo, a.key(dko), &dqh, a.key(dkh),
                                    (float*)ptr(dgq), (float*)ptr(dgk), n ? ptr(ws) : nullptr, n, a.d.stream()));
  return {dq, dk, dgq, dgk};
}

// ------------------------------------------------------------------ distillation
std::tuple<Tensor, OptTensor> distill(uint64_t handle, int index, const Tensor& logits, const Tensor& top_ids, const Tensor& top_logits, double temperature, const OptTensor& row_weight, bool gradient, const OptTensor& out) {
  const Dev d = dev_of(handle, index);
  floating("logits", logits);
  if (logits.dim() != 2) wrong("logits has shape " + shape_of(logits) + ": [rows, vocabulary] is needed");
  const int64_t n = logits.size(0), vocab = logits.size(1); const int wide = index_type("top_ids", top_ids);
  dense("top_logits", top_logits, at::kFloat, {n, -1});
  if (!top_ids.sizes().equals(top_logits.sizes())) wrong("top_ids has shape " + shape_of(top_ids) + ", top_logits " + shape_of(top_logits));
  if (top_ids.size(1) > INT32_MAX) wrong("top_ids has too many columns");
  if (row_weight) { dense("row_weight", *row_weight, at::kFloat, {n}); }
  if (out) { floating("out", *out, &logits); writable("out", *out); }
  here(d, "logits", logits); here(d, "top_ids", top_ids); here(d, "top_logits", top_logits);
  if (row_weight) here(d, "row_weight", *row_weight);
  if (out) here(d, "out", *out);
  const int top = (int)top_ids.size(1);
  Tensor loss = empty(top_logits, {n}); OptTensor grad;
  if (gradient) grad = out ? *out : empty(logits, logits.sizes());
  check(gn_op_distill(d.ctx, dtype_of("logits", logits), n, vocab, top, (float)temperature, ptr(logits), logits.stride(0), ptr(top_ids), wide, (float*)ptr(top_logits), (float*)ptr(row_weight), (float*)ptr(loss), ptr(grad),
                      gradient ? grad->stride(0) : 0, d.stream()));
  if (out) written(*out);
  return {loss, grad};
}

// ------------------------------------------------------------------ embedding
Tensor embedding(uint64_t handle, int index, const Tensor& table, const Tensor& ids, double scale) {
  const Dev d = dev_of(handle, index);
  floating("table", table);
  if (table.dim() != 2 || table.size(1) > INT32_MAX) wrong("table has shape " + shape_of(table) + ": [vocab, dim] is needed");
  const int wide = index_type("ids", ids);
  here(d, "table", table); here(d, "ids", ids);
  std::vector<int64_t> shape(ids.sizes().begin(), ids.sizes().end()); shape.push_back(table.size(1));
  Tensor out = empty(table, shape);
  check(gn_op_embedding(d.ctx, dtype_of("table", table), ids.numel(), table.size(0), (int)table.size(1), (float)scale, ptr(table), table.stride(0), ptr(ids), wide, ptr(out), table.size(1), d.stream()));
  return out;
}

Tensor embedding_backward(uint64_t handle, int index, const Tensor& dout, const Tensor& ids, int64_t vocab, double scale) {
  const Dev d = dev_of(handle, index);
  const int wide = index_type("ids", ids); const Rows r = rows("dout", dout);
  if (!dout.sizes().slice(0, dout.dim() - 1).equals(ids.sizes()) || r.dim > INT32_MAX) wrong("dout has shape " + shape_of(dout) + ": a row for each id is needed");
  if (vocab < 0) wrong("vocab is negative");
  here(d, "ids", ids); here(d, "dout", dout);
  Tensor dtable = empty(dout, {vocab, r.dim}, at::kFloat);
  int64_t need = 0;
  check(gn_op_embedding_workspace(d.ctx, ids.numel(), vocab, (int)r.dim, &need));
  Tensor ws = bytes(dout, need);
  check(gn_op_embedding_backward(d.ctx, dtype_of("dout", dout), ids.numel(), vocab, (int)r.dim, (float)scale, ptr(dout), r.stride, ptr(ids), wide, (float*)ptr(dtable), ptr(ws), need, d.stream()));
  return dtable;
}

// ------------------------------------------------------------------ gated feed-forward block
struct Ffn {
  Dev d; Rows x; int dim, ff, dtype;
  Ffn(const Dev& dev, const Tensor& xt, const Tensor& wg, const Tensor& wu, const Tensor& wd) : d(dev), x(rows("x", xt)), dtype(dtype_of("x", xt)) {
    if (dtype == GN_F32) wrong("x is float32: float16 or bfloat16 is needed, there is no 32-bit form");
    dense("w_gate", wg, xt.scalar_type(), {-1, x.dim});
    const int64_t f = wg.size(0);
    dense("w_up", wu, xt.scalar_type(), {f, x.dim}); dense("w_down", wd, xt.scalar_type(), {x.dim, f});
    if (f > INT32_MAX || x.dim > INT32_MAX) wrong("the weights are too large");
    here(d, "x", xt); here(d, "w_gate", wg); here(d, "w_up", wu); here(d, "w_down", wd);
    dim = (int)x.dim; ff = (int)f;
  }
};

std::tuple<Tensor, OptTensor> gated_ffn(uint64_t handle, int index, const Tensor& x, const Tensor& w_gate, const Tensor& w_up, const Tensor& w_down, int activation, bool save) {
  const Ffn a(dev_of(handle, index), x, w_gate, w_up, w_down);
  int64_t need = 0, keep = 0;
  check(gn_op_gated_ffn_workspace(a.d.ctx, a.x.n, a.dim, a.ff, 0, &need));
  if (save) check(gn_op_gated_ffn_saved(a.d.ctx, a.x.n, a.dim, a.ff, &keep));
  Tensor y = empty(x, x.sizes()), ws = bytes(x, need); OptTensor saved;
  if (save) saved = bytes(x, keep);
  check(gn_op_gated_ffn(a.d.ctx, a.dtype, activation, a.x.n, a.dim, a.ff, ptr(x), a.x.stride, ptr(w_gate), ptr(w_up), ptr(w_down), ptr(y), a.dim, ptr(saved), ptr(ws), need, a.d.stream()));
  return {y, saved};
}

std::tuple<Tensor, Tensor, Tensor, Tensor> gated_ffn_backward(uint64_t handle, int index, const Tensor& dy, const Tensor& x, const Tensor& w_gate, const Tensor& w_up, const Tensor& w_down, const Tensor& saved, int activation) {
  const Ffn a(dev_of(handle, index), x, w_gate, w_up, w_down); const Rows r = rows("dy", dy, &x);
  here(a.d, "dy", dy);
  int64_t need = 0, keep = 0;
  check(gn_op_gated_ffn_saved(a.d.ctx, a.x.n, a.dim, a.ff, &keep));
  dense("saved", saved, at::kByte, {keep}); here(a.d, "saved", saved);
  check(gn_op_gated_ffn_workspace(a.d.ctx, a.x.n, a.dim, a.ff, 1, &need));
  Tensor dx = empty(x, x.sizes()), dwg = empty(w_gate, {a.ff, a.dim}), dwu = empty(w_gate, {a.ff, a.dim}), dwd = empty(w_gate, {a.dim, a.ff}), ws = bytes(x, need);
  check(gn_op_gated_ffn_backward(a.d.ctx, a.dtype, activation, a.x.n, a.dim, a.ff, ptr(dy), r.stride, ptr(x), a.x.stride, ptr(w_gate), ptr(w_up), ptr(w_down), ptr(saved), ptr(dx), a.dim, ptr(dwg), ptr(dwu), ptr(dwd), ptr(ws),
                                 need, a.d.stream()));
  return {dx, dwg, dwu, dwd};
}

void status(uint64_t handle, int index) { const Dev d = dev_of(handle, index); int rc; { void* s = d.stream(); py::gil_scoped_release free; rc = gn_op_status(d.ctx, s); } check(rc); }

}  // namespace

PYBIND11_MODULE(_torch_operators, m) {
  m.def("set_error", [](py::object c) { error_class = new py::object(std::move(c)); });
  m.def("status", &status);
  m.def("qk_norm_rope", &qk_norm_rope);
  m.def("qk_norm_rope_backward", &qk_norm_rope_backward);
  m.def("distill", &distill);
  m.def("embedding", &embedding);
  m.def("embedding_backward", &embedding_backward);
  m.def("gated_ffn", &gated_ffn);
  m.def("gated_ffn_backward", &gated_ffn_backward);
}
