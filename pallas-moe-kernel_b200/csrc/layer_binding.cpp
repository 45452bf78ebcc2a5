// CPython binding of the layer-training entry points (module
// moe_layer_native): argument checks, outputs, workspaces, and the calls into
// libmoe_b200.so, whose function addresses src/_lib.py hands over once.
//
// The other entry points go through ctypes, which costs a call 5 us and more
// on top of its outputs (argument by argument, and each torch.empty from
// Python 2 us).  The calls here come several to a layer and step and are
// themselves 5 to 10 us of GPU work on small batches.
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <sstream>
#include <string>
#include <unordered_map>
#include <vector>

#include "../../include/moe_b200.h"

namespace {

// ---------------------------------------------------------------- the library
decltype(&moe_route_train_workspace_size) p_route_space;
decltype(&moe_route_train_counters) p_route_counters;
decltype(&moe_route_train) p_route_train;
decltype(&moe_route_backward) p_route_backward;
decltype(&moe_combine_rows_backward) p_combine;
decltype(&moe_gather_rows_backward) p_gather;
decltype(&moe_grad_norm_workspace_size) p_norm_space;
decltype(&moe_grad_norm) p_norm;
decltype(&moe_clip_grads) p_clip;
decltype(&moe_last_error) p_error;
PyObject* g_moe_error = nullptr;  // src._lib.MoeError

void check(int rc) {
  if (rc == 0) return;
  PyObject* e = PyObject_CallFunction(g_moe_error, "is", rc, p_error());
  if (e) {
    PyErr_SetObject(g_moe_error, e);
    Py_DECREF(e);
  }
  throw python_error();
}

// ---------------------------------------------------------------- arguments
const at::Tensor& tensor(PyObject* o, const char* name) {
  TORCH_CHECK_TYPE(THPVariable_Check(o), name, " must be a tensor, not ", Py_TYPE(o)->tp_name);
  return THPVariable_Unpack(o);
}
c10::optional<at::Tensor> maybe(PyObject* o, const char* name) {
  if (o == Py_None) return c10::nullopt;
  return tensor(o, name);
}
int64_t integer(PyObject* o) {
  const int64_t v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw python_error();
  return v;
}
bool truth(PyObject* o) {
  const int v = PyObject_IsTrue(o);
  if (v < 0) throw python_error();
  return v != 0;
}
int elem(const at::Tensor& t, const char* name) {
  switch (t.scalar_type()) {
    case at::kFloat: return MOE_ELEM_F32;
    case at::kBFloat16: return MOE_ELEM_BF16;
    case at::kHalf: return MOE_ELEM_F16;
    default: break;
  }
  TORCH_CHECK_TYPE(false, name, " is ", t.scalar_type(), " (float32, bfloat16 or float16)");
}
at::ScalarType elem_type(int code) {
  return code == MOE_ELEM_F32 ? at::kFloat : code == MOE_ELEM_BF16 ? at::kBFloat16 : at::kHalf;
}
void on(const at::Device& dev, const at::Tensor& t, const char* name) {
  TORCH_CHECK_VALUE(t.device() == dev, name, " is on ", t.device(), ", the other operands on ", dev);
}
bool shaped(const at::Tensor& t, int64_t a, int64_t b) { return t.dim() == 2 && t.size(0) == a && t.size(1) == b; }

at::Tensor empty(at::IntArrayRef size, at::ScalarType type, const at::Device& dev) {
  return at::detail::empty_cuda(size, type, dev, c10::nullopt);
}
template <class T = void>
const T* ptr(const c10::optional<at::Tensor>& t) {
  return t ? static_cast<const T*>(t->data_ptr()) : nullptr;
}

// ---------------------------------------------------------------- workspaces
// A workspace shared by the calls of one stream (they run in its order); above
// 64 MiB, and for what a CUDA graph captures, a fresh one.  The map outlives
// the module on purpose: its tensors must not be freed after the driver.
using StreamTensors = std::unordered_map<uint64_t, at::Tensor>;
uint64_t stream_key(const at::Device& dev, cudaStream_t s) {
  return reinterpret_cast<uint64_t>(s) * 64 + (uint64_t)dev.index();
}
bool capturing() {
  return c10::cuda::currentStreamCaptureStatusMayInitCtx() != c10::cuda::CaptureStatus::None;
}
at::Tensor workspace(const at::Device& dev, cudaStream_t s, size_t bytes, bool fresh) {
  static StreamTensors& cache = *new StreamTensors;
  if (fresh || bytes > ((size_t)64 << 20)) return empty({(int64_t)bytes}, at::kByte, dev);
  at::Tensor& w = cache[stream_key(dev, s)];
  if (!w.defined() || (size_t)w.numel() < bytes) w = empty({(int64_t)bytes}, at::kByte, dev);
  return w;
}
// Counters that are zero between the calls of one stream (each call leaves
// them so); a captured call's are set to zero at every replay.
at::Tensor counters(const at::Device& dev, cudaStream_t s, int64_t n, bool fresh) {
  static StreamTensors& cache = *new StreamTensors;
  if (fresh) return empty({n}, at::kInt, dev).zero_();
  at::Tensor& c = cache[stream_key(dev, s)];
  if (!c.defined() || c.numel() < n) c = empty({std::max<int64_t>(n, 1024)}, at::kInt, dev).zero_();
  return c;
}

// ---------------------------------------------------------------- routing
struct Route {
  at::Tensor logits;
  c10::optional<at::Tensor> mask;
  int64_t T, E, ld, sequences;
  int type;
};
Route route(PyObject* logits, PyObject* mask, PyObject* sequences) {
  Route r;
  const at::Tensor& x = tensor(logits, "logits");
  TORCH_CHECK_VALUE(x.is_cuda() && x.dim() == 2, "logits must be a 2-D CUDA tensor");
  r.type = elem(x, "logits");
  r.T = x.size(0);
  r.E = x.size(1);
  r.logits = (r.E > 1 && x.stride(1) != 1) || (r.T > 1 && x.stride(0) < r.E) ? x.contiguous() : x;
  r.ld = r.T > 1 ? r.logits.stride(0) : r.E;
  r.sequences = integer(sequences);
  TORCH_CHECK_VALUE(r.sequences >= 1 && r.T % r.sequences == 0, r.T, " tokens are not ", r.sequences,
                    " sequences of equal length");
  r.mask = maybe(mask, "mask");
  if (r.mask) {
    TORCH_CHECK_VALUE(r.mask->scalar_type() == at::kBool && r.mask->numel() == r.T,
                      "mask must be a bool tensor with one value per token (", r.T, ")");
    on(x.device(), *r.mask, "mask");
    r.mask = r.mask->contiguous();
  }
  return r;
}

// (logits, k, ids, mask, sequences, scoring, normalize, workspace)
PyObject* route_forward(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n == 8, "route_forward takes 8 arguments");
  at::AutoDispatchBelowADInplaceOrView below;
  const Route r = route(a[0], a[3], a[4]);
  const at::Device dev = r.logits.device();
  const int64_t k = integer(a[1]);
  c10::optional<at::Tensor> ids = maybe(a[2], "ids");
  if (ids) {
    TORCH_CHECK_VALUE(shaped(*ids, r.T, k), "ids is ", ids->sizes(), ", expected [", r.T, ", ", k, "]");
    on(dev, *ids, "ids");
    TORCH_CHECK_TYPE(at::isIntegralType(ids->scalar_type(), false), "ids are ", ids->scalar_type(), ", not integers");
    // Far values stay out of range in 32 bits (as int64, those of uint64 are far or negative).
    if (ids->element_size() == 8) ids = ids->to(at::kLong).clamp(-1, r.E);
    ids = ids->to(at::kInt).contiguous();
  }
  TORCH_CHECK_VALUE(1 <= k && k <= 16 && k <= r.E && r.E <= 1024, "k=", k, ", E=", r.E,
                    ": 1 <= k <= min(16, E) and E <= 1024 are supported");
  const c10::cuda::CUDAGuard guard(dev);
  const cudaStream_t stream = c10::cuda::getCurrentCUDAStream(dev.index());
  const bool fresh = capturing();
  const at::Tensor o[6] = {empty({r.T, k}, at::kInt, dev),          empty({r.T, k}, at::kFloat, dev),
                           empty({r.sequences, r.E}, at::kInt, dev), empty({r.sequences}, at::kInt, dev),
                           empty({}, at::kFloat, dev),               empty({}, at::kFloat, dev)};
  const size_t need = p_route_space(r.T, (int32_t)r.E, r.sequences);
  const c10::optional<at::Tensor> given = maybe(a[7], "workspace");
  const at::Tensor ws = given && given->is_cuda() && given->device() == dev && given->is_contiguous() &&
                                given->nbytes() >= need
                            ? *given
                            : workspace(dev, stream, need, fresh);
  const at::Tensor cnt = counters(dev, stream, p_route_counters(r.T, (int32_t)r.E, r.sequences), fresh);
  check(p_route_train(r.logits.data_ptr(), r.type, r.ld, r.T, (int32_t)r.E, (int32_t)k, r.sequences,
                      ptr<uint8_t>(r.mask), ptr<int32_t>(ids), (int32_t)integer(a[5]), truth(a[6]),
                      o[0].data_ptr<int32_t>(), o[1].data_ptr<float>(), o[2].data_ptr<int32_t>(),
                      o[3].data_ptr<int32_t>(), o[4].data_ptr<float>(), o[5].data_ptr<float>(), ws.data_ptr(), need,
                      reinterpret_cast<uint32_t*>(cnt.data_ptr()), stream));
  PyObject* out = PyTuple_New(6);
  if (!out) throw python_error();
  for (int i = 0; i < 6; ++i) PyTuple_SET_ITEM(out, i, THPVariable_Wrap(o[i]));
  return out;
  END_HANDLE_TH_ERRORS
}

// (logits, ids, weights, counts, tokens, d_weights, d_balance, d_z, mask, sequences, scoring, normalize)
PyObject* route_backward(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n == 12, "route_backward takes 12 arguments");
  at::AutoDispatchBelowADInplaceOrView below;
  const Route r = route(a[0], a[8], a[9]);
  const at::Device dev = r.logits.device();
  const at::Tensor &ids = tensor(a[1], "ids"), &weights = tensor(a[2], "weights"), &counts = tensor(a[3], "counts"),
                   &tokens = tensor(a[4], "tokens");
  const int64_t k = ids.dim() == 2 ? ids.size(1) : -1;
  TORCH_CHECK_VALUE(shaped(ids, r.T, k) && shaped(weights, r.T, k) && shaped(counts, r.sequences, r.E) &&
                        tokens.dim() == 1 && tokens.size(0) == r.sequences && ids.device() == dev &&
                        weights.device() == dev && counts.device() == dev && tokens.device() == dev,
                    "routed has ids ", ids.sizes(), ", weights ", weights.sizes(), ", counts ", counts.sizes(),
                    " and tokens ", tokens.sizes(), " on ", ids.device(), ", expected those of ", r.T, " tokens, ", r.E,
                    " experts and ", r.sequences, " sequences on ", dev);
  TORCH_CHECK_TYPE(ids.scalar_type() == at::kInt && weights.scalar_type() == at::kFloat &&
                       counts.scalar_type() == at::kInt && tokens.scalar_type() == at::kInt && ids.is_contiguous() &&
                       weights.is_contiguous() && counts.is_contiguous() && tokens.is_contiguous(),
                   "routed's tensors must be as route_forward_train returns them: int32 and float32, contiguous");
  c10::optional<at::Tensor> dw = maybe(a[5], "d_weights"), db = maybe(a[6], "d_balance"), dz = maybe(a[7], "d_z");
  if (dw) {
    TORCH_CHECK_VALUE(shaped(*dw, r.T, k) && dw->device() == dev, "d_weights is ", dw->sizes(), " on ", dw->device(),
                      ", expected [", r.T, ", ", k, "] on ", dev);
    dw = dw->to(at::kFloat).contiguous();
  }
  for (const auto* g : {&db, &dz})
    TORCH_CHECK_VALUE(!*g || ((*g)->numel() == 1 && (*g)->scalar_type() == at::kFloat && (*g)->device() == dev),
                      "d_balance and d_z must be float32 scalar tensors on the logits' device");
  const c10::cuda::CUDAGuard guard(dev);
  at::Tensor d = empty({r.T, r.E}, r.logits.scalar_type(), dev);
  check(p_route_backward(r.logits.data_ptr(), r.type, r.ld, r.T, (int32_t)r.E, (int32_t)k, r.sequences,
                         ptr<uint8_t>(r.mask), (int32_t)integer(a[10]), truth(a[11]), ids.data_ptr<int32_t>(),
                         weights.data_ptr<float>(), counts.data_ptr<int32_t>(), tokens.data_ptr<int32_t>(),
                         ptr<float>(dw), ptr<float>(db), ptr<float>(dz), d.data_ptr(),
                         c10::cuda::getCurrentCUDAStream(dev.index())));
  return THPVariable_Wrap(d);
  END_HANDLE_TH_ERRORS
}

// ---------------------------------------------------------------- rows
// Rows in whole vectors of four elements: a contiguous view may start anywhere
// in its storage, the kernels read four elements at a time.
at::Tensor rows(const at::Tensor& t, const char* name) {
  TORCH_CHECK_VALUE(t.is_cuda() && t.dim() == 2, name, " must be a 2-D CUDA tensor");
  TORCH_CHECK_VALUE(t.size(1) % 4 == 0 && t.size(1) > 0, name, " has rows of ", t.size(1),
                    " elements: a positive multiple of 4 is needed");
  if (!t.is_contiguous()) return t.contiguous();
  return reinterpret_cast<uintptr_t>(t.data_ptr()) % (4 * t.element_size()) ? t.clone() : t;
}

// (dy, y_sorted, inverse, weights, group_sizes, type of dys)
PyObject* combine_backward(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n == 6, "combine_backward takes 6 arguments");
  at::AutoDispatchBelowADInplaceOrView below;
  const int type = elem(tensor(a[0], "dy"), "dy");
  const at::Tensor dy = rows(tensor(a[0], "dy"), "dy"), ys = rows(tensor(a[1], "y_sorted"), "y_sorted");
  at::Tensor inverse = tensor(a[2], "inverse"), weights = tensor(a[3], "weights"), gs = tensor(a[4], "group_sizes");
  const at::Device dev = dy.device();
  TORCH_CHECK_VALUE(inverse.dim() == 2, "inverse must be (T, k)");
  const int64_t T = inverse.size(0), k = inverse.size(1), N = ys.size(0), D = ys.size(1);
  TORCH_CHECK_VALUE(shaped(dy, T, D) && shaped(weights, T, k), "dy ", dy.sizes(), ", weights ", weights.sizes(),
                    ": expected [", T, ", ", D, "] and [", T, ", ", k, "]");
  TORCH_CHECK_TYPE(ys.scalar_type() == at::kFloat && inverse.scalar_type() == at::kInt,
                   "y_sorted must be float32 and inverse int32");
  on(dev, ys, "y_sorted");
  on(dev, inverse, "inverse");
  on(dev, weights, "weights");
  on(dev, gs, "group_sizes");
  inverse = inverse.contiguous();
  weights = weights.to(at::kFloat).contiguous();
  gs = gs.to(at::kInt).contiguous();
  const int out = (int)integer(a[5]);
  const c10::cuda::CUDAGuard guard(dev);
  at::Tensor dys = empty({N, D}, elem_type(out), dev), dw = empty({T, k}, at::kFloat, dev);
  check(p_combine(dy.data_ptr(), type, ys.data_ptr<float>(), inverse.data_ptr<int32_t>(), weights.data_ptr<float>(),
                  gs.data_ptr<int32_t>(), T, (int32_t)k, (int32_t)D, N, (int32_t)gs.numel(), dys.data_ptr(), out,
                  dw.data_ptr<float>(), c10::cuda::getCurrentCUDAStream(dev.index())));
  PyObject* both = PyTuple_New(2);
  if (!both) throw python_error();
  PyTuple_SET_ITEM(both, 0, THPVariable_Wrap(dys));
  PyTuple_SET_ITEM(both, 1, THPVariable_Wrap(dw));
  return both;
  END_HANDLE_TH_ERRORS
}

// (dxs, inverse, type of dx or -1 for dxs's)
PyObject* gather_backward(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n == 3, "gather_backward takes 3 arguments");
  at::AutoDispatchBelowADInplaceOrView below;
  const int type = elem(tensor(a[0], "dxs"), "dxs");
  const at::Tensor dxs = rows(tensor(a[0], "dxs"), "dxs");
  at::Tensor inverse = tensor(a[1], "inverse");
  const at::Device dev = dxs.device();
  TORCH_CHECK_VALUE(inverse.dim() == 2, "inverse must be (T, k)");
  TORCH_CHECK_TYPE(inverse.scalar_type() == at::kInt, "inverse must be int32");
  on(dev, inverse, "inverse");
  inverse = inverse.contiguous();
  const int64_t T = inverse.size(0), D = dxs.size(1);
  const int out = integer(a[2]) < 0 ? type : (int)integer(a[2]);
  const c10::cuda::CUDAGuard guard(dev);
  at::Tensor dx = empty({T, D}, elem_type(out), dev);
  check(p_gather(dxs.data_ptr(), type, inverse.data_ptr<int32_t>(), T, (int32_t)inverse.size(1), (int32_t)D,
                 dxs.size(0), dx.data_ptr(), out, c10::cuda::getCurrentCUDAStream(dev.index())));
  return THPVariable_Wrap(dx);
  END_HANDLE_TH_ERRORS
}

// ---------------------------------------------------------------- gradient lists
struct Rows {
  int64_t rows = 1, cols = 1, ld = 0;
};
// A tensor whose elements, in some order of its dimensions, are equally long
// contiguous rows at equal distances; false for other strides.
bool rows_of(const at::Tensor& t, Rows* r) {
  std::vector<std::pair<int64_t, int64_t>> dims;  // stride, size
  for (int64_t i = 0; i < t.dim(); ++i)
    if (t.size(i) > 1) dims.emplace_back(t.stride(i), t.size(i));
  std::sort(dims.begin(), dims.end());
  size_t i = 0;
  for (; i < dims.size() && dims[i].first == r->cols; ++i) r->cols *= dims[i].second;
  r->ld = r->cols;
  if (i == dims.size()) return true;
  r->ld = dims[i].first;
  for (; i < dims.size() && dims[i].first == r->ld * r->rows; ++i) r->rows *= dims[i].second;
  return i == dims.size() && r->ld >= r->cols;
}
// Whether the elements of both lie in memory in the same order.
bool same_order(const at::Tensor& a, const at::Tensor& b) {
  std::vector<int64_t> da, db;
  for (int64_t i = 0; i < a.dim(); ++i)
    if (a.size(i) > 1) da.push_back(i);
  db = da;
  std::stable_sort(da.begin(), da.end(), [&](int64_t x, int64_t y) { return a.stride(x) < a.stride(y); });
  std::stable_sort(db.begin(), db.end(), [&](int64_t x, int64_t y) { return b.stride(x) < b.stride(y); });
  return da == db;
}
std::string strides_of(const at::Tensor& t) {
  std::ostringstream s;
  s << t.strides();
  return s.str();
}

struct List {
  std::vector<moe_tensor_desc> d;
  std::vector<at::Tensor> keep;  // the list's tensors, for the length of the call
  c10::optional<at::Device> dev;
};
std::vector<at::Tensor> tensors(PyObject* o, const char* name) {
  PyObject* seq = PySequence_Fast(o, "gradients must be a sequence of tensors");
  if (!seq) throw python_error();
  std::vector<at::Tensor> v;
  const Py_ssize_t n = PySequence_Fast_GET_SIZE(seq);
  v.reserve(n);
  for (Py_ssize_t i = 0; i < n; ++i) {
    PyObject* t = PySequence_Fast_GET_ITEM(seq, i);
    if (!THPVariable_Check(t)) {
      Py_DECREF(seq);
      TORCH_CHECK_TYPE(false, name, " must be tensors, not ", Py_TYPE(t)->tp_name);
    }
    v.push_back(THPVariable_Unpack(t));
  }
  Py_DECREF(seq);
  return v;
}
List describe(PyObject* grads, PyObject* out) {
  List l;
  l.keep = tensors(grads, "gradients");
  const size_t n = l.keep.size();
  std::vector<at::Tensor> outs;
  if (out != Py_None) {
    outs = tensors(out, "outputs");
    TORCH_CHECK_VALUE(outs.size() == n, n, " gradients and ", outs.size(), " outputs");
  }
  l.d.resize(n);
  for (size_t i = 0; i < n; ++i) {
    const at::Tensor &g = l.keep[i], &o = outs.empty() ? g : outs[i];
    if (i == 0) l.dev = g.device();
    TORCH_CHECK_VALUE(g.is_cuda() && g.device() == *l.dev && o.device() == *l.dev,
                      "gradients and outputs must be CUDA tensors on one device");
    moe_tensor_desc& d = l.d[i];
    d = moe_tensor_desc{g.data_ptr(), o.data_ptr(), 1, g.numel(), 0, 0, elem(g, "a gradient"), elem(o, "an output")};
    TORCH_CHECK_VALUE(outs.empty() || g.sizes() == o.sizes(), "tensor ", i,
                      ": an output of another shape than its gradient, ", g.sizes(), ", ", o.sizes());
    if (g.is_contiguous() && o.is_contiguous()) continue;
    Rows rg, ro;
    bool ok = rows_of(g, &rg) && rows_of(o, &ro) && same_order(g, o);
    if (ok) {
      if (rg.rows == 1) rg = Rows{ro.rows, ro.cols, ro.cols};
      if (ro.rows == 1) ro = Rows{rg.rows, rg.cols, rg.cols};
      ok = rg.rows == ro.rows && rg.cols == ro.cols;
    }
    TORCH_CHECK_VALUE(ok, "tensor ", i, ": strides ", strides_of(g), " and ", strides_of(o), " of shape ", g.sizes(),
                      " are not equally spaced rows of one order");
    d.rows = rg.rows;
    d.cols = rg.cols;
    d.in_ld = rg.ld;
    d.out_ld = ro.ld;
  }
  l.keep.insert(l.keep.end(), outs.begin(), outs.end());
  return l;
}
// Tells autograd that a call wrote the outputs (the gradients, in place): a
// graph that saved one of them raises at its backward, as after any in-place
// operation.
void written(const List& l) {
  const size_t n = l.d.size();
  for (size_t i = l.keep.size() > n ? n : 0; i < l.keep.size(); ++i)
    if (!l.keep[i].is_inference()) l.keep[i].unsafeGetTensorImpl()->bump_version();
}
at::Tensor no_gradients() { return at::zeros({}, at::TensorOptions().dtype(at::kFloat).device(at::kCUDA)); }

// (gradients, norm type)
PyObject* grad_norm(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n == 2, "grad_norm takes 2 arguments");
  at::AutoDispatchBelowADInplaceOrView below;
  const List l = describe(a[0], Py_None);
  if (!l.dev) return THPVariable_Wrap(no_gradients());
  const c10::cuda::CUDAGuard guard(*l.dev);
  const cudaStream_t stream = c10::cuda::getCurrentCUDAStream(l.dev->index());
  at::Tensor norm = empty({}, at::kFloat, *l.dev);
  const size_t need = p_norm_space((int32_t)l.d.size());
  const at::Tensor ws = workspace(*l.dev, stream, need, capturing());
  check(p_norm(l.d.data(), (int32_t)l.d.size(), (int32_t)integer(a[1]), norm.data_ptr<float>(), ws.data_ptr(), need,
               stream));
  return THPVariable_Wrap(norm);
  END_HANDLE_TH_ERRORS
}

// (gradients, max_norm, norm type, norm or None, outputs or None)
PyObject* clip(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n == 5, "clip takes 5 arguments");
  at::AutoDispatchBelowADInplaceOrView below;
  const double max_norm = PyFloat_AsDouble(a[1]);
  if (max_norm == -1.0 && PyErr_Occurred()) throw python_error();
  TORCH_CHECK_VALUE(max_norm >= 0.0, "max_norm ", max_norm, " must be at least 0");
  const List l = describe(a[0], a[4]);
  const c10::optional<at::Tensor> given = maybe(a[3], "total_norm");
  if (!l.dev) return THPVariable_Wrap(given ? *given : no_gradients());
  const c10::cuda::CUDAGuard guard(*l.dev);
  const cudaStream_t stream = c10::cuda::getCurrentCUDAStream(l.dev->index());
  if (given) {
    TORCH_CHECK_VALUE(given->device() == *l.dev && given->scalar_type() == at::kFloat && given->numel() == 1,
                      "total_norm must be a float32 scalar tensor on the gradients' device");
    check(p_clip(l.d.data(), (int32_t)l.d.size(), (int32_t)integer(a[2]), max_norm, given->data_ptr<float>(), nullptr,
                 nullptr, 0, stream));
    written(l);
    return THPVariable_Wrap(*given);
  }
  at::Tensor norm = empty({}, at::kFloat, *l.dev);
  const size_t need = p_norm_space((int32_t)l.d.size());
  const at::Tensor ws = workspace(*l.dev, stream, need, capturing());
  check(p_clip(l.d.data(), (int32_t)l.d.size(), (int32_t)integer(a[2]), max_norm, nullptr, norm.data_ptr<float>(),
               ws.data_ptr(), need, stream));
  written(l);
  return THPVariable_Wrap(norm);
  END_HANDLE_TH_ERRORS
}

// (tensor) -> (rows, cols, row stride) or None, as the lists see it
PyObject* tensor_rows(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n == 1, "tensor_rows takes 1 argument");
  Rows r;
  if (!rows_of(tensor(a[0], "t"), &r)) Py_RETURN_NONE;
  return Py_BuildValue("(LLL)", (long long)r.rows, (long long)r.cols, (long long)r.ld);
  END_HANDLE_TH_ERRORS
}

// ({name: address}, MoeError)
PyObject* bind(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n == 2 && PyDict_Check(a[0]), "bind takes a dict of addresses and an exception type");
  auto set = [&](const char* name, auto& fn) {
    PyObject* v = PyDict_GetItemString(a[0], name);
    TORCH_CHECK_VALUE(v, "no address of ", name);
    fn = reinterpret_cast<std::decay_t<decltype(fn)>>(static_cast<uintptr_t>(PyLong_AsUnsignedLongLong(v)));
    if (PyErr_Occurred()) throw python_error();
  };
  set("moe_route_train_workspace_size", p_route_space);
  set("moe_route_train_counters", p_route_counters);
  set("moe_route_train", p_route_train);
  set("moe_route_backward", p_route_backward);
  set("moe_combine_rows_backward", p_combine);
  set("moe_gather_rows_backward", p_gather);
  set("moe_grad_norm_workspace_size", p_norm_space);
  set("moe_grad_norm", p_norm);
  set("moe_clip_grads", p_clip);
  set("moe_last_error", p_error);
  Py_INCREF(a[1]);
  Py_XDECREF(g_moe_error);
  g_moe_error = a[1];
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

#define FAST(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(name)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {FAST(bind),     FAST(route_forward),   FAST(route_backward), FAST(combine_backward),
                         FAST(gather_backward), FAST(grad_norm), FAST(clip),           FAST(tensor_rows),
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "moe_layer_native", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_moe_layer_native(void) { return PyModule_Create(&module); }
