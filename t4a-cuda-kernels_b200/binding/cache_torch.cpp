// The paged-cache operators for Python over torch tensors: t4a_b200/cache.py calls these functions,
// which read the tensors' metadata, allocate results on the current stream and call the C ABI
// (include/t4a_b200/cache.h).  Native because a small call's kernels take some 5 us, and reading
// ten tensors' metadata from Python took 30.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/t4a_b200.h"

namespace {

constexpr int kNoType = -1;

// A tensor's layout (its axes reversed) and reachable elements.
struct Described {
  t4a_cuda_layout layout;
  long long len;
};

Described describe(const at::Tensor& t, const char* name) {
  Described d = {};
  const int64_t rank = t.dim();
  TORCH_CHECK_VALUE(rank <= T4A_CUDA_MAX_RANK, name, " has more than ", T4A_CUDA_MAX_RANK, " axes");
  d.layout.rank = static_cast<int>(rank);
  d.len = 1;
  for (int64_t i = 0; i < rank; ++i) {
    d.layout.extents[i] = t.size(rank - 1 - i);
    d.layout.strides[i] = t.stride(rank - 1 - i);
    d.len += (d.layout.extents[i] - 1) * d.layout.strides[i];
  }
  if (t.numel() == 0) d.len = 0;
  return d;
}

bool is_none(PyObject* o) { return o == Py_None; }

const at::Tensor& tensor(PyObject* o, const char* name) {
  TORCH_CHECK_TYPE(THPVariable_Check(o), name, " is not a tensor");
  return THPVariable_Unpack(o);
}

int row_dtype(const at::Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return T4A_CUDA_F32;
    case at::kHalf: return T4A_F16;
    case at::kBFloat16: return T4A_BF16;
    default: return kNoType;
  }
}

int cache_kind(const at::Tensor& t) {
  switch (t.scalar_type()) {
    case at::kHalf: return T4A_F16;
    case at::kBFloat16: return T4A_BF16;
    case at::kChar: return T4A_I8;
    case at::kFloat8_e4m3fn: return T4A_E4M3;
    default: return kNoType;
  }
}

// What every tensor of a call shares: the current device.
class Call {
 public:
  explicit Call(const at::Tensor& t, const char* name) {
    TORCH_CHECK_VALUE(t.is_cuda(), name, " is not a CUDA tensor");
    device_ = t.device();
    TORCH_CHECK_VALUE(device_.index() == c10::cuda::current_device(), name, " is on ", device_,
                      ", which is not the current device");
  }
  const at::Tensor& on_device(const at::Tensor& t, const char* name) const {
    TORCH_CHECK_VALUE(t.device() == device_, name, " is on ", t.device(), ", not on ", device_);
    return t;
  }
  const at::Tensor& typed(PyObject* o, const char* name, at::ScalarType type) const {
    const at::Tensor& t = on_device(tensor(o, name), name);
    TORCH_CHECK_TYPE(t.scalar_type() == type, name, ": ", t.scalar_type(), " is not supported");
    return t;
  }
  void* stream() const { return c10::cuda::getCurrentCUDAStream(device_.index()).stream(); }
  at::Tensor empty(at::IntArrayRef shape, at::ScalarType type) const {
    return at::empty(shape, at::TensorOptions().dtype(type).device(device_));
  }

 private:
  at::Device device_{at::kCPU};
};

t4a_kv_cache describe_cache(const Call& call, PyObject* k_cache, PyObject* v_cache, PyObject* k_scale,
                            PyObject* v_scale) {
  const at::Tensor& k = call.on_device(tensor(k_cache, "k_cache"), "k_cache");
  const at::Tensor& v = call.typed(v_cache, "v_cache", k.scalar_type());
  t4a_kv_cache c = {};
  c.kind = cache_kind(k);
  TORCH_CHECK_TYPE(c.kind != kNoType, "k_cache: ", k.scalar_type(), " is not supported");
  const bool scaled = c.kind == T4A_I8 || c.kind == T4A_E4M3;
  TORCH_CHECK_VALUE(scaled != is_none(k_scale) && scaled != is_none(v_scale),
                    "k_scale and v_scale go with an 8-bit cache, and only with one");
  Described d = describe(k, "k_cache");
  c.k = k.data_ptr();
  c.k_layout = d.layout;
  c.k_len = d.len;
  d = describe(v, "v_cache");
  c.v = v.data_ptr();
  c.v_layout = d.layout;
  c.v_len = d.len;
  if (scaled) {
    const at::Tensor& ks = call.typed(k_scale, "k_scale", at::kFloat);
    const at::Tensor& vs = call.typed(v_scale, "v_scale", at::kFloat);
    d = describe(ks, "k_scale");
    c.k_scale = static_cast<float*>(ks.data_ptr());
    c.k_scale_layout = d.layout;
    c.k_scale_len = d.len;
    d = describe(vs, "v_scale");
    c.v_scale = static_cast<float*>(vs.data_ptr());
    c.v_scale_layout = d.layout;
    c.v_scale_len = d.len;
  }
  return c;
}

// A status as t4a_b200.T4AError.
PyObject* refuse(int status, const char* where) {
  PyObject* module = PyImport_ImportModule("t4a_b200");
  PyObject* type = module ? PyObject_GetAttrString(module, "T4AError") : nullptr;
  PyObject* error = type ? PyObject_CallFunction(type, "is", status, where) : nullptr;
  if (error) PyErr_SetObject(type, error);
  Py_XDECREF(error);
  Py_XDECREF(type);
  Py_XDECREF(module);
  return nullptr;
}

bool counted(Py_ssize_t n, Py_ssize_t want) {
  if (n == want) return true;
  PyErr_Format(PyExc_TypeError, "%zd arguments, not %zd", n, want);
  return false;
}

int index_dtype(const at::Tensor& slots) {
  TORCH_CHECK_TYPE(slots.scalar_type() == at::kInt || slots.scalar_type() == at::kLong, "slots: ",
                   slots.scalar_type(), " is not supported");
  return slots.scalar_type() == at::kLong ? T4A_CUDA_I64 : T4A_CUDA_I32;
}

// key, value, k_cache, v_cache, slots, k_scale, v_scale
PyObject* write(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!counted(n, 7)) return nullptr;
  const at::Tensor& key = tensor(args[0], "key");
  const Call call(key, "key");
  const int dtype = row_dtype(key);
  TORCH_CHECK_TYPE(dtype != kNoType, "key: ", key.scalar_type(), " is not supported");
  const at::Tensor& value = call.typed(args[1], "value", key.scalar_type());
  const at::Tensor& slots = call.on_device(tensor(args[4], "slots"), "slots");
  const int index = index_dtype(slots);
  const t4a_kv_cache cache = describe_cache(call, args[2], args[3], args[5], args[6]);
  const Described k = describe(key, "key"), v = describe(value, "value"), s = describe(slots, "slots");
  const int status = t4a_cache_write(call.stream(), dtype, index, &cache, key.data_ptr(), &k.layout, k.len,
                                     value.data_ptr(), &v.layout, v.len, slots.data_ptr(), &s.layout, s.len);
  if (status != T4A_OK) return refuse(status, "cache_write");
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

// k_cache, v_cache, slots, row dtype tag, k_scale, v_scale, out key, out value
PyObject* read(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!counted(n, 8)) return nullptr;
  const at::Tensor& k_cache = tensor(args[0], "k_cache");
  const Call call(k_cache, "k_cache");
  const long dtype = PyLong_AsLong(args[3]);
  if (dtype == -1 && PyErr_Occurred()) return nullptr;
  const at::ScalarType type = dtype == T4A_CUDA_F32 ? at::kFloat : dtype == T4A_F16 ? at::kHalf : at::kBFloat16;
  const at::Tensor& slots = call.on_device(tensor(args[2], "slots"), "slots");
  const int index = index_dtype(slots);
  const t4a_kv_cache cache = describe_cache(call, args[0], args[1], args[4], args[5]);
  at::Tensor key, value;
  if (is_none(args[6])) {
    TORCH_CHECK_VALUE(slots.dim() == 1 && k_cache.dim() == 4, "slots is [n] and k_cache [pages, page_size, heads, dim]");
    key = call.empty({slots.size(0), k_cache.size(2), k_cache.size(3)}, type);
    value = call.empty({slots.size(0), k_cache.size(2), k_cache.size(3)}, type);
  } else {
    key = call.typed(args[6], "out[0]", type);
    value = call.typed(args[7], "out[1]", type);
  }
  const Described k = describe(key, "key"), v = describe(value, "value"), s = describe(slots, "slots");
  const int status = t4a_cache_read(call.stream(), static_cast<int>(dtype), index, &cache, key.data_ptr(), &k.layout,
                                    k.len, value.data_ptr(), &v.layout, v.len, slots.data_ptr(), &s.layout, s.len);
  if (status != T4A_OK) return refuse(status, "cache_read");
  return Py_BuildValue("NN", THPVariable_Wrap(std::move(key)), THPVariable_Wrap(std::move(value)));
  END_HANDLE_TH_ERRORS
}

size_t workspace_bytes(const t4a_kv_cache& cache, int dtype, const Described& q, const Described& table, int* status) {
  size_t bytes = 0;
  *status = t4a_tree_attention_workspace_bytes(dtype, &cache, &q.layout, &table.layout, &bytes);
  return bytes;
}

const at::Tensor* vector_of(const Call& call, PyObject* o, const char* name, int64_t batch) {
  if (is_none(o)) return nullptr;
  const at::Tensor& t = call.typed(o, name, at::kInt);
  TORCH_CHECK_VALUE(t.dim() == 1 && t.size(0) == batch && t.is_contiguous(), name, " is a contiguous [batch]");
  return &t;
}

// q, k_cache, v_cache, page_table, k_scale, v_scale
PyObject* attention_bytes(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!counted(n, 6)) return nullptr;
  const at::Tensor& q = tensor(args[0], "q");
  const Call call(q, "q");
  const t4a_kv_cache cache = describe_cache(call, args[1], args[2], args[4], args[5]);
  int status;
  const size_t bytes = workspace_bytes(cache, row_dtype(q), describe(q, "q"),
                                       describe(call.typed(args[3], "page_table", at::kInt), "page_table"), &status);
  if (status != T4A_OK) return refuse(status, "tree_attention_workspace_bytes");
  return PyLong_FromSize_t(bytes);
  END_HANDLE_TH_ERRORS
}

// q, k_cache, v_cache, page_table, context, mask, nodes, k_scale, v_scale, scale, out, lse, workspace
PyObject* attention(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!counted(n, 13)) return nullptr;
  const at::Tensor& q = tensor(args[0], "q");
  const Call call(q, "q");
  const int dtype = row_dtype(q);
  TORCH_CHECK_TYPE(dtype == T4A_F16 || dtype == T4A_BF16, "q: ", q.scalar_type(), " is not supported");
  TORCH_CHECK_VALUE(q.dim() == 4, "q is [batch, nodes, query heads, dim]");
  const at::Tensor& table = call.typed(args[3], "page_table", at::kInt);
  const at::Tensor* context = vector_of(call, args[4], "context", q.size(0));
  const at::Tensor* nodes = vector_of(call, args[6], "nodes", q.size(0));
  TORCH_CHECK_VALUE(context != nullptr, "context is needed");
  const t4a_kv_cache cache = describe_cache(call, args[1], args[2], args[7], args[8]);
  double scale = 0.0;
  if (is_none(args[9])) {
    scale = 1.0 / std::sqrt(static_cast<double>(std::max<int64_t>(1, q.size(3))));
  } else {
    scale = PyFloat_AsDouble(args[9]);
    if (scale == -1.0 && PyErr_Occurred()) return nullptr;
  }
  at::Tensor out = is_none(args[10]) ? call.empty(q.sizes(), q.scalar_type()) : call.typed(args[10], "out", q.scalar_type());
  at::Tensor lse = is_none(args[11]) ? call.empty({q.size(0), q.size(1), q.size(2)}, at::kFloat)
                                     : call.typed(args[11], "lse", at::kFloat);
  const Described dq = describe(q, "q"), dt = describe(table, "page_table"), d_out = describe(out, "out"),
                  dl = describe(lse, "lse");
  at::Tensor workspace;
  if (is_none(args[12])) {
    int status;
    const size_t bytes = workspace_bytes(cache, dtype, dq, dt, &status);
    if (status != T4A_OK) return refuse(status, "tree_attention");
    workspace = call.empty({static_cast<int64_t>(bytes)}, at::kByte);
  } else {
    workspace = call.typed(args[12], "workspace", at::kByte);
    TORCH_CHECK_VALUE(workspace.is_contiguous(), "workspace is contiguous");
  }
  Described dm = {};
  const unsigned char* mask = nullptr;
  if (!is_none(args[5])) {
    const at::Tensor& m = call.on_device(tensor(args[5], "mask"), "mask");
    TORCH_CHECK_TYPE(m.scalar_type() == at::kBool || m.scalar_type() == at::kByte, "mask: ", m.scalar_type(),
                     " is not supported");
    dm = describe(m, "mask");
    mask = static_cast<const unsigned char*>(m.data_ptr());
  }
  const int status = t4a_tree_attention(
      call.stream(), dtype, &cache, out.data_ptr(), &d_out.layout, d_out.len, static_cast<float*>(lse.data_ptr()),
      &dl.layout, dl.len, q.data_ptr(), &dq.layout, dq.len, static_cast<const int*>(table.data_ptr()), &dt.layout,
      dt.len, static_cast<const int*>(context->data_ptr()),
      nodes ? static_cast<const int*>(nodes->data_ptr()) : nullptr, mask, &dm.layout, dm.len,
      static_cast<float>(scale), workspace.data_ptr(), static_cast<size_t>(workspace.numel()));
  if (status != T4A_OK) return refuse(status, "tree_attention");
  return Py_BuildValue("NN", THPVariable_Wrap(std::move(out)), THPVariable_Wrap(std::move(lse)));
  END_HANDLE_TH_ERRORS
}

// logits, tokens, parents, uniforms, draft, race, temperature
PyObject* verify(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!counted(n, 7)) return nullptr;
  const at::Tensor& logits = tensor(args[0], "logits");
  const Call call(logits, "logits");
  const int dtype = row_dtype(logits);
  TORCH_CHECK_TYPE(dtype != kNoType, "logits: ", logits.scalar_type(), " is not supported");
  TORCH_CHECK_VALUE(logits.dim() == 3, "logits is [batch, nodes, vocab]");
  const int64_t batch = logits.size(0), nodes = logits.size(1);
  auto compact = [&](PyObject* o, const char* name, at::ScalarType type) -> void* {
    if (is_none(o)) return nullptr;
    const at::Tensor& t = call.typed(o, name, type);
    TORCH_CHECK_VALUE(t.dim() == 2 && t.size(0) == batch && t.size(1) == nodes && t.is_contiguous(), name,
                      " is a contiguous [batch, nodes]");
    return t.data_ptr();
  };
  const int* tokens = static_cast<const int*>(compact(args[1], "tokens", at::kInt));
  const int* parents = static_cast<const int*>(compact(args[2], "parents", at::kInt));
  const float* uniforms = static_cast<const float*>(compact(args[3], "uniforms", at::kFloat));
  Described dd = {}, dr = {};
  const float *draft = nullptr, *race = nullptr;
  if (!is_none(args[4])) {
    const at::Tensor& t = call.typed(args[4], "draft", at::kFloat);
    dd = describe(t, "draft");
    draft = static_cast<const float*>(t.data_ptr());
  }
  if (!is_none(args[5])) {
    const at::Tensor& t = call.typed(args[5], "race", at::kFloat);
    dr = describe(t, "race");
    race = static_cast<const float*>(t.data_ptr());
  }
  const double temperature = PyFloat_AsDouble(args[6]);
  if (temperature == -1.0 && PyErr_Occurred()) return nullptr;
  at::Tensor count = call.empty({batch}, at::kInt), path = call.empty({batch, nodes}, at::kInt),
             said = call.empty({batch, nodes}, at::kInt), logs = call.empty({batch, nodes}, at::kFloat);
  const Described dl = describe(logits, "logits");
  const int status = t4a_verify_drafts(
      call.stream(), dtype, logits.data_ptr(), &dl.layout, dl.len, tokens, parents, uniforms, draft, &dd.layout, dd.len,
      race, &dr.layout, dr.len, static_cast<float>(temperature), static_cast<int*>(count.data_ptr()),
      static_cast<int*>(path.data_ptr()), static_cast<int*>(said.data_ptr()), static_cast<float*>(logs.data_ptr()));
  if (status != T4A_OK) return refuse(status, "verify_drafts");
  return Py_BuildValue("NNNN", THPVariable_Wrap(std::move(count)), THPVariable_Wrap(std::move(path)),
                       THPVariable_Wrap(std::move(said)), THPVariable_Wrap(std::move(logs)));
  END_HANDLE_TH_ERRORS
}

#define T4A_METHOD(f) \
  { #f, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)), METH_FASTCALL, nullptr }
PyMethodDef methods[] = {T4A_METHOD(write),     T4A_METHOD(read),   T4A_METHOD(attention_bytes),
                         T4A_METHOD(attention), T4A_METHOD(verify), {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_cache_torch", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__cache_torch() { return PyModule_Create(&module); }
