// The short host path of a graph that is one model operator, as a Python type:
//
//   Call(launch, encode, module, kernel, cfg, block, patches, maps, inputs,
//        out_shape, out_dtype, device)
//   call(tensors) -> output tensor, or NotImplemented
//
// The parameter block of such a launch is fixed by the shapes but for the
// pointers (`patches`) and the tensor maps that hold one (`maps`).  A call checks
// the tensors, allocates the output on the current stream, fills the block and
// launches.  For kernels of a few microseconds the same steps in Python took
// longer than the kernel (9.4 to 10.9 us a call; these take 4.3 to 5.9).
//
// NotImplemented stands for every call that is not plain: other shapes, types or
// device, strided or misplaced tensors, a launch that failed (the general path
// repeats it and reports).  Nothing is kept from one call for the next.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/Functions.h>
#include <ATen/core/Tensor.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstdint>
#include <cstring>
#include <new>
#include <string>
#include <vector>

#include "molten_rt.h"

namespace {

typedef int (*LaunchFn)(void*, const char*, const molten_launch_cfg*, const void*, size_t, void*);
typedef int (*EncodeFn)(void*, int, const void*, const uint64_t*, const uint64_t*, const uint32_t*);

constexpr size_t kMaxBlock = 1024;

struct Patch {
  Py_ssize_t at;
  Py_ssize_t tensor;               // -1: the output
};
struct Map {
  Py_ssize_t at, tensor;
  int dtype;
  uint64_t dims[4], strides[3];
  uint32_t box[4];
};
struct Input {
  at::ScalarType dtype;
  std::vector<int64_t> shape;
};
struct Plan {
  LaunchFn launch;
  EncodeFn encode;
  void* module;
  std::string kernel, block;
  molten_launch_cfg cfg;
  std::vector<Patch> patches;
  std::vector<Map> maps;
  std::vector<Input> inputs;
  std::vector<int64_t> out_shape;
  at::ScalarType out_dtype;
  int device;
};

struct Call {
  PyObject_HEAD
  Plan* plan;
};

bool shape_of(PyObject* o, std::vector<int64_t>* out) {
  if (!PyTuple_Check(o)) { PyErr_SetString(PyExc_TypeError, "a shape must be a tuple"); return false; }
  for (Py_ssize_t i = 0; i < PyTuple_GET_SIZE(o); ++i) {
    const long long d = PyLong_AsLongLong(PyTuple_GET_ITEM(o, i));
    if (d == -1 && PyErr_Occurred()) return false;
    out->push_back(d);
  }
  return true;
}

bool fill(Plan& p, PyObject* args) {
  unsigned long long launch, encode, module;
  const char *kernel, *cfg, *block;
  Py_ssize_t nk, nc, nb;
  PyObject *patches, *maps, *inputs, *shape, *dtype;
  if (!PyArg_ParseTuple(args, "KKKy#y#y#O!O!O!OOi", &launch, &encode, &module, &kernel, &nk, &cfg, &nc, &block, &nb,
                        &PyTuple_Type, &patches, &PyTuple_Type, &maps, &PyTuple_Type, &inputs, &shape, &dtype,
                        &p.device))
    return false;
  p.launch = reinterpret_cast<LaunchFn>(launch);
  p.encode = reinterpret_cast<EncodeFn>(encode);
  p.module = reinterpret_cast<void*>(module);
  p.kernel.assign(kernel, nk);
  p.block.assign(block, nb);
  if (nc != (Py_ssize_t)sizeof(p.cfg) || p.block.size() > kMaxBlock || !launch || !module || !THPDtype_Check(dtype)) {
    PyErr_SetString(PyExc_ValueError, "bad launch config, parameter block or output type");
    return false;
  }
  std::memcpy(&p.cfg, cfg, sizeof(p.cfg));
  const Py_ssize_t n = PyTuple_GET_SIZE(inputs);
  for (Py_ssize_t i = 0; i < n; ++i) {
    PyObject *dt, *sh;
    if (!PyArg_ParseTuple(PyTuple_GET_ITEM(inputs, i), "OO", &dt, &sh)) return false;
    Input in;
    if (!THPDtype_Check(dt)) { PyErr_SetString(PyExc_TypeError, "an input's type must be a dtype"); return false; }
    in.dtype = reinterpret_cast<THPDtype*>(dt)->scalar_type;
    if (!shape_of(sh, &in.shape)) return false;
    p.inputs.push_back(in);
  }
  for (Py_ssize_t i = 0; i < PyTuple_GET_SIZE(patches); ++i) {
    Patch q;
    if (!PyArg_ParseTuple(PyTuple_GET_ITEM(patches, i), "nn", &q.at, &q.tensor)) return false;
    if (q.at < 0 || q.at + 8 > nb || q.tensor < -1 || q.tensor >= n) {
      PyErr_SetString(PyExc_ValueError, "a patch lies outside the block or the tensors");
      return false;
    }
    p.patches.push_back(q);
  }
  for (Py_ssize_t i = 0; i < PyTuple_GET_SIZE(maps); ++i) {
    Map q;
    const char *d, *s, *b;
    Py_ssize_t nd, ns, nx;
    if (!PyArg_ParseTuple(PyTuple_GET_ITEM(maps, i), "nniy#y#y#", &q.at, &q.tensor, &q.dtype, &d, &nd, &s, &ns, &b, &nx))
      return false;
    if (q.at < 0 || q.at % 64 || q.at + 128 > nb || q.tensor < 0 || q.tensor >= n || nd != sizeof(q.dims) ||
        ns != sizeof(q.strides) || nx != sizeof(q.box) || !encode) {
      PyErr_SetString(PyExc_ValueError, "a tensor map lies outside the block or the tensors");
      return false;
    }
    std::memcpy(q.dims, d, nd);
    std::memcpy(q.strides, s, ns);
    std::memcpy(q.box, b, nx);
    p.maps.push_back(q);
  }
  if (!shape_of(shape, &p.out_shape)) return false;
  p.out_dtype = reinterpret_cast<THPDtype*>(dtype)->scalar_type;
  return true;
}

PyObject* call_new(PyTypeObject* type, PyObject* args, PyObject* kwargs) {
  HANDLE_TH_ERRORS
  if (kwargs && PyDict_Size(kwargs)) {
    PyErr_SetString(PyExc_TypeError, "Call takes no keyword arguments");
    return nullptr;
  }
  Call* self = reinterpret_cast<Call*>(type->tp_alloc(type, 0));
  if (!self) return nullptr;
  self->plan = new (std::nothrow) Plan();
  if (!self->plan || !fill(*self->plan, args)) {
    if (!PyErr_Occurred()) PyErr_NoMemory();
    Py_DECREF(self);
    return nullptr;
  }
  return reinterpret_cast<PyObject*>(self);
  END_HANDLE_TH_ERRORS
}

void call_dealloc(PyObject* o) {
  delete reinterpret_cast<Call*>(o)->plan;
  Py_TYPE(o)->tp_free(o);
}

PyObject* call_call(PyObject* o, PyObject* args, PyObject* kwargs) {
  HANDLE_TH_ERRORS
  const Plan& p = *reinterpret_cast<Call*>(o)->plan;
  PyObject* tensors;
  if ((kwargs && PyDict_Size(kwargs)) || PyTuple_GET_SIZE(args) != 1 ||
      !PyTuple_Check(tensors = PyTuple_GET_ITEM(args, 0))) {
    PyErr_SetString(PyExc_TypeError, "a call takes one tuple of tensors");
    return nullptr;
  }
  const Py_ssize_t n = PyTuple_GET_SIZE(tensors);
  uintptr_t at[16];
  if (n != (Py_ssize_t)p.inputs.size() || n > 16) Py_RETURN_NOTIMPLEMENTED;
  for (Py_ssize_t i = 0; i < n; ++i) {
    PyObject* v = PyTuple_GET_ITEM(tensors, i);
    if (!THPVariable_CheckExact(v)) Py_RETURN_NOTIMPLEMENTED;
    const at::Tensor& t = THPVariable_Unpack(v);
    const Input& in = p.inputs[i];
    if (!t.is_cuda() || t.scalar_type() != in.dtype || t.layout() != at::kStrided || t.get_device() != p.device ||
        !t.sizes().equals(in.shape) || !t.is_contiguous())
      Py_RETURN_NOTIMPLEMENTED;
    at[i] = reinterpret_cast<uintptr_t>(t.const_data_ptr());
    if (at[i] % 16) Py_RETURN_NOTIMPLEMENTED;
  }
  if (c10::cuda::current_device() != p.device) Py_RETURN_NOTIMPLEMENTED;
  at::Tensor out = at::empty(p.out_shape, at::TensorOptions().dtype(p.out_dtype).device(
                                              c10::Device(c10::kCUDA, (c10::DeviceIndex)p.device)));
  const uintptr_t to = reinterpret_cast<uintptr_t>(out.mutable_data_ptr());
  if (to % 16) Py_RETURN_NOTIMPLEMENTED;
  alignas(64) char block[kMaxBlock];
  std::memcpy(block, p.block.data(), p.block.size());
  for (const Patch& q : p.patches) {
    const uint64_t v = q.tensor < 0 ? to : at[q.tensor];
    std::memcpy(block + q.at, &v, 8);
  }
  for (const Map& q : p.maps)
    if (p.encode(block + q.at, q.dtype, reinterpret_cast<const void*>(at[q.tensor]), q.dims, q.strides, q.box))
      Py_RETURN_NOTIMPLEMENTED;
  void* stream = c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)p.device).stream();
  if (p.launch(p.module, p.kernel.c_str(), &p.cfg, block, p.block.size(), stream)) Py_RETURN_NOTIMPLEMENTED;
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

PyTypeObject CallType = {PyVarObject_HEAD_INIT(nullptr, 0)};

PyModuleDef module_def = {PyModuleDef_HEAD_INIT, "molten_call", "The short host path of one model operator.", -1,
                          nullptr, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_molten_call() {
  CallType.tp_name = "molten_call.Call";
  CallType.tp_basicsize = sizeof(Call);
  CallType.tp_flags = Py_TPFLAGS_DEFAULT;
  CallType.tp_doc = "call(tensors) -> output tensor, or NotImplemented";
  CallType.tp_new = call_new;
  CallType.tp_dealloc = call_dealloc;
  CallType.tp_call = call_call;
  if (PyType_Ready(&CallType) < 0) return nullptr;
  PyObject* m = PyModule_Create(&module_def);
  if (!m) return nullptr;
  Py_INCREF(&CallType);
  if (PyModule_AddObject(m, "Call", reinterpret_cast<PyObject*>(&CallType)) < 0) {
    Py_DECREF(&CallType);
    Py_DECREF(m);
    return nullptr;
  }
  return m;
}
