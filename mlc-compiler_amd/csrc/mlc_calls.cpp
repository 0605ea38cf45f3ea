// Direct calls of the operators of mlc.ops, as a CPython module: what of a call does not
// depend on its operands' values is looked up by their signature (types, shapes, strides,
// device, place within 16 bytes), addresses are put into the launches' arguments, results
// and shared memory come from torch's allocator, and mlc_launch of libmlc_hip.so does the
// rest. One token's operators are bound by the host: a call with four to eight operands
// takes 4-6 us, of which a launch is 2.3 and a result 1; the same in Python took 8-10.
//
// Where something looks on (a tracer, a mode, a transform) a call is handed back, to go through
// torch's dispatcher; a profiler gets a record from here.
//
// Nothing is kept by an operand's address or identity. The table is used under the
// interpreter's lock, which launches are made without.

#define PY_SSIZE_T_CLEAN
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/PyInterpreter.h>
#include <torch/csrc/autograd/python_variable.h>

#include <ATen/PythonTorchFunctionTLS.h>
#include <ATen/ops/empty.h>
#include <ATen/record_function.h>
#include <c10/core/AutogradState.h>
#include <c10/core/GradMode.h>
#include <c10/core/impl/DeviceGuardImplInterface.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>

#include <cstdint>
#include <cstring>
#include <iterator>
#include <memory>
#include <optional>
#include <string>
#include <unordered_map>
#include <vector>

namespace {

using launch_fn = int (*)(void*, uint32_t, uint32_t, uint32_t, const void*, size_t, void*);
using poll_fn = int (*)(void*, int32_t*);

constexpr Py_ssize_t kMostOperands = 16, kMostResults = 2;
constexpr size_t kMostBytes = 1024;  // of a launch's arguments

// The flags of a call. kDispatched: torch's dispatcher has brought it, and whoever looks on
// has seen it.
enum { kPoll = 1, kDispatched = 2 };

// by number, as mlc.ops gives it
constexpr const char* kOperators[] = {"mlc::rotary", "mlc::attention", "mlc::cache_append", "mlc::cache_attention"};

// tensors that stand for others
constexpr c10::DispatchKeySet kWrapped({c10::DispatchKey::Functionalize, c10::DispatchKey::FuncTorchBatched,
                                        c10::DispatchKey::FuncTorchGradWrapper, c10::DispatchKey::Batched,
                                        c10::DispatchKey::Python, c10::DispatchKey::ZeroTensor});

// and what is traced by: a direct call would leave the allocation of its result in a graph
// in the operator's place
constexpr c10::DispatchKeySet kTraced({c10::DispatchKey::Tracer, c10::DispatchKey::Functionalize,
                                       c10::DispatchKey::Python, c10::DispatchKey::PreDispatch,
                                       c10::DispatchKey::PythonDispatcher});

bool is_traced() {
  const auto keys = c10::impl::tls_local_dispatch_key_set();
  return c10::impl::TorchDispatchModeTLS::any_modes_set() || (keys.included_ - keys.excluded_).has_any(kTraced);
}

// torch.utils._device.DeviceContext: a function mode that fills in factories' devices alone
PyTypeObject* device_context = nullptr;

// Whether a function mode (torch.overrides) wants to see calls.
bool is_watched() {
  if (!at::impl::torch_function_mode_enabled()) return false;
  for (int64_t i = 0; i < at::impl::PythonTorchFunctionTLS::stack_len(); ++i) {
    PyObject* const mode = at::impl::PythonTorchFunctionTLS::get_stack_at(i)->ptr(getPyInterpreter());
    if (Py_TYPE(mode) != device_context) return true;
  }
  return false;
}

struct Launch {
  void* fn;
  uint32_t grid, block;
  std::vector<uint8_t> places;  // of its pointers among a call's addresses
  std::string tail;             // and what follows them
};

struct Entry {
  launch_fn launch;
  std::vector<Launch> launches;
  Py_ssize_t changed;  // operands that change: the first ones
  int64_t workspace;   // bytes that the launches share
  poll_fn poll;        // null: cannot meet an invalid input
  void* ctx;
  uint64_t error;
};

std::unordered_map<std::string, std::shared_ptr<Entry>>& table() {
  static auto* entries = new std::unordered_map<std::string, std::shared_ptr<Entry>>;
  return *entries;
}

// Bytes from a tensor's first value to behind its last.
uint64_t extent(const at::Tensor& x) {
  int64_t last = 0;
  for (int64_t i = 0; i < x.dim(); ++i) {
    if (x.size(i) == 0) return 0;
    last += (x.size(i) - 1) * x.stride(i);
  }
  return static_cast<uint64_t>(last + 1) * x.element_size();
}

template <class T> void put(std::string& key, T x) {
  key.append(reinterpret_cast<const char*>(&x), sizeof(x));
}

// call(operator, operands, options, results, stream_of, flags), with the current stream's
// address from stream_of(device):
//   a tuple of results: done;  bytes: the signature, of which nothing is known yet;
//   None: not plain tensors of one GPU, or someone looks on (but for kDispatched);  False: an
//   operand asks for a gradient;  True: an earlier call met an invalid input (where kPoll);
//   NotImplemented: the device is not the current one;  Ellipsis: an operand that changes
//   lies in another's memory;  an int: the launch's error.
PyObject* call(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 6 || !PyTuple_Check(args[1]) || !PyTuple_Check(args[2])) {
    PyErr_SetString(PyExc_TypeError, "call(operator, operands, options, results, stream_of, flags)");
    return nullptr;
  }
  const Py_ssize_t operands = PyTuple_GET_SIZE(args[1]), results = PyLong_AsSsize_t(args[3]);
  if (operands < 1 || operands > kMostOperands || results < 0 || results > kMostResults || results > operands) {
    if (!PyErr_Occurred()) PyErr_SetString(PyExc_TypeError, "call: too many operands or results");
    return nullptr;
  }
  const long op = PyLong_AsLong(args[0]), flags = PyLong_AsLong(args[5]);
  if (PyErr_Occurred()) return nullptr;

  const at::Tensor* x[kMostOperands];
  // forward mode goes on where gradients are off, and ends in inference mode
  const bool grad = at::GradMode::is_enabled(), forward = c10::AutogradState::get_tls_state().get_fw_grad_mode();
  bool plain = (flags & kDispatched) || !(is_traced() || is_watched());
  int device = -1;
  for (Py_ssize_t i = 0; i < operands; ++i) {
    PyObject* const o = PyTuple_GET_ITEM(args[1], i);
    x[i] = nullptr;
    if (o == Py_None) continue;
    if (!THPVariable_Check(o)) {
      PyErr_Format(PyExc_TypeError, "operand %zd: a tensor expected, got %s", i, Py_TYPE(o)->tp_name);
      return nullptr;
    }
    x[i] = &THPVariable_Unpack(o);
    if ((grad && x[i]->requires_grad()) || (forward && x[i]->_fw_grad(0).defined())) Py_RETURN_FALSE;
    plain = plain && THPVariable_CheckExact(o) && x[i]->is_cuda() && x[i]->layout() == at::kStrided &&
            x[i]->has_storage() && !x[i]->is_neg() && !x[i]->is_conj() && !x[i]->key_set().has_any(kWrapped);
    if (plain) {
      if (device < 0) device = x[i]->get_device();
      plain = device == x[i]->get_device();
    }
  }
  if (!plain || x[0] == nullptr) Py_RETURN_NONE;
  if (c10::impl::getDeviceGuardImpl(c10::kCUDA)->getDevice().index() != device) Py_RETURN_NOTIMPLEMENTED;

  std::string key;
  key.reserve(512);
  put(key, static_cast<int8_t>(op));
  for (Py_ssize_t i = 0; i < PyTuple_GET_SIZE(args[2]); ++i) {
    PyObject* const o = PyTuple_GET_ITEM(args[2], i);
    if (o == Py_None) {
      key.push_back('n');
    } else if (PyBool_Check(o)) {
      key.push_back(o == Py_True ? 't' : 'f');
    } else {
      const double v = PyFloat_AsDouble(o);
      if (v == -1.0 && PyErr_Occurred()) return nullptr;
      key.push_back('d');
      put(key, v);
    }
  }
  uint64_t at[kMostOperands + kMostResults + 3];
  for (Py_ssize_t i = 0; i < operands; ++i) {
    at[i] = 0;
    if (x[i] == nullptr) {
      key.push_back('n');
      continue;
    }
    at[i] = reinterpret_cast<uint64_t>(x[i]->const_data_ptr());
    key.push_back('x');
    put(key, static_cast<int8_t>(x[i]->scalar_type()));
    put(key, static_cast<int8_t>(at[i] % 16));
    put(key, static_cast<int16_t>(device));
    put(key, static_cast<int32_t>(x[i]->dim()));
    for (const int64_t s : x[i]->sizes()) put(key, s);
    for (const int64_t s : x[i]->strides()) put(key, s);
  }
  const auto found = table().find(key);
  if (found == table().end()) return PyBytes_FromStringAndSize(key.data(), static_cast<Py_ssize_t>(key.size()));
  const std::shared_ptr<Entry> entry = found->second;

  for (Py_ssize_t i = 0; i < entry->changed && i < operands; ++i)
    if (x[i] != nullptr) at[i] = reinterpret_cast<uint64_t>(x[i]->mutable_data_ptr());  // a lazy copy is made now
  if (entry->changed > 0) {
    uint64_t end[kMostOperands];
    for (Py_ssize_t i = 0; i < operands; ++i) end[i] = x[i] != nullptr ? at[i] + extent(*x[i]) : 0;
    for (Py_ssize_t i = 0; i < entry->changed && i < operands; ++i)
      for (Py_ssize_t j = 0; j < operands; ++j)
        if (j != i && at[i] < end[j] && at[j] < end[i]) {
          Py_INCREF(Py_Ellipsis);
          return Py_Ellipsis;
        }
  }
  if (entry->poll != nullptr && (flags & kPoll)) {
    int32_t word = 0;
    const int rc = entry->poll(entry->ctx, &word);
    if (rc != 0) return PyLong_FromLong(rc);
    if (word != 0) Py_RETURN_TRUE;
  }
  std::vector<c10::IValue> inputs;  // outlives the record
  std::optional<at::RecordFunction> record;
  if (auto callbacks = at::getStepCallbacksUnlessEmpty(at::RecordScope::FUNCTION);
      callbacks.has_value() && !(flags & kDispatched) &&  // the dispatcher makes a record of its own
      op >= 0 && op < static_cast<long>(std::size(kOperators))) {
    record.emplace(std::move(*callbacks));
    if (record->needsInputs())
      for (Py_ssize_t i = 0; i < operands; ++i) inputs.push_back(x[i] ? c10::IValue(*x[i]) : c10::IValue());
    record->before(kOperators[op], &inputs);
  }
  PyObject* const index = PyLong_FromLong(device);
  if (index == nullptr) return nullptr;
  PyObject* const current = PyObject_CallOneArg(args[4], index);
  Py_DECREF(index);
  if (current == nullptr) return nullptr;
  void* const stream = PyLong_AsVoidPtr(current);
  Py_DECREF(current);
  if (PyErr_Occurred()) return nullptr;
  at::Tensor out[kMostResults], space;
  for (Py_ssize_t i = 0; i < results; ++i) {
    out[i] = at::empty(x[i]->sizes(), x[i]->options(), at::MemoryFormat::Contiguous);
    at[operands + i] = reinterpret_cast<uint64_t>(out[i].const_data_ptr());
  }
  uint64_t* const rest = at + operands + results;
  rest[0] = rest[1] = 0;
  rest[2] = entry->error;
  if (entry->workspace > 0) {
    space = at::empty({entry->workspace}, x[0]->options().dtype(at::kByte));
    rest[0] = reinterpret_cast<uint64_t>(space.const_data_ptr());
  }
  int rc = 0;
  Py_BEGIN_ALLOW_THREADS
  alignas(16) char arguments[kMostBytes];
  for (const Launch& l : entry->launches) {
    size_t size = 0;
    for (const uint8_t place : l.places) {
      std::memcpy(arguments + size, &at[place], sizeof(uint64_t));
      size += sizeof(uint64_t);
    }
    std::memcpy(arguments + size, l.tail.data(), l.tail.size());
    rc = entry->launch(l.fn, l.grid, l.block, 0, arguments, size + l.tail.size(), stream);
    if (rc != 0) break;
  }
  Py_END_ALLOW_THREADS
  if (rc != 0) return PyLong_FromLong(rc);
  for (Py_ssize_t i = 0; i < entry->changed && i < operands; ++i)  // autograd asks whether what it kept has changed
    if (x[i] != nullptr && !x[i]->is_inference()) x[i]->unsafeGetTensorImpl()->bump_version();
  PyObject* const made = PyTuple_New(results);
  if (made == nullptr) return nullptr;
  for (Py_ssize_t i = 0; i < results; ++i) PyTuple_SET_ITEM(made, i, THPVariable_Wrap(std::move(out[i])));
  return made;
  END_HANDLE_TH_ERRORS
}

// add(signature, addresses, changed, launch, launches, workspace, poll, ctx, error): launches are
// (function, grid, block, places, tail) with places below ``addresses``.
PyObject* add(PyObject*, PyObject* args) {
  HANDLE_TH_ERRORS
  const char* key;
  Py_ssize_t key_size;
  int addresses, changed;
  unsigned long long launch, poll, ctx, error;
  long long workspace;
  PyObject* launches;
  if (!PyArg_ParseTuple(args, "y#iiKO!LKKK", &key, &key_size, &addresses, &changed, &launch, &PyTuple_Type, &launches,
                        &workspace, &poll, &ctx, &error))
    return nullptr;
  auto entry = std::make_shared<Entry>();
  entry->launch = reinterpret_cast<launch_fn>(launch);
  entry->changed = changed < kMostOperands ? changed : 0;
  entry->workspace = workspace;
  entry->poll = reinterpret_cast<poll_fn>(poll);
  entry->ctx = reinterpret_cast<void*>(ctx);
  entry->error = error;
  for (Py_ssize_t i = 0; i < PyTuple_GET_SIZE(launches); ++i) {
    unsigned long long fn;
    Launch l;
    const char *places, *tail;
    Py_ssize_t places_size, tail_size;
    if (!PyArg_ParseTuple(PyTuple_GET_ITEM(launches, i), "KIIy#y#", &fn, &l.grid, &l.block, &places, &places_size,
                          &tail, &tail_size))
      return nullptr;
    l.fn = reinterpret_cast<void*>(fn);
    l.places.assign(places, places + places_size);
    l.tail.assign(tail, static_cast<size_t>(tail_size));
    bool fits = l.places.size() * sizeof(uint64_t) + l.tail.size() <= kMostBytes && launch != 0 && fn != 0;
    for (const uint8_t place : l.places) fits = fits && place < addresses;
    if (!fits) {
      PyErr_SetString(PyExc_ValueError, "add: a launch that does not fit");
      return nullptr;
    }
    entry->launches.push_back(std::move(l));
  }
  table()[std::string(key, static_cast<size_t>(key_size))] = std::move(entry);
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

PyObject* clear(PyObject*, PyObject*) {
  table().clear();
  Py_RETURN_NONE;
}

PyMethodDef kMethods[] = {
    {"call", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(call)), METH_FASTCALL, nullptr},
    {"add", add, METH_VARARGS, nullptr},
    {"clear", clear, METH_NOARGS, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_calls", nullptr, -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__calls() {
  PyObject* const torch_device = PyImport_ImportModule("torch.utils._device");
  if (torch_device == nullptr) return nullptr;
  PyObject* const type = PyObject_GetAttrString(torch_device, "DeviceContext");  // kept
  Py_DECREF(torch_device);
  if (type == nullptr) return nullptr;
  device_context = reinterpret_cast<PyTypeObject*>(type);
  return PyModule_Create(&kModule);
}
