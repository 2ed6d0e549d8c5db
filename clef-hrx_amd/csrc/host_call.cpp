// Calls from the Python binding into the C ABI: an extension module whose
// functions do in C++ what the binding did per call in Python (argument
// conversion with the device and contiguity checks, the current stream, output
// allocation, the status check). A small projection is two launches of about
// 3 us each; the Python side of it took longer than the GPU.
//
//   entry(address, kinds): a handle for launch and value; kinds has one
//     letter per parameter, 'p' pointer or 'i' integer.
//   launch(entry, *args): entry(args.., current stream). A pointer argument is
//     a tensor (its device pointer), None (NULL) or an int address; an integer
//     is anything with __index__, as through ctypes. A nonzero status goes to
//     the function given to set_check, which raises.
//   value(entry, *args): entry(args..) as int64 (size functions).
//   pointer(tensor): its device pointer, checked as an argument is.
//   holds(device, tensor, dtype, count, ..): whether each is a contiguous tensor of
//     that dtype and at least count elements on that device (-1: the host).
//   empty(like, dtype, *sizes): torch.empty on like's device.
//   linear(entry, bytes_entry, x, weight, bias, activation, residual, out, dtype):
//     clef_linear with its workspace and output, the output returned; None, and
//     nothing done, unless every operand is as the entry takes it (the caller
//     finds out what is wrong).
//   linear_gate_up(entry, bytes_entry, x, gate, up, activation, gate_bias, up_bias,
//     out): clef_linear_gate_up likewise.
//   matrix(buffer, dtype, byte, rows, cols, row_step, col_step): a 2-d tensor of
//     dtype on buffer's memory from its byte `byte`, steps in elements; bounds
//     and alignment checked. (torch's view and as_strided take 1.4 us each.)
//
// Every entry takes integers and pointers only, which the x86-64 calling
// convention passes in 64-bit registers and stack slots.
#include <Python.h>

#include <ATen/ops/empty.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstdint>
#include <cstring>
#include <deque>
#include <utility>

#include "build_id.inc"  // CLEF_BUILD_ID, generated by the Makefile
#include "host_abi.inc"  // CLEF_TORCH_VERSION, likewise

namespace {

constexpr int kMaxArgs = 24;

struct Entry {
  void* f;
  uint32_t pointers;  // bit i: parameter i is a pointer
  int args;
};
std::deque<Entry> g_entries;  // handles are addresses of its elements; kept for the process

PyObject* g_check = nullptr;       // called with a nonzero status
PyObject* g_device = nullptr;      // torch._C._cuda_getDevice
PyObject* g_raw_stream = nullptr;  // torch._C._cuda_getCurrentRawStream

template <size_t... I>
int64_t invoke(void* f, const int64_t* v, std::index_sequence<I...>) {
  return reinterpret_cast<int64_t (*)(decltype((void)I, int64_t{})...)>(f)(v[I]...);
}
using Invoker = int64_t (*)(void*, const int64_t*);
template <size_t N>
int64_t invoke_n(void* f, const int64_t* v) {
  return invoke(f, v, std::make_index_sequence<N>{});
}
template <size_t... N>
constexpr Invoker pick(size_t n, std::index_sequence<N...>) {
  constexpr Invoker table[] = {&invoke_n<N>...};
  return table[n];
}

bool tensor_pointer(PyObject* o, int64_t& out) {
  const at::Tensor& t = THPVariable_Unpack(o);
  if (!t.is_cuda() || !t.is_contiguous()) {
    PyErr_SetString(PyExc_AssertionError, "device tensors must be contiguous CUDA tensors");
    return false;
  }
  out = reinterpret_cast<int64_t>(t.data_ptr());
  return true;
}

bool convert(PyObject* o, bool pointer, int64_t& out) {
  if (PyLong_Check(o)) {
    // device addresses and sizes below 2^64
    out = static_cast<int64_t>(PyLong_AsUnsignedLongLongMask(o));
    return !PyErr_Occurred();
  }
  if (pointer && o == Py_None) {
    out = 0;
    return true;
  }
  if (pointer && THPVariable_Check(o)) return tensor_pointer(o, out);
  if (!pointer && PyIndex_Check(o)) {
    PyObject* i = PyNumber_Index(o);
    if (i == nullptr) return false;
    out = static_cast<int64_t>(PyLong_AsUnsignedLongLongMask(i));
    Py_DECREF(i);
    return !PyErr_Occurred();
  }
  PyErr_Format(PyExc_TypeError, "unsupported argument type %s", Py_TYPE(o)->tp_name);
  return false;
}

// The handle args[0] and the arguments behind it, `missing` fewer than the
// entry has.
bool arguments(PyObject* const* args, Py_ssize_t n, int missing, const Entry*& entry, int64_t* v) {
  entry = n < 1 ? nullptr : static_cast<const Entry*>(PyLong_AsVoidPtr(args[0]));
  if (entry == nullptr) {
    if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "no entry");
    return false;
  }
  if (n - 1 != entry->args - missing) {
    PyErr_Format(PyExc_TypeError, "entry takes %d arguments (%zd given)", entry->args - missing, n - 1);
    return false;
  }
  for (Py_ssize_t i = 1; i < n; ++i)
    if (!convert(args[i], (entry->pointers >> (i - 1)) & 1, v[i - 1])) return false;
  return true;
}

PyObject* entry(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 2) {
    PyErr_SetString(PyExc_TypeError, "entry(address, kinds) expected");
    return nullptr;
  }
  Entry e{PyLong_AsVoidPtr(args[0]), 0, 0};
  Py_ssize_t count = 0;
  const char* kinds = PyErr_Occurred() ? nullptr : PyUnicode_AsUTF8AndSize(args[1], &count);
  if (kinds == nullptr) return nullptr;
  if (e.f == nullptr || count > kMaxArgs) {
    PyErr_SetString(PyExc_ValueError, "no entry, or more than 24 parameters");
    return nullptr;
  }
  e.args = static_cast<int>(count);
  for (int i = 0; i < e.args; ++i) e.pointers |= static_cast<uint32_t>(kinds[i] == 'p') << i;
  g_entries.push_back(e);
  return PyLong_FromVoidPtr(&g_entries.back());
  END_HANDLE_TH_ERRORS
}

PyObject* launch(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  const Entry* entry;
  int64_t v[kMaxArgs];
  if (!arguments(args, n, 1, entry, v)) return nullptr;
  PyObject* device = PyObject_CallNoArgs(g_device);
  if (device == nullptr) return nullptr;
  PyObject* stream = PyObject_CallOneArg(g_raw_stream, device);
  Py_DECREF(device);
  if (stream == nullptr) return nullptr;
  const bool ok = convert(stream, true, v[n - 1]);
  Py_DECREF(stream);
  if (!ok) return nullptr;
  const Invoker call = pick(static_cast<size_t>(n), std::make_index_sequence<kMaxArgs + 1>{});
  int32_t rc;
  Py_BEGIN_ALLOW_THREADS
  rc = static_cast<int32_t>(call(entry->f, v));
  Py_END_ALLOW_THREADS
  if (rc != 0) {
    PyObject* r = PyObject_CallFunction(g_check, "i", rc);
    if (r == nullptr) return nullptr;
    Py_DECREF(r);
  }
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

PyObject* value(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  const Entry* entry;
  int64_t v[kMaxArgs];
  if (!arguments(args, n, 0, entry, v)) return nullptr;
  return PyLong_FromLongLong(pick(static_cast<size_t>(n - 1), std::make_index_sequence<kMaxArgs + 1>{})(entry->f, v));
  END_HANDLE_TH_ERRORS
}

PyObject* pointer(PyObject*, PyObject* o) {
  HANDLE_TH_ERRORS
  int64_t p;
  if (!THPVariable_Check(o)) {
    PyErr_SetString(PyExc_TypeError, "tensor expected");
    return nullptr;
  }
  if (!tensor_pointer(o, p)) return nullptr;
  return PyLong_FromUnsignedLongLong(static_cast<uint64_t>(p));
  END_HANDLE_TH_ERRORS
}

PyObject* holds(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  bool all = n >= 1 && n % 3 == 1;
  for (Py_ssize_t i = 1; all && i < n; i += 3) all = THPVariable_Check(args[i]) && THPDtype_Check(args[i + 1]);
  if (!all) {
    PyErr_SetString(PyExc_TypeError, "holds(device, tensor, dtype, count, ..) expected");
    return nullptr;
  }
  const int64_t device = PyLong_AsLongLong(args[0]);
  if (device == -1 && PyErr_Occurred()) return nullptr;
  for (Py_ssize_t i = 1; i < n; i += 3) {
    const int64_t count = PyLong_AsLongLong(args[i + 2]);
    if (count == -1 && PyErr_Occurred()) return nullptr;
    const at::Tensor& t = THPVariable_Unpack(args[i]);
    const int64_t on = t.is_cuda() ? t.get_device() : t.is_cpu() ? -1 : -2;
    all = all && t.scalar_type() == reinterpret_cast<THPDtype*>(args[i + 1])->scalar_type && t.numel() >= count &&
          on == device && t.is_contiguous();
  }
  return PyBool_FromLong(all);
  END_HANDLE_TH_ERRORS
}

PyObject* empty(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n < 3 || n > 6 || !THPVariable_Check(args[0]) || !THPDtype_Check(args[1])) {
    PyErr_SetString(PyExc_TypeError, "empty(like, dtype, *sizes) expects a tensor, a dtype and one to four sizes");
    return nullptr;
  }
  int64_t sizes[4];
  for (Py_ssize_t i = 2; i < n; ++i) {
    sizes[i - 2] = PyLong_AsLongLong(args[i]);
    if (sizes[i - 2] == -1 && PyErr_Occurred()) return nullptr;
  }
  const at::Tensor& like = THPVariable_Unpack(args[0]);
  at::Tensor out;
  {
    pybind11::gil_scoped_release no_gil;
    out = at::empty(at::IntArrayRef(sizes, static_cast<size_t>(n - 2)),
                    at::TensorOptions().device(like.device()).dtype(
                        reinterpret_cast<THPDtype*>(args[1])->scalar_type));
  }
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// The operands of the bf16 products. Each function gives false for what the C entry
// would not take.
struct Rows {
  int64_t at = 0, rows = 0, cols = 0, pitch = 0;
};

// Rows of contiguous elements of `type` on `device`, a matrix or a column range of one.
bool rows_of(PyObject* o, at::ScalarType type, int64_t device, Rows& r) {
  if (!THPVariable_Check(o)) return false;
  const at::Tensor& t = THPVariable_Unpack(o);
  if (t.dim() != 2 || t.scalar_type() != type || !t.is_cuda() || t.get_device() != device) return false;
  r.rows = t.size(0), r.cols = t.size(1);
  r.at = reinterpret_cast<int64_t>(t.data_ptr());
  r.pitch = r.rows > 1 && !t.is_contiguous() ? t.stride(0) : r.cols;
  return t.is_contiguous() || ((r.cols <= 1 || t.stride(1) == 1) && r.pitch >= r.cols);
}

// A bias of n values, or none.
bool bias_of(PyObject* o, int64_t n, int64_t device, int64_t& at, int64_t& f32) {
  at = f32 = 0;
  if (o == Py_None) return true;
  if (!THPVariable_Check(o)) return false;
  const at::Tensor& t = THPVariable_Unpack(o);
  f32 = t.scalar_type() == at::kFloat;
  at = reinterpret_cast<int64_t>(t.data_ptr());
  return (f32 || t.scalar_type() == at::kBFloat16) && t.dim() == 1 && t.size(0) == n && t.is_cuda() &&
         t.get_device() == device && t.is_contiguous();
}

at::Tensor empty_like(PyObject* o, at::ScalarType type, at::IntArrayRef sizes) {
  pybind11::gil_scoped_release no_gil;
  return at::empty(sizes, at::TensorOptions().device(THPVariable_Unpack(o).device()).dtype(type));
}

bool current(int64_t& device, int64_t& stream) {
  PyObject* d = PyObject_CallNoArgs(g_device);
  if (d == nullptr) return false;
  device = PyLong_AsLongLong(d);
  PyObject* s = PyObject_CallOneArg(g_raw_stream, d);
  Py_DECREF(d);
  if (s == nullptr) return false;
  const bool ok = convert(s, true, stream);
  Py_DECREF(s);
  return ok;
}

// The entry with v's arguments, workspace, its bytes and the stream behind them; the
// status to the function given to set_check.
bool call_with_workspace(const Entry* entry, const Entry* bytes_entry, PyObject* like, int64_t m, int64_t n, int64_t k,
                         int64_t gate_up, int64_t* v, size_t args, int64_t stream) {
  at::Tensor scratch;
  v[args] = v[args + 1] = 0;
  if (m > 8) {  // few rows need none
    const int64_t sizes[] = {m, n, k, gate_up};
    const int64_t bytes = pick(4, std::make_index_sequence<kMaxArgs + 1>{})(bytes_entry->f, sizes);
    if (bytes > 0) {
      scratch = empty_like(like, at::kByte, bytes);
      v[args] = reinterpret_cast<int64_t>(scratch.data_ptr());
      v[args + 1] = bytes;
    }
  }
  v[args + 2] = stream;
  const Invoker call = pick(args + 3, std::make_index_sequence<kMaxArgs + 1>{});
  int32_t rc;
  Py_BEGIN_ALLOW_THREADS
  rc = static_cast<int32_t>(call(entry->f, v));
  Py_END_ALLOW_THREADS
  if (rc == 0) return true;
  PyObject* r = PyObject_CallFunction(g_check, "i", rc);
  Py_XDECREF(r);
  return r != nullptr;
}

// args[0] and args[1] as handles, args[at] as an activation's code.
bool linear_entries(PyObject* const* args, Py_ssize_t n, Py_ssize_t at, const Entry*& entry, const Entry*& bytes_entry,
                    int64_t& activation) {
  if (n != 9) {
    PyErr_SetString(PyExc_TypeError, "two entries and seven arguments expected");
    return false;
  }
  entry = static_cast<const Entry*>(PyLong_AsVoidPtr(args[0]));
  bytes_entry = entry != nullptr ? static_cast<const Entry*>(PyLong_AsVoidPtr(args[1])) : nullptr;
  if (bytes_entry == nullptr) {
    if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "no entry");
    return false;
  }
  activation = PyLong_AsLongLong(args[at]);
  return activation != -1 || !PyErr_Occurred();
}

PyObject* linear(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  const Entry *entry, *bytes_entry;
  int64_t act, device, stream, v[kMaxArgs];
  if (!linear_entries(args, n, 5, entry, bytes_entry, act) || !current(device, stream)) return nullptr;
  if (act < 0) Py_RETURN_NONE;
  PyObject *const x = args[2], *const weight = args[3], *const residual = args[6], *const out = args[7], *const dtype = args[8];
  Rows rx, rw, rr, ro;
  int64_t bias, bias_f32;
  if (!rows_of(x, at::kBFloat16, device, rx) || !rows_of(weight, at::kBFloat16, device, rw) || rx.cols != rw.cols ||
      !bias_of(args[4], rw.rows, device, bias, bias_f32))
    Py_RETURN_NONE;
  rr.pitch = rw.rows;
  if (residual != Py_None &&
      (!rows_of(residual, at::kBFloat16, device, rr) || rr.rows != rx.rows || rr.cols != rw.rows))
    Py_RETURN_NONE;
  at::ScalarType type = at::kBFloat16;
  if (dtype != Py_None) {
    if (!THPDtype_Check(dtype)) Py_RETURN_NONE;
    type = reinterpret_cast<THPDtype*>(dtype)->scalar_type;
  } else if (out != Py_None && THPVariable_Check(out)) {
    type = THPVariable_Unpack(out).scalar_type();
  }
  if (type != at::kBFloat16 && type != at::kFloat) Py_RETURN_NONE;
  at::Tensor made;
  if (out == Py_None) {
    const int64_t sizes[] = {rx.rows, rw.rows};
    made = empty_like(x, type, at::IntArrayRef(sizes, 2));
    ro.at = reinterpret_cast<int64_t>(made.data_ptr()), ro.pitch = rw.rows;
  } else if (!rows_of(out, type, device, ro) || ro.rows != rx.rows || ro.cols != rw.rows) {
    Py_RETURN_NONE;
  }
  const int64_t given[] = {rx.at, rx.rows, rx.cols,  rx.pitch, rw.at,              rw.rows, rw.pitch, bias, bias_f32,
                           act,   rr.at,   rr.pitch, ro.at,    type == at::kFloat, ro.pitch};
  constexpr size_t count = sizeof(given) / sizeof(*given);
  std::memcpy(v, given, sizeof(given));
  if (!call_with_workspace(entry, bytes_entry, x, rx.rows, rw.rows, rx.cols, 0, v, count, stream)) return nullptr;
  if (made.defined()) return THPVariable_Wrap(std::move(made));
  Py_INCREF(out);
  return out;
  END_HANDLE_TH_ERRORS
}

PyObject* linear_gate_up(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  const Entry *entry, *bytes_entry;
  int64_t act, device, stream, v[kMaxArgs];
  if (!linear_entries(args, n, 5, entry, bytes_entry, act) || !current(device, stream)) return nullptr;
  if (act < 0) Py_RETURN_NONE;
  PyObject *const x = args[2], *const out = args[8];
  Rows rx, rg, ru, ro;
  int64_t gate_bias, gate_f32, up_bias, up_f32;
  if (!rows_of(x, at::kBFloat16, device, rx) || !rows_of(args[3], at::kBFloat16, device, rg) ||
      !rows_of(args[4], at::kBFloat16, device, ru) || rx.cols != rg.cols || rg.rows != ru.rows || rg.cols != ru.cols ||
      rg.pitch != ru.pitch || !bias_of(args[6], rg.rows, device, gate_bias, gate_f32) ||
      !bias_of(args[7], rg.rows, device, up_bias, up_f32) || (gate_bias != 0 && up_bias != 0 && gate_f32 != up_f32))
    Py_RETURN_NONE;
  at::Tensor made;
  if (out == Py_None) {
    const int64_t sizes[] = {rx.rows, rg.rows};
    made = empty_like(x, at::kBFloat16, at::IntArrayRef(sizes, 2));
    ro.at = reinterpret_cast<int64_t>(made.data_ptr()), ro.pitch = rg.rows;
  } else if (!rows_of(out, at::kBFloat16, device, ro) || ro.rows != rx.rows || ro.cols != rg.rows) {
    Py_RETURN_NONE;
  }
  const int64_t given[] = {rx.at,    rx.rows,   rx.cols, rx.pitch,          rg.at, ru.at, rg.rows,
                           rg.pitch, gate_bias, up_bias, gate_f32 | up_f32, act,   ro.at, ro.pitch};
  constexpr size_t count = sizeof(given) / sizeof(*given);
  std::memcpy(v, given, sizeof(given));
  if (!call_with_workspace(entry, bytes_entry, x, rx.rows, rg.rows, rx.cols, 1, v, count, stream)) return nullptr;
  if (made.defined()) return THPVariable_Wrap(std::move(made));
  Py_INCREF(out);
  return out;
  END_HANDLE_TH_ERRORS
}

PyObject* matrix(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 7 || !THPVariable_Check(args[0]) || !THPDtype_Check(args[1])) {
    PyErr_SetString(PyExc_TypeError, "matrix(buffer, dtype, byte, rows, cols, row_step, col_step) expected");
    return nullptr;
  }
  int64_t v[5];
  for (int i = 0; i < 5; ++i) {
    v[i] = PyLong_AsLongLong(args[2 + i]);
    if (v[i] == -1 && PyErr_Occurred()) return nullptr;
  }
  const auto [byte, rows, cols, row_step, col_step] = v;
  const at::Tensor& buffer = THPVariable_Unpack(args[0]);
  const caffe2::TypeMeta dtype = c10::scalarTypeToTypeMeta(reinterpret_cast<THPDtype*>(args[1])->scalar_type);
  const int64_t item = static_cast<int64_t>(dtype.itemsize());
  constexpr int64_t most = int64_t{1} << 29;  // of each factor: the sum below stays in 64 bits
  bool fits = buffer.is_contiguous() && !buffer.requires_grad() && byte >= 0;
  for (int i = 1; i < 5; ++i) fits = fits && v[i] >= 0 && v[i] <= most;
  if (fits && rows > 0 && cols > 0)
    fits = byte <= static_cast<int64_t>(buffer.nbytes()) &&
           byte + ((rows - 1) * row_step + (cols - 1) * col_step + 1) * item <= static_cast<int64_t>(buffer.nbytes());
  const int64_t at = fits ? buffer.storage_offset() * static_cast<int64_t>(buffer.itemsize()) + byte : 0;
  if (!fits || at % item != 0) {
    PyErr_SetString(PyExc_ValueError, "matrix does not lie in its buffer");
    return nullptr;
  }
  at::Tensor out = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(buffer.storage()), buffer.key_set(), dtype);
  c10::TensorImpl* impl = out.unsafeGetTensorImpl();
  impl->set_storage_offset(at / item);
  const int64_t sizes[] = {rows, cols}, steps[] = {row_step, col_step};
  impl->set_sizes_and_strides(at::IntArrayRef(sizes, 2), at::IntArrayRef(steps, 2));
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

PyObject* set_check(PyObject*, PyObject* o) {
  Py_XINCREF(o);
  Py_XSETREF(g_check, o);
  Py_RETURN_NONE;
}

PyMethodDef methods[] = {
    {"entry", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&entry)), METH_FASTCALL, nullptr},
    {"launch", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&launch)), METH_FASTCALL, nullptr},
    {"value", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&value)), METH_FASTCALL, nullptr},
    {"pointer", &pointer, METH_O, nullptr},
    {"holds", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&holds)), METH_FASTCALL, nullptr},
    {"empty", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&empty)), METH_FASTCALL, nullptr},
    {"matrix", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&matrix)), METH_FASTCALL, nullptr},
    {"linear", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&linear)), METH_FASTCALL, nullptr},
    {"linear_gate_up", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&linear_gate_up)), METH_FASTCALL, nullptr},
    {"set_check", &set_check, METH_O, nullptr},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef module_def = {PyModuleDef_HEAD_INIT, "clef_host", nullptr, -1, methods};

}  // namespace

namespace {

// The functions above use torch's and Python's class layouts as their headers
// gave them: no other version of either loads this module. (Written with
// functions of Python's stable interface only.)
bool built_for_this_process() {
#define CLEF_STR2(x) #x
#define CLEF_STR(x) CLEF_STR2(x)
  constexpr const char* python = CLEF_STR(PY_MAJOR_VERSION) "." CLEF_STR(PY_MINOR_VERSION) ".";
  PyObject* torch = PyImport_ImportModule("torch");
  PyObject* version = torch != nullptr ? PyObject_GetAttrString(torch, "__version__") : nullptr;
  PyObject* text = version != nullptr ? PyObject_Str(version) : nullptr;
  const char* found = text != nullptr ? PyUnicode_AsUTF8AndSize(text, nullptr) : nullptr;
  const bool same = found != nullptr && std::strcmp(found, CLEF_TORCH_VERSION) == 0 &&
                    std::strncmp(Py_GetVersion(), python, std::strlen(python)) == 0;
  if (found != nullptr && !same)
    PyErr_Format(PyExc_ImportError,
                 "the call module was built for torch %s and Python %sx, this is torch %s and Python %s; run `make -C "
                 "clef-hrx_amd`",
                 CLEF_TORCH_VERSION, python, found, Py_GetVersion());
  Py_XDECREF(text);
  Py_XDECREF(version);
  Py_XDECREF(torch);
  return same;
}

}  // namespace

PyMODINIT_FUNC PyInit_clef_host() {
  if (!built_for_this_process()) return nullptr;
  PyObject* c = PyImport_ImportModule("torch._C");
  if (c == nullptr) return nullptr;
  g_device = PyObject_GetAttrString(c, "_cuda_getDevice");
  g_raw_stream = g_device != nullptr ? PyObject_GetAttrString(c, "_cuda_getCurrentRawStream") : nullptr;
  Py_DECREF(c);
  if (g_raw_stream == nullptr) return nullptr;
  PyObject* m = PyModule_Create(&module_def);
  if (m != nullptr) PyModule_AddStringConstant(m, "build_id", CLEF_BUILD_ID);
  return m;
}
