// Reads pointer, shape, strides and element type out of an array-like Python
// object without depending on any array library at build time.
//
// Accepted, in this order:
//   * objects whose type publishes DLPack's C exchange functions (attribute
//     __dlpack_c_exchange_api__, torch 2.10 and later): one C call, an eighth of
//     the time of the next way;
//   * objects with data_ptr()/shape/stride()/element_size()/dtype - torch
//     tensors (the reference's e2e tests pass torch CUDA tensors,
//     python/hckernel/tests/test_e2e.py:72-75).  torch refuses to export bf16
//     through __cuda_array_interface__, so this branch comes first;
//   * objects with __cuda_array_interface__ (CuPy, Numba device arrays);
//   * objects with __array_interface__ (NumPy) - host memory.
// The reference does the same job with nanobind's ndarray caster
// (python/cpp/py-runtime/src/PyABI.cpp:23-37).
#pragma once

#include <pybind11/pybind11.h>

#include <cstdint>
#include <stdexcept>
#include <string>
#include <utility>
#include <vector>

namespace hc {

namespace py = pybind11;

enum class ElemKind { F32, F64, BF16, F16, I8, U8, I16, I32, I64, E4M3, Other };

struct ArrayArg {
  void *data = nullptr;
  std::vector<int64_t> shape;
  std::vector<int64_t> strides; // in elements
  int64_t itemsize = 0;
  ElemKind kind = ElemKind::Other;
  bool onDevice = false;
  int deviceIndex = -1; // -1: unknown or host

  int rank() const { return int(shape.size()); }
  // Rows are contiguous (last stride 1) - what every kernel here requires.
  bool rowMajor() const { return shape.empty() || strides.back() == 1 || shape.back() <= 1; }
};

inline const char *kindName(ElemKind k) {
  switch (k) {
  case ElemKind::F32: return "float32";
  case ElemKind::F64: return "float64";
  case ElemKind::BF16: return "bfloat16";
  case ElemKind::F16: return "float16";
  case ElemKind::I8: return "int8";
  case ElemKind::U8: return "uint8";
  case ElemKind::I16: return "int16";
  case ElemKind::I32: return "int32";
  case ElemKind::I64: return "int64";
  case ElemKind::E4M3: return "float8_e4m3fn";
  default: return "other";
  }
}

inline ElemKind kindFromTorchName(const std::string &name) {
  // str(tensor.dtype) is "torch.float32" etc.
  auto dot = name.rfind('.');
  std::string n = dot == std::string::npos ? name : name.substr(dot + 1);
  if (n == "float32" || n == "float") return ElemKind::F32;
  if (n == "float64" || n == "double") return ElemKind::F64;
  if (n == "bfloat16") return ElemKind::BF16;
  if (n == "float16" || n == "half") return ElemKind::F16;
  if (n == "int8") return ElemKind::I8;
  if (n == "uint8") return ElemKind::U8;
  if (n == "int16" || n == "short") return ElemKind::I16;
  if (n == "int32" || n == "int") return ElemKind::I32;
  if (n == "int64" || n == "long") return ElemKind::I64;
  if (n == "float8_e4m3fn") return ElemKind::E4M3;
  return ElemKind::Other;
}

inline ElemKind kindFromTypestr(const std::string &t, int64_t &itemsize) {
  // "<f4", "|i1", "<u2", ...
  if (t.size() < 3)
    return ElemKind::Other;
  char c = t[1];
  itemsize = std::stoll(t.substr(2));
  if (c == 'f') return itemsize == 4 ? ElemKind::F32 : itemsize == 8 ? ElemKind::F64
                     : itemsize == 2 ? ElemKind::F16 : ElemKind::Other;
  if (c == 'i') return itemsize == 1 ? ElemKind::I8 : itemsize == 2 ? ElemKind::I16
                     : itemsize == 4 ? ElemKind::I32 : itemsize == 8 ? ElemKind::I64
                     : ElemKind::Other;
  if (c == 'u') return itemsize == 1 ? ElemKind::U8 : ElemKind::Other;
  return ElemKind::Other;
}

inline ArrayArg arrayFromInterface(const py::dict &iface, bool onDevice) {
  ArrayArg a;
  a.onDevice = onDevice;
  auto data = iface["data"].cast<py::tuple>();
  a.data = reinterpret_cast<void *>(data[0].cast<uintptr_t>());
  a.kind = kindFromTypestr(iface["typestr"].cast<std::string>(), a.itemsize);
  for (auto d : iface["shape"].cast<py::tuple>())
    a.shape.push_back(d.cast<int64_t>());
  bool haveStrides = iface.contains("strides") && !iface["strides"].is_none();
  if (haveStrides) {
    for (auto s : iface["strides"].cast<py::tuple>()) {
      int64_t bytes = s.cast<int64_t>();
      if (a.itemsize == 0 || bytes % a.itemsize)
        throw std::runtime_error("Array strides are not a multiple of the element size");
      a.strides.push_back(bytes / a.itemsize);
    }
  } else {
    a.strides.assign(a.shape.size(), 1);
    for (int i = int(a.shape.size()) - 2; i >= 0; --i)
      a.strides[i] = a.strides[i + 1] * a.shape[i + 1];
  }
  return a;
}

// The kind of a dtype object.  torch's dtypes are singletons that live as long as
// torch does; naming one costs more than the rest of a tensor's reading, so each is
// named once (the table holds a reference).
inline ElemKind kindFromTorchDtype(const py::object &dtype) {
  static std::vector<std::pair<PyObject *, ElemKind>> known;
  for (const auto &k : known)
    if (k.first == dtype.ptr())
      return k.second;
  const ElemKind kind = kindFromTorchName(py::str(dtype).cast<std::string>());
  if (known.size() < 64) { // (an array type that makes dtype objects anew is not kept)
    Py_INCREF(dtype.ptr());
    known.emplace_back(dtype.ptr(), kind);
  }
  return kind;
}

// ---- DLPack's C exchange table -----------------------------------------------------
// The public DLPack 1.x binary interface, as far as it is used here.
struct DlVersion {
  uint32_t major, minor;
};
struct DlTensor {
  void *data;
  int32_t deviceType; // 1 host, 2 CUDA, 3 pinned host
  int32_t deviceId;
  int32_t ndim;
  uint8_t code, bits;
  uint16_t lanes;
  int64_t *shape;
  int64_t *strides; // elements; may be null: row-major
  uint64_t byteOffset;
};
struct DlExchange {
  DlVersion version;
  void *previous;
  void *allocate, *toManaged, *fromManaged;
  int (*view)(void *object, DlTensor *out); // borrows: valid while the object lives
  int (*currentStream)(int32_t deviceType, int32_t deviceId, void **stream);
};

inline ElemKind kindFromDl(uint8_t code, uint8_t bits) {
  switch (code) {
  case 0: return bits == 8 ? ElemKind::I8 : bits == 16 ? ElemKind::I16 : bits == 32 ? ElemKind::I32
                : bits == 64 ? ElemKind::I64 : ElemKind::Other;
  case 1: return bits == 8 ? ElemKind::U8 : ElemKind::Other;
  case 2: return bits == 16 ? ElemKind::F16 : bits == 32 ? ElemKind::F32
                : bits == 64 ? ElemKind::F64 : ElemKind::Other;
  case 4: return bits == 16 ? ElemKind::BF16 : ElemKind::Other;
  case 10: return bits == 8 ? ElemKind::E4M3 : ElemKind::Other;
  default: return ElemKind::Other;
  }
}

// The table of an object's type, or null.  Types are asked once (and kept alive).
inline const DlExchange *exchangeOf(py::handle obj) {
  static std::vector<std::pair<PyTypeObject *, const DlExchange *>> known;
  PyTypeObject *type = Py_TYPE(obj.ptr());
  for (const auto &k : known)
    if (k.first == type)
      return k.second;
  const DlExchange *found = nullptr;
  PyObject *capsule =
      PyObject_GetAttrString(reinterpret_cast<PyObject *>(type), "__dlpack_c_exchange_api__");
  if (capsule) {
    if (PyCapsule_IsValid(capsule, "dlpack_exchange_api"))
      found = static_cast<const DlExchange *>(PyCapsule_GetPointer(capsule, "dlpack_exchange_api"));
    if (found && (found->version.major != 1 || !found->view))
      found = nullptr;
    Py_DECREF(capsule); // the table itself is static
  }
  PyErr_Clear();
  if (known.size() < 64) {
    Py_INCREF(type);
    known.emplace_back(type, found);
  }
  return found;
}

// Fills `a` through the exchange table; false where that is not possible (the caller
// then reads the object's attributes).
inline bool arrayFromExchange(py::handle obj, ArrayArg &a) {
  const DlExchange *api = exchangeOf(obj);
  if (!api)
    return false;
  DlTensor t{};
  if (api->view(obj.ptr(), &t) != 0) {
    PyErr_Clear();
    return false;
  }
  if (t.ndim < 0 || t.lanes != 1 || t.bits % 8 || t.deviceType < 1 || t.deviceType > 3)
    return false;
  a.kind = kindFromDl(t.code, t.bits);
  if (a.kind == ElemKind::Other)
    return false;
  a.itemsize = t.bits / 8;
  a.data = static_cast<char *>(t.data) + t.byteOffset;
  a.shape.assign(t.shape, t.shape + t.ndim);
  if (t.strides) {
    a.strides.assign(t.strides, t.strides + t.ndim);
  } else {
    a.strides.assign(size_t(t.ndim), 1);
    for (int d = t.ndim - 2; d >= 0; --d)
      a.strides[d] = a.strides[d + 1] * a.shape[d + 1];
  }
  a.onDevice = t.deviceType == 2;
  a.deviceIndex = a.onDevice ? t.deviceId : -1;
  return true;
}

inline ArrayArg readArray(py::handle obj) {
  {
    ArrayArg a;
    if (arrayFromExchange(obj, a))
      return a;
  }
  if (py::hasattr(obj, "data_ptr") && py::hasattr(obj, "element_size")) {
    ArrayArg a;
    a.data = reinterpret_cast<void *>(obj.attr("data_ptr")().cast<uintptr_t>());
    const py::object shape = obj.attr("shape"), strides = obj.attr("stride")();
    if (PyTuple_Check(shape.ptr()) && PyTuple_Check(strides.ptr())) {
      // torch.Size and the strides are tuples of ints: read them without iterators.
      const Py_ssize_t rank = PyTuple_GET_SIZE(shape.ptr());
      a.shape.reserve(size_t(rank));
      a.strides.reserve(size_t(rank));
      for (Py_ssize_t d = 0; d < rank; ++d)
        a.shape.push_back(PyLong_AsLongLong(PyTuple_GET_ITEM(shape.ptr(), d)));
      for (Py_ssize_t d = 0; d < PyTuple_GET_SIZE(strides.ptr()); ++d)
        a.strides.push_back(PyLong_AsLongLong(PyTuple_GET_ITEM(strides.ptr(), d)));
      if (PyErr_Occurred())
        throw py::error_already_set();
    } else {
      for (auto d : shape)
        a.shape.push_back(d.cast<int64_t>());
      for (auto s : strides)
        a.strides.push_back(s.cast<int64_t>());
    }
    a.itemsize = obj.attr("element_size")().cast<int64_t>();
    a.kind = kindFromTorchDtype(obj.attr("dtype"));
    a.onDevice = obj.attr("is_cuda").cast<bool>();
    if (a.onDevice) {
      py::object idx = obj.attr("device").attr("index");
      a.deviceIndex = idx.is_none() ? 0 : idx.cast<int>();
    }
    return a;
  }
  if (py::hasattr(obj, "__cuda_array_interface__"))
    return arrayFromInterface(obj.attr("__cuda_array_interface__").cast<py::dict>(), true);
  if (py::hasattr(obj, "__array_interface__"))
    return arrayFromInterface(obj.attr("__array_interface__").cast<py::dict>(), false);
  throw std::runtime_error("Object is not an array (no data_ptr, __cuda_array_interface__ "
                           "or __array_interface__)");
}

inline ArrayArg arrayFromPython(py::handle obj) {
  ArrayArg a = readArray(obj);
  if (!a.data) {
    bool empty = false;
    for (int64_t n : a.shape)
      empty = empty || n == 0;
    if (!empty)
      throw std::runtime_error("Array without memory of its own (a meta or fake tensor, or a "
                               "wrapper of others)");
  }
  return a;
}

} // namespace hc
