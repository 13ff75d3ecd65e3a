// paged_binding.cpp -- the Python side of the paged-cache calls, in C++.
//
// A decode step's call is a few microseconds of GPU time, and checking nine tensors' shapes, types and
// strides from Python takes three times that (16 us a call against 6 here), so the checks of
// usagi_b200/paged.py are made here, against the CPython interface.  The C ABI itself is reached
// through the addresses that the package's one loaded library gives (init), so there is one library
// and one set of kernels.
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Device.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <cmath>
#include <map>
#include <string>
#include <utility>

#include "../../include/bsattn.h"

namespace {

constexpr int64_t kHeadDim = 128;
constexpr int64_t kKeptAtLeast = 4 << 20, kKept = 32 << 20;  // bytes of scratch that a stream keeps
constexpr size_t kStreams = 16;                              // streams that keep any, the last ones used

decltype(&bsattn_paged_append) g_append = nullptr;
decltype(&bsattn_paged_fwd) g_fwd = nullptr;
decltype(&bsattn_paged_scratch_bytes) g_scratch_bytes = nullptr;
decltype(&bsattn_paged_counters) g_counters = nullptr;
PyObject* g_workspaces = nullptr;  // the package's error words by (device, stream)
PyObject* g_workspace = nullptr;   // makes one
PyObject* g_error = nullptr;       // BsattnError

// Ends a call with a Python exception that is set already.
struct Raised {};

[[noreturn]] void refuse(PyObject* type, const std::string& text) {
  PyErr_SetString(type, text.c_str());
  throw Raised();
}

std::string shape_text(at::IntArrayRef s) {
  std::string t = "(";
  for (size_t i = 0; i < s.size(); ++i) t += (i ? ", " : "") + std::to_string(s[i]);
  return t + ")";
}

bool is_none(PyObject* o) { return o == nullptr || o == Py_None; }

const at::Tensor& tensor(PyObject* o, const char* name) {
  if (!THPVariable_Check(o)) refuse(PyExc_TypeError, std::string(name) + " must be a tensor");
  return THPVariable_Unpack(o);
}

int64_t integer(PyObject* o, const char* name) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw Raised();
  if (v != static_cast<int>(v)) refuse(PyExc_ValueError, std::string(name) + " is out of range");
  return v;
}

// Stride of a dimension; one of a single entry is never used, whatever torch holds for it.
int64_t stride_of(at::IntArrayRef n, at::IntArrayRef s, int i) { return n[i] > 1 ? s[i] : kHeadDim; }
// Whether rows of 128 contiguous values begin at multiples of 8.
bool rows_of_eight(const at::Tensor& t) {
  const at::IntArrayRef n = t.sizes(), s = t.strides();
  return s[3] == 1 && ((stride_of(n, s, 0) | stride_of(n, s, 1) | stride_of(n, s, 2)) & 7) == 0;
}
bool misaligned(const at::Tensor& t) { return (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15u) != 0; }

void check_call(int rc, const char* where) {
  if (rc == BSATTN_OK) return;
  PyObject* e = PyObject_CallFunction(g_error, "is", rc, where);
  if (e != nullptr) {
    PyErr_SetObject(g_error, e);
    Py_DECREF(e);
  }
  throw Raised();
}

// `t` as int32 on the device with a contiguous last dimension.
at::Tensor index_tensor(const at::Tensor& t, const char* name, c10::Device dev, at::IntArrayRef shape) {
  if (t.sizes() != shape)
    refuse(PyExc_ValueError, std::string(name) + ": expected shape " + shape_text(shape) + ", got " +
                                 shape_text(t.sizes()));
  at::Tensor x = t;
  if (!at::isIntegralType(x.scalar_type(), false))
    refuse(PyExc_TypeError, std::string(name) + " must hold integers");
  // What 32 bits do not hold stays out of range, where the kernels find it.
  if (x.scalar_type() == at::kUInt64) x = x.to(at::kLong);  // what passes 2^63 becomes negative
  if (x.scalar_type() == at::kLong) x = x.clamp(INT32_MIN, INT32_MAX);
  if (x.scalar_type() != at::kInt || x.device() != dev) x = x.to(dev, at::kInt);
  if (x.stride(-1) != 1 && x.size(-1) > 1) x = x.contiguous();
  return x;
}

// A [B, H, T, 128] input as the kernels read it in place: 16-byte rows and strides.
at::Tensor rows_tensor(const at::Tensor& t, const char* name, c10::Device dev, at::ScalarType dtype,
                       at::IntArrayRef shape) {
  if (t.sizes() != shape)
    refuse(PyExc_ValueError,
           std::string(name) + " must be " + shape_text(shape) + ", got " + shape_text(t.sizes()));
  if (t.scalar_type() != dtype || t.device() != dev)
    refuse(PyExc_TypeError, std::string(name) + " must have the dtype and device of the pages");
  if (rows_of_eight(t) && !misaligned(t)) return t;
  at::Tensor x = t.contiguous();
  return misaligned(x) ? x.clone() : x;
}

void check_out(const at::Tensor& t, const char* name, c10::Device dev, at::ScalarType dtype,
               at::IntArrayRef shape, bool aligned) {
  if (t.sizes() != shape || t.scalar_type() != dtype || t.device() != dev || !t.is_contiguous() ||
      (aligned && misaligned(t)))
    refuse(PyExc_ValueError,
           std::string(name) + " has the wrong shape, dtype, device, layout or alignment");
}

// The cache arguments of a call, checked, and the record for the C ABI.
struct Call {
  bsattn_paged_call c{};
  c10::Device dev = c10::Device(at::kCPU);
  at::ScalarType dtype = at::kHalf;
  at::Tensor table, seq_lens, q_lens;  // kept until the launch

  Call(PyObject* k_, PyObject* v_, PyObject* table_, PyObject* lens_, PyObject* q_lens_, int64_t B) {
    const at::Tensor &k = tensor(k_, "k_pages"), &v = tensor(v_, "v_pages");
    if (k.dim() != 4 || k.size(3) != kHeadDim || v.sizes() != k.sizes())
      refuse(PyExc_ValueError, "k_pages and v_pages must be [n_pages, Hkv, page_size, 128] of one shape, got " +
                                   shape_text(k.sizes()) + ", " + shape_text(v.sizes()));
    dev = k.device();
    dtype = k.scalar_type();
    if ((dtype != at::kHalf && dtype != at::kBFloat16) || v.scalar_type() != dtype)
      refuse(PyExc_TypeError, "k_pages and v_pages must both be float16 or both bfloat16");
    if (!k.is_cuda() || v.device() != dev)
      refuse(PyExc_ValueError, "the paged cache needs CUDA tensors on one device (there is no CPU path)");
    const int64_t pages = k.size(0), heads = k.size(1), page = k.size(2);
    if (pages == 0 || heads == 0)
      refuse(PyExc_ValueError, "the cache has no pages or no heads: " + shape_text(k.sizes()));
    if (page < 16 || page > 1024 || (page & (page - 1)) != 0)
      refuse(PyExc_ValueError, "page_size must be a power of two from 16 to 1024, got " + std::to_string(page));
    if (!rows_of_eight(k) || !rows_of_eight(v) || misaligned(k) || misaligned(v))
      refuse(PyExc_ValueError, "k_pages and v_pages must be 16-byte aligned, with a contiguous last "
                               "dimension and strides that are multiples of 8");
    const at::Tensor& t = tensor(table_, "block_table");
    if (t.dim() != 2 || t.size(1) == 0)
      refuse(PyExc_ValueError, "block_table must be [B, max_pages], got " + shape_text(t.sizes()));
    if (pages > INT32_MAX || heads > INT32_MAX || t.size(1) > INT32_MAX || B > INT32_MAX)
      refuse(PyExc_ValueError, "the cache or the batch is too large");
    table = index_tensor(t, "block_table", dev, {B, t.size(1)});
    seq_lens = index_tensor(tensor(lens_, "seq_lens"), "seq_lens", dev, {B});
    if (!is_none(q_lens_)) q_lens = index_tensor(tensor(q_lens_, "q_lens"), "q_lens", dev, {B});
    c.k_pages = k.data_ptr();
    c.v_pages = v.data_ptr();
    const at::IntArrayRef n = k.sizes(), ks = k.strides(), vs = v.strides();
    for (int i = 0; i < 3; ++i) {
      c.page_strides[i] = stride_of(n, ks, i);
      c.page_strides[3 + i] = stride_of(n, vs, i);
    }
    c.block_table = static_cast<const int32_t*>(table.data_ptr());
    c.table_stride = table.stride(0);
    c.seq_lens = static_cast<const int32_t*>(seq_lens.data_ptr());
    c.q_lens = q_lens.defined() ? static_cast<const int32_t*>(q_lens.data_ptr()) : nullptr;
    c.max_pages = static_cast<int32_t>(table.size(1));
    c.n_pages = static_cast<int32_t>(pages);
    c.page_size = static_cast<int32_t>(page);
    c.B = static_cast<int32_t>(B);
    c.Hkv = static_cast<int32_t>(heads);
  }

  // Stream and error word of the current device (the pages').
  cudaStream_t on_stream() {
    const cudaStream_t s = c10::cuda::getCurrentCUDAStream(dev.index()).stream();
    PyObject* key = Py_BuildValue("iK", static_cast<int>(dev.index()),
                                  static_cast<unsigned long long>(reinterpret_cast<uintptr_t>(s)));
    if (key == nullptr) throw Raised();
    PyObject* ws = PyDict_GetItemWithError(g_workspaces, key);  // borrowed
    Py_XINCREF(ws);
    if (ws == nullptr && !PyErr_Occurred()) {
      PyObject* d = THPDevice_New(dev);
      if (d != nullptr)
        ws = PyObject_CallFunctionObjArgs(g_workspace, d, PyTuple_GET_ITEM(key, 1), nullptr);
      Py_XDECREF(d);
    }
    Py_DECREF(key);
    if (ws == nullptr) throw Raised();
    const at::Tensor& t = THPVariable_Unpack(ws);
    c.workspace = t.data_ptr();
    c.workspace_bytes = static_cast<size_t>(t.numel()) * 4;
    c.stream = s;
    Py_DECREF(ws);  // the dictionary keeps it
    return s;
  }
};

int32_t as_int32(int64_t v, const char* what) {
  if (v > INT32_MAX) refuse(PyExc_ValueError, std::string(what) + " is too large");
  return static_cast<int32_t>(v);
}

// Scratch and counters of a call.  The calls of one CUDA stream follow one another, so a stream keeps
// its own (what another stream takes the place of goes back to the allocator, which hands it to that same
// stream again); a captured call gets new ones, which belong to the graph (the counters zeroed by it),
// since graphs captured on one stream may be replayed at the same time.
struct Room {
  at::Tensor scratch, counters;
};
Room room(c10::Device dev, cudaStream_t stream, int64_t need) {
  struct Kept {
    Room room;
    uint64_t call = 0;  // the last one that used it
  };
  static std::map<std::pair<int, cudaStream_t>, Kept> rooms;  // under the interpreter's lock
  static uint64_t calls = 0;
  const auto bytes = at::TensorOptions().device(dev).dtype(at::kByte);
  const auto ints = at::TensorOptions().device(dev).dtype(at::kInt);
  if (c10::cuda::currentStreamCaptureStatusMayInitCtx() != c10::cuda::CaptureStatus::None)
    return {at::empty({need}, bytes), at::zeros({g_counters()}, ints)};
  const std::pair<int, cudaStream_t> key{dev.index(), stream};
  auto at = rooms.find(key);
  if (at == rooms.end()) {
    if (rooms.size() >= kStreams)
      rooms.erase(std::min_element(rooms.begin(), rooms.end(), [](const auto& a, const auto& b) {
        return a.second.call < b.second.call;
      }));
    at = rooms.emplace(key, Kept{}).first;
  }
  at->second.call = ++calls;
  Room& r = at->second.room;
  if (!r.counters.defined()) r.counters = at::zeros({g_counters()}, ints);
  if (need > kKept) return {at::empty({need}, bytes), r.counters};
  if (!r.scratch.defined() || r.scratch.numel() < need)
    r.scratch = at::empty({std::max<int64_t>(need, kKeptAtLeast)}, bytes);
  return r;
}

PyObject* finish(const at::Tensor& t) { return THPVariable_Wrap(t); }

// append(k_pages, v_pages, block_table, seq_lens, k, v, q, q_lens, inv_freq, interleaved, q_out)
PyObject* append_impl(PyObject* const* a) {
  const at::AutoDispatchBelowADInplaceOrView no_grad;
  const at::Tensor& k0 = tensor(a[4], "k");
  if (k0.dim() != 4) refuse(PyExc_ValueError, "k must be [B, Hkv, Tq, 128], got " + shape_text(k0.sizes()));
  const int64_t B = k0.size(0), Tq = k0.size(2);
  Call call(a[0], a[1], a[2], a[3], a[7], B);
  const int64_t Hkv = call.c.Hkv;
  const at::Tensor k = rows_tensor(k0, "k", call.dev, call.dtype, {B, Hkv, Tq, kHeadDim});
  const at::Tensor v = rows_tensor(tensor(a[5], "v"), "v", call.dev, call.dtype, {B, Hkv, Tq, kHeadDim});
  at::Tensor q, q_out;
  int64_t Hq = 0;
  if (!is_none(a[6])) {
    const at::Tensor& x = tensor(a[6], "q");
    Hq = x.dim() == 4 ? x.size(1) : 0;
    if (Hq == 0)
      refuse(PyExc_ValueError, "q must be [B, Hq, Tq, 128] with heads, got " + shape_text(x.sizes()));
    q = rows_tensor(x, "q", call.dev, call.dtype, {B, Hq, Tq, kHeadDim});
    if (is_none(a[10])) {
      q_out = at::empty({B, Hq, Tq, kHeadDim}, q.options());
    } else {
      q_out = tensor(a[10], "q_out");
      check_out(q_out, "q_out", call.dev, call.dtype, {B, Hq, Tq, kHeadDim}, true);
    }
  } else if (!is_none(a[10])) {
    refuse(PyExc_ValueError, "q_out needs q");
  }
  at::Tensor inv;
  if (!is_none(a[8])) {
    const at::Tensor& f = tensor(a[8], "inv_freq");
    if (f.dim() != 1 || f.scalar_type() != at::kDouble || f.device() != call.dev)
      refuse(PyExc_TypeError, "inv_freq must be float64 [rot_dim / 2] on the device of the pages");
    if (f.size(0) % 8 != 0 || f.size(0) < 8 || f.size(0) > kHeadDim / 2)
      refuse(PyExc_ValueError,
             "rot_dim must be a multiple of 16 up to 128, got " + std::to_string(2 * f.size(0)));
    inv = f.contiguous();
  }
  const int interleaved = PyObject_IsTrue(a[9]);
  if (interleaved < 0) throw Raised();
  if (B > 0 && Tq > 0) {
    const c10::cuda::CUDAGuard guard(call.dev);
    call.on_stream();
    call.c.Hq = as_int32(Hq, "Hq");
    call.c.Tq = as_int32(Tq, "Tq");
    call.c.dtype_flags = call.dtype == at::kBFloat16 ? BSATTN_IN_BF16 : 0;
    int64_t st[9] = {0};
    const at::IntArrayRef n = k.sizes(), ks = k.strides(), vs = v.strides();
    for (int i = 0; i < 3; ++i) {
      if (Hq > 0) st[i] = stride_of(q.sizes(), q.strides(), i);
      st[3 + i] = stride_of(n, ks, i);
      st[6 + i] = stride_of(n, vs, i);
    }
    check_call(g_append(&call.c, Hq > 0 ? q.data_ptr() : nullptr, k.data_ptr(), v.data_ptr(), st,
                        Hq > 0 ? q_out.data_ptr() : nullptr,
                        inv.defined() ? static_cast<const double*>(inv.data_ptr()) : nullptr,
                        inv.defined() ? static_cast<int>(2 * inv.size(0)) : 0, interleaved),
               "bsattn_paged_append");
  }
  if (Hq == 0) Py_RETURN_NONE;
  if (!is_none(a[10])) return Py_NewRef(a[10]);
  return finish(q_out);
}

// attn(q, k_pages, v_pages, block_table, seq_lens, q_lens, window, global_blocks, prefix_len, scale,
//      out_dtype, out, lse_out, return_lse)
PyObject* attn_impl(PyObject* const* a) {
  const at::AutoDispatchBelowADInplaceOrView no_grad;
  const at::Tensor& q0 = tensor(a[0], "q");
  if (q0.dim() != 4 || q0.size(3) != kHeadDim)
    refuse(PyExc_ValueError, "q must be [B, Hq, Tq, 128], got " + shape_text(q0.sizes()));
  const int64_t B = q0.size(0), Hq = q0.size(1), Tq = q0.size(2);
  Call call(a[1], a[2], a[3], a[4], a[5], B);
  if (q0.scalar_type() != call.dtype || q0.device() != call.dev)
    refuse(PyExc_TypeError, "q must have the dtype and device of the pages");
  if (Hq == 0 || Hq % call.c.Hkv != 0)
    refuse(PyExc_ValueError, "Hq must be a multiple of Hkv, got " + std::to_string(Hq) + " and " +
                                 std::to_string(call.c.Hkv));
  const int64_t window = integer(a[6], "window"), blocks = integer(a[7], "global_blocks");
  const int64_t prefix = integer(a[8], "prefix_len");
  if (prefix < 0 || prefix % call.c.page_size != 0)
    refuse(PyExc_ValueError, "prefix_len must be whole pages (multiples of " +
                                 std::to_string(call.c.page_size) + "), got " + std::to_string(prefix));
  if (prefix > static_cast<int64_t>(call.c.max_pages) * call.c.page_size)
    refuse(PyExc_ValueError, "prefix_len is more than block_table holds");
  double scale = 0.0;
  if (!is_none(a[9])) {
    scale = PyFloat_AsDouble(a[9]);
    if (scale == -1.0 && PyErr_Occurred()) throw Raised();
    // The C ABI takes 0 for the default.
    if (!(static_cast<float>(scale) > 0.0f) || std::isinf(static_cast<float>(scale)))
      refuse(PyExc_ValueError, "scale must be positive and finite");
  }
  at::ScalarType out_dtype = call.dtype;
  if (!is_none(a[10])) {
    if (THPDtype_Check(a[10])) out_dtype = reinterpret_cast<THPDtype*>(a[10])->scalar_type;
    if (!THPDtype_Check(a[10]) || (out_dtype != at::kHalf && out_dtype != at::kBFloat16))
      refuse(PyExc_TypeError, "out_dtype must be float16 or bfloat16");
  }
  at::Tensor q = q0.contiguous();
  if (misaligned(q)) q = q.clone();
  at::Tensor out, lse;
  if (is_none(a[11])) {
    out = at::empty({B, Hq, Tq, kHeadDim}, q.options().dtype(out_dtype));
  } else {
    out = tensor(a[11], "out");
    check_out(out, "out", call.dev, out_dtype, {B, Hq, Tq, kHeadDim}, true);
  }
  const int want_lse = PyObject_IsTrue(a[13]);
  if (want_lse < 0) throw Raised();
  if (want_lse) {
    if (is_none(a[12])) {
      lse = at::empty({B, Hq, Tq}, q.options().dtype(at::kFloat));
    } else {
      lse = tensor(a[12], "lse_out");
      check_out(lse, "lse_out", call.dev, at::kFloat, {B, Hq, Tq}, false);
    }
  }
  if (B > 0 && Tq > 0) {
    const c10::cuda::CUDAGuard guard(call.dev);
    const cudaStream_t stream = call.on_stream();
    call.c.Hq = as_int32(Hq, "Hq");
    call.c.Tq = as_int32(Tq, "Tq");
    call.c.dtype_flags = (call.dtype == at::kBFloat16 ? BSATTN_IN_BF16 : 0) |
                         (out_dtype == at::kBFloat16 ? BSATTN_OUT_BF16 : 0);
    size_t need = 0;
    check_call(g_scratch_bytes(call.c.B, call.c.Hq, call.c.Hkv, call.c.Tq, call.c.max_pages, call.c.page_size,
                               static_cast<int>(prefix), &need),
               "bsattn_paged_scratch_bytes");
    const Room r = room(call.dev, stream, static_cast<int64_t>(need));
    check_call(g_fwd(&call.c, q.data_ptr(), out.data_ptr(),
                     lse.defined() ? static_cast<float*>(lse.data_ptr()) : nullptr, static_cast<int>(window),
                     static_cast<int>(blocks), static_cast<int>(prefix), static_cast<float>(scale),
                     r.scratch.data_ptr(), need, static_cast<int32_t*>(r.counters.data_ptr())),
               "bsattn_paged_fwd");
  }
  PyObject* o = is_none(a[11]) ? finish(out) : Py_NewRef(a[11]);
  PyObject* l = !want_lse ? Py_NewRef(Py_None) : is_none(a[12]) ? finish(lse) : Py_NewRef(a[12]);
  PyObject* both = o != nullptr && l != nullptr ? PyTuple_Pack(2, o, l) : nullptr;
  Py_XDECREF(o);
  Py_XDECREF(l);
  return both;
}

template <PyObject* (*F)(PyObject* const*), Py_ssize_t N>
PyObject* entry(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != N) {
    PyErr_SetString(PyExc_TypeError, "wrong number of arguments");
    return nullptr;
  }
  if (g_error == nullptr) {
    PyErr_SetString(PyExc_RuntimeError, "not initialised");
    return nullptr;
  }
  try {
    return F(args);
  } catch (const Raised&) {
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}

// init(append, fwd, scratch_bytes, counters, workspaces, workspace, error): addresses and objects
PyObject* init(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 7 || !PyDict_Check(args[4])) {
    PyErr_SetString(PyExc_TypeError, "init takes four addresses, a dict, a function and a class");
    return nullptr;
  }
  void* at[4];
  for (int i = 0; i < 4; ++i) {
    at[i] = PyLong_AsVoidPtr(args[i]);
    if (at[i] == nullptr) {
      if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "a null address");
      return nullptr;
    }
  }
  g_append = reinterpret_cast<decltype(g_append)>(at[0]);
  g_fwd = reinterpret_cast<decltype(g_fwd)>(at[1]);
  g_scratch_bytes = reinterpret_cast<decltype(g_scratch_bytes)>(at[2]);
  g_counters = reinterpret_cast<decltype(g_counters)>(at[3]);
  Py_XSETREF(g_workspaces, Py_NewRef(args[4]));
  Py_XSETREF(g_workspace, Py_NewRef(args[5]));
  Py_XSETREF(g_error, Py_NewRef(args[6]));
  Py_RETURN_NONE;
}

PyMethodDef kMethods[] = {
    {"init", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(init)), METH_FASTCALL, nullptr},
    {"append", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(&entry<append_impl, 11>)), METH_FASTCALL,
     nullptr},
    {"attn", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(&entry<attn_impl, 14>)), METH_FASTCALL,
     nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_paged_binding", nullptr, -1, kMethods, nullptr, nullptr, nullptr,
                       nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__paged_binding() { return PyModule_Create(&kModule); }
