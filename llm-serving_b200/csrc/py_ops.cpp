// py_ops.cpp -- Python binding of the head norm with rotation, the 4-bit pages, the page copies and the
// cache of bounded length.
//
// These calls sit on the path of every decode step, where a launch's host time is the operator's
// time: through ctypes and Python-level checks a call took 17 to 37 us for 2 to 4 us of kernel.
// Here the checks, the output allocation and the C ABI call are one C++ function per operator.
// The C ABI stays the boundary: bind() receives the entry points' addresses from the library that
// model/_native.py loaded, so there is one copy of it in the process and nothing links to it.
//
// Every function takes its arguments by position (the Python modules give them names), raises
// ValueError for a broken contract, RuntimeError for tensors that are not on CUDA, and reports the
// library's status codes through _native.check. No function waits for the device.
#include <ATen/cuda/EmptyTensor.h>
#include <ATen/ops/zeros.h>
#include <Python.h>
#include <c10/cuda/CUDAException.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/python_numbers.h>

#include <algorithm>
#include <cmath>
#include <iterator>
#include <map>
#include <vector>

#include "paged_decode.h"

namespace {

using at::Tensor;

#define PD_ENTRIES(X) \
  X(pd_qk_norm_rope) X(pd_fp4_write_slots) X(pd_fp4_write_table) X(pd_fp4_read_slots) X(pd_fp4_workspace_bytes) \
  X(pd_fp4_decode) X(pd_fp4_prefill) X(pd_block_copy) X(pd_decode_window_workspace_bytes) X(pd_decode_window_small) X(pd_decode_window) \
  X(pd_prefill_window) \
  X(pd_decode_weights_scratch_bytes) X(pd_decode_weights) X(pd_evict_scratch_bytes) X(pd_evict)
#define PD_FIELD(name) decltype(&::name) name = nullptr;
struct Entries {
  PD_ENTRIES(PD_FIELD)
};
Entries lib;
PyObject* check_status = nullptr;  // _native.check(status, what)

#define VALUE(cond, ...) TORCH_CHECK_VALUE(cond, __VA_ARGS__)

// ------------------------------------------------------------------ arguments

void arity(Py_ssize_t got, Py_ssize_t want, const char* what) {
  TORCH_CHECK_TYPE(got == want, what, " takes ", want, " arguments, got ", got);
}

const Tensor& tensor(PyObject* o, const char* name) {
  TORCH_CHECK_TYPE(THPVariable_Check(o), name, " must be a tensor, got ", Py_TYPE(o)->tp_name);
  return THPVariable_Unpack(o);
}

const Tensor* optional(PyObject* o, const char* name) { return o == Py_None ? nullptr : &tensor(o, name); }

void cuda(const Tensor& t, const char* name, const char* what) {
  TORCH_CHECK(t.is_cuda(), what, " requires CUDA tensors, got ", name, " on device ", t.device(),
              "; there is no silent fallback to a dense implementation.");
}

void same_device(const Tensor& t, const char* name, const Tensor& as, const char* as_name) {
  VALUE(t.device() == as.device(), name, " is on ", t.device(), " but ", as_name, " is on ", as.device());
}

int dtype_code(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return PD_F32;
    case at::kHalf: return PD_F16;
    case at::kBFloat16: return PD_BF16;
    default: return -1;
  }
}

bool index_type(const Tensor& t) { return t.scalar_type() == at::kInt || t.scalar_type() == at::kLong; }
int slot_code(const Tensor& t) { return t.scalar_type() == at::kInt ? PD_SLOT_I32 : PD_SLOT_I64; }

Tensor unit_stride(const Tensor& t) { return t.dim() && t.size(-1) != 1 && t.stride(-1) != 1 ? t.contiguous() : t; }
Tensor int32(const Tensor& t) { return (t.scalar_type() == at::kInt ? t : t.to(at::kInt)).contiguous(); }
bool aligned16(const Tensor& t) { return (reinterpret_cast<uintptr_t>(t.const_data_ptr()) & 15u) == 0; }

Tensor new_like(const Tensor& t) {
  return at::detail::empty_cuda(t.sizes(), t.scalar_type(), t.device(), std::nullopt);
}

void* stream_of(const Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.get_device()).stream(); }

// The library's status as a Python exception; true when it raised.
bool failed(int status, const char* what) {
  if (status == PD_OK) return false;
  PyObject* r = PyObject_CallFunction(check_status, "is", status, what);
  Py_XDECREF(r);
  if (!PyErr_Occurred()) PyErr_Format(PyExc_RuntimeError, "%s failed: status %d", what, status);
  return true;
}

PyObject* pair(const Tensor& a, const Tensor& b) {
  PyObject* r = PyTuple_New(2);
  if (r == nullptr) return nullptr;
  PyTuple_SET_ITEM(r, 0, THPVariable_Wrap(a));
  PyTuple_SET_ITEM(r, 1, THPVariable_Wrap(b));
  return r;
}

// ------------------------------------------------------------------ 4-bit pages

struct Pages {
  void* data;
  int64_t n_blocks, hkv;
  int block_size, d;
  const float* units;
};

Pages pages_of(const Tensor& pages, const Tensor* units, const char* what) {
  cuda(pages, "pages", what);
  VALUE(pages.dim() == 4 && pages.scalar_type() == at::kByte,
        "pages must be uint8 (n_blocks, H_kv, block_size / 16, 18 * head_dim), got ", pages.sizes(), " ",
        pages.scalar_type());
  const int64_t rec = pages.size(3), tpb = pages.size(2);
  VALUE((rec == 18 * 64 || rec == 18 * 128 || rec == 18 * 256) && tpb >= 1 && (tpb & (tpb - 1)) == 0 &&
            pages.size(1) >= 1 && pages.size(0) >= 1,
        "pages of shape ", pages.sizes(), " are not 4-bit pages of head_dim 64, 128 or 256");
  VALUE(tpb * pages.size(1) <= 0x7fffffff / rec, "a block of 4-bit pages must be below 2 GiB, got shape ", pages.sizes());
  VALUE(pages.is_contiguous() && aligned16(pages), "pages must be contiguous and 16-byte aligned");
  Pages p;
  p.data = pages.data_ptr();
  p.n_blocks = pages.size(0);
  p.hkv = pages.size(1);
  p.block_size = int(tpb * 16);
  p.d = int(rec / 18);
  p.units = nullptr;
  if (units != nullptr) {
    VALUE(units->scalar_type() == at::kFloat && units->dim() == 2 && units->size(0) == 2 && units->size(1) == p.hkv,
          "units must be float32 (2, ", p.hkv, "), got ", units->sizes(), " ", units->scalar_type());
    same_device(*units, "units", pages, "pages");
    VALUE(units->is_contiguous(), "units must be contiguous");
    p.units = units->const_data_ptr<float>();
  }
  return p;
}

void rows_of(const Pages& p, const Tensor& pages, const Tensor& k, const Tensor& v) {
  VALUE(k.dim() == 3 && k.size(1) == p.hkv && k.size(2) == p.d, "k/v must be (n, ", p.hkv, ", ", p.d,
        ") for these pages, got ", k.sizes(), " / ", v.sizes());
  VALUE(k.sizes() == v.sizes(), "k/v shapes differ: ", k.sizes(), " vs ", v.sizes());
  VALUE(dtype_code(k.scalar_type()) >= 0 && v.scalar_type() == k.scalar_type(),
        "k/v must share one dtype of fp32, fp16 or bf16, got ", k.scalar_type(), " / ", v.scalar_type());
  same_device(k, "k", pages, "pages");
  same_device(v, "v", pages, "pages");
}

void slots_of(const Tensor& slots, const Tensor& pages, int64_t n) {
  VALUE(slots.dim() == 1 && slots.numel() == n, "slot_ids must be 1-D with one entry per token (", n, "), got ",
        slots.sizes());
  VALUE(index_type(slots), "slot_ids must be an integer tensor, got ", slots.scalar_type());
  same_device(slots, "slot_ids", pages, "pages");
}

PyObject* write_slots(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  arity(n, 5, "fp4_write_slots");
  const Tensor& pages = tensor(a[0], "pages");
  const Pages p = pages_of(pages, optional(a[4], "units"), "write_slots_fp4");
  Tensor k = tensor(a[2], "k"), v = tensor(a[3], "v");
  rows_of(p, pages, k, v);
  slots_of(tensor(a[1], "slot_ids"), pages, k.size(0));
  if (k.size(0) == 0) Py_RETURN_NONE;
  const c10::cuda::CUDAGuard guard(pages.device());
  const Tensor slots = tensor(a[1], "slot_ids").contiguous();
  k = unit_stride(k);
  v = unit_stride(v);
  const int64_t ks[2] = {k.stride(0), k.stride(1)}, vs[2] = {v.stride(0), v.stride(1)};
  if (failed(lib.pd_fp4_write_slots(p.data, p.n_blocks, p.block_size, slots.const_data_ptr(), slot_code(slots),
                                    k.const_data_ptr(), ks, v.const_data_ptr(), vs, p.units,
                                    dtype_code(k.scalar_type()), k.size(0), int(p.hkv), p.d, stream_of(pages)),
             "pd_fp4_write_slots"))
    return nullptr;
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

PyObject* write_table(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  arity(n, 6, "fp4_write_table");
  const Tensor& pages = tensor(a[0], "pages");
  const Pages p = pages_of(pages, optional(a[5], "units"), "write_table_fp4");
  const Tensor &table = tensor(a[1], "block_table"), &pos = tensor(a[2], "pos");
  Tensor k = tensor(a[3], "k"), v = tensor(a[4], "v");
  rows_of(p, pages, k, v);
  VALUE(table.dim() == 2 && table.scalar_type() == at::kInt && table.size(0) == k.size(0) &&
            (table.size(1) == 1 || table.stride(1) == 1) && (k.size(0) == 1 || table.stride(0) >= table.size(1)),
        "block_table must be an int32 (", k.size(0), ", max_blocks) tensor with unit columns, got ", table.sizes());
  VALUE(pos.dim() == 1 && pos.scalar_type() == at::kLong && pos.size(0) == k.size(0) && pos.is_contiguous(),
        "pos must be a contiguous int64 (", k.size(0), ",) tensor, got ", pos.sizes());
  same_device(table, "block_table", pages, "pages");
  same_device(pos, "pos", pages, "pages");
  const c10::cuda::CUDAGuard guard(pages.device());
  k = unit_stride(k);
  v = unit_stride(v);
  const int64_t ks[2] = {k.stride(0), k.stride(1)}, vs[2] = {v.stride(0), v.stride(1)};
  if (failed(lib.pd_fp4_write_table(p.data, p.n_blocks, p.block_size, table.const_data_ptr<int32_t>(), table.stride(0),
                                    int(table.size(1)), pos.const_data_ptr<int64_t>(), k.const_data_ptr(), ks,
                                    v.const_data_ptr(), vs, p.units, dtype_code(k.scalar_type()), int(k.size(0)),
                                    int(p.hkv), p.d, stream_of(pages)),
             "pd_fp4_write_table"))
    return nullptr;
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

PyObject* read_slots(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  arity(n, 4, "fp4_read_slots");
  const Tensor& pages = tensor(a[0], "pages");
  const Pages p = pages_of(pages, optional(a[3], "units"), "read_slots_fp4");
  TORCH_CHECK_TYPE(THPDtype_Check(a[2]), "dtype must be a torch.dtype, got ", Py_TYPE(a[2])->tp_name);
  const at::ScalarType dtype = reinterpret_cast<THPDtype*>(a[2])->scalar_type;
  VALUE(dtype_code(dtype) >= 0, "dtype must be fp32, fp16 or bf16, got ", dtype);
  Tensor slots = tensor(a[1], "slot_ids");
  slots_of(slots, pages, slots.numel());
  const c10::cuda::CUDAGuard guard(pages.device());
  slots = slots.contiguous();
  const int64_t count = slots.numel();
  const Tensor k = at::detail::empty_cuda({count, p.hkv, p.d}, dtype, pages.device(), std::nullopt);
  const Tensor v = at::detail::empty_cuda({count, p.hkv, p.d}, dtype, pages.device(), std::nullopt);
  const int64_t s[2] = {p.hkv * p.d, p.d};
  if (count > 0 &&
      failed(lib.pd_fp4_read_slots(p.data, p.n_blocks, p.block_size, slots.const_data_ptr(), slot_code(slots),
                                   k.data_ptr(), s, v.data_ptr(), s, p.units, dtype_code(dtype), count, int(p.hkv),
                                   p.d, stream_of(pages)),
             "pd_fp4_read_slots"))
    return nullptr;
  return pair(k, v);
  END_HANDLE_TH_ERRORS
}

// ------------------------------------------------------------------ attention over 4-bit pages

Tensor new_workspace(const at::Device& device) {
  const c10::cuda::CUDAGuard guard(device);
  return at::zeros({int64_t(lib.pd_fp4_workspace_bytes(256))}, at::TensorOptions(at::kByte).device(device));
}

// The workspace of a call that was given none, of at least what `fresh` makes for it. Eager
// calls share one per (device, stream). A captured call never takes that one, also where its stream has
// it already: the graph may be replayed on another stream beside the eager calls, or beside another graph. A
// capture has its own, per stream (a zero fill is a node of the graph); it is dropped here with the first
// call after the capture's end, its memory staying in the graph's pool.
using Workspaces = std::map<std::pair<int, void*>, Tensor>;
struct StreamWorkspaces {
  Workspaces eager;
  std::map<unsigned long long, Workspaces> captures;  // by capture
};
template <typename Fresh>
Tensor stream_workspace(StreamWorkspaces& all, const at::Device& device, void* stream, int64_t bytes, const Fresh& fresh) {
  Workspaces *eager = &all.eager;
  auto* captures = &all.captures;
  cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
  unsigned long long capture = 0;
  C10_CUDA_CHECK(cudaStreamGetCaptureInfo(static_cast<cudaStream_t>(stream), &status, &capture));
  const bool captured = status != cudaStreamCaptureStatusNone;
  for (auto it = captures->begin(); it != captures->end();)
    it = captured && it->first == capture ? std::next(it) : captures->erase(it);
  Tensor& ws = (captured ? (*captures)[capture] : *eager)[std::make_pair(int(device.index()), stream)];
  if (!ws.defined() || ws.numel() < bytes) ws = fresh();
  return ws;
}

// The 4-bit attention's: zero-filled once and left at zero by every launch.
Tensor fp4_workspace(const at::Device& device, void* stream) {
  static auto* all = new StreamWorkspaces;  // never destroyed: outlives no context
  return stream_workspace(*all, device, stream, 1, [&] { return new_workspace(device); });
}

// The decode kernel's variants': any contents.
Tensor decode_workspace(const at::Device& device, void* stream, int64_t bytes) {
  static auto* all = new StreamWorkspaces;
  return stream_workspace(*all, device, stream, bytes,
                          [&] { return at::detail::empty_cuda({bytes}, at::kByte, device, std::nullopt); });
}

// Rows the kernels read: unit last stride, 16-byte aligned rows; a copy where they are not so already.
Tensor kernel_rows(const Tensor& q) {
  if (q.stride(2) == 1 && q.stride(0) % 8 == 0 && q.stride(1) % 8 == 0 && aligned16(q)) return q;
  const Tensor c = q.contiguous();
  return aligned16(c) && c.data_ptr() != q.data_ptr() ? c : c.clone();
}

PyObject* attend(PyObject* const* a, bool chunk) {
  const char* what = chunk ? "paged_prefill_fp4" : "paged_decode_fp4";
  const Tensor &q0 = tensor(a[0], "q"), &pages = tensor(a[1], "pages"), &table0 = tensor(a[2], "block_table");
  cuda(q0, "q", what);
  const int at = chunk ? 6 : 4;  // units, scale, out, workspace
  const Pages p = pages_of(pages, optional(a[at], "units"), what);
  const Tensor& seqlen = tensor(a[chunk ? 4 : 3], chunk ? "seqlen_k" : "seqlen");
  VALUE(q0.dim() == 3, "q must be (tokens, H, D), got shape ", q0.sizes());
  VALUE(q0.scalar_type() == at::kHalf || q0.scalar_type() == at::kBFloat16, "q dtype must be fp16 or bf16, got ",
        q0.scalar_type());
  VALUE(q0.size(2) == p.d, "q head_dim ", q0.size(2), " != pages head_dim ", p.d);
  VALUE(q0.size(1) >= 1 && q0.size(1) % p.hkv == 0, "n_head (", q0.size(1), ") must be a multiple of n_kv_head (",
        p.hkv, ")");
  VALUE(seqlen.dim() == 1, chunk ? "seqlen_k" : "seqlen", " must be 1-D, got shape ", seqlen.sizes());
  const int64_t rows = chunk ? seqlen.size(0) : q0.size(0);
  VALUE(seqlen.size(0) == rows, "seqlen has ", seqlen.size(0), " entries for a batch of ", rows);
  VALUE(table0.dim() == 2 && table0.size(0) == rows, "block_table must be (", rows, ", max_blocks), got shape ",
        table0.sizes());
  VALUE(table0.scalar_type() == at::kInt, "block_table must be int32, got ", table0.scalar_type());
  VALUE(index_type(seqlen), "seqlen must be int32 or int64, got ", seqlen.scalar_type());
  same_device(pages, "pages", q0, "q");
  same_device(table0, "block_table", q0, "q");
  same_device(seqlen, "seqlen", q0, "q");
  const Tensor* cu = chunk ? &tensor(a[3], "cu_seqlens_q") : nullptr;
  int64_t longest = 1;
  if (chunk) {
    VALUE(cu->dim() == 1 && cu->size(0) == rows + 1, "cu_seqlens_q must be (", rows + 1, ",), got ", cu->sizes());
    VALUE(index_type(*cu), "cu_seqlens_q must be int32 or int64, got ", cu->scalar_type());
    same_device(*cu, "cu_seqlens_q", q0, "q");
    longest = THPUtils_unpackLong(a[5]);
    VALUE(longest <= 0x7fffffff && q0.size(0) <= 0x7fffffff, "too many query tokens");
  }
  double scale = a[at + 1] == Py_None ? 1.0 / std::sqrt(double(p.d)) : PyFloat_AsDouble(a[at + 1]);
  if (PyErr_Occurred()) return nullptr;
  const c10::cuda::CUDAGuard guard(q0.device());
  Tensor out;
  if (const Tensor* o = optional(a[at + 2], "out")) {
    VALUE(o->sizes() == q0.sizes() && o->scalar_type() == q0.scalar_type() && o->device() == q0.device() &&
              o->is_contiguous() && aligned16(*o),
          "out must be a contiguous, 16-byte aligned ", q0.sizes(), " ", q0.scalar_type(), " tensor on ", q0.device());
    out = *o;
  } else {
    out = new_like(q0);
  }
  if (rows == 0 || q0.size(0) == 0 || longest <= 0) return THPVariable_Wrap(out);
  void* stream = stream_of(q0);
  Tensor ws;
  if (const Tensor* w = optional(a[at + 3], "workspace")) {
    VALUE(w->scalar_type() == at::kByte && w->is_contiguous() && w->device() == q0.device(),
          "workspace must be a contiguous uint8 tensor on ", q0.device());
    ws = *w;
  } else {
    ws = fp4_workspace(q0.device(), stream);
  }
  const Tensor q = kernel_rows(q0), lens = int32(seqlen);
  const Tensor table = (table0.size(1) > 1 && table0.stride(1) != 1) || (rows > 1 && table0.stride(0) < table0.size(1))
                           ? table0.contiguous()
                           : table0;
  const int64_t bt_stride = std::max(table.stride(0), table.size(1));  // one row may have any stride
  const int dtype = dtype_code(q.scalar_type());
  const float scale_log2 = float(scale * 1.4426950408889634);
  int status;
  if (chunk) {
    const Tensor offsets = int32(*cu);
    status = lib.pd_fp4_prefill(q.const_data_ptr(), q.size(0), q.stride(0), q.stride(1), p.data, p.n_blocks,
                                p.block_size, p.units, table.const_data_ptr<int32_t>(), bt_stride, int(table.size(1)),
                                offsets.const_data_ptr<int32_t>(), lens.const_data_ptr<int32_t>(), out.data_ptr(),
                                out.stride(0), out.stride(1), int(rows), int(longest), int(q.size(1)), int(p.hkv), p.d,
                                dtype, scale_log2, ws.data_ptr(), size_t(ws.numel()), stream);
  } else {
    status = lib.pd_fp4_decode(q.const_data_ptr(), q.stride(0), q.stride(1), p.data, p.n_blocks, p.block_size, p.units,
                               table.const_data_ptr<int32_t>(), bt_stride, int(table.size(1)),
                               lens.const_data_ptr<int32_t>(), out.data_ptr(), out.stride(0), out.stride(1), int(rows),
                               int(q.size(1)), int(p.hkv), p.d, dtype, scale_log2, ws.data_ptr(), size_t(ws.numel()),
                               stream);
  }
  if (failed(status, chunk ? "pd_fp4_prefill" : "pd_fp4_decode")) return nullptr;
  return THPVariable_Wrap(out);
}

PyObject* decode(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  arity(n, 8, "fp4_decode");
  return attend(a, false);
  END_HANDLE_TH_ERRORS
}

PyObject* prefill(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  arity(n, 10, "fp4_prefill");
  return attend(a, true);
  END_HANDLE_TH_ERRORS
}

PyObject* workspace(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  arity(n, 1, "fp4_workspace");
  const Tensor& like = tensor(a[0], "like");
  cuda(like, "like", "fp4_workspace");
  return THPVariable_Wrap(new_workspace(like.device()));
  END_HANDLE_TH_ERRORS
}

// ------------------------------------------------------------------ head norm with rotation

PyObject* norm_rope(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  arity(n, 11, "qk_norm_rope");
  const Tensor &q0 = tensor(a[0], "q"), &k0 = tensor(a[1], "k");
  cuda(q0, "q", "qk_norm_rope");
  cuda(k0, "k", "qk_norm_rope");
  VALUE(q0.dim() == 3 && k0.dim() == 3, "q must be (T, H, D) and k (T, H_kv, D), got ", q0.sizes(), " / ", k0.sizes());
  const int64_t tokens = q0.size(0), d = q0.size(2);
  VALUE(k0.size(0) == tokens && k0.size(2) == d, "q ", q0.sizes(), " and k ", k0.sizes(),
        " must share their tokens and head_dim");
  VALUE(q0.size(1) >= 1 && k0.size(1) >= 1, "q and k need at least one head each");
  VALUE(d >= 2 && d <= 256, "head_dim ", d, " is outside the kernel's range 2..256");
  const int dtype = dtype_code(q0.scalar_type());
  VALUE(dtype >= 0, "q dtype must be fp16, bf16 or fp32, got ", q0.scalar_type());
  static const char* const names[] = {"q", "k", "q_weight", "k_weight", "cos", "sin"};
  for (int i = 1; i < 6; ++i) {
    const Tensor& t = tensor(a[i], names[i]);
    VALUE(t.scalar_type() == q0.scalar_type(), names[i], " must be ", q0.scalar_type(), " like q, got ",
          t.scalar_type());
    same_device(t, names[i], q0, "q");
    if (i == 2 || i == 3)
      VALUE(t.dim() == 1 && t.size(0) == d, names[i], " must be (", d, ",), got ", t.sizes());
  }
  Tensor cos = tensor(a[4], "cos"), sin = tensor(a[5], "sin");
  VALUE(cos.dim() == 2 && cos.sizes() == sin.sizes(), "cos and sin must be (positions, rotary_dim / 2), got ",
        cos.sizes(), " / ", sin.sizes());
  const int64_t rotary = a[7] == Py_None ? 2 * cos.size(1) : THPUtils_unpackLong(a[7]);
  VALUE(rotary >= 0 && rotary % 2 == 0 && rotary <= d, "rotary_dim must be even and in [0, ", d, "], got ", rotary);
  VALUE(rotary <= 2 * cos.size(1), "rotary_dim ", rotary, " needs ", rotary / 2, " table columns, got ", cos.size(1));
  Tensor pos;
  if (const Tensor* t = optional(a[6], "positions")) {
    VALUE(index_type(*t), "positions must be int32 or int64, got ", t->scalar_type());
    VALUE(t->dim() == 1 && t->size(0) == tokens, "positions must be (", tokens, ",), got ", t->sizes());
    same_device(*t, "positions", q0, "q");
    pos = t->contiguous();
  }
  const double eps = PyFloat_AsDouble(a[8]);
  if (PyErr_Occurred()) return nullptr;
  const c10::cuda::CUDAGuard guard(q0.device());
  const Tensor q = unit_stride(q0), k = unit_stride(k0);
  cos = unit_stride(cos);
  sin = unit_stride(sin);
  const Tensor wq = tensor(a[2], "q_weight").contiguous(), wk = tensor(a[3], "k_weight").contiguous();
  auto output = [](PyObject* o, const char* name, const Tensor& like) -> Tensor {
    const Tensor* t = optional(o, name);
    if (t == nullptr) return new_like(like);
    VALUE(t->sizes() == like.sizes() && t->scalar_type() == like.scalar_type() && t->device() == like.device() &&
              t->stride(2) == 1,
          name, " must be a ", like.sizes(), " ", like.scalar_type(), " tensor on ", like.device(),
          " with a unit last stride");
    return *t;
  };
  const Tensor qo = output(a[9], "q_out", q), ko = output(a[10], "k_out", k);
  if (failed(lib.pd_qk_norm_rope(
                 q.const_data_ptr(), q.stride(0), q.stride(1), k.const_data_ptr(), k.stride(0), k.stride(1),
                 qo.data_ptr(), qo.stride(0), qo.stride(1), ko.data_ptr(), ko.stride(0), ko.stride(1),
                 wq.const_data_ptr(), wk.const_data_ptr(), cos.const_data_ptr(), sin.const_data_ptr(), cos.stride(0),
                 sin.stride(0), cos.size(0), pos.defined() ? pos.const_data_ptr() : nullptr,
                 pos.defined() ? slot_code(pos) : PD_SLOT_I64, tokens, int(q.size(1)), int(k.size(1)), int(d),
                 int(rotary), float(eps), dtype, stream_of(q)),
             "pd_qk_norm_rope"))
    return nullptr;
  return pair(qo, ko);
  END_HANDLE_TH_ERRORS
}

// ------------------------------------------------------------------ page copies

PyObject* block_copy(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  arity(n, 5, "block_copy");
  TORCH_CHECK_TYPE(PyList_Check(a[0]), "pools must be a list");
  const Py_ssize_t count = PyList_GET_SIZE(a[0]);
  VALUE(count >= 1, "copy_blocks needs at least one pool");
  const Tensor& first = tensor(PyList_GET_ITEM(a[0], 0), "pool");
  TORCH_CHECK(first.is_cuda(), "copy_blocks requires CUDA pools, got ", first.device(), "; there is no CPU path.");
  VALUE(first.dim() >= 2 && first.numel() > 0, "a pool needs (n_blocks, ...) elements, got ", first.sizes());
  std::vector<void*> pools(count);
  for (Py_ssize_t i = 0; i < count; ++i) {
    const Tensor& t = tensor(PyList_GET_ITEM(a[0], i), "pool");
    VALUE(t.sizes() == first.sizes() && t.scalar_type() == first.scalar_type() && t.device() == first.device() &&
              t.is_contiguous(),
          "every pool must be a contiguous ", first.sizes(), " ", first.scalar_type(), " tensor on ", first.device());
    pools[i] = t.data_ptr();
  }
  const int64_t n_blocks = first.size(0);
  Tensor ids[2] = {tensor(a[1], "src"), tensor(a[2], "dst")};
  static const char* const names[] = {"src", "dst"};
  const c10::cuda::CUDAGuard guard(first.device());
  for (int i = 0; i < 2; ++i) {
    VALUE(ids[i].dim() == 1 && index_type(ids[i]), names[i], " must be a 1-D int32 or int64 tensor, got ",
          ids[i].sizes(), " ", ids[i].scalar_type());
    same_device(ids[i], names[i], first, "the pools");
  }
  VALUE(ids[0].numel() == ids[1].numel(), "src has ", ids[0].numel(), " blocks and dst ", ids[1].numel());
  const bool mixed = ids[0].scalar_type() != ids[1].scalar_type();
  for (Tensor& t : ids) t = (mixed ? t.to(at::kLong) : t).contiguous();
  const Tensor *table = optional(a[3], "block_table"), *remap0 = optional(a[4], "remap");
  VALUE((table == nullptr) == (remap0 == nullptr), "block_table and remap go together");
  Tensor remap;
  if (table != nullptr) {
    VALUE(table->dim() == 2 && table->scalar_type() == at::kInt, "block_table must be an int32 (B, max_blocks) tensor");
    same_device(*table, "block_table", first, "the pools");
    VALUE(table->size(1) <= 1 || table->stride(1) == 1,
          "block_table needs a unit column stride (it is renumbered in place)");
    VALUE(table->size(0) <= 1 || table->stride(0) >= table->size(1),
          "block_table rows must not overlap (it is renumbered in place)");
    VALUE(remap0->scalar_type() == at::kInt && remap0->dim() == 1 && remap0->size(0) == n_blocks,
          "remap must be an int32 (", n_blocks, ",) tensor");
    same_device(*remap0, "remap", first, "the pools");
    remap = remap0->contiguous();
  }
  const int64_t rows = table ? table->size(0) : 0, cols = table ? table->size(1) : 0;
  if (failed(lib.pd_block_copy(pools.data(), int(count), n_blocks, first.numel() / n_blocks * first.element_size(),
                               ids[0].const_data_ptr(), ids[1].const_data_ptr(), slot_code(ids[0]), ids[0].numel(),
                               table ? table->data_ptr<int32_t>() : nullptr, rows, cols,
                               table ? std::max(table->stride(0), cols) : 0,
                               remap.defined() ? remap.const_data_ptr<int32_t>() : nullptr, stream_of(first)),
             "pd_block_copy"))
    return nullptr;
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

// ------------------------------------------------------------------ a cache of bounded length

struct Pools {
  int64_t n_blocks, hkv;
  int block_size, d, dtype;
  int64_t ks[3], vs[3];
};

// One layer's K and V pools as the kernels take them.
Pools pools_of(const Tensor& k, const Tensor& v, const char* what) {
  cuda(k, "k_cache", what);
  cuda(v, "v_cache", what);
  VALUE(k.dim() == 4 && v.dim() == 4, "k_cache/v_cache must be (n_blocks, block_size, H_kv, D), got ", k.sizes(), " / ",
        v.sizes());
  VALUE(k.sizes() == v.sizes(), "k_cache/v_cache shapes differ: ", k.sizes(), " vs ", v.sizes());
  Pools p;
  p.dtype = dtype_code(k.scalar_type());
  VALUE(p.dtype >= 0 && v.scalar_type() == k.scalar_type(), "k_cache/v_cache must share one dtype of fp32, fp16 or bf16, got ",
        k.scalar_type(), " / ", v.scalar_type());
  same_device(v, "v_cache", k, "k_cache");
  p.n_blocks = k.size(0);
  p.hkv = k.size(2);
  const int64_t bs = k.size(1), d = k.size(3);
  VALUE(p.n_blocks >= 1 && p.hkv >= 1 && p.hkv <= 65535, "k_cache needs blocks and 1 to 65535 heads, got ", k.sizes());
  VALUE(bs >= 1 && (bs & (bs - 1)) == 0 && bs <= (1 << 30), "block_size must be a power of two, got ", bs);
  VALUE(d >= 8 && d <= 256 && (d & (d - 1)) == 0, "head_dim must be a power of two in 8..256, got ", d);
  p.block_size = int(bs);
  p.d = int(d);
  const int64_t es = k.element_size();
  VALUE(std::min(bs * d * es, int64_t(4096)) % 128 == 0, "a block of one head needs a multiple of 128 bytes, got ", bs * d * es);
  for (const bool first : {true, false}) {  // (k and v may be one tensor)
    const Tensor* t = first ? &k : &v;
    VALUE(t->stride(3) == 1 && aligned16(*t), "a pool needs a unit head_dim stride and a 16-byte aligned base");
    for (int i = 0; i < 3; ++i) {
      VALUE(t->stride(i) > 0 && t->stride(i) * es % 16 == 0, "a pool's strides must be positive multiples of 16 bytes, got ",
            t->strides());
      (first ? p.ks : p.vs)[i] = t->stride(i);
    }
  }
  return p;
}

// An int32 block table of `rows` rows with unit columns (a copy where it has other strides).
Tensor table_of(const Tensor& t, const char* name, int64_t rows, const Tensor& as, const char* as_name) {
  VALUE(t.dim() == 2 && t.size(0) == rows, name, " must be (", rows, ", max_blocks), got shape ", t.sizes());
  VALUE(t.scalar_type() == at::kInt, name, " must be int32, got ", t.scalar_type());
  VALUE(t.size(1) <= 0x7fffffff, name, " is too wide");
  same_device(t, name, as, as_name);
  return (t.size(1) > 1 && t.stride(1) != 1) || (rows > 1 && t.stride(0) < t.size(1)) ? t.contiguous() : t;
}

// Whether no two rows (runs of the last, unit-stride dimension) of t share memory, as nested strides tell.
bool disjoint_rows(const Tensor& t) {
  if (t.numel() == 0) return true;
  std::vector<std::pair<int64_t, int64_t>> dims;  // (stride, size)
  for (int64_t i = 0; i + 1 < t.dim(); ++i)
    if (t.size(i) > 1) dims.emplace_back(t.stride(i), t.size(i));
  std::sort(dims.begin(), dims.end());
  int64_t extent = t.size(t.dim() - 1);
  for (const auto& [stride, size] : dims) {
    if (stride < extent) return false;
    extent += stride * (size - 1);
  }
  return true;
}

Tensor aligned_rows(const Tensor& q0) {
  const int64_t es = q0.element_size();
  if (q0.stride(2) == 1 && q0.stride(0) * es % 16 == 0 && q0.stride(1) * es % 16 == 0 && aligned16(q0)) return q0;
  const Tensor q = q0.contiguous();
  return aligned16(q) && q.data_ptr() != q0.data_ptr() ? q : q0.clone(at::MemoryFormat::Contiguous);
}

// window and sinks, cut to what no row exceeds.
void window_of(PyObject* w, PyObject* s, int64_t& window, int64_t& sinks) {
  window = THPUtils_unpackLong(w);
  sinks = THPUtils_unpackLong(s);
  VALUE(window >= 1, "window must be at least 1, got ", window);
  VALUE(sinks >= 0, "sinks must be at least 0, got ", sinks);
  window = std::min<int64_t>(window, 1 << 30);
  sinks = std::min<int64_t>(sinks, 1 << 30);
}

// What every attention call over pools asks of q.
void queries_of(const Tensor& q, const Tensor& k, const Pools& p, const char* shape) {
  VALUE(q.dim() == 3, "q must be ", shape, ", got shape ", q.sizes());
  VALUE(q.scalar_type() == k.scalar_type(), "q/k_cache/v_cache must share one dtype, got ", q.scalar_type(), ", ",
        k.scalar_type());
  VALUE(q.size(2) == p.d, "q head_dim ", q.size(2), " != cache head_dim ", p.d);
  VALUE(q.size(1) >= 1 && q.size(1) % p.hkv == 0, "n_head (", q.size(1), ") must be a multiple of n_kv_head (", p.hkv, ")");
  same_device(k, "k_cache", q, "q");
}

// Whether the spans of memory from the first to the last element of a and b meet.
bool spans_meet(const Tensor& a, const Tensor& b) {
  if (a.numel() == 0 || b.numel() == 0) return false;
  auto end = [](const Tensor& t) {
    int64_t last = 1;
    for (int64_t i = 0; i < t.dim(); ++i) last += (t.size(i) - 1) * t.stride(i);
    return static_cast<const char*>(t.const_data_ptr()) + last * t.element_size();
  };
  return static_cast<const char*>(a.const_data_ptr()) < end(b) && static_cast<const char*>(b.const_data_ptr()) < end(a);
}

// The result of a call: `given` (contiguous, like q, apart from it) or a new tensor.
Tensor result_of(PyObject* given, const Tensor& q) {
  const Tensor* o = optional(given, "out");
  if (o == nullptr) return new_like(q);
  VALUE(o->sizes() == q.sizes() && o->scalar_type() == q.scalar_type() && o->device() == q.device() &&
            o->is_contiguous() && aligned16(*o),
        "out must be a contiguous, 16-byte aligned ", q.sizes(), " ", q.scalar_type(), " tensor on ", q.device());
  VALUE(!spans_meet(*o, q), "out must not share memory with q");
  return *o;
}

// prefill_window(q, k, v, table, cu, seqlen, longest, window, sinks, scale, out)
PyObject* prefill_window(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  arity(n, 11, "prefill_window");
  const Tensor &q0 = tensor(a[0], "q"), &k = tensor(a[1], "k_cache"), &v = tensor(a[2], "v_cache");
  const Tensor &cu = tensor(a[4], "cu_seqlens_q"), &seqlen = tensor(a[5], "seqlen_k");
  cuda(q0, "q", "paged_prefill_window");
  const Pools p = pools_of(k, v, "paged_prefill_window");
  queries_of(q0, k, p, "(total_q, H, D)");
  VALUE(p.dtype != PD_F32, "paged_prefill_window needs fp16 or bf16, got fp32");
  VALUE(p.d >= 64, "head_dim must be 64, 128 or 256, got ", p.d);
  VALUE(p.block_size >= 8, "block_size must be at least 8, got ", p.block_size);
  VALUE(seqlen.dim() == 1, "seqlen_k must be 1-D, got shape ", seqlen.sizes());
  const int64_t rows = seqlen.size(0), heads = q0.size(1), total = q0.size(0);
  VALUE(rows <= 0x7fffffff && total <= (1 << 30) / heads, "too many query rows");
  VALUE(index_type(seqlen), "seqlen_k must be int32 or int64, got ", seqlen.scalar_type());
  same_device(seqlen, "seqlen_k", q0, "q");
  VALUE(cu.dim() == 1 && cu.size(0) == rows + 1, "cu_seqlens_q must be (", rows + 1, ",), got ", cu.sizes());
  VALUE(index_type(cu), "cu_seqlens_q must be int32 or int64, got ", cu.scalar_type());
  same_device(cu, "cu_seqlens_q", q0, "q");
  const c10::cuda::CUDAGuard guard(q0.device());
  const Tensor table = table_of(tensor(a[3], "block_table"), "block_table", rows, q0, "q");
  VALUE(table.size(1) * p.block_size <= (int64_t(1) << 30), "a row's table holds at most 2^30 tokens");
  const int64_t longest = std::min<int64_t>(THPUtils_unpackLong(a[6]), total);
  int64_t window, sinks;
  window_of(a[7], a[8], window, sinks);
  const double scale = a[9] == Py_None ? 1.0 / std::sqrt(double(p.d)) : PyFloat_AsDouble(a[9]);
  if (PyErr_Occurred()) return nullptr;
  const Tensor out = result_of(a[10], q0);
  if (rows == 0 || longest <= 0) return THPVariable_Wrap(out);
  const Tensor q = aligned_rows(q0), offsets = int32(cu), lens = int32(seqlen);
  if (failed(lib.pd_prefill_window(q.const_data_ptr(), total, q.stride(0), q.stride(1), k.const_data_ptr(),
                                   v.const_data_ptr(), p.n_blocks, p.block_size, p.ks, p.vs,
                                   table.const_data_ptr<int32_t>(), std::max(table.stride(0), table.size(1)),
                                   int(table.size(1)), offsets.const_data_ptr<int32_t>(), lens.const_data_ptr<int32_t>(),
                                   int(window), int(sinks), out.data_ptr(), out.stride(0), out.stride(1), int(rows),
                                   int(longest), int(heads), int(p.hkv), p.d, p.dtype,
                                   float(scale * 1.4426950408889634), stream_of(q0)),
             "pd_prefill_window"))
    return nullptr;
  return THPVariable_Wrap(out);
  END_HANDLE_TH_ERRORS
}

// decode_window(q, k, v, table, seqlen, window, sinks, scale, out, workspace) and
// decode_weights(q, k, v, table, seqlen, weights, scale, out, workspace).
PyObject* decode_variant(PyObject* const* a, bool windowed) {
  const char* what = windowed ? "paged_decode_window" : "paged_decode_weights";
  const Tensor &q0 = tensor(a[0], "q"), &k = tensor(a[1], "k_cache"), &v = tensor(a[2], "v_cache");
  const Tensor &table0 = tensor(a[3], "block_table"), &seqlen = tensor(a[4], "seqlen");
  cuda(q0, "q", what);
  const Pools p = pools_of(k, v, what);
  queries_of(q0, k, p, "(B, H, D)");
  const int64_t rows = q0.size(0), heads = q0.size(1);
  VALUE(rows <= 0x7fffffff / heads, "too many query rows");
  VALUE(seqlen.dim() == 1 && seqlen.size(0) == rows, "seqlen must be (", rows, ",), got shape ", seqlen.sizes());
  VALUE(index_type(seqlen), "seqlen must be int32 or int64, got ", seqlen.scalar_type());
  same_device(seqlen, "seqlen", q0, "q");
  const c10::cuda::CUDAGuard guard(q0.device());
  const Tensor table = table_of(table0, "block_table", rows, q0, "q");
  const int64_t capacity = table.size(1) * p.block_size;
  VALUE(capacity <= (int64_t(1) << 30), "a row's table holds at most 2^30 tokens, got ", capacity);
  int64_t window = 0, sinks = 0;
  const Tensor* weights = nullptr;
  if (windowed) {
    window_of(a[5], a[6], window, sinks);
  } else {
    weights = &tensor(a[5], "weights");
    VALUE(weights->scalar_type() == at::kFloat && weights->dim() == 3 && weights->size(0) == rows &&
              weights->size(1) == p.hkv && weights->size(2) >= capacity,
          "weights must be float32 (", rows, ", ", p.hkv, ", at least ", capacity, "), got ", weights->sizes(), " ",
          weights->scalar_type());
    same_device(*weights, "weights", q0, "q");
    VALUE(weights->size(2) <= 1 || weights->stride(2) == 1, "weights needs a unit last stride (it is updated in place)");
    VALUE(disjoint_rows(*weights), "weights rows must not overlap (it is updated in place), got strides ",
          weights->strides());
  }
  const int at = windowed ? 7 : 6;  // scale, out, workspace
  const double scale = a[at] == Py_None ? 1.0 / std::sqrt(double(p.d)) : PyFloat_AsDouble(a[at]);
  if (PyErr_Occurred()) return nullptr;
  const Tensor out = result_of(a[at + 1], q0);
  if (rows == 0) return THPVariable_Wrap(out);
  void* stream = stream_of(q0);
  const bool small = lib.pd_decode_window_small(int(rows), int(heads), int(p.hkv), p.d, p.dtype, p.block_size,
                                                int(table.size(1)), int(window), int(sinks)) != 0;
  const Tensor* w = optional(a[at + 2], "workspace");
  const int64_t need = small && w == nullptr ? 0
                                             : int64_t(lib.pd_decode_window_workspace_bytes(int(rows), int(heads),
                                                                                            int(p.hkv), p.d, p.dtype));
  Tensor ws;
  if (w != nullptr) {
    VALUE(w->scalar_type() == at::kByte && w->is_contiguous() && w->device() == q0.device() && w->numel() >= need,
          "workspace must be a contiguous uint8 tensor of at least ", need, " bytes on ", q0.device());
    ws = *w;
  } else if (!small) {
    ws = decode_workspace(q0.device(), stream, need);
  }
  void* const ws_ptr = ws.defined() ? ws.data_ptr() : nullptr;
  const size_t ws_bytes = ws.defined() ? size_t(ws.numel()) : 0;
  const Tensor q = aligned_rows(q0);
  const Tensor lens = int32(seqlen);
  const int64_t bt_stride = std::max(table.stride(0), table.size(1));  // one row may have any stride
  const float scale_log2 = float(scale * 1.4426950408889634);
  int status;
  if (windowed) {
    status = lib.pd_decode_window(q.const_data_ptr(), q.stride(0), q.stride(1), k.const_data_ptr(), v.const_data_ptr(),
                                  p.n_blocks, p.block_size, p.ks, p.vs, table.const_data_ptr<int32_t>(), bt_stride,
                                  int(table.size(1)), lens.const_data_ptr<int32_t>(), int(window), int(sinks),
                                  out.data_ptr(), out.stride(0), out.stride(1), int(rows), int(heads), int(p.hkv), p.d,
                                  p.dtype, scale_log2, ws_ptr, ws_bytes, stream);
  } else {
    Tensor scratch;
    if (!small)
      scratch = at::detail::empty_cuda(
          {int64_t(lib.pd_decode_weights_scratch_bytes(int(rows), int(heads), int(table.size(1)), p.block_size))}, at::kByte,
          q0.device(), std::nullopt);
    status = lib.pd_decode_weights(q.const_data_ptr(), q.stride(0), q.stride(1), k.const_data_ptr(), v.const_data_ptr(),
                                   p.n_blocks, p.block_size, p.ks, p.vs, table.const_data_ptr<int32_t>(), bt_stride,
                                   int(table.size(1)), lens.const_data_ptr<int32_t>(), weights->data_ptr<float>(),
                                   weights->stride(0), weights->stride(1), weights->size(2), out.data_ptr(),
                                   out.stride(0), out.stride(1), int(rows), int(heads), int(p.hkv), p.d, p.dtype,
                                   scale_log2, ws_ptr, ws_bytes, small ? nullptr : scratch.data_ptr(),
                                   small ? 0 : size_t(scratch.numel()), stream);
  }
  if (failed(status, windowed ? "pd_decode_window" : "pd_decode_weights")) return nullptr;
  return THPVariable_Wrap(out);
}

PyObject* decode_window(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  arity(n, 10, "decode_window");
  return decode_variant(a, true);
  END_HANDLE_TH_ERRORS
}

PyObject* decode_weights(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  arity(n, 9, "decode_weights");
  return decode_variant(a, false);
  END_HANDLE_TH_ERRORS
}

// decode_window_workspace(rows, heads, kv_heads, head_dim, like): a workspace for calls of that shape.
PyObject* decode_window_workspace(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  arity(n, 5, "decode_window_workspace");
  const Tensor& like = tensor(a[4], "like");
  cuda(like, "like", "decode_workspace");
  int64_t x[4];
  for (int i = 0; i < 4; ++i) {
    x[i] = THPUtils_unpackLong(a[i]);
    VALUE(x[i] >= 0 && x[i] <= 0x7fffffff, "sizes must be 31-bit");
  }
  const c10::cuda::CUDAGuard guard(like.device());
  const size_t bytes = lib.pd_decode_window_workspace_bytes(int(x[0]), int(x[1]), int(x[2]), int(x[3]),
                                                            dtype_code(like.scalar_type()));
  VALUE(bytes > 0, "no decode of ", x[0], " rows of ", x[1], " heads on ", x[2], " of ", x[3], " in ", like.scalar_type());
  return THPVariable_Wrap(at::detail::empty_cuda({int64_t(bytes)}, at::kByte, like.device(), std::nullopt));
  END_HANDLE_TH_ERRORS
}

// evict(ks, vs, table, seqlen, weights, keep, recent, sinks, new_table, seqlen_out, weights_out)
PyObject* evict(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  arity(n, 11, "evict");
  TORCH_CHECK_TYPE(PyList_Check(a[0]) && PyList_Check(a[1]), "k_caches and v_caches must be lists");
  const Py_ssize_t layers = PyList_GET_SIZE(a[0]);
  VALUE(layers >= 1 && PyList_GET_SIZE(a[1]) == layers, "evict_tokens needs one k_cache and v_cache per layer, got ", layers,
        " / ", PyList_GET_SIZE(a[1]));
  VALUE(layers <= 65535, "too many layers");
  const Tensor &k0 = tensor(PyList_GET_ITEM(a[0], 0), "k_cache"), &v0 = tensor(PyList_GET_ITEM(a[1], 0), "v_cache");
  const Pools p = pools_of(k0, v0, "evict_tokens");
  std::vector<void*> ks(layers), vs(layers);
  for (Py_ssize_t i = 0; i < layers; ++i) {
    const Tensor &k = tensor(PyList_GET_ITEM(a[0], i), "k_cache"), &v = tensor(PyList_GET_ITEM(a[1], i), "v_cache");
    for (const auto& [t, first] : {std::make_pair(&k, &k0), std::make_pair(&v, &v0)})
      VALUE(t->sizes() == first->sizes() && t->strides() == first->strides() && t->scalar_type() == first->scalar_type() &&
                t->device() == first->device() && aligned16(*t),
            "every layer's pools must have one shape, layout, dtype and device, 16-byte aligned; layer ", i, " has ",
            t->sizes(), " ", t->strides(), " ", t->scalar_type(), " on ", t->device());
    ks[i] = k.data_ptr();
    vs[i] = v.data_ptr();
  }
  std::vector<void*> named(ks);
  named.insert(named.end(), vs.begin(), vs.end());
  std::sort(named.begin(), named.end());
  VALUE(std::adjacent_find(named.begin(), named.end()) == named.end(), "a pool is named twice, and its tokens would be moved twice");
  const Tensor &seqlen0 = tensor(a[3], "seqlen"), &weights = tensor(a[4], "weights");
  VALUE(seqlen0.dim() == 1, "seqlen must be (B,), got shape ", seqlen0.sizes());
  VALUE(index_type(seqlen0), "seqlen must be int32 or int64, got ", seqlen0.scalar_type());
  same_device(seqlen0, "seqlen", k0, "the pools");
  const int64_t rows = seqlen0.size(0);
  const c10::cuda::CUDAGuard guard(k0.device());
  const Tensor table = table_of(tensor(a[2], "block_table"), "block_table", rows, k0, "the pools");
  const int64_t capacity = table.size(1) * p.block_size;
  VALUE(capacity <= (int64_t(1) << 30), "a row's table holds at most 2^30 tokens, got ", capacity);
  auto sums = [&](const Tensor& t, const char* name) {
    VALUE(t.scalar_type() == at::kFloat && t.dim() == 4 && t.size(0) == layers && t.size(1) == rows && t.size(2) == p.hkv &&
              t.size(3) >= capacity,
          name, " must be float32 (", layers, ", ", rows, ", ", p.hkv, ", at least ", capacity, "), got ", t.sizes(), " ",
          t.scalar_type());
    same_device(t, name, k0, "the pools");
    VALUE(t.size(3) <= 1 || t.stride(3) == 1, name, " needs a unit last stride");
  };
  sums(weights, "weights");
  const int64_t keep0 = THPUtils_unpackLong(a[5]), recent = THPUtils_unpackLong(a[6]), sinks = THPUtils_unpackLong(a[7]);
  VALUE(keep0 >= 1, "keep must be at least 1, got ", keep0);
  VALUE(recent >= 0 && sinks >= 0 && recent <= keep0 && sinks <= keep0 - recent,
        "recent and sinks must be at least 0 and fit into keep (", keep0, "), got ", recent, " and ", sinks);
  // a budget that no row exceeds evicts nothing, whatever it is
  const bool all_fit = keep0 > capacity;
  const int keep = all_fit ? int(capacity) + 1 : int(keep0);
  Tensor fresh;
  if (const Tensor* t = optional(a[8], "new_table")) {
    VALUE(t->numel() == 0 || t->const_data_ptr() != tensor(a[2], "block_table").const_data_ptr(),
          "new_table is block_table itself (without it tokens move within their own pages)");
    fresh = table_of(*t, "new_table", rows, k0, "the pools");
    VALUE(fresh.size(1) * p.block_size >= std::min<int64_t>(keep, capacity), "new_table holds ", fresh.size(1) * p.block_size,
          " tokens, but rows may keep ", std::min<int64_t>(keep, capacity));
    VALUE(fresh.size(1) * p.block_size <= (int64_t(1) << 30), "a row's table holds at most 2^30 tokens");
  }
  Tensor lens_out, sums_out;
  if (const Tensor* t = optional(a[9], "seqlen_out")) {
    VALUE(t->dim() == 1 && t->size(0) == rows && t->scalar_type() == at::kInt && t->is_contiguous(),
          "seqlen_out must be a contiguous int32 (", rows, ",) tensor, got ", t->sizes(), " ", t->scalar_type());
    same_device(*t, "seqlen_out", k0, "the pools");
    lens_out = *t;
  } else {
    lens_out = at::detail::empty_cuda({rows}, at::kInt, k0.device(), std::nullopt);
  }
  if (const Tensor* t = optional(a[10], "weights_out")) {
    sums(*t, "weights_out");
    VALUE(t->size(3) == weights.size(3), "weights_out must be as long as weights, got ", t->size(3), " and ", weights.size(3));
    VALUE(t->is_contiguous() || (t->data_ptr() == weights.data_ptr() && t->strides() == weights.strides()),
          "weights_out must be contiguous, or weights itself");
    VALUE((t->data_ptr() == weights.data_ptr() && t->strides() == weights.strides()) || !spans_meet(*t, weights),
          "weights_out shares weights' memory, but not as weights itself");
    VALUE(disjoint_rows(*t), "weights_out rows must not overlap, got strides ", t->strides());
    sums_out = *t;
  } else {
    sums_out = at::detail::empty_cuda(weights.sizes(), at::kFloat, k0.device(), std::nullopt);
  }
  if (rows == 0) return pair(lens_out, sums_out);
  const Tensor lens = int32(seqlen0);
  const int64_t bytes = int64_t(lib.pd_evict_scratch_bytes(int(layers), int(rows), int(p.hkv), keep));
  const Tensor scratch = at::detail::empty_cuda({bytes}, at::kByte, k0.device(), std::nullopt);
  const int64_t w_st[3] = {weights.stride(0), weights.stride(1), weights.stride(2)};
  const int64_t wo_st[3] = {sums_out.stride(0), sums_out.stride(1), sums_out.stride(2)};
  if (failed(lib.pd_evict(ks.data(), vs.data(), int(layers), p.n_blocks, p.block_size, int(p.hkv), p.d, p.dtype, p.ks, p.vs,
                          table.const_data_ptr<int32_t>(), std::max(table.stride(0), table.size(1)), int(table.size(1)),
                          fresh.defined() ? fresh.const_data_ptr<int32_t>() : nullptr,
                          fresh.defined() ? std::max(fresh.stride(0), fresh.size(1)) : 0,
                          fresh.defined() ? int(fresh.size(1)) : 0, lens.const_data_ptr<int32_t>(),
                          lens_out.data_ptr<int32_t>(), weights.const_data_ptr<float>(), w_st, sums_out.data_ptr<float>(),
                          wo_st, weights.size(3), int(rows), keep, all_fit ? 0 : int(recent), all_fit ? 0 : int(sinks),
                          scratch.data_ptr(), size_t(bytes), stream_of(k0)),
             "pd_evict"))
    return nullptr;
  return pair(lens_out, sums_out);
  END_HANDLE_TH_ERRORS
}

// bind(addresses, check): {"pd_...": int} of the loaded library, and _native.check.
PyObject* bind(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  arity(n, 2, "bind");
  TORCH_CHECK_TYPE(PyDict_Check(a[0]), "bind takes a dict of addresses");
#define PD_BIND(name)                                                    \
  {                                                                      \
    PyObject* v = PyDict_GetItemString(a[0], #name);                     \
    VALUE(v != nullptr, "no address of ", #name);                        \
    lib.name = reinterpret_cast<decltype(&::name)>(PyLong_AsVoidPtr(v)); \
  }
  PD_ENTRIES(PD_BIND)
  Py_INCREF(a[1]);
  Py_XDECREF(check_status);
  check_status = a[1];
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

#define PD_METHOD(name, fn) {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(fn)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {
    PD_METHOD("bind", bind),
    PD_METHOD("qk_norm_rope", norm_rope),
    PD_METHOD("fp4_write_slots", write_slots),
    PD_METHOD("fp4_write_table", write_table),
    PD_METHOD("fp4_read_slots", read_slots),
    PD_METHOD("fp4_decode", decode),
    PD_METHOD("fp4_prefill", prefill),
    PD_METHOD("fp4_workspace", workspace),
    PD_METHOD("block_copy", block_copy),
    PD_METHOD("decode_window", decode_window),
    PD_METHOD("decode_weights", decode_weights),
    PD_METHOD("prefill_window", prefill_window),
    PD_METHOD("decode_window_workspace", decode_window_workspace),
    PD_METHOD("evict", evict),
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "pd_ops", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_pd_ops() { return PyModule_Create(&module); }
