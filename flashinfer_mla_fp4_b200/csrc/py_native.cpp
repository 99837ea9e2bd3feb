// Native call path of the Python entry points (extension module `_native`).
//
// A decode step of a short batch takes the GPU ten to twenty microseconds; the same call made of Python attribute
// accesses, ctypes conversions and context managers took the host 22 us (16 us for a cache write), so small steps ran at
// the speed of the interpreter.  Here the common form of a call is checked, filled into the C ABI's argument block and
// launched from one C function.  Every function returns None (False) without having done anything when the call is
// not of the common form: another layout or dtype, a host tensor, an argument that is wrong.  The Python caller then
// goes through its own checks, which also word the error messages, and through ctypes.
//
// The GIL is let go around allocations and launches: a launch blocks while the stream's queue is full, and what is queued may wait
// for another Python thread (a host callback, say).
//
// The kernels stay behind the C ABI: bind() receives the addresses of its functions from the loaded library, so this
// module works with whichever build of the library was loaded and links against none.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <algorithm>
#include <cstdlib>
#include <string>

#include <ATen/ATen.h>
#include <ATen/core/CachingHostAllocator.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <cuda_runtime_api.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/mla_fp4_b200.h"

namespace {

struct Abi {
  decltype(&mla_fp4_decode) decode = nullptr;
  decltype(&mla_fp4_workspace_bytes) workspace_bytes = nullptr;
  decltype(&mla_fp4_cache_write) cache_write = nullptr;
  decltype(&mla_fp4_step_metadata) step_metadata = nullptr;
  decltype(&mla_fp4_last_error) last_error = nullptr;
  decltype(&mla_fp4_summarize_pages) summarize_pages = nullptr;
  decltype(&mla_fp4_summarize_new_pages) summarize_new_pages = nullptr;
  decltype(&mla_fp4_select_workspace_bytes) select_workspace_bytes = nullptr;
  decltype(&mla_fp4_select_pages) select_pages = nullptr;
  decltype(&mla_fp4_pool_workspace_bytes) pool_workspace_bytes = nullptr;
  decltype(&mla_fp4_pool_allocate) pool_allocate = nullptr;
  decltype(&mla_fp4_pool_fork) pool_fork = nullptr;
  decltype(&mla_fp4_pool_free) pool_free = nullptr;
  decltype(&mla_fp4_pool_compact) pool_compact = nullptr;
} abi;

// Without the GIL for as long as it lives.
struct NoGil {
  PyThreadState* state = PyEval_SaveThread();
  NoGil() = default;
  NoGil(const NoGil&) = delete;
  NoGil& operator=(const NoGil&) = delete;
  ~NoGil() { PyEval_RestoreThread(state); }
};

// The exception that the Python binding raises for a status (_cabi.check).
PyObject* raise_status(int rc) {
  const std::string msg = abi.last_error();
  if (rc == MLA_FP4_ERR_BAD_ARG || rc == MLA_FP4_ERR_UNSUPPORTED || rc == MLA_FP4_ERR_WORKSPACE_TOO_SMALL)
    PyErr_SetString(PyExc_ValueError, msg.c_str());
  else
    PyErr_Format(PyExc_RuntimeError, "mla_fp4 error %d: %s", rc, msg.c_str());
  return nullptr;
}

const at::Tensor* tensor(PyObject* o) { return THPVariable_Check(o) ? &THPVariable_Unpack(o) : nullptr; }
bool on(const at::Tensor& t, const at::Device& d) { return t.is_cuda() && t.device() == d; }
bool validating() {
  const char* v = std::getenv("MLA_FP4_VALIDATE");
  return v && *v && !(v[0] == '0' && !v[1]);
}
// A number as a double / an integer; anything else (a tensor, say) is left to the Python path.
bool number(PyObject* o, double* v) {
  if (PyFloat_Check(o)) *v = PyFloat_AS_DOUBLE(o);
  else if (PyLong_Check(o)) *v = PyLong_AsDouble(o);
  else return false;
  if (*v == -1.0 && PyErr_Occurred()) {
    PyErr_Clear();
    return false;
  }
  return true;
}
bool integer(PyObject* o, int64_t* v) {
  if (!PyLong_Check(o)) return false;
  int overflow = 0;
  *v = PyLong_AsLongLongAndOverflow(o, &overflow);
  return overflow == 0;
}

bool addresses(PyObject* const* a, Py_ssize_t n, Py_ssize_t wanted, void** p) {
  if (n != wanted) {
    PyErr_Format(PyExc_TypeError, "bind takes %zd addresses", wanted);
    return false;
  }
  for (Py_ssize_t i = 0; i < n; ++i) {
    p[i] = PyLong_AsVoidPtr(a[i]);
    if (!p[i]) {
      if (!PyErr_Occurred()) PyErr_Format(PyExc_ValueError, "null address");
      return false;
    }
  }
  return true;
}
template <typename F>
void set(F& f, void* p) { f = reinterpret_cast<F>(p); }

// bind(decode, workspace_bytes, cache_write, step_metadata, last_error): addresses in the loaded library
PyObject* bind(PyObject*, PyObject* const* a, Py_ssize_t n) {
  void* p[5];
  if (!addresses(a, n, 5, p)) return nullptr;
  set(abi.decode, p[0]);
  set(abi.workspace_bytes, p[1]);
  set(abi.cache_write, p[2]);
  set(abi.step_metadata, p[3]);
  set(abi.last_error, p[4]);
  Py_RETURN_NONE;
}
// bind_sparse(summarize_pages, summarize_new_pages, select_workspace_bytes, select_pages, pool_workspace_bytes, pool_allocate, pool_fork, pool_free,
// pool_compact)
PyObject* bind_sparse(PyObject*, PyObject* const* a, Py_ssize_t n) {
  void* p[9];
  if (!addresses(a, n, 9, p)) return nullptr;
  set(abi.summarize_pages, p[0]);
  set(abi.summarize_new_pages, p[1]);
  set(abi.select_workspace_bytes, p[2]);
  set(abi.select_pages, p[3]);
  set(abi.pool_workspace_bytes, p[4]);
  set(abi.pool_allocate, p[5]);
  set(abi.pool_fork, p[6]);
  set(abi.pool_free, p[7]);
  set(abi.pool_compact, p[8]);
  Py_RETURN_NONE;
}

// decode(workspace, status, num_heads, page_size, out_code, kernel, num_ctas, pdl, phase_mask, soft_cap, sink, wait_polls,
//        q, kv_cache, block_tables, seq_lens, max_seq_len, softmax_scale, output_scale, out, kv_cache_sf, return_lse, lse_out)
// -> out, (out, lse), or None when the call is not of the common form.
PyObject* decode(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 23) return PyErr_Format(PyExc_TypeError, "decode takes 23 arguments");
  const at::Tensor *ws = tensor(a[0]), *status = tensor(a[1]), *q = tensor(a[12]), *kv = tensor(a[13]), *bt = tensor(a[14]),
                   *sl = tensor(a[15]), *sf = tensor(a[20]);
  if (!ws || !status || !q || !kv || !bt || !sl || !sf) Py_RETURN_NONE;
  int64_t heads, page, out_code, kernel, ctas, phase, polls, max_len;
  double cap, scale, out_scale;
  if (!integer(a[2], &heads) || !integer(a[3], &page) || !integer(a[4], &out_code) || !integer(a[5], &kernel) || !integer(a[6], &ctas) ||
      !integer(a[8], &phase) || !number(a[9], &cap) || !integer(a[11], &polls) || !integer(a[16], &max_len) || !number(a[17], &scale) ||
      !number(a[18], &out_scale))
    Py_RETURN_NONE;
  const at::Device dev = ws->device();
  if (!on(*q, dev) || !on(*kv, dev) || !on(*bt, dev) || !on(*sl, dev) || !on(*sf, dev) || !on(*status, dev)) Py_RETURN_NONE;
  if (q->dim() != 4 || q->size(2) != heads || q->size(3) != MLA_FP4_LATENT_DIM + MLA_FP4_ROPE_DIM || q->stride(3) != 1 ||
      q->scalar_type() != at::kFloat8_e4m3fn)
    Py_RETURN_NONE;
  const int64_t batch = q->size(0), q_len = q->size(1);
  if (kv->dim() != 3 || kv->scalar_type() != at::kByte || kv->size(1) != page || kv->size(2) != MLA_FP4_ROW_BYTES || !kv->is_contiguous())
    Py_RETURN_NONE;
  if (sf->dim() != 3 || sf->scalar_type() != at::kFloat || sf->size(0) != kv->size(0) || sf->size(1) != page || sf->size(2) != 1 ||
      !sf->is_contiguous())
    Py_RETURN_NONE;
  if (bt->dim() != 2 || bt->scalar_type() != at::kInt || bt->stride(1) != 1 || bt->size(0) != batch) Py_RETURN_NONE;
  if (sl->dim() != 1 || sl->scalar_type() != at::kInt || sl->size(0) != batch || !sl->is_contiguous()) Py_RETURN_NONE;
  if (max_len <= 0 || max_len > bt->size(1) * page) Py_RETURN_NONE;
  if (validating()) Py_RETURN_NONE;  // page ids are checked on the host first
  size_t need = 0;
  if (abi.workspace_bytes(int32_t(batch), int32_t(q_len), int32_t(heads), int32_t(ctas), &need) != MLA_FP4_OK || size_t(ws->numel()) < need)
    Py_RETURN_NONE;
  const at::ScalarType out_type =
      out_code == MLA_FP4_OUT_BF16 ? at::kBFloat16 : (out_code == MLA_FP4_OUT_F32 ? at::kFloat : at::kFloat8_e4m3fn);
  const int64_t shape[4] = {batch, q_len, heads, MLA_FP4_LATENT_DIM};
  const bool given = a[19] != Py_None;
  at::Tensor out;
  if (given) {
    const at::Tensor* o = tensor(a[19]);
    if (!o || !on(*o, dev) || o->scalar_type() != out_type || o->sizes() != at::IntArrayRef(shape, 4) || !o->is_contiguous()) Py_RETURN_NONE;
    out = *o;
  }
  const int want_lse = PyObject_IsTrue(a[21]);
  if (want_lse < 0) return nullptr;
  at::Tensor lse;
  const bool lse_given = want_lse && a[22] != Py_None;
  if (lse_given) {
    const at::Tensor* l = tensor(a[22]);
    if (!l || !on(*l, dev) || l->scalar_type() != at::kFloat || l->sizes() != at::IntArrayRef(shape, 3) || !l->is_contiguous()) Py_RETURN_NONE;
    lse = *l;
  }
  const at::Tensor* sink = a[10] == Py_None ? nullptr : tensor(a[10]);
  if (a[10] != Py_None && !sink) Py_RETURN_NONE;
  const int pdl = PyObject_IsTrue(a[7]);
  if (pdl < 0) return nullptr;

  c10::cuda::CUDAGuard guard(dev);
  MlaFp4DecodeArgs d = {};
  d.q = q->data_ptr();
  d.q_stride_batch = q->stride(0); d.q_stride_qpos = q->stride(1); d.q_stride_head = q->stride(2);
  d.kv_cache = kv->data_ptr();
  d.kv_cache_sf = static_cast<const float*>(sf->data_ptr());
  d.block_tables = static_cast<const int32_t*>(bt->data_ptr());
  d.block_table_stride = bt->stride(0);
  d.seq_lens = static_cast<const int32_t*>(sl->data_ptr());
  d.workspace = ws->data_ptr();
  d.workspace_bytes = size_t(ws->numel());
  d.status = static_cast<int32_t*>(status->data_ptr());
  d.batch = int32_t(batch); d.q_len = int32_t(q_len); d.num_heads = int32_t(heads); d.page_size = int32_t(page);
  d.num_pages = kv->size(0);
  d.softmax_scale = float(scale); d.output_scale = float(out_scale);
  d.out_dtype = int32_t(out_code); d.kernel = int32_t(kernel); d.num_ctas = int32_t(ctas);
  d.enable_pdl = pdl; d.phase_mask = int32_t(phase);
  d.stream = c10::cuda::getCurrentCUDAStream(dev.index()).stream();
  d.max_pages_per_request = int32_t(bt->size(1));
  d.max_seq_len = int32_t(max_len < INT32_MAX ? max_len : INT32_MAX);
  d.wait_polls = int32_t(polls);
  d.logits_soft_cap = float(cap);
  d.sink = sink ? static_cast<const float*>(sink->data_ptr()) : nullptr;
  int rc;
  {
    NoGil released;
    if (!given) out = at::empty(at::IntArrayRef(shape, 4), at::TensorOptions().dtype(out_type).device(dev));
    if (want_lse && !lse_given) lse = at::empty(at::IntArrayRef(shape, 3), at::TensorOptions().dtype(at::kFloat).device(dev));
    d.out = out.data_ptr();
    d.lse = want_lse ? static_cast<float*>(lse.data_ptr()) : nullptr;
    rc = abi.decode(&d);
  }
  if (rc != MLA_FP4_OK) return raise_status(rc);
  PyObject* po = given ? Py_NewRef(a[19]) : THPVariable_Wrap(std::move(out));
  if (!po || !want_lse) return po;
  PyObject* pl = lse_given ? Py_NewRef(a[22]) : THPVariable_Wrap(std::move(lse));
  if (!pl) {
    Py_DECREF(po);
    return nullptr;
  }
  PyObject* both = PyTuple_Pack(2, po, pl);
  Py_DECREF(po);
  Py_DECREF(pl);
  return both;
  END_HANDLE_TH_ERRORS
}

// write_tokens(latent, rope, slot_mapping, kv_cache, kv_cache_sf, token_scale) -> whether it was launched
PyObject* write_tokens(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 6) return PyErr_Format(PyExc_TypeError, "write_tokens takes 6 arguments");
  const at::Tensor *lat = tensor(a[0]), *rope = tensor(a[1]), *kv = tensor(a[3]), *sf = tensor(a[4]);
  const at::Tensor *slots = a[2] == Py_None ? nullptr : tensor(a[2]), *ts = a[5] == Py_None ? nullptr : tensor(a[5]);
  if (!lat || !rope || !kv || !sf || (a[2] != Py_None && !slots) || (a[5] != Py_None && !ts)) Py_RETURN_FALSE;
  const at::Device dev = lat->device();
  if (!lat->is_cuda() || !on(*rope, dev) || !on(*kv, dev) || !on(*sf, dev) || (slots && !on(*slots, dev)) || (ts && !on(*ts, dev)))
    Py_RETURN_FALSE;
  if (lat->dim() != 2 || rope->dim() != 2 || lat->size(1) != MLA_FP4_LATENT_DIM || rope->size(1) != MLA_FP4_ROPE_DIM ||
      lat->size(0) != rope->size(0) || lat->stride(1) != 1 || rope->stride(1) != 1 || lat->scalar_type() != rope->scalar_type())
    Py_RETURN_FALSE;
  int in_type;
  if (lat->scalar_type() == at::kBFloat16) in_type = MLA_FP4_IN_BF16;
  else if (lat->scalar_type() == at::kHalf) in_type = MLA_FP4_IN_F16;
  else if (lat->scalar_type() == at::kFloat) in_type = MLA_FP4_IN_F32;
  else Py_RETURN_FALSE;
  const int64_t tokens = lat->size(0);
  if (kv->dim() < 1 || kv->scalar_type() != at::kByte || kv->size(-1) != MLA_FP4_ROW_BYTES || !kv->is_contiguous()) Py_RETURN_FALSE;
  const int64_t num_slots = kv->numel() / MLA_FP4_ROW_BYTES;
  if (sf->scalar_type() != at::kFloat || !sf->is_contiguous() || sf->numel() != num_slots) Py_RETURN_FALSE;
  if (slots && (slots->scalar_type() != at::kLong || slots->numel() != tokens || !slots->is_contiguous())) Py_RETURN_FALSE;
  if (ts && (ts->scalar_type() != at::kFloat || ts->numel() != tokens || !ts->is_contiguous())) Py_RETURN_FALSE;
  c10::cuda::CUDAGuard guard(dev);
  const void *lat_p = lat->data_ptr(), *rope_p = rope->data_ptr();
  const int64_t lat_stride = lat->stride(0), rope_stride = rope->stride(0);
  const float* ts_p = ts ? static_cast<const float*>(ts->data_ptr()) : nullptr;
  const int64_t* slots_p = slots ? static_cast<const int64_t*>(slots->data_ptr()) : nullptr;
  void* kv_p = kv->data_ptr();
  float* sf_p = static_cast<float*>(sf->data_ptr());
  cudaStream_t stream = c10::cuda::getCurrentCUDAStream(dev.index()).stream();
  int rc;
  {
    NoGil released;
    rc = abi.cache_write(lat_p, lat_stride, rope_p, rope_stride, in_type, ts_p, slots_p, tokens, kv_p, sf_p, num_slots, stream);
  }
  if (rc != MLA_FP4_OK) return raise_status(rc);
  Py_RETURN_TRUE;
  END_HANDLE_TH_ERRORS
}

// Where the GPU reads a tensor: its device memory, or pinned host memory through its device address; null when it cannot
// (pageable memory).
const void* readable(const at::Tensor& t, const at::Device& dev) {
  if (t.is_cuda()) return t.device() == dev ? t.data_ptr() : nullptr;
  if (!t.is_cpu()) return nullptr;
  cudaPointerAttributes at;
  if (cudaPointerGetAttributes(&at, t.data_ptr()) != cudaSuccess) {
    (void)cudaGetLastError();
    return nullptr;
  }
  return at.type == cudaMemoryTypeHost ? at.devicePointer : nullptr;
}

// Whether the memory that a tensor at p spans meets that of another (neither is empty).
size_t span(const at::Tensor& t) {
  int64_t elements = 1;
  for (int64_t d = 0; d < t.dim(); ++d) elements += (t.size(d) - 1) * t.stride(d);
  return size_t(elements) * t.element_size();
}
bool meets(const void* p, const at::Tensor& t, const at::Tensor& buffer) {
  const auto a = reinterpret_cast<uintptr_t>(p), b = reinterpret_cast<uintptr_t>(buffer.data_ptr());
  return a < b + span(buffer) && b < a + span(t);
}

// step_metadata(block_tables, seq_lens, slot_mapping, dst_block_tables, dst_seq_lens, dst_slot_mapping, page_size, q_len)
// -> whether it was launched
PyObject* step_metadata(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 8) return PyErr_Format(PyExc_TypeError, "step_metadata takes 8 arguments");
  const at::Tensor *bt = tensor(a[0]), *sl = tensor(a[1]), *dbt = tensor(a[3]), *dsl = tensor(a[4]), *dsm = tensor(a[5]);
  const at::Tensor* sm = a[2] == Py_None ? nullptr : tensor(a[2]);
  int64_t page, q_len;
  if (!bt || !sl || !dbt || !dsl || !dsm || (a[2] != Py_None && !sm) || !integer(a[6], &page) || !integer(a[7], &q_len)) Py_RETURN_FALSE;
  if (bt->dim() != 2 || bt->scalar_type() != at::kInt || bt->stride(1) != 1 || sl->dim() != 1 || sl->stride(0) != 1 ||
      (sl->scalar_type() != at::kInt && sl->scalar_type() != at::kLong) || bt->numel() == 0)
    Py_RETURN_FALSE;
  if (sm && (sm->scalar_type() != at::kLong || !sm->is_contiguous())) Py_RETURN_FALSE;
  if (!dsl->is_cuda()) Py_RETURN_FALSE;
  const at::Device dev = dsl->device();
  // The buffers are public attributes of the backend: what is not of the form it made them in is the general path's.
  if (!on(*dbt, dev) || dbt->dim() != 2 || dbt->scalar_type() != at::kInt || dbt->stride(1) != 1 || dbt->size(0) < bt->size(0) ||
      dbt->size(1) < bt->size(1) || (dbt->size(0) > 1 && dbt->stride(0) < dbt->size(1)) || dsl->dim() != 1 || dsl->scalar_type() != at::kInt ||
      !dsl->is_contiguous() || dsl->size(0) < sl->size(0) || bt->size(0) != sl->size(0) || !on(*dsm, dev) || dsm->scalar_type() != at::kLong ||
      !dsm->is_contiguous() || q_len <= 0 || dsm->numel() != dsl->size(0) * q_len || (sm && sm->numel() != bt->size(0) * q_len))
    Py_RETURN_FALSE;
  c10::cuda::CUDAGuard guard(dev);
  const void *pbt = readable(*bt, dev), *psl = readable(*sl, dev), *psm = sm ? readable(*sm, dev) : nullptr;
  if (!pbt || !psl || (sm && !psm)) Py_RETURN_FALSE;
  // Sources inside the buffers (a backend's own rows, moved up, say) are the general path's: one kernel would read what it writes.
  if (sl->numel() == 0 || (sm && sm->numel() == 0)) Py_RETURN_FALSE;
  for (const at::Tensor* dst : {dbt, dsl, dsm})
    if (meets(pbt, *bt, *dst) || meets(psl, *sl, *dst) || (sm && meets(psm, *sm, *dst))) Py_RETURN_FALSE;
  const c10::cuda::CUDAStream stream = c10::cuda::getCurrentCUDAStream(dev.index());
  const int64_t bt_stride = bt->stride(0), dbt_stride = dbt->stride(0);
  const int32_t width = int32_t(bt->size(1)), batch = int32_t(bt->size(0)), max_batch = int32_t(dsl->size(0)), wide = sl->scalar_type() == at::kLong ? 1 : 0;
  int32_t *dbt_p = static_cast<int32_t*>(dbt->data_ptr()), *dsl_p = static_cast<int32_t*>(dsl->data_ptr());
  int64_t* dsm_p = static_cast<int64_t*>(dsm->data_ptr());
  at::Tensor pinned[3];  // kept while they are handed to the allocator
  int n_pinned = 0;
  for (const at::Tensor* t : {bt, sl, sm})
    if (t && !t->is_cuda()) pinned[n_pinned++] = *t;
  int rc;
  {
    NoGil released;
    rc = abi.step_metadata(static_cast<const int32_t*>(pbt), bt_stride, width, psl, wide, static_cast<const int64_t*>(psm), batch, int32_t(page),
                           int32_t(q_len), dbt_p, dbt_stride, dsl_p, dsm_p, max_batch, stream.stream());
    if (rc == MLA_FP4_OK)
      for (int i = 0; i < n_pinned; ++i)  // pinned memory that the caller lets go now is not handed out again before the kernel has read it
        at::getHostAllocator(at::kCUDA)->record_event(pinned[i].data_ptr(), pinned[i].storage().data_ptr().get_context(), stream);
  }
  if (rc != MLA_FP4_OK) return raise_status(rc);
  Py_RETURN_TRUE;
  END_HANDLE_TH_ERRORS
}

// ---------------------------------------------------------------- sparse decode and the page pool
// A contiguous tensor of that type, those extents (-1: any) and that device.
bool plain(const at::Tensor& t, at::ScalarType type, at::IntArrayRef shape, const at::Device& dev) {
  if (!on(t, dev) || t.scalar_type() != type || size_t(t.dim()) != shape.size() || !t.is_contiguous()) return false;
  for (size_t i = 0; i < shape.size(); ++i)
    if (shape[i] >= 0 && t.size(int64_t(i)) != shape[i]) return false;
  return true;
}
bool cache_ok(const at::Tensor& kv, const at::Tensor& sf) {
  return kv.is_cuda() && kv.dim() == 3 && kv.scalar_type() == at::kByte && kv.size(2) == MLA_FP4_ROW_BYTES && kv.is_contiguous() &&
         plain(sf, at::kFloat, {kv.size(0), kv.size(1), 1}, kv.device());
}
bool summary_ok(const at::Tensor& summary, const at::Tensor& sf, int64_t pages, const at::Device& dev) {
  return plain(summary, at::kChar, {pages, MLA_FP4_LATENT_DIM + MLA_FP4_ROPE_DIM}, dev) && plain(sf, at::kFloat, {summary.size(0)}, dev);
}
bool tables_ok(const at::Tensor& bt, const at::Tensor& sl, const at::Device& dev) {
  return on(bt, dev) && bt.dim() == 2 && bt.scalar_type() == at::kInt && bt.size(1) > 0 && bt.stride(1) == 1 && bt.stride(0) >= 0 &&
         bt.size(1) <= INT32_MAX && plain(sl, at::kInt, {bt.size(0)}, dev);
}
bool query_ok(const at::Tensor& q) {
  return q.is_cuda() && q.dim() == 4 && q.scalar_type() == at::kFloat8_e4m3fn && q.size(3) == MLA_FP4_LATENT_DIM + MLA_FP4_ROPE_DIM && q.stride(3) == 1 &&
         q.size(0) > 0 && q.size(1) > 0 && q.size(2) > 0 && q.size(2) <= 128;
}
// A tensor on the current device for results that a kernel writes in full, and memory for a call's own use: at::empty without its dispatch, of which
// three in a call were a fifth of its time on the host.
at::Tensor room(at::IntArrayRef shape, at::ScalarType type, const at::Device& dev) { return at::Tensor(at::detail::empty_cuda(shape, type, dev, std::nullopt)); }
c10::DataPtr scratch(size_t bytes) { return c10::cuda::CUDACachingAllocator::get()->allocate(bytes); }

// summarize(kv_cache, kv_cache_sf, summary, summary_sf, page_ids, block_tables, seq_lens, new_tokens, status or None) -> whether it was launched; page_ids, or
// the other three
PyObject* summarize(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 9) return PyErr_Format(PyExc_TypeError, "summarize takes 9 arguments");
  const at::Tensor *kv = tensor(a[0]), *sf = tensor(a[1]), *su = tensor(a[2]), *ssf = tensor(a[3]);
  if (!kv || !sf || !su || !ssf || !cache_ok(*kv, *sf)) Py_RETURN_FALSE;
  const at::Device dev = kv->device();
  const int64_t pages = kv->size(0), page = kv->size(1);
  if (!summary_ok(*su, *ssf, pages, dev)) Py_RETURN_FALSE;
  const bool by_id = a[4] != Py_None;
  const at::Tensor *ids = nullptr, *bt = nullptr, *sl = nullptr;
  int64_t fresh = 0;
  if (by_id) {
    ids = tensor(a[4]);
    if (!ids || !plain(*ids, at::kInt, {-1}, dev)) Py_RETURN_FALSE;
  } else {
    bt = tensor(a[5]);
    sl = tensor(a[6]);
    if (!bt || !sl || !integer(a[7], &fresh) || fresh < 0 || fresh > INT32_MAX || !tables_ok(*bt, *sl, dev)) Py_RETURN_FALSE;
  }
  const at::Tensor* st = a[8] == Py_None ? nullptr : tensor(a[8]);
  if (a[8] != Py_None && (!st || !plain(*st, at::kInt, {8}, dev))) Py_RETURN_FALSE;
  int32_t* status = st ? static_cast<int32_t*>(st->data_ptr()) : nullptr;
  c10::cuda::CUDAGuard guard(dev);
  const void* kv_p = kv->data_ptr();
  const float* sf_p = static_cast<const float*>(sf->data_ptr());
  void* su_p = su->data_ptr();
  float* ssf_p = static_cast<float*>(ssf->data_ptr());
  cudaStream_t stream = c10::cuda::getCurrentCUDAStream(dev.index()).stream();
  int rc;
  {
    NoGil released;
    rc = by_id ? abi.summarize_pages(kv_p, sf_p, pages, int32_t(page), static_cast<const int32_t*>(ids->data_ptr()), ids->numel(), su_p, ssf_p, status, stream)
               : abi.summarize_new_pages(kv_p, sf_p, pages, int32_t(page), static_cast<const int32_t*>(bt->data_ptr()), bt->stride(0), int32_t(bt->size(1)),
                                         static_cast<const int32_t*>(sl->data_ptr()), int32_t(bt->size(0)), int32_t(fresh), su_p, ssf_p, status, stream);
  }
  if (rc != MLA_FP4_OK) return raise_status(rc);
  Py_RETURN_TRUE;
  END_HANDLE_TH_ERRORS
}

struct Budget {
  int64_t budget, sink, local;
  int causal;
  // from four Python values; false: not of the common form
  bool from(PyObject* const* a) {
    causal = PyObject_IsTrue(a[3]);
    if (causal < 0) PyErr_Clear();  // (the Python path says what is wrong with it)
    return integer(a[0], &budget) && integer(a[1], &sink) && integer(a[2], &local) && causal >= 0 && sink >= 0 && local >= 1 && sink <= INT32_MAX &&
           local <= INT32_MAX && budget <= INT32_MAX && sink + local <= budget;
  }
};
// What both entry points fill in alike.
MlaFp4SelectArgs select_args(const at::Tensor& q, const at::Tensor& su, const at::Tensor& ssf, const at::Tensor& bt, const at::Tensor& sl, int64_t page,
                             const Budget& b) {
  MlaFp4SelectArgs s = {};
  s.q = q.data_ptr();
  s.q_stride_batch = q.stride(0); s.q_stride_qpos = q.stride(1); s.q_stride_head = q.stride(2);
  s.summary = su.data_ptr();
  s.summary_sf = static_cast<const float*>(ssf.data_ptr());
  s.num_pages = su.size(0);
  s.block_tables = static_cast<const int32_t*>(bt.data_ptr());
  s.block_table_stride = bt.stride(0);
  s.seq_lens = static_cast<const int32_t*>(sl.data_ptr());
  s.batch = int32_t(q.size(0)); s.q_len = int32_t(q.size(1)); s.num_heads = int32_t(q.size(2)); s.page_size = int32_t(page);
  s.width = int32_t(bt.size(1));
  s.budget = int32_t(b.budget); s.sink_pages = int32_t(b.sink); s.local_pages = int32_t(b.local); s.causal = b.causal;
  return s;
}

// select(q, summary, summary_sf, block_tables, seq_lens, page_size, budget, sink_pages, local_pages, causal, selected, selected_lens, workspace, status)
// -> (selected, selected_lens), or None when the call is not of the common form
PyObject* select(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 14) return PyErr_Format(PyExc_TypeError, "select takes 14 arguments");
  const at::Tensor *q = tensor(a[0]), *su = tensor(a[1]), *ssf = tensor(a[2]), *bt = tensor(a[3]), *sl = tensor(a[4]);
  int64_t page;
  Budget b;
  if (!q || !su || !ssf || !bt || !sl || !integer(a[5], &page) || !b.from(a + 6) || !query_ok(*q)) Py_RETURN_NONE;
  const at::Device dev = q->device();
  if (!summary_ok(*su, *ssf, -1, dev) || !tables_ok(*bt, *sl, dev) || bt->size(0) != q->size(0)) Py_RETURN_NONE;
  const int64_t rows = q->size(0) * q->size(1), width = bt->size(1);
  at::Tensor out[3];  // the table, the lengths, the workspace
  for (int i = 0; i < 3; ++i) {
    if (a[10 + i] == Py_None) continue;
    const at::Tensor* t = tensor(a[10 + i]);
    if (!t) Py_RETURN_NONE;
    out[i] = *t;
  }
  const at::Tensor* st = a[13] == Py_None ? nullptr : tensor(a[13]);
  if (a[13] != Py_None && (!st || !plain(*st, at::kInt, {8}, dev))) Py_RETURN_NONE;
  size_t need = 0;
  if (q->size(0) > INT32_MAX || q->size(1) > INT32_MAX || page < 0 || page > 128 ||
      abi.select_workspace_bytes(int32_t(q->size(0)), int32_t(q->size(1)), int32_t(width), &need) != MLA_FP4_OK)
    Py_RETURN_NONE;
  if (width <= b.budget) need = 0;
  if ((out[0].defined() && !plain(out[0], at::kInt, {rows, b.budget}, dev)) || (out[1].defined() && !plain(out[1], at::kInt, {rows}, dev)) ||
      (out[2].defined() && (!plain(out[2], at::kChar, {-1}, dev) || size_t(out[2].numel()) < need)))
    Py_RETURN_NONE;
  c10::cuda::CUDAGuard guard(dev);
  MlaFp4SelectArgs s = select_args(*q, *su, *ssf, *bt, *sl, page, b);
  s.status = st ? static_cast<int32_t*>(st->data_ptr()) : nullptr;
  s.stream = c10::cuda::getCurrentCUDAStream(dev.index()).stream();
  int rc;
  {
    NoGil released;
    if (!out[0].defined()) out[0] = room({rows, b.budget}, at::kInt, dev);
    if (!out[1].defined()) out[1] = room({rows}, at::kInt, dev);
    s.selected = static_cast<int32_t*>(out[0].data_ptr());
    s.selected_lens = static_cast<int32_t*>(out[1].data_ptr());
    c10::DataPtr own;
    if (!out[2].defined() && need > 0) own = scratch(need);
    s.workspace = out[2].defined() ? out[2].data_ptr() : own.get();
    s.workspace_bytes = out[2].defined() ? size_t(out[2].numel()) : need;
    rc = abi.select_pages(&s);
  }
  if (rc != MLA_FP4_OK) return raise_status(rc);
  PyObject* r[2];
  for (int i = 0; i < 2; ++i) r[i] = a[10 + i] != Py_None ? Py_NewRef(a[10 + i]) : THPVariable_Wrap(std::move(out[i]));
  PyObject* both = r[0] && r[1] ? PyTuple_Pack(2, r[0], r[1]) : nullptr;
  Py_XDECREF(r[0]);
  Py_XDECREF(r[1]);
  return both;
  END_HANDLE_TH_ERRORS
}

// sparse_decode(workspace, status, num_heads, page_size, out_code, num_ctas, pdl, soft_cap, sink, wait_polls, budget, sink_pages, local_pages, causal,
//               q, kv_cache, block_tables, seq_lens, max_seq_len, softmax_scale, output_scale, out, kv_cache_sf, summary, summary_sf,
//               return_lse, lse_out)
// -> out, (out, lse), or None when the call is not of the common form.  The workspace: the decode step's, then from the next multiple of 256 on the
// selected table and lengths, then from the next one the scores.
PyObject* sparse_decode(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 27) return PyErr_Format(PyExc_TypeError, "sparse_decode takes 27 arguments");
  const at::Tensor *ws = tensor(a[0]), *status = tensor(a[1]), *q = tensor(a[14]), *kv = tensor(a[15]), *bt = tensor(a[16]), *sl = tensor(a[17]),
                   *sf = tensor(a[22]), *su = tensor(a[23]), *ssf = tensor(a[24]);
  int64_t heads, page, out_code, ctas, polls, max_len;
  double cap, scale, out_scale;
  Budget b;
  if (!ws || !status || !q || !kv || !bt || !sl || !sf || !su || !ssf || !integer(a[2], &heads) || !integer(a[3], &page) || !integer(a[4], &out_code) ||
      !integer(a[5], &ctas) || !number(a[7], &cap) || !integer(a[9], &polls) || !b.from(a + 10) || !integer(a[18], &max_len) || !number(a[19], &scale) ||
      !number(a[20], &out_scale) || !query_ok(*q) || !cache_ok(*kv, *sf) || validating())
    Py_RETURN_NONE;
  const at::Device dev = ws->device();
  if (q->device() != dev || kv->device() != dev || !on(*status, dev) || q->size(2) != heads || kv->size(1) != page || !summary_ok(*su, *ssf, kv->size(0), dev) ||
      !tables_ok(*bt, *sl, dev) || bt->size(0) != q->size(0))
    Py_RETURN_NONE;
  const int64_t batch = q->size(0), q_len = q->size(1), rows = batch * q_len, width = bt->size(1);
  if (rows > INT32_MAX || (q_len > 1 && batch > 1 && q->stride(0) != q_len * q->stride(1)) || max_len <= 0 || max_len > width * page) Py_RETURN_NONE;
  const auto aligned = [](size_t v) { return (v + 255) / 256 * 256; };
  size_t need = 0, scores = 0;
  if (abi.workspace_bytes(int32_t(rows), 1, int32_t(heads), int32_t(ctas), &need) != MLA_FP4_OK ||
      abi.select_workspace_bytes(int32_t(rows), 1, int32_t(width), &scores) != MLA_FP4_OK)
    Py_RETURN_NONE;
  const size_t table_at = aligned(need), lens_at = table_at + size_t(rows) * size_t(b.budget) * 4, scores_at = table_at + aligned(size_t(rows) * (size_t(b.budget) + 1) * 4);
  if (size_t(ws->numel()) < scores_at + (width > b.budget ? scores : 0)) Py_RETURN_NONE;
  const at::ScalarType out_type =
      out_code == MLA_FP4_OUT_BF16 ? at::kBFloat16 : (out_code == MLA_FP4_OUT_F32 ? at::kFloat : at::kFloat8_e4m3fn);
  const int64_t shape[4] = {batch, q_len, heads, MLA_FP4_LATENT_DIM};
  const bool given = a[21] != Py_None;
  at::Tensor out, lse;
  if (given) {
    const at::Tensor* o = tensor(a[21]);
    if (!o || !plain(*o, out_type, at::IntArrayRef(shape, 4), dev)) Py_RETURN_NONE;
    out = *o;
  }
  const int want_lse = PyObject_IsTrue(a[25]), pdl = PyObject_IsTrue(a[6]);
  if (want_lse < 0 || pdl < 0) return nullptr;
  const bool lse_given = want_lse && a[26] != Py_None;
  if (lse_given) {
    const at::Tensor* l = tensor(a[26]);
    if (!l || !plain(*l, at::kFloat, at::IntArrayRef(shape, 3), dev)) Py_RETURN_NONE;
    lse = *l;
  }
  const at::Tensor* sink = a[8] == Py_None ? nullptr : tensor(a[8]);
  if (a[8] != Py_None && !sink) Py_RETURN_NONE;

  c10::cuda::CUDAGuard guard(dev);
  char* base = static_cast<char*>(ws->data_ptr());
  MlaFp4SelectArgs s = select_args(*q, *su, *ssf, *bt, *sl, page, b);
  s.selected = reinterpret_cast<int32_t*>(base + table_at);
  s.selected_lens = reinterpret_cast<int32_t*>(base + lens_at);
  s.workspace = base + scores_at;
  s.workspace_bytes = size_t(ws->numel()) - scores_at;
  s.status = static_cast<int32_t*>(status->data_ptr());
  s.wait_polls = int32_t(polls);
  s.stream = c10::cuda::getCurrentCUDAStream(dev.index()).stream();
  MlaFp4DecodeArgs d = {};
  d.q = s.q;
  d.q_stride_batch = q_len == 1 ? s.q_stride_batch : s.q_stride_qpos;
  d.q_stride_qpos = 16;  // (one position a row: not looked at)
  d.q_stride_head = s.q_stride_head;
  d.kv_cache = kv->data_ptr();
  d.kv_cache_sf = static_cast<const float*>(sf->data_ptr());
  d.block_tables = s.selected;
  d.block_table_stride = b.budget;
  d.seq_lens = s.selected_lens;
  d.workspace = base;
  d.workspace_bytes = table_at;
  d.status = s.status;
  d.batch = int32_t(rows); d.q_len = 1; d.num_heads = int32_t(heads); d.page_size = int32_t(page);
  d.num_pages = kv->size(0);
  d.softmax_scale = float(scale); d.output_scale = float(out_scale);
  d.out_dtype = int32_t(out_code);
  d.num_ctas = int32_t(ctas);
  d.enable_pdl = pdl;
  d.stream = s.stream;
  d.max_pages_per_request = s.budget;
  const int64_t longest = std::min(max_len, b.budget * page);
  d.max_seq_len = int32_t(std::min<int64_t>(longest, INT32_MAX));
  d.wait_polls = int32_t(polls);
  d.logits_soft_cap = float(cap);
  d.sink = sink ? static_cast<const float*>(sink->data_ptr()) : nullptr;
  int rc;
  {
    NoGil released;
    if (!given) out = room(at::IntArrayRef(shape, 4), out_type, dev);
    if (want_lse && !lse_given) lse = room(at::IntArrayRef(shape, 3), at::kFloat, dev);
    d.out = out.data_ptr();
    d.lse = want_lse ? static_cast<float*>(lse.data_ptr()) : nullptr;
    rc = abi.select_pages(&s);
    if (rc == MLA_FP4_OK) rc = abi.decode(&d);
  }
  if (rc != MLA_FP4_OK) return raise_status(rc);
  PyObject* po = given ? Py_NewRef(a[21]) : THPVariable_Wrap(std::move(out));
  if (!po || !want_lse) return po;
  PyObject* pl = lse_given ? Py_NewRef(a[26]) : THPVariable_Wrap(std::move(lse));
  PyObject* both = pl ? PyTuple_Pack(2, po, pl) : nullptr;
  Py_DECREF(po);
  Py_XDECREF(pl);
  return both;
  END_HANDLE_TH_ERRORS
}

// pool(what, layers, num_layers, page_size, num_pages, refcounts, status, block_tables, seq_lens, x, y): what is 0 allocate (x: new_lens), 1 fork (parents,
// children), 2 free (x: rows), 3 compact (x: remap or None); layers is the address of the host array -> remap of a compaction, else True; None
// when the call is not of the common form
PyObject* pool(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 11) return PyErr_Format(PyExc_TypeError, "pool takes 11 arguments");
  int64_t what, layers, page, pages;
  const at::Tensor *ref = tensor(a[5]), *status = tensor(a[6]), *bt = tensor(a[7]), *sl = tensor(a[8]), *x = tensor(a[9]), *y = tensor(a[10]);
  if (!integer(a[0], &what) || !integer(a[2], &layers) || !integer(a[3], &page) || !integer(a[4], &pages) || !ref || !status || !bt || !sl) Py_RETURN_NONE;
  const void* array = PyLong_AsVoidPtr(a[1]);
  if (!array) return PyErr_Occurred() ? nullptr : PyErr_Format(PyExc_ValueError, "null address");
  const at::Device dev = status->device();
  const int64_t rows = bt->size(0);
  if (!plain(*ref, at::kInt, {pages}, dev) || !tables_ok(*bt, *sl, dev) || rows == 0 || rows > INT32_MAX || (rows > 1 && bt->stride(0) < bt->size(1))) Py_RETURN_NONE;
  int64_t count = 0;
  if (what == 0) {
    if (!x || !plain(*x, at::kInt, {rows}, dev)) Py_RETURN_NONE;
  } else if (what == 1 || what == 2) {
    if (!x || !plain(*x, at::kInt, {-1}, dev) || x->numel() == 0 || x->numel() > INT32_MAX) Py_RETURN_NONE;
    count = x->numel();
    if (what == 1 && (!y || !plain(*y, at::kInt, {count}, dev))) Py_RETURN_NONE;
  } else if (a[9] != Py_None && (!x || !plain(*x, at::kInt, {pages}, dev))) {
    Py_RETURN_NONE;
  }
  size_t need = 0;
  if (abi.pool_workspace_bytes(pages, int32_t(rows), int32_t(count), &need) != MLA_FP4_OK) Py_RETURN_NONE;
  c10::cuda::CUDAGuard guard(dev);
  MlaFp4PoolArgs p = {};
  p.layers = static_cast<const MlaFp4PageLayer*>(array);
  p.num_layers = int32_t(layers); p.page_size = int32_t(page);
  p.num_pages = pages;
  p.refcounts = static_cast<int32_t*>(ref->data_ptr());
  p.block_tables = static_cast<int32_t*>(bt->data_ptr());
  p.block_table_stride = bt->stride(0);
  p.width = int32_t(bt->size(1)); p.rows = int32_t(rows);
  p.seq_lens = static_cast<int32_t*>(sl->data_ptr());
  p.workspace_bytes = need;
  p.status = static_cast<int32_t*>(status->data_ptr());
  p.stream = c10::cuda::getCurrentCUDAStream(dev.index()).stream();
  const int32_t *xp = x ? static_cast<const int32_t*>(x->data_ptr()) : nullptr, *yp = y ? static_cast<const int32_t*>(y->data_ptr()) : nullptr;
  at::Tensor remap;
  int rc;
  {
    NoGil released;
    const c10::DataPtr own = scratch(need);
    p.workspace = own.get();
    if (what == 0) rc = abi.pool_allocate(&p, xp);
    else if (what == 1) rc = abi.pool_fork(&p, xp, yp, int32_t(count));
    else if (what == 2) rc = abi.pool_free(&p, xp, int32_t(count));
    else {
      remap = x ? *x : room({pages}, at::kInt, dev);
      rc = abi.pool_compact(&p, static_cast<int32_t*>(remap.data_ptr()));
    }
  }
  if (rc != MLA_FP4_OK) return raise_status(rc);
  if (what != 3) Py_RETURN_TRUE;
  return x ? Py_NewRef(a[9]) : THPVariable_Wrap(std::move(remap));
  END_HANDLE_TH_ERRORS
}

PyMethodDef methods[] = {
    {"bind", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(bind)), METH_FASTCALL, nullptr},
    {"bind_sparse", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(bind_sparse)), METH_FASTCALL, nullptr},
    {"decode", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(decode)), METH_FASTCALL, nullptr},
    {"write_tokens", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(write_tokens)), METH_FASTCALL, nullptr},
    {"step_metadata", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(step_metadata)), METH_FASTCALL, nullptr},
    {"summarize", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(summarize)), METH_FASTCALL, nullptr},
    {"select", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(select)), METH_FASTCALL, nullptr},
    {"sparse_decode", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(sparse_decode)), METH_FASTCALL, nullptr},
    {"pool", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(pool)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_native", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__native() { return PyModule_Create(&module); }
