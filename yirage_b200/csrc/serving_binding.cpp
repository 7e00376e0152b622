// Python binding of the serving operators' hot calls (serving.py).
//
// The rest of the C ABI is bound with ctypes.  These calls are made once per layer and token on
// single tokens, where the kernels take 3 to 10 us: checking six tensors and filling the operand
// structs from Python took 15 to 21 us a call, the same work here 4 to 8.  Every check that the
// C ABI cannot make (types, shapes, devices of tensors) is made here, before anything is
// allocated or enqueued; what the ABI refuses comes back as YpkError.
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/core/grad_mode.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/core/AutogradState.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <math.h>
#include <stdarg.h>

#include <algorithm>

#include "../../include/ypk.h"
#include "strided_rows.h"

namespace {

using at::Tensor;

[[noreturn]] void refuse(PyObject *type, const char *fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  PyErr_FormatV(type, fmt, ap);
  va_end(ap);
  throw python_error();
}

// A failed call of the C ABI, as yirage_b200._native.YpkError(code, message).
[[noreturn]] void refuse_abi(int code) {
  const char *text = ypk_last_error(nullptr);
  PyObject *module = PyImport_ImportModule("yirage_b200._native");
  if (!module) throw python_error();
  PyObject *type = PyObject_GetAttrString(module, "YpkError");
  Py_DECREF(module);
  if (!type) throw python_error();
  PyObject *args = Py_BuildValue("(is)", code, text ? text : "");
  if (args) PyErr_SetObject(type, args);
  Py_XDECREF(args);
  Py_DECREF(type);
  throw python_error();
}

template <class F>
void call_abi(F f) {
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = f();
  Py_END_ALLOW_THREADS
  if (rc != YPK_OK) refuse_abi(rc);
}

const Tensor &tensor(PyObject *o, const char *name) {
  if (!THPVariable_Check(o)) refuse(PyExc_TypeError, "%s must be a tensor, not %s", name, Py_TYPE(o)->tp_name);
  const Tensor &t = THPVariable_Unpack(o);
  if (t.requires_grad() && at::GradMode::is_enabled())
    refuse(PyExc_ValueError, "%s requires a gradient; the serving operators have none (torch.no_grad or detach)", name);
  if (t._fw_grad(/*level=*/0).defined() && c10::AutogradState::get_tls_state().get_fw_grad_mode())
    refuse(PyExc_ValueError, "%s carries a forward-mode tangent; the serving operators have none (detach)", name);
  return t;
}

// A call has written t: what autograd saved of it for a backward pass is no longer there.
void written(const Tensor &t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

const char *type_name(at::ScalarType t) {
  switch (t) {
    case at::kBFloat16: return "torch.bfloat16";
    case at::kHalf: return "torch.float16";
    case at::kFloat: return "torch.float32";
    case at::kDouble: return "torch.float64";
    case at::kInt: return "torch.int32";
    case at::kLong: return "torch.int64";
    default: return c10::toString(t);
  }
}

int abi_type(at::ScalarType t) { return t == at::kBFloat16 ? YPK_BF16 : t == at::kHalf ? YPK_F16 : YPK_F32; }

// The cache of a call: the description that PagedKVCache keeps, and where its tensors are.
struct Cache {
  const ypk_paged_cache *c;
  c10::Device device;
  at::ScalarType dtype;
  int64_t heads, dim;
  const Tensor *keys, *values;
};

int64_t integer(PyObject *o) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw python_error();
  return v;
}

// arg[0]: address of the description; arg[1]: CUDA device of the cache, -1 for the CPU; arg[2], arg[3]:
// its two tensors.
Cache cache_of(PyObject *const *arg) {
  Cache k{reinterpret_cast<const ypk_paged_cache *>(integer(arg[0])), c10::Device(c10::kCPU), at::kBFloat16, 0, 0,
          &tensor(arg[2], "k_cache"), &tensor(arg[3], "v_cache")};
  // (data_ptr of a tensor whose storage was resized or exchanged: the description points elsewhere)
  if (k.keys->const_data_ptr() != k.c->k || k.values->const_data_ptr() != k.c->v)
    refuse(PyExc_ValueError, "k_cache or v_cache is not where it was when PagedKVCache was made");
  const int64_t i = integer(arg[1]);
  if (i >= 0) k.device = c10::Device(c10::kCUDA, static_cast<c10::DeviceIndex>(i));
  if (k.c->dtype == YPK_F16) k.dtype = at::kHalf;
  k.heads = k.c->num_kv_heads;
  k.dim = k.c->head_dim;
  return k;
}

void need_cuda(const c10::Device &d) {
  if (!d.is_cuda())
    refuse(PyExc_RuntimeError, "the serving operators need tensors on a CUDA device (sm_100a); there is no CPU "
                               "execution path");
}

void operand(const Cache &k, const Tensor &t, const char *name) {
  if (t.scalar_type() != k.dtype)
    refuse(PyExc_TypeError, "%s is %s, the cache %s", name, type_name(t.scalar_type()), type_name(k.dtype));
  if (t.device() != k.device)
    refuse(PyExc_ValueError, "%s is on %s, the cache on %s", name, t.device().str().c_str(), k.device.str().c_str());
}

struct Queries {
  int64_t rows, heads, token, group, head;     // strides in elements, 0 over a single entry
};

// [rows, heads, dim] or [rows, kv_heads, group, dim].
Queries queries(const Cache &k, const Tensor &t, const char *name, bool written) {
  operand(k, t, name);
  Queries q{};
  int64_t group = 0, st = 0, sg = 0, sh = 0, last = 0, dim = 0;
  bool good = false;
  if (t.dim() == 3) {
    q.heads = t.size(1);
    good = q.heads > 0 && q.heads % k.heads == 0;
    group = q.heads / k.heads;
    st = t.stride(0), sh = t.stride(1), sg = sh * group;
    dim = t.size(2), last = t.stride(2);
  } else if (t.dim() == 4) {
    group = t.size(2);
    q.heads = k.heads * group;
    good = t.size(1) == k.heads && group > 0;
    st = t.stride(0), sg = t.stride(1), sh = t.stride(2);
    dim = t.size(3), last = t.stride(3);
  }
  if (!good || dim != k.dim || last != 1)
    refuse(PyExc_ValueError, "%s must be [rows, heads, %lld] or [rows, %lld, group, %lld] with heads a multiple of %lld "
                             "and a contiguous last dimension",
           name, (long long)k.dim, (long long)k.heads, (long long)k.dim, (long long)k.heads);
  q.rows = t.size(0);
  if (q.rows > 0x7fffffff || q.heads > 0x7fffffff) refuse(PyExc_ValueError, "%s is too large", name);
  if (written && !ypk::rows_distinct({0, k.dim, {st, sg, sh}, {q.rows, k.heads, group}}))
    refuse(PyExc_ValueError, "%s is written: its rows must not overlap", name);
  q.token = q.rows > 1 ? st : 0;
  q.group = k.heads > 1 ? sg : 0;
  q.head = group > 1 ? sh : 0;
  return q;
}

void kv_rows(const Cache &k, const Tensor &t, const char *name, int64_t *token, int64_t *head) {
  operand(k, t, name);
  if (t.dim() != 3 || t.size(1) != k.heads || t.size(2) != k.dim || t.stride(2) != 1 || t.size(0) > 0x7fffffff)
    refuse(PyExc_ValueError, "%s must be [tokens, %lld, %lld] with a contiguous last dimension", name,
           (long long)k.heads, (long long)k.dim);
  *token = t.size(0) > 1 ? t.stride(0) : 0;
  *head = k.heads > 1 ? t.stride(1) : 0;
}

bool given(PyObject *o) { return o != Py_None; }

// paged_append(cache, device, k_cache, v_cache, k, v, q, q_out, cos, sin, q_norm, k_norm, eps) -> q_out or None
PyObject *paged_append(PyObject *, PyObject *const *arg, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 13) refuse(PyExc_TypeError, "paged_append takes 13 arguments");
  const Cache k = cache_of(arg);
  PyObject *out_obj = arg[7];
  if (!k.c->qo_indptr) refuse(PyExc_ValueError, "append needs the meta tensor 'qo_indptr_buffer'");
  ypk_paged_append_args a = {};
  const Tensor &kt = tensor(arg[4], "k"), &vt = tensor(arg[5], "v");
  kv_rows(k, kt, "k", &a.k_stride_token, &a.k_stride_head);
  kv_rows(k, vt, "v", &a.v_stride_token, &a.v_stride_head);
  const int64_t tokens = kt.size(0);
  if (vt.size(0) != tokens) refuse(PyExc_ValueError, "k has %lld rows, v %lld", (long long)tokens, (long long)vt.size(0));
  a.num_tokens = int32_t(tokens);
  const double eps = PyFloat_AsDouble(arg[12]);
  if (eps == -1.0 && PyErr_Occurred()) throw python_error();
  a.eps = float(eps);
  Queries q{}, qo{};
  if (given(arg[6])) {
    const Tensor &t = tensor(arg[6], "q");
    q = queries(k, t, "q", false);
    if (q.rows != tokens) refuse(PyExc_ValueError, "q has %lld rows, k %lld", (long long)q.rows, (long long)tokens);
    a.q_stride_token = q.token, a.q_stride_group = q.group, a.q_stride_head = q.head;
    a.num_q_heads = int32_t(q.heads);
    if (given(out_obj)) {
      qo = queries(k, tensor(out_obj, "q_out"), "q_out", true);
      if (qo.rows != tokens || qo.heads != q.heads) refuse(PyExc_ValueError, "q_out must have the rows and heads of q");
    }
  } else if (given(out_obj) || given(arg[10])) {
    refuse(PyExc_ValueError, "q_out and q_norm come with q");
  }
  if (given(arg[8]) != given(arg[9])) refuse(PyExc_ValueError, "cos and sin come together");
  if (given(arg[8])) {
    const Tensor &c = tensor(arg[8], "cos"), &s = tensor(arg[9], "sin");
    if ((c.scalar_type() != k.dtype && c.scalar_type() != at::kFloat) || s.scalar_type() != c.scalar_type())
      refuse(PyExc_TypeError, "cos and sin must both be of the cache's type or float32");
    if (c.dim() != 2 || c.sizes() != s.sizes() || c.strides() != s.strides() || c.stride(1) != 1 ||
        c.size(0) > 0x7fffffff || c.size(1) > 0x7fffffff)
      refuse(PyExc_ValueError, "cos and sin must be [positions, rot] alike, rows contiguous");
    if (c.device() != k.device || s.device() != k.device)
      refuse(PyExc_ValueError, "cos and sin must be on the cache's device");
    a.table_dtype = abi_type(c.scalar_type());
    a.max_positions = int32_t(c.size(0));
    a.rot_dim = int32_t(c.size(1));
    a.table_stride = c.size(0) > 1 ? c.stride(0) : (c.size(1) + 7) / 8 * 8;
  }
  for (int i = 10; i < 12; ++i) {
    if (!given(arg[i])) continue;
    const char *name = i == 10 ? "q_norm" : "k_norm";
    const Tensor &w = tensor(arg[i], name);
    operand(k, w, name);
    if (w.dim() != 1 || w.size(0) != k.dim || !w.is_contiguous())
      refuse(PyExc_ValueError, "%s must be a contiguous vector of %lld", name, (long long)k.dim);
  }
  need_cuda(k.device);
  const c10::cuda::CUDAGuard guard(k.device);
  Tensor made;
  if (given(arg[6])) {
    if (given(out_obj)) {
      a.q_out = THPVariable_Unpack(out_obj).data_ptr();
      a.q_out_stride_token = qo.token, a.q_out_stride_group = qo.group, a.q_out_stride_head = qo.head;
    } else {
      made = at::detail::empty_cuda({tokens, q.heads, k.dim}, k.dtype, k.device, std::nullopt);
      a.q_out = made.data_ptr();
      a.q_out_stride_token = q.heads * k.dim;
      a.q_out_stride_group = q.heads / k.heads * k.dim;
      a.q_out_stride_head = k.dim;
    }
    a.q = THPVariable_Unpack(arg[6]).const_data_ptr();
  }
  a.k = kt.const_data_ptr();
  a.v = vt.const_data_ptr();
  if (given(arg[8])) {
    a.cos = THPVariable_Unpack(arg[8]).const_data_ptr();
    a.sin = THPVariable_Unpack(arg[9]).const_data_ptr();
  }
  if (given(arg[10])) a.q_norm = THPVariable_Unpack(arg[10]).const_data_ptr();
  if (given(arg[11])) a.k_norm = THPVariable_Unpack(arg[11]).const_data_ptr();
  void *stream = c10::cuda::getCurrentCUDAStream(k.device.index()).stream();
  call_abi([&] { return ypk_paged_append(k.c, &a, stream); });
  written(*k.keys);
  written(*k.values);
  if (given(out_obj)) written(THPVariable_Unpack(out_obj));
  if (made.defined()) return THPVariable_Wrap(std::move(made));
  return Py_NewRef(out_obj);      // None without queries
  END_HANDLE_TH_ERRORS
}

// paged_decode(cache, device, k_cache, v_cache, q, out, return_lse, sm_scale, window) -> out or (out, lse)
PyObject *paged_decode(PyObject *, PyObject *const *arg, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 9) refuse(PyExc_TypeError, "paged_decode takes 9 arguments");
  const Cache k = cache_of(arg);
  const Tensor &qt = tensor(arg[4], "q");
  const Queries q = queries(k, qt, "q", false);
  if (q.rows > k.c->num_requests)
    refuse(PyExc_ValueError, "q has %lld rows, the tables %d requests", (long long)q.rows, k.c->num_requests);
  Queries o{};
  if (given(arg[5])) {
    const Tensor &t = tensor(arg[5], "out");
    if (t.sizes() != qt.sizes()) refuse(PyExc_ValueError, "out must have the shape of q");
    o = queries(k, t, "out", true);
  }
  const int lse_wanted = PyObject_IsTrue(arg[6]);
  if (lse_wanted < 0) throw python_error();
  ypk_paged_decode_args a = {};
  a.scale = 1.0f / sqrtf(float(k.dim));
  if (given(arg[7])) {
    const double s = PyFloat_AsDouble(arg[7]);
    if (s == -1.0 && PyErr_Occurred()) throw python_error();
    a.scale = float(s);
  }
  const int64_t window = integer(arg[8]);
  if (window < 0) refuse(PyExc_ValueError, "window %lld is negative", (long long)window);
  a.window = int32_t(std::min<int64_t>(window, 0x7fffffff));
  need_cuda(k.device);
  const c10::cuda::CUDAGuard guard(k.device);
  Tensor out, lse;
  if (given(arg[5])) {
    out = THPVariable_Unpack(arg[5]);
    a.out_stride_token = o.token, a.out_stride_group = o.group, a.out_stride_head = o.head;
  } else {
    out = at::detail::empty_cuda(qt.sizes(), k.dtype, k.device, std::nullopt);
    a.out_stride_token = q.heads * k.dim;
    a.out_stride_group = q.heads / k.heads * k.dim;
    a.out_stride_head = k.dim;
  }
  if (lse_wanted) {
    lse = at::detail::empty_cuda({q.rows, q.heads}, at::kFloat, k.device, std::nullopt);
    a.lse = static_cast<float *>(lse.data_ptr());
  }
  uint64_t need = 0;
  if (int rc = ypk_paged_decode_workspace(k.c, int32_t(q.heads), &need)) refuse_abi(rc);
  // Of this call alone, from torch's allocator: calls on several streams and graphs that replay
  // at the same time never share it.
  c10::DataPtr work;
  if (need) work = c10::cuda::CUDACachingAllocator::get()->allocate(need);
  a.q = qt.const_data_ptr();
  a.out = out.data_ptr();
  a.workspace = work.get();
  a.workspace_bytes = need;
  a.q_stride_token = q.token, a.q_stride_group = q.group, a.q_stride_head = q.head;
  a.rows = int32_t(q.rows);
  a.num_q_heads = int32_t(q.heads);
  void *stream = c10::cuda::getCurrentCUDAStream(k.device.index()).stream();
  call_abi([&] { return ypk_paged_decode(k.c, &a, stream); });
  if (given(arg[5])) written(out);
  PyObject *first = given(arg[5]) ? Py_NewRef(arg[5]) : THPVariable_Wrap(std::move(out));
  if (!lse_wanted || !first) return first;
  PyObject *second = THPVariable_Wrap(std::move(lse));
  PyObject *both = second ? PyTuple_Pack(2, first, second) : nullptr;
  Py_DECREF(first);
  Py_XDECREF(second);
  return both;
  END_HANDLE_TH_ERRORS
}

// Results of the logits at `ptr`, as (logprob, entropy, top_logprob, top_token).
PyObject *logprobs(const void *ptr, int dtype, int64_t rows, int64_t vocab, int64_t ld, const Tensor &tokens,
                   int64_t top, const c10::Device &device) {
  if (tokens.scalar_type() != at::kLong)
    refuse(PyExc_TypeError, "tokens must be int64, got %s", type_name(tokens.scalar_type()));
  const bool shaped = tokens.dim() >= 1 && tokens.dim() <= 2 && tokens.size(0) == rows &&
                      (tokens.dim() == 1 || tokens.size(1) == 1);
  if (!shaped || !tokens.is_contiguous())
    refuse(PyExc_ValueError, "tokens must be a contiguous [%lld] or [%lld, 1]", (long long)rows, (long long)rows);
  if (tokens.device() != device)
    refuse(PyExc_ValueError, "tokens are on %s, the logits on %s", tokens.device().str().c_str(), device.str().c_str());
  if (rows > 0x7fffffff || vocab > 0x7fffffff || top < 0 || top > 0x7fffffff)
    refuse(PyExc_ValueError, "logits [%lld, %lld], top_k %lld: out of range", (long long)rows, (long long)vocab, (long long)top);
  need_cuda(device);
  const c10::cuda::CUDAGuard guard(device);
  // One allocation for the four results (a call on a few rows 4.8 us, with four 6.1).
  const int64_t kept = std::min<int64_t>(top, 32);      // (more are refused below)
  const Tensor all = at::detail::empty_cuda({rows * (8 + 12 * kept)}, at::kByte, device, std::nullopt);
  int64_t at = 0;
  const auto take = [&](at::ScalarType type, at::IntArrayRef sizes) {
    Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(all.storage()), all.key_set(),
                                                        c10::scalarTypeToTypeMeta(type));
    t.unsafeGetTensorImpl()->set_storage_offset(at / int64_t(c10::elementSize(type)));
    t.unsafeGetTensorImpl()->set_sizes_contiguous(sizes);
    at += t.numel() * int64_t(c10::elementSize(type));
    return t;
  };
  Tensor top_token, top_logprob;
  if (top > 0) {
    top_token = take(at::kLong, {rows, kept});
    top_logprob = take(at::kFloat, {rows, kept});
  }
  Tensor logprob = take(at::kFloat, {rows}), entropy = take(at::kFloat, {rows});
  void *stream = c10::cuda::getCurrentCUDAStream(device.index()).stream();
  call_abi([&] {
    return ypk_token_logprobs(ptr, dtype, int32_t(rows), int32_t(vocab), ld,
                              static_cast<const int64_t *>(tokens.const_data_ptr()), int32_t(top),
                              static_cast<float *>(logprob.data_ptr()), static_cast<float *>(entropy.data_ptr()),
                              top > 0 ? static_cast<float *>(top_logprob.data_ptr()) : nullptr,
                              top > 0 ? static_cast<int64_t *>(top_token.data_ptr()) : nullptr, stream);
  });
  PyObject *result = PyTuple_New(4);
  if (!result) return nullptr;
  PyTuple_SET_ITEM(result, 0, THPVariable_Wrap(std::move(logprob)));
  PyTuple_SET_ITEM(result, 1, THPVariable_Wrap(std::move(entropy)));
  PyTuple_SET_ITEM(result, 2, top > 0 ? THPVariable_Wrap(std::move(top_logprob)) : Py_NewRef(Py_None));
  PyTuple_SET_ITEM(result, 3, top > 0 ? THPVariable_Wrap(std::move(top_token)) : Py_NewRef(Py_None));
  return result;
}

// token_logprobs(logits, tokens, top_k, valid_cols)
PyObject *token_logprobs(PyObject *, PyObject *const *arg, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 4) refuse(PyExc_TypeError, "token_logprobs takes 4 arguments");
  const Tensor &x = tensor(arg[0], "logits"), &t = tensor(arg[1], "tokens");
  if (x.scalar_type() != at::kBFloat16 && x.scalar_type() != at::kHalf && x.scalar_type() != at::kFloat)
    refuse(PyExc_TypeError, "logits are %s; bfloat16, float16 or float32 wanted", type_name(x.scalar_type()));
  if (x.dim() != 2 || (x.size(1) > 1 && x.stride(1) != 1))
    refuse(PyExc_ValueError, "logits must be [rows, columns] with contiguous rows");
  const int64_t rows = x.size(0), cols = x.size(1), vocab = given(arg[3]) ? integer(arg[3]) : cols;
  if (vocab < 1 || vocab > cols) refuse(PyExc_ValueError, "valid_cols %lld of %lld columns", (long long)vocab, (long long)cols);
  const int64_t ld = rows > 1 ? x.stride(0) : cols;
  if (ld < vocab) refuse(PyExc_ValueError, "rows of logits must not overlap");
  return logprobs(x.const_data_ptr(), abi_type(x.scalar_type()), rows, vocab, ld, t, integer(arg[2]), x.device());
  END_HANDLE_TH_ERRORS
}

// logprobs_at(address, dtype, rows, vocab, ld, tokens, top_k, device index): logits that no tensor holds
PyObject *logprobs_at(PyObject *, PyObject *const *arg, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 8) refuse(PyExc_TypeError, "logprobs_at takes 8 arguments");
  return logprobs(reinterpret_cast<const void *>(integer(arg[0])), int(integer(arg[1])), integer(arg[2]), integer(arg[3]),
                  integer(arg[4]), tensor(arg[5], "tokens"), integer(arg[6]),
                  c10::Device(c10::kCUDA, static_cast<c10::DeviceIndex>(integer(arg[7]))));
  END_HANDLE_TH_ERRORS
}

#define YPK_METHOD(f) {#f, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {YPK_METHOD(paged_append), YPK_METHOD(paged_decode), YPK_METHOD(token_logprobs),
                         YPK_METHOD(logprobs_at), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_serving", "Hot calls of the serving operators.", -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__serving(void) { return PyModule_Create(&module); }
