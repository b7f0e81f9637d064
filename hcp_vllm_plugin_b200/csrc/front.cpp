// Torch front end of the serving-step entry points: checks the tensors, fills the C
// structs of hcp_ring.h and calls the library on the current stream.
//
// These calls last a few microseconds on the GPU, so what the host spends on each
// bounds a serving loop: the same checks in Python cost 10-15 us a call.  The module
// holds no kernels and no state but the addresses of the library's functions, which
// bind() takes from the loaded libhcp_ring.so.
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstdarg>
#include <string>

#include "hcp_ring.h"

namespace {

using at::Tensor;

struct Refused {};  // a Python error is set

[[noreturn]] void refuse(const char* fmt, ...) {
  char text[512];
  va_list a;
  va_start(a, fmt);
  std::vsnprintf(text, sizeof(text), fmt, a);
  va_end(a);
  PyErr_SetString(PyExc_ValueError, text);
  throw Refused{};
}

// ---------------------------------------------------------------- the library
struct Library {
  int (*plan)(const hcp_step_plan_args*, void*);
  int (*rope)(const hcp_norm_rope_args*, void*);
  int (*update)(const void*, const void*, int64_t, int64_t, int64_t, const int64_t*, void*, int64_t, int32_t, int32_t,
                int32_t, int32_t, void*);
  int (*gather)(const void*, int64_t, int32_t, int32_t, int32_t, const int64_t*, int64_t, void*, void*, int64_t, int64_t,
                int32_t, void*);
  int (*decode)(const hcp_decode_q4_args*, void*);
  int64_t (*decode_bytes)(const hcp_decode_q4_args*);
};
Library lib{};
PyObject* check_fn = nullptr;  // raises the library's error for a status that is not 0

void check(int rc, const char* what) {
  if (rc == HCP_OK) return;
  PyObject* r = PyObject_CallFunction(check_fn, "is", rc, what);
  Py_XDECREF(r);
  if (!PyErr_Occurred()) PyErr_Format(PyExc_RuntimeError, "%s failed: %d", what, rc);
  throw Refused{};
}

struct WithoutGil {
  PyThreadState* state = PyEval_SaveThread();
  ~WithoutGil() { PyEval_RestoreThread(state); }
};

// A call of the library on the tensor's device and current stream, other Python threads running
// meanwhile (a launch may wait for room in the stream).
template <typename F>
int on_device_of(const Tensor& t, F&& call) {
  const c10::DeviceIndex dev = t.get_device();
  void* stream = c10::cuda::getCurrentCUDAStream(dev).stream();
  const WithoutGil free;
  if (c10::cuda::current_device() == dev) return call(stream);
  const c10::cuda::CUDAGuard guard(dev);
  return call(stream);
}

// ---------------------------------------------------------------- arguments
const Tensor& tensor(PyObject* o, const char* name) {
  if (!THPVariable_Check(o)) {
    PyErr_Format(PyExc_TypeError, "%s must be a tensor", name);
    throw Refused{};
  }
  return THPVariable_Unpack(o);
}
const Tensor* optional(PyObject* o, const char* name) { return o == Py_None ? nullptr : &tensor(o, name); }
int64_t integer(PyObject* o) {
  PyObject* i = PyNumber_Index(o);
  if (i == nullptr) throw Refused{};
  const long long v = PyLong_AsLongLong(i);
  Py_DECREF(i);
  if (v == -1 && PyErr_Occurred()) throw Refused{};
  return v;
}
double number(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw Refused{};
  return v;
}

// Raw addresses reach the kernels: every tensor has to be on the call's GPU.
void on_gpu(const Tensor& ref) {
  if (!ref.is_cuda()) refuse("tensors must be CUDA tensors (no CPU path)");
}
void beside(const Tensor& ref, const Tensor* t, const char* name) {
  if (t != nullptr && (!t->is_cuda() || t->get_device() != ref.get_device()))
    refuse("%s must be on %s (got %s)", name, ref.device().str().c_str(), t->device().str().c_str());
}
const char* dtype_name(at::ScalarType t) { return c10::toString(t); }
bool rows16(at::ScalarType t) { return t == at::kBFloat16 || t == at::kHalf; }
int32_t code(at::ScalarType t) { return t == at::kBFloat16 ? HCP_BF16 : t == at::kHalf ? HCP_F16 : HCP_F32; }

void* vector(const Tensor& t, const char* name, at::ScalarType type, int64_t n) {
  if (t.scalar_type() != type || t.dim() != 1 || !t.is_contiguous() || t.size(0) < n)
    refuse("%s must be a contiguous %s vector of at least %lld entries", name, dtype_name(type), static_cast<long long>(n));
  return t.data_ptr();
}
// Row stride (elements) of [rows, heads, D] whose last two dims are packed.
int64_t rows_heads(const Tensor& t, const char* name) {
  if (t.dim() != 3) refuse("%s must be [rows, heads, head_dim]", name);
  if (t.stride(2) != 1 || t.stride(1) != t.size(2)) refuse("%s must be contiguous in its last two dims", name);
  return t.size(0) > 1 ? t.stride(0) : t.size(1) * t.size(2);
}
// Row stride (elements) of a 2-D table whose rows are contiguous.
int64_t table_stride(const Tensor& t, const char* name) {
  if (t.dim() != 2 || (t.size(1) > 1 && t.stride(1) != 1)) refuse("%s must be 2-D with contiguous rows", name);
  return t.size(0) > 1 ? t.stride(0) : t.size(1);
}
// Head size of a 4-bit cache, checked against the rows' where given (< 0: not).
int64_t q4_cache(const Tensor& c, int64_t kv_heads, int64_t head_dim) {
  if (c.dim() != 4 || c.scalar_type() != at::kByte || !c.is_contiguous())
    refuse("kv_cache must be a contiguous uint8 [num_blocks, Hkv, block_size, 9*D/8] tensor");
  const int64_t d = c.size(3) * 8 / 9;
  if (9 * d != c.size(3) * 8 || (head_dim >= 0 && d != head_dim))
    refuse("kv_cache's last dimension %lld is not 9*D/8 of the rows' head size", static_cast<long long>(c.size(3)));
  if (kv_heads >= 0 && c.size(1) != kv_heads)
    refuse("kv_cache holds %lld KV heads, the rows %lld", static_cast<long long>(c.size(1)), static_cast<long long>(kv_heads));
  return d;
}
int32_t i32(int64_t v, const char* name) {
  if (v < INT32_MIN || v > INT32_MAX) refuse("%s is out of range", name);
  return static_cast<int32_t>(v);
}

Tensor empty(at::IntArrayRef shape, at::ScalarType type, const Tensor& like) {
  return Tensor(at::detail::empty_cuda(shape, type, like.device(), std::nullopt));
}
// A 1-D piece of a buffer.
Tensor piece(const Tensor& buf, int64_t at, int64_t n) {
  Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::TensorImpl::VIEW, c10::Storage(buf.storage()), buf.key_set(),
                                                      buf.dtype());
  t.unsafeGetTensorImpl()->set_storage_offset(at);
  t.unsafeGetTensorImpl()->set_sizes_contiguous({n});
  return t;
}

template <typename F>
PyObject* guarded(F&& body) {
  HANDLE_TH_ERRORS
  try {
    return body();
  } catch (const Refused&) {
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}
void arity(Py_ssize_t got, Py_ssize_t want) {
  if (got != want) {
    PyErr_Format(PyExc_TypeError, "%zd arguments given, %zd wanted", got, want);
    throw Refused{};
  }
  if (check_fn == nullptr) {
    PyErr_SetString(PyExc_RuntimeError, "the library is not bound");
    throw Refused{};
  }
}

// ---------------------------------------------------------------- the calls
// (context_lens, new_lens, block_table, free_blocks, free_head, block_size, num_tokens, pos_base) -> 8 tensors
PyObject* plan_step(PyObject*, PyObject* const* o, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    arity(n, 8);
    const Tensor &ctx = tensor(o[0], "context_lens"), &add = tensor(o[1], "new_lens"), &bt = tensor(o[2], "block_table"),
                 &fb = tensor(o[3], "free_blocks"), &fh = tensor(o[4], "free_head");
    const Tensor* base = optional(o[7], "pos_base");
    on_gpu(ctx);
    beside(ctx, &add, "new_lens");
    beside(ctx, &bt, "block_table");
    beside(ctx, &fb, "free_blocks");
    beside(ctx, &fh, "free_head");
    beside(ctx, base, "pos_base");
    hcp_step_plan_args a{};
    a.context_lens = static_cast<const int32_t*>(vector(ctx, "context_lens", at::kInt, 0));
    const int64_t reqs = ctx.size(0);
    if (bt.scalar_type() != at::kInt || bt.dim() != 2 || bt.size(0) < reqs)
      refuse("block_table must be an int32 [num_reqs, max_blocks] tensor");
    a.new_lens = static_cast<const int32_t*>(vector(add, "new_lens", at::kInt, reqs));
    if (base != nullptr) a.pos_base = static_cast<const int32_t*>(vector(*base, "pos_base", at::kInt, reqs));
    a.block_table = static_cast<int32_t*>(bt.data_ptr());
    a.block_table_stride = table_stride(bt, "block_table");
    a.block_table_width = bt.size(1);
    a.free_blocks = static_cast<const int32_t*>(vector(fb, "free_blocks", at::kInt, 0));
    a.num_free = fb.size(0);
    a.free_head = static_cast<const int32_t*>(vector(fh, "free_head", at::kInt, 1));
    const int64_t bs = integer(o[5]), tokens = integer(o[6]);
    if (tokens < 0 || tokens > INT32_MAX || bs <= 0) refuse("num_tokens must be >= 0 and block_size positive");
    a.num_reqs = i32(reqs, "num_reqs");
    a.block_size = i32(bs, "block_size");
    a.num_tokens = tokens;
    const Tensor wide = empty({2 * tokens}, at::kLong, ctx), small = empty({2 * reqs + 2 * tokens + 3}, at::kInt, ctx);
    a.positions = static_cast<int64_t*>(wide.data_ptr());
    a.slot_mapping = a.positions + tokens;
    a.query_start = static_cast<int32_t*>(small.data_ptr());
    a.seq_lens = a.query_start + reqs + 1;
    a.token_req = a.seq_lens + reqs;
    a.kv_lens = a.token_req + tokens;
    a.free_head_out = a.kv_lens + tokens;
    a.missing_out = a.free_head_out + 1;
    check(on_device_of(ctx, [&](void* s) { return lib.plan(&a, s); }), "hcp_kv_plan_step");
    // the views are made while the kernel runs
    const Tensor views[8] = {piece(small, 0, reqs + 1),          piece(small, reqs + 1, reqs),
                             piece(wide, 0, tokens),             piece(wide, tokens, tokens),
                             piece(small, 2 * reqs + 1, tokens), piece(small, 2 * reqs + 1 + tokens, tokens),
                             piece(small, 2 * reqs + 1 + 2 * tokens, 1), piece(small, 2 * reqs + 2 + 2 * tokens, 1)};
    PyObject* r = PyTuple_New(8);
    if (r == nullptr) throw Refused{};
    for (int i = 0; i < 8; ++i) {
      PyObject* v = THPVariable_Wrap(views[i]);
      if (v == nullptr) {
        Py_DECREF(r);
        throw Refused{};
      }
      PyTuple_SET_ITEM(r, i, v);
    }
    return r;
  });
}

PyObject* pair(const Tensor& a, const Tensor& b) {
  PyObject *x = THPVariable_Wrap(a), *y = THPVariable_Wrap(b);
  PyObject* r = x != nullptr && y != nullptr ? PyTuple_Pack(2, x, y) : nullptr;
  Py_XDECREF(x);
  Py_XDECREF(y);
  return r;
}

// (q, k, positions, cos_sin, q_weight, k_weight, eps, interleaved, q_out, k_out, value, kv_cache, slot_mapping) -> q_out, k_out
PyObject* norm_rope(PyObject*, PyObject* const* o, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    arity(n, 13);
    const Tensor &q = tensor(o[0], "q"), &k = tensor(o[1], "k"), &pos = tensor(o[2], "positions"), &tab = tensor(o[3], "cos_sin");
    const Tensor *qw = optional(o[4], "q_weight"), *kw = optional(o[5], "k_weight"), *qo = optional(o[8], "q_out"),
                 *ko = optional(o[9], "k_out"), *v = optional(o[10], "value"), *cache = optional(o[11], "kv_cache"),
                 *slots = optional(o[12], "slot_mapping");
    on_gpu(q);
    beside(q, &k, "k");
    beside(q, &pos, "positions");
    beside(q, &tab, "cos_sin");
    beside(q, qw, "q_weight");
    beside(q, kw, "k_weight");
    beside(q, qo, "q_out");
    beside(q, ko, "k_out");
    beside(q, v, "value");
    beside(q, cache, "kv_cache");
    beside(q, slots, "slot_mapping");
    const at::ScalarType type = q.scalar_type();
    if (!rows16(type) || k.scalar_type() != type) refuse("q and k must be bf16 or fp16 rows of one dtype");
    if (q.dim() != 3 || k.dim() != 3 || k.size(0) != q.size(0) || k.size(2) != q.size(2))
      refuse("q must be [T, H, D] and k [T, Hkv, D]");
    const int64_t tokens = q.size(0), d = q.size(2);
    if (tab.scalar_type() != at::kFloat && tab.scalar_type() != type) refuse("cos_sin must be float32 or q's dtype");
    const Tensor q_new = qo != nullptr ? Tensor() : empty(q.sizes(), type, q);
    const Tensor k_new = ko != nullptr ? Tensor() : empty(k.sizes(), type, q);
    const Tensor &q_out = qo != nullptr ? *qo : q_new, &k_out = ko != nullptr ? *ko : k_new;
    if (q_out.sizes() != q.sizes() || q_out.scalar_type() != type) refuse("q_out must have the shape and dtype of q");
    if (k_out.sizes() != k.sizes() || k_out.scalar_type() != type) refuse("k_out must have the shape and dtype of k");
    hcp_norm_rope_args a{};
    a.dtype = code(type);
    a.num_heads = i32(q.size(1), "q's heads");
    a.num_kv_heads = i32(k.size(1), "k's heads");
    a.head_dim = i32(d, "head_dim");
    a.q = q.data_ptr();
    a.q_row_stride = rows_heads(q, "q");
    a.k = k.data_ptr();
    a.k_row_stride = rows_heads(k, "k");
    a.q_out = q_out.data_ptr();
    a.q_out_row_stride = rows_heads(q_out, "q_out");
    a.k_out = k_out.data_ptr();
    a.k_out_row_stride = rows_heads(k_out, "k_out");
    a.positions = static_cast<const int64_t*>(vector(pos, "positions", at::kLong, tokens));
    a.num_tokens = tokens;
    a.table_stride = table_stride(tab, "cos_sin");
    a.cos_sin = tab.data_ptr();
    a.table_rows = tab.size(0);
    a.table_dtype = code(tab.scalar_type());
    a.rotary = i32(tab.size(1), "rotary");
    const int truth = PyObject_IsTrue(o[7]);
    if (truth < 0) throw Refused{};
    a.interleaved = truth;
    a.eps = static_cast<float>(number(o[6]));
    if (qw != nullptr) a.q_weight = vector(*qw, "q_weight", type, d);
    if (kw != nullptr) a.k_weight = vector(*kw, "k_weight", type, d);
    if (cache != nullptr) {
      if (v == nullptr || slots == nullptr) refuse("kv_cache needs value and slot_mapping");
      if (v->sizes() != k.sizes() || v->scalar_type() != type) refuse("value must have k's shape and dtype");
      a.v = v->data_ptr();
      a.v_row_stride = rows_heads(*v, "value");
      if (cache->scalar_type() == at::kByte) {
        q4_cache(*cache, k.size(1), d);
        a.cache_kind = HCP_ROPE_CACHE_Q4;
      } else {
        if (cache->dim() != 4 || !cache->is_contiguous() || cache->scalar_type() != type || cache->size(1) != k.size(1) ||
            cache->size(3) != 2 * d)
          refuse("kv_cache must be a contiguous [num_blocks, Hkv, block_size, 2*D] tensor");
        a.cache_kind = HCP_ROPE_CACHE_SAME;
      }
      a.kv_cache = cache->data_ptr();
      a.num_blocks = cache->size(0);
      a.block_size = i32(cache->size(2), "block_size");
      a.slot_mapping = static_cast<const int64_t*>(vector(*slots, "slot_mapping", at::kLong, tokens));
    } else if (v != nullptr || slots != nullptr) {
      refuse("value and slot_mapping go with kv_cache");
    }
    check(on_device_of(q, [&](void* s) { return lib.rope(&a, s); }), "hcp_qk_norm_rope");
    return pair(q_out, k_out);
  });
}

// (key, value, kv_cache, slot_mapping)
PyObject* update_q4(PyObject*, PyObject* const* o, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    arity(n, 4);
    const Tensor &k = tensor(o[0], "key"), &v = tensor(o[1], "value"), &cache = tensor(o[2], "kv_cache"),
                 &slots = tensor(o[3], "slot_mapping");
    on_gpu(k);
    beside(k, &v, "value");
    beside(k, &cache, "kv_cache");
    beside(k, &slots, "slot_mapping");
    const at::ScalarType type = k.scalar_type();
    if (!rows16(type) || v.scalar_type() != type || v.sizes() != k.sizes())
      refuse("key and value must be bf16 or fp16 rows of one shape");
    if (k.dim() != 3) refuse("key must be [rows, heads, head_dim]");
    q4_cache(cache, k.size(1), k.size(2));
    const int64_t* slot = static_cast<const int64_t*>(vector(slots, "slot_mapping", at::kLong, 0));
    const int64_t rows = std::min(slots.size(0), k.size(0)), ks = rows_heads(k, "key"), vs = rows_heads(v, "value");
    const int32_t bs = i32(cache.size(2), "block_size"), heads = i32(k.size(1), "heads"), d = i32(k.size(2), "head_dim");
    check(on_device_of(k,
                       [&](void* s) {
                         return lib.update(k.data_ptr(), v.data_ptr(), rows, ks, vs, slot, cache.data_ptr(), cache.size(0), bs,
                                           heads, d, code(type), s);
                       }),
          "hcp_kv_cache_update_q4");
    Py_RETURN_NONE;
  });
}

// (kv_cache, slot_mapping, dtype, key, value) -> key, value
PyObject* gather_q4(PyObject*, PyObject* const* o, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    arity(n, 5);
    const Tensor &cache = tensor(o[0], "kv_cache"), &slots = tensor(o[1], "slot_mapping");
    const Tensor *k = optional(o[3], "key"), *v = optional(o[4], "value");
    on_gpu(cache);
    beside(cache, &slots, "slot_mapping");
    beside(cache, k, "key");
    beside(cache, v, "value");
    if (!THPDtype_Check(o[2])) refuse("dtype must be torch.bfloat16 or torch.float16");
    const at::ScalarType type = reinterpret_cast<THPDtype*>(o[2])->scalar_type;
    if (!rows16(type)) refuse("unsupported dtype %s", dtype_name(type));
    const int64_t d = q4_cache(cache, -1, -1), heads = cache.size(1);
    const int64_t* slot = static_cast<const int64_t*>(vector(slots, "slot_mapping", at::kLong, 0));
    const int64_t rows = slots.size(0);
    const Tensor k_new = k != nullptr ? Tensor() : empty({rows, heads, d}, type, cache);
    const Tensor v_new = v != nullptr ? Tensor() : empty({rows, heads, d}, type, cache);
    const Tensor &key = k != nullptr ? *k : k_new, &value = v != nullptr ? *v : v_new;
    for (const Tensor* t : {&key, &value})
      if (t->dim() != 3 || t->size(0) < rows || t->size(1) != heads || t->size(2) != d || t->scalar_type() != type)
        refuse("%s must hold n rows [Hkv, D] of %s", t == &key ? "key" : "value", dtype_name(type));
    const int64_t ks = rows_heads(key, "key"), vs = rows_heads(value, "value");
    const int32_t bs = i32(cache.size(2), "block_size"), hkv = i32(heads, "heads"), hd = i32(d, "head_dim");
    check(on_device_of(cache,
                       [&](void* s) {
                         return lib.gather(cache.data_ptr(), cache.size(0), bs, hkv, hd, slot, rows, key.data_ptr(),
                                           value.data_ptr(), ks, vs, code(type), s);
                       }),
          "hcp_kv_cache_gather_q4");
    return pair(key, value);
  });
}

// (q, kv_cache, block_table, kv_lens, scale, out, lse, token_req, workspace)
PyObject* decode_q4(PyObject*, PyObject* const* o, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    arity(n, 9);
    const Tensor &q = tensor(o[0], "q"), &cache = tensor(o[1], "kv_cache"), &bt = tensor(o[2], "block_table"),
                 &lens = tensor(o[3], "kv_lens"), &out = tensor(o[5], "out");
    const Tensor *lse = optional(o[6], "lse"), *req = optional(o[7], "token_req"), *ws = optional(o[8], "workspace");
    on_gpu(q);
    beside(q, &cache, "kv_cache");
    beside(q, &bt, "block_table");
    beside(q, &lens, "kv_lens");
    beside(q, &out, "out");
    beside(q, lse, "lse");
    beside(q, req, "token_req");
    beside(q, ws, "workspace");
    const at::ScalarType type = q.scalar_type();
    if (!rows16(type)) refuse("q must be a bf16/fp16 CUDA tensor");
    if (q.dim() != 3) refuse("q must be [rows, heads, head_dim]");
    const int64_t rows = q.size(0), heads = q.size(1), d = q.size(2);
    q4_cache(cache, -1, d);
    if (bt.scalar_type() != at::kInt) refuse("block_table must be an int32 [num_reqs, max_blocks] tensor");
    if (out.dim() != 3 || out.size(0) < rows || out.size(1) != heads || out.size(2) != d ||
        (out.scalar_type() != type && out.scalar_type() != at::kFloat))
      refuse("out must be [>= q rows, H, D] of q's dtype or float32");
    hcp_decode_q4_args a{};
    a.dtype = code(type);
    a.num_heads = i32(heads, "heads");
    a.num_kv_heads = i32(cache.size(1), "KV heads");
    a.head_dim = i32(d, "head_dim");
    a.scale = static_cast<float>(number(o[4]));
    a.block_size = i32(cache.size(2), "block_size");
    a.q = q.data_ptr();
    a.q_rows = rows;
    a.q_row_stride = rows_heads(q, "q");
    a.kv_cache = cache.data_ptr();
    a.num_blocks = cache.size(0);
    a.block_table = static_cast<const int32_t*>(bt.data_ptr());
    a.block_table_stride = table_stride(bt, "block_table");
    a.block_table_rows = bt.size(0);
    a.block_table_width = bt.size(1);
    a.kv_lens = static_cast<const int32_t*>(vector(lens, "kv_lens", at::kInt, rows));
    if (req != nullptr) a.token_req = static_cast<const int32_t*>(vector(*req, "token_req", at::kInt, rows));
    else if (bt.size(0) < rows) refuse("block_table needs a row for every query row (or token_req)");
    a.out = out.data_ptr();
    a.out_dtype = code(out.scalar_type());
    a.out_row_stride = rows_heads(out, "out");
    if (lse != nullptr) {
      if (lse->scalar_type() != at::kFloat || lse->dim() != 2 || lse->size(0) != heads || lse->size(1) < rows ||
          (lse->size(1) > 1 && lse->stride(1) != 1))
        refuse("lse must be a float32 [H, >= q rows] tensor with unit column stride");
      a.lse = static_cast<float*>(lse->data_ptr());
      a.lse_stride = heads > 1 ? lse->stride(0) : lse->size(1);
    }
    const int64_t need = lib.decode_bytes(&a);
    if (need < 0) check(HCP_ERR_INVALID, "hcp_decode_q4_workspace_bytes");
    // a buffer of its own per call: torch's allocator orders its reuse on the stream, and a
    // captured call keeps its own with the graph
    const Tensor own = ws != nullptr ? Tensor() : empty({need}, at::kByte, q);
    const Tensor& work = ws != nullptr ? *ws : own;
    if (!work.is_contiguous()) refuse("workspace must be contiguous");
    a.workspace = work.data_ptr();
    a.workspace_bytes = static_cast<int64_t>(work.nbytes());
    check(on_device_of(q, [&](void* s) { return lib.decode(&a, s); }), "hcp_decode_q4_splitkv");
    Py_RETURN_NONE;
  });
}

// (check, plan, rope, update, gather, decode, decode_bytes): the status check and the functions' addresses
PyObject* bind(PyObject*, PyObject* const* o, Py_ssize_t n) {
  if (n != 7) {
    PyErr_SetString(PyExc_TypeError, "bind takes 7 arguments");
    return nullptr;
  }
  void* at[6];
  for (int i = 0; i < 6; ++i) {
    at[i] = PyLong_AsVoidPtr(o[i + 1]);
    if (at[i] == nullptr) {
      if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "null function");
      return nullptr;
    }
  }
  lib.plan = reinterpret_cast<decltype(lib.plan)>(at[0]);
  lib.rope = reinterpret_cast<decltype(lib.rope)>(at[1]);
  lib.update = reinterpret_cast<decltype(lib.update)>(at[2]);
  lib.gather = reinterpret_cast<decltype(lib.gather)>(at[3]);
  lib.decode = reinterpret_cast<decltype(lib.decode)>(at[4]);
  lib.decode_bytes = reinterpret_cast<decltype(lib.decode_bytes)>(at[5]);
  Py_INCREF(o[0]);
  Py_XDECREF(check_fn);
  check_fn = o[0];
  Py_RETURN_NONE;
}

template <typename F>
PyCFunction fast(F f) { return reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)); }

PyMethodDef methods[] = {{"bind", fast(bind), METH_FASTCALL, nullptr},
                         {"plan_step", fast(plan_step), METH_FASTCALL, nullptr},
                         {"norm_rope", fast(norm_rope), METH_FASTCALL, nullptr},
                         {"update_q4", fast(update_q4), METH_FASTCALL, nullptr},
                         {"gather_q4", fast(gather_q4), METH_FASTCALL, nullptr},
                         {"decode_q4", fast(decode_q4), METH_FASTCALL, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_hcp_front", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__hcp_front() {
  PyObject* m = PyModule_Create(&module);
  // the torch and Python that it was built for: another one's insides may differ
  if (m != nullptr && PyModule_AddStringConstant(m, "built_for", HCP_BUILT_FOR) < 0) Py_CLEAR(m);
  return m;
}
