// decoder_bind.cpp -- the Python calls of the decoder operators: checks of the
// tensors, outputs and workspaces from torch's allocator, the current stream,
// and the C ABI of include/cruise_decoder.h.
//
// A small decode step runs a few microseconds on the GPU, so the call itself
// counts: one takes 3 to 4 of the host's so, launch and output tensor included,
// where the same checks in Python with a ctypes call took 14 to 18.
//
// The library's entries come in as addresses (bind), so that this module calls
// the library that cruise_b200._lib loaded.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <c10/core/AutogradState.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <cstdarg>
#include <cstdio>

#include "../../include/cruise_decoder.h"

namespace {

struct Entries {
  decltype(&cruise_decoder_rotate_store) rotate_store;
  decltype(&cruise_decoder_attention) attention;
  decltype(&cruise_decoder_attention_workspace) attention_workspace;
  decltype(&cruise_decoder_choose) choose;
  decltype(&cruise_decoder_last_error) last_error;
};
Entries g_entries{};
PyObject *g_failure = nullptr;   // called with (code, message): the exception of a CUDA error

// A refused argument: becomes ValueError.
struct Refused {
  char text[256];
  explicit Refused(const char *format, ...) __attribute__((format(printf, 2, 3))) {
    va_list args;
    va_start(args, format);
    std::vsnprintf(text, sizeof(text), format, args);
    va_end(args);
  }
};

#define NEED(condition, ...) \
  do {                       \
    if (!(condition)) throw Refused(__VA_ARGS__); \
  } while (0)

const char *type_name(at::ScalarType t) {
  switch (t) {
    case at::kBFloat16: return "torch.bfloat16";
    case at::kHalf: return "torch.float16";
    case at::kFloat: return "torch.float32";
    case at::kInt: return "torch.int32";
    case at::kLong: return "torch.int64";
    default: return "another type";
  }
}

int code(at::ScalarType t) { return t == at::kBFloat16 ? 0 : t == at::kHalf ? 1 : 2; }
bool half(at::ScalarType t) { return t == at::kBFloat16 || t == at::kHalf; }

// The tensors of one call: all on the device of the first.
class Call {
 public:
  const at::Tensor &first(PyObject *o, const char *name) {
    NEED(THPVariable_Check(o), "%s must be a CUDA tensor", name);
    const at::Tensor &t = THPVariable_Unpack(o);
    NEED(t.is_cuda(), "%s must be a CUDA tensor", name);
    device_ = t.get_device();
    plain(t, name);
    return t;
  }
  const at::Tensor &take(PyObject *o, const char *name) {
    NEED(THPVariable_Check(o) && THPVariable_Unpack(o).is_cuda() && THPVariable_Unpack(o).get_device() == device_,
         "%s must be a tensor on cuda:%d", name, device_);
    const at::Tensor &t = THPVariable_Unpack(o);
    plain(t, name);
    return t;
  }
  // nullptr for None
  const at::Tensor *maybe(PyObject *o, const char *name) { return o == Py_None ? nullptr : &take(o, name); }
  int device() const { return device_; }
  void *stream() const { return c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(device_)).stream(); }
  at::Tensor empty(at::IntArrayRef sizes, at::ScalarType type) const {
    return at::empty(sizes, at::TensorOptions().dtype(type).device(at::kCUDA, static_cast<c10::DeviceIndex>(device_)));
  }

 private:
  void plain(const at::Tensor &t, const char *name) const {
    NEED(t.layout() == at::kStrided && !t.is_conj() && !t.is_neg(), "%s must be a plain strided tensor", name);
    NEED(!(t.requires_grad() && c10::GradMode::is_enabled()),
         "%s requires a gradient: the decoder operators are for inference", name);
    NEED(!(c10::AutogradState::get_tls_state().get_fw_grad_mode() && t._fw_grad(0).defined()),
         "%s carries a tangent (forward mode): the decoder operators are for inference", name);
    // (a view of a traced or fake tensor has an address, an offset from nowhere)
    NEED(t.numel() == 0 || (t.has_storage() && t.storage().data() != nullptr), "%s has no memory: the call cannot be traced", name);
  }
  int device_ = -1;
};

void *pointer(const at::Tensor *t) { return t == nullptr ? nullptr : t->data_ptr(); }

const at::Tensor &vector(const at::Tensor &t, const char *name, at::ScalarType type, int64_t count) {
  NEED(t.scalar_type() == type && t.dim() == 1 && t.size(0) == count && (count < 2 || t.stride(0) == 1),
       "%s must be a contiguous %s vector of %lld", name, type_name(type), static_cast<long long>(count));
  return t;
}

// Elements between rows; a single row's stride is its width (torch leaves any value there).
int64_t row_stride(const at::Tensor &t, int64_t width) { return t.size(0) > 1 ? t.stride(0) : std::max<int64_t>(width, 1); }

// [rows, width] with contiguous rows, for a width of 0 too
bool rows_of(const at::Tensor &t, int64_t rows) { return t.dim() == 2 && t.size(0) == rows && (t.size(1) < 2 || t.stride(1) == 1); }

// Row stride of [rows, heads, d] with adjacent heads.
int64_t heads(const at::Tensor &t, const char *name, int64_t rows, int64_t n, int64_t d, at::ScalarType type) {
  NEED(t.scalar_type() == type && t.dim() == 3 && t.size(0) == rows && t.size(1) == n && t.size(2) == d,
       "%s must be %s [%lld, %lld, %lld]", name, type_name(type), static_cast<long long>(rows), static_cast<long long>(n),
       static_cast<long long>(d));
  NEED(rows == 0 || (t.stride(2) == 1 && (n < 2 || t.stride(1) == d)), "%s: the heads of a row must lie next to one another", name);
  return row_stride(t, n * d);
}

struct Caches {
  int64_t blocks, block, nkv, d, stride;
  at::ScalarType type;
};

// Two paged caches [blocks, block_size, kv heads, d] of one block stride.
Caches caches(const at::Tensor &key, const at::Tensor &value) {
  NEED(key.dim() == 4 && value.sizes() == key.sizes() && value.scalar_type() == key.scalar_type() && half(key.scalar_type()),
       "key_cache and value_cache must be bf16 or fp16 [blocks, block_size, kv_heads, head_dim] of one shape");
  NEED(key.numel() > 0, "the caches must not be empty");
  Caches c{key.size(0), key.size(1), key.size(2), key.size(3), 0, key.scalar_type()};
  const int64_t inner[4] = {0, c.nkv * c.d, c.d, 1};
  for (const at::Tensor *t : {&key, &value})
    for (int axis = 1; axis < 4; ++axis)
      NEED(t->size(axis) == 1 || t->stride(axis) == inner[axis], "%s: the slots of a block must be contiguous",
           t == &key ? "key_cache" : "value_cache");
  NEED(c.blocks == 1 || key.stride(0) == value.stride(0), "key_cache and value_cache must have one block stride");
  c.stride = c.blocks > 1 ? key.stride(0) : c.block * c.nkv * c.d;
  return c;
}

int32_t small(int64_t v, const char *what) {
  NEED(v >= 0 && v <= 0x7fffffff, "%s: %lld passes 2^31", what, static_cast<long long>(v));
  return static_cast<int32_t>(v);
}

double number(PyObject *o, const char *name) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred() != nullptr) {
    PyErr_Clear();
    throw Refused("%s must be a number", name);
  }
  return v;
}

// The status of a library call as a Python exception (false) or success.
bool done(int32_t rc) {
  if (rc == 0) return true;
  const char *why = g_entries.last_error();
  if (rc == -1) {
    PyErr_SetString(PyExc_ValueError, why);
  } else {
    PyObject *failure = PyObject_CallFunction(g_failure, "is", static_cast<int>(rc), why);
    if (failure != nullptr) {
      PyErr_SetObject(reinterpret_cast<PyObject *>(Py_TYPE(failure)), failure);
      Py_DECREF(failure);
    }
  }
  return false;
}

// Runs `body`; no C++ exception leaves the module.
template <typename Body>
PyObject *guarded(Body body) {
  try {
    NEED(g_entries.choose != nullptr, "the decoder operators are not bound to the library");
    return body();
  } catch (const Refused &r) {
    PyErr_SetString(PyExc_ValueError, r.text);
  } catch (const std::exception &e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  }
  return nullptr;
}

bool counted(Py_ssize_t n, Py_ssize_t want) {
  if (n == want) return true;
  PyErr_Format(PyExc_TypeError, "%zd arguments expected, got %zd", want, n);
  return false;
}

// The library call without the interpreter lock.
template <typename F>
int32_t unlocked(F call) {
  PyThreadState *state = PyEval_SaveThread();
  const int32_t rc = call();
  PyEval_RestoreThread(state);
  return rc;
}

// What an in-place operation does beside writing: autograd sees that a value it
// keeps for a backward pass is no longer the one it kept.
void written(const at::Tensor *t) {
  if (t != nullptr && !t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
}

// `given` (a borrowed reference) or a wrapped new tensor.
PyObject *answer(PyObject *given, const at::Tensor &made) {
  if (given != Py_None) {
    Py_INCREF(given);
    return given;
  }
  return THPVariable_Wrap(made);
}

// qkv, position, slot, cos, sin, key_cache, value_cache, num_heads, q_norm, k_norm, eps, out
PyObject *rotate_store(PyObject *, PyObject *const *v, Py_ssize_t n) {
  if (!counted(n, 12)) return nullptr;
  return guarded([&]() -> PyObject * {
    Call call;
    const at::Tensor &qkv = call.first(v[0], "qkv"), &position = call.take(v[1], "position"), &slot = call.take(v[2], "slot");
    const at::Tensor &cos = call.take(v[3], "cos"), &sin = call.take(v[4], "sin");
    const at::Tensor &key = call.take(v[5], "key_cache"), &value = call.take(v[6], "value_cache");
    const at::Tensor *q_norm = call.maybe(v[8], "q_norm"), *k_norm = call.maybe(v[9], "k_norm"), *given = call.maybe(v[11], "out");
    const Caches c = caches(key, value);
    const double asked = number(v[7], "num_heads"), eps = number(v[10], "eps");
    NEED(asked >= 1 && asked <= 1024 && asked == std::floor(asked), "num_heads must be a whole number from 1 to 1024");
    const int64_t nq = static_cast<int64_t>(asked), width = (nq + 2 * c.nkv) * c.d;
    NEED(qkv.scalar_type() == c.type, "qkv and the caches must have one type");
    NEED(qkv.dim() == 2 && qkv.size(1) == width, "qkv must be [tokens, %lld] for %lld query and %lld KV heads of %lld",
         static_cast<long long>(width), static_cast<long long>(nq), static_cast<long long>(c.nkv), static_cast<long long>(c.d));
    const int64_t tokens = qkv.size(0);
    NEED(tokens == 0 || qkv.stride(1) == 1, "qkv rows must be contiguous");
    vector(position, "position", at::kLong, tokens);
    vector(slot, "slot", at::kInt, tokens);
    NEED(cos.dim() == 2 && cos.sizes() == sin.sizes() && cos.scalar_type() == sin.scalar_type() &&
             (cos.scalar_type() == at::kBFloat16 || cos.scalar_type() == at::kFloat) && cos.is_contiguous() && sin.is_contiguous(),
         "cos and sin must be contiguous bf16 or fp32 [rows, rotary]");
    NEED((q_norm == nullptr) == (k_norm == nullptr), "pass both norm weights or neither");
    if (q_norm != nullptr) {
      vector(*q_norm, "q_norm", c.type, c.d);
      vector(*k_norm, "k_norm", c.type, c.d);
    }
    at::Tensor made;
    if (given == nullptr) {
      made = call.empty({tokens, nq, c.d}, c.type);
      given = &made;
    }
    const int64_t q_stride = heads(*given, "out", tokens, nq, c.d, c.type);
    const int32_t t = small(tokens, "tokens"), rows = small(cos.size(0), "rows of cos"), rotary = small(cos.size(1), "rotary");
    const int32_t nkv = small(c.nkv, "KV heads"), d = small(c.d, "head size"), block = small(c.block, "block size");
    void *const stream = call.stream();
    const int32_t rc = unlocked([&] {
      return g_entries.rotate_store(qkv.data_ptr(), row_stride(qkv, width), t, static_cast<int32_t>(nq), nkv, d, code(c.type),
                                    static_cast<const int64_t *>(position.data_ptr()), static_cast<const int32_t *>(slot.data_ptr()),
                                    pointer(q_norm), pointer(k_norm), static_cast<float>(eps), cos.data_ptr(), sin.data_ptr(),
                                    code(cos.scalar_type()), rows, rotary, given->data_ptr(), q_stride, key.data_ptr(),
                                    value.data_ptr(), c.blocks, block, c.stride, call.device(), stream);
    });
    if (!done(rc)) return nullptr;
    for (const at::Tensor *t : {&key, &value, given}) written(t);
    return answer(v[11], made);
  });
}

// q, key_cache, value_cache, block_table, seq_len, scale, out, lse
PyObject *paged_attention(PyObject *, PyObject *const *v, Py_ssize_t n) {
  if (!counted(n, 8)) return nullptr;
  return guarded([&]() -> PyObject * {
    Call call;
    const at::Tensor &q = call.first(v[0], "q"), &key = call.take(v[1], "key_cache"), &value = call.take(v[2], "value_cache");
    const at::Tensor &table = call.take(v[3], "block_table"), &seq_len = call.take(v[4], "seq_len");
    const at::Tensor *given = call.maybe(v[6], "out"), *lse = call.maybe(v[7], "lse");
    const Caches c = caches(key, value);
    NEED(q.dim() == 3 && q.size(2) == c.d && q.size(1) > 0 && q.size(1) % c.nkv == 0, "q must be [rows, a multiple of %lld heads, %lld]",
         static_cast<long long>(c.nkv), static_cast<long long>(c.d));
    const int64_t rows = q.size(0), nq = q.size(1);
    const int64_t q_stride = heads(q, "q", rows, nq, c.d, c.type);
    NEED(table.scalar_type() == at::kInt && rows_of(table, rows), "block_table must be int32 [%lld, width] with contiguous rows",
         static_cast<long long>(rows));
    const int64_t width = table.size(1);
    vector(seq_len, "seq_len", at::kInt, rows);
    const double scale = v[5] == Py_None ? 1.0 / std::sqrt(static_cast<double>(c.d)) : number(v[5], "scale");
    at::Tensor made;
    if (given == nullptr) {
      made = call.empty({rows, nq, c.d}, c.type);
      given = &made;
    }
    const int64_t out_stride = heads(*given, "out", rows, nq, c.d, c.type);
    NEED(lse == nullptr || (lse->scalar_type() == at::kFloat && lse->dim() == 2 && lse->size(0) == rows && lse->size(1) == nq &&
                            lse->is_contiguous()),
         "lse must be contiguous torch.float32 [%lld, %lld]", static_cast<long long>(rows), static_cast<long long>(nq));
    const int32_t r = small(rows, "rows"), h = small(nq, "heads"), nkv = small(c.nkv, "KV heads"), d = small(c.d, "head size");
    const int32_t block = small(c.block, "block size"), w = small(width, "table width");
    const int64_t need = g_entries.attention_workspace(r, h, nkv, d, width * c.block, call.device());
    if (need < 0) {
      done(-1);
      return nullptr;
    }
    // from torch's allocator on this stream, so calls on other streams and captured graphs have their own
    at::Tensor workspace;
    if (need > 0) workspace = call.empty({need}, at::kByte);
    void *const stream = call.stream();
    const int32_t rc = unlocked([&] {
      return g_entries.attention(q.data_ptr(), q_stride, r, h, nkv, d, code(c.type), key.data_ptr(), value.data_ptr(), c.blocks, block,
                                 c.stride, width > 0 ? static_cast<const int32_t *>(table.data_ptr()) : nullptr,
                                 row_stride(table, width), w, static_cast<const int32_t *>(seq_len.data_ptr()),
                                 static_cast<float>(scale), given->data_ptr(), out_stride, static_cast<float *>(pointer(lse)),
                                 need > 0 ? workspace.data_ptr() : nullptr, need, call.device(), stream);
    });
    if (!done(rc)) return nullptr;
    for (const at::Tensor *t : {given, lse}) written(t);
    return answer(v[6], made);
  });
}

// logits, history, prompt_len, history_len, repetition, frequency, presence,
// bias_token, bias_value, bias_len, allowed, active, processed, out, append
PyObject *choose(PyObject *, PyObject *const *v, Py_ssize_t n) {
  if (!counted(n, 15)) return nullptr;
  return guarded([&]() -> PyObject * {
    Call call;
    const at::Tensor &logits = call.first(v[0], "logits");
    const at::Tensor *history = call.maybe(v[1], "history"), *prompt_len = call.maybe(v[2], "prompt_len");
    const at::Tensor *history_len = call.maybe(v[3], "history_len");
    const at::Tensor *penalty[3] = {call.maybe(v[4], "repetition"), call.maybe(v[5], "frequency"), call.maybe(v[6], "presence")};
    const at::Tensor *bias_token = call.maybe(v[7], "bias_token"), *bias_value = call.maybe(v[8], "bias_value");
    const at::Tensor *bias_len = call.maybe(v[9], "bias_len"), *allowed = call.maybe(v[10], "allowed");
    const at::Tensor *active = call.maybe(v[11], "active"), *processed = call.maybe(v[12], "processed"), *given = call.maybe(v[13], "out");
    const int append = PyObject_IsTrue(v[14]);
    if (append < 0) return nullptr;
    const at::ScalarType type = logits.scalar_type();
    NEED(logits.dim() == 2 && logits.size(1) > 0 && (half(type) || type == at::kFloat) && rows_of(logits, logits.size(0)),
         "logits must be fp32, bf16 or fp16 [rows, vocab] with contiguous rows");
    const int64_t rows = logits.size(0), vocab = logits.size(1);
    int64_t history_stride = 0, history_width = 0;
    if (history != nullptr) {
      NEED(prompt_len != nullptr && history_len != nullptr, "a history needs prompt_len and history_len");
      NEED(history->scalar_type() == at::kInt && rows_of(*history, rows) && history->size(1) > 0,
           "history must be int32 [%lld, width] with contiguous rows", static_cast<long long>(rows));
      vector(*prompt_len, "prompt_len", at::kInt, rows);
      vector(*history_len, "history_len", at::kInt, rows);
      history_width = history->size(1);
      history_stride = row_stride(*history, history_width);
    } else {
      NEED(prompt_len == nullptr && history_len == nullptr && append == 0 && penalty[0] == nullptr && penalty[1] == nullptr &&
               penalty[2] == nullptr,
           "penalties, lengths and append need a history");
    }
    static const char *const names[3] = {"repetition", "frequency", "presence"};
    for (int i = 0; i < 3; ++i)
      if (penalty[i] != nullptr) vector(*penalty[i], names[i], at::kFloat, rows);
    int64_t bias_width = 0;
    if (bias_token != nullptr) {
      NEED(bias_value != nullptr && bias_len != nullptr, "a bias list needs bias_value and bias_len");
      NEED(bias_token->scalar_type() == at::kInt && bias_value->scalar_type() == at::kFloat && bias_token->dim() == 2 &&
               bias_token->size(0) == rows && bias_token->size(1) > 0 && bias_token->sizes() == bias_value->sizes() &&
               bias_token->is_contiguous() && bias_value->is_contiguous(),
           "bias_token int32 and bias_value fp32 must be contiguous [%lld, width]", static_cast<long long>(rows));
      vector(*bias_len, "bias_len", at::kInt, rows);
      bias_width = bias_token->size(1);
    } else {
      NEED(bias_value == nullptr && bias_len == nullptr, "bias_value and bias_len need bias_token");
    }
    int64_t allowed_stride = 0;
    if (allowed != nullptr) {
      const int64_t words = (vocab + 31) / 32;
      NEED(allowed->scalar_type() == at::kInt && rows_of(*allowed, rows) && allowed->size(1) == words,
           "allowed must be int32 [%lld, %lld] with contiguous rows", static_cast<long long>(rows), static_cast<long long>(words));
      allowed_stride = row_stride(*allowed, words);
    }
    if (active != nullptr) vector(*active, "active", at::kInt, rows);
    int64_t processed_stride = 0;
    if (processed != nullptr) {
      NEED(processed->scalar_type() == at::kFloat && rows_of(*processed, rows) && processed->size(1) == vocab,
           "processed must be fp32 [%lld, %lld] with contiguous rows", static_cast<long long>(rows), static_cast<long long>(vocab));
      processed_stride = row_stride(*processed, vocab);
    }
    at::Tensor made;
    if (given == nullptr) {
      made = call.empty({rows}, at::kLong);
      given = &made;
    } else {
      vector(*given, "out", at::kLong, rows);
    }
    const int32_t r = small(rows, "rows"), width = small(vocab, "vocab"), hist = small(history_width, "history width");
    const int32_t biases = small(bias_width, "bias width");
    void *const stream = call.stream();
    const int32_t rc = unlocked([&] {
      auto ints = [](const at::Tensor *t) { return static_cast<int32_t *>(pointer(t)); };
      auto floats = [](const at::Tensor *t) { return static_cast<float *>(pointer(t)); };
      return g_entries.choose(logits.data_ptr(), row_stride(logits, vocab), r, width, code(type), ints(active), ints(history),
                              history_stride, hist, ints(prompt_len), ints(history_len), floats(penalty[0]), floats(penalty[1]),
                              floats(penalty[2]), ints(bias_token), floats(bias_value), bias_width, biases, ints(bias_len),
                              static_cast<const uint32_t *>(pointer(allowed)), allowed_stride, floats(processed), processed_stride,
                              static_cast<int64_t *>(given->data_ptr()), append, call.device(), stream);
    });
    if (!done(rc)) return nullptr;
    for (const at::Tensor *t : {given, processed, append != 0 ? history : nullptr}) written(t);
    return answer(v[13], made);
  });
}

// rotate_store, attention, attention_workspace, choose, last_error (addresses), failure
PyObject *bind(PyObject *, PyObject *const *v, Py_ssize_t n) {
  if (!counted(n, 6)) return nullptr;
  void *address[5];
  for (int i = 0; i < 5; ++i) {
    address[i] = PyLong_AsVoidPtr(v[i]);
    if (address[i] == nullptr) {
      if (PyErr_Occurred() == nullptr) PyErr_SetString(PyExc_ValueError, "an entry of the library is NULL");
      return nullptr;
    }
  }
  Py_INCREF(v[5]);
  Py_XDECREF(g_failure);
  g_failure = v[5];
  g_entries = {reinterpret_cast<decltype(Entries::rotate_store)>(address[0]), reinterpret_cast<decltype(Entries::attention)>(address[1]),
               reinterpret_cast<decltype(Entries::attention_workspace)>(address[2]),
               reinterpret_cast<decltype(Entries::choose)>(address[3]), reinterpret_cast<decltype(Entries::last_error)>(address[4])};
  Py_RETURN_NONE;
}

#define FAST(name) reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(name))
PyMethodDef g_methods[] = {
    {"bind", FAST(bind), METH_FASTCALL, "Entry addresses of the library and the exception of its failures."},
    {"rotate_store", FAST(rotate_store), METH_FASTCALL, "See cruise_b200.decoder_ops.rotate_store."},
    {"paged_attention", FAST(paged_attention), METH_FASTCALL, "See cruise_b200.decoder_ops.paged_attention."},
    {"choose", FAST(choose), METH_FASTCALL, "See cruise_b200.decoder_ops.choose."},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_decoder_bind", "Python calls of the decoder operators.", -1, g_methods,
                        nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__decoder_bind(void) { return PyModule_Create(&g_module); }
