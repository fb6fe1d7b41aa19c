// CPython binding of the paged-cache and draft-verification calls: checks the tensors and calls the C ABI
// (include/b200decode.h) through the function addresses that b200kernels/_lib.py took from libb200decode.so.
//
// These calls take few microseconds on the GPU, where the same checks in Python and the ctypes conversion of
// 25 to 35 arguments took 15: a decode step that is not captured in a graph would wait for them. Every
// function takes positional arguments only (the Python wrappers hold the signatures), raises ValueError or
// TypeError for what it refuses, and returns an int status where the C ABI refused the call.
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <sstream>
#include <stdexcept>
#include <string>

#include "b200decode.h"

namespace {

decltype(&b2d_paged_rope_append) g_append = nullptr;
decltype(&b2d_paged_attention_workspace_bytes) g_workspace = nullptr;
decltype(&b2d_paged_attention) g_attention = nullptr;
decltype(&b2d_verify_drafts) g_verify = nullptr;

struct TypeErr : std::runtime_error { using std::runtime_error::runtime_error; };
struct ValueErr : std::runtime_error { using std::runtime_error::runtime_error; };
struct PyErr : std::exception {};   // a Python error is already set

std::string show(const at::Tensor& t) {
  std::ostringstream s;
  s << t.scalar_type() << " " << t.sizes() << " strides " << t.strides() << " on " << t.device();
  return s.str();
}
[[noreturn]] void bad_value(const std::string& what) { throw ValueErr(what); }

const at::Tensor& tensor(PyObject* o, const char* name) {
  if (!THPVariable_Check(o)) throw TypeErr(std::string(name) + " is a tensor, got " + Py_TYPE(o)->tp_name);
  return THPVariable_Unpack(o);
}
const at::Tensor* optional(PyObject* o, const char* name) { return o == Py_None ? nullptr : &tensor(o, name); }
int64_t integer(PyObject* o) {
  const int64_t v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw PyErr();
  return v;
}
int integer32(PyObject* o, const char* name) {
  const int64_t v = integer(o);
  if (v < INT32_MIN || v > INT32_MAX) bad_value(std::string(name) + " is out of range");
  return static_cast<int>(v);
}
double number(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw PyErr();
  return v;
}
const b2d_paged_kv* pool(PyObject* o) { return static_cast<const b2d_paged_kv*>(PyLong_AsVoidPtr(o)); }
at::ScalarType pool_dtype(const b2d_paged_kv* kv) { return kv->dtype == B2D_F16 ? at::kHalf : at::kBFloat16; }
int code(at::ScalarType t) { return t == at::kHalf ? B2D_F16 : t == at::kBFloat16 ? B2D_BF16 : B2D_F32; }
const void* ptr(const at::Tensor* t) { return t ? t->const_data_ptr() : nullptr; }
// a contiguous vector of n values
void check_vector(const at::Tensor& t, const char* name, at::ScalarType dtype, int64_t n) {
  if (t.scalar_type() != dtype || t.dim() != 1 || t.size(0) != n || (n > 1 && t.stride(0) != 1)) {
    std::ostringstream s;
    s << name << " is a contiguous " << dtype << " [" << n << "], got " << show(t);
    bad_value(s.str());
  }
}
void check_table(const at::Tensor& t, const char* name, int64_t dim) {
  if (t.scalar_type() != at::kInt || t.dim() != dim || (t.numel() > 0 && t.size(-1) > 1 && t.stride(-1) != 1)) {
    std::ostringstream s;
    s << name << " is int32, " << dim << "-D, contiguous in its last dimension; got " << show(t);
    bad_value(s.str());
  }
}
void check_shape(const at::Tensor& t, const char* name, at::IntArrayRef shape) {
  if (t.sizes() != shape) {
    std::ostringstream s;
    s << name << " is " << shape << ", got " << show(t);
    bad_value(s.str());
  }
}
int narrow(int64_t v, const char* name) {   // a size that the C ABI takes as an int
  if (v > INT32_MAX) bad_value(std::string(name) + " is too large: " + std::to_string(v));
  return static_cast<int>(v);
}
void check_last(const at::Tensor& t, const char* name) {
  if (t.numel() > 0 && t.size(-1) > 1 && t.stride(-1) != 1)
    bad_value(std::string("the last dimension of ") + name + " must be contiguous, got " + show(t));
}
// Whether strides nest: from the smallest on, each is past all that the ones before it span, so that no two
// indices name one element. Every slice, transpose or part of a tensor that does not overlap itself is such.
bool nests(at::IntArrayRef sizes, at::IntArrayRef strides) {
  int64_t order[64], span = 0;   // span: the largest offset so far
  int n = 0;
  for (size_t d = 0; d < sizes.size(); ++d) {
    if (sizes[d] == 0) return true;
    if (sizes[d] == 1) continue;
    int at = n++;
    for (; at > 0 && strides[order[at - 1]] > strides[d]; --at) order[at] = order[at - 1];
    order[at] = d;
  }
  for (int i = 0; i < n; ++i) {
    if (strides[order[i]] <= span) return false;
    span += (sizes[order[i]] - 1) * strides[order[i]];
  }
  return true;
}
// An output that overlaps itself would be written by several blocks at once. (Outputs have at most 4 dimensions.)
void check_output(const at::Tensor& t, const char* name) {
  if (!nests(t.sizes(), t.strides())) bad_value(std::string(name) + " overlaps itself: " + show(t));
}
// The same of the pools that an append writes.
void check_written_pools(const b2d_paged_kv* kv) {
  const int64_t sizes[4] = {kv->num_pages, kv->KVH, kv->page_size, kv->D};
  const int64_t k[4] = {kv->sk_p, kv->sk_h, kv->sk_s, 1}, v[4] = {kv->sv_p, kv->sv_h, kv->sv_s, 1};
  if (!nests(sizes, k) || !nests(sizes, v)) bad_value("the cache's pages overlap one another: an append would write them at once");
  if (kv->k == kv->v && kv->num_pages > 0) bad_value("the cache's keys and values overlap: an append would write both to one memory");
}
void check_device(const at::Tensor* t, const char* name, const at::Device& d) {
  if (t && t->device() != d) {
    std::ostringstream s;
    s << name << " is on " << t->device() << ", not on " << d;
    bad_value(s.str());
  }
}
void check_pool(const at::Device& d, PyObject* index) {   // the cache's device; -1: not a GPU
  if (d.is_cuda() && d.index() != integer(index)) {
    std::ostringstream s;
    s << "q is on " << d << ", the cache on another device";
    bad_value(s.str());
  }
}
void check_cuda(const at::Device& d) {
  if (!d.is_cuda()) {
    std::ostringstream s;
    s << "the tensors are on " << d << "; the kernels run on a CUDA device only";
    bad_value(s.str());
  }
}

// The device of the tensors for the time of a call (the library launches on the current device).
struct OnDevice {
  c10::cuda::OptionalCUDAGuard guard;
  cudaStream_t stream;
  explicit OnDevice(const at::Device& d) {
    if (c10::cuda::current_device() != d.index()) guard.set_device(d);
    stream = c10::cuda::getCurrentCUDAStream(d.index()).stream();
  }
};

template <typename F>
PyObject* guarded(F&& f) {
  try {
    return f();
  } catch (const TypeErr& e) {
    PyErr_SetString(PyExc_TypeError, e.what());
  } catch (const ValueErr& e) {
    PyErr_SetString(PyExc_ValueError, e.what());
  } catch (const PyErr&) {
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  }
  return nullptr;
}
void check_count(Py_ssize_t got, Py_ssize_t want) {
  if (got != want) throw TypeErr("expected " + std::to_string(want) + " arguments, got " + std::to_string(got));
}
PyObject* given(PyObject* o) {
  Py_INCREF(o);
  return o;
}

// (desc, q, k, v, positions, page_table, cos, sin, q_out, seq_ids, q_weight, k_weight, eps, flags, device index)
PyObject* rope_append(PyObject*, PyObject* const* a, Py_ssize_t na) {
  return guarded([&]() -> PyObject* {
    check_count(na, 15);
    const b2d_paged_kv* kv = pool(a[0]);
    const at::Tensor &q = tensor(a[1], "q"), &k = tensor(a[2], "k"), &v = tensor(a[3], "v"),
                     &positions = tensor(a[4], "positions"), &table = tensor(a[5], "page_table"),
                     &cos = tensor(a[6], "cos"), &sin = tensor(a[7], "sin");
    const at::Tensor *seq = optional(a[9], "seq_ids"), *qw = optional(a[10], "q_weight"), *kw = optional(a[11], "k_weight");
    const at::ScalarType dt = pool_dtype(kv);
    if (q.dim() != 3) bad_value("q is [N, H, D], got " + show(q));
    const int64_t N = q.size(0), H = q.size(1), D = q.size(2);
    if (D != kv->D || H % kv->KVH != 0)
      bad_value("q does not fit a cache of " + std::to_string(kv->KVH) + " heads of " + std::to_string(kv->D) + ": " + show(q));
    check_shape(k, "k", {N, kv->KVH, D});
    check_shape(v, "v", {N, kv->KVH, D});
    if (q.scalar_type() != dt || k.scalar_type() != dt || v.scalar_type() != dt)
      throw TypeErr("q, k and v have the cache's dtype, got " + show(q) + ", " + show(k) + ", " + show(v));
    check_vector(positions, "positions", at::kLong, N);
    check_table(table, "page_table", 2);
    const int64_t B = table.size(0);
    if (seq) check_vector(*seq, "seq_ids", at::kInt, N);
    else if (N > 0 && (B == 0 || N % B != 0))
      bad_value(std::to_string(N) + " tokens do not divide over " + std::to_string(B) + " sequences: pass seq_ids");
    if (cos.dim() != 2 || cos.size(1) != D || cos.sizes() != sin.sizes() || cos.strides() != sin.strides())
      bad_value("cos and sin are [S_max, " + std::to_string(D) + "] of one layout, got " + show(cos) + ", " + show(sin));
    check_last(cos, "cos and sin");
    if (cos.scalar_type() != sin.scalar_type() || (cos.scalar_type() != dt && cos.scalar_type() != at::kFloat))
      throw TypeErr("cos and sin are fp32 or have the cache's dtype, got " + show(cos) + ", " + show(sin));
    for (const at::Tensor* w : {qw, kw})
      if (w) check_vector(*w, "q_weight / k_weight", dt, D);
    check_last(q, "q");
    check_last(k, "k");
    check_last(v, "v");
    const at::Device dev = q.device();
    check_device(&k, "k", dev); check_device(&v, "v", dev); check_device(&positions, "positions", dev);
    check_device(&table, "page_table", dev); check_device(&cos, "cos", dev); check_device(&sin, "sin", dev);
    check_device(seq, "seq_ids", dev); check_device(qw, "q_weight", dev); check_device(kw, "k_weight", dev);
    at::Tensor made;
    if (a[8] == Py_None) made = at::empty({N, H, D}, q.options());
    const at::Tensor& out = a[8] == Py_None ? made : tensor(a[8], "q_out");
    if (out.sizes() != q.sizes() || out.scalar_type() != dt) bad_value("q_out has q's shape and dtype, got " + show(out));
    check_last(out, "q_out");
    check_output(out, "q_out");
    check_written_pools(kv);
    check_device(&out, "q_out", dev);
    check_cuda(dev);
    check_pool(dev, a[14]);
    const OnDevice on(dev);
    const int st = g_append(kv, q.const_data_ptr(), q.stride(0), q.stride(1), k.const_data_ptr(), k.stride(0), k.stride(1),
                            v.const_data_ptr(), v.stride(0), v.stride(1), static_cast<const int64_t*>(positions.const_data_ptr()),
                            static_cast<const int32_t*>(ptr(seq)), static_cast<const int32_t*>(table.const_data_ptr()),
                            table.stride(0), narrow(table.size(1), "page_table"), narrow(B, "page_table"), cos.const_data_ptr(),
                            sin.const_data_ptr(), cos.stride(0), narrow(cos.size(0), "cos"), code(cos.scalar_type()),
                            ptr(qw), ptr(kw), static_cast<float>(number(a[12])), out.mutable_data_ptr(), out.stride(0),
                            out.stride(1), narrow(N, "q"), narrow(H, "q"), integer32(a[13], "flags"), on.stream);
    if (st != B2D_OK) return PyLong_FromLong(st);
    return a[8] == Py_None ? THPVariable_Wrap(made) : given(a[8]);
  });
}

at::ScalarType out_type(PyObject* o, at::ScalarType otherwise) {   // torch.dtype or None
  if (o == Py_None) return otherwise;
  if (!THPDtype_Check(o)) throw TypeErr("out_dtype is a torch.dtype");
  return reinterpret_cast<THPDtype*>(o)->scalar_type;
}

// (desc, q, page_table, seqlens, scale, prefix_table, prefix_len, max_len, out, out_dtype, workspace, flags,
// device index)
PyObject* attention(PyObject*, PyObject* const* a, Py_ssize_t na) {
  return guarded([&]() -> PyObject* {
    check_count(na, 13);
    const b2d_paged_kv* kv = pool(a[0]);
    const at::Tensor &q = tensor(a[1], "q"), &table = tensor(a[2], "page_table"), &lens = tensor(a[3], "seqlens");
    const at::ScalarType dt = pool_dtype(kv);
    if (q.dim() != 4) bad_value("q is [B, T, H, D], got " + show(q));
    const int64_t B = q.size(0), T = q.size(1), H = q.size(2), D = q.size(3);
    if (D != kv->D || H % kv->KVH != 0)
      bad_value("q does not fit a cache of " + std::to_string(kv->KVH) + " heads of " + std::to_string(kv->D) + ": " + show(q));
    if (q.scalar_type() != dt) throw TypeErr("q has the cache's dtype, got " + show(q));
    check_table(table, "page_table", 2);
    if (table.size(0) != B) bad_value("page_table has a row per sequence, got " + show(table) + " for " + show(q));
    check_vector(lens, "seqlens", at::kInt, B);
    const int prefix_len = integer32(a[6], "prefix_len"), max_len = integer32(a[7], "max_len");
    const at::Tensor* prefix = nullptr;
    if (prefix_len != 0) {
      prefix = optional(a[5], "prefix_table");
      if (!prefix) bad_value("prefix_len without prefix_table");
      check_table(*prefix, "prefix_table", 1);
      if (prefix_len < 0 || prefix_len > prefix->size(0) * kv->page_size)
        bad_value("prefix_len " + std::to_string(prefix_len) + " is outside the pages of prefix_table: " + show(*prefix));
    }
    const at::Device dev = q.device();
    const at::ScalarType ot = out_type(a[9], dt);
    at::Tensor made;
    if (a[8] == Py_None) made = at::empty({B, T, H, D}, q.options().dtype(ot));
    const at::Tensor& out = a[8] == Py_None ? made : tensor(a[8], "out");
    if (out.sizes() != q.sizes() || (a[9] != Py_None && out.scalar_type() != ot) ||
        (out.scalar_type() != dt && out.scalar_type() != at::kFloat))
      bad_value("out has q's shape and is fp32 or of the cache's dtype (and of out_dtype), got " + show(out));
    check_last(q, "q");
    check_last(out, "out");
    check_output(out, "out");
    check_device(&table, "page_table", dev); check_device(&lens, "seqlens", dev); check_device(&out, "out", dev);
    check_device(prefix, "prefix_table", dev);
    const at::Tensor* ws = optional(a[10], "workspace");
    if (ws && !ws->is_contiguous()) bad_value("workspace is contiguous, got " + show(*ws));   // its bytes are counted below
    check_device(ws, "workspace", dev);
    check_cuda(dev);
    check_pool(dev, a[12]);
    const OnDevice on(dev);
    const int per_seq = narrow(table.size(1), "page_table"), b = narrow(B, "q"), tn = narrow(T, "q"), h = narrow(H, "q");
    at::Tensor scratch;
    if (!ws) {
      const size_t n = g_workspace(kv, b, tn, h, per_seq, prefix_len, max_len);
      if (n > 0) scratch = at::empty({static_cast<int64_t>(n)}, q.options().dtype(at::kByte));
      ws = &scratch;
    }
    const bool has = ws->defined() && ws->numel() > 0;
    const double scale = a[4] == Py_None ? 1.0 / std::sqrt(static_cast<double>(D)) : number(a[4]);
    const int st = g_attention(kv, q.const_data_ptr(), q.stride(0), q.stride(1), q.stride(2),
                               static_cast<const int32_t*>(table.const_data_ptr()), table.stride(0), per_seq,
                               static_cast<const int32_t*>(lens.const_data_ptr()), static_cast<const int32_t*>(ptr(prefix)),
                               prefix_len, max_len, b, tn, h,
                               static_cast<float>(scale), out.mutable_data_ptr(), out.stride(0), out.stride(1), out.stride(2),
                               code(out.scalar_type()), has ? ws->mutable_data_ptr() : nullptr,
                               has ? static_cast<size_t>(ws->nbytes()) : 0, integer32(a[11], "flags"), on.stream);
    if (st != B2D_OK) return PyLong_FromLong(st);
    return a[8] == Py_None ? THPVariable_Wrap(made) : given(a[8]);
  });
}

// (desc, q, page_table, prefix_len, max_len) -> scratch for `attention`
PyObject* attention_workspace(PyObject*, PyObject* const* a, Py_ssize_t na) {
  return guarded([&]() -> PyObject* {
    check_count(na, 5);
    const at::Tensor &q = tensor(a[1], "q"), &table = tensor(a[2], "page_table");
    if (q.dim() != 4) bad_value("q is [B, T, H, D], got " + show(q));
    check_table(table, "page_table", 2);
    check_cuda(q.device());
    const OnDevice on(q.device());
    const size_t n = g_workspace(pool(a[0]), narrow(q.size(0), "q"), narrow(q.size(1), "q"), narrow(q.size(2), "q"),
                                 narrow(table.size(1), "page_table"), integer32(a[3], "prefix_len"), integer32(a[4], "max_len"));
    return THPVariable_Wrap(at::empty({static_cast<int64_t>(n)}, q.options().dtype(at::kByte)));
  });
}

// (draft_tokens, target_probs, uniforms, draft_probs, draft_lens, tokens, accepted, flags)
PyObject* verify(PyObject*, PyObject* const* a, Py_ssize_t na) {
  return guarded([&]() -> PyObject* {
    check_count(na, 8);
    const at::Tensor &draft = tensor(a[0], "draft_tokens"), &target = tensor(a[1], "target_probs"), &u = tensor(a[2], "uniforms");
    const at::Tensor *probs = optional(a[3], "draft_probs"), *lens = optional(a[4], "draft_lens");
    if (draft.dim() != 2 || draft.scalar_type() != at::kLong) bad_value("draft_tokens is int64 [B, K], got " + show(draft));
    const int64_t B = draft.size(0), K = draft.size(1);
    if (K > 31) bad_value("at most 31 drafts per sequence, got " + std::to_string(K));
    if (target.dim() != 3 || target.size(0) != B || target.size(1) != K + 1 || target.size(2) == 0 || target.size(2) > INT32_MAX)
      bad_value("target_probs is [B, K + 1, V], got " + show(target) + " for " + show(draft));
    const int64_t V = target.size(2);
    const at::ScalarType dt = target.scalar_type();
    if (dt != at::kFloat && dt != at::kHalf && dt != at::kBFloat16)
      throw TypeErr("target_probs is fp32, fp16 or bf16, got " + show(target));
    check_last(target, "target_probs");
    if (probs) {
      check_shape(*probs, "draft_probs", {B, K, V});
      if (probs->scalar_type() != dt) throw TypeErr("draft_probs has target_probs' dtype, got " + show(*probs));
      check_last(*probs, "draft_probs");
    }
    if (u.scalar_type() != at::kFloat) bad_value("uniforms is fp32, got " + show(u));
    check_shape(u, "uniforms", {B, K + 1});
    if (lens) check_vector(*lens, "draft_lens", at::kInt, B);
    const at::Device dev = target.device();
    at::Tensor made_t, made_a;
    if (a[5] == Py_None) made_t = at::empty({B, K + 1}, target.options().dtype(at::kLong));
    if (a[6] == Py_None) made_a = at::empty({B}, target.options().dtype(at::kInt));
    const at::Tensor& tok = a[5] == Py_None ? made_t : tensor(a[5], "tokens");
    const at::Tensor& acc = a[6] == Py_None ? made_a : tensor(a[6], "accepted");
    if (tok.scalar_type() != at::kLong) bad_value("tokens is int64, got " + show(tok));
    check_shape(tok, "tokens", {B, K + 1});
    check_vector(acc, "accepted", at::kInt, B);
    check_last(draft, "draft_tokens");
    check_last(u, "uniforms");
    check_last(tok, "tokens");
    check_output(tok, "tokens");
    check_device(&draft, "draft_tokens", dev); check_device(probs, "draft_probs", dev); check_device(&u, "uniforms", dev);
    check_device(lens, "draft_lens", dev); check_device(&tok, "tokens", dev); check_device(&acc, "accepted", dev);
    check_cuda(dev);
    const OnDevice on(dev);
    const int st = g_verify(static_cast<const int64_t*>(draft.const_data_ptr()), B > 1 ? draft.stride(0) : K,
                            static_cast<const int32_t*>(ptr(lens)), target.const_data_ptr(), target.stride(0), target.stride(1),
                            ptr(probs), probs ? probs->stride(0) : 0, probs ? probs->stride(1) : 0, code(dt),
                            static_cast<const float*>(u.const_data_ptr()), B > 1 ? u.stride(0) : K + 1,
                            static_cast<int64_t*>(tok.mutable_data_ptr()), B > 1 ? tok.stride(0) : K + 1,
                            static_cast<int32_t*>(acc.mutable_data_ptr()), narrow(B, "draft_tokens"), static_cast<int>(K),
                            static_cast<int>(V), integer32(a[7], "flags"), on.stream);
    if (st != B2D_OK) return PyLong_FromLong(st);
    PyObject* t = a[5] == Py_None ? THPVariable_Wrap(made_t) : given(a[5]);
    PyObject* c = a[6] == Py_None ? THPVariable_Wrap(made_a) : given(a[6]);
    PyObject* r = PyTuple_Pack(2, t, c);
    Py_DECREF(t);
    Py_DECREF(c);
    return r;
  });
}

// build.py looks for this text in the module, b200kernels/_lib.py asks for it before the first call.
const char kBuiltFor[] = "b2d built for " B2D_HOST_TAG;
PyObject* built_for(PyObject*, PyObject* const*, Py_ssize_t) { return PyUnicode_FromString(kBuiltFor); }

// the addresses of the four entry points, in the order of the globals above
PyObject* bind(PyObject*, PyObject* const* a, Py_ssize_t na) {
  return guarded([&]() -> PyObject* {
    check_count(na, 4);
    g_append = reinterpret_cast<decltype(g_append)>(PyLong_AsVoidPtr(a[0]));
    g_workspace = reinterpret_cast<decltype(g_workspace)>(PyLong_AsVoidPtr(a[1]));
    g_attention = reinterpret_cast<decltype(g_attention)>(PyLong_AsVoidPtr(a[2]));
    g_verify = reinterpret_cast<decltype(g_verify)>(PyLong_AsVoidPtr(a[3]));
    if (PyErr_Occurred()) throw PyErr();
    Py_RETURN_NONE;
  });
}

#define FAST(name) reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(name)), METH_FASTCALL, nullptr
PyMethodDef kMethods[] = {{"rope_append", FAST(rope_append)}, {"attention", FAST(attention)},
                          {"attention_workspace", FAST(attention_workspace)}, {"verify", FAST(verify)},
                          {"bind", FAST(bind)}, {"built_for", FAST(built_for)}, {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_binding", nullptr, -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__binding(void) { return PyModule_Create(&kModule); }
