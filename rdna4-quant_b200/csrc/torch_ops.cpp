// Python module _r4q_torch: the tensor front end of the paged-cache and
// likelihood operators.  Checks of arguments, output and workspace allocation
// (torch's allocator, on the current stream) and the call of the C ABI in one
// native step: written in Python over ctypes, as the older operators in
// r4q/ops.py are, these took 11 to 20 us a call, several times the kernels of a
// decode step.  The C entry points are handed in by r4q/ops.py, from the library
// that r4q/lib.py has loaded.
//
// Every function returns its result, or the C entry point's negative status as
// an int; wrong arguments raise ValueError or TypeError.
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/object_ptr.h>

#include <algorithm>
#include <climits>
#include <vector>

#include "../../include/r4q.h"

namespace {

using at::Tensor;

struct Api {
  decltype(&r4q_paged_kv_write) write;
  decltype(&r4q_paged_flash_decode) attn;
  decltype(&r4q_paged_flash_decode_workspace_bytes) attn_ws;
  decltype(&r4q_kv_copy_pages) copy;
  decltype(&r4q_kv_table_set) table;
  decltype(&r4q_token_logprobs) logprobs;
} api{};

// ------------------------------------------------------------------ arguments
Tensor tensor(PyObject* o, const char* name) {
  TORCH_CHECK_TYPE(THPVariable_Check(o), name, " must be a tensor");
  return THPVariable_Unpack(o);
}
Tensor optional(PyObject* o, const char* name) { return o == Py_None ? Tensor() : tensor(o, name); }

// The one GPU that holds every given tensor.
struct Gpu {
  int index = -1;
  void add(const Tensor& t) {
    if (!t.defined()) return;
    TORCH_CHECK_VALUE(t.is_cuda(), "r4q ops take CUDA tensors only (no CPU fallback)");
    TORCH_CHECK_VALUE(index < 0 || t.get_device() == index, "all tensors must be on the same CUDA device");
    index = t.get_device();
  }
  template <typename... T>
  explicit Gpu(const T&... t) { (add(t), ...); }
};

void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

// fp16 [rows, heads, 128] with the heads of a row side by side; an input laid out otherwise is copied, an output refused.
struct Heads {
  Tensor t;
  int64_t rows = 0, heads = 0, ld = 0;
  Heads() = default;
  Heads(const Tensor& x, const char* name, int64_t want_rows, int64_t want_heads, bool out) : t(x) {
    TORCH_CHECK_TYPE(x.scalar_type() == at::kHalf, name, " must be float16");
    TORCH_CHECK_VALUE(x.dim() == 3 && x.size(2) == 128 && (want_rows < 0 || x.size(0) == want_rows) &&
                          (want_heads < 0 || x.size(1) == want_heads),
                      name, " must be fp16 [rows, heads, 128]", want_rows < 0 ? "" : " with the rows of k",
                      want_heads < 0 ? "" : " and the heads of the cache or of q", ", got ", x.sizes());
    rows = x.size(0);
    heads = x.size(1);
    const int64_t width = heads * 128;
    if (x.numel() && (x.stride(2) != 1 || (heads > 1 && x.stride(1) != 128) || (rows > 1 && x.stride(0) < width))) {
      TORCH_CHECK_VALUE(!out, name, " must hold the heads of a row side by side");
      t = x.contiguous();
    }
    ld = rows > 1 ? t.stride(0) : width;
  }
};

Tensor vector(const Tensor& t, const char* name, at::ScalarType type, int64_t n) {
  TORCH_CHECK_VALUE(t.scalar_type() == type && t.dim() == 1 && t.numel() == n, name, " must be ", type, " [", n,
                    "], got ", t.scalar_type(), " ", t.sizes());
  return t.contiguous();
}

int int_size(int64_t n, const char* what) {
  TORCH_CHECK_VALUE(n <= INT_MAX, what, " of ", n);
  return (int)n;
}

struct Cache {
  r4q_paged_cache c{};
  Cache(const Tensor& k, const Tensor& v, const Tensor& table, const Tensor& ks, const Tensor& vs) {
    TORCH_CHECK_TYPE(k.scalar_type() == at::kByte && v.scalar_type() == at::kByte,
                     "pages must be uint8 (FP8 E4M3 bytes)");
    TORCH_CHECK_VALUE(k.dim() == 4 && k.size(3) == 128 && v.sizes() == k.sizes(),
                      "k_pages and v_pages must be [pages, kv heads, page, 128] of one shape, got ", k.sizes(), " and ",
                      v.sizes());
    const int64_t P = k.size(0), Hk = k.size(1), page = k.size(2);
    for (const Tensor* t : {&k, &v})
      TORCH_CHECK_VALUE(t->stride(3) == 1 && (page == 1 || t->stride(2) == 128) &&
                            (Hk == 1 || t->stride(1) == page * 128) && (P <= 1 || t->stride(0) >= Hk * page * 128),
                        "each page must be contiguous [kv heads, page, 128] and lie behind the one before");
    TORCH_CHECK_TYPE(table.scalar_type() == at::kInt && table.dim() == 2,
                     "block_table must be int32 [sequences, blocks]");
    const int64_t S = table.size(0), nb = table.size(1);
    TORCH_CHECK_VALUE(nb <= 1 || table.stride(1) == 1, "block_table rows must be contiguous");
    for (const Tensor* s : {&ks, &vs})
      TORCH_CHECK_VALUE(!s->defined() || (s->scalar_type() == at::kFloat && s->dim() == 1 && s->numel() == Hk &&
                                          s->is_contiguous()),
                        "k_scale and v_scale must be float32 [", Hk, "], one per kv head");
    c.k_pages = k.data_ptr();
    c.v_pages = v.data_ptr();
    c.k_stride = P > 1 ? k.stride(0) : 0;
    c.v_stride = P > 1 ? v.stride(0) : 0;
    c.n_pages = int_size(P, "pages");
    c.page = int_size(page, "page");
    c.Hk = int_size(Hk, "kv heads");
    c.table = table.data_ptr<int>();
    c.ld_table = S > 1 ? table.stride(0) : nb;
    c.seqs = int_size(S, "sequences");
    c.max_blocks = int_size(nb, "blocks");
    c.k_scale = (const float*)ptr(ks);
    c.v_scale = (const float*)ptr(vs);
  }
};

// Host integers: a sequence, an array or a CPU tensor.
std::vector<int> host_ints(PyObject* o, const char* name) {
  std::vector<int> out;
  const auto put = [&](long long v) {
    TORCH_CHECK_VALUE(v >= INT_MIN && v <= INT_MAX, name, ": ", v, " is no 32-bit integer");
    out.push_back((int)v);
  };
  if (THPVariable_Check(o)) {
    const Tensor& t = THPVariable_Unpack(o);
    TORCH_CHECK_VALUE(!t.is_cuda(), name, " is host data: a list or a CPU tensor");
    TORCH_CHECK_TYPE(t.dim() == 1 && at::isIntegralType(t.scalar_type(), false), name, " must hold integers");
    const Tensor l = t.to(at::kLong).contiguous();
    for (int64_t i = 0; i < l.numel(); ++i) put(l.data_ptr<int64_t>()[i]);
    return out;
  }
  THPObjectPtr seq(PySequence_Fast(o, name));
  if (!seq) throw python_error();
  out.reserve(PySequence_Fast_GET_SIZE(seq.get()));
  for (Py_ssize_t i = 0; i < PySequence_Fast_GET_SIZE(seq.get()); ++i) {     // an item's __index__ may change the list
    PyObject* item = PySequence_Fast_GET_ITEM(seq.get(), i);
    Py_INCREF(item);
    const THPObjectPtr held(item);
    const long long v = PyLong_AsLongLong(item);
    if (v == -1 && PyErr_Occurred()) {
      if (!PyErr_ExceptionMatches(PyExc_OverflowError)) throw python_error();
      PyErr_Clear();
      TORCH_CHECK_VALUE(false, name, " must hold 32-bit integers");
    }
    put(v);
  }
  return out;
}

// Calls f(stream) with the GPU current and the interpreter free for other threads.
template <typename F>
int on(const Gpu& gpu, F f) {
  c10::cuda::OptionalCUDAGuard guard;
  if (c10::cuda::current_device() != gpu.index) guard.set_index(gpu.index);
  const cudaStream_t stream = c10::cuda::getCurrentCUDAStream(gpu.index).stream();
  int st;
  Py_BEGIN_ALLOW_THREADS
  st = f(stream);
  Py_END_ALLOW_THREADS
  return st;
}

PyObject* result(int st, const Tensor& t) {
  if (st) return PyLong_FromLong(st);
  if (t.defined()) return THPVariable_Wrap(t);
  Py_RETURN_NONE;
}

void arity(Py_ssize_t got, Py_ssize_t want) { TORCH_CHECK_TYPE(got == want, "takes ", want, " arguments, got ", got); }

// ------------------------------------------------------------------- operators
// k, v, k_pages, v_pages, block_table, positions, rows, q, q_w, k_w, cos, sin, q_out, k_out, k_scale, v_scale, eps, flags
PyObject* paged_kv_write(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  arity(n_args, 18);
  const Tensor k_ = tensor(a[0], "k"), v_ = tensor(a[1], "v"), kp = tensor(a[2], "k_pages"), vp = tensor(a[3], "v_pages"),
               table = tensor(a[4], "block_table");
  Tensor pos = tensor(a[5], "positions"), rows = optional(a[6], "rows");
  const Tensor q_ = optional(a[7], "q"), q_w = optional(a[8], "q_w"), k_w = optional(a[9], "k_w"),
               cos = optional(a[10], "cos"), sin = optional(a[11], "sin"), q_out_ = optional(a[12], "q_out"),
               k_out_ = optional(a[13], "k_out"), ks = optional(a[14], "k_scale"), vs = optional(a[15], "v_scale");
  const double eps = PyFloat_AsDouble(a[16]);
  if (eps == -1.0 && PyErr_Occurred()) throw python_error();
  int flags = (int)PyLong_AsLong(a[17]);
  const Cache cache(kp, vp, table, ks, vs);
  const Gpu gpu(k_, v_, kp, vp, table, pos, rows, q_, q_w, k_w, cos, sin, q_out_, k_out_, ks, vs);
  const Heads k(k_, "k", -1, cache.c.Hk, false), v(v_, "v", k.rows, cache.c.Hk, false);
  pos = vector(pos, "positions", at::kLong, k.rows);
  if (rows.defined()) rows = vector(rows, "rows", at::kInt, k.rows);
  Heads q, q_out, k_out;
  if (q_.defined()) {
    q = Heads(q_, "q", k.rows, -1, false);
    q_out = Heads(q_out_.defined() ? q_out_ : at::empty({q.rows, q.heads, 128}, q_.options()), "q_out", k.rows, q.heads,
                  true);
  } else {
    TORCH_CHECK_VALUE(!q_out_.defined() && !q_w.defined(), "q_out and q_w need q");
  }
  if (k_out_.defined()) k_out = Heads(k_out_, "k_out", k.rows, cache.c.Hk, true);
  if (k_w.defined() || q_w.defined()) {
    TORCH_CHECK_VALUE(k_w.defined() && q_w.defined() == q_.defined(), "the norm needs a weight for q and for k");
    for (const Tensor* w : {&q_w, &k_w})
      TORCH_CHECK_VALUE(!w->defined() || (w->scalar_type() == at::kHalf && w->dim() == 1 && w->numel() == 128 &&
                                          w->is_contiguous()),
                        "norm weights must be float16 [128]");
    flags |= R4Q_HEAD_NORM;
  }
  int64_t tab_stride = 0, tab_rows = 0;
  if (cos.defined() || sin.defined()) {
    TORCH_CHECK_VALUE(cos.defined() && sin.defined() && cos.scalar_type() == at::kHalf &&
                          sin.scalar_type() == at::kHalf && cos.dim() == 2 && cos.size(1) >= 64 &&
                          cos.stride(1) == 1 && sin.sizes() == cos.sizes() && sin.strides() == cos.strides(),
                      "cos and sin must be float16 [rows, 64] of one layout");
    flags |= R4Q_HEAD_ROPE;
    tab_rows = cos.size(0);
    tab_stride = tab_rows > 1 ? cos.stride(0) : cos.size(1);
  }
  const int M = int_size(k.rows, "tokens"), H = int_size(q.heads, "heads");
  const int st = on(gpu, [&](cudaStream_t s) {
    return api.write(ptr(q.t), q.ld, ptr(k.t), k.ld, ptr(v.t), v.ld, ptr(q_w), ptr(k_w), ptr(cos), ptr(sin), tab_stride,
                     tab_rows, ptr(q_out.t), q_out.ld, ptr(k_out.t), k_out.ld, &cache.c, (const int*)ptr(rows),
                     (const long long*)ptr(pos), M, H, (float)eps, flags, s);
  });
  return result(st, q_out.t);
  END_HANDLE_TH_ERRORS
}

// q, k_pages, v_pages, block_table, seq_lens, k_scale, v_scale, flags, out
PyObject* paged_flash_decode(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  arity(n_args, 9);
  const Tensor q_ = tensor(a[0], "q"), kp = tensor(a[1], "k_pages"), vp = tensor(a[2], "v_pages"),
               table = tensor(a[3], "block_table");
  Tensor seq = tensor(a[4], "seq_lens");
  const Tensor ks = optional(a[5], "k_scale"), vs = optional(a[6], "v_scale"), out_ = optional(a[8], "out");
  const int flags = (int)PyLong_AsLong(a[7]);
  const Cache cache(kp, vp, table, ks, vs);
  const Gpu gpu(q_, kp, vp, table, seq, ks, vs, out_);
  const Heads q(q_, "q", -1, -1, false);
  seq = vector(seq, "seq_lens", at::kLong, q.rows);
  const Heads out(out_.defined() ? out_ : at::empty({q.rows, q.heads, 128}, q_.options()), "out", q.rows, q.heads, true);
  const int B = int_size(q.rows, "sequences"), H = int_size(q.heads, "heads");
  c10::cuda::OptionalCUDAGuard guard;
  if (c10::cuda::current_device() != gpu.index) guard.set_index(gpu.index);
  const size_t need = api.attn_ws(B, H, cache.c.Hk, cache.c.page, cache.c.max_blocks);
  Tensor ws;
  if (need) ws = at::empty({(int64_t)need}, kp.options());
  const int st = on(gpu, [&](cudaStream_t s) {
    return api.attn(ptr(q.t), q.ld, &cache.c, (const long long*)ptr(seq), ptr(out.t), out.ld, B, H, flags, ptr(ws), need,
                    s);
  });
  return result(st, out.t);
  END_HANDLE_TH_ERRORS
}

// pool, src, dst
PyObject* kv_copy_pages(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  arity(n_args, 3);
  const Tensor pool = tensor(a[0], "pool");
  const Gpu gpu(pool);
  TORCH_CHECK_VALUE(pool.scalar_type() == at::kByte && pool.dim() >= 4 && pool.is_contiguous() && pool.numel(),
                    "pool must be uint8 [..., pages, kv heads, page, 128], contiguous and not empty");
  const std::vector<int> src = host_ints(a[1], "src"), dst = host_ints(a[2], "dst");
  TORCH_CHECK_VALUE(src.size() == dst.size(), "src and dst must have one length");
  const int64_t page = pool.size(-3) * pool.size(-2) * pool.size(-1), P = pool.size(-4), outer = pool.numel() / (P * page);
  const int pages = int_size(P, "pages"), n = int_size((int64_t)src.size(), "moves");
  return result(on(gpu, [&](cudaStream_t s) {
                  return api.copy(pool.data_ptr(), outer, P * page, page, page, pages, src.data(), dst.data(), n, s);
                }), Tensor());
  END_HANDLE_TH_ERRORS
}

// table, rows, cols, values
PyObject* kv_table_set(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  arity(n_args, 4);
  const Tensor table = tensor(a[0], "table");
  const Gpu gpu(table);
  TORCH_CHECK_VALUE(table.scalar_type() == at::kInt && table.dim() == 2 &&
                        (table.size(1) <= 1 || table.stride(1) == 1),
                    "table must be int32 [sequences, blocks] with contiguous rows");
  const std::vector<int> r = host_ints(a[1], "rows"), c = host_ints(a[2], "cols"), v = host_ints(a[3], "values");
  TORCH_CHECK_VALUE(r.size() == c.size() && r.size() == v.size(), "rows, cols and values must have one length");
  const int rows = int_size(table.size(0), "rows"), cols = int_size(table.size(1), "columns");
  const int64_t ld = rows > 1 ? table.stride(0) : cols;
  return result(on(gpu, [&](cudaStream_t s) {
                  return api.table((int*)table.data_ptr(), ld, rows, cols, r.data(), c.data(), v.data(), (int)r.size(), s);
                }), Tensor());
  END_HANDLE_TH_ERRORS
}

// logits, tokens, k -> (logprob, rank, entropy, top_ids, top_logprobs)
PyObject* token_logprobs(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  arity(n_args, 3);
  Tensor x = tensor(a[0], "logits"), tokens = optional(a[1], "tokens");
  const long k = PyLong_AsLong(a[2]);
  if (k == -1 && PyErr_Occurred()) throw python_error();
  const Gpu gpu(x, tokens);
  const auto type = x.scalar_type();
  TORCH_CHECK_TYPE(type == at::kHalf || type == at::kBFloat16 || type == at::kFloat,
                   "logits must be float16, bfloat16 or float32, not ", type);
  TORCH_CHECK_VALUE(x.dim() == 2, "logits must be [rows, vocabulary], got ", x.sizes());
  const int M = int_size(x.size(0), "rows"), V = int_size(x.size(1), "vocabulary");
  TORCH_CHECK_VALUE(V >= 1 && k >= 0 && k <= std::min(V, 32), "k must be in [0, ", std::min(V, 32), "], got ", k);
  if ((V > 1 && x.stride(1) != 1) || (M > 1 && x.stride(0) < V)) x = x.contiguous();
  if (tokens.defined()) tokens = vector(tokens, "tokens", at::kLong, M);
  const auto f32 = x.options().dtype(at::kFloat), i64 = x.options().dtype(at::kLong);
  Tensor logprob, rank;
  const Tensor entropy = at::empty({M}, f32), ids = at::empty({M, k}, i64), top = at::empty({M, k}, f32);
  if (tokens.defined()) {
    logprob = at::empty({M}, f32);
    rank = at::empty({M}, i64);
  }
  const int st = on(gpu, [&](cudaStream_t s) {
    return api.logprobs(ptr(x), type == at::kHalf ? R4Q_T_F16 : type == at::kFloat ? R4Q_T_F32 : R4Q_T_BF16,
                        M > 1 ? x.stride(0) : V, (const long long*)ptr(tokens), M, V, (int)k, (float*)ptr(logprob),
                        (long long*)ptr(rank), (float*)ptr(entropy), (long long*)ptr(ids), (float*)ptr(top), s);
  });
  if (st) return PyLong_FromLong(st);
  return PyTuple_Pack(5, THPObjectPtr(result(0, logprob)).get(), THPObjectPtr(result(0, rank)).get(),
                      THPObjectPtr(THPVariable_Wrap(entropy)).get(), THPObjectPtr(THPVariable_Wrap(ids)).get(),
                      THPObjectPtr(THPVariable_Wrap(top)).get());
  END_HANDLE_TH_ERRORS
}

// Addresses of r4q_paged_kv_write, r4q_paged_flash_decode, .._workspace_bytes, r4q_kv_copy_pages, r4q_kv_table_set and
// r4q_token_logprobs
PyObject* bind(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  arity(n_args, 6);
  void* p[6];
  for (int i = 0; i < 6; ++i) {
    p[i] = PyLong_AsVoidPtr(a[i]);
    if (!p[i]) {
      if (PyErr_Occurred()) throw python_error();
      TORCH_CHECK_VALUE(false, "null entry point");
    }
  }
  api.write = (decltype(api.write))p[0];
  api.attn = (decltype(api.attn))p[1];
  api.attn_ws = (decltype(api.attn_ws))p[2];
  api.copy = (decltype(api.copy))p[3];
  api.table = (decltype(api.table))p[4];
  api.logprobs = (decltype(api.logprobs))p[5];
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

#define R4Q_METHOD(name) {#name, (PyCFunction)(void (*)(void))name, METH_FASTCALL, nullptr}
PyMethodDef methods[] = {R4Q_METHOD(bind), R4Q_METHOD(paged_kv_write), R4Q_METHOD(paged_flash_decode),
                         R4Q_METHOD(kv_copy_pages), R4Q_METHOD(kv_table_set), R4Q_METHOD(token_logprobs),
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_r4q_torch", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__r4q_torch() { return PyModule_Create(&module); }
