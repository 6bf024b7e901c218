// Native front-end of the serving operators: argument checks, output allocation
// and the call into libalgx, in one step from Python.
//
// A decode step makes these calls once a layer on tensors of a few kilobytes, so
// the host's time is the call's. Through ctypes a call of 25 arguments costs 2 us
// before the library sees it, the checks and allocations in Python some 8 more;
// here all of it is about 2 us beside the launches. The module binds to the
// library's C ABI by the addresses that algx._lib hands it (bind), so both share
// one loaded libalgx.so.
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <array>
#include <stdexcept>
#include <string>

#include "algx.h"

namespace {

using at::Tensor;

PyObject* g_error = nullptr;  // algx._lib.AlgxError
decltype(&algx_cache_append) g_append = nullptr;
decltype(&algx_paged_attn) g_attn = nullptr;
decltype(&algx_paged_attn_workspace_size) g_attn_ws = nullptr;
decltype(&algx_cache_evict) g_evict = nullptr;
decltype(&algx_cache_evict_workspace_size) g_evict_ws = nullptr;
decltype(&algx_verify_draft) g_verify = nullptr;
decltype(&algx_last_error) g_last_error = nullptr;

struct LibError : std::runtime_error {  // raised as AlgxError
  using std::runtime_error::runtime_error;
};

[[noreturn]] void bad(const std::string& msg) { throw std::invalid_argument(msg); }
void need(bool ok, const char* msg) {
  if (!ok) bad(msg);
}

std::string text(at::IntArrayRef s) {
  std::string r = "(";
  for (size_t i = 0; i < s.size(); ++i) r += (i ? ", " : "") + std::to_string(s[i]);
  return r + (s.size() == 1 ? ",)" : ")");
}

void check(int status, const char* what) {
  if (status == ALGX_OK) return;
  const char* kind = status == ALGX_ERR_INVALID ? "invalid argument" : status == ALGX_ERR_UNSUPPORTED ? "unsupported" : "CUDA error";
  throw LibError(std::string(what) + ": " + kind + ": " + g_last_error());
}

// ------------------------------------------------------------------ arguments
struct Args {
  PyObject* const* at;
  Py_ssize_t count, next = 0;
  PyObject* take() {
    if (next >= count) throw std::runtime_error("too few arguments");
    return at[next++];
  }
  const Tensor& tensor(const char* name) {
    PyObject* o = take();
    if (!THPVariable_Check(o)) bad(std::string(name) + " must be a tensor");
    return THPVariable_Unpack(o);
  }
  const Tensor* maybe(const char* name) {
    if (next < count && at[next] == Py_None) {
      ++next;
      return nullptr;
    }
    return &tensor(name);
  }
  int64_t integer() {
    const long long v = PyLong_AsLongLong(take());
    if (v == -1 && PyErr_Occurred()) throw std::logic_error("");
    return v;
  }
  double number() {
    const double v = PyFloat_AsDouble(take());
    if (v == -1.0 && PyErr_Occurred()) throw std::logic_error("");
    return v;
  }
};

int io_code(at::ScalarType t) {
  return t == at::kBFloat16 ? ALGX_BF16 : t == at::kFloat ? ALGX_F32 : -1;
}

// One device for all, a CUDA one.
void same_device(const Tensor& ref, std::initializer_list<const Tensor*> others) {
  auto cuda_only = [](const Tensor& t) {
    if (!t.is_cuda())
      throw LibError("algx kernels run on CUDA tensors only (no CPU fallback); got a tensor on " + t.device().str());
  };
  for (const Tensor* t : others)
    if (t && t->device() != ref.device()) {
      cuda_only(ref);
      cuda_only(*t);
      bad("tensors on " + ref.device().str() + " and " + t->device().str() + " in one call");
    }
  cuda_only(ref);
}

// Contiguous at a 16-byte boundary, as the kernels load it (a copy where it is not).
Tensor ready(const Tensor& t) {
  Tensor c = t.contiguous();
  return (reinterpret_cast<uintptr_t>(c.data_ptr()) & 15) == 0 ? c : c.clone();
}

void* ptr(const Tensor& t) { return t.data_ptr(); }
void* ptr(const Tensor* t) { return t ? t->data_ptr() : nullptr; }
const int32_t* ints(const Tensor& t) { return static_cast<const int32_t*>(t.data_ptr()); }

void* stream_of(const Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.device().index()).stream(); }

struct Cache {
  int64_t num, heads, size, B, max_pages;
  int code;
};

Cache check_cache(const Tensor& k, const Tensor& v, const Tensor& table, const Tensor& lens) {
  if (k.dim() != 4 || !k.sizes().equals(v.sizes()) || k.scalar_type() != v.scalar_type())
    bad("k_pages and v_pages must both have shape (num_pages, heads, page_size, 64) and one dtype");
  Cache c = {k.size(0), k.size(1), k.size(2), 0, 0, io_code(k.scalar_type())};
  if (k.size(3) != 64) bad("algx paged cache supports head_dim 64, got " + std::to_string(k.size(3)));
  need(c.code >= 0, "paged cache must be bfloat16 or float32");
  if (c.size < 16 || c.size > 256 || (c.size & (c.size - 1)))
    bad("page_size must be a power of two from 16 to 256, got " + std::to_string(c.size));
  need(c.num >= 1 && c.heads >= 1, "paged cache has no pages or no heads");
  need(k.is_contiguous() && v.is_contiguous(), "k_pages and v_pages must be contiguous");
  need(table.dim() == 2 && lens.dim() == 1 && lens.size(0) == table.size(0) && table.size(1) >= 1,
       "table must have shape (B, max_pages) and lens (B,)");
  need(table.scalar_type() == at::kInt && lens.scalar_type() == at::kInt, "table and lens must be int32");
  c.B = table.size(0);
  c.max_pages = table.size(1);
  return c;
}

void check_state(const char* name, const Tensor& t, std::initializer_list<int64_t> shape, at::ScalarType type) {
  if (!t.sizes().equals(at::IntArrayRef(shape)) || t.scalar_type() != type || !t.is_contiguous())
    bad(std::string(name) + " must be a contiguous " + (type == at::kFloat ? "float32" : "int32") + " tensor of shape " +
        text(at::IntArrayRef(shape)));
}

void check_vector(const char* name, const Tensor* t, int64_t B) {
  if (t && (t->dim() != 1 || t->size(0) != B || t->scalar_type() != at::kInt))
    bad(std::string(name) + " must be int32 of shape (" + std::to_string(B) + ",)");
}

Tensor workspace(size_t bytes, const Tensor& like) {
  return at::empty({(int64_t)(bytes ? bytes : 1)}, like.options().dtype(at::kByte));
}

// Where the program has other Python threads, allocations and launches run without
// the interpreter's lock, as torch's own calls do: a launch waits while the stream's
// queue is full. (One token into the cache: 6.9 us a pass with the lock handed back
// and taken again, 6.3 without, which is what a program of one thread pays.)
struct Unlocked {
  PyThreadState* state = nullptr;
  Unlocked() {
    PyThreadState* head = PyInterpreterState_ThreadHead(PyInterpreterState_Get());
    if (head && PyThreadState_Next(head)) state = PyEval_SaveThread();
  }
  ~Unlocked() {
    if (state) PyEval_RestoreThread(state);
  }
  Unlocked(const Unlocked&) = delete;
};

// ------------------------------------------------------------------ operators
Tensor append(Args& in) {
  const Tensor &qkv = in.tensor("qkv"), &k = in.tensor("k_pages"), &v = in.tensor("v_pages"), &table = in.tensor("table"),
               &lens = in.tensor("lens");
  const Tensor *gq = in.maybe("gain_q"), *gk = in.maybe("gain_k"), *cos = in.maybe("cos"), *sin = in.maybe("sin");
  const Tensor *positions = in.maybe("positions"), *counts = in.maybe("counts"), *where = in.maybe("slot_positions");
  const double eps = in.number();
  const Cache c = check_cache(k, v, table, lens);
  if (qkv.dim() != 4 || qkv.size(0) != c.B || qkv.size(3) != 64 || qkv.size(2) < 2 * c.heads)
    bad("qkv must have shape (" + std::to_string(c.B) + ", T, Hq + " + std::to_string(2 * c.heads) + ", 64), got " +
        text(qkv.sizes()));
  need(qkv.scalar_type() == k.scalar_type(), "qkv and the cache must share one dtype");
  need((gq == nullptr) == (gk == nullptr), "give both gain_q and gain_k or neither");
  need(eps > 0, "eps must be positive");
  for (const Tensor* g : {gq, gk})
    need(!g || (g->dim() == 1 && g->size(0) == 64 && g->scalar_type() == at::kFloat), "gains must be float32 of shape (64,)");
  if (cos)
    need(sin && cos->dim() == 2 && cos->size(0) >= 1 && cos->size(1) == 32 && cos->sizes().equals(sin->sizes()) &&
             cos->scalar_type() == at::kFloat && sin->scalar_type() == at::kFloat,
         "rotary tables must both be float32 of shape (rows, 32)");
  check_vector("positions", positions, c.B);
  check_vector("counts", counts, c.B);
  if (where) check_state("slot_positions", *where, {c.B, c.heads, c.max_pages * c.size}, at::kInt);
  same_device(qkv, {&k, &v, &table, &lens, gq, gk, cos, sin, positions, counts, where});
  Unlocked unlocked;
  c10::cuda::CUDAGuard guard(qkv.device());
  const Tensor x = ready(qkv), tb = table.contiguous(), ln = lens.contiguous();
  Tensor g[2], r[2], pos, cnt;
  if (gq) g[0] = ready(*gq), g[1] = ready(*gk);
  if (cos) r[0] = ready(*cos), r[1] = ready(*sin);
  if (positions) pos = positions->contiguous();
  if (counts) cnt = counts->contiguous();
  const int64_t T = x.size(1), Hq = x.size(2) - 2 * c.heads;
  Tensor q = at::empty({c.B, T, Hq, 64}, x.options());
  auto f = [](const Tensor& t) { return t.defined() ? static_cast<const float*>(t.data_ptr()) : nullptr; };
  auto i = [](const Tensor& t) { return t.defined() ? static_cast<const int32_t*>(t.data_ptr()) : nullptr; };
  check(g_append(ptr(x), f(g[0]), f(g[1]), f(r[0]), f(r[1]), cos ? cos->size(0) : 0, ints(tb), ints(ln), i(pos), i(cnt),
                 ptr(q), ptr(k), ptr(v), static_cast<int32_t*>(ptr(where)), c.B, T, Hq, c.heads, c.num, c.size,
                 c.max_pages, 64, c.code, (float)eps, stream_of(x)),
        "algx_cache_append");
  return q;
}

Tensor attend(Args& in) {
  const Tensor &q = in.tensor("q"), &k = in.tensor("k_pages"), &v = in.tensor("v_pages"), &table = in.tensor("table"),
               &lens = in.tensor("lens");
  const Tensor *sink = in.maybe("sink_logit"), *scores = in.maybe("scores"), *out = in.maybe("scores_out");
  algx_paged_config cfg;
  cfg.kind = (int32_t)in.integer();
  cfg.n = (int32_t)in.integer();
  cfg.window = (int32_t)in.integer();
  cfg.first = (int32_t)in.integer();
  cfg.scale = (float)in.number();
  cfg.inv_unit = (float)in.number();
  const Cache c = check_cache(k, v, table, lens);
  if (q.dim() != 4 || q.size(0) != c.B || q.size(3) != 64 || q.size(2) < 1 || q.size(2) % c.heads)
    bad("q must have shape (" + std::to_string(c.B) + ", T, Hq, 64) with Hq a multiple of " + std::to_string(c.heads) +
        ", got " + text(q.sizes()));
  need(q.scalar_type() == k.scalar_type(), "q and the cache must share one dtype");
  const int64_t T = q.size(1), Hq = q.size(2), S = c.max_pages * c.size;
  if (scores) {
    check_state("scores", *scores, {c.B, c.heads, S}, at::kFloat);
    check_state("scores_out", *out, {c.B, c.heads, S}, at::kFloat);
  }
  same_device(q, {&k, &v, &table, &lens, scores, out});
  Unlocked unlocked;
  c10::cuda::CUDAGuard guard(q.device());
  Tensor s;
  if (sink) {
    s = *sink;
    if (s.dim() != 1 || s.size(0) != Hq || s.scalar_type() != at::kFloat || s.device() != q.device())
      s = s.to(q.device(), at::kFloat).reshape({-1}).expand({Hq});
    s = s.contiguous();
  }
  const Tensor x = ready(q), tb = table.contiguous(), ln = lens.contiguous();
  Tensor o = at::empty({c.B, T, Hq, 64}, x.options());
  const size_t bytes = g_attn_ws(c.B, T, Hq, c.heads, c.size, c.max_pages, scores != nullptr, c.code);
  Tensor ws = workspace(bytes, x);
  check(g_attn(&cfg, ptr(x), ptr(k), ptr(v), ints(tb), ints(ln), s.defined() ? static_cast<const float*>(ptr(s)) : nullptr,
               static_cast<const float*>(ptr(scores)), static_cast<float*>(ptr(out)), ptr(o), c.B, T, Hq, c.heads, c.num,
               c.size, c.max_pages, 64, c.code, ptr(ws), bytes, stream_of(x)),
        "algx_paged_attn");
  return o;
}

std::array<Tensor, 4> evict(Args& in) {
  const Tensor &k = in.tensor("k_pages"), &v = in.tensor("v_pages"), &table = in.tensor("table"), &lens = in.tensor("lens"),
               &scores = in.tensor("scores"), &positions = in.tensor("positions");
  const int64_t budget = in.integer(), first = in.integer(), recent = in.integer();
  const Cache c = check_cache(k, v, table, lens);
  need(budget >= 1 && budget < (int64_t)1 << 31, "budget must be positive");
  need(first >= 0 && recent >= 0 && first <= budget && recent <= budget - first,
       "first and recent must not be negative and must fit the budget together");
  check_state("scores", scores, {c.B, c.heads, c.max_pages * c.size}, at::kFloat);
  check_state("positions", positions, {c.B, c.heads, c.max_pages * c.size}, at::kInt);
  same_device(k, {&v, &table, &lens, &scores, &positions});
  Unlocked unlocked;
  c10::cuda::CUDAGuard guard(k.device());
  const Tensor tb = table.contiguous(), ln = lens.contiguous(), sc = ready(scores), po = ready(positions);
  Tensor new_lens = at::empty({c.B}, ln.options());
  Tensor new_scores = at::empty(sc.sizes(), sc.options()), new_positions = at::empty(po.sizes(), po.options());
  Tensor kept = at::empty({c.B, c.heads, budget}, po.options());
  const size_t bytes = g_evict_ws(c.B, c.heads, budget);
  Tensor ws = workspace(bytes, k);
  check(g_evict(ptr(k), ptr(v), ints(tb), ints(ln), static_cast<const float*>(ptr(sc)), ints(po), budget, first, recent,
                static_cast<int32_t*>(ptr(new_lens)), static_cast<float*>(ptr(new_scores)),
                static_cast<int32_t*>(ptr(new_positions)), static_cast<int32_t*>(ptr(kept)), c.B, c.heads, c.num, c.size,
                c.max_pages, 64, c.code, ptr(ws), bytes, stream_of(k)),
        "algx_cache_evict");
  return {new_lens, new_scores, new_positions, kept};
}

std::array<Tensor, 2> verify(Args& in) {
  const Tensor &target = in.tensor("target_logits"), &tokens = in.tensor("draft_tokens");
  const Tensor* draft = in.maybe("draft_logits");
  const Tensor &u = in.tensor("accept_u"), &race = in.tensor("race");
  const Tensor* counts = in.maybe("counts");
  const int64_t kind = in.integer(), n = in.integer();
  const double scale = in.number();
  if (target.dim() != 3 || target.size(1) < 1 || target.size(2) < 1)
    bad("target_logits must have shape (B, K + 1, V), got " + text(target.sizes()));
  const int64_t B = target.size(0), K = target.size(1) - 1, V = target.size(2);
  need(K <= 31, "at most 31 drafted tokens");
  const int code = io_code(target.scalar_type());
  need(code >= 0, "logits must be bfloat16 or float32");
  auto shaped = [](const Tensor& t, std::initializer_list<int64_t> s, at::ScalarType type) {
    return t.sizes().equals(at::IntArrayRef(s)) && t.scalar_type() == type;
  };
  if (draft && !shaped(*draft, {B, K, V}, target.scalar_type()))
    bad("draft_logits must have shape " + text({B, K, V}) + " and target_logits' dtype");
  if (!shaped(tokens, {B, K}, at::kInt)) bad("draft_tokens must be int32 of shape " + text({B, K}));
  if (!shaped(u, {B, K}, at::kFloat)) bad("accept_u must be float32 of shape " + text({B, K}));
  if (!shaped(race, {B, V}, at::kFloat)) bad("race must be float32 of shape " + text({B, V}));
  check_vector("counts", counts, B);
  same_device(target, {draft, &tokens, &u, &race, counts});
  Unlocked unlocked;
  c10::cuda::CUDAGuard guard(target.device());
  const Tensor t = target.contiguous(), tk = tokens.contiguous(), uu = u.contiguous(), rr = race.contiguous();
  Tensor d, cn;
  if (draft) d = draft->contiguous();
  if (counts) cn = counts->contiguous();
  Tensor out = at::empty({B, K + 1}, tk.options()), accepted = at::empty({B}, tk.options());
  check(g_verify((int32_t)kind, (int32_t)n, (float)scale, ptr(t), draft ? ptr(d) : nullptr, ints(tk),
                 counts ? ints(cn) : nullptr, static_cast<const float*>(ptr(uu)), static_cast<const float*>(ptr(rr)),
                 static_cast<int32_t*>(ptr(out)), static_cast<int32_t*>(ptr(accepted)), B, K, V, code, stream_of(t)),
        "algx_verify_draft");
  return {out, accepted};
}

// ------------------------------------------------------------------ the module
template <typename F>
PyObject* guarded(PyObject* const* args, Py_ssize_t n, F f) {
  try {
    Args in{args, n};
    return f(in);
  } catch (const std::invalid_argument& e) {
    PyErr_SetString(PyExc_ValueError, e.what());
  } catch (const LibError& e) {
    PyErr_SetString(g_error ? g_error : PyExc_RuntimeError, e.what());
  } catch (const std::logic_error&) {
    if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, "invalid argument");
  } catch (const c10::OutOfMemoryError& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what_without_backtrace());
  } catch (const c10::Error& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what_without_backtrace());
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  }
  return nullptr;
}

PyObject* py_append(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(a, n, [](Args& in) { return THPVariable_Wrap(append(in)); });
}
PyObject* py_attend(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(a, n, [](Args& in) { return THPVariable_Wrap(attend(in)); });
}
PyObject* py_evict(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(a, n, [](Args& in) {
    const auto t = evict(in);
    return Py_BuildValue("(NNNN)", THPVariable_Wrap(t[0]), THPVariable_Wrap(t[1]), THPVariable_Wrap(t[2]),
                         THPVariable_Wrap(t[3]));
  });
}
PyObject* py_verify(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(a, n, [](Args& in) {
    const auto t = verify(in);
    return Py_BuildValue("(NN)", THPVariable_Wrap(t[0]), THPVariable_Wrap(t[1]));
  });
}

// bind(AlgxError, {name: address})
PyObject* py_bind(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 2 || !PyDict_Check(a[1])) {
    PyErr_SetString(PyExc_TypeError, "bind(error class, {name: address})");
    return nullptr;
  }
  auto find = [&](const char* name, auto& fn) {
    PyObject* v = PyDict_GetItemString(a[1], name);
    void* p = v ? PyLong_AsVoidPtr(v) : nullptr;
    if (!p) {
      PyErr_Format(PyExc_RuntimeError, "no address for %s", name);
      return false;
    }
    fn = reinterpret_cast<std::remove_reference_t<decltype(fn)>>(p);
    return true;
  };
  if (!find("algx_cache_append", g_append) || !find("algx_paged_attn", g_attn) ||
      !find("algx_paged_attn_workspace_size", g_attn_ws) || !find("algx_cache_evict", g_evict) ||
      !find("algx_cache_evict_workspace_size", g_evict_ws) || !find("algx_verify_draft", g_verify) ||
      !find("algx_last_error", g_last_error))
    return nullptr;
  Py_INCREF(a[0]);
  Py_XDECREF(g_error);
  g_error = a[0];
  Py_RETURN_NONE;
}

#define ALGX_METHOD(name, fn, doc) {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(fn)), METH_FASTCALL, doc}
PyMethodDef kMethods[] = {
    ALGX_METHOD("bind", py_bind, "bind(error, {name: address}): the library's entries"),
    ALGX_METHOD("cache_append", py_append, "algx.kernels.paged.cache_append"),
    ALGX_METHOD("paged_attention", py_attend, "algx.kernels.paged.paged_attention"),
    ALGX_METHOD("cache_evict", py_evict, "algx.kernels.paged.cache_evict"),
    ALGX_METHOD("verify_draft", py_verify, "algx.kernels.verify.verify_draft"),
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_native", "Native front-end of the serving operators.", -1, kMethods,
                       nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__native(void) { return PyModule_Create(&kModule); }
