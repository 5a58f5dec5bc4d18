// The entry points of a token step's kernels as Python functions.
//
// A step of one token a sequence is bound by the host: through ctypes an entry point of some thirty arguments
// cost 6 to 7 us, 4 of them for turning Python's numbers and addresses into C's. Here the conversions follow from the entry
// point's own type, and a pointer argument takes the tensor itself (its data_ptr()), a number or None. Two launches of a windowed
// token with the checks before them: 24.5 us through ctypes, 14.4 through this. Latent attention's steps, which are short prompts as
// well, come through here too.
//
// The symbols are libloqa_seqmix.so's and libloqa_lowbit.so's, which are loaded before this module; signatures() lets the loader compare the
// types here with those it knows.
#include <Python.h>
#include <ATen/ops/empty.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <exception>
#include <string>
#include <utility>

typedef void* stream_t;

extern "C" {
int loqa_qk_prep_append(const void*, int, long, int, int, int, int, int, const void*, int, int, float, float, int, const void*, void*,
                        void*, int, int, const void*, void*, int, const void*, const void*, int, const void*, long, float, const void*,
                        long, void*, long, int, int, int, int, stream_t);
int loqa_window_attention(const void*, int, const void*, const void*, int, int, const void*, const void*, const void*, int, const void*,
                          const void*, long, float, float, int, int, int, int, int, int, int, int, int, int, void*, long, int, void*,
                          const void*, const void*, stream_t);
int loqa_window_attention_parts(const void*, int, const void*, const void*, int, int, const void*, const void*, const void*, int,
                                const void*, const void*, long, float, float, int, int, int, int, int, int, int, int, int, int, void*,
                                long, int, void*, const void*, const void*, int, long, void*, long, stream_t);
int loqa_delta_prep(const void*, int, long, const void*, const void*, long, int, int, int, int, int, const void*, int, const void*, int,
                    const void*, const void*, const void*, const void*, const void*, int, int, void*, void*, stream_t);
int loqa_delta_scan(const void*, long, int, int, int, int, int, int, int, int, void*, int, const void*, const void*, const void*,
                    const void*, void*, int, int, stream_t);
int loqa_seq_state_save(const void*, int, const void*, int, int, void*, void*, int, int, int, const void*, const void*, const void*, int,
                        stream_t);
int loqa_gated_rmsnorm(const void*, const void*, const void*, int, long, float, void*, int, int, int, int, int, stream_t);
int loqa_latent_attention(const void*, long, long, const void*, long, long, int, const void*, int, int, const void*, const void*,
                          const void*, int, const void*, const void*, int, const void*, float, int, int, int, int, int, int, void*, int,
                          void*, int, int, stream_t);
int loqa_latent_kv(const void*, long, int, int, const void*, int, const void*, const void*, int, int, const void*, int, int, int, int,
                   int, void*, void*, int, stream_t);
int loqa_latent_prefill(const void*, long, const void*, const void*, void*, long, const void*, const void*, const void*, const void*,
                        const void*, float, int, const void*, long, int, int, int, int, int, int, const void*, int, int, int, int,
                        void*, long, void*, long, stream_t);
int loqa_sigmoid_gate(const void*, long, long, int, const void*, long, void*, long, long, int, int, int, stream_t);
int loqa_head_product(const void*, long, long, const void*, int, int, int, int, void*, long, long, stream_t);
int loqa_moe_route(const void*, const void*, const void*, int, int, int, int, int, int, int, float, void*, void*, int, stream_t);
int loqa_rope_append8(const void*, long, const void*, int, void*, void*, void*, void*, const void*, const void*, const void*, void*, long, int,
                      int, int, int, int, int, int, int, int, int, stream_t);
int loqa_read8(const void*, const void*, const void*, const void*, const void*, const void*, const void*, void*, void*, int, int, int, int, int,
               int, int, int, stream_t);
int loqa_attention8(const void*, long, const void*, const void*, const void*, const void*, const void*, const void*, const void*, void*, long,
                    int, int, int, int, int, int, int, int, int, float, int, int, int, int, int, void*, long, void*, long, stream_t);
int loqa_page_step(const void*, const void*, void*, void*, const void*, void*, void*, void*, void*, void*, void*, void*, void*, int, int, int,
                   int, int, stream_t);
int loqa_linear4(const void*, long, const void*, const void*, const void*, const void*, void*, long, int, int, int, int, int, int, void*, long, void*,
                 long, stream_t);
}

namespace {

bool tensor_of(PyObject* o, const at::Tensor** t) {
  if (!THPVariable_CheckExact(o) && !THPVariable_Check(o)) return false;
  *t = &THPVariable_Unpack(o);
  return true;
}

template <typename T> struct Arg;
template <> struct Arg<void*> {
  static constexpr char code = 'p';
  static bool get(PyObject* o, void** v) {
    const at::Tensor* t;
    if (o == Py_None) *v = nullptr;
    else if (PyLong_Check(o)) *v = PyLong_AsVoidPtr(o);
    else if (tensor_of(o, &t)) *v = t->data_ptr();
    else PyErr_SetString(PyExc_TypeError, "a tensor, an address or None");
    return !PyErr_Occurred();
  }
};
template <> struct Arg<const void*> : Arg<void*> {
  static bool get(PyObject* o, const void** v) { return Arg<void*>::get(o, const_cast<void**>(v)); }
};
template <> struct Arg<long> {
  static constexpr char code = 'l';
  static bool get(PyObject* o, long* v) {
    *v = PyLong_AsLong(o);
    return *v != -1 || !PyErr_Occurred();
  }
};
template <> struct Arg<int> {
  static constexpr char code = 'i';
  static bool get(PyObject* o, int* v) {
    long x;
    if (!Arg<long>::get(o, &x)) return false;
    *v = (int)x;
    if (*v != x) PyErr_SetString(PyExc_OverflowError, "an argument is out of the range of an int");
    return *v == x;
  }
};
template <> struct Arg<float> {
  static constexpr char code = 'f';
  static bool get(PyObject* o, float* v) {
    const double x = PyFloat_AsDouble(o);
    *v = (float)x;
    return x != -1.0 || !PyErr_Occurred();
  }
};

template <auto F> struct Entry;
template <typename... A, int (*F)(A...)> struct Entry<F> {
  static std::string signature() { return {Arg<A>::code...}; }
  template <size_t... I> static PyObject* run(PyObject* const* args, std::index_sequence<I...>) {
    std::tuple<A...> v;
    if (!(Arg<A>::get(args[I], &std::get<I>(v)) && ...)) return nullptr;
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = F(std::get<I>(v)...);
    Py_END_ALLOW_THREADS
    return PyLong_FromLong(rc);
  }
  static PyObject* call(PyObject*, PyObject* const* args, Py_ssize_t n) {
    if (n != (Py_ssize_t)sizeof...(A)) return PyErr_Format(PyExc_TypeError, "takes %d arguments, got %d", (int)sizeof...(A), (int)n);
    try {
      return run(args, std::index_sequence_for<A...>{});
    } catch (const std::exception& e) {          // a tensor without storage
      PyErr_SetString(PyExc_RuntimeError, e.what());
      return nullptr;
    }
  }
};

// Pairs of a tensor and its name, all of them contiguous and of one type.
template <at::ScalarType T> PyObject* contiguous(PyObject*, PyObject* const* args, Py_ssize_t n) {
  for (Py_ssize_t i = 0; i + 1 < n; i += 2) {
    const at::Tensor* t;
    if (!tensor_of(args[i], &t)) return PyErr_Format(PyExc_TypeError, "%U must be a tensor", args[i + 1]);
    try {
      if (t->scalar_type() == T && t->is_contiguous()) continue;
    } catch (const std::exception& e) {
      PyErr_SetString(PyExc_RuntimeError, e.what());
      return nullptr;
    }
    return PyErr_Format(PyExc_TypeError, T == at::kInt ? "%U must be contiguous int32" : "%U must be contiguous float32", args[i + 1]);
  }
  Py_RETURN_NONE;
}

// What ops/seqmix.py asserts of its tensors before these launches, in one call: fifty attributes of tensors took 5 us from Python.
struct Bad { const char* what; };
void need(bool ok, const char* what) {
  if (!ok) throw Bad{what};
}
void need_i32(const at::Tensor& t, const char* name) {
  if (t.scalar_type() == at::kInt && t.is_contiguous()) return;
  PyErr_Format(PyExc_TypeError, "%s must be contiguous int32", name);
  throw Bad{nullptr};
}

// f(tensors, numbers) with the first N arguments as tensors (null for None) and the others as numbers
template <int N, int M, typename Fn> PyObject* checked(PyObject* const* args, Py_ssize_t n, Fn&& f) {
  if (n != N + M) return PyErr_Format(PyExc_TypeError, "takes %d arguments, got %d", N + M, (int)n);
  const at::Tensor* t[N] = {};
  long v[M];
  for (int i = 0; i < N; ++i)
    if (args[i] != Py_None && !tensor_of(args[i], &t[i])) return PyErr_Format(PyExc_TypeError, "argument %d must be a tensor", i);
  for (int i = 0; i < M; ++i)
    if (!Arg<long>::get(args[N + i], &v[i])) return nullptr;
  try {
    return f(t, v);
  } catch (const Bad& b) {
    if (b.what) PyErr_SetString(PyExc_AssertionError, b.what);
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  }
  return nullptr;
}

void need_caches(const at::Tensor& k, const at::Tensor& v, const at::Tensor& x, long G, long D, long Dv) {
  need(k.dim() >= 3 && v.dim() == 3 && k.is_contiguous() && v.is_contiguous(), "contiguous caches [blocks, block, columns]");
  need(k.scalar_type() == x.scalar_type() && v.scalar_type() == x.scalar_type(), "caches of the rows' type");
  need(k.size(2) == G * D && v.size(0) == k.size(0) && v.size(1) == k.size(1) && v.size(2) == G * Dv, "cache columns");
}

// (T, row stride of u, blocks, block, rows of the rotation table) of qk_prep_append
PyObject* qk_shapes(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return checked<6, 6>(args, n, [](const at::Tensor* const* t, const long* v) {
    for (int i = 0; i < 5; ++i) need(t[i], "tensors");
    const at::Tensor &u = *t[0], &k = *t[1], &vc = *t[2], &pos = *t[3], &slots = *t[4];
    const long H = v[0], G = v[1], D = v[2], Dv = v[3], v_off = v[4], dims = v[5];
    need(u.dim() == 2 && u.stride(1) == 1 && (H + G) * D <= u.size(1), "rows with q and k");
    need((v_off < 0 && Dv == D) || (v_off >= (H + G) * D && v_off + G * Dv <= u.size(1)), "values' columns");
    need(dims % 2 == 0 && 0 <= dims && dims <= D, "rotated entries");
    long rows = 0;
    if (dims) {
      need(t[5] && t[5]->dim() >= 2, "a table of rotations");
      if (t[5]->scalar_type() != at::kFloat || !t[5]->is_contiguous()) {
        PyErr_SetString(PyExc_TypeError, "cos_sin must be contiguous float32");
        throw Bad{nullptr};
      }
      need(t[5]->size(1) * 2 == dims, "a table of these rotations");
      rows = t[5]->size(0);
    }
    need_caches(k, vc, u, G, D, Dv);
    need_i32(pos, "positions");
    need_i32(slots, "slots");
    need(pos.numel() >= u.size(0) && slots.numel() >= u.size(0), "a position and a slot for every row");
    return Py_BuildValue("lllll", (long)u.size(0), (long)u.stride(0), (long)k.size(0), (long)k.size(1), rows);
  });
}

// (T, blocks, block, B, columns of the block table, whether the matrix-core token form takes the rows) of window_attention
PyObject* window_shapes(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return checked<7, 4>(args, n, [](const at::Tensor* const* t, const long* v) {
    for (int i = 0; i < 7; ++i) need(t[i], "tensors");
    const at::Tensor &q = *t[0], &k = *t[1], &vc = *t[2], &cu = *t[3], &ctx = *t[4], &bt = *t[5], &pos = *t[6];
    const long H = v[0], G = v[1], D = v[2], Dv = v[3];
    need(q.dim() >= 2 && q.is_contiguous() && q.size(1) == H * D && G > 0 && H % G == 0, "rows of H heads");
    need_caches(k, vc, q, G, D, Dv);
    need(D <= 512 && Dv <= 512, "heads up to 512");
    need_i32(cu, "cu_q");
    need_i32(ctx, "ctx_lens");
    need_i32(bt, "block_tables");
    need_i32(pos, "positions");
    const long B = ctx.numel();
    need(cu.numel() == B + 1 && bt.dim() >= 2 && bt.size(0) == B && pos.numel() >= q.size(0), "feeds, block table and positions");
    // attn_window_token.hip's rule
    const bool token = q.scalar_type() == at::kBFloat16 && D <= 128 && Dv <= 128 && D % 8 == 0 && Dv % 8 == 0 && H / G <= 16 &&
                       (long)k.size(0) * k.size(1) < (1L << 31) &&
                       (((size_t)q.data_ptr() | (size_t)k.data_ptr() | (size_t)vc.data_ptr()) & 15) == 0;
    return Py_BuildValue("lllllO", (long)q.size(0), (long)k.size(0), (long)k.size(1), B, (long)bt.size(1), token ? Py_True : Py_False);
  });
}

// ---- ops/lowbit.py. What its checks ask of a call's tensors, in one go: the numbers of the launch and what it writes to, or None where
// anything is not as a GPU call has it (the checks there then say what, or take the tensors to the CPU's forms).
bool i32_on(const at::Tensor* t, const at::Device& dev) {
  return t && t->scalar_type() == at::kInt && t->is_contiguous() && t->device() == dev;
}
bool rows_on(const at::Tensor& t, long cols, const at::Device& dev) {
  return t.scalar_type() == at::kBFloat16 && t.dim() == 2 && t.size(1) >= cols && (t.stride(1) == 1 || t.size(1) == 1) &&
         (t.size(0) <= 1 || t.stride(0) >= cols) && t.device() == dev;
}
// what a row's stride is where there is a second row, and one that any launch takes where there is none
long row_stride(const at::Tensor& t) { return t.size(0) > 1 ? (long)t.stride(0) : (long)((t.size(1) + 7) / 8 * 8); }
at::Tensor made(at::IntArrayRef size, at::ScalarType type, const at::Device& dev) {
  return at::empty(size, at::TensorOptions().dtype(type).device(dev));
}

// entries at .. at + m of a vector, as a tensor on the same storage (narrow, without its dispatch: seven of them were half of page_step's call)
at::Tensor stretch(const at::Tensor& all, long at, long m) {
  at::Tensor x = at::detail::make_tensor<c10::TensorImpl>(c10::TensorImpl::VIEW, c10::Storage(all.storage()), all.key_set(), all.dtype());
  x.unsafeGetTensorImpl()->set_storage_offset(all.storage_offset() + at);
  x.unsafeGetTensorImpl()->set_sizes_contiguous({m});
  return x;
}

// (rows x, rows y or None, cu_q, ctx_lens, block_tables, the cache's k; columns of x, of y) -> (T, B, columns of the
// table, row strides of x and y, y, device)
PyObject* cache8_rows(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return checked<6, 2>(args, n, [](const at::Tensor* const* t, const long* v) -> PyObject* {
    if (!t[0] || !t[5] || !t[5]->is_cuda()) Py_RETURN_NONE;
    const at::Tensor &x = *t[0], &bt = *t[4];
    const at::Device dev = t[5]->device();
    if (!rows_on(x, v[0], dev) || (t[1] && (!rows_on(*t[1], v[1], dev) || t[1]->size(0) != x.size(0)))) Py_RETURN_NONE;
    if (!i32_on(t[2], dev) || !i32_on(t[3], dev) || !i32_on(t[4], dev)) Py_RETURN_NONE;
    const long T = x.size(0), B = t[3]->numel();
    if (T == 0 || B == 0 || t[2]->numel() != B + 1 || bt.dim() != 2 || bt.size(0) != B || bt.size(1) == 0) Py_RETURN_NONE;
    const at::Tensor y = t[1] ? *t[1] : made({T, v[1]}, at::kBFloat16, dev);
    return Py_BuildValue("lllllNl", T, B, (long)bt.size(1), row_stride(x), row_stride(y), THPVariable_Wrap(y), (long)dev.index());
  });
}

// Whole calls: checks, allocations and the launch, where the tensors are on the current device; None as above.
PyObject* launched(int rc, const char* what) {
  if (rc != 0) PyErr_Format(PyExc_RuntimeError, "%s failed with hipError %d", what, rc);
  return nullptr;
}

// (qkv, q_out or None, cu_q, ctx_lens, block_tables, cos_sin or None, k, v, k_scale, v_scale; heads, kv heads, columns, rows of a page,
// pages, max_q, kind, current device, its stream) -> q
PyObject* rope_append8(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return checked<10, 9>(args, n, [](const at::Tensor* const* t, const long* v) -> PyObject* {
    if (!t[0] || !t[6] || !t[6]->is_cuda() || t[6]->get_device() != v[7]) Py_RETURN_NONE;
    const at::Tensor &x = *t[0], &bt = *t[4];
    const at::Device dev = t[6]->device();
    const long H = v[0], G = v[1], D = v[2];
    if (H <= 0 || !rows_on(x, (H + 2 * G) * D, dev) || (t[1] && (!rows_on(*t[1], H * D, dev) || t[1]->size(0) != x.size(0)))) Py_RETURN_NONE;
    if (!i32_on(t[2], dev) || !i32_on(t[3], dev) || !i32_on(t[4], dev)) Py_RETURN_NONE;
    const long T = x.size(0), B = t[3]->numel();
    if (T == 0 || B == 0 || v[5] <= 0 || t[2]->numel() != B + 1 || bt.dim() != 2 || bt.size(0) != B || bt.size(1) == 0) Py_RETURN_NONE;
    if (t[5] && (t[5]->scalar_type() != at::kFloat || t[5]->dim() != 3 || t[5]->size(1) * 2 != D || t[5]->size(2) != 2 || t[5]->size(0) == 0 ||
                 !t[5]->is_contiguous() || t[5]->device() != dev || ((size_t)t[5]->data_ptr() & 15)))
      Py_RETURN_NONE;
    const at::Tensor q = t[1] ? *t[1] : made({T, H * D}, at::kBFloat16, dev);
    if ((((size_t)x.data_ptr() | (size_t)q.data_ptr()) & 7) || ((row_stride(x) | row_stride(q)) & 3)) Py_RETURN_NONE;
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = loqa_rope_append8(x.data_ptr(), row_stride(x), t[5] ? t[5]->data_ptr() : nullptr, t[5] ? (int)t[5]->size(0) : 0, t[6]->data_ptr(), t[7]->data_ptr(),
                           t[8]->data_ptr(), t[9]->data_ptr(), t[2]->data_ptr(), t[3]->data_ptr(), bt.data_ptr(), q.data_ptr(), row_stride(q), (int)T,
                           (int)B, (int)H, (int)G, (int)D, (int)v[3], (int)v[4], (int)bt.size(1), (int)std::min(v[5], T), (int)v[6], (stream_t)v[8]);
    Py_END_ALLOW_THREADS
    return rc ? launched(rc, "rope_append8") : THPVariable_Wrap(q);
  });
}

// (cu_k, first, block_tables, k, v, k_scale, v_scale; kv heads, columns, rows of a page, pages, total, kind, current device, its stream)
// -> (k, v)
PyObject* read8(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return checked<7, 8>(args, n, [](const at::Tensor* const* t, const long* v) -> PyObject* {
    if (!t[3] || !t[3]->is_cuda() || t[3]->get_device() != v[6]) Py_RETURN_NONE;
    const at::Device dev = t[3]->device();
    if (!i32_on(t[0], dev) || !i32_on(t[1], dev) || !i32_on(t[2], dev)) Py_RETURN_NONE;
    const at::Tensor& bt = *t[2];
    const long B = t[1]->numel(), total = v[4];
    if (B == 0 || total <= 0 || total >= 1L << 31 || t[0]->numel() != B + 1 || bt.dim() != 2 || bt.size(0) != B || bt.size(1) == 0) Py_RETURN_NONE;
    const at::Tensor k = made({total, v[0], v[1]}, at::kBFloat16, dev), u = made({total, v[0], v[1]}, at::kBFloat16, dev);
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = loqa_read8(t[3]->data_ptr(), t[4]->data_ptr(), t[5]->data_ptr(), t[6]->data_ptr(), t[0]->data_ptr(), t[1]->data_ptr(), bt.data_ptr(),
                    k.data_ptr(), u.data_ptr(), (int)total, (int)B, (int)v[0], (int)v[1], (int)v[2], (int)v[3], (int)bt.size(1), (int)v[5],
                    (stream_t)v[7]);
    Py_END_ALLOW_THREADS
    return rc ? launched(rc, "read8") : Py_BuildValue("NN", THPVariable_Wrap(k), THPVariable_Wrap(u));
  });
}

// (new_lens, ctx_lens, block_tables, free_pages, ring, ctx_out or None, ring_out or None, tickets or None; rows of a page, max_tokens, sequences
// at most, current device, its stream) -> (cu_q, positions, slots, last_rows, ctx_out, ring_out, status)
PyObject* page_step(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return checked<8, 5>(args, n, [](const at::Tensor* const* t, const long* v) -> PyObject* {
    if (!t[2] || !t[2]->is_cuda() || t[2]->get_device() != v[3]) Py_RETURN_NONE;
    const at::Device dev = t[2]->device();
    for (int i = 0; i < 7; ++i)
      if (i < 5 ? !i32_on(t[i], dev) : t[i] && !i32_on(t[i], dev)) Py_RETURN_NONE;
    const at::Tensor& bt = *t[2];
    const long B = t[0]->numel(), pool = t[3]->numel(), P = v[0], most = v[1];
    if (B == 0 || B > v[2] || t[1]->numel() != B || bt.dim() != 2 || bt.size(0) != B || bt.size(1) == 0 || t[4]->numel() != 2 || pool == 0)
      Py_RETURN_NONE;
    if (most < 0 || most > 1L << 30 || P <= 0 || (P & (P - 1)) || P >= 1L << 31 || pool * P >= 1L << 31) Py_RETURN_NONE;
    if ((t[5] && t[5]->numel() != B) || (t[6] && t[6]->numel() != 2)) Py_RETURN_NONE;
    // one allocation for all that is int32
    const at::Tensor all = made({B + 1 + 2 * most + B + 2 + 1}, at::kInt, dev), last = made({B}, at::kLong, dev);
    long at = 0;
    auto ints = [&](long m) {
      const at::Tensor x = stretch(all, at, m);
      at += m;
      return x;
    };
    const at::Tensor cu = ints(B + 1), pos = ints(most), slots = ints(most), status = ints(1), ctx = t[5] ? *t[5] : ints(B), ring = t[6] ? *t[6] : ints(2);
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = loqa_page_step(t[0]->data_ptr(), t[1]->data_ptr(), bt.data_ptr(), t[3]->data_ptr(), t[4]->data_ptr(), cu.data_ptr(), pos.data_ptr(),
                        slots.data_ptr(), last.data_ptr(), ctx.data_ptr(), ring.data_ptr(), status.data_ptr(), t[7] ? t[7]->data_ptr() : nullptr,
                        (int)B, (int)bt.size(1), (int)P, (int)pool, (int)most, (stream_t)v[4]);
    Py_END_ALLOW_THREADS
    if (rc) return launched(rc, "page_step");
    return Py_BuildValue("NNNNNNN", THPVariable_Wrap(cu), THPVariable_Wrap(pos), THPVariable_Wrap(slots), THPVariable_Wrap(last),
                         THPVariable_Wrap(ctx), THPVariable_Wrap(ring), THPVariable_Wrap(status));
  });
}

// (x, codes, scales, zeros or None, bias or None; N, K, group, current device, its stream) -> y of up to 16 rows on the current
// device, as a whole call; otherwise (rows, row stride, y to fill, device)
PyObject* linear4_rows(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return checked<5, 5>(args, n, [](const at::Tensor* const* t, const long* v) -> PyObject* {
    if (!t[0] || !t[1] || !t[2] || !t[1]->is_cuda()) Py_RETURN_NONE;
    const at::Tensor& x = *t[0];
    const at::Device dev = t[1]->device();
    const long N = v[0], K = v[1];
    if (x.scalar_type() != at::kBFloat16 || x.device() != dev || x.dim() != 2 || x.size(1) != K || x.size(0) == 0 || x.stride(1) != 1 ||
        row_stride(x) < 0 || row_stride(x) % 8 || ((size_t)x.data_ptr() & 15))
      Py_RETURN_NONE;
    if (t[4] && (t[4]->scalar_type() != at::kBFloat16 || t[4]->dim() != 1 || t[4]->size(0) != N || !t[4]->is_contiguous() || t[4]->device() != dev))
      Py_RETURN_NONE;
    const at::Tensor y = made({x.size(0), N}, at::kBFloat16, dev);
    if (x.size(0) > 16 || dev.index() != v[3])
      return Py_BuildValue("llNl", (long)x.size(0), row_stride(x), THPVariable_Wrap(y), (long)dev.index());
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = loqa_linear4(x.data_ptr(), row_stride(x), t[1]->data_ptr(), t[2]->data_ptr(), t[3] ? t[3]->data_ptr() : nullptr,
                      t[4] ? t[4]->data_ptr() : nullptr, y.data_ptr(), N, (int)x.size(0), (int)N, (int)K, (int)v[2], 0, 1, nullptr, 0, nullptr, 0,
                      (stream_t)v[4]);
    Py_END_ALLOW_THREADS
    return rc ? launched(rc, "linear4") : THPVariable_Wrap(y);
  });
}

#define ENTRIES(X)                                                                                                                \
  X(loqa_qk_prep_append) X(loqa_window_attention) X(loqa_window_attention_parts) X(loqa_delta_prep) X(loqa_delta_scan) \
  X(loqa_seq_state_save) X(loqa_gated_rmsnorm) X(loqa_moe_route) X(loqa_latent_attention) X(loqa_latent_kv) \
  X(loqa_latent_prefill) X(loqa_sigmoid_gate) X(loqa_head_product) \
  X(loqa_rope_append8) X(loqa_read8) X(loqa_attention8) X(loqa_page_step) X(loqa_linear4)

PyObject* signatures(PyObject*, PyObject*) {
  PyObject* d = PyDict_New();
#define SIG(F)                                                                \
  if (d) {                                                                    \
    PyObject* s = PyUnicode_FromString(Entry<&F>::signature().c_str());       \
    if (!s || PyDict_SetItemString(d, #F, s) != 0) Py_CLEAR(d);               \
    Py_XDECREF(s);                                                            \
  }
  ENTRIES(SIG)
#undef SIG
  return d;
}

#define METHOD(F) {#F, (PyCFunction)(void (*)(void))Entry<&F>::call, METH_FASTCALL, nullptr},
PyMethodDef methods[] = {
    ENTRIES(METHOD)
    {"i32c", (PyCFunction)(void (*)(void))contiguous<at::kInt>, METH_FASTCALL, nullptr},
    {"f32c", (PyCFunction)(void (*)(void))contiguous<at::kFloat>, METH_FASTCALL, nullptr},
    {"qk_shapes", (PyCFunction)(void (*)(void))qk_shapes, METH_FASTCALL, nullptr},
    {"window_shapes", (PyCFunction)(void (*)(void))window_shapes, METH_FASTCALL, nullptr},
    {"cache8_rows", (PyCFunction)(void (*)(void))cache8_rows, METH_FASTCALL, nullptr},
    {"rope_append8", (PyCFunction)(void (*)(void))rope_append8, METH_FASTCALL, nullptr},
    {"read8", (PyCFunction)(void (*)(void))read8, METH_FASTCALL, nullptr},
    {"page_step", (PyCFunction)(void (*)(void))page_step, METH_FASTCALL, nullptr},
    {"linear4_rows", (PyCFunction)(void (*)(void))linear4_rows, METH_FASTCALL, nullptr},
    {"signatures", signatures, METH_NOARGS, nullptr},
    {nullptr, nullptr, 0, nullptr}};
#undef METHOD

PyModuleDef module = {PyModuleDef_HEAD_INIT, "libloqa_launch", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_libloqa_launch(void) { return PyModule_Create(&module); }
