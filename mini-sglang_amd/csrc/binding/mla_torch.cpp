// Python calls of the entry points whose launches are short: what kernel/lib.py does with ctypes for the others (checks of
// the tensors, the entry point with their pointers and strides on a stream), with the tensors read in C++. A call of 28
// arguments took 6 us in Python and 2 in ctypes, more than most of these kernels run.
//
// Every function returns the entry point's code, kOtherDevice where the tensors' GPU is not the current one, or kOtherStream
// where it takes memory from torch's allocator for a stream that is not the current one (the caller makes the GPU or the
// stream current and calls again). A tensor that does not fit raises AssertionError, as in lib.py.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/core/LegacyTypeDispatch.h>
#include <ATen/ops/empty.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../../include/mla_amd.h"

namespace {

constexpr long kOtherDevice = -1, kOtherStream = -2;

// set by bind(): the entry points of the loaded library, and torch's current device and raw stream
struct {
  decltype(&mla_gqa_prompt_bf16) prompt;
  decltype(&mla_gqa_workspace_bytes) workspace_bytes;
  decltype(&mla_gqa_chunk_bf16) chunk;
  decltype(&mla_gqa_decode_bf16) decode;
  decltype(&mla_page_tables_from_lengths) tables;
  PyObject* current_device;
  PyObject* current_stream;
} g;

struct Refused {};

void require(bool ok, const char* what) {
  if (ok) return;
  PyErr_SetString(PyExc_AssertionError, what);
  throw Refused();
}

const at::Tensor& tensor(PyObject* o, const char* name) {
  if (!THPVariable_Check(o)) {
    PyErr_Format(PyExc_TypeError, "%s must be a tensor, got %s", name, Py_TYPE(o)->tp_name);
    throw Refused();
  }
  return THPVariable_Unpack(o);
}

long integer(PyObject* o) {
  const long v = PyLong_AsLong(o);
  if (v == -1 && PyErr_Occurred()) throw Refused();
  return v;
}
int32_t int32(PyObject* o, const char* name) {
  const long v = integer(o);
  if (v != (int32_t)v) {
    PyErr_Format(PyExc_OverflowError, "%s %ld does not fit 32 bits", name, v);
    throw Refused();
  }
  return (int32_t)v;
}
float number(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw Refused();
  return (float)v;
}

long gpu_of(const at::Tensor& t) { return t.is_cuda() ? t.get_device() : -1; }

bool is_current(long device) {
  PyObject* r = PyObject_CallNoArgs(g.current_device);
  if (r == nullptr) throw Refused();
  const long now = PyLong_AsLong(r);
  Py_DECREF(r);
  return now == device;
}
void* as_pointer(PyObject* r) {  // takes the reference
  if (r == nullptr) throw Refused();
  void* p = PyLong_AsVoidPtr(r);
  Py_DECREF(r);
  if (p == nullptr && PyErr_Occurred()) throw Refused();
  return p;
}
void* current_stream(long device) {
  PyObject* d = PyLong_FromLong(device);
  PyObject* r = PyObject_CallOneArg(g.current_stream, d);
  Py_XDECREF(d);
  return as_pointer(r);
}
// `stream`: None for the current one, else a torch stream
void* stream_of(PyObject* stream, long device) {
  return stream == Py_None ? current_stream(device) : as_pointer(PyObject_GetAttrString(stream, "cuda_stream"));
}
// Memory from torch's allocator belongs to the current stream: work that is queued there may still use the block's last
// content, and nothing orders another stream's launch behind it.
bool allocates_for(PyObject* stream, void* raw, long device) { return stream == Py_None || raw == current_stream(device); }

const int32_t* index(PyObject* o, const char* name, int64_t n, long device) {
  const at::Tensor& t = tensor(o, name);
  if (t.scalar_type() != at::kInt || t.dim() != 1 || t.size(0) != n || !t.is_contiguous() || gpu_of(t) != device) {
    PyErr_Format(PyExc_AssertionError, "%s must be int32 [%lld], contiguous, on the other tensors' GPU", name, (long long)n);
    throw Refused();
  }
  return static_cast<const int32_t*>(t.data_ptr());
}

// A dimension of one element has no stride of its own: torch gives it any.
int64_t stride_of(const at::Tensor& t, int64_t dim) { return t.size(dim) == 1 ? 0 : t.stride(dim); }
// (an expanded dimension has stride 0, and more than one element)
bool one_apart(const at::Tensor& t, int64_t dim) { return t.size(dim) == 1 || t.stride(dim) == 1; }

// What the attention calls share.
struct Attention {
  const at::Tensor &q, &k, &v, &out;
  const at::Tensor* lse = nullptr;
  long device;
  int64_t T, Hq, Hkv, D;

  Attention(PyObject* q_, PyObject* k_, PyObject* v_, PyObject* out_, PyObject* lse_, int k_dims)
      : q(tensor(q_, "q")), k(tensor(k_, "k")), v(tensor(v_, "v")), out(tensor(out_, "out")), device(gpu_of(q)) {
    if (lse_ != Py_None) lse = &tensor(lse_, "lse");
    require(q.dim() == 3 && k.dim() == k_dims, "q is [T, Hq, D]; k and v are [T, Hkv, D], or pools [pages, ps, Hkv, D]");
    T = q.size(0), Hq = q.size(1), D = q.size(2), Hkv = k.size(-2);
    require(k.size(-1) == D && v.sizes() == k.sizes() && Hkv > 0 && Hq % Hkv == 0, "k and v have q's D and heads that divide q's");
    require(device >= 0 && gpu_of(k) == device && gpu_of(v) == device && gpu_of(out) == device &&
                (lse == nullptr || gpu_of(*lse) == device),
            "all tensors must be on one GPU");
    require(q.scalar_type() == at::kBFloat16 && k.scalar_type() == at::kBFloat16 && v.scalar_type() == at::kBFloat16 &&
                out.scalar_type() == at::kBFloat16 && out.sizes() == q.sizes(),
            "q, k, v and out are bf16, out of q's shape");
    require(lse == nullptr || (lse->scalar_type() == at::kFloat && lse->dim() == 2 && lse->size(0) == T && lse->size(1) == Hq),
            "lse is fp32 [T, Hq]");
    require(q.stride(2) == 1 && k.stride(-1) == 1 && v.stride(-1) == 1 && out.stride(2) == 1 && (lse == nullptr || one_apart(*lse, 1)),
            "rows must be contiguous");
    require(T <= INT32_MAX && Hq <= INT32_MAX && Hkv <= INT32_MAX, "sizes past 32 bits");
  }
  float* lse_ptr() const { return lse == nullptr ? nullptr : static_cast<float*>(lse->data_ptr()); }
  int64_t lse_stride() const { return lse == nullptr || T == 1 ? Hq : lse->stride(0); }
};

// A call's body: its value, or the Python error that it or torch has set.
template <typename F>
PyObject* guarded(Py_ssize_t n, Py_ssize_t want, F&& body) {
  HANDLE_TH_ERRORS
  if (n != want) {
    PyErr_Format(PyExc_TypeError, "%zd arguments, %zd wanted", n, want);
    return nullptr;
  }
  try {
    return body();
  } catch (const Refused&) {
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}
template <typename F>
long launched(F&& call) {
  long rc;
  Py_BEGIN_ALLOW_THREADS;
  rc = call();
  Py_END_ALLOW_THREADS;
  return rc;
}

// gqa_prompt(q, k, v, cu_seqlens, scale, out, lse, stream)
PyObject* gqa_prompt(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 8, [&]() -> PyObject* {
    const Attention x(a[0], a[1], a[2], a[5], a[6], 3);
    require(x.k.size(0) == x.T, "as many keys as queries");
    const at::Tensor& cu = tensor(a[3], "cu_seqlens");
    require(cu.dim() == 1 && cu.size(0) >= 1, "cu_seqlens is [B + 1]");
    const int32_t* cu_ptr = index(a[3], "cu_seqlens", cu.size(0), x.device);
    const float scale = number(a[4]);
    if (!is_current(x.device)) return PyLong_FromLong(kOtherDevice);
    void* stream = stream_of(a[7], x.device);
    return PyLong_FromLong(launched([&] {
      return g.prompt(x.q.data_ptr(), stride_of(x.q, 0), stride_of(x.q, 1), x.k.data_ptr(), stride_of(x.k, 0), stride_of(x.k, 1),
                      x.v.data_ptr(), stride_of(x.v, 0), stride_of(x.v, 1), cu_ptr, (int32_t)(cu.size(0) - 1), (int32_t)x.T,
                      (int32_t)x.Hq, (int32_t)x.Hkv, (int32_t)x.D, scale, x.out.data_ptr(), stride_of(x.out, 0), stride_of(x.out, 1),
                      x.lse_ptr(), x.lse_stride(), stream);
    }));
  });
}

// gqa_paged(q, k_pool, v_pool, page_table, cu_seqlens_q or None, seq_lens, max_seqlen_q, scale, out, lse, workspace, stream)
PyObject* gqa_paged(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 12, [&]() -> PyObject* {
    const Attention x(a[0], a[1], a[2], a[8], a[9], 4);
    const int64_t ps = x.k.size(1);
    // rows lie one stride apart over the whole pool: of its tokens, or of its pages where they hold one
    auto row_stride = [&](const at::Tensor& t) {
      require(t.size(0) == 1 || ps == 1 || t.stride(0) == ps * t.stride(1), "pages of the pools must follow one another");
      return ps == 1 ? stride_of(t, 0) : t.stride(1);
    };
    const int64_t k_row = row_stride(x.k), v_row = row_stride(x.v);
    const at::Tensor& lens = tensor(a[5], "seq_lens");
    require(lens.dim() == 1, "seq_lens is [B]");
    const int64_t B = lens.size(0);
    const int32_t* lens_ptr = index(a[5], "seq_lens", B, x.device);
    const at::Tensor& pt = tensor(a[3], "page_table");
    require(pt.scalar_type() == at::kInt && pt.dim() == 2 && pt.size(0) >= B && one_apart(pt, 1) && gpu_of(pt) == x.device,
            "page_table is int32 [B, cols], on q's GPU");
    const int64_t pt_row = pt.size(0) == 1 ? pt.size(1) : pt.stride(0);
    require(B <= INT32_MAX && pt.size(1) <= INT32_MAX && x.k.size(0) <= INT32_MAX && ps <= INT32_MAX, "sizes past 32 bits");
    const bool decode = a[4] == Py_None;
    const int32_t* cu = nullptr;
    if (decode) require(x.T == B, "one token a request");
    else cu = index(a[4], "cu_seqlens_q", B + 1, x.device);
    const int32_t max_q = (int32_t)std::max<int64_t>(std::min<int64_t>(integer(a[6]), x.T), -1);
    const float scale = number(a[7]);
    if (!is_current(x.device)) return PyLong_FromLong(kOtherDevice);
    void* stream = stream_of(a[11], x.device);
    const int32_t* pt_ptr = static_cast<const int32_t*>(pt.data_ptr());
    auto call = [&](void* ws, int64_t bytes) {
      return launched([&] {
        if (decode)
          return g.decode(x.q.data_ptr(), stride_of(x.q, 0), stride_of(x.q, 1), x.k.data_ptr(), k_row, stride_of(x.k, 2),
                          x.v.data_ptr(), v_row, stride_of(x.v, 2), (int32_t)x.k.size(0), (int32_t)ps, pt_ptr, (int32_t)pt.size(1),
                          pt_row, lens_ptr, (int32_t)B, (int32_t)x.Hq, (int32_t)x.Hkv, (int32_t)x.D, scale, ws, bytes,
                          x.out.data_ptr(), stride_of(x.out, 0), stride_of(x.out, 1), x.lse_ptr(), x.lse_stride(), stream);
        return g.chunk(x.q.data_ptr(), stride_of(x.q, 0), stride_of(x.q, 1), x.k.data_ptr(), k_row, stride_of(x.k, 2),
                       x.v.data_ptr(), v_row, stride_of(x.v, 2), (int32_t)x.k.size(0), (int32_t)ps, pt_ptr, (int32_t)pt.size(1),
                       pt_row, cu, lens_ptr, (int32_t)B, (int32_t)x.T, max_q, (int32_t)x.Hq, (int32_t)x.Hkv, (int32_t)x.D, scale,
                       ws, bytes, x.out.data_ptr(), stride_of(x.out, 0), stride_of(x.out, 1), x.lse_ptr(), x.lse_stride(), stream);
      });
    };
    if (a[10] != Py_None) {
      const at::Tensor& w = tensor(a[10], "workspace");
      require(gpu_of(w) == x.device && w.is_contiguous(), "the workspace is one block on q's GPU");
      return PyLong_FromLong(call(w.data_ptr(), (int64_t)w.nbytes()));
    }
    // without one first; where keys are split, one from torch's allocator, for this call. On the host: a request of 100 keys, in
    // one piece, 3.9 us with or without a workspace given; of 1500, two launches, 7.2 with, 7.2 to 8.0 without
    long rc = call(nullptr, 0);
    if (rc == MLA_ERR_INVALID_ARG) {
      int64_t bytes = 0;
      if ((rc = g.workspace_bytes(max_q, (int32_t)x.Hq, (int32_t)x.Hkv, (int32_t)x.D, &bytes))) return PyLong_FromLong(rc);
      if (!allocates_for(a[11], stream, x.device)) return PyLong_FromLong(kOtherStream);
      const at::Tensor made = at::empty({bytes}, x.q.options().dtype(at::kByte));
      rc = call(made.data_ptr(), bytes);
    }
    return PyLong_FromLong(rc);
  });
}

// page_tables(token_table, table_idx, cached_lens, device_lens, free_slots, page_size, max_device_len, max_extend, total_new,
//             alloc_reqs or None, stream) -> code, or (page_table, out_loc, positions, cu_seqlens_q, pages_taken)
PyObject* page_tables(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 11, [&]() -> PyObject* {
    const at::Tensor& tt = tensor(a[0], "token_table");
    const long device = gpu_of(tt);
    require(device >= 0 && tt.scalar_type() == at::kInt && tt.dim() == 2 && one_apart(tt, 1), "token_table is int32 [rows, cols] on the GPU");
    const at::Tensor &idx = tensor(a[1], "table_idx"), &free = tensor(a[4], "free_slots");
    require(idx.dim() == 1 && free.dim() == 1, "table_idx and free_slots have one dimension");
    const int64_t B = idx.size(0), F = free.size(0);
    require(B <= INT32_MAX && F <= INT32_MAX && tt.size(0) <= INT32_MAX && tt.size(1) <= INT32_MAX, "sizes past 32 bits");
    const int32_t* idx_ptr = index(a[1], "table_idx", B, device);
    const int32_t* cached = index(a[2], "cached_lens", B, device);
    const int32_t* lens = index(a[3], "device_lens", B, device);
    const int32_t* free_ptr = index(a[4], "free_slots", F, device);
    const int32_t ps = int32(a[5], "page_size"), max_len = int32(a[6], "max_device_len"), max_extend = int32(a[7], "max_extend"),
                  total = int32(a[8], "total_new"), alloc = a[9] == Py_None ? (int32_t)B : int32(a[9], "alloc_reqs");
    require(ps > 0 && max_len >= 0 && total >= 0, "page_size is positive, max_device_len and total_new are not negative");
    if (!is_current(device)) return PyLong_FromLong(kOtherDevice);
    void* stream = stream_of(a[10], device);
    if (!allocates_for(a[10], stream, device)) return PyLong_FromLong(kOtherStream);
    const int64_t cols = ((int64_t)max_len + ps - 1) / ps, cells = B * cols;
    at::AutoDispatchBelowADInplaceOrView below;
    // one allocation, which the tables are cut from
    at::Tensor made = at::empty({cells + 2 * (int64_t)total + B + 2}, tt.options());
    int32_t* base = static_cast<int32_t*>(made.data_ptr());
    int32_t *loc = base + cells, *pos = loc + total, *cu = pos + total;
    const long rc = launched([&] {
      return g.tables(static_cast<int32_t*>(tt.data_ptr()), (int32_t)tt.size(0), (int32_t)tt.size(1),
                      tt.size(0) == 1 ? tt.size(1) : tt.stride(0), idx_ptr, cached,
                      lens, (int32_t)B, alloc, free_ptr, (int32_t)F, ps, max_extend, base, (int32_t)cols, cols, loc, pos, total, cu,
                      cu + B + 1, stream);
    });
    if (rc != 0) return PyLong_FromLong(rc);
    auto part = [&](int64_t at, int64_t size) { return THPVariable_Wrap(made.as_strided({size}, {1}, at)); };
    PyObject* r = PyTuple_New(5);
    if (r == nullptr) return nullptr;
    PyTuple_SET_ITEM(r, 0, THPVariable_Wrap(made.as_strided({B, cols}, {cols, 1}, 0)));
    PyTuple_SET_ITEM(r, 1, part(cells, total));
    PyTuple_SET_ITEM(r, 2, part(cells + total, total));
    PyTuple_SET_ITEM(r, 3, part(cells + 2 * (int64_t)total, B + 1));
    PyTuple_SET_ITEM(r, 4, part(cells + 2 * (int64_t)total + B + 1, 1));
    for (int i = 0; i < 5; ++i)
      if (PyTuple_GET_ITEM(r, i) == nullptr) {
        Py_DECREF(r);
        return nullptr;
      }
    return r;
  });
}

// bind(addresses of the five entry points..., torch's current device, torch's current raw stream)
PyObject* bind(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 7, [&]() -> PyObject* {
    auto address = [&](int i) {
      void* p = PyLong_AsVoidPtr(a[i]);
      if (p == nullptr) {
        if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "an entry point's address is null");
        throw Refused();
      }
      return p;
    };
    g.prompt = reinterpret_cast<decltype(g.prompt)>(address(0));
    g.workspace_bytes = reinterpret_cast<decltype(g.workspace_bytes)>(address(1));
    g.chunk = reinterpret_cast<decltype(g.chunk)>(address(2));
    g.decode = reinterpret_cast<decltype(g.decode)>(address(3));
    g.tables = reinterpret_cast<decltype(g.tables)>(address(4));
    Py_INCREF(a[5]);
    Py_INCREF(a[6]);
    g.current_device = a[5];
    g.current_stream = a[6];
    Py_RETURN_NONE;
  });
}

#define MLA_METHOD(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(name)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {MLA_METHOD(bind), MLA_METHOD(gqa_prompt), MLA_METHOD(gqa_paged), MLA_METHOD(page_tables), {}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_mla_torch", nullptr, -1, methods};

}  // namespace

// built_for: the torch and Python whose headers this was compiled with, "torch V, Python X.Y", by the build
PyMODINIT_FUNC PyInit__mla_torch() {
  PyObject* m = PyModule_Create(&module);
  if (m != nullptr && PyModule_AddStringConstant(m, "built_for", MLA_BUILT_FOR) != 0) Py_CLEAR(m);
  return m;
}
