// The 8-bit, Newton-Schulz and embedding calls of kernels/__init__.py from Python in one native call each, as fastcall.cpp has
// it for GEMMs and attention: what can be launched as it lies is checked, allocated for and launched here, every other call
// returns None and goes on to the Python statements, which copy, refuse or explain.
#include "calls_common.h"
#include "../native_ops.h"

namespace {

const at::ScalarType FP8[2] = {at::kFloat8_e4m3fn, at::kFloat8_e5m2};
constexpr int64_t FP8_MOST = (int64_t(1) << 31) - 512;     // rows and columns that kb_fp8_quantize and kb_gemm_fp8 take

bool current(const at::Tensor& t) { return t.device().index() == c10::cuda::getCurrentCUDAStream().device_index(); }
bool aligned(const at::Tensor& t) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0; }

// A tensor of part of a storage; without the dispatcher, which takes three times as long as the allocation behind it.
at::Tensor part(const at::Tensor& base, at::ScalarType type, int64_t offset, c10::IntArrayRef sizes, c10::IntArrayRef strides) {
  at::Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(base.storage()), c10::DispatchKeySet(c10::DispatchKey::CUDA),
                                                          c10::scalarTypeToTypeMeta(type));
  t.unsafeGetTensorImpl()->set_sizes_and_strides(sizes, strides, offset);
  return t;
}
// Data and scales of a matrix in one allocation.  Rows start on 16 bytes, as the kernels read them.
void fp8_matrix(int64_t rows, int64_t cols, int fmt, const at::TensorOptions& o, at::Tensor& data, at::Tensor& scales) {
  const int64_t ld = (cols + 15) / 16 * 16, blocks = (rows + 127) / 128, groups = ((cols + 127) / 128 + 3) / 4;
  const int64_t behind = (rows * ld + 511) / 512 * 512;
  const at::Tensor base = at::empty({behind + blocks * groups * 512}, o.dtype(at::kByte));
  data = part(base, FP8[fmt], 0, {rows, cols}, {ld, 1});
  scales = part(base, at::kByte, behind, {blocks, groups, 32, 4, 4}, {groups * 512, 512, 16, 4, 1});
}

// fp8_quantize(x, rows, cols, square, format) -> (data, scales, data of the transpose, its scales), None for what is not wanted
PyObject* fp8_quantize(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  if (nargs != 5) Py_RETURN_NONE;
  const at::Tensor* x = plain(args[0], at::kBFloat16);
  if (!x || x->dim() != 2 || !current(*x)) Py_RETURN_NONE;
  const int rows = PyObject_IsTrue(args[1]), cols = PyObject_IsTrue(args[2]), square = PyObject_IsTrue(args[3]);
  const long fmt = PyLong_AsLong(args[4]);
  if (rows < 0 || cols < 0 || square < 0 || PyErr_Occurred()) return nullptr;
  const int64_t M = x->size(0), N = x->size(1);
  if (!(rows || cols) || fmt < 0 || fmt > 1 || M < 1 || N < 1 || M > FP8_MOST || N > FP8_MOST) Py_RETURN_NONE;
  const int64_t ld = M > 1 ? x->stride(0) : N;
  if ((x->stride(1) != 1 && N > 1) || ld < N) Py_RETURN_NONE;
  const auto o = x->options().requires_grad(false);
  at::Tensor t[4];
  if (rows) fp8_matrix(M, N, fmt, o, t[0], t[1]);
  if (cols) fp8_matrix(N, M, fmt, o, t[2], t[3]);
  void* p[4];
  for (int i = 0; i < 4; ++i) p[i] = t[i].defined() ? t[i].data_ptr() : nullptr;
  const void* px = x->data_ptr();
  const cudaStream_t stream = c10::cuda::getCurrentCUDAStream().stream();
  const int rc = without_gil([&] {
    return kb_fp8_quantize(px, M, N, ld, p[0], (N + 15) / 16 * 16, p[1], p[2], (M + 15) / 16 * 16, p[3], square, fmt, stream);
  });
  if (!finish(rc, "fp8_quantize", 1)) return nullptr;
  PyObject* r = PyTuple_New(4);
  if (!r) return nullptr;
  for (int i = 0; i < 4; ++i) {
    if (t[i].defined()) {
      PyTuple_SET_ITEM(r, i, THPVariable_Wrap(std::move(t[i])));
    } else {
      Py_INCREF(Py_None);
      PyTuple_SET_ITEM(r, i, Py_None);
    }
  }
  return r;
  END_HANDLE_TH_ERRORS
}

// An 8-bit operand that can be read where it lies; ld 0 otherwise.
struct Operand {
  const at::Tensor *d = nullptr, *s = nullptr;
  int64_t rows = 0, k = 0, ld = 0;
  int fmt = 0;
};
Operand operand(PyObject* data, PyObject* scales) {
  Operand m;
  for (m.fmt = 0; m.fmt < 2 && !(m.d = plain(data, FP8[m.fmt])); ++m.fmt) {}
  m.s = plain(scales, at::kByte);
  if (!m.d || !m.s || m.d->dim() != 2 || m.s->dim() != 5 || m.d->device() != m.s->device() || !m.s->is_contiguous()) return m;
  m.rows = m.d->size(0);
  m.k = m.d->size(1);
  const int64_t want[5] = {(m.rows + 127) / 128, ((m.k + 127) / 128 + 3) / 4, 32, 4, 4};
  for (int i = 0; i < 5; ++i)
    if (m.s->size(i) != want[i]) return m;
  const int64_t ld = m.rows > 1 ? m.d->stride(0) : (m.k + 15) / 16 * 16;
  if (m.rows < 1 || m.k < 1 || m.rows > FP8_MOST || m.k > FP8_MOST || m.d->stride(1) != 1 || ld % 16 || ld < m.k || !aligned(*m.d) ||
      !aligned(*m.s))
    return m;
  m.ld = ld;
  return m;
}

// fp8_gemm(a data, a scales, b data, b scales, accumulate): bf16 output of its own, or accumulate += (fp32)
PyObject* fp8_gemm(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  if (nargs != 5) Py_RETURN_NONE;
  const Operand a = operand(args[0], args[1]), b = operand(args[2], args[3]);
  if (!a.ld || !b.ld || a.k != b.k || a.d->device() != b.d->device() || !current(*a.d)) Py_RETURN_NONE;
  at::Tensor out;
  const bool acc = args[4] != Py_None;
  if (acc) {
    const at::Tensor* c = plain(args[4], at::kFloat);
    if (!c || c->device() != a.d->device() || c->dim() != 2 || c->size(0) != a.rows || c->size(1) != b.rows || !c->is_contiguous())
      Py_RETURN_NONE;
    out = *c;
  } else {
    out = at::empty({a.rows, b.rows}, a.d->options().dtype(at::kBFloat16).requires_grad(false));
  }
  void* pc = out.data_ptr();
  const void *pa = a.d->data_ptr(), *psa = a.s->data_ptr(), *pb = b.d->data_ptr(), *psb = b.s->data_ptr();
  int* status = g_status[a.d->device().index()];
  const cudaStream_t stream = c10::cuda::getCurrentCUDAStream().stream();
  const int rc = without_gil([&] {
    return kb_gemm_fp8(pa, psa, a.fmt, a.ld, pb, psb, b.fmt, b.ld, pc, b.rows, a.rows, b.rows, a.k, acc, acc, status, stream);
  });
  if (rc != 0) {
    char what[96];
    std::snprintf(what, sizeof(what), "fp8_gemm M=%lld N=%lld K=%lld", static_cast<long long>(a.rows), static_cast<long long>(b.rows),
                  static_cast<long long>(a.k));
    finish(rc, what, 1);
    return nullptr;
  }
  if (!finish(rc, "fp8_gemm", 1)) return nullptr;
  if (acc) {
    Py_INCREF(args[4]);
    return args[4];
  }
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// orthogonalize(x, a, b, c, steps, eps, scale, scale_q): contiguous fp32 or bf16 matrices, checked parameters
PyObject* orthogonalize(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  if (nargs != 8) Py_RETURN_NONE;
  const at::Tensor* x = plain(args[0], at::kFloat);
  const bool bf16 = !x;
  if (!x) x = plain(args[0], at::kBFloat16);
  if (!x || x->dim() < 2 || !x->is_contiguous() || !x->numel() || !current(*x)) Py_RETURN_NONE;
  const double a = PyFloat_AsDouble(args[1]), b = PyFloat_AsDouble(args[2]), c = PyFloat_AsDouble(args[3]);
  const long steps = PyLong_AsLong(args[4]);
  const double eps = PyFloat_AsDouble(args[5]), scale = PyFloat_AsDouble(args[6]), scale_q = PyFloat_AsDouble(args[7]);
  if (PyErr_Occurred()) return nullptr;
  const int64_t m = x->size(-2), n = x->size(-1), batch = x->numel() / (m * n);
  const long bytes = kb_newton_schulz_bytes(batch, m, n);
  if (bytes <= 0) Py_RETURN_NONE;
  at::Tensor out = at::empty(x->sizes(), x->options().dtype(at::kBFloat16).requires_grad(false));
  at::Tensor work = at::empty({bytes}, x->options().dtype(at::kByte).requires_grad(false));
  void *po = out.data_ptr(), *pw = work.data_ptr();
  const void* px = x->data_ptr();
  int* status = g_status[x->device().index()];
  const cudaStream_t stream = c10::cuda::getCurrentCUDAStream().stream();
  const int rc = without_gil([&] {
    return kb_newton_schulz(px, bf16, batch, m, n, a, b, c, steps, eps, scale, scale_q, po, pw, status, stream);
  });
  if (!finish(rc, "orthogonalize", kb_newton_schulz_launches(batch, m, n, steps))) return nullptr;
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// Tokens and a table of rows.
bool lookup(const at::Tensor* tokens, const at::Tensor* table) {
  return tokens && table && table->dim() == 2 && tokens->is_contiguous() && table->is_contiguous() && tokens->numel() && table->numel() &&
         table->size(1) <= INT_MAX && tokens->device() == table->device() && current(*table);
}

// embedding_fwd(tokens, weight, vocab_start, scale)
PyObject* embedding_fwd(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  if (nargs != 4 || !PyLong_Check(args[2]) || !PyFloat_Check(args[3])) Py_RETURN_NONE;
  const at::Tensor *t = plain(args[0], at::kLong), *w = plain(args[1], at::kBFloat16);
  if (!lookup(t, w)) Py_RETURN_NONE;
  const long first = PyLong_AsLong(args[2]);
  if (PyErr_Occurred()) return nullptr;
  const double scale = PyFloat_AS_DOUBLE(args[3]);
  std::vector<int64_t> shape(t->sizes().begin(), t->sizes().end());
  const int64_t H = w->size(1), rows = w->size(0), n = t->numel();
  shape.push_back(H);
  at::Tensor out = at::empty(shape, w->options().requires_grad(false));
  const long* pt = reinterpret_cast<const long*>(t->data_ptr());
  const void* pw = w->data_ptr();
  void* po = out.data_ptr();
  const cudaStream_t stream = c10::cuda::getCurrentCUDAStream().stream();
  const int rc = without_gil([&] { return kb_embedding_fwd(pt, pw, po, n, H, first, rows, scale, stream); });
  if (!finish(rc, "embedding_fwd", 1)) return nullptr;
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// embedding_bwd_sorted(dout, tokens, grad, vocab_start, scale)
PyObject* embedding_bwd_sorted(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  if (nargs != 5 || !PyLong_Check(args[3]) || !PyFloat_Check(args[4])) Py_RETURN_NONE;
  const at::Tensor *d = plain(args[0], at::kBFloat16), *t = plain(args[1], at::kLong), *g = plain(args[2], at::kFloat);
  if (!d || !lookup(t, g) || d->device() != g->device() || !d->is_contiguous()) Py_RETURN_NONE;
  const int64_t H = g->size(1), rows = g->size(0), n = t->numel();
  if (d->dim() < 1 || d->size(-1) != H || d->numel() != n * H || rows > INT_MAX) Py_RETURN_NONE;
  const long first = PyLong_AsLong(args[3]);
  if (PyErr_Occurred()) return nullptr;
  const double scale = PyFloat_AS_DOUBLE(args[4]);
  const long bytes = kb_embedding_sorted_bytes(n, H);
  at::Tensor work;
  if (bytes) work = at::empty({bytes}, g->options().dtype(at::kByte).requires_grad(false));
  const long* pt = reinterpret_cast<const long*>(t->data_ptr());
  const void* pd = d->data_ptr();
  float* pg = g->data_ptr<float>();
  void* pw = bytes ? work.data_ptr() : nullptr;
  const cudaStream_t stream = c10::cuda::getCurrentCUDAStream().stream();
  const int rc = without_gil([&] { return kb_embedding_bwd_sorted(pt, pd, pg, n, H, first, rows, scale, pw, stream); });
  if (!finish(rc, "embedding_bwd", kb_embedding_sorted_launches(n))) return nullptr;
  Py_INCREF(args[2]);
  return args[2];
  END_HANDLE_TH_ERRORS
}

#define KB_METHOD(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(name)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {KB_METHOD(fp8_quantize), KB_METHOD(fp8_gemm), KB_METHOD(orthogonalize), KB_METHOD(embedding_fwd),
                         KB_METHOD(embedding_bwd_sorted), KB_METHOD(init), KB_METHOD(set_status), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_opcalls", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__opcalls() {
  PyObject* m = PyModule_Create(&module);
  if (m && PyModule_AddStringConstant(m, "torch_version", KB_TORCH_VERSION) != 0) Py_CLEAR(m);
  return m;
}
