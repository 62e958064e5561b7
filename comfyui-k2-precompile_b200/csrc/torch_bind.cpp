// torch_bind.cpp -- CPython binding of the conditioning operators.
//
// These run at the small end (one token, one latent's timestep), where a call
// costs what its host side costs: through ctypes the checks, allocations and
// the 20 to 35 arguments of a call take 15 to 25 us, as long as five of the
// kernels; here they take 3 to 5.  The checks and messages are the ops'
// own (ValueError, K2BError); k2b/ops.py documents the arguments.
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/k2b.h"

namespace {

PyObject* k2b_error = nullptr;

// Lets other Python threads run while a call allocates and launches.
struct NoGil {
  PyThreadState* state = PyEval_SaveThread();
  ~NoGil() { PyEval_RestoreThread(state); }
};

const at::Tensor& tensor(PyObject* o, const char* what) {
  TORCH_CHECK_VALUE(THPVariable_Check(o), what, ": tensor expected, got ", Py_TYPE(o)->tp_name);
  return THPVariable_Unpack(o);
}
// A null tensor for None.
at::Tensor optional(PyObject* o, const char* what) { return o == Py_None ? at::Tensor() : tensor(o, what); }
const void* ptr(const at::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
bool aligned(const at::Tensor& t, size_t bytes) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % bytes == 0; }

int dtype_code(const at::Tensor& t, const char* what) {
  const auto d = t.scalar_type();
  TORCH_CHECK_VALUE(d == at::kBFloat16 || d == at::kHalf, what, ": bf16 or fp16 expected, got ", d);
  return d == at::kHalf ? 1 : 2;
}

int fits_int(int64_t v, const char* what) {
  TORCH_CHECK_VALUE(v >= 0 && v <= 0x7fffffff, what, ": size ", v, " out of range");
  return (int)v;
}

// Every tensor on the current CUDA device, on whose stream the op launches.
void on_device(const char* what, const at::Tensor& first, std::initializer_list<const at::Tensor*> rest) {
  const auto dev = first.device();
  for (const at::Tensor* t : rest)
    TORCH_CHECK_VALUE(!t->defined() || t->device() == dev, what, ": all tensors on one CUDA device expected, got ",
                      t->device(), " and ", dev);
  TORCH_CHECK_VALUE(dev.is_cuda(), what, ": tensors on a CUDA device expected, got ", dev);
  TORCH_CHECK_VALUE(dev.index() == c10::cuda::current_device(), what, ": tensors on ", dev,
                    ", which is not the current CUDA device");
}

void* stream() { return c10::cuda::getCurrentCUDAStream().stream(); }

PyObject* failed(const char* name, int rc) {
  PyErr_Format(k2b_error, "%s failed with status %d", name, rc);
  return nullptr;
}

// Strides (batch, head, token) of a [B, H, L, D] view whose heads are
// contiguous and start on 16-byte boundaries; that of an axis with one entry
// says nothing.
struct Heads {
  int64_t B, H, L, D, sb, sh, st;
};
Heads heads(const at::Tensor& t, const char* what) {
  TORCH_CHECK_VALUE(t.dim() == 4 && (t.size(3) == 64 || t.size(3) == 128), what,
                    ": [B, H, L, D] with D 64 or 128 expected, got ", t.sizes());
  Heads h = {t.size(0), t.size(1), t.size(2), t.size(3), t.stride(0), t.stride(1), t.stride(2)};
  if (h.B <= 1) h.sb = h.D;
  if (h.H <= 1) h.sh = h.D;
  if (h.L <= 1) h.st = h.D;
  TORCH_CHECK_VALUE(t.numel() == 0 || (t.stride(3) == 1 && h.sb % 8 == 0 && h.sh % 8 == 0 && h.st % 8 == 0 && aligned(t, 16)),
                    what, ": contiguous heads on 16-byte boundaries expected (strides ", t.strides(), ")");
  return h;
}

// ------------------------------------------------------------- w4_linear
// (x, packed, scales, bias, rotate, act)
PyObject* w4_linear(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_VALUE(n_args == 6, "w4_linear: 6 arguments expected");
  const at::Tensor& x = tensor(a[0], "w4_linear: x");
  const at::Tensor& packed = tensor(a[1], "w4_linear: packed");
  const at::Tensor& scales = tensor(a[2], "w4_linear: scales");
  const at::Tensor bias = optional(a[3], "w4_linear: bias");
  const int rotate = PyObject_IsTrue(a[4]);
  const long act = PyLong_AsLong(a[5]);
  if (rotate < 0 || (act == -1 && PyErr_Occurred())) return nullptr;
  const int code = dtype_code(x, "w4_linear: x");
  TORCH_CHECK_VALUE(packed.scalar_type() == at::kByte && scales.scalar_type() == at::kHalf && packed.dim() == 2,
                    "w4_linear: packed uint8 [n, k/2] and fp16 scales expected");
  const int64_t n = packed.size(0), k = 2 * packed.size(1);
  TORCH_CHECK_VALUE(k > 0 && k % 128 == 0 && x.dim() > 0 && x.size(-1) == k && scales.dim() == 2 &&
                        scales.size(0) == n && scales.size(1) == k / 128,
                    "w4_linear: x ", x.sizes(), ", packed ", packed.sizes(), " and scales ", scales.sizes(),
                    " do not fit (k a multiple of 128)");
  TORCH_CHECK_VALUE(packed.is_contiguous() && scales.is_contiguous(), "w4_linear: contiguous packed and scales expected");
  TORCH_CHECK_VALUE(!bias.defined() || (bias.scalar_type() == x.scalar_type() && bias.dim() == 1 && bias.size(0) == n &&
                                        bias.is_contiguous()),
                    "w4_linear: bias [n] in x's dtype expected");
  // the rows of x: one stride over all leading dimensions
  const int64_t m = x.numel() / k;
  int64_t stride = k;
  if (!x.is_contiguous() && m > 0) {
    bool one = x.stride(-1) == 1;
    int64_t expect = -1;
    for (int64_t d = x.dim() - 2; d >= 0; --d) {
      if (x.size(d) == 1) continue;
      if (expect < 0) stride = x.stride(d);
      one = one && (expect < 0 || x.stride(d) == expect);
      expect = x.stride(d) * x.size(d);
    }
    TORCH_CHECK_VALUE(one && (m == 1 || stride >= k), "w4_linear: the rows of x must have one stride and contiguous columns");
  }
  TORCH_CHECK_VALUE(m == 0 || (stride % 4 == 0 && aligned(x, 8)), "w4_linear: x's rows must start on 8-byte boundaries");
  TORCH_CHECK_VALUE(n == 0 || aligned(packed, 16), "w4_linear: packed must start on a 16-byte boundary");
  on_device("w4_linear", x, {&packed, &scales, &bias});
  at::Tensor out;
  int rc = 0;
  {
    NoGil free;
    c10::SmallVector<int64_t, 5> shape(x.sizes().begin(), x.sizes().end() - 1);
    shape.push_back(n);
    out = at::empty(shape, x.options());
    if (out.numel()) {
      const int mi = fits_int(m, "w4_linear"), ni = fits_int(n, "w4_linear"), ki = fits_int(k, "w4_linear");
      const long long bytes = k2b_w4_workspace_bytes(mi, ki);
      at::Tensor work;
      if (bytes > 0) work = at::empty({(int64_t)bytes}, x.options().dtype(at::kByte));
      rc = k2b_w4_linear(x.data_ptr(), stride, packed.data_ptr(), scales.data_ptr(), ptr(bias), out.data_ptr(),
                         work.defined() ? work.data_ptr() : nullptr, mi, ni, ki, code, rotate, (int)act, stream());
    }
  }
  if (rc) return failed("k2b_w4_linear", rc);
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// ---------------------------------------------------------- qk_norm_rope
int rope_batch(const at::Tensor& f, const Heads& h, const char* name) {
  if (!f.defined()) return 1;
  const int64_t per = h.L * h.D * 2;
  TORCH_CHECK_VALUE(f.scalar_type() == at::kFloat && f.is_contiguous() && (f.numel() == 0 || aligned(f, 16)) &&
                        (f.numel() == per || f.numel() == h.B * per),
                    "qk_norm_rope: ", name, " must be contiguous fp32 [L, D/2, 2, 2] (or with a leading B)");
  return f.numel() == per ? 1 : (int)h.B;
}
void norm_weight(const at::Tensor& w, int64_t D, const char* name) {
  TORCH_CHECK_VALUE(w.defined() && w.scalar_type() == at::kFloat && w.numel() == D && w.is_contiguous() && aligned(w, 16),
                    "qk_norm_rope: ", name, " fp32 [D] expected");
}
// [B, H, L, D] over token-major memory, as the attention ops take it
at::Tensor token_major(const Heads& h, const at::Tensor& like) {
  return at::empty_strided({h.B, h.H, h.L, h.D}, {h.L * h.H * h.D, h.D, h.H * h.D, 1}, like.options());
}

// (q, k, wq, wk, freqs_q, freqs_k, eps_q, eps_k)
PyObject* qk_norm_rope(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_VALUE(n_args == 8, "qk_norm_rope: 8 arguments expected");
  const at::Tensor& q = tensor(a[0], "qk_norm_rope: q");
  const at::Tensor k = optional(a[1], "qk_norm_rope: k");
  const at::Tensor& wq = tensor(a[2], "qk_norm_rope: wq");
  const at::Tensor wk = optional(a[3], "qk_norm_rope: wk");
  const at::Tensor fq = optional(a[4], "qk_norm_rope: freqs_q"), fk = optional(a[5], "qk_norm_rope: freqs_k");
  const double eps_q = PyFloat_AsDouble(a[6]), eps_k = PyFloat_AsDouble(a[7]);
  if (PyErr_Occurred()) return nullptr;
  const int code = dtype_code(q, "qk_norm_rope: q");
  const Heads hq = heads(q, "qk_norm_rope: q");
  norm_weight(wq, hq.D, "wq");
  const int fqb = rope_batch(fq, hq, "freqs_q");
  Heads hk = {hq.B, 1, 0, hq.D, 0, 0, 0};
  int fkb = 1;
  if (k.defined()) {
    hk = heads(k, "qk_norm_rope: k");
    TORCH_CHECK_VALUE(hk.B == hq.B && hk.D == hq.D && k.scalar_type() == q.scalar_type(), "qk_norm_rope: k ", k.sizes(),
                      " ", k.scalar_type(), " does not go with q ", q.sizes(), " ", q.scalar_type());
    norm_weight(wk, hk.D, "wk");
    fkb = rope_batch(fk, hk, "freqs_k");
  } else {
    TORCH_CHECK_VALUE(!wk.defined() && !fk.defined(), "qk_norm_rope: wk and freqs_k go with k");
  }
  TORCH_CHECK_VALUE(hq.H > 0 && hk.H > 0, "qk_norm_rope: no heads");
  on_device("qk_norm_rope", q, {&k, &wq, &wk, &fq, &fk});
  at::Tensor qo, ko;
  int rc = 0;
  {
    NoGil free;
    qo = token_major(hq, q);
    if (k.defined()) ko = token_major(hk, q);
    if (hq.B * (hq.L + hk.L) > 0)
      rc = k2b_qk_norm_rope(q.data_ptr(), ptr(k), wq.data_ptr(), ptr(wk), ptr(fq), ptr(fk), qo.data_ptr(),
                            k.defined() ? ko.data_ptr() : nullptr, fits_int(hq.B, "qk_norm_rope"),
                            fits_int(hq.L, "qk_norm_rope"), fits_int(hk.L, "qk_norm_rope"),
                            fits_int(hq.H, "qk_norm_rope"), fits_int(hk.H, "qk_norm_rope"), (int)hq.D, hq.sb, hq.sh,
                            hq.st, hk.sb, hk.sh, hk.st, fqb, fkb, (float)eps_q, (float)eps_k, code, stream());
  }
  if (rc) return failed("k2b_qk_norm_rope", rc);
  PyObject* pair = PyTuple_New(2);
  if (!pair) return nullptr;
  PyTuple_SET_ITEM(pair, 0, THPVariable_Wrap(std::move(qo)));
  if (ko.defined()) {
    PyTuple_SET_ITEM(pair, 1, THPVariable_Wrap(std::move(ko)));
  } else {
    Py_INCREF(Py_None);
    PyTuple_SET_ITEM(pair, 1, Py_None);
  }
  return pair;
  END_HANDLE_TH_ERRORS
}

// ------------------------------------------------------- cross_attention
// (q, k, v, lengths, mask, bias, scale or None)
PyObject* cross_attention(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_VALUE(n_args == 7, "cross_attention: 7 arguments expected");
  const at::Tensor& q = tensor(a[0], "cross_attention: q");
  const at::Tensor& k = tensor(a[1], "cross_attention: k");
  const at::Tensor& v = tensor(a[2], "cross_attention: v");
  const at::Tensor lengths = optional(a[3], "cross_attention: lengths");
  const at::Tensor mask = optional(a[4], "cross_attention: mask");
  const at::Tensor bias = optional(a[5], "cross_attention: bias");
  const int code = dtype_code(q, "cross_attention: q");
  const Heads hq = heads(q, "cross_attention: q");
  Heads hk = heads(k, "cross_attention: k"), hv = heads(v, "cross_attention: v");
  TORCH_CHECK_VALUE(k.sizes() == v.sizes() && hk.D == hq.D && (hk.B == 1 || hk.B == hq.B) && hk.H > 0 &&
                        hq.H % hk.H == 0 && k.scalar_type() == q.scalar_type() && v.scalar_type() == q.scalar_type(),
                    "cross_attention: q ", q.sizes(), " ", q.scalar_type(), ", k ", k.sizes(), " ", k.scalar_type(),
                    " and v ", v.sizes(), " ", v.scalar_type(), " do not go together");
  if (hk.B != hq.B) hk.sb = hv.sb = 0;
  const double scale = a[6] == Py_None ? 1.0 / std::sqrt((double)hq.D) : PyFloat_AsDouble(a[6]);
  if (PyErr_Occurred()) return nullptr;
  const int64_t B = hq.B, H = hq.H, Lq = hq.L, Lk = hk.L;
  TORCH_CHECK_VALUE(!lengths.defined() || (lengths.scalar_type() == at::kInt && lengths.dim() == 1 &&
                                           lengths.size(0) == B && lengths.is_contiguous()),
                    "cross_attention: lengths int32 [B] expected");
  int64_t ms[4] = {0, 0, 0, 0};
  if (mask.defined()) {
    const int64_t d = mask.dim();
    TORCH_CHECK_VALUE(mask.scalar_type() == at::kBool && (d == 2 || d == 4) && mask.size(d - 1) == Lk &&
                          (mask.size(0) == 1 || mask.size(0) == B) &&
                          (d == 2 || ((mask.size(1) == 1 || mask.size(1) == H) && (mask.size(2) == 1 || mask.size(2) == Lq))),
                      "cross_attention: mask bool [B|1, H|1, Lq|1, Lk] or [B|1, Lk] expected, got ", mask.scalar_type(),
                      " ", mask.sizes());
    for (int64_t i = 0; i + 1 < d; ++i) ms[i] = mask.size(i) == 1 ? 0 : mask.stride(i);
    ms[3] = mask.stride(d - 1);
  }
  int64_t bs = 0;
  if (bias.defined()) {
    TORCH_CHECK_VALUE(bias.scalar_type() == at::kFloat && bias.dim() == 2 && (bias.size(0) == 1 || bias.size(0) == B) &&
                          bias.size(1) == Lk && (Lk <= 1 || bias.stride(1) == 1),
                      "cross_attention: bias fp32 [B|1, Lk] with contiguous keys expected");
    bs = bias.size(0) == 1 ? 0 : bias.stride(0);
  }
  on_device("cross_attention", q, {&k, &v, &lengths, &mask, &bias});
  at::Tensor out;
  int rc = 0;
  {
    NoGil free;
    out = at::empty({B, Lq, H * hq.D}, q.options());
    if (out.numel()) {
      const int bi = fits_int(B, "cross_attention"), hi = fits_int(H, "cross_attention"),
                qi = fits_int(Lq, "cross_attention"), ki = fits_int(Lk, "cross_attention");
      at::Tensor work;
      if (ms[1] || ms[2]) {  // depends on the head or the query: packed to bits first
        const long long bytes = k2b_cross_workspace_bytes(bi, hi, (int)hk.H, qi, ki, (int)hq.D, ms[0], ms[1], ms[2]);
        if (bytes > 0) work = at::empty({(int64_t)bytes}, q.options().dtype(at::kByte));
      }
      rc = k2b_cross_attention(q.data_ptr(), k.data_ptr(), v.data_ptr(), ptr(lengths), ptr(mask), ptr(bias),
                               out.data_ptr(), work.defined() ? work.data_ptr() : nullptr, bi, hi,
                               fits_int(hk.H, "cross_attention"), qi, ki, (int)hq.D, hq.sb, hq.sh, hq.st, hk.sb, hk.sh,
                               hk.st, hv.sb, hv.sh, hv.st, ms[0], ms[1], ms[2], ms[3], bs, (float)scale, code, stream());
    }
  }
  if (rc) return failed("k2b_cross_attention", rc);
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

PyMethodDef methods[] = {
    {"w4_linear", (PyCFunction)(void (*)(void))w4_linear, METH_FASTCALL, nullptr},
    {"qk_norm_rope", (PyCFunction)(void (*)(void))qk_norm_rope, METH_FASTCALL, nullptr},
    {"cross_attention", (PyCFunction)(void (*)(void))cross_attention, METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_bind", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__bind() {
  PyObject* native = PyImport_ImportModule("k2b._native");
  if (!native) return nullptr;
  k2b_error = PyObject_GetAttrString(native, "K2BError");
  Py_DECREF(native);
  return k2b_error ? PyModule_Create(&module) : nullptr;
}
