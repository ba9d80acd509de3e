// Host side of the calls whose kernels are shorter than their Python path:
// those an FP8 linear makes (quantisation and GEMM) and those of a paged cache's
// step (append and attention), as a CPython extension: argument checks, output
// allocation and the C ABI call in one crossing.  Through Python checks, torch.empty
// and ctypes a call costs the host 10-13 us (a paged cache's 20-40), more than a
// kernel on a few hundred rows takes; here 5.3
// (GEMM) and 5.6 us (quantisation), of which the launch is about half.  An
// FP8Linear of 512 tokens: 24.6 -> 14.9 us a call, of 2079 tokens per tensor
// 29.5 -> 20.2.
//
// Each function serves the plain case (exact tensors on one GPU, types and
// layouts the kernels take as they are) and returns None for everything else,
// including a call the library refuses: the Python caller then runs its general
// path, which converts, checks and raises as documented there.  A HIP error is
// raised here: the library's status has taken it from the runtime, so a second
// attempt would look clean, on work that may have failed.
//
// The C ABI functions are those of the library the Python side has loaded,
// passed to bind() by address.
#include <Python.h>

#include <cmath>

#include <ATen/ATen.h>
#include <ATen/PythonTorchFunctionTLS.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/fvsr.h"

namespace {

struct Abi {
  decltype(&fvsr_quant_workspace_floats) quant_workspace_floats;
  decltype(&fvsr_quant_fp8_dt) quant_fp8_dt;
  decltype(&fvsr_fp8_gemm) fp8_gemm;
  decltype(&fvsr_gemm_amax_parts) gemm_amax_parts;
} abi{};

// The tensor behind a Python argument, or nullptr if it is not a plain tensor
// (or parameter) on a GPU.
const at::Tensor* plain_gpu(PyObject* o) {
  if (!THPVariable_CheckExact(o)) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(o);
  return t.is_cuda() && t.layout() == at::kStrided ? &t : nullptr;
}

// Modes that intercept torch calls see the Python path's calls instead.
bool modes_active() {
  return at::impl::torch_function_mode_enabled() ||
         c10::impl::TorchDispatchModeTLS::any_modes_set();
}

void* stream_of(const at::Tensor& t) {
  return (void*)c10::hip::getCurrentHIPStream(t.device().index()).stream();
}

int dtype_code(const at::Tensor& t) {
  switch (t.scalar_type()) {
    case at::kBFloat16: return FVSR_DT_BF16;
    case at::kHalf: return FVSR_DT_F16;
    case at::kFloat: return FVSR_DT_F32;
    default: return -1;
  }
}

// What a call returns for a status other than FVSR_OK: None for one decided
// before any launch, an exception for a HIP error (worded as the Python path's).
PyObject* not_done(int rc, const char* what) {
  if (rc != FVSR_EHIP) Py_RETURN_NONE;
  PyErr_Format(PyExc_RuntimeError, "%s failed: HIP launch error (status %d)", what, rc);
  return nullptr;
}

// quantize(x2, per_token, gelu) -> (codes, scale) or None
PyObject* quantize(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 3 || !abi.quant_fp8_dt) Py_RETURN_NONE;
  const at::Tensor* x = plain_gpu(args[0]);
  if (!x || x->dim() != 2 || x->numel() == 0 || x->stride(1) != 1 || modes_active())
    Py_RETURN_NONE;
  const int dt = dtype_code(*x);
  if (dt < 0) Py_RETURN_NONE;
  const int per_token = PyObject_IsTrue(args[1]), gelu = PyObject_IsTrue(args[2]);
  if (per_token < 0 || gelu < 0) return nullptr;  // no truth value: its exception
  const int64_t M = x->size(0), K = x->size(1);
  const int mode = per_token ? FVSR_SCALE_ROW : FVSR_SCALE_TENSOR;
  at::Tensor q = at::empty({M, K}, x->options().dtype(at::kFloat8_e4m3fn));
  const auto f32 = x->options().dtype(at::kFloat);
  at::Tensor s = per_token ? at::empty({M, 1}, f32) : at::empty({1}, f32);
  const int64_t wn = abi.quant_workspace_floats(M, K, mode);
  at::Tensor ws;
  if (wn > 0) ws = at::empty({wn}, f32);
  void* st = stream_of(*x);
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = abi.quant_fp8_dt(x->data_ptr(), dt, M, K, x->stride(0), mode, gelu, q.data_ptr(),
                        (float*)s.data_ptr(), wn > 0 ? (float*)ws.data_ptr() : nullptr, wn, st);
  Py_END_ALLOW_THREADS
  if (rc != FVSR_OK) return not_done(rc, gelu ? "fused_gelu_quant_fp8" : "quantize_fp8");
  PyObject* qo = THPVariable_Wrap(std::move(q));
  PyObject* so = qo ? THPVariable_Wrap(std::move(s)) : nullptr;
  PyObject* r = so ? PyTuple_Pack(2, qo, so) : nullptr;
  Py_XDECREF(qo);
  Py_XDECREF(so);
  return r;
  END_HANDLE_TH_ERRORS
}

// gemm(x8, s, w8, w_scale, bias | None, amax_part | None) -> out or None; with
// amax_part the row-max epilogue.
PyObject* gemm(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 6 || !abi.fp8_gemm) Py_RETURN_NONE;
  const at::Tensor* t[6] = {};
  for (int i = 0; i < 6; ++i) {
    if (args[i] == Py_None) {
      if (i < 4) Py_RETURN_NONE;
      continue;
    }
    t[i] = plain_gpu(args[i]);
    if (!t[i] || t[i]->device() != t[0]->device()) Py_RETURN_NONE;
  }
  const at::Tensor &x = *t[0], &s = *t[1], &w = *t[2], &wsc = *t[3];
  if (x.scalar_type() != at::kFloat8_e4m3fn || w.scalar_type() != at::kFloat8_e4m3fn ||
      x.dim() != 2 || w.dim() != 2 || x.size(1) != w.size(1) || x.stride(1) != 1 ||
      w.stride(1) != 1 || s.scalar_type() != at::kFloat || wsc.scalar_type() != at::kFloat ||
      !s.is_contiguous() || !wsc.is_contiguous())
    Py_RETURN_NONE;
  const int64_t M = x.size(0), K = x.size(1), N = w.size(0), ns = s.numel(), nw = wsc.numel();
  if ((ns != 1 && ns != M) || (nw != 1 && nw != N)) Py_RETURN_NONE;
  if (t[4] && (t[4]->scalar_type() != at::kBFloat16 || t[4]->dim() != 1 || t[4]->numel() != N ||
               !t[4]->is_contiguous()))
    Py_RETURN_NONE;
  if (t[5] && (t[5]->scalar_type() != at::kFloat || !t[5]->is_contiguous() ||
               t[5]->numel() < M * abi.gemm_amax_parts(N)))
    Py_RETURN_NONE;
  if (modes_active()) Py_RETURN_NONE;
  at::Tensor out = at::empty({M, N}, x.options().dtype(at::kBFloat16));
  void* st = stream_of(x);
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = abi.fp8_gemm(x.data_ptr(), x.stride(0), (const float*)s.data_ptr(),
                    ns == M && M != 1 ? FVSR_SCALE_ROW : FVSR_SCALE_TENSOR, w.data_ptr(),
                    w.stride(0), (const float*)wsc.data_ptr(),
                    nw == N && N != 1 ? FVSR_SCALE_ROW : FVSR_SCALE_TENSOR,
                    t[4] ? t[4]->data_ptr() : nullptr, out.data_ptr(), N, M, N, K,
                    t[5] ? FVSR_EPI_ROWMAX : FVSR_EPI_BIAS,
                    t[5] ? (float*)t[5]->data_ptr() : nullptr, nullptr, nullptr, st);
  Py_END_ALLOW_THREADS
  if (rc != FVSR_OK) return not_done(rc, "fp8_gemm");
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// ---------------------------------------------------------------------------
// The paged cache.
// ---------------------------------------------------------------------------
struct PagedAbi {
  decltype(&fvsr_kv_append_workspace_floats) append_floats;
  decltype(&fvsr_kv_append) append;
  decltype(&fvsr_paged_attn_workspace_floats) attn_floats;
  decltype(&fvsr_paged_attn) attn;
} paged{};

// An optional tensor on `dev`: true where there is None (t stays null) or a
// plain tensor of that device.
bool optional_on(PyObject* o, const at::Device& dev, const at::Tensor*& t) {
  if (o == Py_None) return true;
  t = plain_gpu(o);
  return t && t->device() == dev;
}

bool aligned16(const at::Tensor& t) { return ((uintptr_t)t.data_ptr() & 15) == 0; }

// [T, heads, D] rows as the kernels load them.
bool rows_ok(const at::Tensor& x, int64_t T, int64_t D) {
  if (x.dim() != 3 || x.size(0) != T || x.size(2) != D || x.size(1) <= 0 || x.stride(2) != 1)
    return false;
  const int64_t b = x.element_size();
  return aligned16(x) && x.stride(0) * b % 16 == 0 && x.stride(1) * b % 16 == 0;
}

// The cache of a call with T rows from (pages, page_table, lengths, cu_tokens).
bool cache_of(PyObject* pages, PyObject* table, PyObject* lengths, PyObject* cu, int64_t T,
              const at::Device& dev, fvsr_kv_cache& c) {
  if (!PyTuple_Check(pages) || PyTuple_GET_SIZE(pages) != 4) return false;
  const at::Tensor* p[4];
  for (int i = 0; i < 4; ++i) {
    p[i] = plain_gpu(PyTuple_GET_ITEM(pages, i));
    if (!p[i] || p[i]->device() != dev || !p[i]->is_contiguous() ||
        p[i]->scalar_type() != (i < 2 ? at::kFloat8_e4m3fn : at::kFloat8_e8m0fnu))
      return false;
  }
  const at::Tensor &k = *p[0], &v = *p[1];
  if (k.dim() != 4 || v.dim() != 4 || k.size(2) != FVSR_PAGE) return false;
  const int64_t N = k.size(0), H = k.size(1), D = k.size(3);
  if (H <= 0 || v.size(0) != N || v.size(1) != H || v.size(2) != D || v.size(3) != FVSR_PAGE)
    return false;
  for (int i = 2; i < 4; ++i)
    if (p[i]->dim() != 2 || p[i]->size(0) != N || p[i]->size(1) != H) return false;
  const at::Tensor *t = plain_gpu(table), *l = plain_gpu(lengths), *u = nullptr;
  if (!t || !l || t->device() != dev || l->device() != dev || !optional_on(cu, dev, u))
    return false;
  if (t->scalar_type() != at::kInt || l->scalar_type() != at::kInt ||
      (u && u->scalar_type() != at::kInt))
    return false;
  if (t->dim() != 2 || l->dim() != 1) return false;
  const int64_t B = t->size(0), P = t->size(1);
  if (B <= 0 || P <= 0 || t->stride(1) != 1 || (B > 1 && t->stride(0) < P)) return false;
  if (l->size(0) != B || !l->is_contiguous()) return false;
  if (u ? u->dim() != 1 || u->size(0) != B + 1 || !u->is_contiguous() : T % B != 0) return false;
  c = fvsr_kv_cache{k.data_ptr(), v.data_ptr(), p[2]->data_ptr(), p[3]->data_ptr(), N, H, D,
                    (const int32_t*)t->data_ptr(), B > 1 ? t->stride(0) : P, P,
                    (const int32_t*)l->data_ptr(), u ? (const int32_t*)u->data_ptr() : nullptr, B};
  return true;
}

// FVSR_NORM_* of an optional weight, or -1.
int norm_of(const at::Tensor* w, int64_t heads, int64_t D) {
  if (!w) return FVSR_NORM_NONE;
  if (w->dim() != 1 || !w->is_contiguous() || !aligned16(*w) || dtype_code(*w) < 0) return -1;
  return w->size(0) == D ? FVSR_NORM_HEAD : w->size(0) == heads * D ? FVSR_NORM_ROW : -1;
}

// The kernels run on their tensors' device, whichever is current.
bool is_current(const at::Device& dev) {
  return c10::hip::current_device() == dev.index();
}

// append_kv(pages, k, v, page_table, lengths, cu_tokens, freqs_cis, positions,
// k_weight, q, q_weight, eps) -> the turned q, True without a q, or None
PyObject* append_kv(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 12 || !paged.append) Py_RETURN_NONE;
  const at::Tensor *k = plain_gpu(args[1]), *v = plain_gpu(args[2]);
  if (!k || !v || k->dim() != 3 || k->numel() == 0) Py_RETURN_NONE;
  const at::Device dev = k->device();
  const int64_t T = k->size(0);
  const int dt = dtype_code(*k);
  fvsr_kv_cache c;
  if (dt < 0 || !is_current(dev) || v->device() != dev || v->scalar_type() != k->scalar_type() ||
      !cache_of(args[0], args[3], args[4], args[5], T, dev, c))
    Py_RETURN_NONE;
  const int64_t D = c.head_dim;
  if (!rows_ok(*k, T, D) || !rows_ok(*v, T, D) || k->size(1) != c.heads || v->size(1) != c.heads)
    Py_RETURN_NONE;
  const at::Tensor *f = nullptr, *pos = nullptr, *kw = nullptr, *q = nullptr, *qw = nullptr;
  if (!optional_on(args[6], dev, f) || !optional_on(args[7], dev, pos) ||
      !optional_on(args[8], dev, kw) || !optional_on(args[9], dev, q) ||
      !optional_on(args[10], dev, qw))
    Py_RETURN_NONE;
  if (q && (q->scalar_type() != k->scalar_type() || !rows_ok(*q, T, D))) Py_RETURN_NONE;
  const int64_t Hq = q ? q->size(1) : 0;
  if ((qw && !q) || (pos && !f) || (kw && qw && kw->scalar_type() != qw->scalar_type()))
    Py_RETURN_NONE;
  const int kn = norm_of(kw, c.heads, D), qn = norm_of(qw, Hq, D);
  if (kn < 0 || qn < 0) Py_RETURN_NONE;
  int64_t rows = 0;
  if (f) {
    if (f->scalar_type() != at::kComplexFloat || !f->is_contiguous() || f->dim() < 1 ||
        f->size(-1) != D / 2 || !aligned16(*f) || f->is_conj())
      Py_RETURN_NONE;
    rows = f->numel() / (D / 2);
    if (rows <= 0 || (!pos && rows < T)) Py_RETURN_NONE;
    if (pos && (pos->scalar_type() != at::kInt || pos->dim() != 1 || pos->size(0) != T ||
                !pos->is_contiguous()))
      Py_RETURN_NONE;
  }
  const double eps = PyFloat_AsDouble(args[11]);
  if (eps == -1.0 && PyErr_Occurred()) return nullptr;
  if (modes_active()) Py_RETURN_NONE;
  at::Tensor out, ws;
  if (q) out = at::empty({T, Hq, D}, q->options());
  const int64_t wn = paged.append_floats(T, kn);
  if (wn > 0) ws = at::empty({wn}, k->options().dtype(at::kFloat));
  void* st = stream_of(*k);
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = paged.append(&c, k->data_ptr(), k->stride(0), k->stride(1), v->data_ptr(), v->stride(0),
                    v->stride(1), q ? q->data_ptr() : nullptr, q ? q->stride(0) : 0,
                    q ? q->stride(1) : 0, Hq, q ? out.data_ptr() : nullptr, dt, T,
                    kw ? kw->data_ptr() : nullptr, kn, qw ? qw->data_ptr() : nullptr, qn,
                    kw ? dtype_code(*kw) : qw ? dtype_code(*qw) : 0, (float)eps,
                    f ? (const float*)f->data_ptr() : nullptr, rows,
                    pos ? (const int32_t*)pos->data_ptr() : nullptr,
                    wn > 0 ? (float*)ws.data_ptr() : nullptr, wn, st);
  Py_END_ALLOW_THREADS
  if (rc != FVSR_OK) return not_done(rc, "append_kv");
  if (!q) Py_RETURN_TRUE;
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// paged_attention(q, pages, page_table, lengths, cu_tokens, causal, keep,
// sm_scale | None) -> out or None
PyObject* paged_attention(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 8 || !paged.attn) Py_RETURN_NONE;
  const at::Tensor* q = plain_gpu(args[0]);
  if (!q || q->dim() != 3 || q->numel() == 0) Py_RETURN_NONE;
  const at::Device dev = q->device();
  const int64_t T = q->size(0), Hq = q->size(1);
  const int dt = dtype_code(*q);
  fvsr_kv_cache c;
  if ((dt != FVSR_DT_BF16 && dt != FVSR_DT_F16) || !is_current(dev) ||
      !cache_of(args[1], args[2], args[3], args[4], T, dev, c) || !rows_ok(*q, T, c.head_dim))
    Py_RETURN_NONE;
  const int causal = PyObject_IsTrue(args[5]);
  if (causal < 0) return nullptr;  // no truth value: its exception
  const at::Tensor* keep = nullptr;
  if (!optional_on(args[6], dev, keep)) Py_RETURN_NONE;
  int64_t nq = 0, nk = 0;
  if (keep) {
    const int64_t d = keep->dim();
    if (keep->scalar_type() != at::kBool || !keep->is_contiguous() || keep->numel() == 0 ||
        (d != 4 && !(d == 3 && c.sequences == 1)) || keep->size(d - 3) != Hq ||
        (d == 4 && keep->size(0) != c.sequences))
      Py_RETURN_NONE;
    nq = keep->size(d - 2), nk = keep->size(d - 1);
  }
  double scale = 1.0 / std::sqrt((double)c.head_dim);
  if (args[7] != Py_None) {
    scale = PyFloat_AsDouble(args[7]);
    if (scale == -1.0 && PyErr_Occurred()) return nullptr;
  }
  if (modes_active()) Py_RETURN_NONE;
  at::Tensor out = at::empty({T, Hq, c.head_dim}, q->options()), ws;
  const int64_t wn = paged.attn_floats(&c, T, Hq, keep != nullptr);
  if (wn > 0) ws = at::empty({wn}, q->options().dtype(at::kFloat));
  void* st = stream_of(*q);
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = paged.attn(&c, q->data_ptr(), q->stride(0), q->stride(1), Hq, out.data_ptr(), out.stride(0),
                  out.stride(1), dt, T, causal, keep ? (const uint8_t*)keep->data_ptr() : nullptr,
                  nq, nk, (float)scale, 1, wn > 0 ? (float*)ws.data_ptr() : nullptr, wn, st);
  Py_END_ALLOW_THREADS
  if (rc != FVSR_OK) return not_done(rc, "paged_attention");
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// bind_paged(append_workspace_floats, append, attn_workspace_floats, attn).
PyObject* bind_paged(PyObject*, PyObject* args) {
  unsigned long long p[4];
  if (!PyArg_ParseTuple(args, "KKKK", &p[0], &p[1], &p[2], &p[3])) return nullptr;
  paged.append_floats = (decltype(paged.append_floats))(uintptr_t)p[0];
  paged.append = (decltype(paged.append))(uintptr_t)p[1];
  paged.attn_floats = (decltype(paged.attn_floats))(uintptr_t)p[2];
  paged.attn = (decltype(paged.attn))(uintptr_t)p[3];
  Py_RETURN_NONE;
}

// bind(quant_workspace_floats, quant_fp8_dt, fp8_gemm, gemm_amax_parts): the
// addresses of the C ABI functions.
PyObject* bind(PyObject*, PyObject* args) {
  unsigned long long p[4];
  if (!PyArg_ParseTuple(args, "KKKK", &p[0], &p[1], &p[2], &p[3])) return nullptr;
  abi.quant_workspace_floats = (decltype(abi.quant_workspace_floats))(uintptr_t)p[0];
  abi.quant_fp8_dt = (decltype(abi.quant_fp8_dt))(uintptr_t)p[1];
  abi.fp8_gemm = (decltype(abi.fp8_gemm))(uintptr_t)p[2];
  abi.gemm_amax_parts = (decltype(abi.gemm_amax_parts))(uintptr_t)p[3];
  Py_RETURN_NONE;
}

PyMethodDef kMethods[] = {
    {"bind", bind, METH_VARARGS, "addresses of the C ABI functions"},
    {"quantize", (PyCFunction)(void*)quantize, METH_FASTCALL, "quantize(x2, per_token, gelu)"},
    {"gemm", (PyCFunction)(void*)gemm, METH_FASTCALL, "gemm(x8, s, w8, w_scale, bias, amax_part)"},
    {"bind_paged", bind_paged, METH_VARARGS, "addresses of the paged cache's C ABI functions"},
    {"append_kv", (PyCFunction)(void*)append_kv, METH_FASTCALL,
     "append_kv(pages, k, v, page_table, lengths, cu_tokens, freqs_cis, positions, k_weight, q, "
     "q_weight, eps)"},
    {"paged_attention", (PyCFunction)(void*)paged_attention, METH_FASTCALL,
     "paged_attention(q, pages, page_table, lengths, cu_tokens, causal, keep, sm_scale)"},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_fvsr_host", nullptr, -1, kMethods};

}  // namespace

// torch_version: the torch whose headers this was compiled against.
PyMODINIT_FUNC PyInit__fvsr_host() {
  PyObject* m = PyModule_Create(&kModule);
  if (m && PyModule_AddStringConstant(m, "torch_version", FVSR_TORCH_VERSION) < 0) Py_CLEAR(m);
  return m;
}
