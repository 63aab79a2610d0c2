// The language-model launches (include/edsl_hip_lm.h) on torch tensors: the
// operand checks of mlir_edsl_hip/lm.py and the calls, natively, as
// csrc/torch_launch.cpp does for the dense layer. Each function returns the
// entry's status, or None where an argument is not taken: the Python path then
// names what is wrong. Checking a norm's operands through Python takes 9 us, here
// 0.4.
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/edsl_hip_lm.h"

#include "torch_lm.hpp"

namespace {

// What a call has found: an argument that is not taken ends it with None.
struct NotTaken {};

int type_code(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return EDSL_LM_F32;
    case at::kBFloat16: return EDSL_LM_BF16;
    case at::kHalf: return EDSL_LM_F16;
    case at::kChar: return EDSL_LM_I8;
    case at::kFloat8_e4m3fn: return EDSL_LM_E4M3;
    default: throw NotTaken{};
  }
}

const at::Tensor& tensor(PyObject* o) {
  if (!THPVariable_CheckExact(o)) throw NotTaken{};
  return THPVariable_Unpack(o);
}

bool given(PyObject* o) { return o != Py_None; }

void require(bool ok) {
  if (!ok) throw NotTaken{};
}

struct Mat {
  void* p = nullptr;
  int64_t ld = 0, rows = 0, cols = 0;
  int type = 0;
};

// A 2-D GPU tensor with unit inner stride.
Mat mat(const at::Tensor& t) {
  require(t.is_cuda() && t.layout() == at::kStrided && t.dim() == 2);
  require(t.size(1) <= 1 || t.stride(1) == 1);
  return {t.data_ptr(), t.stride(0), t.size(0), t.size(1), type_code(t.scalar_type())};
}

// One of `like`'s shape on its device.
Mat mat_like(PyObject* o, const at::Tensor& like, int64_t rows, int64_t cols) {
  const at::Tensor& t = tensor(o);
  const Mat m = mat(t);
  require(m.rows == rows && m.cols == cols && t.device() == like.device());
  return m;
}

// A contiguous vector of n elements on `like`'s device, or null for None.
const at::Tensor* vec(PyObject* o, const at::Tensor& like, int64_t n) {
  if (!given(o)) return nullptr;
  const at::Tensor& t = tensor(o);
  require(t.is_cuda() && t.layout() == at::kStrided && t.dim() == 1 && t.size(0) == n && t.is_contiguous() &&
          t.device() == like.device());
  return &t;
}

float* vec_f32(PyObject* o, const at::Tensor& like, int64_t n) {
  const at::Tensor* t = vec(o, like, n);
  if (!t) return nullptr;
  require(t->scalar_type() == at::kFloat);
  return static_cast<float*>(t->data_ptr());
}

// Tokens: the pointer and whether they are 64 bits; null for None.
void* ids(PyObject* o, const at::Tensor& like, int64_t n, int* ids64) {
  const at::Tensor* t = vec(o, like, n);
  if (!t) return nullptr;
  require(t->scalar_type() == at::kLong || t->scalar_type() == at::kInt);
  *ids64 = t->scalar_type() == at::kLong;
  return t->data_ptr();
}

bool is_float(int type) { return type <= EDSL_LM_F16; }

float number(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw NotTaken{};
  return static_cast<float>(v);
}

int64_t integer(PyObject* o) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw NotTaken{};
  return v;
}

// The handle of the caller's stream object, or of the current stream. Asked for
// after the checks, so that host tensors are refused without the GPU.
void* stream_of(PyObject* stream, PyObject* current) {
  PyObject* handle = given(stream) ? PyObject_GetAttrString(stream, "cuda_stream") : PyObject_CallNoArgs(current);
  if (handle == nullptr) throw NotTaken{};
  void* s = PyLong_AsVoidPtr(handle);
  Py_DECREF(handle);
  if (s == nullptr && PyErr_Occurred()) throw NotTaken{};
  return s;
}

// Runs f(args) -> status without the GIL's checks leaking C++ exceptions.
template <typename F>
PyObject* taken(PyObject* const* args, Py_ssize_t n, Py_ssize_t want, F&& f) {
  if (n != want) {
    PyErr_SetString(PyExc_TypeError, "wrong number of arguments");
    return nullptr;
  }
  int rc;
  try {
    rc = f(args);
  } catch (...) {  // NotTaken, or a tensor without storage: the Python path raises
    PyErr_Clear();
    Py_RETURN_NONE;
  }
  return PyLong_FromLong(rc);
}

template <typename F>
int released(F&& call) {
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = call();
  Py_END_ALLOW_THREADS
  return rc;
}

}  // namespace

// rms_norm(X, weight, Y, residual, total, scales, rstd, eps, stream, current)
PyObject* edsl_torch_rms_norm(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return taken(args, n, 10, [](PyObject* const* a) {
    const at::Tensor& X = tensor(a[0]);
    const Mat x = mat(X), y = mat_like(a[2], X, x.rows, x.cols);
    const at::Tensor* w = vec(a[1], X, x.cols);
    require(w && is_float(x.type));
    const int wt = type_code(w->scalar_type());
    require(wt == x.type || wt == EDSL_LM_F32);
    const bool eight = y.type > EDSL_LM_F16;
    require((eight || y.type == x.type) && eight == given(a[5]));
    const Mat r = given(a[3]) ? mat_like(a[3], X, x.rows, x.cols) : Mat{};
    const Mat t = given(a[4]) ? mat_like(a[4], X, x.rows, x.cols) : Mat{};
    require((!given(a[3]) || r.type == x.type) && (!given(a[4]) || t.type == x.type));
    float* const scales = vec_f32(a[5], X, x.rows);
    float* const rstd = vec_f32(a[6], X, x.rows);
    const float eps = number(a[7]);
    void* const stream = stream_of(a[8], a[9]);
    const void* const wp = w->data_ptr();
    return released([&] {
      return edsl_hip_rms_norm_launch(x.p, x.ld, r.p, r.ld, wp, wt, t.p, t.ld, y.p, y.ld, y.type, scales, rstd, x.rows,
                                      x.cols, x.type, eps, stream);
    });
  });
}

// rms_norm_backward(dY, H, weight, rstd, dX, dweight, dh, stream, current)
PyObject* edsl_torch_rms_norm_backward(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return taken(args, n, 9, [](PyObject* const* a) {
    const at::Tensor& DY = tensor(a[0]);
    const Mat dy = mat(DY), h = mat_like(a[1], DY, dy.rows, dy.cols), dx = mat_like(a[4], DY, dy.rows, dy.cols);
    const Mat dh = given(a[6]) ? mat_like(a[6], DY, dy.rows, dy.cols) : Mat{};
    require(is_float(dy.type) && h.type == dy.type && dx.type == dy.type && (!given(a[6]) || dh.type == dy.type));
    const at::Tensor* w = vec(a[2], DY, dy.cols);
    require(w && given(a[3]));
    const int wt = type_code(w->scalar_type());
    require(wt == dy.type || wt == EDSL_LM_F32);
    float* const rstd = vec_f32(a[3], DY, dy.rows);
    float* const dw = vec_f32(a[5], DY, dy.cols);
    void* const stream = stream_of(a[7], a[8]);
    const void* const wp = w->data_ptr();
    return released([&] {
      return edsl_hip_rms_norm_backward_launch(dy.p, dy.ld, h.p, h.ld, wp, wt, rstd, dh.p, dh.ld, dx.p, dx.ld, dw,
                                               dy.rows, dy.cols, dy.type, stream);
    });
  });
}

// q4_dense(X, packed, K, N, group_size, scale_type, has_zeros, b, Y, epilogue, alpha, x_scales, stream, current)
PyObject* edsl_torch_q4_dense(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return taken(args, n, 14, [](PyObject* const* a) {
    const at::Tensor &X = tensor(a[0]), &W = tensor(a[1]);
    const int64_t K = integer(a[2]), N = integer(a[3]);
    const Mat x = mat(X), y = mat_like(a[8], X, x.rows, N);
    require(x.cols == K && is_float(y.type) && W.is_cuda() && W.device() == X.device());
    const at::Tensor* b = vec(a[7], X, N);
    const int bt = b ? type_code(b->scalar_type()) : 0;
    require(is_float(bt));
    const float* const xs = vec_f32(a[11], X, x.rows);
    const int group = static_cast<int>(integer(a[4])), st = static_cast<int>(integer(a[5]));
    const int zeros = static_cast<int>(integer(a[6])), epi = static_cast<int>(integer(a[9]));
    const float alpha = number(a[10]);
    void* const stream = stream_of(a[12], a[13]);
    const void *const wp = W.data_ptr(), *const bp = b ? b->data_ptr() : nullptr;
    return released([&] {
      return edsl_hip_q4_dense_launch(x.p, x.ld, x.type, xs, wp, bp, bt, y.p, y.ld, y.type, x.rows, N, K, group, st,
                                      zeros, epi, alpha, stream);
    });
  });
}

// token_logprobs(logits, tokens, logprobs, lse, entropy, top_logprobs, top_ids, scale, stream, current)
PyObject* edsl_torch_token_logprobs(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return taken(args, n, 10, [](PyObject* const* a) {
    const at::Tensor& L = tensor(a[0]);
    const Mat l = mat(L);
    require(is_float(l.type));
    int ids64 = 1, k = 0;
    void* const tokens = ids(a[1], L, l.rows, &ids64);
    float *const lp = vec_f32(a[2], L, l.rows), *const lse = vec_f32(a[3], L, l.rows),
                 *const ent = vec_f32(a[4], L, l.rows);
    require(!lp || tokens);
    require(given(a[5]) == given(a[6]));
    float* top = nullptr;
    void* top_ids = nullptr;
    if (given(a[6])) {
      const at::Tensor &T = tensor(a[5]), &I = tensor(a[6]);
      for (const at::Tensor* t : {&T, &I})
        require(t->is_cuda() && t->layout() == at::kStrided && t->dim() == 2 && t->is_contiguous() &&
                t->size(0) == l.rows && t->device() == L.device());
      require(T.size(1) == I.size(1) && I.size(1) <= EDSL_LM_MAX_TOP && T.scalar_type() == at::kFloat);
      require(I.scalar_type() == at::kLong || I.scalar_type() == at::kInt);
      const int wide = I.scalar_type() == at::kLong;
      require(!tokens || wide == ids64);
      ids64 = wide;
      k = static_cast<int>(I.size(1));
      top = static_cast<float*>(T.data_ptr());
      top_ids = I.data_ptr();
    }
    const float scale = number(a[7]);
    void* const stream = stream_of(a[8], a[9]);
    return released([&] {
      return edsl_hip_token_logprobs_launch(l.p, l.ld, l.type, tokens, ids64, lp, lse, ent, top, top_ids, k, l.rows,
                                            l.cols, scale, stream);
    });
  });
}

// token_logprobs_backward(logits, tokens, lse, dlogits, dlogprobs, entropy, dentropy, scale, stream, current)
PyObject* edsl_torch_token_logprobs_backward(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return taken(args, n, 10, [](PyObject* const* a) {
    const at::Tensor& L = tensor(a[0]);
    const Mat l = mat(L), dl = mat_like(a[3], L, l.rows, l.cols);
    require(is_float(l.type) && dl.type == l.type && given(a[2]));
    int ids64 = 1;
    void* const tokens = ids(a[1], L, l.rows, &ids64);
    float *const lse = vec_f32(a[2], L, l.rows), *const dlp = vec_f32(a[4], L, l.rows),
                 *const ent = vec_f32(a[5], L, l.rows), *const dent = vec_f32(a[6], L, l.rows);
    require((!dlp || tokens) && (!dent || ent));
    const float scale = number(a[7]);
    void* const stream = stream_of(a[8], a[9]);
    return released([&] {
      return edsl_hip_token_logprobs_backward_launch(l.p, l.ld, l.type, tokens, ids64, lse, dlp, ent, dent, dl.p, dl.ld,
                                                     l.rows, l.cols, scale, stream);
    });
  });
}
