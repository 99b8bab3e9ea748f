// The tensor-level calls of the Python package (forward, backward, linear_*, layernorm_*, embedding_*, paged_*, sample) as a CPython extension
// over the C ABI of libattn_sm100.so.
//
// What bounds small calls is the host: with these functions written in Python, a forward and backward of
// B=1 T=40 H=2 spent 39 us per pass on the host (three allocations of 2.6 us each, 3.2 us to find the current
// stream, 11 to 13 converted arguments per ctypes call) around 16 us of GPU work.  Here the arguments are taken
// from the tensor objects directly, outputs come from the caching allocator without going through the operator
// dispatcher, and the stream is a thread-local read.  The GIL is released around the C ABI call, as ctypes does.
// The element-wise entry points and size queries that programs call through lib() get the same treatment (shorten_calls):
// converting their arguments took ctypes 0.5 to 1 us of the 2.8 us of a call, 2.3 of which the launch itself needs.
#include <Python.h>

#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/attn_sm100.h"
#include "../../include/layernorm_sm100.h"
#include "../../include/linear_sm100.h"
#include "../../include/tensor_sm100.h"
#include "../../include/xent_sm100.h"

#include <algorithm>
#include <cmath>
#include <tuple>
#include <utility>

namespace {

PyObject *g_error = nullptr;  // the package's AttnError(code, where)

// Raises AttnError for a non-zero status.
bool failed(int code, const char *where) {
    if (code == ATTN_OK) return false;
    PyObject *args = Py_BuildValue("(is)", code, where);
    PyObject *e = args && g_error ? PyObject_CallObject(g_error, args) : nullptr;
    Py_XDECREF(args);
    if (e) {
        PyErr_SetObject(g_error, e);
        Py_DECREF(e);
    } else if (!PyErr_Occurred()) {
        PyErr_Format(PyExc_RuntimeError, "%s failed with status %d", where, code);
    }
    return true;
}

// One positional argument list, read with checks that set a Python error; `ok` turns false on the first bad one.
struct Args {
    PyObject *const *v;
    bool ok = true;

    Args(PyObject *const *args, Py_ssize_t n, Py_ssize_t want) : v(args) {
        if (n != want) {
            PyErr_Format(PyExc_TypeError, "expected %zd arguments, got %zd", want, n);
            ok = false;
        }
    }
    const at::Tensor *tensor(int i) {
        if (!ok) return nullptr;
        if (!THPVariable_Check(v[i])) {
            PyErr_Format(PyExc_TypeError, "argument %d must be a tensor", i);
            ok = false;
            return nullptr;
        }
        return &THPVariable_Unpack(v[i]);
    }
    // A tensor an output is allocated next to: on a CUDA device, with at least one dimension.
    const at::Tensor *cuda(int i) {
        const at::Tensor *t = tensor(i);
        if (ok && (!t->is_cuda() || t->dim() < 1 || t->size(-1) < 1)) {
            PyErr_SetString(PyExc_ValueError, "expected a CUDA tensor with a non-empty last dimension");
            ok = false;
        }
        return ok ? t : nullptr;
    }
    template <class T>
    T *ptr(int i) {  // None gives NULL
        if (!ok || v[i] == Py_None) return nullptr;
        const at::Tensor *t = tensor(i);
        return ok ? static_cast<T *>(t->data_ptr()) : nullptr;
    }
    float *f32(int i) { return ptr<float>(i); }
    long integer(int i) {
        if (!ok) return 0;
        const long r = PyLong_AsLong(v[i]);
        if (r == -1 && PyErr_Occurred()) ok = false;
        return r;
    }
    double real(int i) {
        if (!ok) return 0;
        const double r = PyFloat_AsDouble(v[i]);
        if (r == -1.0 && PyErr_Occurred()) ok = false;
        return r;
    }
    // None: the current stream of the current device; else a cudaStream_t as an integer.
    void *stream(int i) {
        if (!ok) return nullptr;
        if (v[i] == Py_None) return c10::cuda::getCurrentCUDAStream().stream();
        void *s = PyLong_AsVoidPtr(v[i]);
        if (PyErr_Occurred()) ok = false;
        return s;
    }
};

at::Tensor alloc(at::IntArrayRef shape, at::ScalarType type, const at::Tensor &beside) {
    return at::detail::empty_cuda(shape, type, beside.device(), std::nullopt);
}

PyObject *value_error(const char *text) {
    PyErr_SetString(PyExc_ValueError, text);
    return nullptr;
}

// forward(qkv, n_heads, flags, keep_copy) -> (out, out_copy or None, lse, saved, (B, T, H, D))
PyObject *forward(PyObject *, PyObject *const *args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    Args a(args, n, 4);
    const at::Tensor *qkv = a.tensor(0);
    const long H = a.integer(1), flags = a.integer(2);
    const int keep = a.ok ? PyObject_IsTrue(args[3]) : 0;
    if (!a.ok || keep < 0) return nullptr;
    if (!(qkv->is_cuda() && qkv->scalar_type() == at::kFloat && qkv->is_contiguous() && qkv->dim() == 3))
        return value_error("qkv must be a contiguous fp32 CUDA tensor of shape [B, T, 3C]");
    const int64_t B = qkv->size(0), T = qkv->size(1), C3 = qkv->size(2);
    if (H <= 0 || C3 % (3 * H) != 0) return value_error("last dimension must be 3 * n_heads * head_size");
    const int64_t C = C3 / 3, D = C / H;
    const size_t saved_bytes = attn_sm100_saved_bytes((int)B, (int)T, (int)H, (int)D);
    at::Tensor out = alloc({B, T, C}, at::kFloat, *qkv);
    at::Tensor copy;
    if (keep) copy = alloc({B, T, C}, at::kFloat, *qkv);
    at::Tensor lse = alloc({B, H, T}, at::kFloat, *qkv);
    at::Tensor saved = alloc({(int64_t)saved_bytes}, at::kByte, *qkv);
    void *stream = c10::cuda::getCurrentCUDAStream().stream();
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = attn_sm100_forward(static_cast<const float *>(qkv->data_ptr()), static_cast<float *>(out.data_ptr()),
                            keep ? static_cast<float *>(copy.data_ptr()) : nullptr, static_cast<float *>(lse.data_ptr()),
                            saved.data_ptr(), (int)B, (int)T, (int)H, (int)D, (int)flags, stream);
    Py_END_ALLOW_THREADS
    if (failed(rc, "attn_sm100_forward")) return nullptr;
    PyObject *second = keep ? THPVariable_Wrap(copy) : Py_NewRef(Py_None);
    return Py_BuildValue("(NNNN(iiii))", THPVariable_Wrap(out), second, THPVariable_Wrap(lse), THPVariable_Wrap(saved), (int)B,
                         (int)T, (int)H, (int)D);
    END_HANDLE_TH_ERRORS
}

// backward(saved, out, lse, dout, (B, T, H, D), flags) -> dqkv
PyObject *backward(PyObject *, PyObject *const *args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    Args a(args, n, 6);
    const void *saved = a.ptr<void>(0);
    const float *out = a.f32(1), *lse = a.f32(2);
    const at::Tensor *dout = a.tensor(3);
    const long flags = a.integer(5);
    int B, T, H, D;
    if (!a.ok || !PyArg_ParseTuple(args[4], "iiii", &B, &T, &H, &D)) return nullptr;
    if (!(dout->is_cuda() && dout->scalar_type() == at::kFloat && dout->is_contiguous() && dout->dim() == 3 &&
          dout->size(0) == B && dout->size(1) == T && dout->size(2) == (int64_t)H * D))
        return value_error("dout must be a contiguous fp32 CUDA tensor of shape [B, T, C]");
    at::Tensor dqkv = alloc({B, T, 3 * (int64_t)H * D}, at::kFloat, *dout);
    at::Tensor scratch = alloc({(int64_t)attn_sm100_backward_scratch_bytes(B, T, H, D)}, at::kByte, *dout);
    void *stream = c10::cuda::getCurrentCUDAStream().stream();
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = attn_sm100_backward(saved, out, lse, static_cast<const float *>(dout->data_ptr()),
                             static_cast<float *>(dqkv.data_ptr()), scratch.data_ptr(), B, T, H, D, (int)flags, stream);
    Py_END_ALLOW_THREADS
    if (failed(rc, "attn_sm100_backward")) return nullptr;
    return THPVariable_Wrap(dqkv);
    END_HANDLE_TH_ERRORS
}

// forward_into(qkv, out, out_copy, lse, saved, n_heads, flags, stream)
PyObject *forward_into(PyObject *, PyObject *const *args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    Args a(args, n, 8);
    const at::Tensor *qkv = a.tensor(0);
    float *out = a.f32(1), *copy = a.f32(2), *lse = a.f32(3);
    void *saved = a.ptr<void>(4);
    const long H = a.integer(5), flags = a.integer(6);
    void *stream = a.stream(7);
    if (!a.ok) return nullptr;
    if (qkv->dim() != 3 || H == 0) return value_error("qkv must have the shape [B, T, 3C]");
    const int B = (int)qkv->size(0), T = (int)qkv->size(1), D = (int)(qkv->size(2) / 3 / H);
    const float *x = static_cast<const float *>(qkv->data_ptr());
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = attn_sm100_forward(x, out, copy, lse, saved, B, T, (int)H, D, (int)flags, stream);
    Py_END_ALLOW_THREADS
    if (failed(rc, "attn_sm100_forward")) return nullptr;
    Py_RETURN_NONE;
    END_HANDLE_TH_ERRORS
}

// backward_into(saved, out, lse, dout, dqkv, scratch, n_heads, flags, stream)
PyObject *backward_into(PyObject *, PyObject *const *args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    Args a(args, n, 9);
    const void *saved = a.ptr<void>(0);
    const float *out = a.f32(1), *lse = a.f32(2);
    const at::Tensor *dout = a.tensor(3);
    float *dqkv = a.f32(4);
    void *scratch = a.ptr<void>(5);
    const long H = a.integer(6), flags = a.integer(7);
    void *stream = a.stream(8);
    if (!a.ok) return nullptr;
    if (dout->dim() != 3 || H == 0) return value_error("dout must have the shape [B, T, C]");
    const int B = (int)dout->size(0), T = (int)dout->size(1), D = (int)(dout->size(2) / H);
    const float *g = static_cast<const float *>(dout->data_ptr());
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = attn_sm100_backward(saved, out, lse, g, dqkv, scratch, B, T, (int)H, D, (int)flags, stream);
    Py_END_ALLOW_THREADS
    if (failed(rc, "attn_sm100_backward")) return nullptr;
    Py_RETURN_NONE;
    END_HANDLE_TH_ERRORS
}

// linear_forward(x, w, bias, planes, stream) -> y
PyObject *linear_forward(PyObject *, PyObject *const *args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    Args a(args, n, 5);
    const at::Tensor *x = a.cuda(0), *w = a.cuda(1);
    const float *bias = a.f32(2);
    void *planes = a.ptr<void>(3);
    void *stream = a.stream(4);
    if (!a.ok) return nullptr;
    const int64_t K = x->size(-1), N = w->size(0), M = x->numel() / K;
    c10::SmallVector<int64_t, 6> shape(x->sizes().begin(), x->sizes().end());
    shape.back() = N;
    at::Tensor y = alloc(shape, at::kFloat, *x);
    const float *xp = static_cast<const float *>(x->data_ptr()), *wp = static_cast<const float *>(w->data_ptr());
    float *yp = static_cast<float *>(y.data_ptr());
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = linear_sm100_forward(xp, wp, bias, yp, planes, (int)M, (int)N, (int)K, stream);
    Py_END_ALLOW_THREADS
    if (failed(rc, "linear_sm100_forward")) return nullptr;
    return THPVariable_Wrap(y);
    END_HANDLE_TH_ERRORS
}

// linear_backward(dy, x, w, dw, db, stream, want_dx) -> dx or None
PyObject *linear_backward(PyObject *, PyObject *const *args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    Args a(args, n, 7);
    const float *dy = a.f32(0);
    const at::Tensor *x = a.cuda(1), *w = a.cuda(2);
    float *dw = a.f32(3), *db = a.f32(4);
    void *stream = a.stream(5);
    const int want_dx = a.ok ? PyObject_IsTrue(args[6]) : 0;
    if (!a.ok || want_dx < 0) return nullptr;
    const int64_t K = x->size(-1), N = w->size(0), M = x->numel() / K;
    at::Tensor dx, scratch;
    if (want_dx) dx = alloc(x->sizes(), at::kFloat, *x);
    const size_t bytes = linear_sm100_backward_scratch_bytes((int)M, (int)N, (int)K);
    if (bytes) scratch = alloc({(int64_t)bytes}, at::kByte, *x);
    const float *xp = static_cast<const float *>(x->data_ptr()), *wp = static_cast<const float *>(w->data_ptr());
    float *dxp = want_dx ? static_cast<float *>(dx.data_ptr()) : nullptr;
    void *sp = bytes ? scratch.data_ptr() : nullptr;
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = linear_sm100_backward(dy, xp, wp, dxp, dw, db, sp, (int)M, (int)N, (int)K, stream);
    Py_END_ALLOW_THREADS
    if (failed(rc, "linear_sm100_backward")) return nullptr;
    if (!want_dx) Py_RETURN_NONE;
    return THPVariable_Wrap(dx);
    END_HANDLE_TH_ERRORS
}

// layernorm_forward(x, w, b, eps, stream) -> (y, mean, rstd)
PyObject *layernorm_forward(PyObject *, PyObject *const *args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    Args a(args, n, 5);
    const at::Tensor *x = a.cuda(0);
    const float *w = a.f32(1), *b = a.f32(2);
    const double eps = a.real(3);
    void *stream = a.stream(4);
    if (!a.ok) return nullptr;
    const int64_t C = x->size(-1), rows = x->numel() / C;
    at::Tensor y = alloc(x->sizes(), at::kFloat, *x);
    at::Tensor mean = alloc({rows}, at::kFloat, *x), rstd = alloc({rows}, at::kFloat, *x);
    const float *xp = static_cast<const float *>(x->data_ptr());
    float *yp = static_cast<float *>(y.data_ptr()), *mp = static_cast<float *>(mean.data_ptr()),
          *rp = static_cast<float *>(rstd.data_ptr());
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = layernorm_sm100_forward(xp, w, b, (float)eps, mp, rp, yp, (int)rows, (int)C, stream);
    Py_END_ALLOW_THREADS
    if (failed(rc, "layernorm_sm100_forward")) return nullptr;
    return Py_BuildValue("(NNN)", THPVariable_Wrap(y), THPVariable_Wrap(mean), THPVariable_Wrap(rstd));
    END_HANDLE_TH_ERRORS
}

// layernorm_backward(dy, x, mean, rstd, w, dw, db, dx, stream)
PyObject *layernorm_backward(PyObject *, PyObject *const *args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    Args a(args, n, 9);
    const at::Tensor *x = a.cuda(1);
    const float *dy = a.f32(0), *mean = a.f32(2), *rstd = a.f32(3), *w = a.f32(4);
    float *dw = a.f32(5), *db = a.f32(6), *dx = a.f32(7);
    void *stream = a.stream(8);
    if (!a.ok) return nullptr;
    const int64_t C = x->size(-1), rows = x->numel() / C;
    const float *xp = static_cast<const float *>(x->data_ptr());
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = layernorm_sm100_backward(dy, xp, mean, rstd, w, dw, db, dx, (int)rows, (int)C, stream);
    Py_END_ALLOW_THREADS
    if (failed(rc, "layernorm_sm100_backward")) return nullptr;
    Py_RETURN_NONE;
    END_HANDLE_TH_ERRORS
}

// ------------------------------------------------------------------------------------------
// Generation: the paged cache and the draw of a token.  These take tensors on any one device, current or not, and views
// whose rows lie apart; without a stream they run on the current stream of that device.
// ------------------------------------------------------------------------------------------
// The device of a call's tensors made current, and the stream of the call: outputs are allocated for it.
struct On {
    c10::cuda::CUDAGuard device;
    c10::cuda::OptionalCUDAStreamGuard own;
    void *stream;
    On(const at::Tensor &t, PyObject *s) : device(t.device()) {
        if (s == Py_None) {
            stream = c10::cuda::getCurrentCUDAStream().stream();
        } else {
            stream = PyLong_AsVoidPtr(s);
            if (!PyErr_Occurred()) own.reset_stream(c10::cuda::getStreamFromExternal(static_cast<cudaStream_t>(stream), t.device().index()));
        }
    }
};

bool is(const at::Tensor &t, at::ScalarType type, const at::Tensor &beside) {
    return t.scalar_type() == type && t.device() == beside.device();
}

struct Pages {
    const at::Tensor *k, *v, *table, *cu, *past;
    int type = 0, tokens = 0, seqs = 0, kv_heads = 0, D = 0, page_size = 0, pages = 0, width = 0;
    long long stride = 0;

    // `x` [tokens, ...] beside the cache in arguments i .. i + 4; false with a Python error set
    bool read(Args &a, const at::Tensor &x, int i) {
        k = a.tensor(i), v = a.tensor(i + 1), table = a.tensor(i + 2), cu = a.tensor(i + 3), past = a.tensor(i + 4);
        if (!a.ok) return false;
        if (!(x.is_cuda() && x.scalar_type() == at::kFloat && x.dim() == 2 && (x.size(1) < 2 || x.stride(1) == 1)))
            return value_error("the first argument must be an fp32 CUDA tensor of shape [tokens, columns] with its columns side by side") != nullptr;
        if (!((k->scalar_type() == at::kFloat || k->scalar_type() == at::kBFloat16) && k->dim() == 4 && k->device() == x.device()))
            return value_error("k_pages must be an fp32 or bf16 tensor of shape [pages, kv_heads, page_size, head_size] on the same device") != nullptr;
        if (!(v->scalar_type() == k->scalar_type() && v->sizes() == k->sizes() && v->device() == x.device()))
            return value_error("v_pages must be like k_pages") != nullptr;
        const auto size = k->sizes(), ks = k->strides(), vs = v->strides();
        const int64_t page = size[1] * size[2] * size[3];
        for (const auto &st : {ks, vs})  // (a dimension of one element may have any stride)
            if (size[0] * page <= 0 || (size[3] > 1 && st[3] != 1) || (size[2] > 1 && st[2] != size[3]) || (size[1] > 1 && st[1] != size[2] * size[3]) ||
                (size[0] > 1 && (st[0] != ks[0] || st[0] < page)))
                return value_error("pages must each be contiguous, and as far apart in v_pages as in k_pages") != nullptr;
        if (!(is(*table, at::kInt, x) && table->dim() == 2 && table->is_contiguous()))
            return value_error("page_table must be a contiguous int32 tensor of shape [sequences, pages] on the same device") != nullptr;
        if (!(is(*cu, at::kInt, x) && cu->dim() == 1 && cu->is_contiguous() && cu->size(0) == table->size(0) + 1))
            return value_error("cu_seqlens must be an int32 tensor of sequences + 1 values on the same device") != nullptr;
        if (!(is(*past, at::kInt, x) && past->dim() == 1 && past->is_contiguous() && past->size(0) == table->size(0)))
            return value_error("past must be an int32 tensor of one value a sequence on the same device") != nullptr;
        for (int64_t n : {x.size(0), k->size(0), k->size(1), k->size(2), table->size(0), table->size(1)})
            if (n > 0x7fffffff) return value_error("a size does not fit 31 bits") != nullptr;
        if (x.size(0) > 1 && x.stride(0) < x.size(1)) return value_error("rows must not overlap") != nullptr;
        type = k->scalar_type() == at::kBFloat16 ? ATTN_CACHE_BF16 : ATTN_CACHE_F32;
        tokens = (int)x.size(0), seqs = (int)table->size(0), width = (int)table->size(1);
        pages = (int)k->size(0), kv_heads = (int)k->size(1), page_size = (int)k->size(2), D = (int)k->size(3);
        stride = pages > 1 ? k->stride(0) : (long long)kv_heads * page_size * D;
        return true;
    }
};

// x[:, :columns] cut off from autograd, as every result here is: no gradient could come back for the keys and values beside
// them.  Without a trip through the dispatcher (a quarter of the time of a small append).
at::Tensor first_columns(const at::Tensor &x, int64_t columns) {
    const c10::TensorImpl *impl = x.unsafeGetTensorImpl();
    auto view = impl->shallow_copy_and_detach(impl->version_counter(), true);
    const int64_t sizes[2] = {x.size(0), columns}, strides[2] = {x.stride(0), x.stride(1)};
    view->set_sizes_and_strides(sizes, strides);
    return at::Tensor(std::move(view));
}

long long row_stride(const at::Tensor &x) { return x.size(0) > 1 ? x.stride(0) : x.size(1); }

// paged_append(qkv, k_pages, v_pages, page_table, cu_seqlens, past, rotary or None, rotary_pairs, stream) -> q
PyObject *paged_append(PyObject *, PyObject *const *args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    Args a(args, n, 9);
    const at::Tensor *qkv = a.tensor(0);
    Pages p;
    if (!a.ok || !p.read(a, *qkv, 1)) return nullptr;
    const at::Tensor *rotary = args[6] == Py_None ? nullptr : a.tensor(6);
    const int pairs = a.ok ? PyObject_IsTrue(args[7]) : 0;
    if (!a.ok || pairs < 0) return nullptr;
    const int64_t C = qkv->size(1) - 2 * (int64_t)p.kv_heads * p.D;
    if (C <= 0 || C % ((int64_t)p.kv_heads * p.D)) return value_error("qkv must have (n_heads + 2 kv_heads) * head_size columns, n_heads a multiple of kv_heads");
    if (rotary && !(is(*rotary, at::kFloat, *qkv) && rotary->dim() == 2 && rotary->is_contiguous() && rotary->size(0) > 0 && rotary->size(0) <= 0x7fffffff &&
                    rotary->size(1) > 0 && rotary->size(1) <= p.D && rotary->size(1) % 2 == 0))
        return value_error("rotary must be a contiguous fp32 tensor of shape [positions, an even number of columns up to head_size] on the same device");
    const On on(*qkv, args[8]);
    if (PyErr_Occurred()) return nullptr;
    at::Tensor q = rotary ? alloc({qkv->size(0), C}, at::kFloat, *qkv) : first_columns(*qkv, C);
    const int heads = (int)(C / p.D), positions = rotary ? (int)rotary->size(0) : 0, dim = rotary ? (int)rotary->size(1) : 0;
    const float *x = static_cast<const float *>(qkv->data_ptr()), *angles = rotary ? static_cast<const float *>(rotary->data_ptr()) : nullptr;
    float *out = rotary ? static_cast<float *>(q.data_ptr()) : nullptr;
    int rc = ATTN_OK;
    Py_BEGIN_ALLOW_THREADS
    if (p.tokens)
        rc = attn_sm100_paged_append(x, out, p.k->data_ptr(), p.v->data_ptr(), static_cast<const int *>(p.table->data_ptr()),
                                     static_cast<const int *>(p.cu->data_ptr()), static_cast<const int *>(p.past->data_ptr()), angles, row_stride(*qkv), p.stride,
                                     p.type, p.tokens, p.seqs, heads, p.kv_heads, p.D, p.page_size, p.pages, p.width, positions, dim, pairs, on.stream);
    Py_END_ALLOW_THREADS
    if (failed(rc, "attn_sm100_paged_append")) return nullptr;
    return THPVariable_Wrap(q);
    END_HANDLE_TH_ERRORS
}

// paged_attention(q, k_pages, v_pages, page_table, cu_seqlens, past, max_new, scale or None, out or None, stream) -> out
PyObject *paged_attention(PyObject *, PyObject *const *args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    Args a(args, n, 10);
    const at::Tensor *q = a.tensor(0);
    Pages p;
    if (!a.ok || !p.read(a, *q, 1)) return nullptr;
    const long max_new = a.integer(6);
    const double scale = args[7] == Py_None ? 1.0 / std::sqrt((double)p.D) : a.real(7);
    const at::Tensor *given = args[8] == Py_None ? nullptr : a.tensor(8);
    if (!a.ok) return nullptr;
    if (q->size(1) == 0 || q->size(1) % ((int64_t)p.kv_heads * p.D)) return value_error("q must have n_heads * head_size columns, n_heads a multiple of kv_heads");
    if (max_new < 0 || max_new > 0x7fffffff) return value_error("max_new must be a count, or 0 where it is not known");
    if (given && !(is(*given, at::kFloat, *q) && given->is_contiguous() && given->sizes() == q->sizes()))
        return value_error("out must be a contiguous fp32 tensor of the shape of q on the same device");
    if (given && p.tokens) {
        const char *a = static_cast<const char *>(q->data_ptr()), *b = static_cast<const char *>(given->data_ptr());
        if (a < b + given->nbytes() && b < a + 4 * ((p.tokens - 1) * row_stride(*q) + q->size(1))) return value_error("out must not overlap q");
    }
    const On on(*q, args[9]);
    if (PyErr_Occurred()) return nullptr;
    at::Tensor out = given ? *given : alloc(q->sizes(), at::kFloat, *q);
    const int heads = (int)(q->size(1) / p.D);
    const float *x = static_cast<const float *>(q->data_ptr());
    float *y = static_cast<float *>(out.data_ptr());
    int rc = ATTN_OK;
    Py_BEGIN_ALLOW_THREADS
    if (p.tokens)
        rc = attn_sm100_paged_forward(x, p.k->data_ptr(), p.v->data_ptr(), static_cast<const int *>(p.table->data_ptr()),
                                      static_cast<const int *>(p.cu->data_ptr()), static_cast<const int *>(p.past->data_ptr()), y, row_stride(*q), p.stride, p.type,
                                      p.tokens, p.seqs, heads, p.kv_heads, p.D, p.page_size, p.pages, p.width, (int)max_new, (float)scale, on.stream);
    Py_END_ALLOW_THREADS
    if (failed(rc, "attn_sm100_paged_forward")) return nullptr;
    return THPVariable_Wrap(out);
    END_HANDLE_TH_ERRORS
}

// sample(logits, u, temperature or None, top_k or None, top_p or None, min_p or None, stream) -> tokens
PyObject *sample(PyObject *, PyObject *const *args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    Args a(args, n, 7);
    const at::Tensor *x = a.tensor(0);
    if (!a.ok) return nullptr;
    if (!(x->is_cuda() && x->scalar_type() == at::kFloat && x->dim() == 2 && x->size(1) > 0 && (x->size(1) == 1 || x->stride(1) == 1) &&
          (x->size(0) < 2 || x->stride(0) >= x->size(1)) && x->size(0) <= 0x7fffffff && x->size(1) <= 0x7fffffff))
        return value_error("logits must be an fp32 CUDA tensor of shape [rows, classes] with a row's values side by side");
    const void *each[5] = {};  // u, temperature, top_k, top_p, min_p
    for (int i = 0; i < 5; i++) {
        if (i > 0 && args[1 + i] == Py_None) continue;
        const at::Tensor *t = a.tensor(1 + i);
        if (!a.ok) return nullptr;
        if (!(is(*t, i == 2 ? at::kInt : at::kFloat, *x) && t->is_contiguous() && t->dim() == 1 && t->size(0) == x->size(0)))
            return value_error("u, temperature, top_p and min_p must be fp32, top_k int32, with one value a row of logits, on the same device");
        each[i] = t->data_ptr();
    }
    const On on(*x, args[6]);
    if (PyErr_Occurred()) return nullptr;
    at::Tensor out = alloc({x->size(0)}, at::kInt, *x);
    const float *logits = static_cast<const float *>(x->data_ptr());
    int *y = static_cast<int *>(out.data_ptr()), rc = ATTN_OK;
    const int rows = (int)x->size(0), C = (int)x->size(1);
    Py_BEGIN_ALLOW_THREADS
    if (rows)
        rc = xent_sm100_sample(logits, static_cast<const float *>(each[0]), static_cast<const float *>(each[1]), static_cast<const int *>(each[2]),
                               static_cast<const float *>(each[3]), static_cast<const float *>(each[4]), y, rows > 1 ? x->stride(0) : C, rows, C, on.stream);
    Py_END_ALLOW_THREADS
    if (failed(rc, "xent_sm100_sample")) return nullptr;
    return THPVariable_Wrap(out);
    END_HANDLE_TH_ERRORS
}

// ------------------------------------------------------------------------------------------
// Both ends of a training step: these take fp32 or bf16 tensors, on any one device like the calls above.
// ------------------------------------------------------------------------------------------
// x [..., columns] as rows `ld` elements apart: one row stride with the columns side by side.
struct Rows {
    const void *p = nullptr;
    int64_t rows = 0, columns = 0;
    long long ld = 0;

    bool read(const at::Tensor &t) {
        if (t.dim() < 1 || t.size(-1) < 1 || (t.size(-1) > 1 && t.stride(-1) != 1)) return false;
        columns = t.size(-1), rows = t.numel() / columns, ld = columns, p = t.data_ptr();
        if (t.dim() == 2 && rows > 1) ld = t.stride(0);
        else if (t.dim() != 2 && !t.is_contiguous()) return false;
        return ld >= columns && rows <= 0x7fffffff && columns <= 0x7fffffff;
    }
};
// 0 fp32, 1 bf16, -1 neither
int float_type(const at::Tensor &t) { return t.scalar_type() == at::kFloat ? TENSOR_F32 : t.scalar_type() == at::kBFloat16 ? TENSOR_BF16 : -1; }
int id_type(const at::Tensor &t) {
    return t.scalar_type() == at::kInt ? TENSOR_INT32 : t.scalar_type() == at::kLong ? TENSOR_INT64 : t.scalar_type() == at::kFloat ? TENSOR_IDS_F32 : -1;
}

struct Head {
    const at::Tensor *x, *w, *targets;
    Rows xr, wr;
    int type, ids;
    // x, w, targets in arguments i .. i + 2; false with a Python error set
    bool read(Args &a, int i) {
        x = a.tensor(i), w = a.tensor(i + 1), targets = a.tensor(i + 2);
        if (!a.ok) return false;
        type = float_type(*x);
        if (!(x->is_cuda() && type >= 0 && xr.read(*x)))
            return value_error("x must be an fp32 or bf16 CUDA tensor of shape [..., features], contiguous, or of two dimensions with its columns side by side") != nullptr;
        if (!(is(*w, x->scalar_type(), *x) && w->dim() == 2 && wr.read(*w) && wr.rows > 0 && wr.columns == xr.columns))
            return value_error("w must be a tensor of the type of x and of shape [classes, features] on the same device, with its columns side by side") != nullptr;
        ids = id_type(*targets);
        if (!(ids >= 0 && targets->device() == x->device() && targets->is_contiguous() && targets->sizes() == x->sizes().slice(0, x->dim() - 1)))
            return value_error("targets must be a contiguous int32, int64 or fp32 tensor with one value a row of x, on the same device") != nullptr;
        return true;
    }
};

// linear_xent_forward(x, w, targets, stream) -> (losses, lse)
PyObject *linear_xent_forward(PyObject *, PyObject *const *args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    Args a(args, n, 4);
    Head h;
    if (!a.ok || !h.read(a, 0)) return nullptr;
    const On on(*h.x, args[3]);
    if (PyErr_Occurred()) return nullptr;
    const auto shape = h.targets->sizes();
    const int rows = (int)h.xr.rows, V = (int)h.wr.rows, K = (int)h.xr.columns;
    at::Tensor losses = alloc(shape, at::kFloat, *h.x), lse = alloc(shape, at::kFloat, *h.x), scratch;
    int rc = ATTN_OK;
    if (rows) {
        const size_t bytes = xent_sm100_linear_forward_scratch_bytes(h.xr.p, h.wr.p, h.xr.ld, h.wr.ld, h.type, rows, V, K);
        scratch = alloc({(int64_t)bytes}, at::kByte, *h.x);
        float *lp = static_cast<float *>(losses.data_ptr()), *ep = static_cast<float *>(lse.data_ptr());
        const void *tp = h.targets->data_ptr();
        void *sp = bytes ? scratch.data_ptr() : nullptr;  // (none: sizes that the call refuses)
        Py_BEGIN_ALLOW_THREADS
        rc = xent_sm100_linear_forward(h.xr.p, h.wr.p, tp, lp, ep, sp, h.xr.ld, h.wr.ld, h.type, h.ids, rows, V, K, on.stream);
        Py_END_ALLOW_THREADS
    }
    if (failed(rc, "xent_sm100_linear_forward")) return nullptr;
    return Py_BuildValue("(NN)", THPVariable_Wrap(losses), THPVariable_Wrap(lse));
    END_HANDLE_TH_ERRORS
}

// linear_xent_backward(g, x, w, targets, lse, dw or None, want_dx, stream) -> dx or None
PyObject *linear_xent_backward(PyObject *, PyObject *const *args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    Args a(args, n, 8);
    const at::Tensor *g = a.tensor(0);
    Head h;
    if (!a.ok || !h.read(a, 1)) return nullptr;
    const at::Tensor *lse = a.tensor(4), *dw = args[5] == Py_None ? nullptr : a.tensor(5);
    const int want_dx = a.ok ? PyObject_IsTrue(args[6]) : 0;
    if (!a.ok || want_dx < 0) return nullptr;
    if (!(is(*g, at::kFloat, *h.x) && g->is_contiguous() && (g->numel() == 1 || g->sizes() == h.targets->sizes())))
        return value_error("g must be a contiguous fp32 tensor of one value, or of one for each row of x, on the same device");
    if (!(is(*lse, at::kFloat, *h.x) && lse->is_contiguous() && lse->sizes() == h.targets->sizes()))
        return value_error("lse must be a contiguous fp32 tensor with one value a row of x, on the same device");
    Rows dr;
    if (dw && !(is(*dw, h.w->scalar_type(), *h.w) && dw->sizes() == h.w->sizes() && dr.read(*dw)))
        return value_error("dw must be a tensor like w, with its columns side by side");
    if (!dw && !want_dx) return value_error("neither dx nor dw is wanted");
    const On on(*h.x, args[7]);
    if (PyErr_Occurred()) return nullptr;
    const int rows = (int)h.xr.rows, V = (int)h.wr.rows, K = (int)h.xr.columns;
    at::Tensor dx, scratch;
    if (want_dx) dx = alloc(h.x->sizes(), h.x->scalar_type(), *h.x);
    int rc = ATTN_OK;
    if (rows) {
        const size_t bytes = xent_sm100_linear_backward_scratch_bytes(h.xr.p, h.wr.p, h.xr.ld, h.wr.ld, h.type, rows, V, K);
        scratch = alloc({(int64_t)bytes}, at::kByte, *h.x);
        const float *gp = static_cast<const float *>(g->data_ptr()), *ep = static_cast<const float *>(lse->data_ptr());
        const void *tp = h.targets->data_ptr();
        void *dxp = want_dx ? dx.data_ptr() : nullptr, *dwp = dw ? dw->data_ptr() : nullptr, *sp = bytes ? scratch.data_ptr() : nullptr;
        const int one = g->numel() == 1;
        Py_BEGIN_ALLOW_THREADS
        rc = xent_sm100_linear_backward(gp, h.xr.p, h.wr.p, tp, ep, dxp, dwp, sp, h.xr.ld, h.wr.ld, dr.ld, one, h.type, h.ids, rows, V, K, on.stream);
        Py_END_ALLOW_THREADS
    }
    if (failed(rc, "xent_sm100_linear_backward")) return nullptr;
    if (!want_dx) Py_RETURN_NONE;
    return THPVariable_Wrap(dx);
    END_HANDLE_TH_ERRORS
}

// The table of an embedding or of its gradient: [rows, columns] of fp32 or bf16 beside the tokens.
bool table_of(const at::Tensor &t, const at::Tensor &beside, Rows &r) {
    return float_type(t) >= 0 && t.device() == beside.device() && t.dim() == 2 && r.read(t) && r.rows > 0;
}
// positions: like tokens, or None
bool ids_of(const at::Tensor *tokens, const at::Tensor *positions) {
    return id_type(*tokens) >= 0 && tokens->is_cuda() && tokens->is_contiguous() &&
           (!positions || (is(*positions, tokens->scalar_type(), *tokens) && positions->is_contiguous() && positions->sizes() == tokens->sizes()));
}
int sequence_length(const at::Tensor &tokens) { return tokens.dim() ? (int)std::min<int64_t>(tokens.size(-1), 0x7fffffff) : 1; }

// embedding_forward(tokens, table, positions or None, pos_table or None, scale, stream) -> y
PyObject *embedding_forward(PyObject *, PyObject *const *args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    Args a(args, n, 6);
    const at::Tensor *tokens = a.tensor(0), *table = a.tensor(1);
    const at::Tensor *positions = a.ok && args[2] != Py_None ? a.tensor(2) : nullptr, *pos = a.ok && args[3] != Py_None ? a.tensor(3) : nullptr;
    const double scale = a.real(4);
    if (!a.ok) return nullptr;
    if (!ids_of(tokens, positions)) return value_error("tokens, and positions if given, must be contiguous int32, int64 or fp32 CUDA tensors of the same type and shape");
    Rows tr, pr;
    if (!table_of(*table, *tokens, tr)) return value_error("table must be an fp32 or bf16 tensor of shape [tokens, features] on the same device, with its columns side by side");
    if (pos && !(pos->scalar_type() == table->scalar_type() && table_of(*pos, *tokens, pr) && pr.columns == tr.columns))
        return value_error("pos_table must be a tensor like table, with a row for each position");
    if (positions && !pos) return value_error("positions without pos_table");
    const On on(*tokens, args[5]);
    if (PyErr_Occurred()) return nullptr;
    c10::SmallVector<int64_t, 6> shape(tokens->sizes().begin(), tokens->sizes().end());
    shape.push_back(tr.columns);
    at::Tensor y = alloc(shape, table->scalar_type(), *tokens);
    const int64_t count = tokens->numel();
    const void *tp = tokens->data_ptr(), *pp = positions ? positions->data_ptr() : nullptr;
    void *yp = y.data_ptr();
    const int type = float_type(*table), ids = id_type(*tokens), T = sequence_length(*tokens);
    int rc = ATTN_OK;
    Py_BEGIN_ALLOW_THREADS
    if (count)
        rc = tensor_sm100_embedding_forward(tp, tr.p, pp, pr.p, yp, count, tr.ld, pr.ld, (float)scale, type, ids, T, (int)tr.columns, (int)tr.rows, (int)pr.rows, on.stream);
    Py_END_ALLOW_THREADS
    if (failed(rc, "tensor_sm100_embedding_forward")) return nullptr;
    return THPVariable_Wrap(y);
    END_HANDLE_TH_ERRORS
}

// embedding_backward(dy, tokens, dtable or None, positions or None, dpos_table or None, scale, stream)
PyObject *embedding_backward(PyObject *, PyObject *const *args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    Args a(args, n, 7);
    const at::Tensor *dy = a.tensor(0), *tokens = a.tensor(1), *grad = a.ok && args[2] != Py_None ? a.tensor(2) : nullptr;
    const at::Tensor *positions = a.ok && args[3] != Py_None ? a.tensor(3) : nullptr, *pos = a.ok && args[4] != Py_None ? a.tensor(4) : nullptr;
    const double scale = a.real(5);
    if (!a.ok) return nullptr;
    if (!ids_of(tokens, positions)) return value_error("tokens, and positions if given, must be contiguous int32, int64 or fp32 CUDA tensors of the same type and shape");
    Rows dr, gr, pr;
    if (!(float_type(*dy) >= 0 && dy->device() == tokens->device() && dy->dim() == tokens->dim() + 1 && dy->sizes().slice(0, tokens->dim()) == tokens->sizes() && dr.read(*dy)))
        return value_error("dy must be an fp32 or bf16 tensor with a row for each token on the same device, contiguous, or of two dimensions with its columns side by side");
    if (!grad && !pos) return value_error("neither dtable nor dpos_table is given");
    if (grad && !(table_of(*grad, *tokens, gr) && gr.columns == dr.columns))
        return value_error("dtable must be an fp32 or bf16 tensor of shape [tokens, features] on the same device, with its columns side by side");
    if (pos && !(table_of(*pos, *tokens, pr) && pr.columns == dr.columns && (!grad || pos->scalar_type() == grad->scalar_type())))
        return value_error("dpos_table must be a tensor like dtable, with a row for each position");
    if (positions && !pos) return value_error("positions without dpos_table");
    const On on(*tokens, args[6]);
    if (PyErr_Occurred()) return nullptr;
    const int64_t count = tokens->numel();
    int rc = ATTN_OK;
    if (count) {
        const int C = (int)dr.columns, V = (int)gr.rows, P = (int)pr.rows;
        const size_t bytes = tensor_sm100_embedding_backward_scratch_bytes(count, C, V, positions ? P : 0);
        at::Tensor scratch;
        if (bytes) scratch = alloc({(int64_t)bytes}, at::kByte, *tokens);
        void *sp = bytes ? scratch.data_ptr() : nullptr;
        const void *tp = tokens->data_ptr(), *pp = positions ? positions->data_ptr() : nullptr;
        const int type = float_type(*dy), grad_type = float_type(grad ? *grad : *pos), ids = id_type(*tokens), T = sequence_length(*tokens);
        void *gp = const_cast<void *>(gr.p), *qp = const_cast<void *>(pr.p);
        Py_BEGIN_ALLOW_THREADS
        rc = tensor_sm100_embedding_backward(dr.p, tp, gp, pp, qp, sp, count, dr.ld, gr.ld, pr.ld, (float)scale, type, grad_type, ids, T, C, V, P, on.stream);
        Py_END_ALLOW_THREADS
    }
    if (failed(rc, "tensor_sm100_embedding_backward")) return nullptr;
    Py_RETURN_NONE;
    END_HANDLE_TH_ERRORS
}

// ------------------------------------------------------------------------------------------
// What calling a ctypes function of the library does instead, as the tp_call of its function object's class: a call with
// exactly as many plain numbers (or None for a pointer) as the function has arguments goes to the C ABI from here, every
// other one to ctypes.
// ------------------------------------------------------------------------------------------
template <class T>
bool take(PyObject *o, T *&out) {
    if (o == Py_None) out = nullptr;
    else if (PyLong_Check(o)) out = reinterpret_cast<T *>(static_cast<uintptr_t>(PyLong_AsUnsignedLongLongMask(o)));
    else return false;
    return true;
}
bool take(PyObject *o, int &out) { return PyLong_Check(o) && (out = static_cast<int>(PyLong_AsUnsignedLongLongMask(o)), true); }
bool take(PyObject *o, size_t &out) { return PyLong_Check(o) && (out = static_cast<size_t>(PyLong_AsUnsignedLongLongMask(o)), true); }
bool take(PyObject *o, float &out) { return PyFloat_Check(o) && (out = static_cast<float>(PyFloat_AS_DOUBLE(o)), true); }

template <class R, class... A, size_t... I>
PyObject *invoke(R (*fn)(A...), ternaryfunc own, PyObject *self, PyObject *args, PyObject *keywords, std::index_sequence<I...>) {
    std::tuple<A...> v;
    if (keywords != nullptr || PyTuple_GET_SIZE(args) != (Py_ssize_t)sizeof...(A) || !(take(PyTuple_GET_ITEM(args, I), std::get<I>(v)) && ...)) {
        PyTypeObject *base = Py_TYPE(self)->tp_base;  // of the function's class, or of one derived from it
        while (base->tp_call == own) base = base->tp_base;
        return base->tp_call(self, args, keywords);
    }
    R rc;
    Py_BEGIN_ALLOW_THREADS
    rc = fn(std::get<I>(v)...);
    Py_END_ALLOW_THREADS
    return std::is_signed_v<R> ? PyLong_FromLong(static_cast<long>(rc)) : PyLong_FromSize_t(static_cast<size_t>(rc));
}
template <class R, class... A>
constexpr size_t arity(R (*)(A...)) { return sizeof...(A); }
template <auto kFn>
PyObject *call(PyObject *self, PyObject *args, PyObject *keywords) {
    return invoke(kFn, call<kFn>, self, args, keywords, std::make_index_sequence<arity(kFn)>());
}

#define ENTRY(name) {#name, call<name>}
const struct {
    const char *name;
    ternaryfunc call;
} kEntries[] = {ENTRY(tensor_sm100_fill),        ENTRY(tensor_sm100_arange),        ENTRY(tensor_sm100_copy),
                ENTRY(tensor_sm100_axpy),        ENTRY(tensor_sm100_gelu_forward),  ENTRY(tensor_sm100_gelu_backward),
                ENTRY(xent_sm100_forward),       ENTRY(xent_sm100_backward),        ENTRY(attn_sm100_saved_bytes),
                ENTRY(attn_sm100_backward_scratch_bytes)};

// shorten_calls({name of an entry point: class of its function alone, a Python class derived from ctypes' own})
PyObject *shorten_calls(PyObject *, PyObject *classes) {
    for (const auto &e : kEntries) {
        PyObject *cls = PyDict_Check(classes) ? PyDict_GetItemString(classes, e.name) : nullptr;
        if (cls == nullptr || !PyType_Check(cls) || !PyType_HasFeature(reinterpret_cast<PyTypeObject *>(cls), Py_TPFLAGS_HEAPTYPE) ||
            reinterpret_cast<PyTypeObject *>(cls)->tp_base->tp_call == nullptr) {
            PyErr_Format(PyExc_TypeError, "%s: expected a class derived from that of ctypes functions", e.name);
            return nullptr;
        }
        reinterpret_cast<PyTypeObject *>(cls)->tp_call = e.call;
        PyType_Modified(reinterpret_cast<PyTypeObject *>(cls));
    }
    Py_RETURN_NONE;
}

// set_error(cls): the exception class raised for a non-zero status
PyObject *set_error(PyObject *, PyObject *cls) {
    Py_INCREF(cls);
    Py_XDECREF(g_error);
    g_error = cls;
    Py_RETURN_NONE;
}

#define FAST(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(name)), METH_FASTCALL, nullptr}
PyMethodDef kMethods[] = {FAST(forward), FAST(backward), FAST(forward_into), FAST(backward_into), FAST(linear_forward),
                          FAST(linear_backward), FAST(layernorm_forward), FAST(layernorm_backward), FAST(paged_append), FAST(paged_attention), FAST(sample),
                          FAST(linear_xent_forward), FAST(linear_xent_backward), FAST(embedding_forward), FAST(embedding_backward),
                          {"set_error", set_error, METH_O, nullptr}, {"shorten_calls", shorten_calls, METH_O, nullptr}, {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "gptc_b200_calls", nullptr, -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_gptc_b200_calls(void) { return PyModule_Create(&kModule); }
