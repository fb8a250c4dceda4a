// binding.cpp -- Python calls of the norm, KV cache and attention entry points
// (module luisaml_amd._binding, host code only).
//
// A decode step makes these calls for every layer and token, and their kernels
// take 4 to 10 us; through ctypes a call's argument handling alone took as
// long (cache write 8.4 us, attention 9.4 us).  Each function checks its
// tensors (ValueError), their device among it, calls the C ABI on the stream
// handle given, and returns its status; allocation and status handling stay in
// capi.py.
#include <Python.h>

#include <torch/csrc/autograd/python_variable.h>

#include <string>

#include "lcml_fp8.h"

namespace {

struct Bad {
    std::string what;
};
void need(bool ok, const char *what) {
    if (!ok) throw Bad{what};
}

using Args = PyObject *const *;

// the tensors of one call, all on one device
struct Tensors {
    int device = -1;
    const at::Tensor &operator()(PyObject *o, const char *name) {
        if (!THPVariable_Check(o)) throw Bad{std::string(name) + ": a tensor is expected"};
        const at::Tensor &t = THPVariable_Unpack(o);
        if (!t.is_cuda()) throw Bad{std::string(name) + ": a device tensor is expected"};
        const int at = t.get_device();
        if (device >= 0 && at != device) throw Bad{std::string(name) + ": the other tensors' device is expected"};
        device = at;
        return t;
    }
};
int64_t integer(PyObject *o, const char *name) {
    const long long v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) {
        PyErr_Clear();
        throw Bad{std::string(name) + ": an integer is expected"};
    }
    return v;
}
float number(PyObject *o, const char *name) {
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) {
        PyErr_Clear();
        throw Bad{std::string(name) + ": a number is expected"};
    }
    return (float)v;
}
int dtype_code(const at::Tensor &t) {
    const auto s = t.scalar_type();
    return s == at::kFloat ? LCML_DTYPE_FLOAT : s == at::kBFloat16 ? LCML_DTYPE_BFLOAT16 : 0;
}
// a matrix whose rows are contiguous
void rows(const at::Tensor &t, int64_t M, int64_t H, const char *what) {
    need(t.dim() == 2 && t.size(0) == M && t.size(1) == H && (t.stride(1) == 1 || H <= 1), what);
}
// from row to row, which a single row's stride does not say
int64_t pitch(const at::Tensor &t) { return t.size(0) > 1 || t.stride(0) > t.size(1) ? t.stride(0) : t.size(1); }

// the call's stream, at the end of its checks: the handle and the device that
// are its last two arguments
void *stream_of(const Tensors &t, Args a) {
    const int64_t current = integer(a[1], "device");
    if (current >= 0 && t.device != current)
        throw Bad{"tensors on cuda:" + std::to_string(t.device) + ", current device cuda:" + std::to_string(current)};
    return reinterpret_cast<void *>(integer(a[0], "stream"));
}

template <class F>
PyObject *guarded(Py_ssize_t n, Py_ssize_t want, F f) {
    try {
        need(n == want, "wrong number of arguments");
        return PyLong_FromLong(f());
    } catch (const Bad &b) {
        PyErr_SetString(PyExc_ValueError, b.what.c_str());
    } catch (const std::exception &e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
    } catch (...) {
        PyErr_SetString(PyExc_RuntimeError, "unknown failure");
    }
    return nullptr;
}

// x, gamma, eps, residual, residual_out, mode, scale, out, workspace, stream, device
PyObject *rms_norm(PyObject *, Args a, Py_ssize_t n) {
    return guarded(n, 11, [&] {
        Tensors tensor;
        const at::Tensor &x = tensor(a[0], "x"), &gamma = tensor(a[1], "gamma"), &scale = tensor(a[6], "scale"),
                         &y = tensor(a[7], "out");
        need(x.dim() == 2, "x: a matrix is expected");
        const int64_t M = x.size(0), H = x.size(1), mode = integer(a[5], "mode");
        rows(x, M, H, "x: contiguous rows are expected");
        need(gamma.scalar_type() == at::kFloat && gamma.numel() == H && gamma.is_contiguous(), "gamma: H floats are expected");
        need(y.scalar_type() == at::kByte, "out: uint8 is expected");
        rows(y, M, H, "out: x's shape and contiguous rows are expected");
        need(scale.scalar_type() == at::kFloat && scale.is_contiguous() && scale.numel() >= (mode == LCML_SCALE_ROW ? M : 1),
             "scale: floats, one for the tensor or each row, are expected");
        const void *r = nullptr;
        void *ro = nullptr;
        int64_t ldr = 0, ldro = 0;
        int rt = 0;
        if (a[3] != Py_None) {
            const at::Tensor &res = tensor(a[3], "residual"), &out = tensor(a[4], "residual_out");
            rows(res, M, H, "residual: x's shape and contiguous rows are expected");
            rows(out, M, H, "residual_out: x's shape and contiguous rows are expected");
            need(res.scalar_type() == out.scalar_type(), "residual_out: the residual's type is expected");
            r = res.data_ptr(), ro = out.data_ptr(), ldr = pitch(res), ldro = pitch(out), rt = dtype_code(res);
        } else {
            need(a[4] == Py_None, "residual_out without residual");
        }
        void *ws = nullptr;
        int64_t bytes = 0;
        if (a[8] != Py_None) {
            const at::Tensor &w = tensor(a[8], "workspace");
            ws = w.data_ptr(), bytes = (int64_t)w.nbytes();
        }
        return lcml_fp8_rms_norm(M, H, x.data_ptr(), dtype_code(x), pitch(x), r, ro, rt, ldr, ldro,
                                 static_cast<const float *>(gamma.data_ptr()), number(a[2], "eps"),
                                 static_cast<uint8_t *>(y.data_ptr()), pitch(y), (int)mode,
                                 static_cast<float *>(scale.data_ptr()), ws, bytes, stream_of(tensor, a + 9));
    });
}

struct Cache {
    uint8_t *k, *v;
    float *ks, *vs;
    const int32_t *table, *kv_len, *cu_q;
    int64_t pages, heads, dim, page, stride, cols, seqs;
};
// k_cache, v_cache, k_scale, v_scale, block_table, kv_len, cu_q
Cache cache(Tensors &tensor, Args a) {
    const at::Tensor &k = tensor(a[0], "k_cache"), &v = tensor(a[1], "v_cache"), &ks = tensor(a[2], "k_scale"),
                     &vs = tensor(a[3], "v_scale"), &table = tensor(a[4], "block_table"), &len = tensor(a[5], "kv_len"),
                     &cu = tensor(a[6], "cu_q");
    need(k.dim() == 4 && k.scalar_type() == at::kByte && k.is_contiguous(),
         "k_cache: contiguous uint8 [pages, kv_heads, page_tokens, head_dim] is expected");
    need(v.scalar_type() == at::kByte && v.is_contiguous() && v.sizes() == k.sizes(), "v_cache: k_cache's shape and type are expected");
    for (const at::Tensor *s : {&ks, &vs})
        need(s->scalar_type() == at::kFloat && s->dim() == 2 && s->size(0) == k.size(0) && s->size(1) == k.size(1) && s->is_contiguous(),
             "k_scale, v_scale: contiguous float [pages, kv_heads] is expected");
    need(table.scalar_type() == at::kInt && table.dim() == 2 && (table.stride(1) == 1 || table.size(1) <= 1),
         "block_table: int32 [seqs, columns] with contiguous rows is expected");
    const int64_t seqs = table.size(0), cols = table.size(1);
    need(seqs <= 1 || table.stride(0) >= cols, "block_table: rows that do not overlap are expected (an expanded table's do)");
    need(len.scalar_type() == at::kInt && len.numel() == seqs && len.is_contiguous(), "kv_len: contiguous int32 [seqs] is expected");
    need(cu.scalar_type() == at::kInt && cu.numel() == seqs + 1 && cu.is_contiguous(), "cu_q: contiguous int32 [seqs + 1] is expected");
    return Cache{static_cast<uint8_t *>(k.data_ptr()), static_cast<uint8_t *>(v.data_ptr()), static_cast<float *>(ks.data_ptr()),
                 static_cast<float *>(vs.data_ptr()), static_cast<const int32_t *>(table.data_ptr()),
                 static_cast<const int32_t *>(len.data_ptr()), static_cast<const int32_t *>(cu.data_ptr()), k.size(0), k.size(1),
                 k.size(3), k.size(2), table.stride(0) > cols ? table.stride(0) : cols, cols, seqs};
}
// tokens of `heads` heads whose elements are contiguous
void heads_of(const at::Tensor &t, int64_t heads, int64_t dim, const char *what) {
    need(t.dim() == 3 && (heads < 0 || t.size(1) == heads) && t.size(2) == dim && t.stride(2) == 1, what);
}

// k, v, the cache's seven, max_q, stream, device
PyObject *kv_cache_write(PyObject *, Args a, Py_ssize_t n) {
    return guarded(n, 12, [&] {
        Tensors tensor;
        const at::Tensor &k = tensor(a[0], "k"), &v = tensor(a[1], "v");
        const Cache c = cache(tensor, a + 2);
        heads_of(k, c.heads, c.dim, "k: [tokens, kv_heads, head_dim] is expected");
        heads_of(v, c.heads, c.dim, "v: [tokens, kv_heads, head_dim] is expected");
        need(k.size(0) == v.size(0) && k.scalar_type() == v.scalar_type(), "v: k's tokens and type are expected");
        return lcml_fp8_kv_cache_write(k.data_ptr(), v.data_ptr(), dtype_code(k), k.size(0), k.stride(0), k.stride(1), v.stride(0),
                                       v.stride(1), c.k, c.v, c.ks, c.vs, c.pages, c.heads, c.dim, c.page, c.table, c.stride,
                                       c.cols, c.kv_len, c.cu_q, c.seqs, integer(a[9], "max_q"),
                                       stream_of(tensor, a + 10));
    });
}

// the cache's seven, max_q, k_out, v_out, stream, device
PyObject *kv_cache_read(PyObject *, Args a, Py_ssize_t n) {
    return guarded(n, 12, [&] {
        Tensors tensor;
        const Cache c = cache(tensor, a);
        const at::Tensor &k = tensor(a[8], "k_out"), &v = tensor(a[9], "v_out");
        heads_of(k, c.heads, c.dim, "k_out: [tokens, kv_heads, head_dim] is expected");
        heads_of(v, c.heads, c.dim, "v_out: [tokens, kv_heads, head_dim] is expected");
        need(k.size(0) == v.size(0) && k.scalar_type() == v.scalar_type(), "v_out: k_out's tokens and type are expected");
        return lcml_fp8_kv_cache_read(c.k, c.v, c.ks, c.vs, c.pages, c.heads, c.dim, c.page, c.table, c.stride, c.cols, c.kv_len,
                                      c.cu_q, c.seqs, integer(a[7], "max_q"), k.data_ptr(), v.data_ptr(), dtype_code(k), k.size(0),
                                      k.stride(0), k.stride(1), v.stride(0), v.stride(1),
                                      stream_of(tensor, a + 10));
    });
}

// q, out, the cache's seven, max_q, max_kv, scale, causal, window, workspace, stream, device
PyObject *attention(PyObject *, Args a, Py_ssize_t n) {
    return guarded(n, 17, [&] {
        Tensors tensor;
        const at::Tensor &q = tensor(a[0], "q"), &o = tensor(a[1], "out");
        const Cache c = cache(tensor, a + 2);
        heads_of(q, -1, c.dim, "q: [tokens, q_heads, head_dim] is expected");
        heads_of(o, q.size(1), c.dim, "out: q's shape is expected");
        need(o.size(0) == q.size(0), "out: q's shape is expected");
        void *ws = nullptr;
        int64_t bytes = 0;
        if (a[14] != Py_None) {
            const at::Tensor &w = tensor(a[14], "workspace");
            ws = w.data_ptr(), bytes = (int64_t)w.nbytes();
        }
        return lcml_fp8_attention(q.data_ptr(), dtype_code(q), q.size(0), q.size(1), q.stride(0), q.stride(1), o.data_ptr(),
                                  dtype_code(o), o.stride(0), o.stride(1), c.k, c.v, c.ks, c.vs, c.pages, c.heads, c.dim, c.page,
                                  c.table, c.stride, c.cols, c.kv_len, c.cu_q, c.seqs, integer(a[9], "max_q"),
                                  integer(a[10], "max_kv"), number(a[11], "scale"), (int)integer(a[12], "causal"),
                                  integer(a[13], "window"), ws, bytes, stream_of(tensor, a + 15));
    });
}

#define METHOD(f) {#f, reinterpret_cast<PyCFunction>(reinterpret_cast<void *>(f)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {METHOD(rms_norm), METHOD(kv_cache_write), METHOD(kv_cache_read), METHOD(attention), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_binding", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__binding() { return PyModule_Create(&module); }
