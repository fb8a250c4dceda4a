// binding.cpp -- Python calls of the norm, rotation, KV cache and attention entry points
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

struct Workspace {
    void *p = nullptr;
    int64_t bytes = 0;
};
Workspace workspace(Tensors &tensor, PyObject *o) {
    if (o == Py_None) return {};
    const at::Tensor &w = tensor(o, "workspace");
    need(w.is_contiguous(), "workspace: a contiguous tensor is expected");
    return {w.data_ptr(), (int64_t)w.nbytes()};
}

// q, out, the cache's seven, max_q, max_kv, scale, causal, window, sinks, workspace, stream, device
PyObject *attention(PyObject *, Args a, Py_ssize_t n) {
    return guarded(n, 18, [&] {
        Tensors tensor;
        const at::Tensor &q = tensor(a[0], "q"), &o = tensor(a[1], "out");
        const Cache c = cache(tensor, a + 2);
        heads_of(q, -1, c.dim, "q: [tokens, q_heads, head_dim] is expected");
        heads_of(o, q.size(1), c.dim, "out: q's shape is expected");
        need(o.size(0) == q.size(0), "out: q's shape is expected");
        const int64_t sinks = integer(a[14], "sinks");
        void *ws = nullptr;
        int64_t bytes = 0;
        if (a[15] != Py_None) {
            const at::Tensor &w = tensor(a[15], "workspace");
            ws = w.data_ptr(), bytes = (int64_t)w.nbytes();
        }
        if (sinks != 0)
            return lcml_fp8_attention_sinks(q.data_ptr(), dtype_code(q), q.size(0), q.size(1), q.stride(0), q.stride(1),
                                            o.data_ptr(), dtype_code(o), o.stride(0), o.stride(1), c.k, c.v, c.ks, c.vs, c.pages,
                                            c.heads, c.dim, c.page, c.table, c.stride, c.cols, c.kv_len, c.cu_q, c.seqs,
                                            integer(a[9], "max_q"), integer(a[10], "max_kv"), number(a[11], "scale"),
                                            (int)integer(a[12], "causal"), integer(a[13], "window"), sinks, ws, bytes,
                                            stream_of(tensor, a + 16));
        return lcml_fp8_attention(q.data_ptr(), dtype_code(q), q.size(0), q.size(1), q.stride(0), q.stride(1), o.data_ptr(),
                                  dtype_code(o), o.stride(0), o.stride(1), c.k, c.v, c.ks, c.vs, c.pages, c.heads, c.dim, c.page,
                                  c.table, c.stride, c.cols, c.kv_len, c.cu_q, c.seqs, integer(a[9], "max_q"),
                                  integer(a[10], "max_kv"), number(a[11], "scale"), (int)integer(a[12], "causal"),
                                  integer(a[13], "window"), ws, bytes, stream_of(tensor, a + 16));
    });
}

// `count` contiguous int32, for any count if it is negative
int32_t *ints(const at::Tensor &t, int64_t count, const char *what) {
    need(t.scalar_type() == at::kInt && t.is_contiguous() && (count < 0 || t.numel() == count), what);
    return static_cast<int32_t *>(t.data_ptr());
}

// rows of an int32 table that do not overlap
struct Table {
    int32_t *p;
    int64_t stride, cols;
};
Table table_of(const at::Tensor &t, int64_t rows, const char *what) {
    need(t.scalar_type() == at::kInt && t.dim() == 2 && t.size(0) == rows && (t.stride(1) == 1 || t.size(1) <= 1), what);
    need(rows <= 1 || t.stride(0) >= t.size(1), what);
    return {static_cast<int32_t *>(t.data_ptr()), t.stride(0) > t.size(1) ? t.stride(0) : t.size(1), t.size(1)};
}

// q, out, the cache's seven, group_seq, prefix_table, prefix_len, max_q, max_own, max_prefix, scale, causal, workspace,
// stream, device
PyObject *attention_shared(PyObject *, Args a, Py_ssize_t n) {
    return guarded(n, 20, [&] {
        Tensors tensor;
        const at::Tensor &q = tensor(a[0], "q"), &o = tensor(a[1], "out");
        const Cache c = cache(tensor, a + 2);
        heads_of(q, -1, c.dim, "q: [tokens, q_heads, head_dim] is expected");
        heads_of(o, q.size(1), c.dim, "out: q's shape is expected");
        need(o.size(0) == q.size(0), "out: q's shape is expected");
        const at::Tensor &len = tensor(a[11], "prefix_len");
        const int64_t groups = len.numel();
        const int32_t *prefix_len = ints(len, groups, "prefix_len: contiguous int32 [groups] is expected");
        const int32_t *group_seq = ints(tensor(a[9], "group_seq"), groups + 1, "group_seq: contiguous int32 [groups + 1] is expected");
        const Table t = table_of(tensor(a[10], "prefix_table"), groups,
                                 "prefix_table: int32 [groups, columns] with contiguous rows that do not overlap is expected");
        const Workspace w = workspace(tensor, a[17]);
        return lcml_fp8_attention_shared(q.data_ptr(), dtype_code(q), q.size(0), q.size(1), q.stride(0), q.stride(1),
                                         o.data_ptr(), dtype_code(o), o.stride(0), o.stride(1), c.k, c.v, c.ks, c.vs, c.pages,
                                         c.heads, c.dim, c.page, c.table, c.stride, c.cols, c.kv_len, c.cu_q, c.seqs, group_seq,
                                         t.p, t.stride, t.cols, prefix_len, groups, integer(a[12], "max_q"),
                                         integer(a[13], "max_own"), integer(a[14], "max_prefix"), number(a[15], "scale"),
                                         (int)integer(a[16], "causal"), w.p, w.bytes, stream_of(tensor, a + 18));
    });
}

// new_tokens, kv_len, block_table, free_pages, free_count, page_tokens, ended, first_own, kv_len_out, cu_q, left, positions,
// slots, workspace, stream, device
PyObject *kv_cache_plan(PyObject *, Args a, Py_ssize_t n) {
    return guarded(n, 16, [&] {
        Tensors tensor;
        const at::Tensor &len = tensor(a[1], "kv_len"), &free = tensor(a[3], "free_pages");
        const int64_t seqs = len.numel(), pages = free.numel();
        const Table t = table_of(tensor(a[2], "block_table"), seqs,
                                 "block_table: int32 [seqs, columns] with contiguous rows that do not overlap is expected");
        const auto some = [&](int i, const char *name, const char *what) -> int32_t * {
            return a[i] == Py_None ? nullptr : ints(tensor(a[i], name), seqs, what);
        };
        int64_t rows = -1;
        int32_t *positions = nullptr;
        int64_t *slots = nullptr;
        if (a[11] != Py_None) {
            const at::Tensor &p = tensor(a[11], "positions");
            positions = ints(p, -1, "positions: contiguous int32 is expected"), rows = p.numel();
        }
        if (a[12] != Py_None) {
            const at::Tensor &s = tensor(a[12], "slots");
            need(s.scalar_type() == at::kLong && s.is_contiguous() && (rows < 0 || s.numel() == rows),
                 "slots: contiguous int64, as many as positions, is expected");
            slots = static_cast<int64_t *>(s.data_ptr()), rows = s.numel();
        }
        const Workspace w = workspace(tensor, a[13]);
        return lcml_fp8_kv_cache_plan(
            ints(tensor(a[0], "new_tokens"), seqs, "new_tokens: contiguous int32 [seqs] is expected"),
            ints(len, seqs, "kv_len: contiguous int32 [seqs] is expected"),
            some(6, "ended", "ended: contiguous int32 [seqs] is expected"),
            some(7, "first_own", "first_own: contiguous int32 [seqs] is expected"), seqs,
            ints(free, pages, "free_pages: contiguous int32 [pages] is expected"),
            ints(tensor(a[4], "free_count"), 1, "free_count: int32 [1] is expected"), pages, integer(a[5], "page_tokens"), t.p,
            t.stride, t.cols, ints(tensor(a[8], "kv_len_out"), seqs, "kv_len_out: contiguous int32 [seqs] is expected"),
            ints(tensor(a[9], "cu_q"), seqs + 1, "cu_q: contiguous int32 [seqs + 1] is expected"),
            ints(tensor(a[10], "left"), 1, "left: int32 [1] is expected"), positions, slots, rows < 0 ? 0 : rows, w.p, w.bytes,
            stream_of(tensor, a + 14));
    });
}

// q, k, positions, table, q_gamma, k_gamma, eps, interleaved, q_out, k_out, stream, device
PyObject *qk_norm_rope(PyObject *, Args a, Py_ssize_t n) {
    return guarded(n, 12, [&] {
        Tensors tensor;
        const at::Tensor &q = tensor(a[0], "q"), &qo = tensor(a[8], "q_out");
        need(q.dim() == 3, "q: [tokens, q_heads, head_dim] is expected");
        const int64_t tokens = q.size(0), dim = q.size(2);
        heads_of(q, -1, dim, "q: [tokens, q_heads, head_dim] is expected");
        heads_of(qo, q.size(1), dim, "q_out: q's shape is expected");
        need(qo.size(0) == tokens, "q_out: q's shape is expected");
        const void *k = nullptr;
        void *ko = nullptr;
        int64_t k_heads = 0, kt = 0, kh = 0, kot = 0, koh = 0;
        if (a[1] != Py_None) {
            const at::Tensor &x = tensor(a[1], "k"), &y = tensor(a[9], "k_out");
            heads_of(x, -1, dim, "k: [tokens, k_heads, head_dim] is expected");
            heads_of(y, x.size(1), dim, "k_out: k's shape is expected");
            need(x.size(0) == tokens && x.scalar_type() == q.scalar_type(), "k: q's tokens and type are expected");
            need(y.size(0) == tokens && y.scalar_type() == qo.scalar_type(), "k_out: k's shape and q_out's type are expected");
            k = x.data_ptr(), ko = y.data_ptr(), k_heads = x.size(1);
            kt = x.stride(0), kh = x.stride(1), kot = y.stride(0), koh = y.stride(1);
        } else {
            need(a[9] == Py_None, "k_out without k");
        }
        const auto gamma = [&](int i, const char *name, const char *what) -> const float * {
            if (a[i] == Py_None) return nullptr;
            const at::Tensor &g = tensor(a[i], name);
            need(g.scalar_type() == at::kFloat && g.numel() == dim && g.is_contiguous(), what);
            return static_cast<const float *>(g.data_ptr());
        };
        const float *table = nullptr;
        int64_t table_rows = 0, rot = 0;
        if (a[3] != Py_None) {
            const at::Tensor &t = tensor(a[3], "table");
            need(t.scalar_type() == at::kFloat && t.dim() == 2 && t.is_contiguous(), "table: contiguous float [rows, rot_dim] is expected");
            table = static_cast<const float *>(t.data_ptr()), table_rows = t.size(0), rot = t.size(1);
        }
        const int32_t *positions = a[2] == Py_None ? nullptr : ints(tensor(a[2], "positions"), tokens, "positions: contiguous int32 [tokens] is expected");
        return lcml_fp8_qk_norm_rope(q.data_ptr(), k, dtype_code(q), tokens, q.size(1), k_heads, dim, q.stride(0), q.stride(1), kt,
                                     kh, gamma(4, "q_gamma", "q_gamma: head_dim floats are expected"),
                                     gamma(5, "k_gamma", "k_gamma: head_dim floats are expected"), number(a[6], "eps"), positions,
                                     table, table_rows, rot, (int)integer(a[7], "interleaved"), qo.data_ptr(), ko, dtype_code(qo),
                                     qo.stride(0), qo.stride(1), kot, koh, stream_of(tensor, a + 10));
    });
}

#define METHOD(f) {#f, reinterpret_cast<PyCFunction>(reinterpret_cast<void *>(f)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {METHOD(rms_norm), METHOD(kv_cache_write), METHOD(kv_cache_read), METHOD(attention), METHOD(attention_shared),
                         METHOD(kv_cache_plan), METHOD(qk_norm_rope), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_binding", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__binding() { return PyModule_Create(&module); }
