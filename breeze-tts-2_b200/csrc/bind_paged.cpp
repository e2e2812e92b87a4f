// Host side of breeze_b200.fused.paged's and paged_fp8's calls: reads the tensors, fills the
// descriptor, allocates the output and the workspace and calls the library's C
// entry. It takes plain calls only: whatever it would have to refuse, convert or
// explain it hands back to Python (None), whose checks of the same conditions are
// the ones that raise. A status other than BQ_OK comes back as an int.
//
// Measured (two streams, calls in a row): paged_append 13.1 -> 5.8 us, paged_attention
// with an lse of its own 14.9 -> 8.4 us, of which 2.3 us are the launch; reading and
// checking the tensors from Python took 5 to 6 us, an allocation 1.9 us.
#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <torch/csrc/autograd/python_variable.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>

#include <climits>
#include <cmath>
#include <cstring>

#include "breeze_b200.h"

namespace {

decltype(&bq_paged_append) f_append = nullptr;
decltype(&bq_paged_attention) f_attention = nullptr;
decltype(&bq_paged_attention_workspace_bytes) f_workspace = nullptr;
decltype(&bq_paged8_append) f_append8 = nullptr;
decltype(&bq_paged8_attention) f_attention8 = nullptr;
decltype(&bq_paged8_attention_workspace_bytes) f_workspace8 = nullptr;
decltype(&bq_paged8_read) f_read8 = nullptr;

struct NotPlain {};  // to Python's checks

void need(bool ok) {
    if (!ok) throw NotPlain{};
}
int32_t i32(int64_t v) {
    need(v >= 0 && v <= INT32_MAX);
    return int32_t(v);
}
const at::Tensor& tensor(PyObject* o) {
    need(THPVariable_Check(o));
    return THPVariable_Unpack(o);
}
long integer(PyObject* o) {
    need(PyLong_Check(o));
    const long v = PyLong_AsLong(o);
    if (v == -1 && PyErr_Occurred()) throw NotPlain{};
    return v;
}
float real(PyObject* o) {
    need(PyFloat_Check(o) || PyLong_Check(o));
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) throw NotPlain{};
    need(std::isfinite(v) && std::fabs(v) < 3.4e38);
    return float(v);
}
bool on(const at::Tensor& t, int dev) { return t.is_cuda() && t.get_device() == dev; }
// Row stride of a 2-D tensor with contiguous rows (a dimension of size one has no stride).
int64_t row_stride(const at::Tensor& t) {
    need(t.dim() == 2 && (t.stride(1) == 1 || t.size(1) == 1));
    return t.size(0) > 1 ? t.stride(0) : t.size(1);
}
bool vector(const at::Tensor& t, at::ScalarType type, int64_t n, int dev) {
    return t.scalar_type() == type && t.dim() == 1 && t.size(0) == n && (t.stride(0) == 1 || n == 1) && on(t, dev);
}

// The cache part of both descriptors. rows: new tokens, of dtype `type`.
int fill(bq_paged_kv* kv, const at::Tensor& rows, PyObject* k_, PyObject* v_, PyObject* table_, PyObject* lens_, PyObject* starts_) {
    const at::Tensor &k = tensor(k_), &v = tensor(v_), &table = tensor(table_), &lens = tensor(lens_);
    need(rows.is_cuda());
    const int dev = int(rows.get_device());
    need(dev == int(c10::cuda::current_device()));
    const at::ScalarType type = rows.scalar_type();
    need(type == at::kBFloat16 || type == at::kHalf);
    need(on(k, dev) && on(v, dev) && on(table, dev) && k.scalar_type() == type && v.scalar_type() == type);
    need(k.dim() == 4 && v.sizes() == k.sizes() && k.stride(3) == 1 && v.stride(3) == 1 && k.numel() > 0);
    need(table.scalar_type() == at::kInt && table.dim() == 2 && (table.stride(1) == 1 || table.size(1) == 1) && table.numel() > 0);
    const int64_t batch = table.size(0);
    need(vector(lens, at::kInt, batch, dev));
    kv->B = i32(batch);
    kv->HKV = i32(k.size(1));
    kv->D = i32(k.size(3));
    kv->page_size = i32(k.size(2));
    kv->num_pages = i32(k.size(0));
    kv->max_pages = i32(table.size(1));
    kv->dtype = type == at::kHalf ? BQ_DT_F16 : BQ_DT_BF16;
    kv->k_pages = k.data_ptr();
    kv->v_pages = v.data_ptr();
    for (int i = 0; i < 3; ++i) {
        kv->k_stride[i] = k.stride(i);
        kv->v_stride[i] = v.stride(i);
    }
    kv->page_table = static_cast<const int32_t*>(table.data_ptr());
    kv->ld_table = batch > 1 ? table.stride(0) : table.size(1);
    kv->seq_lens = static_cast<const int32_t*>(lens.data_ptr());
    if (starts_ == Py_None) {
        need(rows.size(0) == batch);
    } else {
        const at::Tensor& starts = tensor(starts_);
        need(vector(starts, at::kInt, batch + 1, dev));
        kv->q_starts = static_cast<const int32_t*>(starts.data_ptr());
    }
    return dev;
}

// The cache part of the 8-bit descriptors, from a: k_pages, v_pages, k_scales, v_scales, page_table, seq_lens.
// rows of dtype `type`.
int fill8(bq_paged8_kv* kv, int64_t rows, at::ScalarType type, PyObject* const* a, PyObject* starts_) {
    const at::Tensor &k = tensor(a[0]), &v = tensor(a[1]), &ks = tensor(a[2]), &vs = tensor(a[3]), &table = tensor(a[4]), &lens = tensor(a[5]);
    need(k.is_cuda());
    const int dev = int(k.get_device());
    need(dev == int(c10::cuda::current_device()));
    need(type == at::kBFloat16 || type == at::kHalf || type == at::kFloat);
    need(on(v, dev) && on(ks, dev) && on(vs, dev) && on(table, dev));
    need(k.scalar_type() == at::kFloat8_e4m3fn && v.scalar_type() == at::kFloat8_e4m3fn);
    need(ks.scalar_type() == at::kFloat8_e8m0fnu && vs.scalar_type() == at::kFloat8_e8m0fnu);
    need(k.dim() == 4 && v.sizes() == k.sizes() && k.stride(3) == 1 && v.stride(3) == 1 && k.numel() > 0);
    need(ks.dim() == 3 && vs.sizes() == ks.sizes() && ks.size(0) == k.size(0) && ks.size(1) == k.size(1) && ks.size(2) > 0);
    need(((ks.stride(2) == 1 && vs.stride(2) == 1) || ks.size(2) == 1) && k.size(2) % ks.size(2) == 0);
    need(table.scalar_type() == at::kInt && table.dim() == 2 && (table.stride(1) == 1 || table.size(1) == 1) && table.numel() > 0);
    const int64_t batch = table.size(0);
    need(vector(lens, at::kInt, batch, dev));
    kv->B = i32(batch);
    kv->HKV = i32(k.size(1));
    kv->D = i32(k.size(3));
    kv->page_size = i32(k.size(2));
    kv->num_pages = i32(k.size(0));
    kv->max_pages = i32(table.size(1));
    kv->block = i32(k.size(2) / ks.size(2));
    kv->dtype = type == at::kHalf ? BQ_DT_F16 : type == at::kFloat ? BQ_DT_F32 : BQ_DT_BF16;
    kv->k_pages = k.data_ptr();
    kv->v_pages = v.data_ptr();
    kv->k_scales = ks.data_ptr();
    kv->v_scales = vs.data_ptr();
    for (int i = 0; i < 3; ++i) {
        kv->k_stride[i] = k.stride(i);
        kv->v_stride[i] = v.stride(i);
    }
    for (int i = 0; i < 2; ++i) {
        kv->k_scale_stride[i] = ks.stride(i);
        kv->v_scale_stride[i] = vs.stride(i);
    }
    kv->page_table = static_cast<const int32_t*>(table.data_ptr());
    kv->ld_table = batch > 1 ? table.stride(0) : table.size(1);
    kv->seq_lens = static_cast<const int32_t*>(lens.data_ptr());
    if (starts_ == Py_None) {
        need(rows == batch);
    } else {
        const at::Tensor& starts = tensor(starts_);
        need(vector(starts, at::kInt, batch + 1, dev));
        kv->q_starts = static_cast<const int32_t*>(starts.data_ptr());
    }
    return dev;
}

// `given`, or a new (rows, width) tensor like `like`.
at::Tensor output(PyObject* given, const at::Tensor& like, int64_t rows, int64_t width, int dev, int64_t* ld) {
    if (given == Py_None) {
        *ld = width;
        return at::empty({rows, width}, like.options());
    }
    const at::Tensor& out = tensor(given);
    need(out.dim() == 2 && out.size(0) == rows && out.size(1) == width && out.scalar_type() == like.scalar_type() && on(out, dev));
    *ld = row_stride(out);
    return out;
}

template <typename Call>
int32_t launched(const Call& call) {
    int32_t rc;
    Py_BEGIN_ALLOW_THREADS
    rc = call();
    Py_END_ALLOW_THREADS
    return rc;
}

PyObject* result(int32_t rc, const at::Tensor& out, PyObject* given) {
    if (rc != BQ_OK) return PyLong_FromLong(rc);
    if (given == Py_None) return THPVariable_Wrap(out);
    Py_INCREF(given);
    return given;
}

template <typename Body>
PyObject* guarded(const Body& body) {
    try {
        return body();
    } catch (const NotPlain&) {
        PyErr_Clear();
        Py_RETURN_NONE;
    } catch (const c10::OutOfMemoryError&) {
        Py_RETURN_NONE;  // Python's own allocation raises it as torch does
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
        return nullptr;
    }
}

// The rows, tables, norms and output of an append's descriptor, whose cache part `kv` is filled; arguments a[at] and on:
// q_norm_w, k_norm_w, eps, out, flags.
template <typename Desc>
at::Tensor fill_append(Desc& d, const at::Tensor& qkv, const at::Tensor& cos, const at::Tensor& sin, PyObject* const* a, int dev) {
    const int64_t rows = qkv.size(0), width = qkv.size(1), hq = width / d.kv.D - 2 * int64_t(d.kv.HKV);
    need(hq > 0 && (hq + 2 * int64_t(d.kv.HKV)) * d.kv.D == width);
    const at::ScalarType type = qkv.scalar_type(), cs = cos.scalar_type();
    d.ldcs = row_stride(cos);
    need(cos.size(1) == d.kv.D && sin.sizes() == cos.sizes() && sin.scalar_type() == cs && row_stride(sin) == d.ldcs);
    need((cs == type || cs == at::kFloat) && on(cos, dev) && on(sin, dev));
    if (a[0] != Py_None || a[1] != Py_None) {
        const at::Tensor &qn = tensor(a[0]), &kn = tensor(a[1]);
        need(vector(qn, type, d.kv.D, dev) && vector(kn, type, d.kv.D, dev));
        d.q_norm = qn.data_ptr();
        d.k_norm = kn.data_ptr();
    }
    d.T = i32(rows);
    d.HQ = i32(hq);
    d.cs_dtype = cs == at::kFloat ? BQ_DT_F32 : d.kv.dtype;
    d.rope_rows = i32(cos.size(0));
    d.eps = real(a[2]);
    d.flags = uint32_t(integer(a[4]));
    d.qkv = qkv.data_ptr();
    d.cos = cos.data_ptr();
    d.sin = sin.data_ptr();
    const at::Tensor out = output(a[3], qkv, rows, hq * d.kv.D, dev, &d.ldq);
    d.q_out = out.data_ptr();
    return out;
}

// The rows and outputs of an attention's descriptor, whose cache part is filled.
template <typename Desc>
at::Tensor fill_attention(Desc& d, const at::Tensor& q, PyObject* scale, PyObject* max_q, PyObject* given, PyObject* lse_, PyObject* flags,
                          int dev) {
    const int64_t rows = q.size(0), width = q.size(1), hq = width / d.kv.D;
    need(hq > 0 && hq * d.kv.D == width && hq % d.kv.HKV == 0);
    d.T = i32(rows);
    d.HQ = i32(hq);
    d.max_q = max_q == Py_None ? 0 : i32(integer(max_q));
    d.scale = scale == Py_None ? float(1.0 / std::sqrt(double(d.kv.D))) : real(scale);
    d.flags = uint32_t(integer(flags));
    d.q = q.data_ptr();
    if (lse_ != Py_None) {
        const at::Tensor& lse = tensor(lse_);
        need(lse.dim() == 2 && lse.size(0) == rows && lse.size(1) == hq && lse.scalar_type() == at::kFloat && on(lse, dev));
        d.lse = static_cast<float*>(lse.data_ptr());
        d.ldl = row_stride(lse);
    }
    const at::Tensor out = output(given, q, rows, width, dev, &d.ldo);
    d.out = out.data_ptr();
    return out;
}

void* stream_of(int dev) { return c10::cuda::getCurrentCUDAStream(c10::DeviceIndex(dev)).stream(); }

// Workspace from torch's allocator (calls on other streams, and other graphs, have their own), then the call.
template <typename Desc, typename Size, typename Call>
PyObject* attend(const Desc& d, Size* size, Call* call, const at::Tensor& q, const at::Tensor& out, PyObject* given, int dev) {
    size_t bytes = 0;
    const int32_t rc = size(&d, &bytes);
    if (rc != BQ_OK) return PyLong_FromLong(rc);
    at::Tensor ws;
    if (bytes) ws = at::empty({int64_t(bytes)}, q.options().dtype(at::kByte));
    void* stream = stream_of(dev);
    return result(launched([&] { return call(&d, bytes ? ws.data_ptr() : nullptr, bytes, stream); }), out, given);
}

// append(qkv, cos, sin, k_pages, v_pages, page_table, seq_lens, q_starts, q_norm_w, k_norm_w, eps, out, flags)
PyObject* append(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        need(n == 13 && f_append);
        const at::Tensor &qkv = tensor(a[0]), &cos = tensor(a[1]), &sin = tensor(a[2]);
        bq_paged_append_desc d;
        std::memset(&d, 0, sizeof(d));
        d.ldqkv = row_stride(qkv);
        const int dev = fill(&d.kv, qkv, a[3], a[4], a[5], a[6], a[7]);
        const at::Tensor out = fill_append(d, qkv, cos, sin, a + 8, dev);
        void* stream = stream_of(dev);
        return result(launched([&] { return f_append(&d, stream); }), out, a[11]);
    });
}

// attention(q, k_pages, v_pages, page_table, seq_lens, prefix_len, q_starts, scale, max_q, out, lse, flags)
PyObject* attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        need(n == 12 && f_attention && f_workspace);
        const at::Tensor& q = tensor(a[0]);
        bq_paged_attn_desc d;
        std::memset(&d, 0, sizeof(d));
        d.ldq = row_stride(q);
        const int dev = fill(&d.kv, q, a[1], a[2], a[3], a[4], a[6]);
        d.prefix_len = i32(integer(a[5]));
        const at::Tensor out = fill_attention(d, q, a[7], a[8], a[9], a[10], a[11], dev);
        return attend(d, f_workspace, f_attention, q, out, a[9], dev);
    });
}

// append8(qkv, cos, sin, k_pages, v_pages, k_scales, v_scales, page_table, seq_lens, q_starts, q_norm_w, k_norm_w, eps,
//         out, flags)
PyObject* append8(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        need(n == 15 && f_append8);
        const at::Tensor &qkv = tensor(a[0]), &cos = tensor(a[1]), &sin = tensor(a[2]);
        bq_paged8_append_desc d;
        std::memset(&d, 0, sizeof(d));
        d.ldqkv = row_stride(qkv);
        const int dev = fill8(&d.kv, qkv.size(0), qkv.scalar_type(), a + 3, a[9]);
        need(on(qkv, dev));
        const at::Tensor out = fill_append(d, qkv, cos, sin, a + 10, dev);
        void* stream = stream_of(dev);
        return result(launched([&] { return f_append8(&d, stream); }), out, a[13]);
    });
}

// attention8(q, k_pages, v_pages, k_scales, v_scales, page_table, seq_lens, q_starts, scale, max_q, out, lse, flags)
PyObject* attention8(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        need(n == 13 && f_attention8 && f_workspace8);
        const at::Tensor& q = tensor(a[0]);
        bq_paged8_attn_desc d;
        std::memset(&d, 0, sizeof(d));
        d.ldq = row_stride(q);
        const int dev = fill8(&d.kv, q.size(0), q.scalar_type(), a + 1, a[7]);
        need(on(q, dev));
        const at::Tensor out = fill_attention(d, q, a[8], a[9], a[10], a[11], a[12], dev);
        return attend(d, f_workspace8, f_attention8, q, out, a[10], dev);
    });
}

// `given`, or a new (rows, heads, dim) tensor, and its strides of a row and a head.
at::Tensor read_out(PyObject* given, const at::Tensor& like, int64_t rows, int64_t heads, int64_t dim, at::ScalarType type, int dev,
                    int64_t* strides) {
    at::Tensor out;
    if (given == Py_None) {
        out = at::empty({rows, heads, dim}, like.options().dtype(type));
    } else {
        out = tensor(given);
        need(out.dim() == 3 && out.size(0) == rows && out.size(1) == heads && out.size(2) == dim && out.scalar_type() == type && on(out, dev));
        need(out.stride(2) == 1);
    }
    strides[0] = rows > 1 ? out.stride(0) : heads * dim;
    strides[1] = heads > 1 ? out.stride(1) : dim;
    return out;
}

// read8(k_pages, v_pages, k_scales, v_scales, page_table, seq_lens, q_starts, rows, dtype, k_out, v_out, flags) -> (k, v);
// dtype: BQ_DT_*
PyObject* read8(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        need(n == 12 && f_read8);
        const long code = integer(a[8]);
        need(code == BQ_DT_BF16 || code == BQ_DT_F16 || code == BQ_DT_F32);
        const at::ScalarType type = code == BQ_DT_BF16 ? at::kBFloat16 : code == BQ_DT_F16 ? at::kHalf : at::kFloat;
        bq_paged8_read_desc d;
        std::memset(&d, 0, sizeof(d));
        const int64_t rows = integer(a[7]);
        const int dev = fill8(&d.kv, rows, type, a, a[6]);
        d.T = i32(rows);
        d.flags = uint32_t(integer(a[11]));
        const at::Tensor& like = tensor(a[0]);
        const at::Tensor k = read_out(a[9], like, rows, d.kv.HKV, d.kv.D, type, dev, d.ko_stride),
                         v = read_out(a[10], like, rows, d.kv.HKV, d.kv.D, type, dev, d.vo_stride);
        d.k_out = k.data_ptr();
        d.v_out = v.data_ptr();
        void* stream = stream_of(dev);
        const int32_t rc = launched([&] { return f_read8(&d, stream); });
        if (rc != BQ_OK) return PyLong_FromLong(rc);
        PyObject* pair = PyTuple_New(2);
        if (!pair) return nullptr;
        for (int i = 0; i < 2; ++i) {
            PyObject* o = a[9 + i];
            if (o == Py_None)
                o = THPVariable_Wrap(i ? v : k);
            else
                Py_INCREF(o);
            if (!o) {
                Py_DECREF(pair);
                return nullptr;
            }
            PyTuple_SET_ITEM(pair, i, o);
        }
        return pair;
    });
}

// The addresses of N entries of the loaded library.
template <int N>
bool addresses(PyObject* const* a, Py_ssize_t n, const char* many, void* (&p)[N]) {
    if (n != N) {
        PyErr_SetString(PyExc_TypeError, many);
        return false;
    }
    for (int i = 0; i < N; ++i) {
        p[i] = PyLong_AsVoidPtr(a[i]);
        if (!p[i]) {
            if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "address 0");
            return false;
        }
    }
    return true;
}

// bind(append, attention, workspace)
PyObject* bind(PyObject*, PyObject* const* a, Py_ssize_t n) {
    void* p[3];
    if (!addresses(a, n, "bind takes three addresses", p)) return nullptr;
    f_append = reinterpret_cast<decltype(f_append)>(p[0]);
    f_attention = reinterpret_cast<decltype(f_attention)>(p[1]);
    f_workspace = reinterpret_cast<decltype(f_workspace)>(p[2]);
    Py_RETURN_NONE;
}

// bind8(append, attention, workspace, read)
PyObject* bind8(PyObject*, PyObject* const* a, Py_ssize_t n) {
    void* p[4];
    if (!addresses(a, n, "bind8 takes four addresses", p)) return nullptr;
    f_append8 = reinterpret_cast<decltype(f_append8)>(p[0]);
    f_attention8 = reinterpret_cast<decltype(f_attention8)>(p[1]);
    f_workspace8 = reinterpret_cast<decltype(f_workspace8)>(p[2]);
    f_read8 = reinterpret_cast<decltype(f_read8)>(p[3]);
    Py_RETURN_NONE;
}

PyMethodDef methods[] = {
    {"append", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&append)), METH_FASTCALL, nullptr},
    {"attention", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&attention)), METH_FASTCALL, nullptr},
    {"append8", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&append8)), METH_FASTCALL, nullptr},
    {"attention8", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&attention8)), METH_FASTCALL, nullptr},
    {"read8", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&read8)), METH_FASTCALL, nullptr},
    {"bind8", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&bind8)), METH_FASTCALL, nullptr},
    {"bind", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&bind)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_paged_bind", "Calls of the paged-cache operators.", -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__paged_bind() {
    PyObject* m = PyModule_Create(&module);
    // the torch whose classes this file was compiled for; no other may use it
    if (m && PyModule_AddStringConstant(m, "torch_version", BREEZE_TORCH_VERSION) < 0) Py_CLEAR(m);
    return m;
}
