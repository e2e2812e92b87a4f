// Host side of breeze_b200.fused.paged's calls: reads the tensors, fills the
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

// append(qkv, cos, sin, k_pages, v_pages, page_table, seq_lens, q_starts, q_norm_w, k_norm_w, eps, out, flags)
PyObject* append(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        need(n == 13 && f_append);
        const at::Tensor &qkv = tensor(a[0]), &cos = tensor(a[1]), &sin = tensor(a[2]);
        bq_paged_append_desc d;
        std::memset(&d, 0, sizeof(d));
        d.ldqkv = row_stride(qkv);
        const int dev = fill(&d.kv, qkv, a[3], a[4], a[5], a[6], a[7]);
        const int64_t rows = qkv.size(0), width = qkv.size(1), hq = width / d.kv.D - 2 * int64_t(d.kv.HKV);
        need(hq > 0 && (hq + 2 * int64_t(d.kv.HKV)) * d.kv.D == width);
        const at::ScalarType type = qkv.scalar_type(), cs = cos.scalar_type();
        d.ldcs = row_stride(cos);
        need(cos.size(1) == d.kv.D && sin.sizes() == cos.sizes() && sin.scalar_type() == cs && row_stride(sin) == d.ldcs);
        need((cs == type || cs == at::kFloat) && on(cos, dev) && on(sin, dev));
        if (a[8] != Py_None || a[9] != Py_None) {
            const at::Tensor &qn = tensor(a[8]), &kn = tensor(a[9]);
            need(vector(qn, type, d.kv.D, dev) && vector(kn, type, d.kv.D, dev));
            d.q_norm = qn.data_ptr();
            d.k_norm = kn.data_ptr();
        }
        d.T = i32(rows);
        d.HQ = i32(hq);
        d.cs_dtype = cs == at::kFloat ? BQ_DT_F32 : d.kv.dtype;
        d.rope_rows = i32(cos.size(0));
        d.eps = real(a[10]);
        d.flags = uint32_t(integer(a[12]));
        d.qkv = qkv.data_ptr();
        d.cos = cos.data_ptr();
        d.sin = sin.data_ptr();
        const at::Tensor out = output(a[11], qkv, rows, hq * d.kv.D, dev, &d.ldq);
        d.q_out = out.data_ptr();
        void* stream = c10::cuda::getCurrentCUDAStream(c10::DeviceIndex(dev)).stream();
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
        const int64_t rows = q.size(0), width = q.size(1), hq = width / d.kv.D;
        need(hq > 0 && hq * d.kv.D == width && hq % d.kv.HKV == 0);
        d.T = i32(rows);
        d.HQ = i32(hq);
        d.prefix_len = i32(integer(a[5]));
        d.max_q = a[8] == Py_None ? 0 : i32(integer(a[8]));
        d.scale = a[7] == Py_None ? float(1.0 / std::sqrt(double(d.kv.D))) : real(a[7]);
        d.flags = uint32_t(integer(a[11]));
        d.q = q.data_ptr();
        if (a[10] != Py_None) {
            const at::Tensor& lse = tensor(a[10]);
            need(lse.dim() == 2 && lse.size(0) == rows && lse.size(1) == hq && lse.scalar_type() == at::kFloat && on(lse, dev));
            d.lse = static_cast<float*>(lse.data_ptr());
            d.ldl = row_stride(lse);
        }
        const at::Tensor out = output(a[9], q, rows, width, dev, &d.ldo);
        d.out = out.data_ptr();
        size_t bytes = 0;
        int32_t rc = f_workspace(&d, &bytes);
        if (rc != BQ_OK) return PyLong_FromLong(rc);
        at::Tensor ws;  // from torch's allocator: calls on other streams, and other graphs, have their own
        if (bytes) ws = at::empty({int64_t(bytes)}, q.options().dtype(at::kByte));
        void* stream = c10::cuda::getCurrentCUDAStream(c10::DeviceIndex(dev)).stream();
        return result(launched([&] { return f_attention(&d, bytes ? ws.data_ptr() : nullptr, bytes, stream); }), out, a[9]);
    });
}

// bind(append, attention, workspace): addresses of the loaded library's entries
PyObject* bind(PyObject*, PyObject* const* a, Py_ssize_t n) {
    if (n != 3) {
        PyErr_SetString(PyExc_TypeError, "bind takes three addresses");
        return nullptr;
    }
    void* p[3];
    for (int i = 0; i < 3; ++i) {
        p[i] = PyLong_AsVoidPtr(a[i]);
        if (!p[i]) {
            if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "address 0");
            return nullptr;
        }
    }
    f_append = reinterpret_cast<decltype(f_append)>(p[0]);
    f_attention = reinterpret_cast<decltype(f_attention)>(p[1]);
    f_workspace = reinterpret_cast<decltype(f_workspace)>(p[2]);
    Py_RETURN_NONE;
}

PyMethodDef methods[] = {
    {"append", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&append)), METH_FASTCALL, nullptr},
    {"attention", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&attention)), METH_FASTCALL, nullptr},
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
