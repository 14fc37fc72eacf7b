// The operators over a paged cache called from Python without ctypes in between (megacute_b200/paged.py).  Each function looks at its tensors, makes the
// result and calls the C ABI; arguments that are not plainly right, and whatever fails, give None, and the caller's own checks then say why.
// A call of one token takes the host 4 to 6 us that way, launch included, 12 to 17 through ctypes.
#include <Python.h>
#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>

#include "megacute_b200.h"

namespace {

struct Abi {
    decltype(&mk_rotary) rotary = nullptr;
    decltype(&mk_paged_append) append = nullptr;
    decltype(&mk_paged_attention) attention = nullptr;
    decltype(&mk_paged_attention_workspace) workspace = nullptr;
} abi;

struct Rows {                                         // a 2-D tensor whose rows start on 16-byte boundaries
    char* p = nullptr;
    long long ld = 0, rows = 0, cols = 0;
    int size = 0, dtype = -1;                         // dtype: the ABI's code
    long long bytes() const { return ((rows - 1) * ld + cols) * size; }
};

int code_of(at::ScalarType t) {
    return t == at::kBFloat16 ? 0 : t == at::kFloat ? 1 : t == at::kHalf ? 2 : -1;
}
const at::Tensor* tensor(PyObject* o, int device) {
    if (!THPVariable_Check(o)) return nullptr;
    const at::Tensor& t = THPVariable_Unpack(o);
    if (!t.defined() || t.layout() != at::kStrided || !t.is_cuda() || (device >= 0 && t.get_device() != device)) return nullptr;
    return &t;
}
// cols < 0: any number
bool rows_of(PyObject* o, int device, long long cols, Rows& r) {
    const at::Tensor* const t = tensor(o, device);
    if (!t || t->dim() != 2) return false;
    r.dtype = code_of(t->scalar_type());
    if (r.dtype < 0) return false;
    r.size = r.dtype == 1 ? 4 : 2;
    r.rows = t->size(0);
    r.cols = t->size(1);
    const long long ld = t->stride(0);
    if (cols >= 0 && r.cols != cols) return false;
    if ((t->stride(1) != 1 && r.cols > 1) || (ld < r.cols && r.rows > 1) || ld * r.size % 16) return false;
    r.ld = ld > r.cols ? ld : r.cols;
    r.p = static_cast<char*>(t->data_ptr());
    return (reinterpret_cast<uintptr_t>(r.p) & 15) == 0;
}
// int32, unit stride in the last of `dim` dimensions
const at::Tensor* ints(PyObject* o, int device, int dim) {
    const at::Tensor* const t = tensor(o, device);
    if (!t || t->scalar_type() != at::kInt || t->dim() != dim || t->stride(0) < 0 || (t->stride(dim - 1) != 1 && t->size(dim - 1) > 1)) return nullptr;
    return t;
}
bool batch_of(PyObject* pos, PyObject* starts, int device, long long rows, mk_batch& b) {
    const at::Tensor* const p = ints(pos, device, 2);
    if (!p || p->size(1) != 1 || rows <= 0 || rows > 0x7fffffff) return false;
    const long long seqs = p->size(0);
    if (seqs <= 0 || seqs > 0x7ffffffe) return false;
    b = mk_batch{};
    b.pos = p->const_data_ptr<int32_t>();
    b.pos_ld = p->stride(0);
    b.rows = (int)rows;
    b.seqs = (int)seqs;
    if (starts == Py_None) return rows % seqs == 0;
    const at::Tensor* const s = ints(starts, device, 1);
    if (!s || s->size(0) != seqs + 1) return false;
    b.starts = s->const_data_ptr<int32_t>();
    return true;
}
bool rotation_of(PyObject* cos, PyObject* sin, bool interleaved, long long head_dim, int device, mk_rotation& r) {
    Rows c, s;
    if (!rows_of(cos, device, -1, c) || !rows_of(sin, device, c.cols, s) || c.rows != s.rows || c.dtype != s.dtype) return false;
    if (c.cols % 8 || c.cols == 0 || 2 * c.cols > head_dim || c.rows == 0 || c.rows > 0x7fffffff) return false;
    r = mk_rotation{c.p, s.p, c.ld, s.ld, (int)c.rows, (int)c.cols, c.dtype, interleaved ? 1 : 0};
    return true;
}
bool cache_of(PyObject* kc, PyObject* vc, PyObject* table, long long seqs, long long kv_heads, long long head_dim, long long page_size, int dtype, int device,
              mk_paged_cache& c, Rows& k, Rows& v) {
    if (kv_heads <= 0 || page_size < 16 || page_size > 0x40000000 || (page_size & (page_size - 1))) return false;
    if (!rows_of(kc, device, kv_heads * head_dim, k) || !rows_of(vc, device, kv_heads * head_dim, v) || k.dtype != dtype || v.dtype != dtype) return false;
    const at::Tensor* const t = ints(table, device, 2);
    if (!t || t->size(0) != seqs || k.rows != v.rows || k.rows % page_size || k.rows > 0x7fffffff || t->size(1) > 0x7fff0000ll / page_size) return false;
    c = mk_paged_cache{k.p, v.p, t->const_data_ptr<int32_t>(), k.ld, v.ld, t->stride(0), (int)(k.rows / page_size), (int)page_size, (int)t->size(1),
                       (int)kv_heads, (int)head_dim, dtype};
    return true;
}
// no memory in common, or different columns of one tensor's rows
bool apart(const Rows& a, const Rows& b) {
    if (a.rows == 0 || b.rows == 0 || a.p >= b.p + b.bytes() || b.p >= a.p + a.bytes()) return true;
    const long long pitch = a.ld * a.size;
    if (pitch != b.ld * b.size) return false;
    const long long at = ((b.p - a.p) % pitch + pitch) % pitch;
    return at >= a.cols * a.size && at + b.cols * b.size <= pitch;
}
at::Tensor make(at::ScalarType type, long long rows, long long cols, int device) {
    return at::empty({rows, cols}, at::TensorOptions().dtype(type).device(at::kCUDA, (c10::DeviceIndex)device));
}
at::ScalarType type_of(int code) { return code == 0 ? at::kBFloat16 : code == 1 ? at::kFloat : at::kHalf; }
void* stream_of(int device) { return c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)device).stream(); }

// whole numbers of 32 bits from args[0 ..]
bool numbers(PyObject* const* args, int n, long long* to) {
    for (int i = 0; i < n; ++i) {
        if (!PyLong_Check(args[i])) return false;
        to[i] = PyLong_AsLongLong(args[i]);
        if (PyErr_Occurred() || to[i] < -0x7fffffffll || to[i] > 0x7fffffffll) return false;
    }
    return true;
}
// heads, kv heads, elements of a head: positive, and products of them far from 63 bits
bool sizes(const long long* v, int n) {
    for (int i = 0; i < n; ++i)
        if (v[i] <= 0 || v[i] > 1 << 24) return false;
    return true;
}
PyObject* none() {
    PyErr_Clear();
    Py_RETURN_NONE;
}
int device_of(PyObject* x) {
    const at::Tensor* const t = tensor(x, -1);
    return t ? (int)t->get_device() : -1;
}

// (x, cos, sin, pos, starts, heads, head_dim, interleaved)
PyObject* rotary(PyObject*, PyObject* const* args, Py_ssize_t n) {
    try {
        long long v[2];
        Rows x;
        mk_batch batch;
        mk_rotation rot;
        const int device = n == 8 && abi.rotary ? device_of(args[0]) : -1, pairs = device < 0 ? -1 : PyObject_IsTrue(args[7]);
        if (pairs < 0 || !numbers(args + 5, 2, v) || !sizes(v, 2) || v[1] % 16) return none();
        if (!rows_of(args[0], device, v[0] * v[1], x) || !rotation_of(args[1], args[2], pairs, v[1], device, rot) ||
            !batch_of(args[3], args[4], device, x.rows, batch))
            return none();
        at::Tensor out = make(type_of(x.dtype), x.rows, x.cols, device);
        if (abi.rotary(device, &batch, &rot, x.p, x.ld, out.data_ptr(), x.cols, x.dtype, (int)v[0], (int)v[1], stream_of(device))) return none();
        return THPVariable_Wrap(std::move(out));
    } catch (...) {
        return none();
    }
}
// (qkv, cos, sin, pos, k_cache, v_cache, pages, starts, heads, kv_heads, head_dim, page_size, interleaved)
PyObject* paged_append(PyObject*, PyObject* const* args, Py_ssize_t n) {
    try {
        long long v[4];
        Rows x, k, vv;
        mk_batch batch;
        mk_rotation rot;
        mk_paged_cache cache;
        const int device = n == 13 && abi.append ? device_of(args[0]) : -1, pairs = device < 0 ? -1 : PyObject_IsTrue(args[12]);
        if (pairs < 0 || !numbers(args + 8, 4, v) || !sizes(v, 3) || v[2] % 16) return none();
        if (!rows_of(args[0], device, (v[0] + 2 * v[1]) * v[2], x) || x.dtype == 1 ||
            !rotation_of(args[1], args[2], pairs, v[2], device, rot) || !batch_of(args[3], args[7], device, x.rows, batch) ||
            !cache_of(args[4], args[5], args[6], batch.seqs, v[1], v[2], v[3], x.dtype, device, cache, k, vv))
            return none();
        if (!apart(k, x) || !apart(vv, x) || !apart(k, vv)) return none();
        at::Tensor out = make(type_of(x.dtype), x.rows, v[0] * v[2], device);
        if (abi.append(device, &batch, &rot, &cache, x.p, x.ld, out.data_ptr(), v[0] * v[2], (int)v[0], stream_of(device))) return none();
        return THPVariable_Wrap(std::move(out));
    } catch (...) {
        return none();
    }
}
// (q, k_cache, v_cache, pos, pages, starts, heads, kv_heads, head_dim, page_size, scale, window, max_new)
PyObject* paged_attention(PyObject*, PyObject* const* args, Py_ssize_t n) {
    try {
        long long v[4], window = 0, max_new = 0;
        Rows x, k, vv;
        mk_batch batch;
        mk_paged_cache cache;
        const int device = n == 13 && abi.attention ? device_of(args[0]) : -1;
        if (device < 0 || !numbers(args + 6, 4, v) || !sizes(v, 3) || v[0] % v[1] || (v[2] != 64 && v[2] != 128)) return none();
        if (args[10] != Py_None && !PyFloat_Check(args[10]) && !PyLong_Check(args[10])) return none();
        const double scale = args[10] == Py_None ? std::pow((double)v[2], -0.5) : PyFloat_AsDouble(args[10]);
        if (PyErr_Occurred() || (args[11] != Py_None && !numbers(args + 11, 1, &window)) || window < 0) return none();
        if (!rows_of(args[0], device, v[0] * v[2], x) || x.dtype == 1 || !batch_of(args[3], args[5], device, x.rows, batch) ||
            !cache_of(args[1], args[2], args[4], batch.seqs, v[1], v[2], v[3], x.dtype, device, cache, k, vv))
            return none();
        if (!batch.starts) max_new = batch.rows / batch.seqs;
        else if (args[12] == Py_None) max_new = batch.rows;
        else if (!numbers(args + 12, 1, &max_new)) return none();
        const long long bytes = abi.workspace(device, (int)v[0], (int)v[1], (int)v[2], (int)max_new);
        if (bytes < 0) return none();
        at::Tensor out = make(type_of(x.dtype), x.rows, x.cols, device), workspace = make(at::kByte, 1, bytes, device);
        if (abi.attention(device, &batch, &cache, x.p, x.ld, out.data_ptr(), x.cols, (int)v[0], (float)scale, (int)window, (int)max_new,
                          workspace.data_ptr(), (size_t)bytes, stream_of(device)))
            return none();
        return THPVariable_Wrap(std::move(out));
    } catch (...) {
        return none();
    }
}
// the ABI's functions by address: mk_rotary, mk_paged_append, mk_paged_attention, mk_paged_attention_workspace
PyObject* bind(PyObject*, PyObject* const* args, Py_ssize_t n) {
    void* p[4];
    for (int i = 0; i < 4; ++i) {
        p[i] = n == 4 ? PyLong_AsVoidPtr(args[i]) : nullptr;
        if (PyErr_Occurred() || !p[i]) {
            PyErr_SetString(PyExc_ValueError, "bind: four addresses");
            return nullptr;
        }
    }
    abi.rotary = reinterpret_cast<decltype(abi.rotary)>(p[0]);
    abi.append = reinterpret_cast<decltype(abi.append)>(p[1]);
    abi.attention = reinterpret_cast<decltype(abi.attention)>(p[2]);
    abi.workspace = reinterpret_cast<decltype(abi.workspace)>(p[3]);
    Py_RETURN_NONE;
}

PyMethodDef methods[] = {
    {"bind", (PyCFunction)(void (*)(void))bind, METH_FASTCALL, nullptr},
    {"rotary", (PyCFunction)(void (*)(void))rotary, METH_FASTCALL, nullptr},
    {"paged_append", (PyCFunction)(void (*)(void))paged_append, METH_FASTCALL, nullptr},
    {"paged_attention", (PyCFunction)(void (*)(void))paged_attention, METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_binding", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

// (the module's view of a tensor is that of the torch it was built against: `built_for` names it)
PyMODINIT_FUNC PyInit__binding(void) {
    PyObject* const m = PyModule_Create(&module);
    if (m && PyModule_AddStringConstant(m, "built_for", MK_TORCH_VERSION)) {
        Py_DECREF(m);
        return nullptr;
    }
    return m;
}
