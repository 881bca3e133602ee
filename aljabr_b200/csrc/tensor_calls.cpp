// Tensors straight to the C-ABI: the calls of kv4.py whose kernels take less
// time than Python needs to look at their arguments (a rotated append of one
// token: 10 us of host time through ctypes, 3 us on the GPU).
//
// Each function checks everything that its method in kv4.py checks.  Where all
// is as it should be it makes the call and gives the result; otherwise it gives
// NotImplemented, touches nothing, and kv4.py says what is wrong.  A C-ABI call
// that refuses gives its status, an int.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <initializer_list>
#include <vector>

#include "../../include/aljabr_blackwell.h"

namespace {

using at::Tensor;

const Tensor* tensor(PyObject* o) { return THPVariable_Check(o) ? &THPVariable_Unpack(o) : nullptr; }

bool here(const Tensor& t, int index) { return t.is_cuda() && t.get_device() == index; }

bool ints(const Tensor* t, int index, at::IntArrayRef shape) {
    return t && t->scalar_type() == at::kInt && here(*t, index) && t->sizes() == shape && t->is_contiguous();
}

// Rows of [tokens, heads, D] (or, with flat, [tokens, heads * D]) that are contiguous each: elements between them, -1 otherwise.
long long rows(const Tensor* t, int index, at::ScalarType type, int64_t tokens, int64_t heads, int64_t D, bool flat) {
    if (!t || t->scalar_type() != type || !here(*t, index)) return -1;
    if (t->dim() == 3) {
        if (t->size(0) != tokens || t->size(1) != heads || t->size(2) != D || t->stride(2) != 1 || (heads > 1 && t->stride(1) != D)) return -1;
    } else if (!flat || t->dim() != 2 || t->size(0) != tokens || t->size(1) != heads * D || t->stride(1) != 1) {
        return -1;
    }
    return tokens > 1 ? t->stride(0) : heads * D;
}

// A raw stream from the argument: None or 0 is torch's current one, whose legacy stream the C-ABI knows as 1.
bool stream_of(PyObject* o, int index, void** stream, bool* current) {
    void* now = c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(index)).stream();
    if (!now) now = reinterpret_cast<void*>(1);
    *stream = now;
    if (o != Py_None) {
        const unsigned long long given = PyLong_Check(o) ? PyLong_AsUnsignedLongLong(o) : ~0ull;
        if (PyErr_Occurred() || given == ~0ull) {
            PyErr_Clear();
            return false;
        }
        if (given) *stream = reinterpret_cast<void*>(given);
    }
    *current = *stream == now;
    return true;
}

PyObject* no() { Py_RETURN_NOTIMPLEMENTED; }

// rotate_append(address, pages, page_size, kv_heads, head_dim, index, q, k, v, slots, positions, rope, interleaved, q_out,
//               k_back, v_back, stream) -> q_out
PyObject* rotate_append(PyObject*, PyObject* const* a, Py_ssize_t n) {
    if (n != 17) return no();
    const unsigned long long address = PyLong_AsUnsignedLongLong(a[0]);
    long dims[5];
    for (int i = 0; i < 5; ++i) dims[i] = PyLong_AsLong(a[1 + i]);
    if (PyErr_Occurred()) return nullptr;
    const int index = static_cast<int>(dims[4]);
    const int64_t heads = dims[2], D = dims[3];
    const Tensor *q = tensor(a[6]), *k = tensor(a[7]), *v = tensor(a[8]), *slots = tensor(a[9]), *positions = tensor(a[10]), *rope = tensor(a[11]);
    if (!q || !k || !slots || !rope || slots->dim() != 1 || q->dim() != 3 || rope->dim() != 3) return no();
    const int64_t tokens = slots->size(0), q_heads = q->size(1);
    if (tokens > INT32_MAX || rope->size(0) > INT32_MAX) return no();
    const at::ScalarType type = k->scalar_type();
    if ((type != at::kFloat && type != at::kBFloat16) || !ints(slots, index, {tokens}) || !ints(positions, index, {tokens})) return no();
    const long long qs = rows(q, index, type, tokens, q_heads, D, false), ks = rows(k, index, type, tokens, heads, D, true),
                    vs = rows(v, index, type, tokens, heads, D, true);
    if (qs < 0 || ks < 0 || vs < 0) return no();
    if (rope->scalar_type() != at::kFloat || !here(*rope, index) || rope->size(2) != 2 || !rope->is_contiguous()) return no();
    void* back[2] = {};
    for (int i = 0; i < 2; ++i) {
        if (a[14 + i] == Py_None) continue;
        const Tensor* t = tensor(a[14 + i]);
        if (!t || t->scalar_type() != type || !here(*t, index) || t->numel() != tokens * heads * D || !t->is_contiguous()) return no();
        back[i] = t->data_ptr();
    }
    const int inter = PyObject_IsTrue(a[12]);
    if (inter < 0) return nullptr;
    void* stream;
    bool current;
    if (!stream_of(a[16], index, &stream, &current)) return no();
    Tensor made;
    const Tensor* out = a[13] == Py_None ? nullptr : tensor(a[13]);
    if (a[13] == Py_None) {
        if (!current) return no();                 // memory of another stream's pool
        made = at::empty(q->sizes(), q->options());
        out = &made;
    }
    const long long os = rows(out, index, type, tokens, q_heads, D, false);
    if (os < 0) return no();
    // a tensor without memory of its own (a fake one) throws here, with the interpreter held
    const void *qp = q->data_ptr(), *kp = k->data_ptr(), *vp = v->data_ptr();
    void* const op = out->data_ptr();
    const int *sp = slots->data_ptr<int>(), *pp = positions->data_ptr<int>();
    const float* rp = rope->data_ptr<float>();
    const int n_rope = static_cast<int>(rope->size(0)), rotary = static_cast<int>(2 * rope->size(1));
    const int kind = type == at::kFloat ? ALJ_KV_F32 : ALJ_KV_BF16;
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = aljabr_blackwell_kv4_rotate_append_dev(reinterpret_cast<void*>(address), static_cast<int>(dims[0]), static_cast<int>(dims[1]),
                                                static_cast<int>(heads), static_cast<int>(D), op, os, qp, kp, vp, kind, qs, ks, vs,
                                                static_cast<int>(q_heads), sp, pp, rp, n_rope, rotary, inter, static_cast<int>(tokens),
                                                back[0], back[1], stream);
    Py_END_ALLOW_THREADS
    if (rc) return PyLong_FromLong(rc);
    if (a[13] == Py_None) return THPVariable_Wrap(made);
    Py_INCREF(a[13]);
    return a[13];
}

// accept_tree([addresses], pages, page_size, kv_heads, head_dim, index, seq_lens, parents, drafted, picked, block_table, out, stream)
//   -> (path, count, token, lens)
PyObject* accept_tree(PyObject*, PyObject* const* a, Py_ssize_t n) {
    if (n != 13 || !PyList_CheckExact(a[0])) return no();
    long dims[5];
    for (int i = 0; i < 5; ++i) dims[i] = PyLong_AsLong(a[1 + i]);
    if (PyErr_Occurred()) return nullptr;
    const int index = static_cast<int>(dims[4]);
    const Tensor *lens = tensor(a[6]), *parents = tensor(a[7]), *drafted = tensor(a[8]), *picked = tensor(a[9]), *table = nullptr;
    if (!drafted || !parents || drafted->dim() != 2) return no();
    const int64_t batch = drafted->size(0), nodes = drafted->size(1);
    if (!ints(drafted, index, {batch, nodes}) || !ints(picked, index, {batch, nodes}) || !ints(lens, index, {batch})) return no();
    const bool each = parents->dim() == 2;
    if (each ? !ints(parents, index, {batch, nodes}) : !ints(parents, index, {nodes})) return no();
    int64_t width = 0;
    if (a[10] != Py_None) {
        table = tensor(a[10]);
        if (!table || table->dim() != 2) return no();
        width = table->size(1);
        if (width < 1 || !ints(table, index, {batch, width})) return no();
    }
    const Py_ssize_t layers = PyList_GET_SIZE(a[0]);
    if (layers < 1 || layers > 256) return no();
    void* caches[256];
    for (Py_ssize_t i = 0; i < layers; ++i) caches[i] = reinterpret_cast<void*>(PyLong_AsUnsignedLongLong(PyList_GET_ITEM(a[0], i)));
    if (PyErr_Occurred()) return nullptr;
    void* stream;
    bool current;
    if (!stream_of(a[12], index, &stream, &current)) return no();
    Tensor path, count, token, left;
    if (a[11] == Py_None) {
        if (!current) return no();
        // one allocation; the small ones lie behind the path
        const Tensor all = at::empty({batch * (nodes + 3)}, drafted->options());
        path = all.as_strided({batch, nodes}, {nodes, 1}, 0);
        count = all.as_strided({batch}, {1}, batch * nodes);
        token = all.as_strided({batch}, {1}, batch * (nodes + 1));
        left = all.as_strided({batch}, {1}, batch * (nodes + 2));
    } else {
        if (!PyTuple_CheckExact(a[11]) || PyTuple_GET_SIZE(a[11]) != 4) return no();
        const Tensor* out[4];
        for (int i = 0; i < 4; ++i) out[i] = tensor(PyTuple_GET_ITEM(a[11], i));
        if (!ints(out[0], index, {batch, nodes}) || !ints(out[1], index, {batch}) || !ints(out[2], index, {batch}) || !ints(out[3], index, {batch}))
            return no();
        path = *out[0], count = *out[1], token = *out[2], left = *out[3];
    }
    int* const outs[4] = {path.data_ptr<int>(), count.data_ptr<int>(), token.data_ptr<int>(), left.data_ptr<int>()};
    const int *tp = table ? table->data_ptr<int>() : nullptr, *lp = lens->data_ptr<int>(), *pp = parents->data_ptr<int>(),
              *dp = drafted->data_ptr<int>(), *kp = picked->data_ptr<int>();
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = aljabr_blackwell_kv4_accept_tree_dev(outs[0], outs[1], outs[2], outs[3], caches, static_cast<int>(layers), static_cast<int>(dims[0]),
                                              static_cast<int>(dims[1]), static_cast<int>(dims[2]), static_cast<int>(dims[3]), tp,
                                              static_cast<int>(width), lp, static_cast<int>(batch), pp, each ? static_cast<int>(nodes) : 0,
                                              static_cast<int>(nodes), dp, kp, stream);
    Py_END_ALLOW_THREADS
    if (rc) return PyLong_FromLong(rc);
    if (a[11] != Py_None) {
        Py_INCREF(a[11]);
        return a[11];
    }
    PyObject* got = PyTuple_New(4);
    if (!got) return nullptr;
    const Tensor* all[4] = {&path, &count, &token, &left};
    for (int i = 0; i < 4; ++i) {
        PyObject* t = THPVariable_Wrap(*all[i]);
        if (!t) {
            Py_DECREF(got);
            return nullptr;
        }
        PyTuple_SET_ITEM(got, i, t);
    }
    return got;
}

// What torch throws (no memory, a stream of no device) as a Python error.
template <PyObject* (*F)(PyObject*, PyObject* const*, Py_ssize_t)>
PyObject* guarded(PyObject* self, PyObject* const* a, Py_ssize_t n) {
    try {
        return F(self, a, n);
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
        return nullptr;
    }
}

PyMethodDef methods[] = {
    {"rotate_append", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(guarded<rotate_append>)), METH_FASTCALL, nullptr},
    {"accept_tree", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(guarded<accept_tree>)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "tensor_calls", ALJ_MARK, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_tensor_calls(void) {
    PyObject* m = PyModule_Create(&module);
    if (m && PyModule_AddStringConstant(m, "torch", ALJ_TORCH)) {   // the torch it was built with, which kv4.py compares
        Py_DECREF(m);
        return nullptr;
    }
    return m;
}
