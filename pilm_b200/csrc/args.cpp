// Python entry of the 8-bit KV cache calls: checks the tensors and makes the C call.
//
// A verify step makes two of these calls per layer, each a few microseconds on the GPU.  Checking
// fourteen tensors from Python (dtype, device, size, contiguity, address: five attribute calls
// each) and passing them through ctypes takes longer than the kernels; here it takes under a
// microsecond.  The functions' addresses come from the library that bindings.py has loaded.
#include <Python.h>
#include <torch/csrc/autograd/python_variable.h>

#include <exception>
#include <string>

#include "../../include/pilm_cuda.h"

namespace {

decltype(&ekernel_qk_norm_rope_kv_append_kv8) g_append = nullptr;
decltype(&ekernel_qk_norm_rope_kv_append_kv8_splitk) g_append_splitk = nullptr;
decltype(&ekernel_paged_attention_verify_kv8) g_attention = nullptr;

// Collects the addresses of a call's tensors; after the first bad one the rest are skipped and a
// ValueError is set.
struct Args {
    int dev;
    bool ok = true;

    const at::Tensor *tensor(const char *name, PyObject *o) {
        if (!ok) return nullptr;
        if (!THPVariable_Check(o)) {
            ok = false;
            PyErr_Format(PyExc_ValueError, "%s must be a tensor, got %s", name, Py_TYPE(o)->tp_name);
            return nullptr;
        }
        return &THPVariable_Unpack(o);
    }
    void *at(const char *name, PyObject *o, at::ScalarType dtype, size_t numel) {
        const at::Tensor *t = tensor(name, o);
        if (!t) return nullptr;
        if (!t->is_cuda() || t->get_device() != dev || t->scalar_type() != dtype || (size_t)t->numel() < numel ||
            !t->is_contiguous()) {
            ok = false;
            std::string shape;
            for (const int64_t n : t->sizes()) shape += (shape.empty() ? "" : ", ") + std::to_string(n);
            PyErr_Format(PyExc_ValueError,
                         "%s must be a contiguous %s CUDA tensor of at least %zu elements on cuda:%d, got %s [%s] on %s%s",
                         name, at::toString(dtype), numel, dev, at::toString(t->scalar_type()), shape.c_str(),
                         t->device().str().c_str(), t->is_contiguous() ? "" : " (not contiguous)");
            return nullptr;
        }
        return t->data_ptr();
    }
    void *maybe(const char *name, PyObject *o, bool used, at::ScalarType dtype, size_t numel) {
        return !ok || !used || o == Py_None ? nullptr : at(name, o, dtype, numel);
    }
};

// The descriptor inside a ctypes structure.
struct Desc {
    Py_buffer buf{};
    const ekernel_paged_attn_desc_t *d = nullptr;
    explicit Desc(PyObject *o) {
        if (PyObject_GetBuffer(o, &buf, PyBUF_SIMPLE) != 0) return;
        if (buf.len == (Py_ssize_t)sizeof(ekernel_paged_attn_desc_t))
            d = static_cast<const ekernel_paged_attn_desc_t *>(buf.buf);
        else
            PyErr_SetString(PyExc_ValueError, "desc must be a PagedAttnDesc");
    }
    ~Desc() {
        if (buf.obj) PyBuffer_Release(&buf);
    }
};

template <typename T>
T *as(void *p) {
    return static_cast<T *>(p);
}

bool unsigned_arg(const char *name, PyObject *o, size_t *out) {
    const long long v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) return false;
    if (v < 0) {
        PyErr_Format(PyExc_ValueError, "%s must not be negative, got %lld", name, v);
        return false;
    }
    *out = (size_t)v;
    return true;
}

PyObject *result(int rc) { return PyLong_FromLong(rc); }

bool bound(PyObject *const *, Py_ssize_t n, Py_ssize_t want) {
    if (!g_append || !g_append_splitk || !g_attention) {
        PyErr_SetString(PyExc_RuntimeError, "bind() has not been called");
        return false;
    }
    if (n != want) {
        PyErr_Format(PyExc_TypeError, "expected %zd arguments, got %zd", want, n);
        return false;
    }
    return true;
}

// bind(append, append_splitk, attention): the functions' addresses
PyObject *py_bind(PyObject *, PyObject *const *a, Py_ssize_t n) {
    if (n != 3) {
        PyErr_SetString(PyExc_TypeError, "bind takes three addresses");
        return nullptr;
    }
    void *p[3];
    for (int i = 0; i < 3; ++i)
        if (!(p[i] = PyLong_AsVoidPtr(a[i]))) {
            if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "null address");
            return nullptr;
        }
    g_append = reinterpret_cast<decltype(g_append)>(p[0]);
    g_append_splitk = reinterpret_cast<decltype(g_append_splitk)>(p[1]);
    g_attention = reinterpret_cast<decltype(g_attention)>(p[2]);
    Py_RETURN_NONE;
}

// append(dev, desc, src, splits (0: src is the bf16 projection), q_norm_w, k_norm_w, rope_cos,
//        rope_sin, positions, slot_mapping, k_cache, v_cache, k_scale, v_scale, q_out, gate_out)
PyObject *py_append(PyObject *, PyObject *const *a, Py_ssize_t n) {
    if (!bound(a, n, 16)) return nullptr;
    const long dev = PyLong_AsLong(a[0]);
    size_t splits = 0;
    if ((dev == -1 && PyErr_Occurred()) || !unsigned_arg("splits", a[3], &splits)) return nullptr;
    Desc desc(a[1]);
    const auto *d = desc.d;
    if (!d) return nullptr;
    const auto bf = at::kBFloat16, f32 = at::kFloat, i32 = at::kInt, u8 = at::kByte;
    const size_t t = d->total_q, hd = d->head_dim, rows = t * d->n_heads * hd, table = d->rope_rows * (d->rot_dim / 2);
    const size_t pages = d->num_blocks * d->n_kv_heads, codes = pages * d->block_size * hd;
    Args c{(int)dev};
    void *src = splits ? c.at("partials", a[2], f32, splits * t * d->qkv_stride) : c.at("qkv", a[2], bf, t * d->qkv_stride);
    auto *qn = as<uint16_t>(c.at("q_norm_w", a[4], bf, hd)), *kn = as<uint16_t>(c.at("k_norm_w", a[5], bf, hd));
    auto *cos = as<float>(c.at("rope_cos", a[6], f32, table)), *sin = as<float>(c.at("rope_sin", a[7], f32, table));
    auto *pos = as<int32_t>(c.at("positions", a[8], i32, t)), *slots = as<int32_t>(c.at("slot_mapping", a[9], i32, t));
    auto *kc = as<uint8_t>(c.at("k_cache", a[10], u8, codes)), *vc = as<uint8_t>(c.at("v_cache", a[11], u8, codes));
    auto *ks = as<float>(c.at("k_scale", a[12], f32, pages)), *vs = as<float>(c.at("v_scale", a[13], f32, pages));
    auto *q = as<uint16_t>(c.at("q_out", a[14], bf, rows));
    auto *g = as<uint16_t>(c.maybe("gate_out", a[15], d->output_gate != 0, bf, rows));
    if (!c.ok) return nullptr;
    return result(splits ? g_append_splitk(d, as<float>(src), (int32_t)splits, qn, kn, cos, sin, pos, slots, kc, vc, ks, vs, q, g)
                         : g_append(d, as<uint16_t>(src), qn, kn, cos, sin, pos, slots, kc, vc, ks, vs, q, g));
}

// attention(dev, desc, q, k_cache, v_cache, k_scale, v_scale, block_table, cu_q, context_lens, gate,
//           out, window, sinks, workspace)
PyObject *py_attention(PyObject *, PyObject *const *a, Py_ssize_t n) {
    if (!bound(a, n, 15)) return nullptr;
    const long dev = PyLong_AsLong(a[0]);
    size_t window = 0, sinks = 0;
    if ((dev == -1 && PyErr_Occurred()) || !unsigned_arg("window", a[12], &window) || !unsigned_arg("sinks", a[13], &sinks))
        return nullptr;
    Desc desc(a[1]);
    const auto *d = desc.d;
    if (!d) return nullptr;
    const auto bf = at::kBFloat16, f32 = at::kFloat, i32 = at::kInt, u8 = at::kByte;
    const size_t rows = d->total_q * d->n_heads * d->head_dim, seqs = d->num_seqs;
    const size_t pages = d->num_blocks * d->n_kv_heads, codes = pages * d->block_size * d->head_dim;
    Args c{(int)dev};
    auto *q = as<uint16_t>(c.at("q", a[2], bf, rows));
    auto *kc = as<uint8_t>(c.at("k_cache", a[3], u8, codes)), *vc = as<uint8_t>(c.at("v_cache", a[4], u8, codes));
    auto *ks = as<float>(c.at("k_scale", a[5], f32, pages)), *vs = as<float>(c.at("v_scale", a[6], f32, pages));
    auto *table = as<int32_t>(c.at("block_table", a[7], i32, seqs * d->max_blocks_per_seq));
    auto *cu = as<int32_t>(c.at("cu_q", a[8], i32, seqs + 1)), *ctx = as<int32_t>(c.at("context_lens", a[9], i32, seqs));
    auto *gate = as<uint16_t>(c.maybe("gate", a[10], d->output_gate != 0, bf, rows));
    auto *out = as<uint16_t>(c.at("out", a[11], bf, rows));
    void *ws = c.at("workspace", a[14], u8, 0);
    if (!c.ok) return nullptr;
    return result(g_attention(d, q, kc, vc, ks, vs, table, cu, ctx, gate, window, sinks, ws,
                              (size_t)THPVariable_Unpack(a[14]).numel(), out));
}

// torch reports trouble by exceptions (a tensor without storage, say): they end here as Python's
using Fast = PyObject *(*)(PyObject *, PyObject *const *, Py_ssize_t);
template <Fast F>
PyObject *guarded(PyObject *self, PyObject *const *a, Py_ssize_t n) {
    try {
        return F(self, a, n);
    } catch (const std::exception &e) {
        if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, e.what());
    } catch (...) {
        if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, "unknown C++ exception");
    }
    return nullptr;
}
template <Fast F>
PyCFunction method() {
    return reinterpret_cast<PyCFunction>(reinterpret_cast<void *>(&guarded<F>));
}

PyMethodDef kMethods[] = {
    {"bind", method<py_bind>(), METH_FASTCALL, nullptr},
    {"append", method<py_append>(), METH_FASTCALL, nullptr},
    {"attention", method<py_attention>(), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_args", "Checked calls of the 8-bit KV cache kernels.", -1, kMethods,
                       nullptr, nullptr, nullptr, nullptr};

}  // namespace

extern "C" __attribute__((visibility("default"))) PyObject *PyInit__args(void) { return PyModule_Create(&kModule); }
