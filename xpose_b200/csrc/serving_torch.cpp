// Torch tensors to the serving entry points of include/xp_cuda.h: the checks
// of xpose_b200/serving.py in C++, because a decode step's kernels take less
// time than the same checks in Python. Every function returns None, or
// (status, message) for the caller to raise.
#include <Python.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <string>

#include "../../include/xp_cuda.h"

namespace {

struct Bad {
    std::string message;
};
[[noreturn]] void bad(const std::string& m) { throw Bad{m}; }

const at::Tensor& tensor(PyObject* o, const char* name) {
    if (!THPVariable_Check(o)) bad(std::string("'") + name + "' must be a tensor");
    const at::Tensor& t = THPVariable_Unpack(o);
    if (!t.is_cuda()) bad(std::string("'") + name + "' must be a CUDA tensor");
    return t;
}

xp_rows rows(PyObject* o, const char* name) {
    const at::Tensor& t = tensor(o, name);
    xp_rows r{};
    switch (t.scalar_type()) {
        case at::kFloat: r.dtype = XP_F32; break;
        case at::kHalf: r.dtype = XP_F16; break;
        case at::kBFloat16: r.dtype = XP_BF16; break;
        default: bad(std::string("'") + name + "' must be float32, float16 or bfloat16");
    }
    if (t.dim() != 3) bad(std::string("'") + name + "' must be [tokens, heads, dim]");
    if (t.size(2) > 1 && t.stride(2) != 1) bad(std::string("the last axis of '") + name + "' must be contiguous");
    if (t.size(0) > 0x7FFFFFFF || t.size(1) > 0x7FFFFFFF || t.size(2) > 0x7FFFFFFF)
        bad(std::string("'") + name + "' is too large");
    r.data = t.data_ptr();
    r.tokens = (uint32_t)t.size(0);
    r.heads = (uint32_t)t.size(1);
    r.dim = (uint32_t)t.size(2);
    r.token_stride = r.tokens > 1 ? t.stride(0) : 0;  // a lone row or head has no stride
    r.head_stride = r.heads > 1 ? t.stride(1) : 0;
    return r;
}

// a contiguous tensor of n values (n < 0: any number)
void* flat(PyObject* o, const char* name, at::ScalarType type, int64_t n) {
    const at::Tensor& t = tensor(o, name);
    if (t.scalar_type() != type || !t.is_contiguous() || (n >= 0 && t.numel() != n))
        bad(std::string("'") + name + "' must be contiguous, of type " + c10::toString(type) +
            (n >= 0 ? " and of " + std::to_string(n) + " values" : std::string()));
    return t.data_ptr();
}

xp_pages pages(PyObject* const* a) {  // k, v, k_scale, v_scale
    const at::Tensor &k = tensor(a[0], "k_pages"), &v = tensor(a[1], "v_pages");
    xp_pages p{};
    switch (k.scalar_type()) {
        case at::kHalf: p.dtype = XP_F16; break;
        case at::kBFloat16: p.dtype = XP_BF16; break;
        case at::kChar: p.dtype = XP_INT8; break;
        case at::kFloat8_e4m3fn: p.dtype = XP_FP8_E4M3; break;
        default: bad("the pages must be float16, bfloat16, int8 or float8_e4m3fn");
    }
    if (k.dim() != 4 || v.sizes() != k.sizes() || v.scalar_type() != k.scalar_type() || !k.is_contiguous() ||
        !v.is_contiguous())
        bad("the pages must be two contiguous tensors [pages, kv heads, page size, dim] of one type");
    if (k.size(1) > 0x7FFFFFFF || k.size(2) > 0x7FFFFFFF || k.size(3) > 0x7FFFFFFF) bad("the pages are too large");
    p.k = k.data_ptr();
    p.v = v.data_ptr();
    p.num_pages = (uint64_t)k.size(0);
    p.kv_heads = (uint32_t)k.size(1);
    p.page_size = (uint32_t)k.size(2);
    p.head_dim = (uint32_t)k.size(3);
    if (k.element_size() == 1) {
        if (a[2] == Py_None || a[3] == Py_None) bad("8-bit pages need k_scale and v_scale");
        const int64_t n = k.size(0) * k.size(1) * k.size(2);
        p.k_scale = static_cast<float*>(flat(a[2], "k_scale", at::kFloat, n));
        p.v_scale = static_cast<float*>(flat(a[3], "v_scale", at::kFloat, n));
    }
    return p;
}

xp_rotary rotary(PyObject* positions, PyObject* turns, PyObject* layout, PyObject* magnitude, PyObject* inverse,
                 uint32_t tokens) {
    xp_rotary r{};
    r.turns = static_cast<const uint64_t*>(flat(turns, "turns", at::kLong, -1));
    r.positions = static_cast<const int32_t*>(flat(positions, "positions", at::kInt, tokens));
    const int64_t n = THPVariable_Unpack(turns).numel();
    if (n > 0x3FFFFFFF) bad("'turns' is too long");
    r.rot_dim = (uint32_t)(2 * n);
    r.layout = (uint32_t)PyLong_AsLong(layout);
    r.magnitude = (float)PyFloat_AsDouble(magnitude);
    r.inverse = PyObject_IsTrue(inverse) ? 1u : 0u;
    return r;
}

void* stream_of(PyObject* o) { return c10::cuda::getCurrentCUDAStream(THPVariable_Unpack(o).device().index()).stream(); }

void* scratch(PyObject* o) {
    const at::Tensor& t = tensor(o, "scratch");
    if (!t.is_contiguous() || t.nbytes() < XP_SERVING_SCRATCH_BYTES)
        bad("'scratch' must be contiguous and of " + std::to_string(XP_SERVING_SCRATCH_BYTES) + " bytes (new_scratch)");
    return t.data_ptr();
}

float* lse_of(PyObject* o, const xp_rows& q) {
    if (o == Py_None) return nullptr;
    return static_cast<float*>(flat(o, "lse", at::kFloat, (int64_t)q.tokens * q.heads));
}

uint32_t count(PyObject* o, const char* name) {
    const long v = PyLong_AsLong(o);
    if (v < 0 || v > 0x7FFFFFFF) {
        PyErr_Clear();
        bad(std::string("'") + name + "' must be a whole number, not negative");
    }
    return (uint32_t)v;
}

PyObject* failed(int status, const std::string& message) {
    return Py_BuildValue("(is)", status, message.c_str());
}

// Runs f, which returns an xp_status, and turns what goes wrong into a result.
template <class F> PyObject* guarded(Py_ssize_t got, Py_ssize_t want, F f) {
    if (got != want) return failed(XP_ERR_ARITY, "expects " + std::to_string(want) + " arguments");
    try {
        const xp_status s = f();
        if (PyErr_Occurred()) return nullptr;
        if (s != XP_OK) return failed(s, xp_last_error());
        Py_RETURN_NONE;
    } catch (const Bad& b) {
        PyErr_Clear();
        return failed(XP_ERR_INVALID, b.message);
    } catch (const std::exception& e) {
        return failed(XP_ERR_INVALID, e.what());
    }
}

PyObject* py_rope_rows(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 7, [&] {
        const xp_rows out = rows(a[0], "out"), in = rows(a[1], "x");
        const xp_rotary r = rotary(a[2], a[3], a[4], a[5], a[6], in.tokens);
        return xp_rope_rows(stream_of(a[1]), &out, &in, &r);
    });
}
PyObject* py_kv_write(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 11, [&] {
        const xp_pages p = pages(a);
        const xp_rows k = rows(a[4], "k"), v = rows(a[5], "v");
        const auto* slots = static_cast<const int64_t*>(flat(a[6], "slots", at::kLong, k.tokens));
        if (a[8] == Py_None) return xp_kv_write(stream_of(a[4]), &p, &k, &v, slots, nullptr);
        const xp_rotary r = rotary(a[7], a[8], a[9], a[10], Py_False, k.tokens);
        return xp_kv_write(stream_of(a[4]), &p, &k, &v, slots, &r);
    });
}
PyObject* py_kv_read(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 7, [&] {
        const xp_pages p = pages(a);
        const xp_rows k = rows(a[4], "k"), v = rows(a[5], "v");
        return xp_kv_read(stream_of(a[4]), &p, &k, &v, static_cast<const int64_t*>(flat(a[6], "slots", at::kLong, k.tokens)));
    });
}
PyObject* py_attention_packed(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 9, [&] {
        const xp_rows out = rows(a[0], "out"), q = rows(a[1], "q"), k = rows(a[2], "k"), v = rows(a[3], "v");
        const auto* starts = static_cast<const int32_t*>(flat(a[4], "starts", at::kInt, -1));
        const int64_t batch = THPVariable_Unpack(a[4]).numel() - 1;
        if (batch < 0 || batch > 0x7FFFFFFF) bad("'starts' must have one value more than there are sequences");
        return xp_attention_packed(stream_of(a[1]), &out, &q, &k, &v, starts, (uint32_t)batch, count(a[6], "window"),
                                   (float)PyFloat_AsDouble(a[7]), lse_of(a[8], q), scratch(a[5]));
    });
}
PyObject* py_attention_paged(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 14, [&] {
        const xp_rows out = rows(a[0], "out"), q = rows(a[1], "q");
        const xp_pages p = pages(a + 2);
        const auto* lens = static_cast<const int32_t*>(flat(a[7], "kv_lens", at::kInt, -1));
        const int64_t batch = THPVariable_Unpack(a[7]).numel();
        const at::Tensor& t = tensor(a[6], "table");
        if (t.dim() != 2 || t.size(0) != batch || batch > 0x7FFFFFFF || t.size(1) > 0x7FFFFFFF)
            bad("'table' must be [sequences, pages of a sequence]");
        const auto* table = static_cast<const int32_t*>(flat(a[6], "table", at::kInt, -1));
        const auto* starts = static_cast<const int32_t*>(flat(a[8], "starts", at::kInt, batch + 1));
        return xp_attention_paged(stream_of(a[1]), &out, &q, &p, table, (uint32_t)t.size(1), lens, starts, (uint32_t)batch,
                                  count(a[9], "q_most"), count(a[11], "window"), (float)PyFloat_AsDouble(a[12]),
                                  lse_of(a[13], q), scratch(a[10]));
    });
}

#define METHOD(f) {#f, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_##f)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {METHOD(rope_rows), METHOD(kv_write), METHOD(kv_read), METHOD(attention_packed),
                         METHOD(attention_paged), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_serving", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__serving(void) { return PyModule_Create(&module); }
