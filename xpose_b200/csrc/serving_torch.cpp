// Torch tensors to the serving entry points of include/xp_cuda.h: the checks
// of xpose_b200/serving.py in C++, because a decode step's kernels take less
// time than the same checks in Python. Every function returns None, or
// (status, message) for the caller to raise. The tensors of a call are all on
// one device, which is the current one while the call is enqueued.
#include <Python.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <string>

#include "../../include/xp_cuda.h"

namespace {

struct Bad {
    std::string message;
};
[[noreturn]] void bad(const std::string& m) { throw Bad{m}; }

// The device of one call: that of the first tensor looked at.
struct Device {
    int index = -1;
    c10::cuda::OptionalCUDAGuard guard;
    // torch's current stream there, for which the device is made the current one
    void* stream() {
        guard.set_index((c10::DeviceIndex)index);
        return c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)index).stream();
    }
};

const at::Tensor& tensor(Device& d, PyObject* o, const char* name) {
    if (!THPVariable_Check(o)) bad(std::string("'") + name + "' must be a tensor");
    const at::Tensor& t = THPVariable_Unpack(o);
    if (!t.is_cuda()) bad(std::string("'") + name + "' must be a CUDA tensor");
    const int index = t.device().index();
    if (d.index < 0) d.index = index;
    if (index != d.index)
        bad(std::string("'") + name + "' is on device " + std::to_string(index) + ", others of the call on device " +
            std::to_string(d.index));
    return t;
}

xp_rows rows(Device& d, PyObject* o, const char* name) {
    const at::Tensor& t = tensor(d, o, name);
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
void* flat(Device& d, PyObject* o, const char* name, at::ScalarType type, int64_t n) {
    const at::Tensor& t = tensor(d, o, name);
    if (t.scalar_type() != type || !t.is_contiguous() || (n >= 0 && t.numel() != n))
        bad(std::string("'") + name + "' must be contiguous, of type " + c10::toString(type) +
            (n >= 0 ? " and of " + std::to_string(n) + " values" : std::string()));
    return t.data_ptr();
}

float number(PyObject* o, const char* name) {
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) bad(std::string("'") + name + "' must be a number");
    return (float)v;
}

xp_pages pages(Device& d, PyObject* const* a) {  // k, v, k_scale, v_scale
    const at::Tensor &k = tensor(d, a[0], "k_pages"), &v = tensor(d, a[1], "v_pages");
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
        p.k_scale = static_cast<float*>(flat(d, a[2], "k_scale", at::kFloat, n));
        p.v_scale = static_cast<float*>(flat(d, a[3], "v_scale", at::kFloat, n));
    }
    return p;
}

xp_rotary rotary(Device& d, PyObject* positions, PyObject* turns, PyObject* layout, PyObject* magnitude,
                 PyObject* inverse, uint32_t tokens) {
    xp_rotary r{};
    r.turns = static_cast<const uint64_t*>(flat(d, turns, "turns", at::kLong, -1));
    r.positions = static_cast<const int32_t*>(flat(d, positions, "positions", at::kInt, tokens));
    const int64_t n = THPVariable_Unpack(turns).numel();
    if (n > 0x3FFFFFFF) bad("'turns' is too long");
    r.rot_dim = (uint32_t)(2 * n);
    r.layout = (uint32_t)PyLong_AsLong(layout);
    r.magnitude = number(magnitude, "magnitude");
    const int back = PyObject_IsTrue(inverse);
    if (back < 0) bad("'inverse' must be true or false");
    r.inverse = (uint32_t)back;
    return r;
}

void* scratch(Device& d, PyObject* o) {
    const at::Tensor& t = tensor(d, o, "scratch");
    if (!t.is_contiguous() || t.nbytes() < XP_SERVING_SCRATCH_BYTES)
        bad("'scratch' must be contiguous and of " + std::to_string(XP_SERVING_SCRATCH_BYTES) + " bytes (new_scratch)");
    return t.data_ptr();
}

float* lse_of(Device& d, PyObject* o, const xp_rows& q) {
    if (o == Py_None) return nullptr;
    return static_cast<float*>(flat(d, o, "lse", at::kFloat, (int64_t)q.tokens * q.heads));
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

// Runs f(device), which returns an xp_status, and turns what goes wrong into a result.
template <class F> PyObject* guarded(Py_ssize_t got, Py_ssize_t want, F f) {
    if (got != want) return failed(XP_ERR_ARITY, "expects " + std::to_string(want) + " arguments");
    try {
        Device d;
        const xp_status s = f(d);
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
    return guarded(n, 7, [&](Device& d) {
        const xp_rows out = rows(d, a[0], "out"), in = rows(d, a[1], "x");
        const xp_rotary r = rotary(d, a[2], a[3], a[4], a[5], a[6], in.tokens);
        return xp_rope_rows(d.stream(), &out, &in, &r);
    });
}
PyObject* py_kv_write(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 11, [&](Device& d) {
        const xp_pages p = pages(d, a);
        const xp_rows k = rows(d, a[4], "k"), v = rows(d, a[5], "v");
        const auto* slots = static_cast<const int64_t*>(flat(d, a[6], "slots", at::kLong, k.tokens));
        if (a[8] == Py_None) return xp_kv_write(d.stream(), &p, &k, &v, slots, nullptr);
        const xp_rotary r = rotary(d, a[7], a[8], a[9], a[10], Py_False, k.tokens);
        return xp_kv_write(d.stream(), &p, &k, &v, slots, &r);
    });
}
PyObject* py_kv_read(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 7, [&](Device& d) {
        const xp_pages p = pages(d, a);
        const xp_rows k = rows(d, a[4], "k"), v = rows(d, a[5], "v");
        return xp_kv_read(d.stream(), &p, &k, &v, static_cast<const int64_t*>(flat(d, a[6], "slots", at::kLong, k.tokens)));
    });
}
PyObject* py_attention_packed(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 9, [&](Device& d) {
        const xp_rows out = rows(d, a[0], "out"), q = rows(d, a[1], "q"), k = rows(d, a[2], "k"), v = rows(d, a[3], "v");
        const auto* starts = static_cast<const int32_t*>(flat(d, a[4], "starts", at::kInt, -1));
        const int64_t batch = THPVariable_Unpack(a[4]).numel() - 1;
        if (batch < 0 || batch > 0x7FFFFFFF) bad("'starts' must have one value more than there are sequences");
        float* const lse = lse_of(d, a[8], q);
        void* const work = scratch(d, a[5]);
        const uint32_t window = count(a[6], "window");
        const float scale = number(a[7], "scale");
        return xp_attention_packed(d.stream(), &out, &q, &k, &v, starts, (uint32_t)batch, window, scale, lse, work);
    });
}
PyObject* py_attention_paged(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 14, [&](Device& d) {
        const xp_rows out = rows(d, a[0], "out"), q = rows(d, a[1], "q");
        const xp_pages p = pages(d, a + 2);
        const auto* lens = static_cast<const int32_t*>(flat(d, a[7], "kv_lens", at::kInt, -1));
        const int64_t batch = THPVariable_Unpack(a[7]).numel();
        const at::Tensor& t = tensor(d, a[6], "table");
        if (t.dim() != 2 || t.size(0) != batch || batch > 0x7FFFFFFF || t.size(1) > 0x7FFFFFFF)
            bad("'table' must be [sequences, pages of a sequence]");
        const auto* table = static_cast<const int32_t*>(flat(d, a[6], "table", at::kInt, -1));
        const auto* starts = static_cast<const int32_t*>(flat(d, a[8], "starts", at::kInt, batch + 1));
        float* const lse = lse_of(d, a[13], q);
        void* const work = scratch(d, a[10]);
        const uint32_t most = count(a[9], "q_most"), window = count(a[11], "window");
        const float scale = number(a[12], "scale");
        return xp_attention_paged(d.stream(), &out, &q, &p, table, (uint32_t)t.size(1), lens, starts, (uint32_t)batch, most,
                                  window, scale, lse, work);
    });
}

#define METHOD(f) {#f, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_##f)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {METHOD(rope_rows), METHOD(kv_write), METHOD(kv_read), METHOD(attention_packed),
                         METHOD(attention_paged), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_serving", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__serving(void) { return PyModule_Create(&module); }
