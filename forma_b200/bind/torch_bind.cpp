// Python entry of the serving operators (attention_window, attention_prefix,
// token_logprobs, token_logprobs_grad): torch tensors to fb_tensor
// descriptors, outputs from torch's allocator, one call of the C ABI on the
// current stream.
//
// These run once per layer and token, where the host's time per call is what
// a small call costs: token_logprobs with alternatives took 43 us through
// ctypes (seven descriptors filled field by field from Python) and takes 10 us
// here, a windowed decode step 6 us.  All checks of shapes and
// types stay in the C ABI; only what concerns torch (device memory, one
// device, known dtypes) is checked here, as describe() and _device() of
// api.py do.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ops/empty.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <string>

#include "../../include/forma_b200.h"

namespace {

PyObject* g_error = nullptr;  // api.TensorError(status, detail)

struct Fail {};  // a Python exception is set

[[noreturn]] void fail(int status, const std::string& detail) {
    if (PyObject* e = PyObject_CallFunction(g_error, "is", status, detail.c_str())) {
        PyErr_SetObject(g_error, e);
        Py_DECREF(e);
    }
    throw Fail();
}

// One call's operands: their common device.
struct Call {
    c10::Device device{c10::kCPU};
    bool any = false;

    // The tensor behind `o`, or null for None.
    const at::Tensor* tensor(PyObject* o) {
        if (o == Py_None) return nullptr;
        if (!THPVariable_Check(o)) {
            PyErr_SetString(PyExc_TypeError, "expected a torch tensor");
            throw Fail();
        }
        const at::Tensor& t = THPVariable_Unpack(o);
        if (!t.is_cuda()) fail(FB_ERR_INVALID_INPUT, "tensors must be CUDA device memory (no CPU fallback)");
        if (any && t.device() != device)
            fail(FB_ERR_FOREIGN_RUNTIME, "operands on " + device.str() + " and " + t.device().str() + ": one call runs on one device");
        device = t.device();
        any = true;
        return &t;
    }
    const at::Tensor& required(PyObject* o) {
        const at::Tensor* t = tensor(o);
        if (!t) fail(FB_ERR_INVALID_INPUT, "no tensor");
        return *t;
    }
};

struct Desc {
    fb_tensor t;
    fb_tensor* p = nullptr;  // null: absent
    Desc() = default;
    explicit Desc(const at::Tensor* x) {
        if (x) fill(*x);
    }
    void fill(const at::Tensor& x) {
        switch (x.scalar_type()) {
            case at::kFloat: t.dtype = FB_F32; break;
            case at::kInt: t.dtype = FB_U32; break;
            case at::kHalf: t.dtype = FB_F16; break;
            case at::kBFloat16: t.dtype = FB_BF16; break;
            default: fail(FB_ERR_DTYPE, std::string("unsupported dtype ") + c10::toString(x.scalar_type()));
        }
        const int64_t n = x.dim();
        if (n > FB_MAX_RANK) fail(FB_ERR_INVALID_INPUT, "rank " + std::to_string(n) + " exceeds " + std::to_string(FB_MAX_RANK));
        const c10::Storage& s = x.storage();
        t.data = s.nbytes() ? const_cast<void*>(s.data()) : nullptr;
        t.storage_len = s.nbytes() / x.element_size();
        t.rank = (uint32_t)n;
        for (int64_t i = 0; i < n; ++i) {
            t.dims[i] = (uint64_t)x.size(i);
            t.strides[i] = (uint64_t)x.stride(i);
        }
        t.offset = (uint64_t)x.storage_offset();
        p = &t;
    }
};

uint64_t count_of(PyObject* o) {  // a count of keys; more than 2^63 - 1 is as good as that
    int overflow = 0;
    const long long v = PyLong_AsLongLongAndOverflow(o, &overflow);
    if (v == -1 && !overflow && PyErr_Occurred()) throw Fail();
    if (overflow > 0) return INT64_MAX;
    if (overflow < 0 || v < 0) fail(FB_ERR_INVALID_ATTENTION, "invalid attention: window and sinks count keys");
    return (uint64_t)v;
}

fb_attention_options options_of(PyObject* scale, PyObject* causal) {
    fb_attention_options o{};
    if (scale != Py_None) {
        o.has_scale = 1;
        o.scale = (float)PyFloat_AsDouble(scale);
    }
    if (causal != Py_None) {
        o.has_causal = 1;
        const long v = PyLong_AsLong(causal);
        if (!PyErr_Occurred() && (v > INT32_MAX || v < INT32_MIN)) fail(FB_ERR_INVALID_INPUT, "causal offset exceeds i32");
        o.causal = (int32_t)v;
    }
    if (PyErr_Occurred()) throw Fail();
    return o;
}

// Runs one C ABI call on the operands' device and current stream.
template <typename F>
void run(const Call& c, F call) {
    c10::cuda::CUDAGuard guard(c.device);
    void* stream = c10::cuda::getCurrentCUDAStream(c.device.index()).stream();
    int status;
    Py_BEGIN_ALLOW_THREADS
    status = call(stream);
    Py_END_ALLOW_THREADS
    if (status != FB_OK) fail(status, fb_last_error());
}

at::Tensor empty(at::IntArrayRef dims, at::ScalarType dtype, const Call& c) {
    return at::empty(dims, at::TensorOptions().dtype(dtype).device(c.device));
}

// attention's output dims: the query's with the value's depth where the batch
// axes agree, else what the plan says (broadcast batches, errors).
at::Tensor attention_out(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, fb_attention_options o, const Call& c) {
    const int64_t r = q.dim();
    if (r >= 3 && k.dim() == r && v.dim() == r && q.sizes().slice(0, r - 3) == k.sizes().slice(0, r - 3) &&
        q.sizes().slice(0, r - 3) == v.sizes().slice(0, r - 3)) {
        c10::SmallVector<int64_t, 8> dims(q.sizes().begin(), q.sizes().end());
        dims[r - 1] = v.size(r - 1);
        return empty(dims, q.scalar_type(), c);
    }
    uint64_t d[3][FB_MAX_RANK], out[FB_MAX_RANK];
    const at::Tensor* x[3] = {&q, &k, &v};
    for (int i = 0; i < 3; ++i) {
        if (x[i]->dim() > FB_MAX_RANK) fail(FB_ERR_INVALID_INPUT, "rank exceeds " + std::to_string(FB_MAX_RANK));
        for (int64_t a = 0; a < x[i]->dim(); ++a) d[i][a] = (uint64_t)x[i]->size(a);
    }
    uint32_t rank = 0;
    const int status = fb_attention_plan(d[0], (uint32_t)q.dim(), d[1], (uint32_t)k.dim(), d[2], (uint32_t)v.dim(), nullptr, 0, o,
                                         out, &rank);
    if (status != FB_OK) fail(status, fb_last_error());
    c10::SmallVector<int64_t, 8> dims(out, out + rank);
    return empty(dims, q.scalar_type(), c);
}

// C++ exceptions (torch's allocator) become Python ones.
template <typename F>
PyObject* guarded(Py_ssize_t n, Py_ssize_t want, F body) {
    if (n != want) {
        PyErr_Format(PyExc_TypeError, "expected %zd arguments, got %zd", want, n);
        return nullptr;
    }
    try {
        return body();
    } catch (const Fail&) {
        return nullptr;
    } catch (const c10::OutOfMemoryError& e) {
        PyErr_SetString(PyExc_MemoryError, e.what_without_backtrace());
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
    }
    return nullptr;
}

// (query, key, value, window, sinks, lengths, scale, causal, out)
PyObject* attention_window(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 9, [&]() -> PyObject* {
        Call c;
        const at::Tensor &q = c.required(a[0]), &k = c.required(a[1]), &v = c.required(a[2]);
        const uint64_t window = count_of(a[3]), sinks = count_of(a[4]);
        const Desc dl(c.tensor(a[5]));
        const fb_attention_options o = options_of(a[6], a[7]);
        const at::Tensor* given = c.tensor(a[8]);
        const Desc dq(&q), dk(&k), dv(&v);
        at::Tensor made;
        if (!given) made = attention_out(q, k, v, o, c);
        Desc out(given ? given : &made);
        run(c, [&](void* s) { return fb_attention_window(&dq.t, &dk.t, &dv.t, dl.p ? &dl.t : nullptr, window, sinks, o, &out.t, s); });
        return given ? Py_NewRef(a[8]) : THPVariable_Wrap(std::move(made));
    });
}

// (query, prefix_key, prefix_value, key, value, lengths, scale, causal, out)
PyObject* attention_prefix(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 9, [&]() -> PyObject* {
        Call c;
        const at::Tensor &q = c.required(a[0]), &pk = c.required(a[1]), &pv = c.required(a[2]), &k = c.required(a[3]),
                         &v = c.required(a[4]);
        const Desc dl(c.tensor(a[5]));
        const fb_attention_options o = options_of(a[6], a[7]);
        const at::Tensor* given = c.tensor(a[8]);
        const Desc dq(&q), dpk(&pk), dpv(&pv), dk(&k), dv(&v);
        at::Tensor made;
        if (!given) made = attention_out(q, k, v, o, c);
        Desc out(given ? given : &made);
        run(c, [&](void* s) {
            return fb_attention_prefix(&dq.t, &dpk.t, &dpv.t, &dk.t, &dv.t, dl.p ? &dl.t : nullptr, o, &out.t, s);
        });
        return given ? Py_NewRef(a[8]) : THPVariable_Wrap(std::move(made));
    });
}

// (logits, targets, top) -> (logprob, entropy, logsumexp, top_logprob, top_index)
PyObject* token_logprobs(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 3, [&]() -> PyObject* {
        Call c;
        const at::Tensor& x = c.required(a[0]);
        const Desc dt(c.tensor(a[1]));
        const long top = PyLong_AsLong(a[2]);
        if (PyErr_Occurred()) throw Fail();
        if (top < 0) fail(FB_ERR_INVALID_INPUT, "a negative number of alternatives");
        if (top > FB_MAX_TOP) fail(FB_ERR_INVALID_INPUT, "at most " + std::to_string(FB_MAX_TOP) + " alternatives");
        const Desc dx(&x);
        if (x.dim() == 0) fail(FB_ERR_INVALID_INPUT, "logits need rank at least one");
        c10::SmallVector<int64_t, 9> dims(x.sizes().begin(), x.sizes().end() - 1);
        at::Tensor out[5];
        Desc d[5];
        for (int i = 0; i < 5; ++i) {
            if (i == 0 && !dt.p) continue;
            if (i == 3) {
                if (!top) break;
                dims.push_back(top);
            }
            out[i] = empty(dims, i == 4 ? at::kInt : at::kFloat, c);
            d[i].fill(out[i]);
        }
        run(c, [&](void* s) {
            return fb_token_logprobs(&dx.t, dt.p ? &dt.t : nullptr, d[0].p, d[1].p, d[2].p, d[3].p, d[4].p, s);
        });
        PyObject* r = PyTuple_New(5);
        if (!r) return nullptr;
        for (int i = 0; i < 5; ++i)
            PyTuple_SET_ITEM(r, i, d[i].p ? THPVariable_Wrap(std::move(out[i])) : Py_NewRef(Py_None));
        return r;
    });
}

// (logits, targets, logsumexp, grad_logprob, entropy, grad_entropy, out)
PyObject* token_logprobs_grad(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 7, [&]() -> PyObject* {
        Call c;
        const at::Tensor& x = c.required(a[0]);
        const Desc dx(&x), dt(&c.required(a[1])), dl(&c.required(a[2])), dg(&c.required(a[3])), de(c.tensor(a[4])),
            dh(c.tensor(a[5]));
        const at::Tensor* given = c.tensor(a[6]);
        at::Tensor made;
        if (!given) made = empty(x.sizes(), x.scalar_type(), c);
        Desc out(given ? given : &made);
        run(c, [&](void* s) {
            return fb_token_logprobs_grad(&dx.t, &dt.t, &dl.t, &dg.t, de.p ? &de.t : nullptr, dh.p ? &dh.t : nullptr, &out.t, s);
        });
        return given ? Py_NewRef(a[6]) : THPVariable_Wrap(std::move(made));
    });
}

// set_error(TensorError): the exception class for non-zero statuses
PyObject* set_error(PyObject*, PyObject* cls) {
    Py_XSETREF(g_error, Py_NewRef(cls));
    Py_RETURN_NONE;
}

PyMethodDef methods[] = {
    {"attention_window", (PyCFunction)(void (*)(void))attention_window, METH_FASTCALL, nullptr},
    {"attention_prefix", (PyCFunction)(void (*)(void))attention_prefix, METH_FASTCALL, nullptr},
    {"token_logprobs", (PyCFunction)(void (*)(void))token_logprobs, METH_FASTCALL, nullptr},
    {"token_logprobs_grad", (PyCFunction)(void (*)(void))token_logprobs_grad, METH_FASTCALL, nullptr},
    {"set_error", set_error, METH_O, nullptr},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_torch_bind", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__torch_bind() { return PyModule_Create(&module); }
