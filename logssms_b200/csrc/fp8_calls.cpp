// The calls of the 8-bit operators from Python to their launchers, without a detour: what `kernels.py` checks, allocates and
// converts in a dozen microseconds per call takes two here, which is what a single token outside a captured graph waits for.
//
// Only what is plainly in order is taken: every function returns the new tensors, or None, whereupon the caller goes the
// ordinary way and says what is wrong with the arguments (or finds that all is well), or a launcher's error code.  Nothing is
// kept between calls but the addresses of the launchers and of each device's error word, which `kernels.py` hands over.
#include <Python.h>
#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

namespace {
constexpr int kDevices = 64;
int* error_words[kDevices];

typedef int (*NormFn)(const void*, long, const void*, long, const void*, long, void*, long, const float*, void*, long, float*, long,
                      long, int, int, float, float, float, float, int, void*);
typedef int (*QuantFn)(const void*, long, void*, long, float*, long, long, long, int, int, int, void*);
typedef int (*LinearFn)(const void*, long, const float*, long, long, const void*, long, const float*, long, long, const float*, void*,
                        long, int, int, int, float, int, int, int, int*, void*);
typedef int (*SwigluFn)(const void*, long, const float*, long, long, const void*, const void*, long, const float*, const float*, long,
                        long, void*, long, float*, long, long, int, int, int, float, int, int, int*, void*);
NormFn norm_fn;
QuantFn quant_fn;
LinearFn linear_fn;
SwigluFn swiglu_fn;

// the argument's tensor, or null
const at::Tensor* tensor(PyObject* o) { return THPVariable_Check(o) ? &THPVariable_Unpack(o) : nullptr; }

// [rows, width] on the current device, columns side by side
bool matrix(const at::Tensor& t, int device) {
    return t.is_cuda() && t.get_device() == device && t.dim() == 2 && t.size(1) > 0 && (t.stride(1) == 1 || t.size(1) == 1);
}
int dtype_code(const at::Tensor& t) { return t.scalar_type() == at::kFloat ? 0 : t.scalar_type() == at::kBFloat16 ? 1 : -1; }
bool vector(const at::Tensor& t, int device, int64_t n) {
    return t.is_cuda() && t.get_device() == device && t.scalar_type() == at::kFloat && t.dim() == 1 && t.size(0) == n && t.is_contiguous();
}
bool fits(int64_t n) { return n <= 0x7fffffff; }

struct Fp8 { const at::Tensor *v, *s; long pitch; };
// an 8-bit operand with a scale for each block_rows x 128 block; rows at multiples of 16 bytes
bool operand(Fp8& f, PyObject* values, PyObject* scales, int block_rows, int device) {
    f.v = tensor(values);
    f.s = tensor(scales);
    if (f.v == nullptr || f.s == nullptr || !matrix(*f.v, device) || f.v->scalar_type() != at::kFloat8_e4m3fn) return false;
    const int64_t rows = f.v->size(0), width = f.v->size(1);
    if (!f.s->is_cuda() || f.s->get_device() != device || f.s->scalar_type() != at::kFloat || f.s->dim() != 2
        || f.s->size(0) != (rows + block_rows - 1) / block_rows || f.s->size(1) != (width + 127) / 128) return false;
    f.pitch = rows > 1 ? f.v->stride(0) : (width + 15) / 16 * 16;
    return f.pitch % 16 == 0 && f.pitch >= width && ((uintptr_t)f.v->data_ptr() & 15) == 0 && fits(rows) && fits(width);
}
// whole rows of the pitch, the last one too: kernels write what fills up a row
at::Tensor values_for(int64_t rows, int64_t width, at::Device device) {
    const int64_t pitch = (width + 15) / 16 * 16;
    at::Tensor t = at::detail::empty_strided_cuda({rows, pitch}, {pitch, 1}, at::kFloat8_e4m3fn, device);
    const int64_t sizes[2] = {rows, width}, strides[2] = {pitch, 1};
    if (pitch != width) t.unsafeGetTensorImpl()->set_sizes_and_strides(at::IntArrayRef(sizes), at::IntArrayRef(strides));
    return t;
}
at::Tensor scales_for(int64_t rows, int64_t width, at::Device device, bool side_by_side) {
    const int64_t blocks = (width + 127) / 128;
    return side_by_side ? at::detail::empty_strided_cuda({rows, blocks}, {1, rows}, at::kFloat, device)
                        : at::detail::empty_strided_cuda({rows, blocks}, {blocks, 1}, at::kFloat, device);
}
PyObject* two(const at::Tensor& a, const at::Tensor& b) {
    PyObject *pa = THPVariable_Wrap(a), *pb = THPVariable_Wrap(b);
    PyObject* r = pa != nullptr && pb != nullptr ? PyTuple_Pack(2, pa, pb) : nullptr;
    Py_XDECREF(pa);
    Py_XDECREF(pb);
    return r;
}
PyObject* none() { Py_RETURN_NONE; }
bool numbers(double* to, PyObject* const* from, int n) {
    for (int i = 0; i < n; ++i) {
        to[i] = PyFloat_AsDouble(from[i]);
        if (to[i] == -1.0 && PyErr_Occurred()) { PyErr_Clear(); return false; }
    }
    return true;
}
// what Python's `if` would say of each; false where that raises (the ordinary way then raises it)
bool truths(bool* to, PyObject* const* from, int n) {
    for (int i = 0; i < n; ++i) {
        const int yes = PyObject_IsTrue(from[i]);
        if (yes < 0) { PyErr_Clear(); return false; }
        to[i] = yes != 0;
    }
    return true;
}
// no C++ exception reaches the interpreter: what throws here (an allocation that fails) goes the ordinary way and says so there
template <typename F> PyObject* guarded(F f) {
    try {
        return f();
    } catch (...) {
        PyErr_Clear();
        return none();
    }
}
void* stream_of(int device) { return (void*)c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)device).stream(); }

// (x, weight, eps, residual | None, other | None, in0, in1, out_scale, want_residual, in_place) -> (values, scales, residual | None)
PyObject* norm(PyObject*, PyObject* const* args, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        const int device = (int)c10::cuda::current_device();
        double num[4];
        bool flags[2];
        if (n != 10 || norm_fn == nullptr || !numbers(num, args + 2, 1) || !numbers(num + 1, args + 5, 3) || !truths(flags, args + 8, 2)) return none();
        const at::Tensor *x = tensor(args[0]), *w = tensor(args[1]), *res = nullptr, *other = nullptr;
        if (x == nullptr || w == nullptr || !matrix(*x, device) || dtype_code(*x) < 0) return none();
        const int64_t rows = x->size(0), width = x->size(1);
        if (!fits(rows) || !fits(width) || !vector(*w, device, width)) return none();
        for (int i = 0; i < 2; ++i) {
            if (args[3 + i] == Py_None) continue;
            const at::Tensor* t = tensor(args[3 + i]);
            if (t == nullptr || !matrix(*t, device) || t->size(0) != rows || t->size(1) != width || t->scalar_type() != x->scalar_type()) return none();
            (i == 0 ? res : other) = t;
        }
        at::Tensor fresh;
        const bool want = flags[0], in_place = flags[1];
        const at::Tensor* to = nullptr;
        if (want && res != nullptr && in_place) to = res;
        else if (want) {
            fresh = at::detail::empty_strided_cuda({rows, width}, {width, 1}, x->scalar_type(), x->device());
            to = &fresh;
        }
        const at::Tensor q = values_for(rows, width, x->device()), s = scales_for(rows, width, x->device(), true);
        const int code = norm_fn(x->data_ptr(), x->stride(0), other ? other->data_ptr() : nullptr, other ? other->stride(0) : 0,
                                 res ? res->data_ptr() : nullptr, res ? res->stride(0) : 0, to ? to->data_ptr() : nullptr,
                                 to ? to->stride(0) : 0, (const float*)w->data_ptr(), q.data_ptr(), q.stride(0), (float*)s.data_ptr(), 1,
                                 rows, (int)rows, (int)width, (float)num[0], (float)num[1], (float)num[2], (float)num[3], dtype_code(*x),
                                 stream_of(device));
        if (code != 0) return PyLong_FromLong(code);
        PyObject *pq = THPVariable_Wrap(q), *ps = THPVariable_Wrap(s), *pr;
        if (to == nullptr) { pr = Py_None; Py_INCREF(pr); }
        else if (to == res) { pr = args[3]; Py_INCREF(pr); }
        else pr = THPVariable_Wrap(fresh);
        PyObject* r = pq && ps && pr ? PyTuple_Pack(3, pq, ps, pr) : nullptr;
        Py_XDECREF(pq);
        Py_XDECREF(ps);
        Py_XDECREF(pr);
        return r;
    });
}

// (x, block_rows) -> (values, scales)
PyObject* quantize(PyObject*, PyObject* const* args, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        const int device = (int)c10::cuda::current_device();
        const at::Tensor* x = n == 2 ? tensor(args[0]) : nullptr;
        if (x == nullptr || quant_fn == nullptr || !matrix(*x, device) || dtype_code(*x) < 0 || !fits(x->size(1))) return none();
        const long block_rows = PyLong_AsLong(args[1]);
        const int64_t rows = x->size(0), width = x->size(1), scale_rows = block_rows == 1 ? rows : (rows + 127) / 128;
        const at::Tensor q = values_for(rows, width, x->device()), s = scales_for(scale_rows, width, x->device(), block_rows == 1);
        const int code = quant_fn(x->data_ptr(), x->stride(0), q.data_ptr(), q.stride(0), (float*)s.data_ptr(),
                                  block_rows == 1 ? 1 : (width + 127) / 128, block_rows == 1 ? rows : 1, rows, (int)width, (int)block_rows,
                                  dtype_code(*x), stream_of(device));
        return code != 0 ? PyLong_FromLong(code) : two(q, s);
    });
}

// (x values, x scales, w values, w scales, bias | None, out_scale, float32 out, settled, form) -> tensor
PyObject* linear(PyObject*, PyObject* const* args, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        const int device = (int)c10::cuda::current_device();
        Fp8 x, w;
        double out_scale;
        bool flags[2];
        if (n != 9 || linear_fn == nullptr || device >= kDevices || error_words[device] == nullptr || !numbers(&out_scale, args + 5, 1)
            || !truths(flags, args + 6, 2)
            || !operand(x, args[0], args[1], 1, device) || !operand(w, args[2], args[3], 128, device) || x.v->size(1) != w.v->size(1)) return none();
        const int64_t M = x.v->size(0), N = w.v->size(0), K = x.v->size(1);
        const at::Tensor* bias = nullptr;
        if (args[4] != Py_None && ((bias = tensor(args[4])) == nullptr || !vector(*bias, device, N))) return none();
        const bool f32 = flags[0];
        const at::Tensor out = at::detail::empty_strided_cuda({M, N}, {N, 1}, f32 ? at::kFloat : at::kBFloat16, x.v->device());
        const int code = linear_fn(x.v->data_ptr(), x.pitch, (const float*)x.s->data_ptr(), x.s->stride(0), x.s->stride(1), w.v->data_ptr(),
                                   w.pitch, (const float*)w.s->data_ptr(), w.s->stride(0), w.s->stride(1),
                                   bias ? (const float*)bias->data_ptr() : nullptr, out.data_ptr(), N, (int)M, (int)N, (int)K,
                                   (float)out_scale, f32, flags[1], (int)PyLong_AsLong(args[8]), error_words[device], stream_of(device));
        return code != 0 ? PyLong_FromLong(code) : THPVariable_Wrap(out);
    });
}

// (x values, x scales, gate values, gate scales, up values, up scales, act_scale, settled, form) -> (values, scales)
PyObject* swiglu(PyObject*, PyObject* const* args, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        const int device = (int)c10::cuda::current_device();
        Fp8 x, g, u;
        double act_scale;
        bool settled;
        if (n != 9 || swiglu_fn == nullptr || device >= kDevices || error_words[device] == nullptr || !numbers(&act_scale, args + 6, 1)
            || !truths(&settled, args + 7, 1)
            || !operand(x, args[0], args[1], 1, device) || !operand(g, args[2], args[3], 128, device)
            || !operand(u, args[4], args[5], 128, device) || x.v->size(1) != g.v->size(1) || g.v->sizes() != u.v->sizes()
            || g.pitch != u.pitch || g.s->strides() != u.s->strides()) return none();
        const int64_t M = x.v->size(0), N = g.v->size(0), K = x.v->size(1);
        const at::Tensor q = values_for(M, N, x.v->device()), s = scales_for(M, N, x.v->device(), true);
        const int code = swiglu_fn(x.v->data_ptr(), x.pitch, (const float*)x.s->data_ptr(), x.s->stride(0), x.s->stride(1), g.v->data_ptr(),
                                   u.v->data_ptr(), g.pitch, (const float*)g.s->data_ptr(), (const float*)u.s->data_ptr(), g.s->stride(0),
                                   g.s->stride(1), q.data_ptr(), q.stride(0), (float*)s.data_ptr(), 1, M, (int)M, (int)N, (int)K,
                                   (float)act_scale, settled, (int)PyLong_AsLong(args[8]), error_words[device], stream_of(device));
        return code != 0 ? PyLong_FromLong(code) : two(q, s);
    });
}

// the launchers' addresses
PyObject* launchers(PyObject*, PyObject* const* args, Py_ssize_t n) {
    if (n != 4) { PyErr_SetString(PyExc_TypeError, "four addresses"); return nullptr; }
    norm_fn = (NormFn)PyLong_AsVoidPtr(args[0]);
    quant_fn = (QuantFn)PyLong_AsVoidPtr(args[1]);
    linear_fn = (LinearFn)PyLong_AsVoidPtr(args[2]);
    swiglu_fn = (SwigluFn)PyLong_AsVoidPtr(args[3]);
    return none();
}
// (device index, address of its error word)
PyObject* error_word(PyObject*, PyObject* const* args, Py_ssize_t n) {
    const long device = n == 2 ? PyLong_AsLong(args[0]) : -1;
    if (device < 0 || device >= kDevices) { PyErr_SetString(PyExc_ValueError, "a device index and an address"); return nullptr; }
    error_words[device] = (int*)PyLong_AsVoidPtr(args[1]);
    return none();
}

PyMethodDef methods[] = {
    {"norm", (PyCFunction)(void*)norm, METH_FASTCALL, nullptr},         {"quantize", (PyCFunction)(void*)quantize, METH_FASTCALL, nullptr},
    {"linear", (PyCFunction)(void*)linear, METH_FASTCALL, nullptr},     {"swiglu", (PyCFunction)(void*)swiglu, METH_FASTCALL, nullptr},
    {"launchers", (PyCFunction)(void*)launchers, METH_FASTCALL, nullptr}, {"error_word", (PyCFunction)(void*)error_word, METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "fp8_calls", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};
}  // namespace

PyMODINIT_FUNC PyInit_fp8_calls(void) { return PyModule_Create(&module); }
