// The calls of some operators from Python to their launchers, without a detour: the 8-bit operators and the serving operators
// (attention over a shared prefix, adapters, rules on logits).  What `kernels.py` checks, allocates and converts in a dozen
// microseconds or two per call takes a few here, which is what a single token outside a captured graph waits for.
//
// Only what is plainly in order is taken: every function returns the new tensors, or None, whereupon the caller goes the ordinary
// way and says what is wrong with the arguments (or finds that all is well), or a launcher's error code.  Nothing is kept between
// calls but the addresses of the launchers and of each device's error word, which `kernels.py` hands over.
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

// ------------------------------------------------------------ serving operators
namespace serving {
typedef int (*SplitsFn)(const void*, long, const void*, const void*, long, int, int, int, int, int, int, long, long, int);
typedef int (*AttentionFn)(const void*, long, const void*, const void*, void*, const int*, long, int, int, const int*, const int*, const int*,
                           const int*, int, float*, float*, long, int, int, int, int, int, int, int, long, long, float, int*, int, void*);
typedef int (*AdaptersFn)(const void*, long, const void*, long, const void*, long, long, const void*, long, long, const int*, const float*,
                          const int*, void*, long, void*, int*, long, int, int, int, int, int, int*, void*);
typedef int (*ScratchFn)(const void*, long, const void*, long, const void*, long, long, const void*, long, long, const void*, long, long, int, int, int, int,
                         int);
typedef int (*RulesFn)(const float*, long, float*, long, int, int, const int*, long, int, int, const int*, const int*, const int*, const float*,
                       const float*, const float*, const int*, const int*, const float*, int, const int*, long, int, const int*, void*);
SplitsFn splits_fn;
AttentionFn attention_fn;
AdaptersFn adapters_fn;
ScratchFn scratch_fn;
RulesFn rules_fn;


// the argument's tensor on the current device, or null
const at::Tensor* tensor(PyObject* o, int device) {
    if (!THPVariable_Check(o)) return nullptr;
    const at::Tensor& t = THPVariable_Unpack(o);
    return t.is_cuda() && t.get_device() == device ? &t : nullptr;
}
int dtype_code(const at::Tensor& t) { return t.scalar_type() == at::kFloat ? 0 : t.scalar_type() == at::kBFloat16 ? 1 : -1; }
constexpr int64_t kFits = 0x3fffffff;
// [rows, columns], columns side by side, rows that do not overlap
bool matrix(const at::Tensor& t) {
    return t.dim() == 2 && t.size(0) > 0 && t.size(1) > 0 && t.size(0) <= kFits && t.size(1) <= kFits && t.stride(1) == 1 && t.stride(0) >= t.size(1);
}
bool ints(const at::Tensor* t, int64_t n) { return t != nullptr && t->scalar_type() == at::kInt && t->dim() == 1 && t->size(0) == n && t->is_contiguous(); }
bool floats(const at::Tensor* t, int64_t n) { return t != nullptr && t->scalar_type() == at::kFloat && t->dim() == 1 && t->size(0) == n && t->is_contiguous(); }
template <typename T> const T* data(const at::Tensor* t) { return t == nullptr ? nullptr : (const T*)t->data_ptr(); }
bool number(double* to, PyObject* from) {
    *to = PyFloat_AsDouble(from);
    if (*to == -1.0 && PyErr_Occurred()) { PyErr_Clear(); return false; }
    return true;
}
bool whole(long* to, PyObject* from) {
    if (!PyLong_CheckExact(from)) return false;
    *to = PyLong_AsLong(from);
    if (*to == -1 && PyErr_Occurred()) { PyErr_Clear(); return false; }
    return true;
}

// (q, k_cache, v_cache, block_table, token_req, positions, group_start, prefix_lens, scale, max_prefix, max_context) -> out
PyObject* attention(PyObject*, PyObject* const* args, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        const int device = (int)c10::cuda::current_device();
        if (n != 11 || attention_fn == nullptr || device >= kDevices || error_words[device] == nullptr) return none();
        const at::Tensor* t[8];
        for (int i = 0; i < 8; ++i)
            if ((t[i] = tensor(args[i], device)) == nullptr) return none();
        double scale;
        long max_prefix, max_context;
        if (!number(&scale, args[8]) || !whole(&max_prefix, args[9]) || !whole(&max_context, args[10])) return none();
        const at::Tensor &q = *t[0], &k = *t[1], &v = *t[2], &bt = *t[3];
        if (!((float)scale > 0.f && (float)scale < INFINITY) || (((uintptr_t)k.data_ptr() | (uintptr_t)v.data_ptr()) & 15) != 0) return none();
        if (q.dim() != 3 || k.dim() != 4 || dtype_code(q) < 0 || k.scalar_type() != q.scalar_type() || v.scalar_type() != q.scalar_type()) return none();
        const int64_t tokens = q.size(0), Hq = q.size(1), hd = q.size(2), pages = k.size(0), page = k.size(1), Hkv = k.size(2), groups = t[7]->numel();
        if (tokens < 1 || groups < 1 || hd < 8 || hd > 256 || hd % 8 != 0 || Hkv < 1 || Hq < 1 || Hq % Hkv != 0 || pages < 1 || page < 1 || tokens > kFits || Hq > 65535
            || page > kFits || groups > kFits || q.stride(2) != 1 || (Hq > 1 && q.stride(1) != hd) || k.size(3) != hd || !k.is_contiguous() || !v.is_contiguous() || v.sizes() != k.sizes()
            || !matrix(bt) || bt.scalar_type() != at::kInt || !ints(t[4], tokens) || !ints(t[5], tokens) || !ints(t[6], groups + 1) || !ints(t[7], groups)) return none();
        const int code = dtype_code(q);
        const int splits = splits_fn(q.data_ptr(), q.stride(0), k.data_ptr(), v.data_ptr(), pages, (int)tokens, (int)Hq, (int)Hkv, (int)hd, (int)page,
                                     (int)groups, max_prefix, max_context - max_prefix, code);
        const int sp = splits >> 16, so = splits & 0xffff;
        const int64_t rows = tokens * Hq * (sp + so);
        const at::Tensor out = at::detail::empty_strided_cuda({tokens, Hq, hd}, {Hq * hd, hd, 1}, q.scalar_type(), q.device());
        const at::Tensor parts = at::detail::empty_strided_cuda({rows * (hd + 2)}, {1}, at::kFloat, q.device());
        float* part_o = (float*)parts.data_ptr();
        const int rc = attention_fn(q.data_ptr(), q.stride(0), k.data_ptr(), v.data_ptr(), out.data_ptr(), (const int*)bt.data_ptr(), bt.stride(0),
                                    (int)bt.size(1), (int)bt.size(0), data<int>(t[4]), data<int>(t[5]), data<int>(t[6]), data<int>(t[7]), (int)groups,
                                    part_o, part_o + rows * hd, pages, (int)tokens, (int)Hq, (int)Hkv, (int)hd, (int)page, sp, so, max_prefix, max_context - max_prefix,
                                    (float)scale, error_words[device], code, stream_of(device));
        return rc != 0 ? PyLong_FromLong(rc) : THPVariable_Wrap(out);
    });
}

// (y, x, a, b, index, scales | None, ranks | None) -> (out, kernels launched)
PyObject* adapters(PyObject*, PyObject* const* args, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        const int device = (int)c10::cuda::current_device();
        if (n != 7 || adapters_fn == nullptr || device >= kDevices || error_words[device] == nullptr) return none();
        const at::Tensor *y = tensor(args[0], device), *x = tensor(args[1], device), *a = tensor(args[2], device), *b = tensor(args[3], device);
        const at::Tensor *index = tensor(args[4], device), *scales = nullptr, *ranks = nullptr;
        if (y == nullptr || x == nullptr || a == nullptr || b == nullptr || !matrix(*y) || !matrix(*x) || a->dim() != 3 || b->dim() != 3) return none();
        const int64_t rows = y->size(0), features = y->size(1), width = x->size(1), count = a->size(0), rank = a->size(1);
        if (x->size(0) != rows || a->size(2) != width || b->size(0) != count || b->size(1) != features || b->size(2) != rank || count < 1 || rank < 1
            || count > kFits || rank > kFits || a->stride(2) != 1 || b->stride(2) != 1 || dtype_code(*y) < 0 || x->scalar_type() != y->scalar_type()
            || a->scalar_type() != y->scalar_type() || b->scalar_type() != y->scalar_type() || !ints(index, rows)) return none();
        if (args[5] != Py_None && !floats(scales = tensor(args[5], device), count)) return none();
        if (args[6] != Py_None && !ints(ranks = tensor(args[6], device), count)) return none();
        const int code = dtype_code(*y);
        const at::Tensor out = at::detail::empty_strided_cuda({rows, features}, {features, 1}, y->scalar_type(), y->device());
        at::Tensor scratch;
        const int64_t pieces = scratch_fn(y->data_ptr(), y->stride(0), x->data_ptr(), x->stride(0), a->data_ptr(), a->stride(0), a->stride(1), b->data_ptr(),
                                          b->stride(0), b->stride(1), out.data_ptr(), features, rows, (int)width, (int)features, (int)rank, (int)count, code);
        if (pieces > 0) scratch = at::detail::empty_strided_cuda({64 * pieces}, {1}, at::kInt, y->device());
        int launches = 0;
        const int rc = adapters_fn(y->data_ptr(), y->stride(0), x->data_ptr(), x->stride(0), a->data_ptr(), a->stride(0), a->stride(1), b->data_ptr(),
                                   b->stride(0), b->stride(1), data<int>(index), data<float>(scales), data<int>(ranks), out.data_ptr(), features,
                                   pieces > 0 ? scratch.data_ptr() : nullptr, error_words[device], rows, (int)width, (int)features, (int)rank, (int)count, code, &launches, stream_of(device));
        if (rc != 0) return PyLong_FromLong(rc);
        PyObject *po = THPVariable_Wrap(out), *pn = PyLong_FromLong(launches);
        PyObject* r = po != nullptr && pn != nullptr ? PyTuple_Pack(2, po, pn) : nullptr;
        Py_XDECREF(po);
        Py_XDECREF(pn);
        return r;
    });
}

// (logits, history, lengths, prompt_lengths, slots, repetition, frequency, presence, bias_start, bias_ids, bias_values, allowed,
//  allowed_row, each but the first may be None) -> edited
PyObject* rules(PyObject*, PyObject* const* args, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        const int device = (int)c10::cuda::current_device();
        if (n != 13 || rules_fn == nullptr) return none();
        const at::Tensor* t[13] = {};
        for (int i = 0; i < 13; ++i)
            if (args[i] != Py_None && (t[i] = tensor(args[i], device)) == nullptr) return none();
        const at::Tensor *logits = t[0], *history = t[1], *biases = t[8], *allowed = t[11];
        if (logits == nullptr || !matrix(*logits) || logits->scalar_type() != at::kFloat) return none();
        const int64_t rows = logits->size(0), V = logits->size(1);
        int64_t slots = 0, capacity = 0, words = 0, masks = 0, n_biases = 0;
        if (history != nullptr) {
            if (!matrix(*history) || history->scalar_type() != at::kInt || t[2] == nullptr) return none();
            slots = history->size(0);
            capacity = history->size(1);
            if (t[4] == nullptr && slots < rows) return none();
        } else {
            for (int i = 2; i < 8; ++i) if (t[i] != nullptr) return none();
        }
        for (int i : {2, 3, 4, 12}) if (t[i] != nullptr && !ints(t[i], rows)) return none();
        for (int i : {5, 6, 7}) if (t[i] != nullptr && !floats(t[i], rows)) return none();
        if (biases != nullptr) {
            if (t[9] == nullptr || !ints(biases, rows + 1)) return none();
            n_biases = t[9]->numel();
            if (n_biases > kFits || !ints(t[9], n_biases) || !floats(t[10], n_biases)) return none();
        } else if (t[9] != nullptr || t[10] != nullptr) {
            return none();
        }
        if (allowed != nullptr) {
            if (!matrix(*allowed) || allowed->scalar_type() != at::kInt) return none();
            masks = allowed->size(0);
            words = allowed->stride(0);
            if (allowed->size(1) * 32 < V || (t[12] == nullptr && masks < rows)) return none();
        } else if (t[12] != nullptr) {
            return none();
        }
        const at::Tensor out = at::detail::empty_strided_cuda({rows, V}, {V, 1}, at::kFloat, logits->device());
        const int rc = rules_fn(data<float>(logits), logits->stride(0), (float*)out.data_ptr(), V, (int)rows, (int)V, data<int>(history),
                                history != nullptr ? history->stride(0) : 0, (int)capacity, (int)slots, data<int>(t[4]), data<int>(t[2]), data<int>(t[3]),
                                data<float>(t[5]), data<float>(t[6]), data<float>(t[7]), data<int>(biases), data<int>(t[9]), data<float>(t[10]), (int)n_biases,
                                data<int>(allowed), words, (int)masks, data<int>(t[12]), stream_of(device));
        return rc != 0 ? PyLong_FromLong(rc) : THPVariable_Wrap(out);
    });
}

// the launchers' addresses, each operator's by itself: its library is not loaded for the others'
PyObject* attention_launchers(PyObject*, PyObject* const* args, Py_ssize_t n) {
    if (n != 2) { PyErr_SetString(PyExc_TypeError, "two addresses"); return nullptr; }
    splits_fn = (SplitsFn)PyLong_AsVoidPtr(args[0]);
    attention_fn = (AttentionFn)PyLong_AsVoidPtr(args[1]);
    return none();
}
PyObject* adapters_launchers(PyObject*, PyObject* const* args, Py_ssize_t n) {
    if (n != 2) { PyErr_SetString(PyExc_TypeError, "two addresses"); return nullptr; }
    scratch_fn = (ScratchFn)PyLong_AsVoidPtr(args[0]);
    adapters_fn = (AdaptersFn)PyLong_AsVoidPtr(args[1]);
    return none();
}
PyObject* rules_launchers(PyObject*, PyObject* const* args, Py_ssize_t n) {
    if (n != 1) { PyErr_SetString(PyExc_TypeError, "one address"); return nullptr; }
    rules_fn = (RulesFn)PyLong_AsVoidPtr(args[0]);
    return none();
}
}  // namespace serving

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
    {"attention", (PyCFunction)(void*)serving::attention, METH_FASTCALL, nullptr}, {"adapters", (PyCFunction)(void*)serving::adapters, METH_FASTCALL, nullptr},
    {"rules", (PyCFunction)(void*)serving::rules, METH_FASTCALL, nullptr},
    {"attention_launchers", (PyCFunction)(void*)serving::attention_launchers, METH_FASTCALL, nullptr},
    {"adapters_launchers", (PyCFunction)(void*)serving::adapters_launchers, METH_FASTCALL, nullptr},
    {"rules_launchers", (PyCFunction)(void*)serving::rules_launchers, METH_FASTCALL, nullptr},
    {"launchers", (PyCFunction)(void*)launchers, METH_FASTCALL, nullptr}, {"error_word", (PyCFunction)(void*)error_word, METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "host_calls", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};
}  // namespace

PyMODINIT_FUNC PyInit_host_calls(void) { return PyModule_Create(&module); }
