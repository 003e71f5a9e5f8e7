// The FP8 entry points for Python callers, checked and called in C++.
//
// A decode step calls these operators a few hundred times, eagerly or while it
// is being captured; in Python the checks of a call's tensors take longer than
// the launch.  Each function here makes the checks of its namesake in
// lightreason_b200/fp8.py and, where all hold, calls the C ABI (whose addresses
// fp8.py hands over from the loaded library) on the tensors' device and its
// current stream.  It returns the result; None where a check fails, for
// fp8.py to find the fault and name it; or the status of a failed call.
#include <ATen/ATen.h>
#include <c10/core/AutogradState.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include "moe_b200.h"

namespace {

decltype(&moe_rmsnorm_fp8) g_rows;
decltype(&moe_quantize_fp8_blocks) g_blocks;
decltype(&moe_linear_fp8) g_linear;
decltype(&moe_experts_fp8) g_experts;
decltype(&moe_experts_fp8_workspace_bytes) g_experts_workspace;

constexpr auto kE4M3 = at::kFloat8_e4m3fn;
constexpr int64_t kGroup = 128;

int64_t groups(int64_t n) { return (n + kGroup - 1) / kGroup; }

// An argument as a tensor; null if it is None or something else.
const at::Tensor *tensor(PyObject *o) { return THPVariable_Check(o) ? &THPVariable_Unpack(o) : nullptr; }

// No gradient to be tracked and no forward-mode tangent to be carried on.
bool plain(const at::Tensor &t) {
    if (t.requires_grad() && c10::GradMode::is_enabled()) return false;
    return !(c10::AutogradState::get_tls_state().get_fw_grad_mode() && t._fw_grad(0).defined());
}
// A dense plain CUDA tensor of this type and shape on device `index`.
bool fits(const at::Tensor *t, at::ScalarType type, at::IntArrayRef shape, int index) {
    return t && t->scalar_type() == type && t->is_cuda() && t->get_device() == index && t->sizes() == shape &&
           t->is_contiguous() && plain(*t);
}
// BF16 rows [T, H], dense within a row.
bool fits_rows(const at::Tensor *t, int64_t *stride) {
    if (!t || t->scalar_type() != at::kBFloat16 || !t->is_cuda() || t->dim() != 2 || !plain(*t))
        return false;
    const int64_t tokens = t->size(0), hidden = t->size(1);
    if (hidden < 1 || (hidden > 1 && t->stride(1) != 1) || (tokens > 1 && t->stride(0) < hidden)) return false;
    *stride = tokens > 1 ? t->stride(0) : hidden;
    return true;
}
bool small(int64_t n) { return n >= 0 && n < (1ll << 31); }

at::Tensor make(at::IntArrayRef shape, at::ScalarType type, const at::Tensor &like) {
    return at::empty(shape, like.options().dtype(type).requires_grad(false));
}
template <class T>
T *ptr(const at::Tensor *t) {
    if (!t) return nullptr;
    void *p = t->data_ptr();
    TORCH_CHECK(p || t->numel() == 0, "the FP8 operators need tensors with storage");
    return static_cast<T *>(p);
}

// Runs f(stream) on device `index` without the interpreter's lock.  f may throw
// (a fake tensor has no storage): device and lock are
// back before the exception is turned into Python's.
template <class F>
int on(int index, F &&f) {
    struct Device {
        const c10::DeviceIndex before;
        const bool changed;
        explicit Device(int i) : before(c10::cuda::current_device()), changed(before != i) {
            if (changed) c10::cuda::set_device(static_cast<c10::DeviceIndex>(i));
        }
        ~Device() {
            if (changed) c10::cuda::MaybeSetDevice(before);
        }
    } device(index);
    struct Unlocked {
        PyThreadState *state = PyEval_SaveThread();
        ~Unlocked() { PyEval_RestoreThread(state); }
    };
    void *stream = c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(index)).stream();
    Unlocked unlocked;
    return f(stream);
}

PyObject *none() { Py_RETURN_NONE; }
PyObject *own(PyObject *given, const at::Tensor &made) {
    if (given == Py_None) return THPVariable_Wrap(made);
    Py_INCREF(given);
    return given;
}

// rows(x, weight, residual, eps, weight_offset, q, scales, normed, residual_out)
// with every output given; True
PyObject *rows(PyObject *, PyObject *const *a, Py_ssize_t n) {
    if (n != 9) return none();
    const at::Tensor *x = tensor(a[0]), *weight = tensor(a[1]), *residual = tensor(a[2]), *q = tensor(a[5]),
                     *scales = tensor(a[6]), *normed = tensor(a[7]), *total = tensor(a[8]);
    int64_t stride = 0, rstride = 0;
    if (!fits_rows(x, &stride)) return none();
    const int index = x->get_device();
    const int64_t tokens = x->size(0), hidden = x->size(1);
    if (!small(tokens) || !small(hidden)) return none();
    auto absent = [&](int i) { return a[i] == Py_None; };
    if (!(absent(1) || fits(weight, at::kBFloat16, {hidden}, index)) ||
        !(absent(2) || (fits_rows(residual, &rstride) && residual->sizes() == x->sizes() &&
                        residual->get_device() == index)) ||
        !fits(q, kE4M3, x->sizes(), index) || !fits(scales, at::kFloat, {tokens, groups(hidden)}, index) ||
        !(absent(7) || fits(normed, at::kBFloat16, x->sizes(), index)) ||
        !(absent(8) || (residual && fits(total, at::kBFloat16, x->sizes(), index))))
        return none();
    const double eps = PyFloat_AsDouble(a[3]), offset = PyFloat_AsDouble(a[4]);
    if (PyErr_Occurred()) {
        PyErr_Clear();
        return none();
    }
    const int rc = on(index, [&](void *stream) {
        return g_rows(ptr<uint16_t>(x), stride, ptr<uint16_t>(residual), rstride, ptr<uint16_t>(weight),
                      static_cast<float>(offset), static_cast<float>(eps), static_cast<int>(tokens),
                      static_cast<int>(hidden), ptr<uint8_t>(q), ptr<float>(scales), ptr<uint16_t>(normed),
                      ptr<uint16_t>(total), stream);
    });
    if (rc) return PyLong_FromLong(rc);
    Py_RETURN_TRUE;
}

// blocks(w, q or None, scales or None) -> (q, scales)
PyObject *blocks(PyObject *, PyObject *const *a, Py_ssize_t n) {
    if (n != 3) return none();
    const at::Tensor *w = tensor(a[0]), *q = tensor(a[1]), *scales = tensor(a[2]);
    if (!w || w->scalar_type() != at::kBFloat16 || !w->is_cuda() || !(w->dim() == 2 || w->dim() == 3) ||
        !w->is_contiguous() || !plain(*w))
        return none();
    const int index = w->get_device();
    const int64_t banks = w->dim() == 3 ? w->size(0) : 1, nr = w->size(-2), nc = w->size(-1);
    if (nr < 1 || nc < 1 || !small(banks) || !small(nr) || !small(nc)) return none();
    const int64_t three[3] = {banks, groups(nr), groups(nc)};
    const at::IntArrayRef shape = w->dim() == 3 ? at::IntArrayRef(three, 3) : at::IntArrayRef(three + 1, 2);
    at::Tensor made[2];
    if (a[1] == Py_None && a[2] == Py_None) {
        q = &(made[0] = make(w->sizes(), kE4M3, *w));
        scales = &(made[1] = make(shape, at::kFloat, *w));
    } else if (!fits(q, kE4M3, w->sizes(), index) || !fits(scales, at::kFloat, shape, index)) {
        return none();
    }
    const int rc = on(index, [&](void *stream) {
        return g_blocks(ptr<uint16_t>(w), static_cast<int>(banks), static_cast<int>(nr), static_cast<int>(nc),
                        ptr<uint8_t>(q), ptr<float>(scales), stream);
    });
    if (rc) return PyLong_FromLong(rc);
    return Py_BuildValue("NN", own(a[1], made[0]), own(a[2], made[1]));
}

// linear(x, x_scales, w, w_scales, out or None, out is FP32, status or None) -> out
PyObject *linear(PyObject *, PyObject *const *a, Py_ssize_t n) {
    if (n != 7) return none();
    const at::Tensor *x = tensor(a[0]), *xs = tensor(a[1]), *w = tensor(a[2]), *ws = tensor(a[3]), *out = tensor(a[4]),
                     *status = tensor(a[6]);
    if (!x || !w || x->dim() != 2 || w->dim() != 2 || !x->is_cuda()) return none();
    const int index = x->get_device();
    const int64_t tokens = x->size(0), cols = x->size(1), nr = w->size(0), g = groups(cols);
    if (!small(tokens) || !small(nr) || !small(cols) || nr < 1 || cols < 16 || cols % 16) return none();
    if (!fits(x, kE4M3, {tokens, cols}, index) || !fits(xs, at::kFloat, {tokens, g}, index) ||
        !fits(w, kE4M3, {nr, cols}, index) || !fits(ws, at::kFloat, {groups(nr), g}, index) ||
        !(a[6] == Py_None || fits(status, at::kInt, {1}, index)))
        return none();
    at::Tensor made;
    if (a[4] == Py_None) {
        const int wide = PyObject_IsTrue(a[5]);
        out = &(made = make({tokens, nr}, wide == 1 ? at::kFloat : at::kBFloat16, *x));
    } else if (!out || !(out->scalar_type() == at::kFloat || out->scalar_type() == at::kBFloat16) ||
               !fits(out, out->scalar_type(), {tokens, nr}, index)) {
        return none();
    }
    const int rc = on(index, [&](void *stream) {
        return g_linear(ptr<uint8_t>(x), ptr<float>(xs), ptr<uint8_t>(w), ptr<float>(ws), static_cast<int>(tokens),
                        static_cast<int>(nr), static_cast<int>(cols), ptr<void>(out),
                        out->scalar_type() == at::kFloat, ptr<int32_t>(status), stream);
    });
    if (rc) return PyLong_FromLong(rc);
    return own(a[4], made);
}

// experts(x, x_scales, gate_up, gate_up_scales, down, down_scales, idx, weights, out or None, status or None) -> out
PyObject *experts(PyObject *, PyObject *const *a, Py_ssize_t n) {
    if (n != 10) return none();
    const at::Tensor *x = tensor(a[0]), *xs = tensor(a[1]), *gu = tensor(a[2]), *gus = tensor(a[3]), *dn = tensor(a[4]),
                     *dns = tensor(a[5]), *idx = tensor(a[6]), *wt = tensor(a[7]), *out = tensor(a[8]),
                     *status = tensor(a[9]);
    if (!x || !gu || !dn || !idx || x->dim() != 2 || gu->dim() != 3 || dn->dim() != 3 || idx->dim() != 2 ||
        !x->is_cuda())
        return none();
    const int index = x->get_device();
    const int64_t tokens = x->size(0), hidden = x->size(1), count = gu->size(0), inner = dn->size(2), k = idx->size(1);
    if (!small(tokens) || !small(hidden) || !small(count) || !small(inner) || !small(k)) return none();
    const int64_t g = groups(hidden), gi = groups(inner);
    if (!fits(x, kE4M3, {tokens, hidden}, index) || !fits(xs, at::kFloat, {tokens, g}, index) ||
        !fits(gu, kE4M3, {count, 2 * inner, hidden}, index) ||
        !fits(gus, at::kFloat, {count, groups(2 * inner), g}, index) ||
        !fits(dn, kE4M3, {count, hidden, inner}, index) || !fits(dns, at::kFloat, {count, g, gi}, index) ||
        !fits(idx, at::kLong, {tokens, k}, index) || !fits(wt, at::kBFloat16, {tokens, k}, index) ||
        !(a[9] == Py_None || fits(status, at::kInt, {1}, index)))
        return none();
    at::Tensor made;
    if (a[8] == Py_None) out = &(made = make({tokens, hidden}, at::kBFloat16, *x));
    else if (!fits(out, at::kBFloat16, {tokens, hidden}, index)) return none();
    const size_t bytes =
        g_experts_workspace(static_cast<int>(tokens), static_cast<int>(count), static_cast<int>(k),
                            static_cast<int>(hidden), static_cast<int>(inner));
    at::Tensor ws_t;
    if (bytes) ws_t = make({static_cast<int64_t>(bytes)}, at::kByte, *x);
    const int rc = on(index, [&](void *stream) {
        return g_experts(ptr<uint8_t>(x), ptr<float>(xs), ptr<uint8_t>(gu), ptr<float>(gus), ptr<uint8_t>(dn),
                         ptr<float>(dns), ptr<int64_t>(idx), ptr<uint16_t>(wt), static_cast<int>(tokens),
                         static_cast<int>(count), static_cast<int>(k), static_cast<int>(hidden),
                         static_cast<int>(inner), ptr<uint16_t>(out), bytes ? ws_t.data_ptr() : nullptr, bytes,
                         ptr<int32_t>(status), stream);
    });
    if (rc) return PyLong_FromLong(rc);
    return own(a[8], made);
}

// A C++ exception (out of memory, a tensor without storage) becomes Python's.
template <PyObject *(*F)(PyObject *, PyObject *const *, Py_ssize_t)>
PyObject *guarded(PyObject *self, PyObject *const *a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    return F(self, a, n);
    END_HANDLE_TH_ERRORS
}

// bind(rows, blocks, linear, experts, experts_workspace): addresses in the loaded library
PyObject *bind(PyObject *, PyObject *args) {
    unsigned long long p[5];
    if (!PyArg_ParseTuple(args, "KKKKK", &p[0], &p[1], &p[2], &p[3], &p[4])) return nullptr;
    g_rows = reinterpret_cast<decltype(g_rows)>(p[0]);
    g_blocks = reinterpret_cast<decltype(g_blocks)>(p[1]);
    g_linear = reinterpret_cast<decltype(g_linear)>(p[2]);
    g_experts = reinterpret_cast<decltype(g_experts)>(p[3]);
    g_experts_workspace = reinterpret_cast<decltype(g_experts_workspace)>(p[4]);
    Py_RETURN_NONE;
}

PyMethodDef methods[] = {
    {"rows", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(guarded<rows>)), METH_FASTCALL, nullptr},
    {"blocks", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(guarded<blocks>)), METH_FASTCALL, nullptr},
    {"linear", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(guarded<linear>)), METH_FASTCALL, nullptr},
    {"experts", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(guarded<experts>)), METH_FASTCALL, nullptr},
    {"bind", bind, METH_VARARGS, nullptr},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_fp8_bind", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__fp8_bind() { return PyModule_Create(&module); }
