// gradops.cpp -- nvdr_grad_norm and nvdr_grad_clip for lists of Python tensors (optim.py grad_norm, clip_grad_norm_, FusedAdam.measure_norm).
//
// The kernels of a short list take 5 us, and a network has hundreds of parameters: asking each gradient for address, length, type, device and
// layout through Python takes 0.4 us a tensor, and the call around them some 6 us -- more than the work.  Here it is 20 ns a tensor and 2 us a
// call.  A CPython extension of its own against the installed torch; the C library stays free of torch, and its entries are handed over as
// addresses (bind), so that there is one copy of it in the process.
#define PY_SSIZE_T_CLEAN
#include <torch/csrc/autograd/python_variable.h>
#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <c10/core/DeviceGuard.h>
#include <algorithm>
#include <vector>

#include "nvdr_hip.h"

static decltype(&nvdr_grad_norm) grad_norm_entry = nullptr;
static decltype(&nvdr_grad_clip) grad_clip_entry = nullptr;
static decltype(&nvdr_grad_norm_workspace) workspace_entry = nullptr;
static decltype(&nvdr_last_error) last_error_entry = nullptr;
static PyObject *raw_stream = nullptr;              // device index -> handle of its current stream

namespace {

struct Lists {
    std::vector<void *> data;
    std::vector<int64_t> n;
    std::vector<uint8_t> type;
    std::vector<Py_ssize_t> irregular;              // tensors whose elements do not fill their memory exactly once
    // of a call that writes to them:
    std::vector<c10::TensorImpl *> written;         // (until Python code or another thread can run)
    std::vector<c10::Storage> held;                 // their memory: another thread may drop a parameter's gradient during the call
    int device = -1;
    int64_t count() const { return (int64_t)n.size(); }
};

// The gradients in `seq`, a list: tensors, or parameters whose gradients are meant (None is left out).  writes: what the call needs that writes to
// them (references to the memory, not to each tensor: an atomic a tensor would cost a list of 400 views 3 us).  false: an exception is set.
bool collect(PyObject *seq, bool grads, bool writes, Lists &l)
{
    if (!PyList_Check(seq)) {
        PyErr_SetString(PyExc_TypeError, "a list is expected");
        return false;
    }
    const size_t most = (size_t)PyList_GET_SIZE(seq);
    l.data.reserve(most); l.n.reserve(most); l.type.reserve(most);
    if (writes) l.written.reserve(most);
    const c10::StorageImpl *memory = nullptr;
    for (Py_ssize_t k = 0; k < PyList_GET_SIZE(seq); ++k)               // (the check of a subclass runs Python code: in front of everything else)
        if (!THPVariable_Check(PyList_GET_ITEM(seq, k))) {
            PyErr_Format(PyExc_TypeError, "gradients must be tensors (got %s)", Py_TYPE(PyList_GET_ITEM(seq, k))->tp_name);
            return false;
        }
    for (Py_ssize_t k = 0; k < PyList_GET_SIZE(seq); ++k) {
        PyObject *item = PyList_GET_ITEM(seq, k);
        const at::Tensor &own = THPVariable_Unpack(item);          // (the list is the caller's own: nobody takes the item out)
        const at::Tensor &t = grads ? own.grad() : own;
        if (!t.defined()) continue;
        int type = -1;
        switch (t.scalar_type()) {
        case at::kFloat: type = NVDR_GRAD_F32; break;
        case at::kBFloat16: type = NVDR_GRAD_BF16; break;
        case at::kHalf: type = NVDR_GRAD_F16; break;
        default: break;
        }
        if (type < 0) {
            PyObject *d = PyObject_GetAttrString(item, "dtype");
            if (d) PyErr_Format(PyExc_ValueError, "gradients must be float32, bfloat16 or float16 (got %S)", d);
            Py_XDECREF(d);
            return false;
        }
        const c10::Device device = t.device();
        if (!device.is_cuda() || (l.device >= 0 && device.index() != l.device)) {
            PyErr_SetString(PyExc_RuntimeError, "gradients must reside on one GPU; this path has no CPU fallback");
            return false;
        }
        if (t.layout() != at::kStrided) {
            PyErr_SetString(PyExc_ValueError, "gradients must be dense");
            return false;
        }
        l.device = device.index();
        if (!t.is_non_overlapping_and_dense()) l.irregular.push_back((Py_ssize_t)l.n.size());
        l.data.push_back(t.data_ptr());
        l.n.push_back(t.numel());
        l.type.push_back((uint8_t)type);
        if (writes && t.numel()) {
            c10::TensorImpl *const impl = t.unsafeGetTensorImpl();
            l.written.push_back(impl);
            const c10::Storage &storage = impl->unsafe_storage();
            if (storage.unsafeGetStorageImpl() != memory) l.held.push_back(storage);
            memory = storage.unsafeGetStorageImpl();
        }
    }
    return true;
}

// ---- which tensors share memory ------------------------------------------------------------------------------------------------------------
// The bytes of a strided tensor: `run` bytes at `at` + sum over the dims of stride * index.  Dims from the longest stride on, none with one index;
// reach[k]: bytes from the first to behind the last one of the dims from k on.
struct Bytes {
    struct Dim { int64_t stride, n; };
    int64_t at, run;
    std::vector<Dim> dims;
    std::vector<int64_t> reach;
    size_t index;
};

Bytes bytes_of(const at::Tensor &t, size_t index)              // t has elements
{
    Bytes b;
    const int64_t size = (int64_t)t.element_size();
    b.at = (int64_t)(uintptr_t)t.data_ptr();
    b.run = size;
    b.index = index;
    for (int64_t d = 0; d < t.dim(); ++d)
        if (t.size(d) != 1) b.dims.push_back({t.stride(d) * size, t.size(d)});
    std::sort(b.dims.begin(), b.dims.end(), [](const Bytes::Dim &x, const Bytes::Dim &y) { return x.stride < y.stride; });
    std::vector<Bytes::Dim> kept;
    for (const Bytes::Dim &d : b.dims) {                           // dims that continue the run or one another are one
        if (kept.empty() && d.stride == b.run) b.run *= d.n;
        else if (!kept.empty() && d.stride == kept.back().stride * kept.back().n) kept.back().n *= d.n;
        else kept.push_back(d);
    }
    b.dims.assign(kept.rbegin(), kept.rend());
    b.reach.assign(b.dims.size() + 1, b.run);
    for (size_t k = b.dims.size(); k-- > 0;) b.reach[k] = b.reach[k + 1] + (b.dims[k].n - 1) * b.dims[k].stride;
    return b;
}

int64_t floor_div(int64_t a, int64_t b) { return a / b - (a % b < 0 ? 1 : 0); }       // b > 0

// Have the dims of a from ka on, placed at pa, and those of b from kb on, placed at pb, a byte in common?  Exact: the longer stride is taken apart,
// index by index where the other reaches, and of two equal strides only the difference of their indices counts, of which one or two are
// in reach for views that interleave.  Strides that fit one another badly can take many steps: after `steps` of them the answer is yes.
bool meet(const Bytes &a, size_t ka, int64_t pa, const Bytes &b, size_t kb, int64_t pb, int &steps)
{
    if (--steps < 0) return true;
    if (pa + a.reach[ka] <= pb || pb + b.reach[kb] <= pa) return false;
    const bool last_a = ka == a.dims.size(), last_b = kb == b.dims.size();
    if (last_a && last_b) return true;
    if (!last_a && !last_b && a.dims[ka].stride == b.dims[kb].stride) {
        const int64_t s = a.dims[ka].stride;
        const int64_t lo = std::max(1 - a.dims[ka].n, floor_div(pa - pb - b.reach[kb + 1], s) + 1), hi = std::min(b.dims[kb].n - 1, floor_div(pa + a.reach[ka + 1] - pb - 1, s));
        for (int64_t d = lo; d <= hi; ++d)
            if (meet(a, ka + 1, pa, b, kb + 1, pb + s * d, steps)) return true;
        return false;
    }
    if (last_a || (!last_b && b.dims[kb].stride > a.dims[ka].stride)) return meet(b, kb, pb, a, ka, pa, steps);
    const int64_t s = a.dims[ka].stride;
    const int64_t lo = std::max<int64_t>(0, floor_div(pb - pa - a.reach[ka + 1], s) + 1), hi = std::min(a.dims[ka].n - 1, floor_div(pb + b.reach[kb] - pa - 1, s));
    for (int64_t i = lo; i <= hi; ++i)
        if (meet(a, ka + 1, pa + s * i, b, kb, pb, steps)) return true;
    return false;
}

bool meets_itself(const Bytes &a, int &steps)
{
    for (size_t k = a.dims.size(); k-- > 0;) {
        const int64_t s = a.dims[k].stride;
        if (s == 0) return true;
        for (int64_t d = 1; d < a.dims[k].n && d * s < a.reach[k + 1]; ++d)
            if (meet(a, k + 1, 0, a, k + 1, d * s, steps)) return true;
    }
    return false;
}

// two tensors that share memory, or one whose own elements do (then *first == *second); false: none
bool shared(const std::vector<at::Tensor> &tensors, size_t *first, size_t *second)
{
    constexpr int STEPS = 1 << 14;
    std::vector<Bytes> all;
    all.reserve(tensors.size());
    for (size_t k = 0; k < tensors.size(); ++k) {
        if (tensors[k].numel() == 0) continue;
        all.push_back(bytes_of(tensors[k], k));
        int steps = STEPS;
        if (meets_itself(all.back(), steps)) { *first = *second = k; return true; }
    }
    std::sort(all.begin(), all.end(), [](const Bytes &x, const Bytes &y) { return x.at < y.at; });
    for (size_t i = 0; i < all.size(); ++i)
        for (size_t j = i + 1; j < all.size() && all[j].at < all[i].at + all[i].reach[0]; ++j) {
            int steps = STEPS;
            if (meet(all[i], 0, all[i].at, all[j], 0, all[j].at, steps)) {
                *first = std::min(all[i].index, all[j].index);
                *second = std::max(all[i].index, all[j].index);
                return true;
            }
        }
    return false;
}

PyObject *irregular_list(const Lists &l)
{
    PyObject *r = PyList_New((Py_ssize_t)l.irregular.size());
    for (size_t i = 0; r && i < l.irregular.size(); ++i) {
        PyObject *v = PyLong_FromSsize_t(l.irregular[i]);
        if (!v) { Py_DECREF(r); return nullptr; }
        PyList_SET_ITEM(r, (Py_ssize_t)i, v);
    }
    return r;
}

bool current_stream(int device, void **stream)
{
    PyObject *i = PyLong_FromLong(device), *h = i ? PyObject_CallFunctionObjArgs(raw_stream, i, nullptr) : nullptr;
    *stream = h ? PyLong_AsVoidPtr(h) : nullptr;
    Py_XDECREF(i);
    Py_XDECREF(h);
    return !PyErr_Occurred();
}

at::Tensor empty(at::IntArrayRef size, at::ScalarType type, int device)
{
    return at::empty(size, at::TensorOptions().dtype(type).device(at::Device(at::kCUDA, (at::DeviceIndex)device)));
}

PyObject *failed(const char *what, int rc)
{
    const char *why = last_error_entry();
    return PyErr_Format(PyExc_RuntimeError, "%s failed (code %d): %s", what, rc, why ? why : "?");
}

// no C++ exception passes into the interpreter
template <class F>
PyObject *guarded(F f)
{
    try {
        return f();
    } catch (const std::exception &e) {
        if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, e.what());
    } catch (...) {
        if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, "reading the gradients failed");
    }
    return nullptr;
}

}  // namespace

// norm(tensors, scales, norm_type, max_norm, out, work): a new 0-d tensor, or into `out` (norm, factor) with the workspace `work`; None for no
// tensors; the positions of irregular ones as a list (then nothing was done).  scales: fp32 bytes or None
static PyObject *norm(PyObject *, PyObject *args)
{
    PyObject *seq, *scales, *out, *work;
    int code;
    double max_norm;
    if (!PyArg_ParseTuple(args, "OOidOO", &seq, &scales, &code, &max_norm, &out, &work)) return nullptr;
    return guarded([&]() -> PyObject * {
        Lists l;
        if (!collect(seq, false, false, l)) return nullptr;
        if (!l.irregular.empty()) return irregular_list(l);
        if (out == Py_None && l.device < 0) Py_RETURN_NONE;
        if (scales != Py_None && (!PyBytes_Check(scales) || PyBytes_GET_SIZE(scales) != 4 * (Py_ssize_t)l.count())) return PyErr_Format(PyExc_ValueError, "a scale for each tensor is expected");
        at::Tensor result, room;
        if (out != Py_None) {
            result = THPVariable_Unpack(out);
            room = THPVariable_Unpack(work);
            if (l.device >= 0 && l.device != result.get_device()) return PyErr_Format(PyExc_RuntimeError, "gradients must reside on one GPU; this path has no CPU fallback");
            l.device = (int)result.get_device();
        }
        const c10::DeviceGuard device(at::Device(at::kCUDA, (at::DeviceIndex)l.device));
        void *stream;
        if (!current_stream(l.device, &stream)) return nullptr;
        if (out == Py_None) {
            result = empty({}, at::kFloat, l.device);
            room = empty({workspace_entry(l.n.data(), l.type.data(), l.count(), 0)}, at::kDouble, l.device);
        }
        float *at = (float *)result.data_ptr();
        int rc;
        const float *s = scales == Py_None ? nullptr : (const float *)PyBytes_AS_STRING(scales);
        Py_BEGIN_ALLOW_THREADS
        rc = grad_norm_entry(l.data.data(), l.n.data(), l.type.data(), s, l.count(), code, max_norm, (double *)room.data_ptr(), room.numel(), at, out == Py_None ? nullptr : at + 1, stream);
        Py_END_ALLOW_THREADS
        if (rc) return failed("grad_norm", rc);
        return THPVariable_Wrap(result);
    });
}

// clip(sequence, grads, norm_type, max_norm): the gradients scaled in place; results as norm's
static PyObject *clip(PyObject *, PyObject *args)
{
    PyObject *seq;
    int grads, code;
    double max_norm;
    if (!PyArg_ParseTuple(args, "Opid", &seq, &grads, &code, &max_norm)) return nullptr;
    return guarded([&]() -> PyObject * {
        Lists l;
        if (!collect(seq, grads != 0, true, l)) return nullptr;
        auto gradient = [&](Py_ssize_t k) -> const at::Tensor & {
            const at::Tensor &own = THPVariable_Unpack(PyList_GET_ITEM(seq, k));
            return grads ? own.grad() : own;
        };
        if (!l.irregular.empty()) {
            std::vector<at::Tensor> tensors;
            for (Py_ssize_t k = 0; k < PyList_GET_SIZE(seq); ++k)
                if (gradient(k).defined()) tensors.push_back(gradient(k));
            size_t i, j;
            if (!shared(tensors, &i, &j)) return irregular_list(l);
            return i == j ? PyErr_Format(PyExc_RuntimeError, "clip_grad_norm_: a gradient whose elements share memory (an expanded tensor) cannot be scaled in place")
                          : PyErr_Format(PyExc_RuntimeError, "clip_grad_norm_: two gradients share memory (the same tensor twice, or overlapping views)");
        }
        if (l.device < 0) Py_RETURN_NONE;
        // versions go up, as with any operation in place
        for (c10::TensorImpl *t : l.written)
            if (!t->is_inference()) t->bump_version();
        const c10::DeviceGuard device(at::Device(at::kCUDA, (at::DeviceIndex)l.device));
        void *stream;
        if (!current_stream(l.device, &stream)) return nullptr;
        const at::Tensor result = empty({}, at::kFloat, l.device);
        const int64_t size = workspace_entry(l.n.data(), l.type.data(), l.count(), 1);
        at::Tensor room;
        if (size) room = empty({size}, at::kDouble, l.device);
        float *at = (float *)result.data_ptr();
        double *w = size ? (double *)room.data_ptr() : nullptr;
        int rc;
        Py_BEGIN_ALLOW_THREADS
        rc = grad_clip_entry(l.data.data(), l.n.data(), l.type.data(), l.count(), code, max_norm, w, size, at, stream);
        Py_END_ALLOW_THREADS
        if (rc == -1) {                     // refused, nothing written: they come down again (of gradients that are still the parameters')
            size_t at = 0;
            for (Py_ssize_t k = 0; k < PyList_GET_SIZE(seq); ++k) {
                const at::Tensor &t = gradient(k);
                if (at >= l.written.size() || t.unsafeGetTensorImpl() != l.written[at]) continue;
                ++at;
                c10::VariableVersion version = t.unsafeGetTensorImpl()->version_counter();
                if (!t.is_inference() && version.current_version() > 0) version.set_version((int64_t)version.current_version() - 1);
            }
        }
        if (rc) return failed("clip_grad_norm_", rc);
        return THPVariable_Wrap(result);
    });
}

// shared(tensors): the positions of two tensors that share memory -- of one whose own elements do: its position twice -- or None (host or GPU: nothing is read)
static PyObject *shared_pair(PyObject *, PyObject *seq)
{
    return guarded([&]() -> PyObject * {
        std::vector<at::Tensor> tensors;
        if (!PyList_Check(seq)) return PyErr_Format(PyExc_TypeError, "a list is expected");
        for (Py_ssize_t k = 0; k < PyList_GET_SIZE(seq); ++k) {
            if (!THPVariable_Check(PyList_GET_ITEM(seq, k))) return PyErr_Format(PyExc_TypeError, "tensors are expected");
            tensors.push_back(THPVariable_Unpack(PyList_GET_ITEM(seq, k)));
        }
        size_t i, j;
        if (!shared(tensors, &i, &j)) Py_RETURN_NONE;
        return Py_BuildValue("nn", (Py_ssize_t)i, (Py_ssize_t)j);
    });
}

// bind(nvdr_grad_norm, nvdr_grad_clip, nvdr_grad_norm_workspace, nvdr_last_error, raw_stream): the library's entries, and where the stream comes from
static PyObject *bind(PyObject *, PyObject *args)
{
    unsigned long long a, b, c, d;
    PyObject *stream;
    if (!PyArg_ParseTuple(args, "KKKKO", &a, &b, &c, &d, &stream)) return nullptr;
    grad_norm_entry = (decltype(grad_norm_entry))(uintptr_t)a;
    grad_clip_entry = (decltype(grad_clip_entry))(uintptr_t)b;
    workspace_entry = (decltype(workspace_entry))(uintptr_t)c;
    last_error_entry = (decltype(last_error_entry))(uintptr_t)d;
    Py_INCREF(stream);
    Py_XDECREF(raw_stream);
    raw_stream = stream;
    Py_RETURN_NONE;
}

static PyMethodDef methods[] = {{"norm", norm, METH_VARARGS, "norm(tensors, scales, norm_type, max_norm, out, work)"},
                                {"clip", clip, METH_VARARGS, "clip(sequence, grads, norm_type, max_norm)"},
                                {"shared", shared_pair, METH_O, "shared(tensors)"},
                                {"bind", bind, METH_VARARGS, "bind(nvdr_grad_norm, nvdr_grad_clip, nvdr_grad_norm_workspace, nvdr_last_error, raw_stream)"},
                                {nullptr, nullptr, 0, nullptr}};
static PyModuleDef module = {PyModuleDef_HEAD_INIT, "_gradops", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

PyMODINIT_FUNC PyInit__gradops(void) { return PyModule_Create(&module); }
