// gradlist.cpp -- the lists that nvdr_grad_norm / nvdr_grad_clip take, read out of Python tensors in one call.
//
// A network has hundreds of parameters, and asking each of its gradients for address, length, type, device and layout through Python takes
// about 0.4 us a tensor: for many short tensors several times what the kernels take.  Here it is some 20 ns.  A CPython extension of its own:
// the C library stays free of torch.
#define PY_SSIZE_T_CLEAN
#include <torch/csrc/autograd/python_variable.h>
#include <ATen/core/Tensor.h>

// collect(sequence, grads, written) -> (device, data, n, types, irregular)
//   sequence   a list or tuple of tensors; grads: of parameters, whose gradients are meant (None is left out)
//   written    the call is going to write to them: their versions go up, as with any operation in place
//   device     the index of their GPU, -1 if there is no tensor
//   data, n, types   the library's lists as bytes
//   irregular  positions (among the gradients) of tensors whose elements do not fill their memory exactly once; the lists are of use if it is empty
static PyObject *collect(PyObject *, PyObject *args)
{
    PyObject *seq;
    int grads, written;
    if (!PyArg_ParseTuple(args, "Opp", &seq, &grads, &written)) return nullptr;
    PyObject *fast = PySequence_Fast(seq, "gradients must be a list or tuple");
    if (!fast) return nullptr;
    PyObject *result = nullptr, *data = nullptr, *n = nullptr, *types = nullptr, *irregular = PyList_New(0);
    try {
        const Py_ssize_t most = PySequence_Fast_GET_SIZE(fast);
        data = PyBytes_FromStringAndSize(nullptr, most * 8);
        n = PyBytes_FromStringAndSize(nullptr, most * 8);
        types = PyBytes_FromStringAndSize(nullptr, most);
        bool ok = irregular && data && n && types;
        Py_ssize_t count = 0;
        long device = -1;
        for (Py_ssize_t k = 0; ok && k < most; ++k) {
            PyObject *item = PySequence_Fast_GET_ITEM(fast, k);
            if (!THPVariable_Check(item)) {
                PyErr_Format(PyExc_TypeError, "gradients must be tensors (got %s)", Py_TYPE(item)->tp_name);
                ok = false;
                break;
            }
            const at::Tensor &own = THPVariable_Unpack(item);
            const at::Tensor &t = grads ? own.grad() : own;
            if (!t.defined()) continue;
            int type;
            switch (t.scalar_type()) {
            case at::kFloat: type = 0; break;
            case at::kBFloat16: type = 1; break;
            case at::kHalf: type = 2; break;
            default: type = -1;
            }
            ok = false;
            if (type < 0) {
                PyObject *d = PyObject_GetAttrString(item, "dtype");
                if (d) PyErr_Format(PyExc_ValueError, "gradients must be float32, bfloat16 or float16 (got %S)", d);
                Py_XDECREF(d);
            } else if (!t.is_cuda() || (device >= 0 && t.get_device() != device)) {
                PyErr_SetString(PyExc_RuntimeError, "gradients must reside on one GPU; this path has no CPU fallback");
            } else if (t.layout() != at::kStrided) {
                PyErr_SetString(PyExc_ValueError, "gradients must be dense");
            } else {
                ok = true;
                device = t.get_device();
                if (!t.is_non_overlapping_and_dense()) {
                    PyObject *i = PyLong_FromSsize_t(count);
                    ok = i && PyList_Append(irregular, i) == 0;
                    Py_XDECREF(i);
                }
                ((int64_t *)PyBytes_AS_STRING(data))[count] = (int64_t)(uintptr_t)t.data_ptr();
                ((int64_t *)PyBytes_AS_STRING(n))[count] = t.numel();
                PyBytes_AS_STRING(types)[count] = (char)type;
                if (written && !t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
                ++count;
            }
        }
        ok = ok && _PyBytes_Resize(&data, count * 8) == 0 && _PyBytes_Resize(&n, count * 8) == 0 && _PyBytes_Resize(&types, count) == 0;
        if (ok) result = Py_BuildValue("lOOOO", device, data, n, types, irregular);
    } catch (const std::exception &e) {
        if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, e.what());
    } catch (...) {
        if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, "reading the gradients failed");
    }
    Py_XDECREF(irregular);
    Py_XDECREF(types);
    Py_XDECREF(n);
    Py_XDECREF(data);
    Py_DECREF(fast);
    return result;
}

static PyMethodDef methods[] = {{"collect", collect, METH_VARARGS, "collect(sequence, grads, written) -> (device, data, n, types, irregular)"}, {nullptr, nullptr, 0, nullptr}};
static PyModuleDef module = {PyModuleDef_HEAD_INIT, "_gradlist", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

PyMODINIT_FUNC PyInit__gradlist(void) { return PyModule_Create(&module); }
