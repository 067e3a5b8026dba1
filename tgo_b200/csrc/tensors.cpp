// What a wrapper asks of its tensors, asked natively: a Python attribute of a tensor costs 40 to 60 ns, and a wrapper of
// twelve tensors spends more on four of each than on its launch.
//
//   look(kinds, *tensors) -> [address, ...] + [how many numbers, ...], a letter of `kinds` a tensor: i int32, l int64, f float32,
//     b bfloat16. None: 0 and 0. One that is no contiguous tensor of that type on a GPU: None instead of the list
//   rows(tensor) -> (rows, columns, stride of a row, stride of a column, address) of a matrix on a GPU, else None
//   pages(tensor, axis) -> (places of a page, numbers, address, what lies before the pages, pages, heads, bytes of a row) of a contiguous
//     tensor on a GPU whose pages [heads, places, width] or [places, width] lie along `axis`, else None
//
// The caller finds out what is wrong and says so. (What a tensor throws is a None too.)
//
// MEASURED, host time of a call on a B200's host: logits_constrain with eleven tensors 8.4 us by attributes,
// 5.8 so; tree_accept 5.9 and 4.2, attention_tree 10.1 and 8.3 (the launches themselves take 2 us, its workspace 1.5).
#include <torch/csrc/autograd/python_variable.h>

static bool there(const at::Tensor& t) { return t.is_cuda() && t.layout() == at::kStrided; }

static PyObject* ten_look(PyObject*, PyObject* const* args, Py_ssize_t n) {
    Py_ssize_t length = 0;
    const char* kinds = n > 0 && PyUnicode_Check(args[0]) ? PyUnicode_AsUTF8AndSize(args[0], &length) : nullptr;
    if (!kinds || length != n - 1) {
        if (!PyErr_Occurred()) PyErr_SetString(PyExc_TypeError, "look(kinds, *tensors): a letter a tensor");
        return nullptr;
    }
    PyObject* out = PyList_New(2 * length);
    if (!out) return nullptr;
    for (Py_ssize_t k = 0; k < length; ++k) {
        unsigned long long address = 0;
        long long count = 0;
        PyObject* o = args[k + 1];
        if (o != Py_None) {
            const at::ScalarType want = kinds[k] == 'i' ? at::kInt : kinds[k] == 'l' ? at::kLong : kinds[k] == 'f' ? at::kFloat : at::kBFloat16;
            bool ok = THPVariable_Check(o);
            if (ok) try {
                const at::Tensor& t = THPVariable_Unpack(o);
                ok = there(t) && t.scalar_type() == want && t.is_contiguous();
                if (ok) {
                    address = (unsigned long long)(uintptr_t)t.const_data_ptr();
                    count = t.numel();
                    ok = address || !count;               // one without storage
                }
            } catch (const std::exception&) { ok = false; }
            if (!ok) {
                Py_DECREF(out);
                Py_RETURN_NONE;
            }
        }
        PyObject *a = PyLong_FromUnsignedLongLong(address), *c = PyLong_FromLongLong(count);
        if (!a || !c) {
            Py_XDECREF(a);
            Py_XDECREF(c);
            Py_DECREF(out);
            return nullptr;
        }
        PyList_SET_ITEM(out, k, a);
        PyList_SET_ITEM(out, length + k, c);
    }
    return out;
}

static PyObject* ten_rows(PyObject*, PyObject* o) {
    if (!THPVariable_Check(o)) Py_RETURN_NONE;
    long long size[2], stride[2];
    unsigned long long address;
    try {
        const at::Tensor& t = THPVariable_Unpack(o);
        if (!there(t) || t.dim() != 2) Py_RETURN_NONE;
        for (int i = 0; i < 2; ++i) {
            size[i] = t.size(i);
            stride[i] = t.stride(i);
        }
        address = (unsigned long long)(uintptr_t)t.const_data_ptr();
        if (!address && size[0] && size[1]) Py_RETURN_NONE;
    } catch (const std::exception&) { Py_RETURN_NONE; }
    return Py_BuildValue("LLLLK", size[0], size[1], stride[0], stride[1], address);
}

static PyObject* ten_pages(PyObject*, PyObject* const* args, Py_ssize_t n) {
    const long long axis = n == 2 ? PyLong_AsLongLong(args[1]) : -1;
    if (n != 2 || (axis == -1 && PyErr_Occurred())) {
        if (!PyErr_Occurred()) PyErr_SetString(PyExc_TypeError, "pages(tensor, axis)");
        return nullptr;
    }
    if (!THPVariable_Check(args[0])) Py_RETURN_NONE;
    long long outer = 1, pages, heads, places, bytes, count;
    unsigned long long address;
    try {
        const at::Tensor& t = THPVariable_Unpack(args[0]);
        const long long rest = t.dim() - axis;
        if (!there(t) || axis < 0 || (rest != 3 && rest != 4) || !t.is_contiguous()) Py_RETURN_NONE;
        for (long long i = 0; i < axis; ++i) outer *= t.size(i);
        pages = t.size(axis);
        heads = rest == 4 ? t.size(axis + 1) : 1;
        places = t.size(-2);
        bytes = t.size(-1) * (long long)t.element_size();
        count = t.numel();
        address = (unsigned long long)(uintptr_t)t.const_data_ptr();
        if (!address && count) Py_RETURN_NONE;
    } catch (const std::exception&) { Py_RETURN_NONE; }
    return Py_BuildValue("LLKLLLL", places, count, address, outer, pages, heads, bytes);
}

static PyMethodDef ten_methods[] = {
    {"look", (PyCFunction)(void (*)(void))ten_look, METH_FASTCALL, "look(kinds, *tensors) -> addresses and counts, or None"},
    {"rows", ten_rows, METH_O, "rows(matrix) -> sizes, strides and address, or None"},
    {"pages", (PyCFunction)(void (*)(void))ten_pages, METH_FASTCALL, "pages(tensor, axis) -> sizes and address, or None"},
    {nullptr, nullptr, 0, nullptr}};
static PyModuleDef ten_module = {PyModuleDef_HEAD_INIT, "tgo_tensors", nullptr, -1, ten_methods, nullptr, nullptr, nullptr, nullptr};

PyMODINIT_FUNC PyInit_tgo_tensors() { return PyModule_Create(&ten_module); }
