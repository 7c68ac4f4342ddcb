// tensor_list.cpp - reads a list of tensors for the entry points that take many (gs_b200.grad, the clipped steps of
// gs_b200.adam): their addresses, sizes and types as packed arrays, in one call from Python.
//
// Asked through Python, a tensor's five properties cost about 0.4 us, which for a few hundred tensors is ten times
// what the kernels take. This module launches nothing; the kernels stay behind the C ABI.
#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstdint>
#include <exception>
#include <vector>

namespace {

// SPLAT_F32 ... SPLAT_F64 of include/splat_b200.h, or -1.
int code_of(at::ScalarType t) {
    switch (t) {
        case at::ScalarType::Float: return 0;
        case at::ScalarType::BFloat16: return 1;
        case at::ScalarType::Half: return 2;
        case at::ScalarType::Double: return 3;
        default: return -1;
    }
}

// The entries of a list or tuple, or no entries for anything else.
struct Entries {
    PyObject** items = nullptr;
    Py_ssize_t count = 0;
    explicit Entries(PyObject* seq) {
        if (PyList_Check(seq) || PyTuple_Check(seq)) {
            items = PySequence_Fast_ITEMS(seq);
            count = PySequence_Fast_GET_SIZE(seq);
        }
    }
};

// describe(list or tuple) -> (addresses uint64, element counts int64, type codes uint8, all contiguous, device index,
// whether that is the current device, its current stream), the first three as bytes, when every entry is a dense
// strided CUDA tensor of a known type, all on one device; otherwise None (the caller then says which is not, and why).
PyObject* describe(PyObject*, PyObject* seq) {
    const Entries e(seq);
    if (e.count == 0) Py_RETURN_NONE;
    try {
        std::vector<uint64_t> address(e.count);
        std::vector<int64_t> size(e.count);
        std::vector<uint8_t> code(e.count);
        int device = -1;
        bool contiguous = true;
        for (Py_ssize_t i = 0; i < e.count; ++i) {
            if (!THPVariable_Check(e.items[i])) Py_RETURN_NONE;
            const at::Tensor& t = THPVariable_Unpack(e.items[i]);
            if (!t.defined() || !t.is_cuda() || t.layout() != at::kStrided) Py_RETURN_NONE;
            const int c = code_of(t.scalar_type());
            if (c < 0 || (i > 0 && t.get_device() != device)) Py_RETURN_NONE;
            device = static_cast<int>(t.get_device());
            size[i] = t.numel();
            if (!t.is_contiguous()) {
                contiguous = false;
                if (size[i] > 0 && !t.is_non_overlapping_and_dense()) Py_RETURN_NONE;
            }
            code[i] = static_cast<uint8_t>(c);
            address[i] = reinterpret_cast<uint64_t>(t.data_ptr());
        }
        const auto index = static_cast<c10::DeviceIndex>(device);
        const auto stream = reinterpret_cast<unsigned long long>(c10::cuda::getCurrentCUDAStream(index).stream());
        return Py_BuildValue("(y#y#y#OiOK)", reinterpret_cast<const char*>(address.data()), e.count * Py_ssize_t(8),
                             reinterpret_cast<const char*>(size.data()), e.count * Py_ssize_t(8),
                             reinterpret_cast<const char*>(code.data()), e.count, contiguous ? Py_True : Py_False,
                             device, c10::cuda::current_device() == index ? Py_True : Py_False, stream);
    } catch (const std::exception&) {  // a tensor without storage of its own (fake, functional)
        Py_RETURN_NONE;
    }
}

// same_form(a, b) -> whether the two lists' tensors agree one by one in shape, type and (with elements) strides.
PyObject* same_form(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    if (nargs != 2) {
        PyErr_SetString(PyExc_TypeError, "same_form takes two lists");
        return nullptr;
    }
    const Entries a(args[0]), b(args[1]);
    if (a.count != b.count) Py_RETURN_FALSE;
    try {
        for (Py_ssize_t i = 0; i < a.count; ++i) {
            if (!THPVariable_Check(a.items[i]) || !THPVariable_Check(b.items[i])) Py_RETURN_FALSE;
            const at::Tensor &x = THPVariable_Unpack(a.items[i]), &y = THPVariable_Unpack(b.items[i]);
            if (x.scalar_type() != y.scalar_type() || x.sizes() != y.sizes()) Py_RETURN_FALSE;
            if (x.numel() > 0 && !(x.is_contiguous() && y.is_contiguous()) && x.strides() != y.strides())
                Py_RETURN_FALSE;
        }
    } catch (const std::exception&) {
        Py_RETURN_FALSE;
    }
    Py_RETURN_TRUE;
}

PyMethodDef kMethods[] = {
    {"describe", describe, METH_O, "describe(tensors) -> (addresses, sizes, codes, contiguous, device, current, stream)"},
    {"same_form", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(same_form)), METH_FASTCALL,
     "same_form(a, b) -> shapes, types and strides agree"},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_tensors", nullptr, -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__tensors() { return PyModule_Create(&kModule); }
