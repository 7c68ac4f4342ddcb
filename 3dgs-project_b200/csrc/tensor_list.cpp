// tensor_list.cpp - the Python side's reading of tensors for the entry points that take many (gs_b200.grad, the clipped
// steps of gs_b200.adam): addresses, sizes and types as the C ABI's arrays, in one call from Python, and the buffers
// that such a call needs.
//
// Asked through Python, a tensor's five properties cost about 0.4 us, which for a few hundred tensors is ten times
// what the kernels take. This module launches nothing; the kernels stay behind the C ABI.
#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <ATen/ops/empty.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstdint>
#include <exception>
#include <vector>

#include "../../include/splat_b200.h"

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

// describe(list or tuple) -> (addresses uint64, element counts int64, type codes uint8, device index, whether that is
// the current device, its current stream), the first three as bytes, when every entry is a dense
// strided CUDA tensor of a known type whose memory holds its values (no lazy negation), all on one device; otherwise
// None (the caller then says which is not, and why).
PyObject* describe(PyObject*, PyObject* seq) {
    const Entries e(seq);
    if (e.count == 0) Py_RETURN_NONE;
    try {
        std::vector<uint64_t> address(e.count);
        std::vector<int64_t> size(e.count);
        std::vector<uint8_t> code(e.count);
        int device = -1;
        for (Py_ssize_t i = 0; i < e.count; ++i) {
            if (!THPVariable_Check(e.items[i])) Py_RETURN_NONE;
            const at::Tensor& t = THPVariable_Unpack(e.items[i]);
            if (!t.defined() || !t.is_cuda() || t.layout() != at::kStrided || t.is_neg()) Py_RETURN_NONE;
            const int c = code_of(t.scalar_type());
            if (c < 0 || (i > 0 && t.get_device() != device)) Py_RETURN_NONE;
            device = static_cast<int>(t.get_device());
            size[i] = t.numel();
            if (size[i] > 0 && !t.is_contiguous() && !t.is_non_overlapping_and_dense()) Py_RETURN_NONE;
            code[i] = static_cast<uint8_t>(c);
            address[i] = reinterpret_cast<uint64_t>(t.data_ptr());
        }
        const auto index = static_cast<c10::DeviceIndex>(device);
        const auto stream = reinterpret_cast<unsigned long long>(c10::cuda::getCurrentCUDAStream(index).stream());
        return Py_BuildValue("(y#y#y#iOK)", reinterpret_cast<const char*>(address.data()), e.count * Py_ssize_t(8),
                             reinterpret_cast<const char*>(size.data()), e.count * Py_ssize_t(8),
                             reinterpret_cast<const char*>(code.data()), e.count, device,
                             c10::cuda::current_device() == index ? Py_True : Py_False, stream);
    } catch (const std::exception&) {  // a tensor without storage of its own (fake, functional)
        Py_RETURN_NONE;
    }
}

// Two tensors of one shape lie alike in memory: their strides agree where a dimension has more than one entry.
bool lie_alike(const at::Tensor& x, const at::Tensor& y) {
    if (x.numel() == 0 || (x.is_contiguous() && y.is_contiguous())) return true;
    for (int64_t d = 0; d < x.dim(); ++d)
        if (x.size(d) != 1 && x.stride(d) != y.stride(d)) return false;
    return true;
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
            if (!lie_alike(x, y)) Py_RETURN_FALSE;
        }
    } catch (const std::exception&) {
        Py_RETURN_FALSE;
    }
    Py_RETURN_TRUE;
}

// scratch(device, float64, bytes) -> (a 0-d tensor for a norm, its address, a byte tensor, its address), on the device.
PyObject* scratch(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    if (nargs != 3) {
        PyErr_SetString(PyExc_TypeError, "scratch takes a device, a truth value and a size");
        return nullptr;
    }
    const long device = PyLong_AsLong(args[0]);
    const int f64 = PyObject_IsTrue(args[1]);
    const long long bytes = PyLong_AsLongLong(args[2]);
    if (PyErr_Occurred()) return nullptr;
    HANDLE_TH_ERRORS  // out of memory is torch.OutOfMemoryError
    const auto on = at::TensorOptions().device(at::Device(at::kCUDA, static_cast<c10::DeviceIndex>(device)));
    at::Tensor norm = at::empty({}, on.dtype(f64 ? at::kDouble : at::kFloat));
    at::Tensor space = at::empty({bytes}, on.dtype(at::kByte));
    const auto norm_at = reinterpret_cast<unsigned long long>(norm.data_ptr());
    const auto space_at = reinterpret_cast<unsigned long long>(space.data_ptr());
    return Py_BuildValue("(NKNK)", THPVariable_Wrap(std::move(norm)), norm_at, THPVariable_Wrap(std::move(space)),
                         space_at);
    END_HANDLE_TH_ERRORS
}

// adam_table(groups, lean) -> (adam_group or adam_lean_group array as bytes, device index, whether that is the current
// device, its current stream) for groups (param, grad, exp_avg, exp_avg_sq, lr) of contiguous CUDA tensors of one size
// on one device: float32, or for the lean table both moments bfloat16; lr a Python float. None where a group is not that.
// A parameter that appears twice raises.
PyObject* adam_table(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    if (nargs != 2) {
        PyErr_SetString(PyExc_TypeError, "adam_table takes groups and a truth value");
        return nullptr;
    }
    const Entries groups(args[0]);
    const int lean = PyObject_IsTrue(args[1]);
    if (groups.count == 0 || lean < 0) Py_RETURN_NONE;
    try {
        std::vector<adam_group> dense(lean ? 0 : groups.count);
        std::vector<adam_lean_group> sparse(lean ? groups.count : 0);
        std::vector<const void*> params(groups.count);
        c10::DeviceIndex device = -1;
        for (Py_ssize_t i = 0; i < groups.count; ++i) {
            const Entries g(groups.items[i]);
            if (g.count != 5) Py_RETURN_NONE;
            void* at[4];
            at::ScalarType kind[4];
            long long n = 0, rows = 1;
            for (int k = 0; k < 4; ++k) {
                if (!THPVariable_Check(g.items[k])) Py_RETURN_NONE;
                const at::Tensor& t = THPVariable_Unpack(g.items[k]);
                if (!t.defined() || !t.is_cuda() || t.layout() != at::kStrided || !t.is_contiguous() || t.is_neg())
                    Py_RETURN_NONE;
                if (i == 0 && k == 0) device = t.get_device();
                if (k == 0) {
                    n = t.numel();
                    if (lean && t.dim() == 0) Py_RETURN_NONE;
                    rows = lean && t.size(0) > 0 ? t.size(0) : 1;
                }
                if (t.get_device() != device || t.numel() != n) Py_RETURN_NONE;
                kind[k] = t.scalar_type();
                at[k] = t.data_ptr();
            }
            const bool low = kind[2] == at::kBFloat16;
            if (kind[0] != at::kFloat || kind[1] != at::kFloat || kind[2] != kind[3] ||
                !(kind[2] == at::kFloat || (lean && low)))
                Py_RETURN_NONE;
            if (!PyFloat_Check(g.items[4])) Py_RETURN_NONE;  // anything else may run code that changes the lists
            const double lr = PyFloat_AS_DOUBLE(g.items[4]);
            params[i] = n > 0 ? at[0] : nullptr;
            for (Py_ssize_t j = 0; j < i; ++j)
                if (params[i] && params[i] == params[j]) {
                    PyErr_SetString(PyExc_RuntimeError, "a parameter appears in two groups");
                    return nullptr;
                }
            if (lean)
                sparse[i] = {static_cast<float*>(at[0]), static_cast<const float*>(at[1]), at[2], at[3], n, lr,
                             static_cast<int>(n / rows), low ? 1 : 0};
            else
                dense[i] = {static_cast<float*>(at[0]), static_cast<const float*>(at[1]), static_cast<float*>(at[2]),
                            static_cast<float*>(at[3]), n, lr};
        }
        const char* table = lean ? reinterpret_cast<const char*>(sparse.data()) : reinterpret_cast<const char*>(dense.data());
        const Py_ssize_t size = groups.count * static_cast<Py_ssize_t>(lean ? sizeof(adam_lean_group) : sizeof(adam_group));
        const auto stream = reinterpret_cast<unsigned long long>(c10::cuda::getCurrentCUDAStream(device).stream());
        return Py_BuildValue("(y#iOK)", table, size, static_cast<int>(device),
                             c10::cuda::current_device() == device ? Py_True : Py_False, stream);
    } catch (const std::exception&) {
        Py_RETURN_NONE;
    }
}

void bump(PyObject* item) {
    if (!THPVariable_Check(item)) return;
    const at::Tensor& t = THPVariable_Unpack(item);
    if (t.defined() && !t.is_inference()) t.unsafeGetTensorImpl()->bump_version();  // inference tensors count nothing
}

// written(entries): tells autograd that a kernel wrote the entries, tensors or the groups (param, grad, exp_avg,
// exp_avg_sq, lr) of a step, so that a backward that saved their old values raises.
PyObject* written(PyObject*, PyObject* seq) {
    HANDLE_TH_ERRORS
    const Entries e(seq);
    for (Py_ssize_t i = 0; i < e.count; ++i) {
        const Entries group(e.items[i]);
        if (group.count == 0) bump(e.items[i]);
        for (Py_ssize_t k = 0; k < group.count && k < 4; ++k)
            if (k != 1) bump(group.items[k]);
    }
    Py_RETURN_NONE;
    END_HANDLE_TH_ERRORS
}

PyMethodDef kMethods[] = {
    {"describe", describe, METH_O, "describe(tensors) -> (addresses, sizes, codes, device, current, stream)"},
    {"same_form", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(same_form)), METH_FASTCALL,
     "same_form(a, b) -> shapes, types and strides agree"},
    {"scratch", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(scratch)), METH_FASTCALL,
     "scratch(device, float64, bytes) -> (norm, address, workspace, address)"},
    {"adam_table", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(adam_table)), METH_FASTCALL,
     "adam_table(groups, lean) -> (table, device, current, stream)"},
    {"written", written, METH_O, "written(tensors or groups): counts a write for autograd"},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_tensors", nullptr, -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__tensors() { return PyModule_Create(&kModule); }
