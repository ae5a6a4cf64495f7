// Python's way to the C entry points for operators of a few microseconds: one call checks every tensor against what the operator expects, takes
// their addresses and the device's current stream, and calls the entry point. (Checked and converted one by one in Python, the eight tensors of a block
// norm took 7 us of the host, twice as long as the call itself.)
//
//   specs = make_specs(((dtype, shape), ...))                          what the operands have to be; kept by the caller
//   status = call(entry, descriptor, specs, workspace, offset, operands...)
//
// `entry` is the address of int f(const void* descriptor, operands..., [void* workspace, size_t bytes,] void* stream), every argument of which takes an integer
// register; an operand is a tensor or None (a null pointer); `workspace` is a tensor or None, used from byte `offset` on. Returns the entry point's status, or
// 1 + i where operand i is not what its spec says (nothing is called then): the caller raises what is wrong with it. With 0 for `entry` the operands are checked
// only.
#include <Python.h>

#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/python_variable.h>

#include <vector>

namespace {

struct Spec {
    c10::ScalarType dtype;
    std::vector<int64_t> shape;
};
typedef std::vector<Spec> Specs;
constexpr const char* SPECS = "phoenix_core_b200.specs";
constexpr int MAX_OPERANDS = 16;

void free_specs(PyObject* capsule) { delete static_cast<Specs*>(PyCapsule_GetPointer(capsule, SPECS)); }

PyObject* make_specs(PyObject*, PyObject* list) {
    if (!PyTuple_Check(list) || PyTuple_GET_SIZE(list) > MAX_OPERANDS) {
        PyErr_SetString(PyExc_TypeError, "a tuple of at most 16 (dtype, shape) expected");
        return nullptr;
    }
    Specs* specs = new Specs;
    for (Py_ssize_t i = 0; i < PyTuple_GET_SIZE(list); ++i) {
        PyObject *dtype, *shape;
        if (!PyArg_ParseTuple(PyTuple_GET_ITEM(list, i), "OO!", &dtype, &PyTuple_Type, &shape) || !THPDtype_Check(dtype)) {
            if (!PyErr_Occurred()) PyErr_SetString(PyExc_TypeError, "(dtype, shape) expected");
            delete specs;
            return nullptr;
        }
        Spec s{reinterpret_cast<THPDtype*>(dtype)->scalar_type, {}};
        for (Py_ssize_t k = 0; k < PyTuple_GET_SIZE(shape); ++k) s.shape.push_back(PyLong_AsLongLong(PyTuple_GET_ITEM(shape, k)));
        if (PyErr_Occurred()) {
            delete specs;
            return nullptr;
        }
        specs->push_back(std::move(s));
    }
    PyObject* capsule = PyCapsule_New(specs, SPECS, free_specs);
    if (!capsule) delete specs;
    return capsule;
}

typedef uintptr_t W;
// f(words[0 .. n - 1])
int invoke(W f, const W* w, int n) {
#define A(i) w[i]
    switch (n) {
        case 4: return reinterpret_cast<int (*)(W, W, W, W)>(f)(A(0), A(1), A(2), A(3));
        case 5: return reinterpret_cast<int (*)(W, W, W, W, W)>(f)(A(0), A(1), A(2), A(3), A(4));
        case 8: return reinterpret_cast<int (*)(W, W, W, W, W, W, W, W)>(f)(A(0), A(1), A(2), A(3), A(4), A(5), A(6), A(7));
        case 9: return reinterpret_cast<int (*)(W, W, W, W, W, W, W, W, W)>(f)(A(0), A(1), A(2), A(3), A(4), A(5), A(6), A(7), A(8));
        case 10: return reinterpret_cast<int (*)(W, W, W, W, W, W, W, W, W, W)>(f)(A(0), A(1), A(2), A(3), A(4), A(5), A(6), A(7), A(8), A(9));
        case 17:
            return reinterpret_cast<int (*)(W, W, W, W, W, W, W, W, W, W, W, W, W, W, W, W, W)>(f)(A(0), A(1), A(2), A(3), A(4), A(5), A(6), A(7), A(8), A(9), A(10), A(11), A(12), A(13),
                                                                                                A(14), A(15), A(16));
        default: return -2;                                        // (no entry point has another number of arguments)
    }
#undef A
}

PyObject* checked_call(PyObject* const* args, Py_ssize_t nargs) {
    if (nargs < 6) {
        PyErr_SetString(PyExc_TypeError, "call(entry, descriptor, specs, workspace, offset, operands...)");
        return nullptr;
    }
    const W entry = PyLong_AsUnsignedLongLong(args[0]), descriptor = PyLong_AsUnsignedLongLong(args[1]);
    const Specs* specs = static_cast<const Specs*>(PyCapsule_GetPointer(args[2], SPECS));
    const W offset = PyLong_AsUnsignedLongLong(args[4]);
    if (!specs || PyErr_Occurred()) return nullptr;
    const int n = (int)(nargs - 5);
    if ((size_t)n != specs->size()) {
        PyErr_SetString(PyExc_TypeError, "an operand for each spec expected");
        return nullptr;
    }
    W words[MAX_OPERANDS + 4];
    int count = 0, device = -1;
    words[count++] = descriptor;
    for (int i = 0; i < n; ++i) {
        PyObject* o = args[5 + i];
        if (o == Py_None) {
            words[count++] = 0;
            continue;
        }
        if (!THPVariable_Check(o)) return PyLong_FromLong(1 + i);
        const at::Tensor& t = THPVariable_Unpack(o);
        const Spec& s = (*specs)[i];
        if (!t.is_cuda() || t.layout() != c10::kStrided || t.scalar_type() != s.dtype || t.sizes() != c10::IntArrayRef(s.shape) || !t.is_contiguous()) return PyLong_FromLong(1 + i);
        if (device < 0) device = t.get_device();
        else if (t.get_device() != device) return PyLong_FromLong(1 + i);
        words[count++] = reinterpret_cast<W>(t.data_ptr());
    }
    if (device < 0) return PyLong_FromLong(1);
    if (entry == 0) return PyLong_FromLong(0);
    if (args[3] != Py_None) {
        if (!THPVariable_Check(args[3])) {
            PyErr_SetString(PyExc_TypeError, "a workspace is a tensor");
            return nullptr;
        }
        const at::Tensor& t = THPVariable_Unpack(args[3]);
        if (t.get_device() != device || t.nbytes() < offset) {
            PyErr_SetString(PyExc_ValueError, "the workspace does not suit the call");
            return nullptr;
        }
        words[count++] = reinterpret_cast<W>(t.data_ptr()) + offset;
        words[count++] = t.nbytes() - offset;
    }
    c10::cuda::OptionalCUDAGuard guard;
    if (c10::cuda::current_device() != device) guard.set_index((c10::DeviceIndex)device);
    words[count++] = reinterpret_cast<W>(c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)device).stream());
    int status;
    Py_BEGIN_ALLOW_THREADS
    status = invoke(entry, words, count);
    Py_END_ALLOW_THREADS
    return PyLong_FromLong(status);
}

PyObject* call(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    try {
        return checked_call(args, nargs);
    } catch (const std::exception& e) {                            // (no exception leaves through the interpreter's C frames)
        PyErr_SetString(PyExc_RuntimeError, e.what());
        return nullptr;
    }
}

PyMethodDef methods[] = {{"make_specs", make_specs, METH_O, "What a call's operands have to be."},
                         {"call", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(call)), METH_FASTCALL, "Checks the operands and calls an entry point."},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_binding", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__binding() { return PyModule_Create(&module); }
