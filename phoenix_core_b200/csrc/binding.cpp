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

#include <cuda_runtime_api.h>

#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/python_variable.h>

#include <atomic>
#include <new>
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

// The capture that a stream is part of, as a number of its own (0: none). A capture holds on to what its kernels use until the graph and everything
// instantiated from it are gone: watch_capture gives the graph an object that the runtime releases then, ended(watch) says whether it has.
unsigned long long capture_of(W stream, cudaGraph_t* graph = nullptr) {
    cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
    unsigned long long id = 0;
    if (cudaStreamGetCaptureInfo(reinterpret_cast<cudaStream_t>(stream), &status, &id, graph) != cudaSuccess) {
        cudaGetLastError();                                        // (the legacy stream beside a capture: it is part of none)
        return 0;
    }
    return status == cudaStreamCaptureStatusActive ? id + 1 : 0;
}
PyObject* capture_id(PyObject*, PyObject* stream) {
    const W s = PyLong_AsUnsignedLongLong(stream);
    return PyErr_Occurred() ? nullptr : PyLong_FromUnsignedLongLong(capture_of(s));
}

constexpr const char* WATCH = "phoenix_core_b200.watch";
std::atomic<long long> g_ended{0};                                  // graphs that are gone
struct Watch {
    std::atomic<int> holders{2};                                   // the graph and Python
    std::atomic<bool> told{false}, ended{false};                   // told: the graph took the object (where it took none, it never ends for us)
    void drop() {
        if (holders.fetch_sub(1) == 1) delete this;
    }
};
void CUDART_CB watch_released(void* w) {                            // (on a thread of the runtime's: no call into it or into Python)
    static_cast<Watch*>(w)->ended = true;
    ++g_ended;
    static_cast<Watch*>(w)->drop();
}
void free_watch(PyObject* capsule) { static_cast<Watch*>(PyCapsule_GetPointer(capsule, WATCH))->drop(); }

PyObject* watch_capture(PyObject*, PyObject* stream) {
    const W s = PyLong_AsUnsignedLongLong(stream);
    if (PyErr_Occurred()) return nullptr;
    cudaGraph_t graph = nullptr;
    if (capture_of(s, &graph) == 0) {
        PyErr_SetString(PyExc_RuntimeError, "the stream is not being captured");
        return nullptr;
    }
    Watch* watch = new (std::nothrow) Watch;
    if (!watch) return PyErr_NoMemory();
    PyObject* capsule = PyCapsule_New(watch, WATCH, free_watch);
    if (!capsule) {
        delete watch;
        return nullptr;
    }
    cudaUserObject_t object = nullptr;
    if (cudaUserObjectCreate(&object, watch, watch_released, 1, cudaUserObjectNoDestructorSync) != cudaSuccess) {
        watch->drop();                                             // (the graph's share: nothing will say when it ends)
    } else {
        watch->told = true;
        if (cudaGraphRetainUserObject(graph, object, 1, cudaGraphUserObjectMove) != cudaSuccess) {
            watch->told = false;
            cudaUserObjectRelease(object, 1);
        }
    }
    cudaGetLastError();
    return capsule;
}
PyObject* ended_count(PyObject*, PyObject*) { return PyLong_FromLongLong(g_ended); }
PyObject* ended(PyObject*, PyObject* capsule) {
    const Watch* watch = static_cast<const Watch*>(PyCapsule_GetPointer(capsule, WATCH));
    return watch ? PyBool_FromLong(watch->told && watch->ended) : nullptr;
}

// Status words of captured calls: memory that no graph's and no stream's allocations are given, zero from the start, never given back.
// new_words(device, count) -> address; take_words(device, stream, address, count) -> what they held, as a tuple; what was not zero is from then on. Both wait for the stream.
struct RelaxedCapture {                                            // (an allocation beside somebody's capture is no part of it)
    cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
    RelaxedCapture() { cudaThreadExchangeStreamCaptureMode(&mode); }
    ~RelaxedCapture() { cudaThreadExchangeStreamCaptureMode(&mode); }
};
PyObject* cuda_failed(const char* what, cudaError_t e) {
    cudaGetLastError();
    PyErr_Format(PyExc_RuntimeError, "%s: %s", what, cudaGetErrorString(e));
    return nullptr;
}
PyObject* new_words(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    const long device = nargs == 2 ? PyLong_AsLong(args[0]) : -1, count = nargs == 2 ? PyLong_AsLong(args[1]) : 0;
    if (PyErr_Occurred()) return nullptr;
    if (device < 0 || count <= 0) {
        PyErr_SetString(PyExc_ValueError, "new_words(device, count)");
        return nullptr;
    }
    int before = 0;
    cudaGetDevice(&before);
    cudaError_t e = cudaSetDevice((int)device);
    void* words = nullptr;
    cudaStream_t stream = nullptr;
    {
        const RelaxedCapture relaxed;
        if (e == cudaSuccess) e = cudaMalloc(&words, (size_t)count * 4);
        if (e == cudaSuccess) e = cudaStreamCreateWithFlags(&stream, cudaStreamNonBlocking);
        if (e == cudaSuccess) e = cudaMemsetAsync(words, 0, (size_t)count * 4, stream);
        if (e == cudaSuccess) e = cudaStreamSynchronize(stream);
        if (stream) cudaStreamDestroy(stream);
        if (e != cudaSuccess && words) cudaFree(words);
    }
    cudaSetDevice(before);
    return e == cudaSuccess ? PyLong_FromUnsignedLongLong(reinterpret_cast<W>(words)) : cuda_failed("status words", e);
}
PyObject* take_words(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    if (nargs != 4) {
        PyErr_SetString(PyExc_TypeError, "take_words(device, stream, address, count)");
        return nullptr;
    }
    const long device = PyLong_AsLong(args[0]), count = PyLong_AsLong(args[3]);
    const W stream = PyLong_AsUnsignedLongLong(args[1]), words = PyLong_AsUnsignedLongLong(args[2]);
    if (PyErr_Occurred()) return nullptr;
    int held[1024];
    const size_t n = count > 0 ? (size_t)count : 0;
    if (n > sizeof(held) / 4) {
        PyErr_SetString(PyExc_ValueError, "up to 1024 words at a time");
        return nullptr;
    }
    bool any = false;
    int before = 0;
    cudaGetDevice(&before);
    cudaError_t e = cudaSetDevice((int)device);
    Py_BEGIN_ALLOW_THREADS
    if (e == cudaSuccess) e = cudaMemcpyAsync(held, reinterpret_cast<const void*>(words), n * 4, cudaMemcpyDeviceToHost, reinterpret_cast<cudaStream_t>(stream));
    if (e == cudaSuccess) e = cudaStreamSynchronize(reinterpret_cast<cudaStream_t>(stream));
    // (only those: another one may be written meanwhile)
    for (size_t i = 0; e == cudaSuccess && i < n; ++i)
        if (held[i] != 0) {
            e = cudaMemsetAsync(reinterpret_cast<int*>(words) + i, 0, 4, reinterpret_cast<cudaStream_t>(stream));
            any = true;
        }
    if (e == cudaSuccess && any) e = cudaStreamSynchronize(reinterpret_cast<cudaStream_t>(stream));
    Py_END_ALLOW_THREADS
    cudaSetDevice(before);
    if (e != cudaSuccess) return cuda_failed("status words", e);
    PyObject* tuple = PyTuple_New((Py_ssize_t)n);
    for (size_t i = 0; tuple && i < n; ++i) PyTuple_SET_ITEM(tuple, (Py_ssize_t)i, PyLong_FromLong(held[i]));
    return tuple;
}
template <PyObject* (*F)(PyObject*, PyObject* const*, Py_ssize_t)> PyCFunction fast() { return reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(F)); }

PyMethodDef methods[] = {{"make_specs", make_specs, METH_O, "What a call's operands have to be."},
                         {"capture_id", capture_id, METH_O, "A number for the capture that a stream is part of, 0 for none."},
                         {"watch_capture", watch_capture, METH_O, "What tells when the graph that a stream is captured into is gone."},
                         {"new_words", fast<new_words>(), METH_FASTCALL, "Status words of captured calls."},
                         {"take_words", fast<take_words>(), METH_FASTCALL, "What status words hold; zero from then on."},
                         {"ended_count", ended_count, METH_NOARGS, "Watched graphs that are gone."},
                         {"ended", ended, METH_O, "Whether a watched graph and all that was instantiated from it are gone."},
                         {"call", fast<call>(), METH_FASTCALL, "Checks the operands and calls an entry point."},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_binding", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__binding() { return PyModule_Create(&module); }
