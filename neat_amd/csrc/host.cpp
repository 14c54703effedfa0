// What the C ABI takes of a list of tensors, read from the tensors themselves.
//
// A step over many small tensors is bound by the host where each is asked for its type, device, size, layout and address from
// Python: twelve questions of 30 to 50 ns, 31 us of a step over 48 tensors that the GPU does in 6.  Here they cost 30 ns a tensor
// together.  Part of the Python package alone (libneat_hip.so knows no torch): called through ctypes with the interpreter's lock
// held.  Nothing is kept from one call for the next.
#include <Python.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstdint>

// the torch and Python that this was compiled for: others lay their objects out otherwise
extern "C" const char* neat_host_for() { return NEAT_HOST_FOR; }

static bool plain(const at::Tensor& t, at::ScalarType type, int device, int64_t numel) {
    return t.defined() && t.layout() == at::kStrided && t.scalar_type() == type && t.get_device() == device && t.numel() == numel &&
           t.is_contiguous();
}

// Addresses of the tensors in the list ``params`` (p) and of their gradients (g), and the step counts ``steps`` + 1 (now): 1 if
// every tensor has a gradient and all of both are contiguous, of one type (bf16: bfloat16, else float32), on ``device`` and of the
// sizes ``numel``.  Otherwise 0, with nothing said about p, g and now: the caller finds out what the matter is.
extern "C" int neat_host_step_list(PyObject* params, int64_t count, const int64_t* numel, int bf16, int device, const int32_t* steps,
                                   uint64_t* p, uint64_t* g, int32_t* now) {
    if (!PyList_CheckExact(params) || PyList_GET_SIZE(params) != count) return 0;
    const at::ScalarType type = bf16 ? at::kBFloat16 : at::kFloat;
    try {                                               // no exception crosses the C entry
        for (int64_t i = 0; i < count; ++i) {
            PyObject* const o = PyList_GET_ITEM(params, i);
            if (!THPVariable_Check(o)) return 0;
            const at::Tensor& t = THPVariable_Unpack(o);
            if (!plain(t, type, device, numel[i])) return 0;
            const at::Tensor& d = t.grad();
            if (!plain(d, type, device, numel[i])) return 0;
            p[i] = (uint64_t)t.data_ptr();
            g[i] = (uint64_t)d.data_ptr();
            now[i] = steps[i] + 1;
        }
    } catch (...) {
        return 0;
    }
    return 1;
}

// Says to autograd that the tensors in the list ``params`` (of the kind that neat_host_step_list takes) have been written: a backward
// pass that saved one of them raises an error instead of using what is there now.
extern "C" void neat_host_written(PyObject* params) {
    if (!PyList_CheckExact(params)) return;
    const Py_ssize_t n = PyList_GET_SIZE(params);
    for (Py_ssize_t i = 0; i < n; ++i) {
        PyObject* const o = PyList_GET_ITEM(params, i);
        if (!THPVariable_Check(o)) continue;
        const at::Tensor& t = THPVariable_Unpack(o);
        if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();     // inference tensors have no version
    }
}
