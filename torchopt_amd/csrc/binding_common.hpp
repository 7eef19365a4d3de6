// What the bindings of the extension module share: dtype codes, layout checks, device and stream
// of a call, and the conversion of Python lists.
#pragma once

#include <c10/hip/HIPStream.h>
#include <hip/hip_runtime_api.h>
#include <pybind11/stl.h>
#include <torch/extension.h>

#include <string>
#include <vector>

#include "toa_adam.h"

namespace toa_binding {

namespace py = pybind11;
using at::Tensor;
using TensorList = std::vector<Tensor>;

inline int dtypeCode(const Tensor &t, const char *name) {
    switch (t.scalar_type()) {
        case at::kFloat: return TOA_F32;
        case at::kDouble: return TOA_F64;
        case at::kHalf: return TOA_F16;
        case at::kBFloat16: return TOA_BF16;
        default:
            // wording of ATen's dispatch failure, which is what the reference raises
            TORCH_CHECK(false, "\"", name, "\" not implemented for '", t.scalar_type(), "'");
    }
}

inline void requireDense(const char *name, const char *what, const Tensor &t) {
    TORCH_CHECK(t.is_non_overlapping_and_dense(), name, ": `", what,
                "` must be contiguous (non-overlapping and dense), got sizes ", t.sizes(),
                " strides ", t.strides());
}

inline bool sameLayout(const Tensor &a, const Tensor &b) {
    return a.numel() <= 1 || a.strides() == b.strides();
}

// A read-only operand in the memory order of `donor`, copying only if it is not already.
// (The reference makes incoming gradients .contiguous(), adam_op.cpp:107,123,143.)
inline Tensor asLayoutOf(const Tensor &x, const Tensor &donor) {
    if (x.numel() <= 1 || (x.is_contiguous() && donor.is_contiguous())) return x;
    // a wrong device or dtype is the gate's to report, not to be papered over by a copy
    if (x.device() != donor.device() || x.scalar_type() != donor.scalar_type()) return x;
    if (x.sizes() == donor.sizes())
        return x.strides() == donor.strides() ? x : at::empty_like(donor).copy_(x);
    TORCH_CHECK(donor.is_contiguous(), "operands of different shapes must be contiguous");
    return x.contiguous();
}

// Makes the tensors' device current for the launch (the C ABI uses the current device) and
// hands out PyTorch's current stream on it.
class OnDeviceOf {
  public:
    explicit OnDeviceOf(const Tensor &t) : index_((int)t.get_device()) {
        if (hipGetDevice(&prev_) != hipSuccess) prev_ = index_;
        if (prev_ != index_) TORCH_CHECK(hipSetDevice(index_) == hipSuccess, "hipSetDevice failed");
    }
    ~OnDeviceOf() {
        if (prev_ != index_) (void)hipSetDevice(prev_);
    }
    void *stream() const {
        return (void *)c10::hip::getCurrentHIPStream((c10::DeviceIndex)index_).stream();
    }

  private:
    int index_;
    int prev_ = 0;
};

// A Python list or tuple of tensors -> TensorList without the generic sequence caster (which
// costs ~40 ns per element; long lists of small tensors are bound by exactly this).
inline TensorList toTensorList(const py::object &o, const char *what) {
    PyObject *seq = o.ptr();
    const bool is_list = PyList_Check(seq);
    if (!is_list && !PyTuple_Check(seq)) return o.cast<TensorList>();
    const Py_ssize_t num = is_list ? PyList_GET_SIZE(seq) : PyTuple_GET_SIZE(seq);
    TensorList out;
    out.reserve((size_t)num);
    for (Py_ssize_t k = 0; k < num; ++k) {
        PyObject *item = is_list ? PyList_GET_ITEM(seq, k) : PyTuple_GET_ITEM(seq, k);
        if (!THPVariable_Check(item))
            throw py::type_error(std::string(what) + ": expected a list of tensors");
        out.push_back(THPVariable_Unpack(item));
    }
    return out;
}

}  // namespace toa_binding
