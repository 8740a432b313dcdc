// What the operators' autograd nodes share (torch_ops.cpp, torch_mixer.cpp): argument helpers over torch's C++ API.
#pragma once
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>

#include "../../include/pdw.h"

namespace pdw_torch {

using at::Tensor;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;

inline int dtype_code(at::ScalarType t) {
    switch (t) {
        case at::kFloat: return PDW_F32;
        case at::kHalf: return PDW_F16;
        case at::kBFloat16: return PDW_BF16;
        default: return -1;
    }
}

inline void check(int status, const char* what) {
    TORCH_CHECK(status == 0, what, ": ", pdw_last_error(), " (status ", status, ")");
}

inline void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

// Contiguous and 16-byte aligned (the kernels move 16-byte pieces; a view at an odd storage offset is copied).
inline Tensor dense(const Tensor& t) {
    Tensor c = t.is_contiguous() ? t : t.contiguous();
    return reinterpret_cast<uintptr_t>(c.data_ptr()) % 16 == 0 ? c : c.clone(at::MemoryFormat::Contiguous);
}

// What a node keeps of an input: the input itself where it went to the kernels as it is, so that a later change of it in
// place is noticed, else the copy that they read.
inline SavedVariable save(const Tensor& in, const Tensor& read) { return SavedVariable(read.is_same(in) ? in : read, false); }

// What a node has saved, as it comes back: a saved-tensor hook may have put another tensor in its place, and the kernels
// take addresses.  (Of another type: converted.)
inline Tensor restored(const SavedVariable& v, const std::shared_ptr<torch::autograd::Node>& node, at::IntArrayRef sizes,
                at::ScalarType type, c10::Device device) {
    Tensor t = v.unpack(node);
    TORCH_CHECK(t.defined() && t.sizes() == sizes && t.device() == device, node->name(),
                ": a saved tensor came back as another one (", sizes, " on ", device, " was saved)");
    return t.scalar_type() == type ? t : t.to(type);
}

// The gradient of a node's only output; zeros where the engine has none (a later node's backward returned none), as
// torch.autograd.Function gives them, so that inputs and parameters get gradients of zero and not none.
inline Tensor output_gradient(const torch::autograd::Node& node, const variable_list& grads) {
    return grads[0].defined() ? grads[0] : node.input_metadata(0).zeros_like();
}

inline void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

inline Tensor bytes(size_t n, const Tensor& like) { return at::empty({(int64_t)n}, like.options().dtype(at::kByte)); }

// Whether a call belongs to the nodes below.  They have no forward-mode derivative and no batching rule, so such calls go
// on to the torch.autograd.Function forms, which refuse them; and a trace (torch.jit.trace) would record of them the
// allocation of the result alone, where a Function becomes a node of the graph that calls it again.
inline bool plain_call(const Tensor* in, int n) {
    if (torch::jit::tracer::isTracing()) return false;
    if (c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::FuncTorchDynamicLayerFrontMode)) return false;
    for (int i = 0; i < n; ++i)
        if (in[i].defined() && in[i]._fw_grad(0).defined()) return false;
    return true;
}

inline bool tensor_arg(PyObject* o, Tensor* t) {
    if (o == Py_None) return true;
    if (!THPVariable_Check(o)) {
        PyErr_Format(PyExc_TypeError, "expected a Tensor or None, got %s", Py_TYPE(o)->tp_name);
        return false;
    }
    *t = THPVariable_Unpack(o);
    return true;
}

}  // namespace pdw_torch
