// Arguments, gradients and what autograd nodes keep, of the operators around and beside a mixing block (torch_mixer.cpp, torch_delta.cpp).
#pragma once
#include "torch_node.h"

#include <torch/csrc/autograd/functions/accumulate_grad.h>

namespace pdw_torch {

// A gradient accumulator works on the stream that its leaf first met a graph on, and lives as long as any graph of that leaf.  If that is the
// default stream, which no capture may make wait, a captured backward would end the process when the engine hands the gradient over: so it
// is refused here, before anything is handed over.  (A leaf whose gradient this pass does not ask for is handed nothing.)
inline void no_eager_accumulators(const torch::autograd::Node& node, c10::Device device) {
    const auto current = c10::hip::getCurrentHIPStream(device.index());
    const auto eager = c10::hip::getDefaultHIPStream(device.index());
    if (current == eager) return;
    hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
    if (hipStreamIsCapturing(current.stream(), &status) != hipSuccess || status == hipStreamCaptureStatusNone) return;
    for (size_t i = 0; i < node.num_outputs(); ++i) {
        const auto& edge = node.next_edge(i);
        if (!node.task_should_compute_output(i) || !dynamic_cast<torch::autograd::AccumulateGrad*>(edge.function.get())) continue;
        const auto stream = edge.function->stream();
        TORCH_CHECK(!stream || stream->id() != eager.id(), node.name(), ": this backward pass cannot be captured while an output of an eager pass "
                    "over the same tensors lives, whose gradients go to the default stream: drop that output first");
    }
}

// Neither node has a second derivative: its gradients are results of kernels, which a graph of the backward would take for
// constants.
inline void no_second_derivative(const torch::autograd::Node& node) {
    TORCH_CHECK(!at::GradMode::is_enabled(), node.name(), ": no derivative of the gradient (create_graph=True)");
}

// Types and shapes are checked before devices.
inline void check_devices(const Tensor* in, int n) {
    for (int i = 0; i < n; ++i) {
        if (!in[i].defined()) continue;
        TORCH_CHECK(in[i].is_cuda(), "pyramid dwconv kernels run on a HIP device only (tensor is on ", in[i].device(),
                    "); there is no CPU path");
        TORCH_CHECK(in[i].device() == in[0].device(), "tensors on different devices: ", in[0].device(), " vs ", in[i].device());
    }
}

// t is of x's type
inline void check_like(const Tensor& x, const Tensor& t, const char* name) {
    TORCH_CHECK_TYPE(!t.defined() || t.scalar_type() == x.scalar_type(), name, " is ", t.scalar_type(), " and x ", x.scalar_type());
}

inline void check_param(const Tensor& x, const Tensor& t, const char* name) {
    check_like(x, t, name);
    TORCH_CHECK_VALUE(!t.defined() || (t.dim() == 1 && t.size(0) == x.size(-1)), name, " has to be [", x.size(-1), "], got ",
                      t.sizes());
}

inline void check_x(const Tensor& x) {
    TORCH_CHECK_TYPE(x.defined(), "x has to be a tensor");
    TORCH_CHECK_TYPE(dtype_code(x.scalar_type()) >= 0, "pyramid dwconv kernels support float32/float16/bfloat16, got ",
                     x.scalar_type());
}

inline void check_channels(const Tensor& x) {
    TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) >= 1 && x.size(-1) <= PDW_NORM_MAX_CHANNELS, "expected [..., C] with 1 <= C <= ",
                      PDW_NORM_MAX_CHANNELS, ", got ", x.sizes());
}

inline bool wants_grad(const Tensor* in, int n) {
    if (!at::GradMode::is_enabled()) return false;
    for (int i = 0; i < n; ++i)
        if (in[i].defined() && in[i].requires_grad()) return true;
    return false;
}

inline Tensor packed(const Tensor& t) { return !t.defined() || t.is_contiguous() ? t : t.contiguous(); }

inline Tensor floats(at::IntArrayRef sizes, const Tensor& like) { return at::empty(sizes, like.options().dtype(at::kFloat)); }

inline Tensor new_like(const Tensor& t) { return at::empty(t.sizes(), t.options()); }

// The gradients of a call's parameters, as pieces of one allocation of 64-byte multiples: an allocation each is 1.4 us on the backward's
// thread (a gated residual's backward with seven gradients: 75 us of host time, this way 69).
class ParamGrads {
  public:
    // Wants a gradient like t (of these sizes) in *to, unless there is no t.
    void add(bool want, at::IntArrayRef sizes, Tensor* to) {
        if (!want) return;
        parts_.push_back({sizes.vec(), total_, to});
        int64_t n = 1;
        for (int64_t e : sizes) n *= e;
        total_ += (n + 31) / 32 * 32;
    }
    // Makes them (zeros for a call without rows).
    void make(const at::TensorOptions& options, bool zero) {
        if (parts_.empty()) return;
        const Tensor all = zero ? at::zeros({total_}, options) : at::empty({total_}, options);
        for (const Part& q : parts_) {
            *q.to = at::detail::make_tensor<c10::TensorImpl>(c10::TensorImpl::VIEW, c10::Storage(all.storage()), all.key_set(), all.dtype());
            q.to->unsafeGetTensorImpl()->set_storage_offset(q.offset);
            q.to->unsafeGetTensorImpl()->set_sizes_contiguous(q.sizes);
        }
    }
    bool any() const { return !parts_.empty(); }

  private:
    struct Part {
        std::vector<int64_t> sizes;
        int64_t offset;
        Tensor* to;
    };
    std::vector<Part> parts_;
    int64_t total_ = 0;
};

// What a node keeps: the input, and its sizes.
struct Kept {
    SavedVariable v;
    at::DimVector sizes;
    bool there = false;
    void keep(const Tensor& in, const Tensor& read) {
        if (!read.defined()) return;
        v = save(in, read), sizes = read.sizes(), there = true;
    }
    Tensor get(const std::shared_ptr<torch::autograd::Node>& node, at::ScalarType type, c10::Device device) const {
        return there ? restored(v, node, sizes, type, device) : Tensor();
    }
};

// Strides of t's axes [first, last) as one axis; false where they are none.
inline bool collapse(const Tensor& t, int64_t first, int64_t last, long long* stride) {
    bool any = false;
    int64_t next = 0;
    *stride = 0;
    for (int64_t d = last - 1; d >= first; --d) {
        if (t.size(d) == 1) continue;
        if (!any) *stride = next = t.stride(d), any = true;
        if (t.stride(d) != next) return false;
        next *= t.size(d);
    }
    return true;
}

// Whether a tensor that is written may change what another call's elements are read from: they share memory, and not element by element.
inline bool overlap(const Tensor& read, const Tensor& written) {
    if (!read.defined() || read.numel() == 0) return false;
    int64_t last = 0;
    for (int64_t d = 0; d < read.dim(); ++d) last += (read.size(d) - 1) * read.stride(d);
    const char *p = (const char*)read.data_ptr(), *q = (const char*)written.data_ptr();
    const bool same = p == q && read.is_contiguous() && read.scalar_type() == written.scalar_type() && read.sizes() == written.sizes();
    return !same && p < q + written.nbytes() && q < p + (last + 1) * (int64_t)read.element_size();
}

inline bool int_arg(PyObject* o, int64_t* v) {
    *v = PyLong_AsLong(o);
    return !PyErr_Occurred();
}

// (a code of ops.py's tables)
inline bool code_arg(PyObject* o, int* v) {
    int64_t n;
    if (!int_arg(o, &n)) return false;
    TORCH_CHECK_VALUE(n >= 0 && n < 3, "unknown code ", n);
    *v = (int)n;
    return true;
}

inline PyObject* pair(Tensor&& a, Tensor&& b) {
    PyObject* x = THPVariable_Wrap(std::move(a));
    if (!x) return nullptr;
    PyObject* y = THPVariable_Wrap(std::move(b));
    if (!y) {
        Py_DECREF(x);
        return nullptr;
    }
    PyObject* t = PyTuple_Pack(2, x, y);
    Py_DECREF(x), Py_DECREF(y);
    return t;
}

}  // namespace pdw_torch
