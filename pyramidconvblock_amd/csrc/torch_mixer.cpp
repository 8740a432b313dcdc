// The host path of what goes around and beside a mixing block: channel norm, gated residual and gated scan as autograd nodes over
// libpdw.so (torch_ops.cpp has the block and the convolution, and says why they are native).
#include "torch_node.h"

#include <torch/csrc/autograd/functions/accumulate_grad.h>

namespace {

using namespace pdw_torch;

// A gradient accumulator works on the stream that its leaf first met a graph on, and lives as long as any graph of that leaf.  If that is the
// default stream, which no capture may make wait, a captured backward would end the process when the engine hands the gradient over: so it
// is refused here, before anything is handed over.  (A leaf whose gradient this pass does not ask for is handed nothing.)
void no_eager_accumulators(const torch::autograd::Node& node, c10::Device device) {
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
void no_second_derivative(const torch::autograd::Node& node) {
    TORCH_CHECK(!at::GradMode::is_enabled(), node.name(), ": no derivative of the gradient (create_graph=True)");
}

// Types and shapes are checked before devices.
void check_devices(const Tensor* in, int n) {
    for (int i = 0; i < n; ++i) {
        if (!in[i].defined()) continue;
        TORCH_CHECK(in[i].is_cuda(), "pyramid dwconv kernels run on a HIP device only (tensor is on ", in[i].device(),
                    "); there is no CPU path");
        TORCH_CHECK(in[i].device() == in[0].device(), "tensors on different devices: ", in[0].device(), " vs ", in[i].device());
    }
}

// t is of x's type
void check_like(const Tensor& x, const Tensor& t, const char* name) {
    TORCH_CHECK_TYPE(!t.defined() || t.scalar_type() == x.scalar_type(), name, " is ", t.scalar_type(), " and x ", x.scalar_type());
}

void check_param(const Tensor& x, const Tensor& t, const char* name) {
    check_like(x, t, name);
    TORCH_CHECK_VALUE(!t.defined() || (t.dim() == 1 && t.size(0) == x.size(-1)), name, " has to be [", x.size(-1), "], got ",
                      t.sizes());
}

void check_x(const Tensor& x) {
    TORCH_CHECK_TYPE(x.defined(), "x has to be a tensor");
    TORCH_CHECK_TYPE(dtype_code(x.scalar_type()) >= 0, "pyramid dwconv kernels support float32/float16/bfloat16, got ",
                     x.scalar_type());
}

void check_channels(const Tensor& x) {
    TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) >= 1 && x.size(-1) <= PDW_NORM_MAX_CHANNELS, "expected [..., C] with 1 <= C <= ",
                      PDW_NORM_MAX_CHANNELS, ", got ", x.sizes());
}

bool wants_grad(const Tensor* in, int n) {
    if (!at::GradMode::is_enabled()) return false;
    for (int i = 0; i < n; ++i)
        if (in[i].defined() && in[i].requires_grad()) return true;
    return false;
}

Tensor packed(const Tensor& t) { return !t.defined() || t.is_contiguous() ? t : t.contiguous(); }

Tensor floats(at::IntArrayRef sizes, const Tensor& like) { return at::empty(sizes, like.options().dtype(at::kFloat)); }

Tensor new_like(const Tensor& t) { return at::empty(t.sizes(), t.options()); }

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

// ---------------------------------------------------------------------------------------------------------------
// The channel norm

enum { kNX, kNWeight, kNBias, kNormInputs };

struct NormNode : public torch::autograd::Node {
    Kept x, weight, stats;
    bool has_bias;
    int kind;

    std::string name() const override { return "ChannelNormBackward"; }
    void release_variables() override {
        std::lock_guard<std::mutex> lock(mutex_);
        for (Kept* k : {&x, &weight, &stats}) k->v.reset_data();
    }

    variable_list apply(variable_list&& grads) override {
        std::lock_guard<std::mutex> lock(mutex_);
        no_second_derivative(*this);
        const Tensor grad = output_gradient(*this, grads);
        no_eager_accumulators(*this, grad.device());
        const auto self = shared_from_this();
        const auto type = grad.scalar_type();
        Tensor xs = x.get(self, type, grad.device()), w = weight.get(self, type, grad.device()),
               st = stats.get(self, at::kFloat, grad.device());
        at::AutoDispatchBelowADInplaceOrView below;
        xs = packed(xs), w = packed(w), st = packed(st);
        const Tensor gy = packed(grad);
        const c10::DeviceGuard guard(xs.device());
        const int C = (int)xs.size(-1), dt = dtype_code(type);
        const int64_t N = xs.numel() / C;
        variable_list out(kNormInputs);
        if (task_should_compute_output(kNX)) out[kNX] = new_like(xs);
        ParamGrads params;
        params.add(w.defined() && task_should_compute_output(kNWeight), {C}, &out[kNWeight]);
        params.add(has_bias && task_should_compute_output(kNBias), {C}, &out[kNBias]);
        params.make(xs.options(), N == 0);
        if (N == 0) return out;
        Tensor ws;
        if (params.any()) ws = bytes(pdw_norm_bwd_workspace_bytes(N, C, dt), xs);
        check(pdw_norm_bwd(ptr(gy), ptr(xs), ptr(w), (const float*)ptr(st), ptr(out[kNX]), ptr(out[kNWeight]), ptr(out[kNBias]), ptr(ws),
                           ws.defined() ? ws.numel() : 0, N, C, kind, dt, stream_of(xs)),
              "pdw_norm_bwd");
        return out;
    }
};

Tensor norm_forward(const Tensor* in, int kind, double eps, bool grad) {
    const c10::DeviceGuard guard(in[kNX].device());
    Tensor d[kNormInputs], y, stats;
    {
        at::AutoDispatchBelowADInplaceOrView below;
        for (int i = 0; i < kNormInputs; ++i) d[i] = packed(in[i]);
        const Tensor& x = d[kNX];
        const int C = (int)x.size(-1);
        const int64_t N = x.numel() / C;
        y = at::empty(x.sizes(), x.options());
        if (grad) stats = floats({N, 2}, x);
        if (N)
            check(pdw_norm_fwd(ptr(x), ptr(d[kNWeight]), ptr(d[kNBias]), ptr(y), (float*)ptr(stats), N, C, kind, (float)eps,
                               dtype_code(x.scalar_type()), stream_of(x)),
                  "pdw_norm_fwd");
    }
    if (grad) {
        auto node = std::shared_ptr<NormNode>(new NormNode(), torch::autograd::deleteNode);
        node->set_next_edges(torch::autograd::collect_next_edges(in[kNX], in[kNWeight], in[kNBias]));
        node->x.keep(in[kNX], d[kNX]), node->weight.keep(in[kNWeight], d[kNWeight]), node->stats.keep(stats, stats);
        node->has_bias = in[kNBias].defined(), node->kind = kind;
        torch::autograd::set_history(y, node);
    }
    return y;
}

// ---------------------------------------------------------------------------------------------------------------
// The gated residual

enum { kRX, kRY, kRGate, kRScale, kRWeight, kRBias, kRNextWeight, kRNextBias, kResidualInputs };

struct ResidualShape {
    int64_t N, P, ldgate;   // rows; rows of a gate row; elements between gate rows
    int C, act, kind, next_kind, dtype;
};

// The gate as the kernels read it: rows of C neighbouring channels, ldgate elements apart.
Tensor gate_rows(const Tensor& gate, int C, int64_t* ld) {
    *ld = C;
    if (!gate.defined() || gate.is_contiguous() || gate.numel() == 0) return gate;
    // (a slice of a wider tensor's channels, say)
    bool rows = gate.stride(-1) == 1 || C == 1;
    int64_t step = 0, next = 0;
    for (int64_t d = gate.dim() - 2; d >= 0 && rows; --d) {
        if (gate.size(d) == 1) continue;
        if (step == 0) step = next = gate.stride(d);
        rows = gate.stride(d) == next && next >= C;
        next *= gate.size(d);
    }
    if (!rows) return gate.contiguous();
    if (step) *ld = step;
    return gate;
}

struct ResidualNode : public torch::autograd::Node {
    Kept x, y, gate, scale, weight, next_weight, bias, stats, next_stats;
    ResidualShape s;
    bool has_next_bias;

    std::string name() const override { return "GatedResidualBackward"; }
    void release_variables() override {
        std::lock_guard<std::mutex> lock(mutex_);
        for (Kept* k : {&x, &y, &gate, &scale, &weight, &next_weight, &bias, &stats, &next_stats}) k->v.reset_data();
    }

    variable_list apply(variable_list&& grads) override {
        std::lock_guard<std::mutex> lock(mutex_);
        no_second_derivative(*this);
        const bool next = s.next_kind != PDW_NORM_NONE;
        Tensor gout = grads[0], gnext = next ? grads[1] : Tensor();
        // (an output that nothing was made of has a gradient of zero)
        if (!gout.defined()) gout = input_metadata(0).zeros_like();
        if (next && !gnext.defined()) gnext = input_metadata(1).zeros_like();
        const auto self = shared_from_this();
        const auto type = gout.scalar_type();
        const auto dev = gout.device();
        no_eager_accumulators(*this, dev);
        auto take = [&](const Kept& k) { return k.get(self, type, dev); };
        Tensor xv = take(x), yv = take(y), q = take(gate), sc = take(scale), w = take(weight), nw = take(next_weight), b = take(bias);
        Tensor st = stats.get(self, at::kFloat, dev), nst = next_stats.get(self, at::kFloat, dev);
        at::AutoDispatchBelowADInplaceOrView below;
        for (Tensor* t : {&xv, &yv, &sc, &w, &nw, &b, &st, &nst}) *t = packed(*t);
        q = gate_rows(q, s.C, &s.ldgate);
        const Tensor go = packed(gout), gn = packed(gnext);
        const c10::DeviceGuard guard(dev);
        const bool empty = s.N == 0;
        variable_list r(kResidualInputs);
        auto want = [&](int i) { return task_should_compute_output(i); };
        if (want(kRX)) r[kRX] = next ? new_like(yv) : gout;   // without a next norm x's gradient is out's
        if (want(kRY)) r[kRY] = new_like(yv);
        ParamGrads params;
        const bool image_gate = q.defined() && s.P > 1 && want(kRGate);
        if (q.defined() && !image_gate && want(kRGate)) r[kRGate] = at::empty(q.sizes(), yv.options());
        params.add(image_gate, q.defined() ? q.sizes() : at::IntArrayRef(), &r[kRGate]);
        params.add(sc.defined() && want(kRScale), {s.C}, &r[kRScale]);
        params.add(w.defined() && want(kRWeight), {s.C}, &r[kRWeight]);
        params.add(b.defined() && want(kRBias), {s.C}, &r[kRBias]);
        params.add(nw.defined() && want(kRNextWeight), {s.C}, &r[kRNextWeight]);
        params.add(has_next_bias && want(kRNextBias), {s.C}, &r[kRNextBias]);
        params.make(yv.options(), empty);
        if (empty) {
            if (r[kRGate].defined()) r[kRGate].zero_();
            return r;
        }
        Tensor ws;
        if (params.any()) ws = bytes(pdw_residual_bwd_workspace_bytes(s.N, s.C, s.P, s.next_kind, s.dtype), yv);
        check(pdw_residual_bwd(ptr(go), ptr(gn), ptr(xv), ptr(yv), ptr(q), ptr(sc), ptr(w), ptr(b), ptr(nw), (const float*)ptr(st),
                               (const float*)ptr(nst), next ? ptr(r[kRX]) : nullptr, ptr(r[kRY]), ptr(r[kRGate]), ptr(r[kRScale]),
                               ptr(r[kRWeight]), ptr(r[kRBias]), ptr(r[kRNextWeight]), ptr(r[kRNextBias]), ptr(ws),
                               ws.defined() ? ws.numel() : 0, s.N, s.C, s.P, s.ldgate, s.act, s.kind, s.next_kind, s.dtype, stream_of(yv)),
              "pdw_residual_bwd");
        return r;
    }
};

void residual_forward(const Tensor* in, ResidualShape s, double eps, bool grad, Tensor* out, Tensor* next) {
    const c10::DeviceGuard guard(in[kRX].device());
    const bool norm = s.kind != PDW_NORM_NONE, nnorm = s.next_kind != PDW_NORM_NONE;
    Tensor d[kResidualInputs], stats, next_stats;
    {
        at::AutoDispatchBelowADInplaceOrView below;
        for (int i = 0; i < kResidualInputs; ++i) d[i] = i == kRGate ? gate_rows(in[i], s.C, &s.ldgate) : packed(in[i]);
        const Tensor& x = d[kRX];
        *out = at::empty(x.sizes(), x.options());
        if (nnorm) *next = at::empty(x.sizes(), x.options());
        if (grad && norm) stats = floats({s.N, 2}, x);
        if (grad && nnorm) next_stats = floats({s.N, 2}, x);
        if (s.N)
            check(pdw_residual_fwd(ptr(x), ptr(d[kRY]), ptr(d[kRGate]), ptr(d[kRScale]), ptr(d[kRWeight]), ptr(d[kRBias]),
                                   ptr(d[kRNextWeight]), ptr(d[kRNextBias]), ptr(*out), ptr(*next), (float*)ptr(stats),
                                   (float*)ptr(next_stats), s.N, s.C, s.P, s.ldgate, s.act, s.kind, s.next_kind, (float)eps, s.dtype,
                                   stream_of(x)),
                  "pdw_residual_fwd");
    }
    if (grad) {
        auto node = std::shared_ptr<ResidualNode>(new ResidualNode(), torch::autograd::deleteNode);
        node->set_next_edges(torch::autograd::collect_next_edges(in[kRX], in[kRY], in[kRGate], in[kRScale], in[kRWeight], in[kRBias],
                                                                 in[kRNextWeight], in[kRNextBias]));
        auto keep = [&](Kept& k, int i) { k.keep(in[i], d[i]); };
        keep(node->y, kRY), keep(node->gate, kRGate), keep(node->scale, kRScale), keep(node->weight, kRWeight);
        keep(node->bias, kRBias), keep(node->next_weight, kRNextWeight);
        if (nnorm) keep(node->x, kRX);
        node->stats.keep(stats, stats), node->next_stats.keep(next_stats, next_stats);
        node->s = s, node->has_next_bias = in[kRNextBias].defined();
        torch::autograd::set_history(*out, node);
        if (nnorm) torch::autograd::set_history(*next, node);
    }
}

// ---------------------------------------------------------------------------------------------------------------
// The gated scan

enum { kSX, kSG, kSState, kScanInputs };

struct ScanShape {
    int64_t T;
    int O, W, I, reverse, dtype, dim;
    bool halves;   // x and g are the halves of one tensor's channels
};

// A tensor [lead..., T, mid..., channels] as [O][T][W][I]: where it lies, and the strides in elements.
struct ScanView {
    Tensor t;
    long long s[3];
};

// Strides of t's axes [first, last) as one axis; false where they are none.
bool collapse(const Tensor& t, int64_t first, int64_t last, long long* stride) {
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

ScanView scan_view(const Tensor& t, int dim) {
    ScanView v{t, {0, 0, 0}};
    const int64_t last = t.dim() - 1;
    auto read = [&](const Tensor& u) {
        v.s[1] = u.stride(dim);
        return (u.stride(last) == 1 || u.size(last) == 1) && collapse(u, 0, dim, &v.s[0]) && collapse(u, dim + 1, last, &v.s[2]);
    };
    if (t.numel() && !read(t)) {
        v.t = t.contiguous();
        read(v.t);
    }
    return v;
}

// The halves of xg's channels.
void split(const Tensor& xg, Tensor* x, Tensor* g) {
    const int64_t C = xg.size(-1) / 2;
    *x = xg.narrow(-1, 0, C), *g = xg.narrow(-1, C, C);
}

// Where the axes behind the recurrence's are dense in every tensor they are one axis of chains, [O][T][1][W * I].  Never with halves: rows
// of x and g may lie side by side (windows that overlap), but those of their gradients, halves of one dense tensor, do not.
bool mergeable(const ScanShape& s, std::initializer_list<const ScanView*> views) {
    if (s.halves || s.W == 1 || (int64_t)s.W * s.I > 0x7fffffff) return false;
    for (const ScanView* v : views)
        if (v->s[2] != s.I) return false;
    return true;
}

ScanShape merged(ScanShape s) {
    s.I *= s.W, s.W = 1;
    return s;
}

struct ScanNode : public torch::autograd::Node {
    Kept x, g, lengths, states;   // (halves: x is the whole tensor)
    ScanShape s;
    bool one_axis;   // how the forward was called: the states lie by it
    at::DimVector state_sizes;

    std::string name() const override { return "GatedScanBackward"; }
    void release_variables() override {
        std::lock_guard<std::mutex> lock(mutex_);
        for (Kept* k : {&x, &g, &lengths, &states}) k->v.reset_data();
    }

    variable_list apply(variable_list&& grads) override {
        std::lock_guard<std::mutex> lock(mutex_);
        no_second_derivative(*this);
        Tensor gy = grads[0], glast = grads[1];
        if (!gy.defined() && !glast.defined()) gy = input_metadata(0).zeros_like();
        const auto self = shared_from_this();
        const auto type = input_metadata(0).options().dtype().toScalarType();
        const auto dev = gy.defined() ? gy.device() : glast.device();
        no_eager_accumulators(*this, dev);
        Tensor xv = x.get(self, type, dev), gv = g.get(self, type, dev);
        Tensor len = lengths.get(self, at::kInt, dev), st = states.get(self, at::kFloat, dev);
        at::AutoDispatchBelowADInplaceOrView below;
        gy = packed(gy), glast = packed(glast), len = packed(len), st = packed(st);
        const c10::DeviceGuard guard(dev);
        variable_list r(kScanInputs);
        Tensor xh = xv, gh = gv, gx, gg;
        if (s.halves) {
            split(xv, &xh, &gh);
            if (task_should_compute_output(kSX)) {
                r[kSX] = at::empty(xv.sizes(), xv.options());
                split(r[kSX], &gx, &gg);
            }
        } else {
            if (task_should_compute_output(kSX)) gx = r[kSX] = at::empty(xh.sizes(), xh.options());
            if (task_should_compute_output(kSG)) gg = r[kSG] = at::empty(gh.sizes(), gh.options());
        }
        if (task_should_compute_output(kSState)) r[kSState] = floats(state_sizes, xh);
        if (s.O == 0 || s.W == 0 || s.I == 0) return r;
        ScanView vx = scan_view(xh, s.dim), vg = scan_view(gh, s.dim), vgx{gx, {0, 0, 0}}, vgg{gg, {0, 0, 0}};
        if (gx.defined()) vgx = scan_view(gx, s.dim);
        if (gg.defined()) vgg = scan_view(gg, s.dim);
        // (a saved-tensor hook may have brought x and g back in another layout)
        if (one_axis && !mergeable(s, {&vx, &vg})) vx = scan_view(xh.contiguous(), s.dim), vg = scan_view(gh.contiguous(), s.dim);
        const ScanShape m = one_axis ? merged(s) : s;
        const size_t need = pdw_scan_workspace_bytes(m.O, m.T, m.W, m.I, 1);
        Tensor ws;
        if (need) ws = bytes(need, xh);
        check(pdw_scan_bwd(ptr(gy), (const float*)ptr(glast), ptr(vx.t), ptr(vg.t), (const int*)ptr(len), (const float*)ptr(st), ptr(gx),
                           ptr(gg), (float*)ptr(r[kSState]), ptr(ws), need, m.O, m.T, m.W, m.I, vx.s, vg.s, vgx.s, vgg.s, m.reverse,
                           m.dtype, stream_of(xh)),
              "pdw_scan_bwd");
        return r;
    }
};

void scan_forward(const Tensor* in, const Tensor& lengths, const ScanShape& s, at::IntArrayRef y_sizes, at::IntArrayRef state_sizes,
                  bool grad, Tensor* y, Tensor* last) {
    const c10::DeviceGuard guard(in[kSX].device());
    Tensor states, len, h0;
    Tensor keep_x = in[kSX], keep_g = in[kSG];   // what the kernels read
    bool one_axis = false;
    {
        at::AutoDispatchBelowADInplaceOrView below;
        Tensor xh = in[kSX], gh = in[kSG];
        if (s.halves) split(in[kSX], &xh, &gh);
        ScanView vx = scan_view(xh, s.dim), vg = scan_view(gh, s.dim);
        if (s.halves) {
            if (!vx.t.is_same(xh) || !vg.t.is_same(gh)) {   // (neither half lies in rows: one copy of the whole)
                keep_x = in[kSX].contiguous();
                split(keep_x, &xh, &gh);
                vx = scan_view(xh, s.dim), vg = scan_view(gh, s.dim);
            }
        } else {
            keep_x = vx.t, keep_g = vg.t;
        }
        one_axis = mergeable(s, {&vx, &vg});
        const ScanShape m = one_axis ? merged(s) : s;
        len = packed(lengths), h0 = packed(in[kSState]);
        *y = at::empty(y_sizes, in[kSX].options());
        *last = floats(state_sizes, in[kSX]);
        if (grad) states = bytes(pdw_scan_states_bytes(m.O, m.T, m.W, m.I), *y).view(at::kFloat);
        if (m.O && m.W && m.I) {
            const size_t need = pdw_scan_workspace_bytes(m.O, m.T, m.W, m.I, 0);
            Tensor ws;
            if (need) ws = bytes(need, *y);
            check(pdw_scan_fwd(ptr(vx.t), ptr(vg.t), (const float*)ptr(h0), (const int*)ptr(len), ptr(*y), (float*)ptr(*last),
                               (float*)ptr(states), ptr(ws), need, m.O, m.T, m.W, m.I, vx.s, vg.s, m.reverse, m.dtype, stream_of(*y)),
                  "pdw_scan_fwd");
        }
    }
    if (grad) {
        auto node = std::shared_ptr<ScanNode>(new ScanNode(), torch::autograd::deleteNode);
        node->set_next_edges(torch::autograd::collect_next_edges(in[kSX], in[kSG], in[kSState]));
        node->x.keep(in[kSX], keep_x), node->g.keep(in[kSG], keep_g);
        node->lengths.keep(lengths, len), node->states.keep(states, states);
        node->s = s, node->one_axis = one_axis, node->state_sizes = state_sizes;
        torch::autograd::set_history(*y, node);
        torch::autograd::set_history(*last, node);
    }
}

// ---------------------------------------------------------------------------------------------------------------
// Python entry points

bool int_arg(PyObject* o, int64_t* v) {
    *v = PyLong_AsLong(o);
    return !PyErr_Occurred();
}

// (a code of ops.py's tables)
bool code_arg(PyObject* o, int* v) {
    int64_t n;
    if (!int_arg(o, &n)) return false;
    TORCH_CHECK_VALUE(n >= 0 && n < 3, "unknown code ", n);
    *v = (int)n;
    return true;
}

PyObject* pair(Tensor&& a, Tensor&& b) {
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

// A call's arguments, checked; false with a Python error.  (The Function forms, which a trace's replays call with other tensors, have theirs checked
// by check_norm, check_residual and check_scan.)
bool norm_args(PyObject* const* args, Py_ssize_t n, Tensor* in, int* kind, double* eps) {
    TORCH_CHECK(n == 5, "norm: 5 arguments expected");
    for (int i = 0; i < kNormInputs; ++i)
        if (!tensor_arg(args[i], &in[i])) return false;
    if (!code_arg(args[3], kind)) return false;
    *eps = PyFloat_AsDouble(args[4]);
    if (PyErr_Occurred()) return false;
    check_x(in[kNX]);
    check_channels(in[kNX]);
    TORCH_CHECK_VALUE(*eps >= 0, "eps is ", *eps);
    check_param(in[kNX], in[kNWeight], "weight"), check_param(in[kNX], in[kNBias], "bias");
    check_devices(in, kNormInputs);
    return true;
}

PyObject* py_check_norm(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    Tensor in[kNormInputs];
    int kind;
    double eps;
    if (!norm_args(args, n, in, &kind, &eps)) return nullptr;
    Py_RETURN_NONE;
    END_HANDLE_TH_ERRORS
}

// norm(x, weight, bias, kind, eps): the norm; None where ChannelNormFunction has to answer (a transform, a trace).
PyObject* py_norm(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    Tensor in[kNormInputs];
    int kind;
    double eps;
    if (!norm_args(args, n, in, &kind, &eps)) return nullptr;
    if (!plain_call(in, kNormInputs)) Py_RETURN_NONE;
    Tensor y;
    {
        pybind11::gil_scoped_release no_gil;
        y = norm_forward(in, kind, eps, wants_grad(in, kNormInputs));
    }
    return THPVariable_Wrap(std::move(y));
    END_HANDLE_TH_ERRORS
}

bool residual_args(PyObject* const* args, Py_ssize_t n, Tensor* in, ResidualShape* shape, double* eps_out) {
    ResidualShape& s = *shape;
    TORCH_CHECK(n == 12, "residual: 12 arguments expected");
    for (int i = 0; i < kResidualInputs; ++i)
        if (!tensor_arg(args[i], &in[i])) return false;
    if (!code_arg(args[8], &s.act) || !code_arg(args[9], &s.kind) || !code_arg(args[10], &s.next_kind)) return false;
    const double eps = *eps_out = PyFloat_AsDouble(args[11]);
    if (PyErr_Occurred()) return false;
    const Tensor &x = in[kRX], &gate = in[kRGate];
    check_x(x);
    check_channels(x);
    TORCH_CHECK_VALUE(eps >= 0, "eps is ", eps);
    TORCH_CHECK_TYPE(in[kRY].defined(), "y has to be a tensor");
    check_like(x, in[kRY], "y"), check_like(x, gate, "gate");
    TORCH_CHECK_VALUE(x.sizes() == in[kRY].sizes(), "x and y have to be of one shape, got ", x.sizes(), " and ", in[kRY].sizes());
    static const char* const names[] = {"x", "y", "gate", "scale", "weight", "bias", "next_weight", "next_bias"};
    for (int i = kRScale; i < kResidualInputs; ++i) check_param(x, in[i], names[i]);
    s.C = (int)x.size(-1), s.N = x.numel() / s.C, s.P = 1, s.ldgate = s.C, s.dtype = dtype_code(x.scalar_type());
    if (gate.defined() && gate.sizes() != x.sizes()) {
        TORCH_CHECK_VALUE(x.dim() >= 2 && gate.dim() == 2 && gate.size(0) == x.size(0) && gate.size(1) == s.C,
                          "gate has to be of x's shape or [", x.dim() >= 2 ? x.size(0) : 1, ", ", s.C, "], got ", gate.sizes());
        s.P = s.N ? s.N / x.size(0) : 1;   // (1: every row has a gate row of its own after all)
    }
    check_devices(in, kResidualInputs);
    return true;
}

PyObject* py_check_residual(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    Tensor in[kResidualInputs];
    ResidualShape s;
    double eps;
    if (!residual_args(args, n, in, &s, &eps)) return nullptr;
    Py_RETURN_NONE;
    END_HANDLE_TH_ERRORS
}

// residual(x, y, gate, scale, weight, bias, next_weight, next_bias, act, kind, next_kind, eps): out, or (out, next); None where
// GatedResidualFunction has to answer.
PyObject* py_residual(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    Tensor in[kResidualInputs];
    ResidualShape s;
    double eps;
    if (!residual_args(args, n, in, &s, &eps)) return nullptr;
    if (!plain_call(in, kResidualInputs)) Py_RETURN_NONE;
    Tensor out, next;
    {
        pybind11::gil_scoped_release no_gil;
        residual_forward(in, s, eps, wants_grad(in, kResidualInputs), &out, &next);
    }
    if (!next.defined()) return THPVariable_Wrap(std::move(out));
    return pair(std::move(out), std::move(next));
    END_HANDLE_TH_ERRORS
}

// (x, g, the state; lengths; the result's sizes and the state's)
struct ScanArguments {
    Tensor in[kScanInputs], lengths;
    ScanShape s;
    at::DimVector y_sizes, state_sizes;
};

bool scan_args(PyObject* const* args, Py_ssize_t n, ScanArguments* a) {
    Tensor(&in)[kScanInputs] = a->in;
    Tensor& lengths = a->lengths;
    ScanShape& s = a->s;
    at::DimVector &y_sizes = a->y_sizes, &state_sizes = a->state_sizes;
    TORCH_CHECK(n == 6, "scan: 6 arguments expected");
    for (int i = 0; i < kScanInputs; ++i)
        if (!tensor_arg(args[i], &in[i])) return false;
    if (!tensor_arg(args[3], &lengths)) return false;
    int64_t dim;
    if (!int_arg(args[4], &dim)) return false;
    s.reverse = PyObject_IsTrue(args[5]);
    if (s.reverse < 0) return false;
    const Tensor& x = in[kSX];
    check_x(x);
    s.halves = !in[kSG].defined(), s.dtype = dtype_code(x.scalar_type());
    const int64_t rank = x.dim();
    TORCH_CHECK_VALUE(rank >= 2, "expected [..., T, ..., C], got ", x.sizes());
    TORCH_CHECK_INDEX(dim >= -rank && dim < rank, "dim ", dim, " of a tensor of ", rank, " dimensions");
    if (dim < 0) dim += rank;
    TORCH_CHECK_VALUE(dim != rank - 1, "the recurrence runs along any dimension but the channels' (", x.sizes(), ", dim ", dim, ")");
    if (s.halves) {
        TORCH_CHECK_VALUE(x.size(-1) % 2 == 0, "without g, x holds both in halves of its channels: an even number, got ", x.size(-1));
    } else {
        check_like(x, in[kSG], "g");
        TORCH_CHECK_VALUE(in[kSG].sizes() == x.sizes(), "x and g have to be of one shape, got ", x.sizes(), " and ", in[kSG].sizes());
    }
    y_sizes = at::DimVector(x.sizes());
    if (s.halves) y_sizes.back() /= 2;
    int64_t O = 1, W = 1;
    for (int64_t d = 0; d < rank; ++d) {
        if (d != dim) state_sizes.push_back(y_sizes[d]);
        if (d < dim) O *= y_sizes[d];
        else if (d > dim && d < rank - 1) W *= y_sizes[d];
    }
    TORCH_CHECK_VALUE(O <= 0x7fffffff && W <= 0x7fffffff && O * W <= 0x7fffffff && y_sizes.back() <= 0x7fffffff && y_sizes[dim] <= 0x7fffffff,
                      "more than 2^31 - 1 chains, channels or steps: ", x.sizes());
    s.O = (int)O, s.T = y_sizes[dim], s.W = (int)W, s.I = (int)y_sizes.back(), s.dim = (int)dim;
    const Tensor& state = in[kSState];
    if (state.defined()) {
        TORCH_CHECK_TYPE(state.scalar_type() == at::kFloat, "state is float32, got ", state.scalar_type());
        TORCH_CHECK_VALUE(state.sizes() == at::IntArrayRef(state_sizes), "state has to be ", at::IntArrayRef(state_sizes), ", got ",
                          state.sizes());
    }
    if (lengths.defined()) {
        TORCH_CHECK_TYPE(lengths.scalar_type() == at::kInt, "lengths is int32, got ", lengths.scalar_type());
        TORCH_CHECK_VALUE(lengths.sizes() == x.sizes().slice(0, dim), "lengths has to be ", x.sizes().slice(0, dim), ", got ",
                          lengths.sizes());
    }
    const Tensor all[] = {x, in[kSG], state, lengths};
    check_devices(all, 4);
    return true;
}

PyObject* py_check_scan(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    ScanArguments a;
    if (!scan_args(args, n, &a)) return nullptr;
    Py_RETURN_NONE;
    END_HANDLE_TH_ERRORS
}

// scan(x, g, state, lengths, dim, reverse): (y, last); None where GatedScanFunction has to answer.  g None: x holds both, in halves.
PyObject* py_scan(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    ScanArguments a;
    if (!scan_args(args, n, &a)) return nullptr;
    if (!plain_call(a.in, kScanInputs)) Py_RETURN_NONE;
    Tensor y, last;
    {
        pybind11::gil_scoped_release no_gil;
        scan_forward(a.in, a.lengths, a.s, a.y_sizes, a.state_sizes, wants_grad(a.in, kScanInputs), &y, &last);
    }
    return pair(std::move(y), std::move(last));
    END_HANDLE_TH_ERRORS
}

// Whether a tensor that is written may change what another call's elements are read from: they share memory, and not element by element.
bool overlap(const Tensor& read, const Tensor& written) {
    if (!read.defined() || read.numel() == 0) return false;
    int64_t last = 0;
    for (int64_t d = 0; d < read.dim(); ++d) last += (read.size(d) - 1) * read.stride(d);
    const char *p = (const char*)read.data_ptr(), *q = (const char*)written.data_ptr();
    const bool same = p == q && read.is_contiguous() && read.scalar_type() == written.scalar_type() && read.sizes() == written.sizes();
    return !same && p < q + written.nbytes() && q < p + (last + 1) * (int64_t)read.element_size();
}

// scan_step(x, g, state, new_state): y; new_state (or state in place, None) is written.
PyObject* py_scan_step(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    TORCH_CHECK(n == 4, "scan_step: 4 arguments expected");
    Tensor x, g, state, to;
    if (!tensor_arg(args[0], &x) || !tensor_arg(args[1], &g) || !tensor_arg(args[2], &state) || !tensor_arg(args[3], &to)) return nullptr;
    check_x(x);
    TORCH_CHECK_TYPE(state.defined(), "state has to be a tensor");
    TORCH_CHECK_VALUE(x.dim() >= 1, "expected [..., C]");
    const bool halves = !g.defined();
    if (halves) TORCH_CHECK_VALUE(x.size(-1) % 2 == 0, "without g, x holds both in halves of its channels: an even number, got ", x.size(-1));
    check_like(x, g, "g");
    TORCH_CHECK_VALUE(halves || g.sizes() == x.sizes(), "x and g have to be of one shape, got ", x.sizes(), " and ", g.sizes());
    at::DimVector sizes(x.sizes());
    if (halves) sizes.back() /= 2;
    TORCH_CHECK_VALUE(sizes.back() <= 0x7fffffff, "more than 2^31 - 1 channels: ", x.sizes());
    for (const Tensor* t : {&state, &to}) {
        if (!t->defined()) continue;
        TORCH_CHECK_TYPE(t->scalar_type() == at::kFloat, "the state is float32, got ", t->scalar_type());
        TORCH_CHECK_VALUE(t->sizes() == at::IntArrayRef(sizes) && t->is_contiguous(), "the state has to be dense and ",
                          at::IntArrayRef(sizes), ", got ", t->sizes());
    }
    const Tensor into = to.defined() ? to : state;
    TORCH_CHECK_VALUE(!overlap(state, into) && !overlap(x, into) && !overlap(g, into),
                      to.defined() ? "new_state" : "state", " overlaps what is read beside it");
    const Tensor all[] = {x, g, state, into};
    check_devices(all, 4);
    TORCH_CHECK(!wants_grad(all, 4), "gated_scan_step has no gradient: call it under torch.no_grad(), or gated_scan");
    TORCH_CHECK(plain_call(all, 4), "gated_scan_step takes part in no transform or trace");
    Tensor y;
    {
        pybind11::gil_scoped_release no_gil;
        const c10::DeviceGuard guard(x.device());
        at::AutoDispatchBelowADInplaceOrView below;
        const int C = (int)sizes.back();
        Tensor xh = x, gh = g;
        if (halves) split(x, &xh, &gh);
        int64_t ldx, ldg;
        xh = gate_rows(xh, C, &ldx), gh = gate_rows(gh, C, &ldg);
        y = at::empty(sizes, x.options());
        if (y.numel())
            check(pdw_scan_step(ptr(xh), ptr(gh), (const float*)ptr(state), (float*)ptr(into), ptr(y), y.numel() / C, C, ldx, ldg,
                                dtype_code(x.scalar_type()), stream_of(x)),
                  "pdw_scan_step");
        if (!into.is_inference()) into.unsafeGetTensorImpl()->bump_version();
    }
    return THPVariable_Wrap(std::move(y));
    END_HANDLE_TH_ERRORS
}

PyMethodDef kMixerMethods[] = {
    {"check_norm", (PyCFunction)(void (*)(void))py_check_norm, METH_FASTCALL, nullptr},
    {"check_residual", (PyCFunction)(void (*)(void))py_check_residual, METH_FASTCALL, nullptr},
    {"check_scan", (PyCFunction)(void (*)(void))py_check_scan, METH_FASTCALL, nullptr},
    {"norm", (PyCFunction)(void (*)(void))py_norm, METH_FASTCALL, nullptr},
    {"residual", (PyCFunction)(void (*)(void))py_residual, METH_FASTCALL, nullptr},
    {"scan", (PyCFunction)(void (*)(void))py_scan, METH_FASTCALL, nullptr},
    {"scan_step", (PyCFunction)(void (*)(void))py_scan_step, METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};

}  // namespace

PyMethodDef* pdw_mixer_methods() { return kMixerMethods; }
