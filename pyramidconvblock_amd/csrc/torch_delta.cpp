// The host path of head norms with rotated positions and of the gated delta rule, as autograd nodes over libpdw.so (as torch_mixer.cpp).
#include "torch_args.h"

namespace {

using namespace pdw_torch;

// ---------------------------------------------------------------------------------------------------------------
// Head norms with rotated positions

enum { kHQ, kHK, kHWeight, kHKeyWeight, kHPositions, kHFrequencies, kRotaryInputs };

struct RotaryCall {
    Tensor in[kRotaryInputs];
    pdw_rotary c;   // but for addresses and strides
};

// A tensor [tokens.., heads, d] where its tokens have one stride and its channels lie side by side, else a copy.
Tensor head_view(const Tensor& t, long long* xt, long long* xh) {
    auto read = [&](const Tensor& u) {
        const int64_t h = u.dim() - 2;
        *xh = u.stride(h);
        return (u.stride(h + 1) == 1 || u.size(h + 1) == 1) && collapse(u, 0, h, xt);
    };
    *xt = *xh = 0;
    if (t.numel() == 0 || read(t)) return t;
    const Tensor c = t.contiguous();
    read(c);
    return c;
}

struct RotaryNode : public torch::autograd::Node {
    Kept x[2], w[2], positions, frequencies;
    pdw_rotary c;
    at::DimVector sizes[2];

    std::string name() const override { return "HeadRotaryBackward"; }
    void release_variables() override {
        std::lock_guard<std::mutex> lock(mutex_);
        for (Kept* k : {&x[0], &x[1], &w[0], &w[1], &positions, &frequencies}) k->v.reset_data();
    }

    variable_list apply(variable_list&& grads) override {
        std::lock_guard<std::mutex> lock(mutex_);
        no_second_derivative(*this);
        const auto options = input_metadata(0).options();
        const auto type = options.dtype().toScalarType();
        const auto dev = options.device();
        no_eager_accumulators(*this, dev);
        const auto self = shared_from_this();
        static const at::ScalarType kinds[] = {at::kInt, at::kInt, at::kLong, at::kFloat};
        Tensor xs[2], ws[2], pos = positions.get(self, kinds[c.position_type], dev), freq = frequencies.get(self, at::kFloat, dev);
        for (int s = 0; s < 2; ++s) xs[s] = x[s].get(self, type, dev), ws[s] = w[s].get(self, type, dev);
        at::AutoDispatchBelowADInplaceOrView below;
        const c10::DeviceGuard guard(dev);
        variable_list out(kRotaryInputs);
        pdw_rotary call = c;
        Tensor gy[2], gw[2];
        ParamGrads params;
        for (int s = 0; s < 2; ++s) {
            const bool want = c.heads[s] && task_should_compute_output(kHQ + s);
            ws[s] = packed(ws[s]), call.weight[s] = ptr(ws[s]);
            params.add(ws[s].defined() && task_should_compute_output(kHWeight + s), {c.d}, &out[kHWeight + s]);
            if (want) out[kHQ + s] = at::empty(sizes[s], options);
            if (!want && !(ws[s].defined() && task_should_compute_output(kHWeight + s))) call.heads[s] = 0;
            if (!call.heads[s]) continue;
            gy[s] = grads.size() > (size_t)s && grads[s].defined() ? packed(grads[s]) : at::zeros(sizes[s], options);
            if (xs[s].defined()) xs[s] = head_view(xs[s], &call.xt[s], &call.xh[s]);
            // (without a norm the input itself is not read)
            call.x[s] = xs[s].defined() ? ptr(xs[s]) : ptr(gy[s]);
        }
        const bool none = c.tokens == 0 || (call.heads[0] == 0 && call.heads[1] == 0);
        params.make(options, none);
        if (none) return out;
        pos = packed(pos), freq = packed(freq);
        call.positions = ptr(pos), call.frequencies = (const float*)ptr(freq);
        Tensor work;
        if (params.any()) work = at::empty({(int64_t)pdw_rotary_bwd_workspace_bytes(c.d)}, options.dtype(at::kByte));
        const void* const gys[2] = {ptr(gy[0]), ptr(gy[1])};
        void* const gxs[2] = {ptr(out[kHQ]), ptr(out[kHK])};
        void* const gws[2] = {ptr(out[kHWeight]), ptr(out[kHKeyWeight])};
        check(pdw_rotary_bwd(&call, gys, gxs, gws, ptr(work), work.defined() ? work.numel() : 0,
                             c10::hip::getCurrentHIPStream(dev.index()).stream()),
              "pdw_rotary_bwd");
        return out;
    }
};

void rotary_forward(const RotaryCall& a, bool grad, Tensor* y) {
    const Tensor(&in)[kRotaryInputs] = a.in;
    const c10::DeviceGuard guard(in[kHQ].device());
    pdw_rotary c = a.c;
    Tensor x[2], w[2], pos, freq;
    {
        at::AutoDispatchBelowADInplaceOrView below;
        for (int s = 0; s < 2; ++s) {
            if (!in[kHQ + s].defined()) continue;
            x[s] = head_view(in[kHQ + s], &c.xt[s], &c.xh[s]), w[s] = packed(in[kHWeight + s]);
            c.x[s] = ptr(x[s]), c.weight[s] = ptr(w[s]);
            y[s] = at::empty(in[kHQ + s].sizes(), in[kHQ].options());
        }
        pos = packed(in[kHPositions]), freq = packed(in[kHFrequencies]);
        c.positions = ptr(pos), c.frequencies = (const float*)ptr(freq);
        void* const ys[2] = {ptr(y[0]), ptr(y[1])};
        check(pdw_rotary_fwd(&c, ys, stream_of(in[kHQ])), "pdw_rotary_fwd");
    }
    if (!grad) return;
    auto node = std::shared_ptr<RotaryNode>(new RotaryNode(), torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(in[kHQ], in[kHK], in[kHWeight], in[kHKeyWeight], in[kHPositions], in[kHFrequencies]));
    for (int s = 0; s < 2; ++s) {
        if (!in[kHQ + s].defined()) continue;
        if (c.kind != PDW_HEAD_NONE) node->x[s].keep(in[kHQ + s], x[s]);
        node->w[s].keep(in[kHWeight + s], w[s]);
        node->sizes[s] = in[kHQ + s].sizes();
    }
    node->positions.keep(in[kHPositions], pos), node->frequencies.keep(in[kHFrequencies], freq);
    node->c = a.c;
    for (int s = 0; s < 2; ++s)
        if (y[s].defined()) torch::autograd::set_history(y[s], node);
}

// (q, k, weight, key_weight, positions, frequencies, axes, sections, base, kind, neighbours, eps)
bool rotary_args(PyObject* const* args, Py_ssize_t n, RotaryCall* a) {
    TORCH_CHECK(n == 12, "rotary: 12 arguments expected");
    Tensor(&in)[kRotaryInputs] = a->in;
    pdw_rotary& c = a->c;
    c = pdw_rotary{};
    for (int i = 0; i < kRotaryInputs; ++i)
        if (!tensor_arg(args[i], &in[i])) return false;
    int64_t axes;
    if (!int_arg(args[6], &axes)) return false;
    const Tensor &q = in[kHQ], &k = in[kHK], &pos = in[kHPositions], &freq = in[kHFrequencies];
    TORCH_CHECK_TYPE(q.defined(), "q has to be a tensor");
    TORCH_CHECK_TYPE(dtype_code(q.scalar_type()) >= 0, "pyramid dwconv kernels support float32/float16/bfloat16, got ", q.scalar_type());
    TORCH_CHECK_VALUE(axes >= 1 && axes <= 3, "axes has to be 1, 2 or 3, got ", axes);
    const int64_t rank = q.dim();
    TORCH_CHECK_VALUE(rank >= 2 && q.size(-1) >= 1 && q.size(-1) <= PDW_HEAD_MAX_CHANNELS, "expected [..., heads, d] with 1 <= d <= ",
                      PDW_HEAD_MAX_CHANNELS, ", got ", q.sizes());
    c.d = (int)q.size(-1), c.axes = (int)axes, c.dtype = dtype_code(q.scalar_type());
    const auto lead = q.sizes().slice(0, rank - 2);
    c.tokens = 1;
    for (int64_t e : lead) c.tokens *= e;
    if (k.defined()) {
        TORCH_CHECK_TYPE(k.scalar_type() == q.scalar_type(), "k is ", k.scalar_type(), " and q ", q.scalar_type());
        TORCH_CHECK_VALUE(k.dim() == rank && k.sizes().slice(0, rank - 2) == lead && k.size(-1) == c.d,
                          "q and k have to be alike but for their heads, got ", q.sizes(), " and ", k.sizes());
    }
    TORCH_CHECK_VALUE(q.size(-2) <= 65536 && (!k.defined() || k.size(-2) <= 65536), "more than 65536 heads: ", q.sizes());
    c.heads[0] = (int)q.size(-2), c.heads[1] = k.defined() ? (int)k.size(-2) : 0;
    TORCH_CHECK_TYPE(PyTuple_Check(args[7]) && PyTuple_GET_SIZE(args[7]) == axes, "sections has to be a tuple of ", axes, " numbers of pairs");
    int64_t P = 0;
    for (int64_t i = 0; i < axes; ++i) {
        int64_t v;
        if (!int_arg(PyTuple_GET_ITEM(args[7], i), &v)) return false;
        TORCH_CHECK_VALUE(v >= 0 && v <= c.d, "section ", i, " has ", v, " pairs, a head ", c.d, " channels");
        c.sections[i] = (int)v, P += v;
    }
    TORCH_CHECK_VALUE(2 * P <= c.d, "sections of ", P, " pairs, a head has ", c.d, " channels");
    c.base = PyFloat_AsDouble(args[8]);
    if (PyErr_Occurred()) return false;
    TORCH_CHECK_VALUE(c.base > 0, "base is ", c.base);
    if (!code_arg(args[9], &c.kind)) return false;
    c.neighbours = PyObject_IsTrue(args[10]);
    if (c.neighbours < 0) return false;
    const double eps = PyFloat_AsDouble(args[11]);
    if (PyErr_Occurred()) return false;
    TORCH_CHECK_VALUE(eps >= 0, "eps is ", eps);
    c.eps = (float)eps;
    static const char* const names[] = {"weight", "key_weight"};
    for (int s = 0; s < 2; ++s) {
        const Tensor& w = in[kHWeight + s];
        if (!w.defined()) continue;
        TORCH_CHECK_VALUE(c.kind != PDW_HEAD_NONE, names[s], " without a norm");
        TORCH_CHECK_VALUE(s == 0 || k.defined(), "key_weight without k");
        check_param(q, w, names[s]);
    }
    if (pos.defined()) {
        c.position_type = pos.scalar_type() == at::kInt     ? PDW_POSITIONS_I32
                          : pos.scalar_type() == at::kLong  ? PDW_POSITIONS_I64
                          : pos.scalar_type() == at::kFloat ? PDW_POSITIONS_F32
                                                            : -1;
        TORCH_CHECK_TYPE(c.position_type > 0, "positions are int32, int64 or float32, got ", pos.scalar_type());
        const int64_t m = pos.dim() - 1;
        TORCH_CHECK_VALUE(m >= 0 && m <= rank - 2 && pos.size(-1) == axes && pos.sizes().slice(0, m) == lead.slice(lead.size() - m),
                          "positions have to be ", lead, " or its last dimensions, and ", axes, " axes; got ", pos.sizes());
        TORCH_CHECK(!pos.requires_grad(), "positions have no gradient");
        c.positions_rows = pos.numel() / axes;
    } else {
        TORCH_CHECK_VALUE(rank - 2 >= axes, "without positions the ", axes, " dimensions before the heads are the grid, got ", q.sizes());
        for (int64_t i = 0; i < axes; ++i) {
            const int64_t e = lead[rank - 2 - axes + i];
            TORCH_CHECK_VALUE(e <= 0x7fffffff, "more than 2^31 - 1 places along an axis: ", q.sizes());
            c.grid[i] = (int)e;
        }
    }
    if (freq.defined()) {
        TORCH_CHECK_TYPE(freq.scalar_type() == at::kFloat, "frequencies are float32, got ", freq.scalar_type());
        TORCH_CHECK_VALUE(freq.dim() == 1 && freq.size(0) == P, "frequencies have to be [", P, "], got ", freq.sizes());
        TORCH_CHECK(!freq.requires_grad(), "frequencies have no gradient");
    }
    check_devices(in, kRotaryInputs);
    return true;
}

PyObject* py_check_rotary(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    RotaryCall a;
    if (!rotary_args(args, n, &a)) return nullptr;
    Py_RETURN_NONE;
    END_HANDLE_TH_ERRORS
}

PyObject* one_or_pair(Tensor* y) {
    if (!y[1].defined()) return THPVariable_Wrap(std::move(y[0]));
    return pair(std::move(y[0]), std::move(y[1]));
}

// rotary(...): y, or (y, k's); None where HeadRotaryFunction has to answer (a transform, a trace).
PyObject* py_rotary(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    RotaryCall a;
    if (!rotary_args(args, n, &a)) return nullptr;
    if (!plain_call(a.in, kRotaryInputs)) Py_RETURN_NONE;
    Tensor y[2];
    {
        pybind11::gil_scoped_release no_gil;
        rotary_forward(a, wants_grad(a.in, 4), y);
    }
    return one_or_pair(y);
    END_HANDLE_TH_ERRORS
}

// ---------------------------------------------------------------------------------------------------------------
// The gated delta rule

enum { kDQ, kDK, kDV, kDG, kDB, kDState, kDeltaInputs };

struct DeltaCall {
    Tensor in[kDeltaInputs], lengths;
    pdw_delta c;   // but for addresses and strides
    int dim;
    at::DimVector state_sizes;
};

// A tensor [lead.., T, mid.., heads, channels] (gates: without channels) by strides of [O][T][W][heads]; a copy where it has none.
Tensor delta_view(const Tensor& t, int dim, bool channels, long long* s) {
    auto read = [&](const Tensor& u) {
        const int64_t h = u.dim() - (channels ? 2 : 1);
        s[1] = u.stride(dim), s[3] = u.stride(h);
        return (!channels || u.stride(h + 1) == 1 || u.size(h + 1) == 1) && collapse(u, 0, dim, &s[0]) && collapse(u, dim + 1, h, &s[2]);
    };
    s[0] = s[1] = s[2] = s[3] = 0;
    if (t.numel() == 0 || read(t)) return t;
    const Tensor c = t.contiguous();
    read(c);
    return c;
}

// Addresses and strides of the five tensors; read: what the kernels read of them.
void delta_addresses(const Tensor* in, int dim, pdw_delta* c, Tensor* read) {
    long long* const strides[] = {c->qs, c->ks, c->vs, c->gs, c->bs};
    for (int i = 0; i < 5; ++i) read[i] = delta_view(in[i], dim, i < 3, strides[i]);
    c->q = ptr(read[0]), c->k = ptr(read[1]), c->v = ptr(read[2]), c->g = ptr(read[3]), c->b = ptr(read[4]);
}

struct DeltaNode : public torch::autograd::Node {
    Kept in[5], lengths, states;
    pdw_delta c;
    int dim;
    at::ScalarType gates;
    at::DimVector state_sizes;

    std::string name() const override { return "GatedDeltaBackward"; }
    void release_variables() override {
        std::lock_guard<std::mutex> lock(mutex_);
        for (Kept& k : in) k.v.reset_data();
        lengths.v.reset_data(), states.v.reset_data();
    }

    variable_list apply(variable_list&& grads) override {
        std::lock_guard<std::mutex> lock(mutex_);
        no_second_derivative(*this);
        Tensor gy = grads[0], glast = grads[1];
        if (!gy.defined()) gy = input_metadata(0).zeros_like();
        const auto self = shared_from_this();
        const auto type = input_metadata(0).options().dtype().toScalarType();
        const auto dev = gy.device();
        no_eager_accumulators(*this, dev);
        Tensor t[5], read[5];
        for (int i = 0; i < 5; ++i) t[i] = in[i].get(self, i < 3 ? type : gates, dev);
        Tensor len = lengths.get(self, at::kInt, dev), st = states.get(self, at::kByte, dev);
        at::AutoDispatchBelowADInplaceOrView below;
        gy = packed(gy), glast = packed(glast), len = packed(len), st = packed(st);
        const c10::DeviceGuard guard(dev);
        pdw_delta call = c;
        delta_addresses(t, dim, &call, read);
        call.lengths = (const int*)ptr(len);
        variable_list r(kDeltaInputs);
        for (int i = 0; i < 5; ++i)
            if (task_should_compute_output(i)) r[i] = at::empty(in[i].sizes, t[i].options());
        if (task_should_compute_output(kDState)) r[kDState] = floats(state_sizes, t[0]);
        const size_t need = pdw_delta_workspace_bytes(&call, 1, 1);
        Tensor ws;
        if (need) ws = bytes(need, t[0]);
        check(pdw_delta_bwd(&call, ptr(gy), (const float*)ptr(glast), ptr(st), ptr(r[0]), ptr(r[1]), ptr(r[2]), ptr(r[3]), ptr(r[4]),
                            (float*)ptr(r[kDState]), ptr(ws), need, stream_of(t[0])),
              "pdw_delta_bwd");
        return r;
    }
};

void delta_forward(const DeltaCall& a, bool grad, Tensor* y, Tensor* last) {
    const Tensor(&in)[kDeltaInputs] = a.in;
    const c10::DeviceGuard guard(in[kDQ].device());
    pdw_delta c = a.c;
    Tensor read[5], len, h0, states;
    {
        at::AutoDispatchBelowADInplaceOrView below;
        delta_addresses(in, a.dim, &c, read);
        len = packed(a.lengths), h0 = packed(in[kDState]);
        c.lengths = (const int*)ptr(len), c.h0 = (const float*)ptr(h0);
        *y = at::empty(in[kDV].sizes(), in[kDQ].options());
        *last = floats(a.state_sizes, in[kDQ]);
        if (grad) states = bytes(pdw_delta_states_bytes(&c), *y);
        const size_t need = pdw_delta_workspace_bytes(&c, 0, grad);
        Tensor ws;
        if (need) ws = bytes(need, *y);
        // (an empty tensor has no address: a call for gradients says so with any that is not null)
        check(pdw_delta_fwd(&c, ptr(*y), (float*)ptr(*last), grad && states.numel() ? ptr(states) : nullptr, ptr(ws), need, stream_of(*y)),
              "pdw_delta_fwd");
    }
    if (!grad) return;
    auto node = std::shared_ptr<DeltaNode>(new DeltaNode(), torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(in[kDQ], in[kDK], in[kDV], in[kDG], in[kDB], in[kDState]));
    for (int i = 0; i < 5; ++i) node->in[i].keep(in[i], read[i]);
    node->lengths.keep(a.lengths, len), node->states.keep(states, states);
    node->c = a.c, node->dim = a.dim, node->gates = in[kDG].scalar_type(), node->state_sizes = a.state_sizes;
    torch::autograd::set_history(*y, node);
    torch::autograd::set_history(*last, node);
}

// What a whole call and a step have in common: q, k, v and the gates, [lead.., heads(, channels)].
void check_delta(const Tensor* in, pdw_delta* c) {
    const Tensor &q = in[kDQ], &k = in[kDK], &v = in[kDV], &g = in[kDG], &b = in[kDB];
    static const char* const names[] = {"q", "k", "v", "g", "b"};
    for (int i = 0; i < 5; ++i) TORCH_CHECK_TYPE(in[i].defined(), names[i], " has to be a tensor");
    TORCH_CHECK_TYPE(dtype_code(q.scalar_type()) >= 0, "pyramid dwconv kernels support float32/float16/bfloat16, got ", q.scalar_type());
    for (int i = 1; i < 3; ++i)
        TORCH_CHECK_TYPE(in[i].scalar_type() == q.scalar_type(), names[i], " is ", in[i].scalar_type(), " and q ", q.scalar_type());
    TORCH_CHECK_TYPE(g.scalar_type() == q.scalar_type() || g.scalar_type() == at::kFloat, "g is ", g.scalar_type(), ", q ", q.scalar_type(),
                     " (float32 is possible, too)");
    TORCH_CHECK_TYPE(b.scalar_type() == g.scalar_type(), "b is ", b.scalar_type(), " and g ", g.scalar_type());
    const int64_t rank = q.dim();
    TORCH_CHECK_VALUE(rank >= 2, "expected [..., heads, channels], got ", q.sizes());
    TORCH_CHECK_VALUE(k.sizes() == q.sizes(), "q and k have to be of one shape, got ", q.sizes(), " and ", k.sizes());
    TORCH_CHECK_VALUE(v.dim() == rank && v.sizes().slice(0, rank - 2) == q.sizes().slice(0, rank - 2),
                      "q and v have to be alike but for heads and channels, got ", q.sizes(), " and ", v.sizes());
    const int64_t hk = q.size(-2), hv = v.size(-2);
    TORCH_CHECK_VALUE(hk >= 1 && hv >= 1 && hv % hk == 0, "v's heads have to be a multiple of q's, got ", hv, " and ", hk);
    at::DimVector sizes(q.sizes().slice(0, rank - 1));
    sizes.back() = hv;
    TORCH_CHECK_VALUE(g.sizes() == at::IntArrayRef(sizes), "g has to be ", at::IntArrayRef(sizes), ", got ", g.sizes());
    TORCH_CHECK_VALUE(b.sizes() == at::IntArrayRef(sizes), "b has to be ", at::IntArrayRef(sizes), ", got ", b.sizes());
    TORCH_CHECK_VALUE(q.size(-1) >= 1 && q.size(-1) <= PDW_DELTA_MAX_CHANNELS && v.size(-1) >= 1 && v.size(-1) <= PDW_DELTA_MAX_CHANNELS,
                      "1 to ", PDW_DELTA_MAX_CHANNELS, " channels a head, got ", q.sizes(), " and ", v.sizes());
    TORCH_CHECK_VALUE(hv <= 0x7fffffff, "more than 2^31 - 1 heads");
    c->Hk = (int)hk, c->Hv = (int)hv, c->dk = (int)q.size(-1), c->dv = (int)v.size(-1);
    c->dtype = dtype_code(q.scalar_type()), c->gates_f32 = g.scalar_type() == at::kFloat;
}

// (q, k, v, g, b, state, lengths, dim, reverse, scale, logits)
bool delta_args(PyObject* const* args, Py_ssize_t n, DeltaCall* a) {
    TORCH_CHECK(n == 11, "delta: 11 arguments expected");
    Tensor(&in)[kDeltaInputs] = a->in;
    pdw_delta& c = a->c;
    c = pdw_delta{};
    for (int i = 0; i < kDeltaInputs; ++i)
        if (!tensor_arg(args[i], &in[i])) return false;
    if (!tensor_arg(args[6], &a->lengths)) return false;
    int64_t dim;
    if (!int_arg(args[7], &dim)) return false;
    c.reverse = PyObject_IsTrue(args[8]), c.logits = PyObject_IsTrue(args[10]);
    if (c.reverse < 0 || c.logits < 0) return false;
    c.scale = (float)PyFloat_AsDouble(args[9]);
    if (PyErr_Occurred()) return false;
    check_delta(in, &c);
    const Tensor& q = in[kDQ];
    const int64_t rank = q.dim();
    TORCH_CHECK_VALUE(rank >= 3, "expected [..., T, ..., heads, channels], got ", q.sizes());
    TORCH_CHECK_INDEX(dim >= -rank && dim < rank, "dim ", dim, " of a tensor of ", rank, " dimensions");
    if (dim < 0) dim += rank;
    TORCH_CHECK_VALUE(dim < rank - 2, "the rule runs along any dimension but the heads' and the channels' (", q.sizes(), ", dim ", dim, ")");
    int64_t O = 1, W = 1;
    for (int64_t d = 0; d < rank - 2; ++d) {
        if (d != dim) a->state_sizes.push_back(q.size(d));
        if (d < dim) O *= q.size(d);
        else if (d > dim) W *= q.size(d);
    }
    TORCH_CHECK_VALUE(O <= 0x7fffffff && W <= 0x7fffffff && O * W <= 0x7fffffff / c.Hv && q.size(dim) <= 0x7fffffff,
                      "more than 2^31 - 1 chains or steps: ", q.sizes());
    c.O = (int)O, c.W = (int)W, c.T = q.size(dim), a->dim = (int)dim;
    for (int64_t e : {(int64_t)c.Hv, (int64_t)c.dk, (int64_t)c.dv}) a->state_sizes.push_back(e);
    const Tensor& state = in[kDState];
    if (state.defined()) {
        TORCH_CHECK_TYPE(state.scalar_type() == at::kFloat, "state is float32, got ", state.scalar_type());
        TORCH_CHECK_VALUE(state.sizes() == at::IntArrayRef(a->state_sizes), "state has to be ", at::IntArrayRef(a->state_sizes), ", got ",
                          state.sizes());
    }
    if (a->lengths.defined()) {
        TORCH_CHECK_TYPE(a->lengths.scalar_type() == at::kInt, "lengths is int32, got ", a->lengths.scalar_type());
        TORCH_CHECK_VALUE(a->lengths.sizes() == q.sizes().slice(0, dim), "lengths has to be ", q.sizes().slice(0, dim), ", got ",
                          a->lengths.sizes());
    }
    const Tensor all[] = {in[0], in[1], in[2], in[3], in[4], state, a->lengths};
    check_devices(all, 7);
    return true;
}

PyObject* py_check_delta(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    DeltaCall a;
    if (!delta_args(args, n, &a)) return nullptr;
    Py_RETURN_NONE;
    END_HANDLE_TH_ERRORS
}

// delta(...): (y, last); None where GatedDeltaFunction has to answer.
PyObject* py_delta(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    DeltaCall a;
    if (!delta_args(args, n, &a)) return nullptr;
    if (!plain_call(a.in, kDeltaInputs)) Py_RETURN_NONE;
    Tensor y, last;
    {
        pybind11::gil_scoped_release no_gil;
        delta_forward(a, wants_grad(a.in, kDeltaInputs), &y, &last);
    }
    return pair(std::move(y), std::move(last));
    END_HANDLE_TH_ERRORS
}

// delta_step(q, k, v, g, b, state, new_state, scale, logits): y; new_state (or state in place, None) is written.
PyObject* py_delta_step(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    TORCH_CHECK(n == 9, "delta_step: 9 arguments expected");
    Tensor in[kDeltaInputs], to;
    for (int i = 0; i < kDeltaInputs; ++i)
        if (!tensor_arg(args[i], &in[i])) return nullptr;
    if (!tensor_arg(args[6], &to)) return nullptr;
    pdw_delta c{};
    c.scale = (float)PyFloat_AsDouble(args[7]);
    c.logits = PyObject_IsTrue(args[8]);
    if (PyErr_Occurred()) return nullptr;
    check_delta(in, &c);
    const Tensor &q = in[kDQ], &state = in[kDState];
    TORCH_CHECK_TYPE(state.defined(), "state has to be a tensor");
    at::DimVector sizes(q.sizes().slice(0, q.dim() - 2));
    int64_t B = 1;
    for (int64_t e : sizes) B *= e;
    TORCH_CHECK_VALUE(B <= 0x7fffffff / c.Hv, "more than 2^31 - 1 chains: ", q.sizes());
    for (int64_t e : {(int64_t)c.Hv, (int64_t)c.dk, (int64_t)c.dv}) sizes.push_back(e);
    for (const Tensor* t : {&state, (const Tensor*)&to}) {
        if (!t->defined()) continue;
        TORCH_CHECK_TYPE(t->scalar_type() == at::kFloat, "the state is float32, got ", t->scalar_type());
        TORCH_CHECK_VALUE(t->sizes() == at::IntArrayRef(sizes) && t->is_contiguous(), "the state has to be dense and ", at::IntArrayRef(sizes),
                          ", got ", t->sizes());
    }
    const Tensor into = to.defined() ? to : state;
    const char* what = to.defined() ? "new_state" : "state";
    TORCH_CHECK_VALUE(!overlap(state, into), what, " overlaps what is read beside it");
    for (int i = 0; i < 5; ++i) TORCH_CHECK_VALUE(!overlap(in[i], into), what, " overlaps what is read beside it");
    const Tensor all[] = {in[0], in[1], in[2], in[3], in[4], state, into};
    check_devices(all, 7);
    TORCH_CHECK(!wants_grad(all, 7), "gated_delta_step has no gradient: call it under torch.no_grad(), or gated_delta");
    TORCH_CHECK(plain_call(all, 7), "gated_delta_step takes part in no transform or trace");
    Tensor y;
    {
        pybind11::gil_scoped_release no_gil;
        const c10::DeviceGuard guard(q.device());
        at::AutoDispatchBelowADInplaceOrView below;
        c.O = (int)B, c.T = 1, c.W = 1;
        Tensor read[5];
        long long* const strides[] = {c.qs, c.ks, c.vs, c.gs, c.bs};
        for (int i = 0; i < 5; ++i) {
            // (all leading dimensions as one, ahead of a step's own)
            auto look = [&](const Tensor& u) {
                const int64_t h = u.dim() - (i < 3 ? 2 : 1);
                strides[i][3] = u.stride(h);
                return (i >= 3 || u.stride(h + 1) == 1 || u.size(h + 1) == 1) && collapse(u, 0, h, &strides[i][0]);
            };
            read[i] = in[i];
            if (in[i].numel() && !look(in[i])) read[i] = in[i].contiguous(), look(read[i]);
        }
        c.q = ptr(read[0]), c.k = ptr(read[1]), c.v = ptr(read[2]), c.g = ptr(read[3]), c.b = ptr(read[4]);
        c.h0 = (const float*)ptr(state);
        y = at::empty(in[kDV].sizes(), q.options());
        if (y.numel()) check(pdw_delta_step(&c, ptr(y), (float*)ptr(into), stream_of(q)), "pdw_delta_step");
        if (!into.is_inference()) into.unsafeGetTensorImpl()->bump_version();
    }
    return THPVariable_Wrap(std::move(y));
    END_HANDLE_TH_ERRORS
}

PyMethodDef kDeltaMethods[] = {
    {"check_rotary", (PyCFunction)(void (*)(void))py_check_rotary, METH_FASTCALL, nullptr},
    {"rotary", (PyCFunction)(void (*)(void))py_rotary, METH_FASTCALL, nullptr},
    {"check_delta", (PyCFunction)(void (*)(void))py_check_delta, METH_FASTCALL, nullptr},
    {"delta", (PyCFunction)(void (*)(void))py_delta, METH_FASTCALL, nullptr},
    {"delta_step", (PyCFunction)(void (*)(void))py_delta_step, METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};

}  // namespace

PyMethodDef* pdw_delta_methods() { return kDeltaMethods; }
