// PyTorch binding of the layer operators: argument checks, output allocation, autograd nodes.  No arithmetic; every
// result comes from the C ABI of libplconvlstm (include/plconvlstm.h), whose entry points are handed in as addresses, so
// that the library the rest of the package has loaded is the one that runs.
//
// Native because these operators are often small: a training pass over one of them took 143 us of host time through
// Python autograd functions and ctypes, of which the kernels were 10 to 30 us.
#include <torch/extension.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/variable.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <c10/core/AutogradState.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPStream.h>

#include <unordered_set>

#include "../../include/plconvlstm.h"

namespace {

using at::Tensor;
using OptTensor = std::optional<Tensor>;

struct Library {
    const char* (*last_error)(void) = nullptr;
    size_t (*scan_states_bytes)(int, int, long long) = nullptr;
    size_t (*scan_workspace_bytes)(const plc_scan_desc*, int) = nullptr;
    int (*scan_fwd)(const plc_scan_desc*, void*) = nullptr;
    int (*scan_bwd)(const plc_scan_desc*, void*) = nullptr;
    int (*dropout)(const void*, const void*, void*, long long, int, double, unsigned long long, unsigned long long, const long long*,
                   long long*, void*) = nullptr;
    size_t (*norm_workspace_bytes)(const plc_norm_desc*, int) = nullptr;
    int (*norm_fwd)(const plc_norm_desc*, void*) = nullptr;
    int (*norm_bwd)(const plc_norm_desc*, void*) = nullptr;
} lib;

template <class F>
void bind_one(const py::dict& d, const char* name, F& f) {
    f = reinterpret_cast<F>(d[name].cast<uintptr_t>());
}
void bind(const py::dict& d) {
    bind_one(d, "plc_last_error", lib.last_error);
    bind_one(d, "plc_gated_scan_states_bytes", lib.scan_states_bytes);
    bind_one(d, "plc_gated_scan_workspace_bytes", lib.scan_workspace_bytes);
    bind_one(d, "plc_gated_scan_fwd", lib.scan_fwd);
    bind_one(d, "plc_gated_scan_bwd", lib.scan_bwd);
    bind_one(d, "plc_dropout", lib.dropout);
    bind_one(d, "plc_group_norm_workspace_bytes", lib.norm_workspace_bytes);
    bind_one(d, "plc_group_norm_fwd", lib.norm_fwd);
    bind_one(d, "plc_group_norm_bwd", lib.norm_bwd);
}

void check_rc(int rc, const char* what) {
    if (rc == 0) return;
    const char* msg = lib.last_error();
    TORCH_CHECK_NOT_IMPLEMENTED(rc != PLC_EUNSUPPORTED, what, ": ", msg);
    TORCH_CHECK_VALUE(rc != PLC_EINVAL, what, ": ", msg);
    TORCH_CHECK(false, what, " failed (code ", rc, "): ", msg);
}

// A recorder of PyTorch's own operations sees the allocation of a result and not the kernel that fills it: what it made of
// such a call would return memory that nothing has written.
void check_not_recorded() {
    TORCH_CHECK(!torch::jit::tracer::isTracing() && !c10::impl::TorchDispatchModeTLS::get_mode(c10::impl::TorchDispatchModeKey::PROXY).has_value(),
                "the layer operators cannot be recorded by torch.jit.trace or torch.fx: their kernels are not PyTorch operations (a HIP graph captures them)");
}

void on_gpu(const Tensor& t, const char* name) {
    TORCH_CHECK(t.is_cuda(), name, " is on ", t.device(), ": the layer operators run on MI355X (HIP) only; there is no CPU fallback");
    TORCH_CHECK(t.layout() == at::kStrided, name, " must be a dense tensor");
}
int dtype_of(const Tensor& t, const char* name) {
    on_gpu(t, name);
    switch (t.scalar_type()) {
        case at::kFloat: return PLC_F32;
        case at::kBFloat16: return PLC_BF16;
        case at::kHalf: return PLC_F16;
        default: TORCH_CHECK_TYPE(false, name, " must be float32, bfloat16 or float16 (got ", t.scalar_type(), ")");
    }
    return -1;
}
void like(const Tensor& t, const char* name, const Tensor& x, at::ScalarType dtype) {
    on_gpu(t, name);
    TORCH_CHECK_TYPE(t.scalar_type() == dtype, name, " must be ", dtype, " (got ", t.scalar_type(), ")");
    TORCH_CHECK_VALUE(t.device() == x.device(), name, " is on ", t.device(), ", the input on ", x.device());
}
void shaped(const Tensor& t, const char* name, at::IntArrayRef shape) {
    TORCH_CHECK_VALUE(t.sizes() == shape, name, " must be ", shape, " (got ", t.sizes(), ")");
}
int to_int(int64_t n, const char* what) {
    TORCH_CHECK_NOT_IMPLEMENTED(n <= std::numeric_limits<int>::max(), what, " = ", n, " is more than 2^31 - 1");
    return (int)n;
}
void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }
template <class T = void>
T* ptr(const Tensor& t) { return t.defined() ? reinterpret_cast<T*>(t.data_ptr()) : nullptr; }
Tensor get(const OptTensor& t) { return t.has_value() ? *t : Tensor(); }
// A kernel has written into a caller's tensor: a backward pass that kept it has to notice.
void written(const Tensor& t) {
    if (t.defined() && !t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}
Tensor workspace(size_t bytes, const Tensor& x) {
    return bytes ? at::empty({(int64_t)bytes}, x.options().dtype(at::kByte)) : Tensor();
}

// a gradient that is asked to be differentiable again says so when that is tried, instead of being taken for a constant
torch::autograd::variable_list once(torch::autograd::variable_list grads, const char* what) {
    if (!at::GradMode::is_enabled()) return grads;
    torch::autograd::variable_list in;
    for (Tensor& g : grads) in.push_back(g.defined() ? g.detach().requires_grad_() : g);
    torch::autograd::DelayedError err(std::string("second derivatives of ") + what + " are not available", (int64_t)in.size());
    return err.apply(std::move(in));
}

// A leaf's accumulation node lives as long as any autograd graph that uses the leaf, and belongs to the stream that graph was
// made on.  Where that is the default stream, which cannot be captured, a backward pass that is being captured and reaches
// the node ends the process when the capture ends: refused here, while it can be.  (Another stream joins the capture and is
// joined again: that works, and is what a warm-up on a side stream leaves behind.)
//
// The forward call looks through what was computed during the capture (and leads, if anything does, into the captured
// backward pass) down to the leaves.  A graph made on the default stream before the capture may stay outside that pass, so it is
// looked at when a backward pass of these operators is about to lead there.
bool capturing(const c10::hip::HIPStream& stream) {
    if (!stream.stream()) return false;      // (the default stream; asking the runtime takes a microsecond of a training call)
    hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
    return hipStreamIsCapturing(stream.stream(), &status) == hipSuccess && status != hipStreamCaptureStatusNone;
}
void check_captured(std::vector<torch::autograd::Node*> nodes, int device, bool in_backward) {
    const auto fixed = c10::hip::getDefaultHIPStream(device).id();       // (by id: autograd's streams name the device's type differently)
    std::unordered_set<torch::autograd::Node*> seen;
    while (!nodes.empty()) {
        torch::autograd::Node* n = nodes.back();
        nodes.pop_back();
        if (!seen.insert(n).second) continue;
        const auto made = n->stream();
        if (made.has_value() && made->device_index() == device && made->id() == fixed) {
            TORCH_CHECK(n->num_outputs() > 0 && !in_backward,
                        "a graph is being captured while outputs of an earlier pass over the same leaf tensor, on the default stream, are alive: "
                        "its gradient would be accumulated there.  Detach or delete those outputs first.");
            continue;
        }
        for (uint32_t i = 0; i < n->num_outputs(); ++i)
            if (n->next_edge(i).is_valid() && (!in_backward || n->task_should_compute_output(i))) nodes.push_back(n->next_edge(i).function.get());
    }
}
// called by the backward pass of an operator on a tensor of that device, before it launches anything
void check_captured_backward(const Tensor& g) {
    if (!g.is_cuda() || !capturing(c10::hip::getCurrentHIPStream(g.device().index()))) return;
    if (const auto node = torch::autograd::get_current_node()) check_captured({node.get()}, g.device().index(), true);
}

// ---------------------------------------------------------------------------------------------- gated recurrence
// [B, T, ...] with the trailing dimensions contiguous: read in place with the strides of a sample and of a step
Tensor steps(const Tensor& t, long long inner, long long& batch, long long& step) {
    Tensor r = t;
    if (t.is_contiguous()) {
        batch = t.size(1) * inner;
        step = inner;
        return r;
    }
    long long want = 1;
    bool fine = t.numel() > 0;
    for (int64_t d = t.dim() - 1; d >= 2 && fine; --d) {
        fine = t.size(d) == 1 || t.stride(d) == want;
        want *= t.size(d);
    }
    if (!fine) {
        r = t.contiguous();
        batch = t.size(1) * inner;
        step = inner;
    } else {
        batch = t.stride(0);
        step = t.stride(1);
    }
    return r;
}

struct Scan {
    plc_scan_desc d;
    Tensor x, f, h0, lengths;            // as the kernels take them
    std::vector<int64_t> state;          // shape of a state
    Scan(const Tensor& x_, const Tensor& f_, const Tensor& h0_, const Tensor& lengths_, bool coupled) {
        memset(&d, 0, sizeof(d));
        d.dtype = dtype_of(x_, "x");
        like(f_, "f", x_, x_.scalar_type());
        TORCH_CHECK_VALUE(x_.dim() >= 2 && x_.sizes() == f_.sizes(), "x and f must both be [B, T, ...] (got ", x_.sizes(), " and ", f_.sizes(), ")");
        state.push_back(x_.size(0));
        long long inner = 1;
        for (int64_t i = 2; i < x_.dim(); ++i) {
            state.push_back(x_.size(i));
            inner *= x_.size(i);
        }
        if (h0_.defined()) {
            like(h0_, "h0", x_, at::kFloat);
            shaped(h0_, "h0", state);
            h0 = h0_.contiguous();
        }
        if (lengths_.defined()) {
            like(lengths_, "lengths", x_, at::kInt);
            shaped(lengths_, "lengths", {x_.size(0)});
            lengths = lengths_.contiguous();
        }
        d.B = to_int(x_.size(0), "B");
        d.T = to_int(x_.size(1), "T");
        d.D = inner;
        d.coupled = coupled;
        x = steps(x_, inner, d.x_batch, d.x_step);
        f = steps(f_, inner, d.f_batch, d.f_step);
        d.x = ptr(x);
        d.f = ptr(f);
        d.h0 = ptr<float>(h0);
        d.lengths = ptr<int>(lengths);
    }
};

std::tuple<Tensor, Tensor, Tensor> scan_forward(const Tensor& x, const Tensor& f, const Tensor& h0, const Tensor& lengths, bool coupled,
                                                bool save_states, const Tensor& into) {
    check_not_recorded();
    Scan s(x, f, h0, lengths, coupled);
    const c10::OptionalDeviceGuard guard(x.device());
    const auto f32 = x.options().dtype(at::kFloat);
    Tensor y = at::empty(x.sizes(), x.options()), states;
    if (into.defined()) {
        like(into, "h_last", x, at::kFloat);
        shaped(into, "h_last", s.state);
        TORCH_CHECK_VALUE(into.is_contiguous(), "h_last must be contiguous");
    }
    Tensor h = into.defined() ? into : at::empty(s.state, f32);
    if (save_states)
        if (const size_t n = lib.scan_states_bytes(s.d.B, s.d.T, s.d.D)) states = at::empty({(int64_t)(n / 4)}, f32);
    s.d.y = ptr(y);
    s.d.h_last = ptr<float>(h);
    s.d.states = ptr<float>(states);
    const size_t n = lib.scan_workspace_bytes(&s.d, 0);
    Tensor ws = workspace(n, x);
    s.d.workspace = ptr(ws);
    s.d.workspace_bytes = n;
    check_rc(lib.scan_fwd(&s.d, stream_of(x)), "plc_gated_scan_fwd");
    written(into);
    return {y, h, states};
}

std::tuple<Tensor, Tensor, Tensor> scan_backward(const Tensor& x, const Tensor& f, const Tensor& h0, const Tensor& lengths, bool coupled,
                                                 const Tensor& states, const Tensor& dy_, const Tensor& dh_, bool need_dh0) {
    check_not_recorded();
    Scan s(x, f, h0, lengths, coupled);
    const c10::OptionalDeviceGuard guard(x.device());
    const auto f32 = x.options().dtype(at::kFloat);
    Tensor dy = dy_, dh = dh_;
    if (!dy.defined()) dy = at::zeros(x.sizes(), x.options());
    like(dy, "dy", x, x.scalar_type());
    shaped(dy, "dy", x.sizes());
    dy = steps(dy, s.d.D, s.d.dy_batch, s.d.dy_step);
    if (dh.defined()) {
        like(dh, "dh_last", x, at::kFloat);
        shaped(dh, "dh_last", s.state);
        dh = dh.contiguous();
    }
    if (const size_t n = lib.scan_states_bytes(s.d.B, s.d.T, s.d.D)) {
        TORCH_CHECK_VALUE(states.defined(), "the backward pass needs the states the forward pass stored");
        like(states, "states", x, at::kFloat);
        TORCH_CHECK_VALUE(states.is_contiguous() && (size_t)states.numel() * 4 >= n, "states do not belong to these inputs");
    }
    Tensor dx = at::empty(x.sizes(), x.options()), df = at::empty(x.sizes(), x.options());
    Tensor dh0 = need_dh0 ? at::empty(s.state, f32) : Tensor();
    s.d.states = ptr<float>(states);
    s.d.dy = ptr(dy);
    s.d.dh_last = ptr<float>(dh);
    s.d.dx = ptr(dx);
    s.d.df = ptr(df);
    s.d.dh0 = ptr<float>(dh0);
    const size_t n = lib.scan_workspace_bytes(&s.d, 1);
    Tensor ws = workspace(n, x);
    s.d.workspace = ptr(ws);
    s.d.workspace_bytes = n;
    check_rc(lib.scan_bwd(&s.d, stream_of(x)), "plc_gated_scan_bwd");
    return {dx, df, dh0};
}

struct ScanFn : public torch::autograd::Function<ScanFn> {
    static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const Tensor& x, const Tensor& f, const OptTensor& h0,
                                                  const OptTensor& lengths, bool coupled) {
        at::AutoDispatchBelowADInplaceOrView below;
        auto [y, h, states] = scan_forward(x, f, get(h0), get(lengths), coupled, true, Tensor());
        ctx->save_for_backward({x, f, get(h0), get(lengths), states});
        ctx->saved_data["coupled"] = coupled;
        ctx->saved_data["need_dh0"] = h0.has_value() && h0->requires_grad();
        ctx->set_materialize_grads(false);
        return {y, h};
    }
    static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list g) {
        if (!g[0].defined() && !g[1].defined()) return {Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
        check_captured_backward(g[0].defined() ? g[0] : g[1]);
        const auto s = ctx->get_saved_variables();
        torch::autograd::variable_list out;
        {
            const at::AutoGradMode off(false);
            auto [dx, df, dh0] = scan_backward(s[0], s[1], s[2], s[3], ctx->saved_data["coupled"].toBool(), s[4], g[0], g[1],
                                               ctx->saved_data["need_dh0"].toBool());
            out = {dx, df, dh0, Tensor(), Tensor()};
        }
        return once(std::move(out), "gated_linear_scan");
    }
};

// There are no forward-mode derivatives: a tensor that carries a tangent is refused, since the result would carry none.
void check_no_tangent(std::initializer_list<const Tensor*> ts) {
    if (!c10::AutogradState::get_tls_state().get_fw_grad_mode()) return;
    for (const Tensor* t : ts)
        TORCH_CHECK_NOT_IMPLEMENTED(!t->defined() || !t->_fw_grad(/*level=*/0).defined(),
                                    "forward-mode derivatives of the layer operators are not available");
}
bool wants_grad(std::initializer_list<const Tensor*> ts) {
    check_no_tangent(ts);
    if (!at::GradMode::is_enabled()) return false;
    const Tensor* any = nullptr;
    for (const Tensor* t : ts)
        if (t->defined() && t->requires_grad()) any = t;
    if (!any) return false;
    if (any->is_cuda() && capturing(c10::hip::getCurrentHIPStream(any->device().index()))) {
        std::vector<torch::autograd::Node*> nodes;
        std::vector<std::shared_ptr<torch::autograd::Node>> kept;
        for (const Tensor* t : ts)
            if (t->defined() && t->requires_grad())
                if (auto node = t->is_leaf() ? torch::autograd::impl::try_get_grad_accumulator(*t) : t->grad_fn()) {
                    nodes.push_back(node.get());
                    kept.push_back(std::move(node));
                }
        check_captured(std::move(nodes), any->device().index(), false);
    }
    return true;
}

std::tuple<Tensor, Tensor> scan(const Tensor& x, const Tensor& f, const OptTensor& h0, const OptTensor& lengths, bool coupled) {
    const Tensor h = get(h0);
    if (wants_grad({&x, &f, &h})) {
        auto r = ScanFn::apply(x, f, h0, lengths, coupled);
        return {r[0], r[1]};
    }
    auto [y, last, states] = scan_forward(x, f, h, get(lengths), coupled, false, Tensor());
    return {y, last};
}

std::tuple<Tensor, Tensor> scan_one_step(const Tensor& x_, const Tensor& f_, const Tensor& state_, bool coupled, bool inplace) {
    check_no_tangent({&x_, &f_, &state_});
    check_not_recorded();
    const at::AutoGradMode off(false);
    const Tensor x = x_.detach(), f = f_.detach(), state = state_.detach();
    dtype_of(x, "x");
    like(state, "state", x, at::kFloat);
    TORCH_CHECK_VALUE(x.dim() >= 1 && x.sizes() == f.sizes() && x.sizes() == state.sizes(), "x, f and state must have one shape (got ", x.sizes(),
                      ", ", f.sizes(), " and ", state.sizes(), ")");
    TORCH_CHECK_VALUE(!inplace || state.is_contiguous(), "a state that is updated in place must be contiguous");
    auto [y, h, states] = scan_forward(x.unsqueeze(1), f.unsqueeze(1), state, Tensor(), coupled, false, inplace ? state : Tensor());
    return {y.squeeze(1), inplace ? state_ : h};
}

// ---------------------------------------------------------------------------------------------- dropout
struct Draw {          // what a mask is made of; offset_t: an int64 on the device that takes the place of offset
    double p;
    uint64_t seed, offset;
    Tensor offset_t;
    Draw(double p_, uint64_t seed_, uint64_t offset_, const Tensor& t, const Tensor& x) : p(p_), seed(seed_), offset(offset_), offset_t(t) {
        TORCH_CHECK_VALUE(p >= 0.0 && p <= 1.0, "p must be a probability (got ", p, ")");
        if (t.defined()) {
            like(t, "offset", x, at::kLong);
            TORCH_CHECK_VALUE(t.numel() == 1, "offset must have one element (got ", t.numel(), ")");
        }
    }
};

Tensor dropout_forward(const Tensor& x_, double p, uint64_t seed, uint64_t offset, const Tensor& offset_t, const Tensor& residual, const Tensor& used) {
    check_not_recorded();
    const int dtype = dtype_of(x_, "x");
    const Draw w(p, seed, offset, offset_t, x_);
    const c10::OptionalDeviceGuard guard(x_.device());
    const Tensor x = x_.contiguous();
    Tensor r;
    if (residual.defined()) {
        like(residual, "residual", x, x.scalar_type());
        shaped(residual, "residual", x.sizes());
        r = residual.contiguous();
    }
    if (used.defined()) like(used, "used_offset", x, at::kLong);
    Tensor y = at::empty(x.sizes(), x.options().memory_format(at::MemoryFormat::Contiguous));
    check_rc(lib.dropout(ptr(x), ptr(r), ptr(y), x.numel(), dtype, p, seed, offset, ptr<long long>(offset_t), ptr<long long>(used), stream_of(x)),
             "plc_dropout");
    written(used);
    return y;
}

struct DropoutFn : public torch::autograd::Function<DropoutFn> {
    static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& x, const OptTensor& residual, double p, int64_t seed, int64_t offset,
                          const OptTensor& offset_t) {
        at::AutoDispatchBelowADInplaceOrView below;
        Tensor used = offset_t.has_value() ? at::empty_like(*offset_t) : Tensor();
        Tensor y = dropout_forward(x, p, (uint64_t)seed, (uint64_t)offset, get(offset_t), get(residual), used);
        ctx->save_for_backward({used});
        ctx->saved_data["p"] = p;
        ctx->saved_data["seed"] = seed;
        ctx->saved_data["offset"] = offset;
        ctx->saved_data["dx"] = x.requires_grad();
        ctx->saved_data["dr"] = residual.has_value() && residual->requires_grad();
        return y;
    }
    static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list g) {
        check_captured_backward(g[0]);
        Tensor dx;
        if (ctx->saved_data["dx"].toBool()) {
            const at::AutoGradMode off(false);
            dx = dropout_forward(g[0], ctx->saved_data["p"].toDouble(), (uint64_t)ctx->saved_data["seed"].toInt(), (uint64_t)ctx->saved_data["offset"].toInt(),
                                 ctx->get_saved_variables()[0], Tensor(), Tensor());
        }
        const Tensor dr = ctx->saved_data["dr"].toBool() ? g[0] : Tensor();
        return once({dx, dr, Tensor(), Tensor(), Tensor(), Tensor()}, "counter_dropout");
    }
};

Tensor dropout(const Tensor& x, double p, uint64_t seed, uint64_t offset, const OptTensor& offset_t, const OptTensor& residual) {
    const Tensor r = get(residual);
    if (wants_grad({&x, &r})) return DropoutFn::apply(x, residual, p, (int64_t)seed, (int64_t)offset, offset_t);
    return dropout_forward(x, p, seed, offset, get(offset_t), r, Tensor());
}

// ---------------------------------------------------------------------------------------------- group norm
struct Norm {
    plc_norm_desc d;
    Tensor x, w, b;
    Norm(const Tensor& x_, int64_t groups, const Tensor& w_, const Tensor& b_, double eps, int64_t act, const Draw& draw) {
        memset(&d, 0, sizeof(d));
        d.dtype = dtype_of(x_, "x");
        TORCH_CHECK_VALUE(x_.dim() == 4, "x must be [N, C, H, W] (got ", x_.sizes(), ")");
        const int64_t ch = x_.size(1);
        TORCH_CHECK_VALUE(groups >= 1 && ch >= 1 && ch % groups == 0, ch, " channels do not divide into ", groups, " groups");
        TORCH_CHECK_VALUE(eps >= 0.0, "eps must not be negative (got ", eps, ")");
        const Tensor* from[2] = {&w_, &b_};
        Tensor* to[2] = {&w, &b};
        for (int i = 0; i < 2; ++i)
            if (from[i]->defined()) {
                like(*from[i], i ? "bias" : "weight", x_, at::kFloat);
                shaped(*from[i], i ? "bias" : "weight", {ch});
                *to[i] = from[i]->contiguous();
            }
        x = x_.contiguous(at::MemoryFormat::ChannelsLast);
        d.N = to_int(x.size(0), "N");
        d.C = to_int(ch, "C");
        d.G = (int)groups;
        d.HW = to_int(x.size(2) * x.size(3), "H * W");
        d.layout = PLC_NHWC;
        d.act = (int)act;
        d.eps = (float)eps;
        d.x = ptr(x);
        d.weight = ptr<float>(w);
        d.bias = ptr<float>(b);
        d.p = draw.p;
        d.seed = draw.seed;
        d.offset = draw.offset;
        d.offset_ptr = ptr<long long>(draw.offset_t);
    }
};
Tensor channels_last_like(const Tensor& x) { return at::empty(x.sizes(), x.options().memory_format(at::MemoryFormat::ChannelsLast)); }

std::tuple<Tensor, Tensor> norm_forward(const Tensor& x, int64_t groups, const Tensor& w, const Tensor& b, double eps, int64_t act, double p,
                                        uint64_t seed, uint64_t offset, const Tensor& offset_t, const Tensor& used) {
    check_not_recorded();
    dtype_of(x, "x");
    const Draw draw(p, seed, offset, offset_t, x);
    const c10::OptionalDeviceGuard guard(x.device());
    Norm s(x, groups, w, b, eps, act, draw);
    if (used.defined()) like(used, "used_offset", x, at::kLong);
    Tensor y = channels_last_like(x), stats = at::empty({x.size(0), groups, 2}, x.options().dtype(at::kFloat).memory_format(at::MemoryFormat::Contiguous));
    s.d.y = ptr(y);
    s.d.stats = ptr<float>(stats);
    s.d.used_offset = ptr<long long>(used);
    const size_t n = lib.norm_workspace_bytes(&s.d, 0);
    Tensor ws = workspace(n, x);
    s.d.workspace = ptr(ws);
    s.d.workspace_bytes = n;
    check_rc(lib.norm_fwd(&s.d, stream_of(x)), "plc_group_norm_fwd");
    written(used);
    return {y, stats};
}

std::tuple<Tensor, Tensor, Tensor> norm_backward(const Tensor& x, int64_t groups, const Tensor& w, const Tensor& b, double eps, int64_t act, double p,
                                                 uint64_t seed, uint64_t offset, const Tensor& offset_t, const Tensor& stats, const Tensor& dy_) {
    check_not_recorded();
    dtype_of(x, "x");
    const Draw draw(p, seed, offset, offset_t, x);
    const c10::OptionalDeviceGuard guard(x.device());
    Norm s(x, groups, w, b, eps, act, draw);
    like(dy_, "dy", x, x.scalar_type());
    shaped(dy_, "dy", x.sizes());
    const Tensor dy = dy_.contiguous(at::MemoryFormat::ChannelsLast);
    like(stats, "stats", x, at::kFloat);
    TORCH_CHECK_VALUE(stats.sizes() == at::IntArrayRef({x.size(0), groups, 2}) && stats.is_contiguous(), "stats do not belong to these inputs");
    Tensor dx = channels_last_like(x), dw, db;
    if (w.defined()) dw = at::empty({x.size(1)}, w.options());
    if (b.defined()) db = at::empty({x.size(1)}, b.options());
    s.d.stats = ptr<float>(stats);
    s.d.dy = ptr(dy);
    s.d.dx = ptr(dx);
    s.d.dweight = ptr<float>(dw);
    s.d.dbias = ptr<float>(db);
    const size_t n = lib.norm_workspace_bytes(&s.d, 1);
    Tensor ws = workspace(n, x);
    s.d.workspace = ptr(ws);
    s.d.workspace_bytes = n;
    check_rc(lib.norm_bwd(&s.d, stream_of(x)), "plc_group_norm_bwd");
    return {dx, dw, db};
}

struct NormFn : public torch::autograd::Function<NormFn> {
    static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& x, const OptTensor& w, const OptTensor& b, int64_t groups, double eps,
                          int64_t act, double p, int64_t seed, int64_t offset, const OptTensor& offset_t) {
        at::AutoDispatchBelowADInplaceOrView below;
        Tensor used = p > 0 && offset_t.has_value() ? at::empty_like(*offset_t) : Tensor();
        auto [y, stats] = norm_forward(x, groups, get(w), get(b), eps, act, p, (uint64_t)seed, (uint64_t)offset, get(offset_t), used);
        ctx->save_for_backward({x, get(w), get(b), stats, used});
        ctx->saved_data["groups"] = groups;
        ctx->saved_data["eps"] = eps;
        ctx->saved_data["act"] = act;
        ctx->saved_data["p"] = p;
        ctx->saved_data["seed"] = seed;
        ctx->saved_data["offset"] = offset;
        return y;
    }
    static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list g) {
        check_captured_backward(g[0]);
        const auto s = ctx->get_saved_variables();
        auto& d = ctx->saved_data;
        torch::autograd::variable_list out(10);
        {
            const at::AutoGradMode off(false);
            std::tie(out[0], out[1], out[2]) = norm_backward(s[0], d["groups"].toInt(), s[1], s[2], d["eps"].toDouble(), d["act"].toInt(), d["p"].toDouble(),
                                                             (uint64_t)d["seed"].toInt(), (uint64_t)d["offset"].toInt(), s[4], s[3], g[0]);
        }
        return once(std::move(out), "group_norm_act");
    }
};

Tensor norm(const Tensor& x, int64_t groups, const OptTensor& w, const OptTensor& b, double eps, int64_t act, double p, uint64_t seed, uint64_t offset,
            const OptTensor& offset_t) {
    const Tensor wt = get(w), bt = get(b);
    if (wants_grad({&x, &wt, &bt})) return NormFn::apply(x, w, b, groups, eps, act, p, (int64_t)seed, (int64_t)offset, offset_t);
    return std::get<0>(norm_forward(x, groups, wt, bt, eps, act, p, seed, offset, get(offset_t), Tensor()));
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
    m.doc() = "PyTorch binding of libplconvlstm's layer operators (see pl_convlstm_gan_amd/ops.py and layers.py)";
    using release = py::call_guard<py::gil_scoped_release>;
    m.attr("abi_version") = PLC_VERSION;
    m.def("bind", &bind);
    m.def("scan_forward", [](const Tensor& x, const Tensor& f, const OptTensor& h0, const OptTensor& lengths, bool coupled, bool save, const OptTensor& into) {
        return scan_forward(x, f, get(h0), get(lengths), coupled, save, get(into)); }, release());
    m.def("scan_backward", [](const Tensor& x, const Tensor& f, const OptTensor& h0, const OptTensor& lengths, bool coupled, const OptTensor& states,
                              const OptTensor& dy, const OptTensor& dh, bool need) {
        return scan_backward(x, f, get(h0), get(lengths), coupled, get(states), get(dy), get(dh), need); }, release());
    m.def("scan", &scan, release());
    m.def("step", &scan_one_step, release());
    m.def("dropout_forward", [](const Tensor& x, double p, uint64_t seed, uint64_t offset, const OptTensor& t, const OptTensor& r, const OptTensor& used) {
        return dropout_forward(x, p, seed, offset, get(t), get(r), get(used)); }, release());
    m.def("dropout", &dropout, release());
    m.def("norm_forward", [](const Tensor& x, int64_t g, const OptTensor& w, const OptTensor& b, double eps, int64_t act, double p, uint64_t seed,
                             uint64_t offset, const OptTensor& t, const OptTensor& used) {
        return norm_forward(x, g, get(w), get(b), eps, act, p, seed, offset, get(t), get(used)); }, release());
    m.def("norm_backward", [](const Tensor& x, int64_t g, const OptTensor& w, const OptTensor& b, double eps, int64_t act, double p, uint64_t seed,
                              uint64_t offset, const OptTensor& t, const Tensor& stats, const Tensor& dy) {
        return norm_backward(x, g, get(w), get(b), eps, act, p, seed, offset, get(t), stats, dy); }, release());
    m.def("norm", &norm, release());
}
