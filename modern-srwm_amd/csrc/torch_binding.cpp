// The selective-scan, convolution and norm operators for torch tensors, over the C entry points of include/srwm_hip.h:
// checks of the arguments, allocation, the current stream, and autograd.  Single-token calls and small training steps are
// bound by the host, and this is what it costs them: a call of one token takes 14 us with the checks in Python over ctypes,
// and a backward pass then waits for the interpreter in autograd's own thread.  No kernel is launched other than through the
// C entry points, and there is no CPU path.
#include <ATen/ATen.h>
#include <ATen/TracerMode.h>
#include <c10/core/AutogradState.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/accumulate_grad.h>
#include <torch/csrc/utils/pybind.h>
#include <torch/python.h>

#include <string>
#include <tuple>
#include <unordered_set>
#include <vector>

#include "../../include/srwm_hip.h"

namespace {

namespace py = pybind11;
using at::IntArrayRef;
using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::Function;
using torch::autograd::variable_list;
using MaybeTensor = std::optional<Tensor>;   // autograd's Function takes absent tensors in this form only

Tensor or_none(const MaybeTensor &t) { return t.has_value() ? *t : Tensor(); }

void check_code(int code, const char *what) {
    TORCH_CHECK(code != SRWM_ESIZE, what, ": sizes beyond what the kernels take");
    TORCH_CHECK(code == 0, what, " failed with code ", code, ": ", srwm_hip_strerror(code));
}

const char *type_name(at::ScalarType t) {
    return t == at::kFloat ? "torch.float32" : t == at::kBFloat16 ? "torch.bfloat16" : t == at::kInt ? "torch.int32" : c10::toString(t);
}

// float32 or bfloat16 rows; true: bfloat16
bool io_type(const Tensor &t, const char *name) {
    const auto s = t.scalar_type();
    TORCH_CHECK_TYPE(s == at::kFloat || s == at::kBFloat16, name, " must be torch.float32 or torch.bfloat16 (got ", type_name(s), ")");
    return s == at::kBFloat16;
}

void on_gpu(const Tensor &t, const char *name) {
    TORCH_CHECK(t.is_cuda(), name, " must live on the GPU (got ", t.device(), "); there is no CPU path");
}

void fits(const Tensor &t, const char *name, IntArrayRef shape, at::ScalarType type, const at::Device &dev) {
    TORCH_CHECK(t.is_cuda(), name, " must live on the GPU (got ", t.device(), "); there is no CPU path");
    TORCH_CHECK_TYPE(t.scalar_type() == type, name, " must be ", type_name(type), " (got ", type_name(t.scalar_type()), ")");
    TORCH_CHECK_VALUE(t.sizes() == shape, name, " has shape ", t.sizes(), ", expected ", shape);
    TORCH_CHECK(t.device() == dev, name, " lives on ", t.device(), ", the call's other tensors on ", dev);
}

bool aligned(const Tensor &t) { return (reinterpret_cast<uintptr_t>(t.const_data_ptr()) & 15) == 0; }

// A tensor as the kernels read it through strides: its last axis contiguous (other layouts are copied).  Rows of one step
// have three axes; their third stride is not used.
struct Rows {
    Tensor t;
    int64_t st[3] = {0, 0, 0};
    Rows() = default;
    explicit Rows(const Tensor &x) : t(x) {
        if (!t.defined()) return;
        const int nd = (int)t.dim();
        if (t.stride(nd - 1) != 1 && t.size(nd - 1) != 1) t = t.contiguous();
        for (int i = 0; i + 1 < nd; ++i) st[i] = t.stride(i);
    }
    const int64_t *strides() const { return t.defined() ? st : nullptr; }
    template <typename T>
    T *ptr() const { return t.defined() ? static_cast<T *>(t.data_ptr()) : nullptr; }
};

Rows rows_in(const Tensor &t, const char *name, IntArrayRef shape, at::ScalarType type, const at::Device &dev) {
    if (!t.defined()) return Rows();
    fits(t, name, shape, type, dev);
    return Rows(t);
}

// A dense tensor that starts at a multiple of 16 bytes (copied where it is not); undefined stays undefined.
Tensor dense_in(const Tensor &t, const char *name, IntArrayRef shape, at::ScalarType type, const at::Device &dev) {
    if (!t.defined()) return t;
    fits(t, name, shape, type, dev);
    Tensor d = t.contiguous();
    return aligned(d) ? d : d.clone();
}
template <typename T>
T *ptr(const Tensor &t) { return t.defined() ? static_cast<T *>(t.data_ptr()) : nullptr; }

// An empty tensor of t's shape and type in the memory order of t's rows, its last axis contiguous.
Tensor rows_like(const Tensor &t) {
    Tensor out = at::empty_like(t);
    const int nd = (int)t.dim();
    if (nd > 0 && out.stride(nd - 1) != 1 && out.size(nd - 1) != 1) out = at::empty(t.sizes(), t.options());
    return out;
}
Tensor like_or_none(const Tensor &t) { return t.defined() ? at::empty_like(t) : Tensor(); }

void *stream_of(const Tensor &t) { return c10::hip::getCurrentHIPStream(t.get_device()).stream(); }
at::TensorOptions f32_on(const Tensor &t) { return t.options().dtype(at::kFloat); }
Tensor floats(int64_t n, const Tensor &like) { return n ? at::empty({n}, f32_on(like)) : Tensor(); }

bool wants_grad(std::initializer_list<Tensor> ts) {
    if (!at::GradMode::is_enabled()) return false;
    for (const Tensor &t : ts)
        if (t.defined() && t.requires_grad()) return true;
    return false;
}

// The kernels carry no tangents, and a dual tensor does not say that it requires a gradient: without this its derivative
// would count as zero.
void no_tangents(const char *what, std::initializer_list<Tensor> ts) {
    if (!c10::AutogradState::get_tls_state().get_fw_grad_mode()) return;
    for (const Tensor &t : ts)
        TORCH_CHECK(!t.defined() || !t._fw_grad(/*level=*/0).defined(), what, " has no derivative in forward mode");
}

// A trace holds the allocations of a call and not its kernels: run again, it would return memory that nobody wrote.
void not_traced(const char *what) {
    using Modes = c10::impl::TorchDispatchModeTLS;
    using Mode = c10::impl::TorchDispatchModeKey;
    bool traced = at::tracer::impl::is_dispatch_enabled();
    if (Modes::any_modes_set())
        for (const Mode m : {Mode::FAKE, Mode::PROXY, Mode::FUNCTIONAL}) traced = traced || Modes::get_mode(m).has_value();
    TORCH_CHECK(!traced, what, " cannot be traced: its kernels are launched outside torch's dispatcher");
}
void plain_call(const char *what, std::initializer_list<Tensor> ts) {
    no_tangents(what, ts);
    not_traced(what);
}

// A captured backward joins the streams of the leaves' gradient accumulators, those of leaves that reach the call through
// other operations among them.  One that a live graph outside the capture recorded on the default stream cannot be joined:
// the process would end inside the backward, so the forward refuses.  The graph behind the inputs is walked in captures only.
void not_held_outside(const char *what, c10::ArrayRef<Tensor> ts) {
    hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
    int dev = -1;
    for (const Tensor &t : ts)
        if (dev < 0 && t.defined() && t.is_cuda()) dev = t.get_device();
    if (dev < 0) return;
    if (hipStreamIsCapturing(c10::hip::getCurrentHIPStream(dev).stream(), &status) != hipSuccess)
        (void)hipGetLastError();   // the default stream while another one is captured: the launch will say so
    if (status == hipStreamCaptureStatusNone) return;
    std::vector<torch::autograd::Node *> open;
    std::vector<std::shared_ptr<torch::autograd::Node>> leaves;   // hold what the open list points to
    for (const Tensor &t : ts) {
        if (!t.defined() || !t.requires_grad()) continue;
        if (auto node = t.is_leaf() ? torch::autograd::impl::try_get_grad_accumulator(t) : t.grad_fn()) {
            open.push_back(node.get());
            leaves.push_back(std::move(node));
        }
    }
    std::unordered_set<torch::autograd::Node *> seen(open.begin(), open.end());
    while (!open.empty()) {
        torch::autograd::Node *node = open.back();
        open.pop_back();
        if (dynamic_cast<torch::autograd::AccumulateGrad *>(node)) {
            const auto on = node->stream();
            TORCH_CHECK(!on || on->id() != c10::Stream(c10::Stream::DEFAULT, on->device()).id(), what,
                        ": a stream is being captured while a graph recorded on the default stream still holds the gradient of a leaf of "
                        "this call; drop that graph and its outputs first, or record it on a side stream");
        }
        for (const torch::autograd::Edge &e : node->next_edges())
            if (e.function && seen.insert(e.function.get()).second) open.push_back(e.function.get());
    }
}

// What a backward returns.  Where a graph of it is recorded (create_graph), a derivative of these gradients raises instead
// of counting them as constants.  The node that raises leads on to the inputs of the forward and to the gradients that came in:
// a derivative that is asked for some tensors only follows the paths to them and would pass a node without any by.
struct NoDerivative : torch::autograd::Node {
    std::string what;
    NoDerivative(const char *what, torch::autograd::edge_list &&next) : Node(std::move(next)), what(what) {}
    variable_list apply(variable_list &&) override { TORCH_CHECK(false, what, " has no second derivative"); }
};
variable_list once_differentiable(variable_list g, const char *what, const variable_list &incoming) {
    if (!at::GradMode::is_enabled()) return g;
    torch::autograd::edge_list next;
    if (const auto forward = torch::autograd::get_current_node()) next = forward->next_edges();
    for (const Tensor &t : incoming)
        if (t.defined() && t.requires_grad()) next.push_back(torch::autograd::impl::gradient_edge(t));
    const std::shared_ptr<NoDerivative> node(new NoDerivative(what, std::move(next)), torch::autograd::deleteNode);
    for (Tensor &t : g) {
        if (!t.defined()) continue;
        t = t.detach();
        const uint32_t nr = node->add_input_metadata(t);
        torch::autograd::impl::set_gradient_edge(t, {node, nr});
    }
    return g;
}

// A tensor that a kernel overwrites: itself where it is dense and aligned, else a copy that is written back.
struct Overwritten {
    Tensor orig, work;
    explicit Overwritten(const Tensor &t) : orig(t), work(t) {
        if (!t.is_contiguous() || !aligned(t)) work = t.clone(at::MemoryFormat::Contiguous);
    }
    void done() {
        if (!work.is_same(orig)) orig.copy_(work);
        else if (!orig.is_inference()) orig.unsafeGetTensorImpl()->bump_version();
    }
};

// ---- selective scan
struct ScanSizes {
    int64_t N, H, L, E, S, G;
};
ScanSizes scan_sizes(const Tensor &u, const Tensor &A, const Tensor &B, bool step) {
    const int nd = step ? 3 : 4;
    TORCH_CHECK_VALUE(u.dim() == nd && A.dim() == 3 && B.dim() == nd,
                      step ? "u must be (N, H, E), A (H, E, S), B and C (N, G, S)" : "u must be (N, H, L, E), A (H, E, S), B and C (N, G, L, S)");
    const ScanSizes z{u.size(0), u.size(1), step ? 1 : u.size(2), u.size(nd - 1), A.size(2), B.size(1)};
    TORCH_CHECK_VALUE(z.G > 0 && z.H % z.G == 0, "the ", z.H, " heads must divide into the ", z.G, " groups of B and C");
    TORCH_CHECK_VALUE(z.S > 0, "a channel needs at least one state");
    return z;
}
struct ScanIn {   // the inputs, checked and laid out
    ScanSizes z;
    bool bf16;
    Rows u, delta, zz, B, C;
    Tensor A, D, bias, keep, lengths;
    ScanIn(const Tensor &u_, const Tensor &delta_, const Tensor &A_, const Tensor &B_, const Tensor &C_, const Tensor &D_,
           const Tensor &z_, const Tensor &bias_, const Tensor &keep_, const Tensor &lengths_, bool step)
        : z(scan_sizes(u_, A_, B_, step)), bf16(io_type(u_, "u")) {
        on_gpu(u_, "u");
        const auto io = u_.scalar_type();
        const auto dev = u_.device();
        const auto sh = u_.sizes();
        const int64_t bc4[4] = {z.N, z.G, z.L, z.S}, bc3[3] = {z.N, z.G, z.S};
        const IntArrayRef bc = step ? IntArrayRef(bc3, 3) : IntArrayRef(bc4, 4);
        u = Rows(u_);
        delta = rows_in(delta_, "delta", sh, io, dev);
        zz = rows_in(z_, "z", sh, io, dev);
        B = rows_in(B_, "B", bc, io, dev);
        C = rows_in(C_, "C", bc, io, dev);
        A = dense_in(A_, "A", {z.H, z.E, z.S}, at::kFloat, dev);
        D = dense_in(D_, "D", {z.H, z.E}, at::kFloat, dev);
        bias = dense_in(bias_, "delta_bias", {z.H, z.E}, at::kFloat, dev);
        if (step) keep = dense_in(keep_, "keep", {z.N}, at::kFloat, dev);
        else keep = dense_in(keep_, "keep", {z.N, z.L}, at::kFloat, dev);
        lengths = dense_in(lengths_, "lengths", {z.N}, at::kInt, dev);
    }
    bool empty() const { return z.N * z.H * z.L * z.E * z.S == 0; }
    IntArrayRef state_shape() { return shape4 = {z.N, z.H, z.E, z.S}, IntArrayRef(shape4); }
    std::array<int64_t, 4> shape4;
};
int64_t scan_workspace(const ScanSizes &z, int backward) {
    int64_t n[1];
    check_code(selective_scan_workspace(n, z.N, z.H, z.L, z.E, z.S, z.G, backward), "selective_scan_workspace");
    return n[0];
}
// what no entry point could count in its ints
void check_ints(std::initializer_list<int64_t> sizes) {
    for (const int64_t s : sizes) TORCH_CHECK_VALUE(s <= INT32_MAX, "a size of ", s, " does not fit the kernels");
}

std::tuple<Tensor, Tensor, Tensor> scan_forward(ScanIn &in, const Tensor &state_, bool softplus, bool save) {
    const ScanSizes &z = in.z;
    const Tensor &u = in.u.t;
    if (save && !in.empty()) {   // what the backward could not take is refused in front of it
        check_ints({z.N, z.H, z.L, z.E, z.S});
        scan_workspace(z, 1);
    }
    const Tensor state = dense_in(state_, "state", in.state_shape(), at::kFloat, u.device());
    Tensor out = rows_like(u), last = at::empty(in.state_shape(), f32_on(u));
    Tensor saved = save ? at::empty({z.N, (z.L + 15) / 16, z.H * z.E, z.S}, f32_on(u)) : Tensor();
    if (in.empty()) {
        out.zero_();
        if (state.defined()) last.copy_(state);
        else last.zero_();
        return {out, last, saved};
    }
    check_ints({z.N, z.H, z.L, z.E, z.S});
    const c10::DeviceGuard guard(u.device());
    const Tensor work = floats(scan_workspace(z, 0), u);
    const Rows o(out);
    const unsigned flags = softplus ? SRWM_FLAG_SOFTPLUS : 0;
    auto call = [&](auto *fn, auto *type) {
        using T = std::remove_pointer_t<decltype(type)>;
        return fn(in.u.ptr<T>(), in.u.st, in.delta.ptr<T>(), in.delta.st, in.zz.ptr<T>(), in.zz.strides(), in.B.ptr<T>(), in.B.st,
                  in.C.ptr<T>(), in.C.st, ptr<float>(in.A), ptr<float>(in.D), ptr<float>(in.bias), ptr<float>(state),
                  ptr<float>(in.keep), ptr<int>(in.lengths), o.ptr<T>(), o.st, ptr<float>(last), ptr<float>(saved),
                  ptr<float>(work), z.N, z.H, z.L, z.E, z.S, z.G, flags, stream_of(u));
    };
    check_code(in.bf16 ? call(selective_scan_forward_bf16, (uint16_t *)nullptr) : call(selective_scan_forward_f32, (float *)nullptr),
               "selective_scan_forward");
    return {out, last, saved};
}

// gradients of u, delta, A, B, C, D, z, delta_bias, state
variable_list scan_backward(ScanIn &in, const Tensor &saved, const Tensor &grad_out, const Tensor &grad_last, bool softplus,
                            bool with_state) {
    const ScanSizes &z = in.z;
    const Tensor &u = in.u.t;
    const auto dev = u.device();
    const Rows go = rows_in(grad_out, "grad_out", u.sizes(), u.scalar_type(), dev);
    const Tensor glast = dense_in(grad_last, "grad_last", in.state_shape(), at::kFloat, dev);
    const Rows gu(rows_like(u)), gd(rows_like(in.delta.t)), gB(rows_like(in.B.t)), gC(rows_like(in.C.t));
    const Rows gz = in.zz.t.defined() ? Rows(rows_like(in.zz.t)) : Rows();
    const Tensor gA = at::empty_like(in.A), gD = like_or_none(in.D), gbias = like_or_none(in.bias);
    const Tensor gstate = with_state ? at::empty(in.state_shape(), f32_on(u)) : Tensor();
    if (in.empty()) {
        for (const Tensor &t : {gu.t, gd.t, gz.t, gB.t, gC.t, gA, gD, gbias})
            if (t.defined()) t.zero_();
        if (gstate.defined() && glast.defined()) gstate.copy_(glast);
        else if (gstate.defined()) gstate.zero_();
    } else {
        const c10::DeviceGuard guard(dev);
        const Tensor work = floats(scan_workspace(z, 1), u);
        const unsigned flags = softplus ? SRWM_FLAG_SOFTPLUS : 0;
        auto call = [&](auto *fn, auto *type) {
            using T = std::remove_pointer_t<decltype(type)>;
            return fn(in.u.ptr<T>(), in.u.st, in.delta.ptr<T>(), in.delta.st, in.zz.ptr<T>(), in.zz.strides(), in.B.ptr<T>(),
                      in.B.st, in.C.ptr<T>(), in.C.st, ptr<float>(in.A), ptr<float>(in.D), ptr<float>(in.bias),
                      ptr<float>(in.keep), ptr<int>(in.lengths), ptr<float>(saved), go.ptr<T>(), go.st, ptr<float>(glast),
                      gu.ptr<T>(), gu.st, gd.ptr<T>(), gd.st, gz.ptr<T>(), gz.strides(), gB.ptr<T>(), gB.st, gC.ptr<T>(), gC.st,
                      ptr<float>(gA), ptr<float>(gD), ptr<float>(gbias), ptr<float>(gstate), ptr<float>(work), z.N, z.H, z.L, z.E,
                      z.S, z.G, flags, stream_of(u));
        };
        check_code(in.bf16 ? call(selective_scan_backward_bf16, (uint16_t *)nullptr) : call(selective_scan_backward_f32, (float *)nullptr),
                   "selective_scan_backward");
    }
    return {gu.t, gd.t, gA, gB.t, gC.t, gD, gz.t, gbias, gstate};
}

// The states of every 16th step are kept for the backward.
struct SelectiveScan : Function<SelectiveScan> {
    static variable_list forward(AutogradContext *ctx, const Tensor &u, const Tensor &delta, const Tensor &A, const Tensor &B,
                                 const Tensor &C, const MaybeTensor &D_, const MaybeTensor &z_, const MaybeTensor &bias_,
                                 const MaybeTensor &state_, const MaybeTensor &keep_, const MaybeTensor &lengths_, bool softplus) {
        const Tensor D = or_none(D_), z = or_none(z_), bias = or_none(bias_), state = or_none(state_), keep = or_none(keep_),
                     lengths = or_none(lengths_);
        ScanIn in(u, delta, A, B, C, D, z, bias, keep, lengths, false);
        auto [out, last, saved] = scan_forward(in, state, softplus, true);
        ctx->set_materialize_grads(false);
        ctx->save_for_backward({u, delta, A, B, C, D, z, bias, keep, lengths, saved});
        ctx->saved_data["softplus"] = softplus;
        ctx->saved_data["state"] = state.defined();
        return {out, last};
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        plain_call("the backward of selective_scan", {grads[0], grads[1]});
        const variable_list s = ctx->get_saved_variables();
        ScanIn in(s[0], s[1], s[2], s[3], s[4], s[5], s[6], s[7], s[8], s[9], false);
        const Tensor go = grads[0].defined() ? grads[0] : at::zeros_like(s[0]);
        variable_list g = scan_backward(in, s[10], go, grads[1], ctx->saved_data["softplus"].toBool(), ctx->saved_data["state"].toBool());
        g.resize(12);
        return once_differentiable(std::move(g), "selective_scan", grads);
    }
};

std::tuple<Tensor, Tensor> selective_scan(const Tensor &u, const Tensor &delta, const Tensor &A, const Tensor &B, const Tensor &C,
                                          const MaybeTensor &D_, const MaybeTensor &z_, const MaybeTensor &bias_,
                                          const MaybeTensor &state_, const MaybeTensor &keep_, const MaybeTensor &lengths_,
                                          bool softplus) {
    const Tensor D = or_none(D_), z = or_none(z_), bias = or_none(bias_), state = or_none(state_), keep = or_none(keep_),
                 lengths = or_none(lengths_);
    plain_call("selective_scan", {u, delta, A, B, C, D, z, bias, state});
    if (wants_grad({u, delta, A, B, C, D, z, bias, state})) {
        not_held_outside("selective_scan", {u, delta, A, B, C, D, z, bias, state});
        const variable_list r = SelectiveScan::apply(u, delta, A, B, C, D_, z_, bias_, state_, keep_, lengths_, softplus);
        return {r[0], r[1]};
    }
    ScanIn in(u, delta, A, B, C, D, z, bias, keep, lengths, false);
    const at::NoGradGuard none;
    auto [out, last, saved] = scan_forward(in, state, softplus, false);
    return {out, last};
}

Tensor selective_scan_step(const Tensor &u, const Tensor &delta, const Tensor &state, const Tensor &A, const Tensor &B,
                           const Tensor &C, const MaybeTensor &D_, const MaybeTensor &z_, const MaybeTensor &bias_,
                           const MaybeTensor &keep_, bool softplus) {
    const Tensor D = or_none(D_), z = or_none(z_), bias = or_none(bias_);
    plain_call("selective_scan_step", {u, delta, A, B, C, D, z, bias, state});
    TORCH_CHECK(!wants_grad({u, delta, A, B, C, D, z, bias, state}),
                "selective_scan_step has no backward: call it under torch.no_grad(), or selective_scan with L = 1");
    const at::NoGradGuard none;
    ScanIn in(u, delta, A, B, C, D, z, bias, or_none(keep_), Tensor(), true);
    const ScanSizes &s = in.z;
    fits(state, "state", in.state_shape(), at::kFloat, u.device());
    const Tensor out = at::empty(u.sizes(), u.options());
    if (in.empty()) return out.zero_();
    check_ints({s.N, s.H, s.E, s.S});
    const c10::DeviceGuard guard(u.device());
    Overwritten h(state);
    const Rows o(out);
    const unsigned flags = softplus ? SRWM_FLAG_SOFTPLUS : 0;
    auto call = [&](auto *fn, auto *type) {
        using T = std::remove_pointer_t<decltype(type)>;
        return fn(in.u.ptr<T>(), in.u.st, in.delta.ptr<T>(), in.delta.st, in.zz.ptr<T>(), in.zz.strides(), in.B.ptr<T>(), in.B.st,
                  in.C.ptr<T>(), in.C.st, ptr<float>(in.A), ptr<float>(in.D), ptr<float>(in.bias), ptr<float>(in.keep),
                  ptr<float>(h.work), o.ptr<T>(), o.st, s.N, s.H, s.E, s.S, s.G, flags, stream_of(u));
    };
    check_code(in.bf16 ? call(selective_scan_step_bf16, (uint16_t *)nullptr) : call(selective_scan_step_f32, (float *)nullptr),
               "selective_scan_step");
    h.done();
    return out;
}

// ---- convolution
struct ConvIn {
    int64_t N, H, L, E, W;
    bool bf16;
    Rows x;
    Tensor weight, bias, keep, lengths;
    ConvIn(const Tensor &x_, const Tensor &weight_, const Tensor &bias_, const Tensor &keep_, const Tensor &lengths_, bool step) {
        const int nd = step ? 3 : 4;
        TORCH_CHECK_VALUE(x_.dim() == nd && weight_.dim() == 3,
                          step ? "x must be (N, H, E), weight (H, E, W)" : "x must be (N, H, L, E), weight (H, E, W)");
        N = x_.size(0), H = x_.size(1), L = step ? 1 : x_.size(2), E = x_.size(nd - 1), W = weight_.size(2);
        bf16 = io_type(x_, "x");
        on_gpu(x_, "x");
        TORCH_CHECK_VALUE(W >= 2 && W <= 4, "the convolution has 2 to 4 taps (got ", W, ")");
        const auto dev = x_.device();
        x = Rows(x_);
        weight = dense_in(weight_, "weight", {H, E, W}, at::kFloat, dev);
        bias = dense_in(bias_, "bias", {H, E}, at::kFloat, dev);
        if (step) keep = dense_in(keep_, "keep", {N}, at::kFloat, dev);
        else keep = dense_in(keep_, "keep", {N, L}, at::kFloat, dev);
        lengths = dense_in(lengths_, "lengths", {N}, at::kInt, dev);
    }
    bool empty() const { return N * H * L * E == 0; }
    Tensor carried(const Tensor &t, const char *name) const {
        return dense_in(t, name, {N, H, W - 1, E}, x.t.scalar_type(), x.t.device());
    }
};

std::tuple<Tensor, Tensor> conv_forward(const ConvIn &in, const Tensor &state_, bool silu) {
    const Tensor &x = in.x.t;
    const Tensor state = in.carried(state_, "state");
    Tensor out = rows_like(x), last = at::empty({in.N, in.H, in.W - 1, in.E}, x.options());
    if (in.empty()) {
        if (state.defined()) last.copy_(state);
        else last.zero_();
        return {out, last};
    }
    check_ints({in.N, in.H, in.L, in.E});
    const c10::DeviceGuard guard(x.device());
    const Rows o(out);
    auto call = [&](auto *fn, auto *type) {
        using T = std::remove_pointer_t<decltype(type)>;
        return fn(in.x.ptr<T>(), in.x.st, ptr<float>(in.weight), ptr<float>(in.bias), ptr<T>(state), ptr<float>(in.keep),
                  ptr<int>(in.lengths), o.ptr<T>(), o.st, ptr<T>(last), in.N, in.H, in.L, in.E, in.W, silu ? SRWM_FLAG_SILU : 0,
                  stream_of(x));
    };
    check_code(in.bf16 ? call(causal_conv_forward_bf16, (uint16_t *)nullptr) : call(causal_conv_forward_f32, (float *)nullptr),
               "causal_conv_forward");
    return {out, last};
}

struct CausalConv : Function<CausalConv> {
    static variable_list forward(AutogradContext *ctx, const Tensor &x, const Tensor &weight, const MaybeTensor &bias_,
                                 const MaybeTensor &state_, const MaybeTensor &keep_, const MaybeTensor &lengths_, bool silu) {
        const Tensor bias = or_none(bias_), state = or_none(state_), keep = or_none(keep_), lengths = or_none(lengths_);
        const ConvIn in(x, weight, bias, keep, lengths, false);
        auto [out, last] = conv_forward(in, state, silu);
        ctx->set_materialize_grads(false);
        ctx->save_for_backward({x, weight, bias, state, keep, lengths});
        ctx->saved_data["silu"] = silu;
        return {out, last};
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        plain_call("the backward of causal_conv", {grads[0], grads[1]});
        const variable_list s = ctx->get_saved_variables();
        const ConvIn in(s[0], s[1], s[2], s[4], s[5], false);
        const Tensor &x = in.x.t;
        const Tensor state = in.carried(s[3], "state"), glast = in.carried(grads[1], "grad_last");
        const Rows go = rows_in(grads[0].defined() ? grads[0] : at::zeros_like(s[0]), "grad_out", x.sizes(), x.scalar_type(), x.device());
        const Rows gx(rows_like(x));
        const Tensor gw = at::empty_like(in.weight), gb = like_or_none(in.bias), gs = like_or_none(state);
        if (in.empty()) {
            gw.zero_();
            if (gb.defined()) gb.zero_();
            if (gs.defined() && glast.defined()) gs.copy_(glast);
            else if (gs.defined()) gs.zero_();
        } else {
            const c10::DeviceGuard guard(x.device());
            int64_t n[1];
            check_code(causal_conv_workspace(n, in.N, in.H, in.L, in.E, in.W), "causal_conv_workspace");
            const Tensor work = floats(n[0], x);
            const bool silu = ctx->saved_data["silu"].toBool();
            auto call = [&](auto *fn, auto *type) {
                using T = std::remove_pointer_t<decltype(type)>;
                return fn(in.x.ptr<T>(), in.x.st, ptr<float>(in.weight), ptr<float>(in.bias), ptr<T>(state), ptr<float>(in.keep),
                          ptr<int>(in.lengths), go.ptr<T>(), go.st, ptr<T>(glast), gx.ptr<T>(), gx.st, ptr<float>(gw), ptr<float>(gb),
                          ptr<T>(gs), ptr<float>(work), in.N, in.H, in.L, in.E, in.W, silu ? SRWM_FLAG_SILU : 0, stream_of(x));
            };
            check_code(in.bf16 ? call(causal_conv_backward_bf16, (uint16_t *)nullptr) : call(causal_conv_backward_f32, (float *)nullptr),
                       "causal_conv_backward");
        }
        return once_differentiable({gx.t, gw, gb, gs, Tensor(), Tensor(), Tensor()}, "causal_conv", grads);
    }
};

std::tuple<Tensor, Tensor> causal_conv(const Tensor &x, const Tensor &weight, const MaybeTensor &bias_, const MaybeTensor &state_,
                                       const MaybeTensor &keep_, const MaybeTensor &lengths_, bool silu) {
    const Tensor bias = or_none(bias_), state = or_none(state_), keep = or_none(keep_), lengths = or_none(lengths_);
    plain_call("causal_conv", {x, weight, bias, state});
    if (wants_grad({x, weight, bias, state})) {
        not_held_outside("causal_conv", {x, weight, bias, state});
        const variable_list r = CausalConv::apply(x, weight, bias_, state_, keep_, lengths_, silu);
        return {r[0], r[1]};
    }
    const at::NoGradGuard none;
    return conv_forward(ConvIn(x, weight, bias, keep, lengths, false), state, silu);
}

Tensor causal_conv_step(const Tensor &x, const Tensor &state, const Tensor &weight, const MaybeTensor &bias_, const MaybeTensor &keep_,
                        bool silu) {
    const Tensor bias = or_none(bias_);
    plain_call("causal_conv_step", {x, weight, bias, state});
    TORCH_CHECK(!wants_grad({x, weight, bias, state}),
                "causal_conv_step has no backward: call it under torch.no_grad(), or causal_conv with L = 1");
    const at::NoGradGuard none;
    const ConvIn in(x, weight, bias, or_none(keep_), Tensor(), true);
    fits(state, "state", {in.N, in.H, in.W - 1, in.E}, x.scalar_type(), x.device());
    const Tensor out = at::empty(x.sizes(), x.options());
    if (in.empty()) return out;
    check_ints({in.N, in.H, in.E});
    const c10::DeviceGuard guard(x.device());
    Overwritten h(state);
    const Rows o(out);
    auto call = [&](auto *fn, auto *type) {
        using T = std::remove_pointer_t<decltype(type)>;
        return fn(in.x.ptr<T>(), in.x.st, ptr<float>(in.weight), ptr<float>(in.bias), ptr<float>(in.keep), ptr<T>(h.work), o.ptr<T>(),
                  o.st, in.N, in.H, in.E, in.W, silu ? SRWM_FLAG_SILU : 0, stream_of(x));
    };
    check_code(in.bf16 ? call(causal_conv_step_bf16, (uint16_t *)nullptr) : call(causal_conv_step_f32, (float *)nullptr),
               "causal_conv_step");
    h.done();
    return out;
}

// ---- norm
constexpr int64_t kNormBackwardMax = 16384;

struct NormIn {
    bool bf16;
    at::ScalarType rtype;
    Tensor x, residual, weight;
    int64_t rows, D;
    unsigned flags;
    NormIn(const Tensor &x_, const Tensor &residual_, const Tensor &weight_) {
        bf16 = io_type(x_, "x");
        TORCH_CHECK_VALUE(x_.dim() > 0 && x_.size(-1) > 0, "x must have a last axis to normalise over");
        on_gpu(x_, "x");
        const auto dev = x_.device();
        rtype = x_.scalar_type();
        x = dense_in(x_, "x", x_.sizes(), rtype, dev);
        if (residual_.defined()) {
            rtype = residual_.scalar_type();
            io_type(residual_, "residual");
            TORCH_CHECK_TYPE(bf16 || rtype == at::kFloat, "a float32 x takes a float32 residual");
            residual = dense_in(residual_, "residual", x_.sizes(), rtype, dev);
        }
        D = x_.size(-1);
        rows = x_.numel() / D;
        weight = dense_in(weight_, "weight", {D}, at::kFloat, dev);
        flags = bf16 && rtype == at::kFloat ? SRWM_FLAG_RESIDUAL_F32 : 0;
        check_ints({rows, D});
    }
    Tensor sum() const { return residual.defined() ? at::empty(x.sizes(), x.options().dtype(rtype)) : x; }
};

// out, sum (x itself without a residual), the rows' reciprocal norms (undefined without `save`)
std::tuple<Tensor, Tensor, Tensor> norm_forward(const NormIn &in, double eps_, bool save) {
    const Tensor out = at::empty(in.x.sizes(), in.x.options()), sum = in.sum();
    const Tensor rstd = save ? at::empty({in.rows}, f32_on(in.x)) : Tensor();
    const float eps[1] = {(float)eps_};
    if (in.rows) {
        const c10::DeviceGuard guard(in.x.device());
        void *s = in.residual.defined() ? sum.data_ptr() : nullptr;
        const int code =
            in.bf16 ? residual_rms_norm_forward_bf16(ptr<uint16_t>(in.x), ptr<void>(in.residual), ptr<float>(in.weight),
                                                     ptr<uint16_t>(out), s, ptr<float>(rstd), eps, in.rows, in.D, in.flags, stream_of(in.x))
                    : residual_rms_norm_forward_f32(ptr<float>(in.x), ptr<void>(in.residual), ptr<float>(in.weight), ptr<float>(out), s,
                                                    ptr<float>(rstd), eps, in.rows, in.D, in.flags, stream_of(in.x));
        check_code(code, "residual_rms_norm_forward");
    }
    return {out, sum, rstd};
}

struct ResidualRMSNorm : Function<ResidualRMSNorm> {
    static variable_list forward(AutogradContext *ctx, const Tensor &x, const MaybeTensor &residual_, const Tensor &weight, double eps) {
        const Tensor residual = or_none(residual_);
        const NormIn in(x, residual, weight);
        auto [out, sum, rstd] = norm_forward(in, eps, true);
        ctx->set_materialize_grads(false);
        ctx->save_for_backward({residual.defined() ? sum : x, weight, rstd});
        ctx->saved_data["residual"] = residual.defined();
        ctx->saved_data["bf16"] = in.bf16;
        if (residual.defined()) return {out, sum};
        return {out};
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        const variable_list s = ctx->get_saved_variables();
        const bool with_residual = ctx->saved_data["residual"].toBool();
        plain_call("the backward of residual_rms_norm", {grads[0], with_residual ? grads[1] : Tensor()});
        const auto io = ctx->saved_data["bf16"].toBool() ? at::kBFloat16 : at::kFloat;
        return run(s[0].contiguous(), s[1], s[2], grads[0], with_residual ? grads[1] : Tensor(), io, with_residual, s[0].device());
    }
    static variable_list run(const Tensor &total_, const Tensor &weight_, const Tensor &rstd, const Tensor &go_, const Tensor &gt_,
                             at::ScalarType io, bool with_residual, const at::Device &dev) {
        const Tensor total = aligned(total_) ? total_ : total_.clone();
        const auto rtype = total.scalar_type();
        const int64_t D = total.size(-1), rows = total.numel() / D;
        const Tensor weight = dense_in(weight_, "weight", {D}, at::kFloat, dev);
        const Tensor go = go_.defined() ? dense_in(go_, "grad_out", total.sizes(), io, dev) : at::zeros(total.sizes(), total.options().dtype(io));
        const Tensor gt = dense_in(gt_, "grad_total", total.sizes(), rtype, dev);
        const Tensor gx = at::empty(total.sizes(), total.options().dtype(io));
        const Tensor gr = with_residual ? at::empty(total.sizes(), total.options()) : Tensor();
        const Tensor gw = at::empty_like(weight);
        if (rows) {
            const c10::DeviceGuard guard(dev);
            int64_t n[1];
            check_code(residual_rms_norm_workspace(n, rows, D), "residual_rms_norm_workspace");
            const Tensor work = floats(n[0], total);
            const unsigned flags = io == at::kBFloat16 && rtype == at::kFloat ? SRWM_FLAG_RESIDUAL_F32 : 0;
            const int code =
                io == at::kBFloat16
                    ? residual_rms_norm_backward_bf16(ptr<void>(total), ptr<float>(weight), ptr<float>(rstd), ptr<uint16_t>(go),
                                                      ptr<void>(gt), ptr<uint16_t>(gx), ptr<void>(gr), ptr<float>(gw), ptr<float>(work),
                                                      rows, D, flags, stream_of(total))
                    : residual_rms_norm_backward_f32(ptr<void>(total), ptr<float>(weight), ptr<float>(rstd), ptr<float>(go), ptr<void>(gt),
                                                     ptr<float>(gx), ptr<void>(gr), ptr<float>(gw), ptr<float>(work), rows, D, flags,
                                                     stream_of(total));
            check_code(code, "residual_rms_norm_backward");
        } else {
            gw.zero_();
        }
        return once_differentiable({gx, gr, gw, Tensor()}, "residual_rms_norm", {go_, gt_});
    }
};

std::tuple<Tensor, Tensor> residual_rms_norm(const Tensor &x, const MaybeTensor &residual_, const Tensor &weight, double eps) {
    const Tensor residual = or_none(residual_);
    plain_call("residual_rms_norm", {x, residual, weight});
    if (wants_grad({x, residual, weight})) {
        TORCH_CHECK_VALUE(x.dim() == 0 || x.size(-1) <= kNormBackwardMax, "residual_rms_norm has no backward for rows longer than ",
                          kNormBackwardMax);
        not_held_outside("residual_rms_norm", {x, residual, weight});
        const variable_list r = ResidualRMSNorm::apply(x, residual_, weight, eps);
        return {r[0], residual.defined() ? r[1] : x};
    }
    const at::NoGradGuard none;
    const NormIn in(x, residual, weight);
    auto [out, sum, rstd] = norm_forward(in, eps, false);
    return {out, residual.defined() ? sum : x};
}

std::tuple<Tensor, Tensor, Tensor> residual_rms_norm_e4m3(const Tensor &x, const MaybeTensor &residual_, const Tensor &weight, double eps_) {
    const Tensor residual = or_none(residual_);
    plain_call("residual_rms_norm_e4m3", {x, residual, weight});
    TORCH_CHECK(!wants_grad({x, residual, weight}), "residual_rms_norm_e4m3 has no backward: call it under torch.no_grad()");
    const at::NoGradGuard none;
    const NormIn in(x, residual, weight);
    const Tensor out = at::empty(x.sizes(), x.options().dtype(at::kFloat8_e4m3fn)), sum = in.sum();
    auto shape = x.sizes().vec();
    shape.back() = 1;
    const Tensor scale = at::empty(shape, f32_on(x));
    const float eps[1] = {(float)eps_};
    if (in.rows) {
        const c10::DeviceGuard guard(x.device());
        void *s = residual.defined() ? sum.data_ptr() : nullptr;
        const int code =
            in.bf16 ? residual_rms_norm_e4m3_bf16(ptr<uint16_t>(in.x), ptr<void>(in.residual), ptr<float>(in.weight), ptr<uint8_t>(out),
                                                  ptr<float>(scale), s, eps, in.rows, in.D, in.flags, stream_of(x))
                    : residual_rms_norm_e4m3_f32(ptr<float>(in.x), ptr<void>(in.residual), ptr<float>(in.weight), ptr<uint8_t>(out),
                                                 ptr<float>(scale), s, eps, in.rows, in.D, in.flags, stream_of(x));
        check_code(code, "residual_rms_norm_e4m3");
    }
    return {out, scale, residual.defined() ? sum : x};
}

}  // namespace

PYBIND11_MODULE(srwm_torch, m) {
    using release = py::call_guard<py::gil_scoped_release>;
    m.def("abi_version", &srwm_hip_abi_version);
    m.def("not_held_outside", [](const std::string &what, const std::vector<Tensor> &ts) { not_held_outside(what.c_str(), ts); });
    m.def("rows_like", &rows_like, release());
    m.def("selective_scan", &selective_scan, release());
    m.def("selective_scan_step", &selective_scan_step, release());
    m.def("causal_conv", &causal_conv, release());
    m.def("causal_conv_step", &causal_conv_step, release());
    m.def("residual_rms_norm", &residual_rms_norm, release());
    m.def("residual_rms_norm_e4m3", &residual_rms_norm_e4m3, release());
}
