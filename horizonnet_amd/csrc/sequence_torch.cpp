// The sequence operators on torch tensors: argument checks, workspaces, autograd nodes over the C entry points of libhorizonnet_hip.so.
//
// Small calls are bound by the host: the same calls through ctypes and Python autograd functions took 10.0 us for a single step (B 1, C 1024)
// against 4.2 here, and 86 us for dropout's forward and backward pass against 48: a node here runs in the engine's thread without the interpreter.
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/accumulate_grad.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/extension.h>

#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/AutogradState.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>

#include <unordered_set>
#include <vector>

#include "../../include/horizonnet_hip.h"

namespace {

using torch::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// a failed entry point: HipEngineError in Python (a RuntimeError)
struct EngineError : std::runtime_error {
    using std::runtime_error::runtime_error;
};
void check(int rc, const char* what)
{
    if (rc != 0) {
        const char* msg = hn_last_error();
        throw EngineError(std::string(what) + " failed (rc=" + std::to_string(rc) + "): " + (msg ? msg : "?"));
    }
}

void* stream_of(const Tensor& t) { return (void*)c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.get_device()).stream(); }
template <class T = void>
T* addr(const Tensor& t)
{
    return t.defined() ? static_cast<T*>(t.data_ptr()) : nullptr;
}
int dtype_of(const Tensor& t) { return t.scalar_type() == at::kBFloat16 ? 1 : 0; }

// What sees torch's own operations alone has to be told: a tangent would be dropped, which counts as zero, and a trace would keep the outputs' memory
// without what fills it
void check_seen(const char* who, std::initializer_list<const Tensor*> ts)
{
    TORCH_CHECK(!torch::jit::tracer::isTracing() && !c10::impl::TorchDispatchModeTLS::get_mode(c10::impl::TorchDispatchModeKey::PROXY), who,
                " cannot be traced: a trace does not record its kernels");
    if (!c10::AutogradState::get_tls_state().get_fw_grad_mode()) return;
    for (const Tensor* t : ts)
        TORCH_CHECK(!t || !t->defined() || !t->_fw_grad(0).defined(), who, " has no forward-mode derivative");
}
template <class Optional>
const Tensor* in(const Optional& t) { return t ? &*t : nullptr; }

void check_main(const char* who, const char* name, const Tensor& t)
{
    TORCH_CHECK(t.is_cuda(), who, " needs cuda/ROCm tensors (no CPU fallback): ", name, " is on ", t.device());
    TORCH_CHECK_VALUE(t.scalar_type() == at::kFloat || t.scalar_type() == at::kBFloat16, who, ": ", name, " is ", t.scalar_type(),
                      "; float32 and bfloat16 are supported");
}
void check_like(const char* who, const char* name, const Tensor& t, at::IntArrayRef shape, at::ScalarType dtype, at::Device device)
{
    TORCH_CHECK(t.device() == device, who, ": ", name, " is on ", t.device(), ", expected ", device);
    TORCH_CHECK_VALUE(t.scalar_type() == dtype, who, ": ", name, " is ", t.scalar_type(), ", expected ", dtype);
    TORCH_CHECK_VALUE(t.sizes() == shape, who, ": ", name, " has shape ", t.sizes(), ", expected ", shape);
}
// What a kernel reads: a view whose sign is pending (torch's imaginary part of a conjugate is one, and so is the gradient that reaches an imaginary part) is
// copied with its sign
Tensor plain(const Tensor& t) { return t.defined() && t.is_neg() ? t.resolve_neg() : t; }
// channels next to each other; the other axes as they are
Tensor rows(const Tensor& t_)
{
    const Tensor t = plain(t_);
    return !t.defined() || t.size(-1) <= 1 || t.stride(-1) == 1 ? t : t.contiguous();
}
Tensor whole(const Tensor& t) { return t.defined() ? plain(t).contiguous() : t; }
// row stride of a matrix; of a single row any: the one that keeps it aligned
int64_t row_stride(const Tensor& t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); }
int64_t stride_of(const Tensor& t, int axis) { return t.defined() ? t.stride(axis) : 0; }
// An input that may be missing goes to an autograd node as std::optional: the node takes the defined ones alone as its edges, in order
typedef std::optional<Tensor> Maybe;
Maybe maybe(const Tensor& t) { return t.defined() ? Maybe(t) : std::nullopt; }
Tensor open(const Maybe& t) { return t ? *t : Tensor(); }
bool wants_grad(std::initializer_list<const Tensor*> ts)
{
    if (!at::GradMode::is_enabled()) return false;
    for (const Tensor* t : ts)
        if (t->defined() && t->requires_grad()) return true;
    return false;
}

// The gradients are kernels' outputs: a second derivative through them has to fail instead of being zero
variable_list once(const char* who, variable_list grads)
{
    if (!at::GradMode::is_enabled()) return grads;
    variable_list in;
    for (auto& g : grads) in.push_back(g.defined() ? g.detach().set_requires_grad(true) : g);
    auto node = std::make_shared<torch::autograd::DelayedError>(std::string("trying to differentiate twice a function that is differentiable once: ") + who,
                                                                (int64_t)in.size());
    return (*node)(std::move(in));
}

// A gradient accumulator that an eager graph keeps alive belongs to the stream that graph was made on.  On its way there a captured backward
// pass would draw the default stream into the capture, which ends the process: refused before that.  The operator's own leaves count, and every node
// that this pass will run behind it (the leaf may lie behind a reshaped batch, the copy of an input whose channels lie apart, a cast weight)
bool draws_default_stream(torch::autograd::Node* node)
{
    std::vector<torch::autograd::Node*> todo{node};
    std::unordered_set<torch::autograd::Node*> seen;
    while (!todo.empty()) {
        const auto at = todo.back();
        todo.pop_back();
        for (size_t i = 0; i < at->num_outputs(); ++i) {
            const auto next = at->next_edge(i).function.get();
            if (!next) continue;
            const bool run = at->task_should_compute_output(i);
            if (run || (at == node && dynamic_cast<torch::autograd::AccumulateGrad*>(next))) {
                const auto its = next->stream();
                if (its && its->id() == 0) return true;
            }
            if (run && seen.insert(next).second) todo.push_back(next);
        }
    }
    return false;
}
void check_capture(const char* who, const Tensor& t)
{
    const auto stream = c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.get_device());
    hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
    if (hipStreamIsCapturing(stream.stream(), &status) != hipSuccess || status == hipStreamCaptureStatusNone) return;
    const auto node = torch::autograd::get_current_node();
    if (!node) return;
    TORCH_CHECK(!draws_default_stream(node.get()), who, ": the backward pass is being captured while a graph made on the default stream holds one of its leaves; "
                "let go of that graph first, or make it on a side stream");
}

// ---- gated linear recurrence ----
struct RecurrenceOut {
    Tensor y, last, states;
};
RecurrenceOut recurrence_forward(const Tensor& f, const Tensor& v, const Tensor& o, const Tensor& h0, const Tensor& lengths, int64_t direction, bool keep)
{
    const c10::DeviceGuard guard(f.device());
    const int64_t T = f.size(0), B = f.size(1), C = f.size(2);
    const auto f32 = f.options().dtype(at::kFloat);
    RecurrenceOut r;
    r.y = at::empty({T, B, C}, f.options());
    r.last = at::empty({B, C}, f32);
    const size_t n = hn_gated_recurrence_workspace(T, B, C, (int)direction);
    Tensor ws;
    if (n) ws = at::empty({(int64_t)n}, f32);
    if (keep) r.states = at::empty({(int64_t)hn_gated_recurrence_states(T, B, C)}, f32);
    check(hn_gated_recurrence(addr(f), f.stride(0), f.stride(1), addr(v), v.stride(0), v.stride(1), addr(o), stride_of(o, 0), stride_of(o, 1), addr<float>(h0),
                              addr<int>(lengths), addr(r.y), addr<float>(r.last), addr<float>(r.states), addr<float>(ws), n, T, B, C, dtype_of(f), (int)direction,
                              stream_of(f)),
          "hn_gated_recurrence");
    return r;
}

struct Recurrence : torch::autograd::Function<Recurrence> {
    static variable_list forward(AutogradContext* ctx, const Tensor& f, const Tensor& v, const Maybe& o_, const Maybe& h0_, const Maybe& lengths_,
                                 int64_t direction)
    {
        const Tensor o = open(o_), h0 = open(h0_), lengths = open(lengths_);
        RecurrenceOut r = recurrence_forward(f, v, o, h0, lengths, direction, true);
        ctx->save_for_backward({f, v, o, lengths, r.states});
        ctx->saved_data["direction"] = direction;
        ctx->saved_data["h0"] = h0.defined();
        ctx->set_materialize_grads(false);
        return {r.y, r.last};
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads)
    {
        const auto saved = ctx->get_saved_variables();
        const Tensor &f = saved[0], &v = saved[1], &o = saved[2], &lengths = saved[3], &states = saved[4];
        const int64_t direction = ctx->saved_data["direction"].toInt();
        const c10::DeviceGuard guard(f.device());
        check_seen("gated_recurrence", {&grads[0], &grads[1]});
        check_capture("gated_recurrence", f);
        const int64_t T = f.size(0), B = f.size(1), C = f.size(2);
        variable_list out(6);
        {
            at::AutoGradMode off(false);
            const auto f32 = f.options().dtype(at::kFloat);
            const Tensor dy = grads[0].defined() ? rows(grads[0]) : at::zeros({T, B, C}, f.options());
            const Tensor dlast = whole(grads[1]);
            out[0] = at::empty({T, B, C}, f.options());
            out[1] = at::empty({T, B, C}, f.options());
            if (o.defined()) out[2] = at::empty({T, B, C}, f.options());
            if (ctx->saved_data["h0"].toBool()) out[3] = at::empty({B, C}, f32);
            const size_t n = hn_gated_recurrence_workspace(T, B, C, (int)direction);
            Tensor ws;
            if (n) ws = at::empty({(int64_t)n}, f32);
            check(hn_gated_recurrence_bwd(addr(f), f.stride(0), f.stride(1), addr(v), v.stride(0), v.stride(1), addr(o), stride_of(o, 0), stride_of(o, 1), addr(dy),
                                          dy.stride(0), dy.stride(1), addr<float>(dlast), addr<int>(lengths), addr<float>(states), addr(out[0]), addr(out[1]),
                                          addr(out[2]), addr<float>(out[3]), addr<float>(ws), n, T, B, C, dtype_of(f), (int)direction, stream_of(f)),
                  "hn_gated_recurrence_bwd");
        }
        return once("gated_recurrence", std::move(out));
    }
};

std::tuple<Tensor, Tensor> gated_recurrence(const Tensor& forget, const Tensor& value, const Maybe& out_gate, const Maybe& h0_,
                                            const Maybe& lengths_, const std::string& direction)
{
    const char* who = "gated_recurrence";
    check_seen(who, {&forget, &value, in(out_gate), in(h0_)});
    check_main(who, "forget", forget);
    TORCH_CHECK_VALUE(forget.dim() == 3, who, ": forget must be [T, B, C], got shape ", forget.sizes());
    const int64_t dir = direction == "forward" ? 0 : direction == "reverse" ? 1 : direction == "both" ? 2 : -1;
    TORCH_CHECK_VALUE(dir >= 0, who, ": direction must be 'forward', 'reverse' or 'both', got '", direction, "'");
    const int64_t T = forget.size(0), B = forget.size(1), C = forget.size(2);
    const auto dev = forget.device();
    const auto dt = forget.scalar_type();
    check_like(who, "value", value, forget.sizes(), dt, dev);
    Tensor o, h0, lengths;
    if (out_gate) { check_like(who, "out_gate", *out_gate, forget.sizes(), dt, dev); o = rows(*out_gate); }
    if (h0_) { check_like(who, "h0", *h0_, {B, C}, at::kFloat, dev); h0 = whole(*h0_); }
    TORCH_CHECK_VALUE(dir != 2 || C % 2 == 0, who, ": direction 'both' needs an even number of channels, got ", C);
    if (lengths_) {
        const auto lt = lengths_->scalar_type();
        TORCH_CHECK_TYPE(lt == at::kInt || lt == at::kLong, who, ": lengths must be an int32 or int64 tensor");
        check_like(who, "lengths", *lengths_, {B}, lt, dev);
        lengths = lt == at::kInt ? whole(*lengths_) : lengths_->clamp(0, T).to(at::kInt);
    }
    const Tensor f = rows(forget), v = rows(value);
    if (wants_grad({&f, &v, &o, &h0})) {
        const auto r = Recurrence::apply(f, v, maybe(o), maybe(h0), maybe(lengths), dir);
        return {r[0], r[1]};
    }
    RecurrenceOut r = recurrence_forward(f, v, o, h0, lengths, dir, false);
    return {r.y, r.last};
}

// Whether t [B, C] shares memory with the contiguous state, other than by being it: a thread reads its own elements alone before it writes them, so
// the same tensor may be both, but not one shifted against the other
bool meets(const Tensor& state, const Tensor& t)
{
    if (!t.defined() || t.numel() == 0) return false;
    const auto s0 = (intptr_t)state.data_ptr(), s1 = s0 + (intptr_t)state.nbytes(), t0 = (intptr_t)t.data_ptr();
    const int64_t size = (int64_t)t.element_size(), B = t.size(0), width = t.size(1) * size, step = t.stride(0) * size;
    if (t0 == s0 && t.scalar_type() == state.scalar_type() && (B == 1 || step == width)) return false;
    const int64_t first = t0 + width > s0 || step == 0 ? 0 : (s0 - t0 - width) / step + 1;         // the first row that ends behind the state's start
    return first < B && t0 + first * step + width > s0 && t0 + first * step < s1;
}

Tensor gated_recurrence_step(const Tensor& forget, const Tensor& value, const Tensor& state, const Maybe& out_gate)
{
    const char* who = "gated_recurrence_step";
    check_seen(who, {&forget, &value, &state, in(out_gate)});
    check_main(who, "forget", forget);
    TORCH_CHECK_VALUE(forget.dim() == 2, who, ": forget must be [B, C], got shape ", forget.sizes());
    const auto dev = forget.device();
    check_like(who, "value", value, forget.sizes(), forget.scalar_type(), dev);
    Tensor o;
    if (out_gate) { check_like(who, "out_gate", *out_gate, forget.sizes(), forget.scalar_type(), dev); o = rows(*out_gate); }
    check_like(who, "state", state, forget.sizes(), at::kFloat, dev);
    TORCH_CHECK_VALUE(state.is_contiguous() && !state.is_neg(), who, ": state is updated in place and must be contiguous");
    TORCH_CHECK(!wants_grad({&forget, &value, &o, &state}), who, " is not differentiable: call it under torch.no_grad() or use gated_recurrence");
    const at::AutoGradMode off(false);
    const Tensor f = rows(forget), v = rows(value);
    TORCH_CHECK(!meets(state, f) && !meets(state, v) && !meets(state, o), who, ": state is updated in place and shares memory with an input");
    const c10::DeviceGuard guard(dev);
    Tensor y = at::empty(forget.sizes(), f.options());
    check(hn_gated_recurrence_step(addr(f), f.stride(0), addr(v), v.stride(0), addr(o), stride_of(o, 0), addr<float>(state), addr(y), f.size(0), f.size(1),
                                   dtype_of(f), stream_of(f)),
          "hn_gated_recurrence_step");
    if (!state.is_inference()) state.unsafeGetTensorImpl()->bump_version();      // a graph that saved the state has to notice
    return y;
}

// ---- gated linear block ----
Tensor linear_forward(const Tensor& x, const Tensor& wg, const Tensor& wu, const Tensor& bg, const Tensor& bu, int64_t act, Tensor* kept)
{
    const c10::DeviceGuard guard(x.device());
    const int64_t M = x.size(0), K = x.size(1), F = wg.size(0);
    Tensor y = at::empty({M, F}, x.options()), ws;
    const size_t n = hn_gated_linear_workspace(addr(x), row_stride(x), addr(wg), row_stride(wg), addr(wu), row_stride(wu), M, K, F, dtype_of(x), 0);
    if (n) ws = at::empty({(int64_t)n}, x.options().dtype(at::kByte));
    if (kept)
        if (const size_t floats = hn_gated_linear_kept(M, K, F, dtype_of(x))) *kept = at::empty({(int64_t)floats}, x.options().dtype(at::kFloat));
    check(hn_gated_linear(addr(x), row_stride(x), addr(wg), row_stride(wg), addr(wu), row_stride(wu), addr(bg), addr(bu), addr(y),
                          kept ? addr<float>(*kept) : nullptr, addr(ws), n, M, K, F, dtype_of(x),
                          (int)act, stream_of(x)),
          "hn_gated_linear");
    return y;
}

struct Linear : torch::autograd::Function<Linear> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& wg, const Tensor& wu, const Maybe& bg_, const Maybe& bu_, int64_t act)
    {
        const Tensor bg = open(bg_), bu = open(bu_);
        Tensor kept;
        const Tensor y = linear_forward(x, wg, wu, bg, bu, act, &kept);
        ctx->save_for_backward({x, wg, wu, bg, bu, kept});
        ctx->saved_data["act"] = act;
        return y;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads)
    {
        const auto saved = ctx->get_saved_variables();
        const Tensor &x = saved[0], &wg = saved[1], &wu = saved[2], &bg = saved[3], &bu = saved[4], &kept = saved[5];
        const c10::DeviceGuard guard(x.device());
        check_seen("gated_linear", {&grads[0]});
        check_capture("gated_linear", x);
        const int64_t M = x.size(0), K = x.size(1), F = wg.size(0);
        variable_list out(6);
        {
            at::AutoGradMode off(false);
            const Tensor dy = rows(grads[0]);
            if (ctx->needs_input_grad(0)) out[0] = at::empty({M, K}, x.options());
            if (ctx->needs_input_grad(1)) out[1] = at::empty({F, K}, x.options());
            if (ctx->needs_input_grad(2)) out[2] = at::empty({F, K}, x.options());
            if (bg.defined() && ctx->needs_input_grad(3)) out[3] = at::empty({F}, x.options());
            if (bu.defined() && ctx->needs_input_grad(bg.defined() ? 4 : 3)) out[4] = at::empty({F}, x.options());
            const size_t n = hn_gated_linear_workspace(addr(x), row_stride(x), addr(wg), row_stride(wg), addr(wu), row_stride(wu), M, K, F, dtype_of(x), 1);
            Tensor ws;
            if (n) ws = at::empty({(int64_t)n}, x.options().dtype(at::kByte));
            check(hn_gated_linear_bwd(addr(x), row_stride(x), addr(wg), row_stride(wg), addr(wu), row_stride(wu), addr(bg), addr(bu), addr(dy), row_stride(dy),
                                      addr<float>(kept), addr(out[0]),
                                      addr(out[1]), addr(out[2]), addr(out[3]), addr(out[4]), addr(ws), n, M, K, F, dtype_of(x),
                                      (int)ctx->saved_data["act"].toInt(), stream_of(x)),
                  "hn_gated_linear_bwd");
        }
        return once("gated_linear", std::move(out));
    }
};

Tensor gated_linear(const Tensor& x, const Tensor& w_gate, const Tensor& w_up, const Maybe& b_gate, const Maybe& b_up,
                    const std::string& activation)
{
    const char* who = "gated_linear";
    check_seen(who, {&x, &w_gate, &w_up, in(b_gate), in(b_up)});
    check_main(who, "x", x);
    TORCH_CHECK_VALUE(x.dim() >= 1, who, ": x must be [..., K]");
    const int64_t act = activation == "silu" ? 0 : activation == "gelu" ? 1 : activation == "sigmoid" ? 2 : activation == "relu" ? 3 : -1;
    TORCH_CHECK_VALUE(act >= 0, who, ": activation must be 'silu', 'gelu', 'sigmoid' or 'relu', got '", activation, "'");
    TORCH_CHECK_VALUE(w_gate.dim() == 2, who, ": w_gate must be [F, K], got shape ", w_gate.sizes());
    const auto dev = x.device();
    const auto dt = x.scalar_type();
    const int64_t K = x.size(-1), F = w_gate.size(0);
    check_like(who, "w_gate", w_gate, {F, K}, dt, dev);
    check_like(who, "w_up", w_up, {F, K}, dt, dev);
    Tensor bg, bu;
    if (b_gate) { check_like(who, "b_gate", *b_gate, {F}, dt, dev); bg = whole(*b_gate); }
    if (b_up) { check_like(who, "b_up", *b_up, {F}, dt, dev); bu = whole(*b_up); }
    int64_t M = 1;
    for (int64_t i = 0; i + 1 < x.dim(); ++i) M *= x.size(i);
    const Tensor x2 = rows(x.dim() == 2 ? x : x.reshape({M, K})), wg = rows(w_gate), wu = rows(w_up);
    const Tensor y = wants_grad({&x2, &wg, &wu, &bg, &bu}) ? Linear::apply(x2, wg, wu, maybe(bg), maybe(bu), act) : linear_forward(x2, wg, wu, bg, bu, act, nullptr);
    if (x.dim() == 2) return y;
    auto shape = x.sizes().vec();
    shape.back() = F;
    return y.view(shape);
}

// ---- dropout ----
Tensor drop(const Tensor& x, const Tensor& residual, double p, uint64_t number, const Tensor& seed)
{
    const c10::DeviceGuard guard(x.device());
    Tensor y = at::empty(x.sizes(), x.options());
    check(hn_dropout(addr(x), addr(residual), addr(y), x.numel(), dtype_of(x), (float)p, number, addr(seed), stream_of(x)), "hn_dropout");
    return y;
}

struct Dropout : torch::autograd::Function<Dropout> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const Maybe& residual_, double p, int64_t number, const Maybe& seed_)
    {
        const Tensor residual = open(residual_), seed = open(seed_);
        ctx->saved_data["residual"] = residual.defined();
        if (seed.defined()) ctx->save_for_backward({seed});
        ctx->saved_data["p"] = p;
        ctx->saved_data["number"] = number;
        ctx->saved_data["tensor"] = seed.defined();
        return drop(x, residual, p, (uint64_t)number, seed);
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads)
    {
        variable_list out(5);
        Tensor seed;
        check_seen("dropout", {&grads[0]});
        check_capture("dropout", grads[0]);
        if (ctx->saved_data["tensor"].toBool()) seed = ctx->get_saved_variables()[0];
        {
            at::AutoGradMode off(false);
            if (ctx->needs_input_grad(0))
                out[0] = drop(whole(grads[0]), Tensor(), ctx->saved_data["p"].toDouble(), (uint64_t)ctx->saved_data["number"].toInt(), seed);
            if (ctx->saved_data["residual"].toBool() && ctx->needs_input_grad(1)) out[1] = grads[0];
        }
        return once("dropout", std::move(out));
    }
};

Tensor dropout(const Tensor& x_, double p, const py::object& seed_, const Maybe& residual_)
{
    const char* who = "dropout";
    check_seen(who, {&x_, in(residual_)});
    check_main(who, "x", x_);
    TORCH_CHECK_VALUE(p >= 0.0 && (float)p < 1.0f, who, ": p must be in [0, 1), got ", p);
    Tensor seed, residual;
    uint64_t number = 0;
    if (THPVariable_Check(seed_.ptr())) {
        seed = plain(THPVariable_Unpack(seed_.ptr()));
        TORCH_CHECK_VALUE(seed.scalar_type() == at::kLong && seed.numel() == 1 && seed.device() == x_.device(), who, ": a seed tensor must be one int64 on ",
                          x_.device(), ", got ", seed.sizes(), " ", seed.scalar_type(), " on ", seed.device());
    } else {
        const py::object whole = PyBool_Check(seed_.ptr()) ? py::object() : py::reinterpret_steal<py::object>(PyNumber_Index(seed_.ptr()));
        if (whole) number = PyLong_AsUnsignedLongLong(whole.ptr());
        if (!whole || PyErr_Occurred()) {
            PyErr_Clear();
            TORCH_CHECK_VALUE(false, who, ": seed must be an int in 0 .. 2**64 - 1 or an int64 tensor");
        }
    }
    py::gil_scoped_release free;
    if (residual_) {
        check_like(who, "residual", *residual_, x_.sizes(), x_.scalar_type(), x_.device());
        residual = whole(*residual_);
    }
    const Tensor x = whole(x_);
    if (wants_grad({&x, &residual})) return Dropout::apply(x, maybe(residual), p, (int64_t)number, maybe(seed));
    return drop(x, residual, p, number, seed);
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m)
{
    static py::object engine_error = py::module_::import("horizonnet_amd._lib").attr("HipEngineError");
    py::register_exception_translator([](std::exception_ptr p) {
        try {
            if (p) std::rethrow_exception(p);
        } catch (const EngineError& e) {
            PyErr_SetString(engine_error.ptr(), e.what());
        }
    });
    using free = py::call_guard<py::gil_scoped_release>;
    m.def("gated_recurrence", &gated_recurrence, free());
    m.def("gated_recurrence_step", &gated_recurrence_step, free());
    m.def("gated_linear", &gated_linear, free());
    m.def("dropout", &dropout);
}
