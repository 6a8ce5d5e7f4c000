// Torch binding of the state-space operators of libtgru.so (tgru_conv_* and tgru_scan_* of include/tgru.h): argument
// checks, memory from torch's caching allocator, torch's current stream of the tensors' device, and the operators as C++
// autograd functions whose backward pass runs in autograd's own thread without entering Python.  timegan_amd/ssm.py
// documents the arguments.
#include <torch/extension.h>
#include <ATen/hip/impl/HIPGuardImplMasqueradingAsCUDA.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>

#include <string>
#include <vector>

#include "tgru.h"

namespace {

using torch::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using OptTensor = c10::optional<Tensor>;

// What Python sees as timegan_amd.TgruError.
struct NoGpu : std::runtime_error { using std::runtime_error::runtime_error; };

void check(int rc, const char *what) {
    TORCH_CHECK(rc == TGRU_OK, what, " failed: ", tgru_error_string(rc), " (", rc, ")");
}

int dtype_code(const Tensor &t, const char *what) {
    switch (t.scalar_type()) {
    case torch::kFloat32: return TGRU_DTYPE_F32;
    case torch::kBFloat16: return TGRU_DTYPE_BF16;
    case torch::kFloat16: return TGRU_DTYPE_F16;
    default: TORCH_CHECK(false, what, " must be float32, bfloat16 or float16, got ", t.scalar_type());
    }
}

std::string shape_of(const Tensor &t) {
    std::string s = "(";
    for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.size(i));
    return s + ")";
}

void require_shape(const Tensor &t, at::IntArrayRef want, const char *what) {
    std::string w = "(";
    for (size_t i = 0; i < want.size(); ++i) w += (i ? ", " : "") + std::to_string(want[i]);
    TORCH_CHECK(t.sizes() == want, what, " must have shape ", w, "), got ", shape_of(t));
}

// A sequence tensor of the call: the element type of the first one, and its device.
void require_like(const Tensor &t, const Tensor &first, const char *what) {
    TORCH_CHECK(t.scalar_type() == first.scalar_type(), what, " must have the element type of the input, ", first.scalar_type(),
                ", got ", t.scalar_type());
    TORCH_CHECK(t.device() == first.device(), what, " is on ", t.device(), ", the input on ", first.device());
}

// A parameter (or a scan state): any floating type, computed with in fp32.
Tensor param(const Tensor &t, const Tensor &first, const char *what) {
    TORCH_CHECK(t.is_floating_point(), what, " must be a floating-point tensor, got ", t.scalar_type());
    TORCH_CHECK(t.device() == first.device(), what, " is on ", t.device(), ", the input on ", first.device());
    return t.to(torch::kFloat32).contiguous();
}

void require_index(const OptTensor &t, int64_t n, const Tensor &first, const char *what) {
    if (!t) return;
    TORCH_CHECK(t->scalar_type() == torch::kInt32 && t->is_contiguous(), what, " must be a dense int32 tensor");
    require_shape(*t, {n}, what);
    TORCH_CHECK(t->device() == first.device(), what, " is on ", t->device(), ", the input on ", first.device());
}

void require_gpu(const Tensor &t) {
    if (!t.is_cuda())
        throw NoGpu("input is on " + t.device().str() + ": the tgru operators only run on a gfx950 GPU and have no CPU fallback");
}

// Consecutive elements in the last dimension (the other strides are passed on as they are).
Tensor rows(const Tensor &t) { return (t.size(-1) == 1 || t.stride(-1) == 1) ? t : t.contiguous(); }
Tensor dense(const Tensor &t) { return t.defined() ? t.contiguous() : t; }
// For the scan also steps that are less than TGRU_SCAN_MAX_ROW_STRIDE elements apart.
Tensor near_rows(const Tensor &t) { return t.stride(1) < TGRU_SCAN_MAX_ROW_STRIDE ? rows(t) : t.clone(at::MemoryFormat::Contiguous); }

// A new tensor of the (B, T, D) shape of `t`, in the order of steps and sequences that `t` has in memory (as far as the
// scan's limit on the distance of two steps allows).  Not a view: autograd forbids to change a view that a function returns.
Tensor like(const Tensor &t) {
    if (t.size(0) > 1 && t.stride(1) > t.stride(0) && t.stride(0) > 0 && t.size(0) * t.size(2) < TGRU_SCAN_MAX_ROW_STRIDE)
        return torch::empty_strided(t.sizes(), {t.size(2), t.size(0) * t.size(2), 1}, t.options());
    return torch::empty(t.sizes(), t.options());
}

const float *fptr(const Tensor &t) { return t.defined() ? t.data_ptr<float>() : nullptr; }
float *fout(const Tensor &t) { return t.defined() ? t.data_ptr<float>() : nullptr; }
const void *ptr(const Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; }
void *out(const Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; }
const int32_t *iptr(const Tensor &t) { return t.defined() ? t.data_ptr<int32_t>() : nullptr; }
void strides2(int64_t (&to)[2], const Tensor &t) {
    if (t.defined()) { to[0] = t.stride(0); to[1] = t.stride(1); }
}
void strides3(int64_t (&to)[3], const Tensor &t) { to[0] = t.stride(0); to[1] = t.stride(1); to[2] = t.stride(2); }

Tensor scratch(size_t bytes, const Tensor &like) {
    return bytes ? torch::empty({(int64_t)(bytes / 4)}, like.options().dtype(torch::kFloat32)) : Tensor();
}

hipStream_t stream_of(const Tensor &t) {
    return c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.device().index()).stream();
}

int as_int(int64_t v, const char *what) {
    TORCH_CHECK(v > 0 && v <= INT32_MAX, what, " must be between 1 and 2^31 - 1, got ", v);
    return (int)v;
}

bool wants(const Tensor &t) { return t.defined() && t.requires_grad(); }

void no_second_derivative(const char *what) {
    TORCH_CHECK(!torch::GradMode::is_enabled(), what, " has no second derivative (backward was called with create_graph=True)");
}

// ---- convolution -----------------------------------------------------------------------------------------------------

tgru_conv_args conv_args(const Tensor &x, const Tensor &weight, const Tensor &bias, const Tensor &initial, const Tensor &lengths, bool silu) {
    tgru_conv_args a{};
    a.x = ptr(x);
    a.weight = fptr(weight);
    a.bias = fptr(bias);
    a.initial_state = (initial.defined() && initial.numel()) ? ptr(initial) : nullptr;
    a.lengths = iptr(lengths);
    strides2(a.x_stride, x);
    a.B = (int)x.size(0);
    a.T = (int)x.size(1);
    a.D = (int)x.size(2);
    a.K = (int)weight.size(1);
    a.dtype = dtype_code(x, "input");
    a.silu = silu;
    return a;
}

class ConvFunction : public torch::autograd::Function<ConvFunction> {
public:
    static variable_list forward(AutogradContext *ctx, const Tensor &x, const Tensor &weight, const OptTensor &bias_, const OptTensor &initial_,
                                 const OptTensor &lengths_, bool silu, bool want_state, bool grad_mode) {
        const Tensor bias = bias_.value_or(Tensor()), initial = initial_.value_or(Tensor()), lengths = lengths_.value_or(Tensor());
        const c10::hip::HIPGuardMasqueradingAsCUDA guard(x.device());
        tgru_conv_args a = conv_args(x, weight, bias, initial, lengths, silu);
        Tensor y = like(x), state;
        if (want_state) state = torch::empty({a.B, a.K - 1, a.D}, x.options());
        a.y = out(y);
        strides2(a.y_stride, y);
        a.final_state = (want_state && a.K > 1) ? out(state) : nullptr;
        check(tgru_conv_forward(&a, stream_of(x)), "tgru_conv_forward");
        const bool need = grad_mode && (wants(x) || wants(weight) || wants(bias) || wants(initial));
        ctx->saved_data["need"] = std::vector<bool>{wants(x), wants(weight), wants(bias), wants(initial)};
        ctx->saved_data["silu"] = silu;
        ctx->set_materialize_grads(false);
        if (need) ctx->save_for_backward({x, weight, bias, initial, lengths});
        if (want_state) return {y, state};
        return {y};
    }

    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        no_second_derivative("short_conv");
        const auto saved = ctx->get_saved_variables();
        const Tensor x = saved[0], weight = saved[1], bias = saved[2], initial = saved[3], lengths = saved[4];
        const auto need = ctx->saved_data["need"].toBoolList();
        const c10::hip::HIPGuardMasqueradingAsCUDA guard(x.device());
        tgru_conv_args a = conv_args(x, weight, bias, initial, lengths, ctx->saved_data["silu"].toBool());
        const Tensor dy = grads[0].defined() ? rows(grads[0]) : Tensor();
        const Tensor dfinal = grads.size() > 1 ? dense(grads[1]) : Tensor();
        a.dy = ptr(dy);
        strides2(a.dy_stride, dy);
        a.dfinal = (dfinal.defined() && a.K > 1) ? ptr(dfinal) : nullptr;
        Tensor dx, dinitial, dweight, dbias, ws;
        if (need[0]) {
            dx = like(x);
            a.dx = out(dx);
            strides2(a.dx_stride, dx);
        }
        if (need[1]) dweight = torch::empty_like(weight);
        if (need[2]) dbias = torch::empty_like(bias);
        if (need[3]) dinitial = torch::empty(initial.sizes(), initial.options());
        a.dweight = fout(dweight);
        a.dbias = fout(dbias);
        a.dinitial = (dinitial.defined() && a.K > 1) ? out(dinitial) : nullptr;
        if (need[1] || need[2]) ws = scratch(tgru_conv_backward_workspace_bytes(a.B, a.T, a.D, a.K), x);
        a.workspace = fout(ws);
        check(tgru_conv_backward(&a, stream_of(x)), "tgru_conv_backward");
        return {dx, dweight, dbias, dinitial, Tensor(), Tensor(), Tensor(), Tensor()};
    }
};

std::vector<Tensor> short_conv(const Tensor &x_, const Tensor &weight_, const OptTensor &bias_, bool silu, const OptTensor &initial_,
                               const OptTensor &lengths, bool return_state) {
    dtype_code(x_, "input");
    TORCH_CHECK(x_.dim() == 3, "input must be (B, T, D), got ", shape_of(x_));
    const int64_t B = as_int(x_.size(0), "the batch"), D = as_int(x_.size(2), "the number of channels");
    as_int(x_.size(1), "the number of steps");
    TORCH_CHECK(weight_.dim() == 2 && weight_.size(0) == D, "weight must be (D, K) = (", D, ", K), got ", shape_of(weight_));
    const int64_t K = weight_.size(1);
    TORCH_CHECK(K >= 1 && K <= TGRU_CONV_MAX_TAPS, "weight has ", K, " taps, 1 to ", TGRU_CONV_MAX_TAPS, " are built");
    const Tensor weight = param(weight_, x_, "weight");
    OptTensor bias, initial;
    if (bias_) {
        require_shape(*bias_, {D}, "bias");
        bias = param(*bias_, x_, "bias");
    }
    if (initial_) {
        require_shape(*initial_, {B, K - 1, D}, "initial_state");
        require_like(*initial_, x_, "initial_state");
        initial = initial_->contiguous();
    }
    require_index(lengths, B, x_, "lengths");
    require_gpu(x_);
    auto r = ConvFunction::apply(rows(x_), weight, bias, initial, lengths, silu, return_state, torch::GradMode::is_enabled());
    return r;
}

// ---- scan ------------------------------------------------------------------------------------------------------------

struct ScanInputs { Tensor u, delta, A, b, c, skip, z, delta_bias, initial, lengths; };

tgru_scan_args scan_args(const ScanInputs &in, bool softplus) {
    tgru_scan_args a{};
    a.u = ptr(in.u);
    a.delta = ptr(in.delta);
    a.z = ptr(in.z);
    a.b = ptr(in.b);
    a.c = ptr(in.c);
    a.a = fptr(in.A);
    a.skip = fptr(in.skip);
    a.delta_bias = fptr(in.delta_bias);
    a.initial_state = fptr(in.initial);
    a.lengths = iptr(in.lengths);
    strides2(a.u_stride, in.u);
    strides2(a.delta_stride, in.delta);
    strides2(a.z_stride, in.z);
    strides3(a.b_stride, in.b);
    strides3(a.c_stride, in.c);
    a.B = (int)in.u.size(0);
    a.T = (int)in.u.size(1);
    a.D = (int)in.u.size(2);
    a.N = (int)in.A.size(1);
    a.G = (int)in.b.size(2);
    a.dtype = dtype_code(in.u, "input");
    a.softplus = softplus;
    return a;
}

class ScanFunction : public torch::autograd::Function<ScanFunction> {
public:
    static variable_list forward(AutogradContext *ctx, const Tensor &u, const Tensor &delta, const Tensor &A, const Tensor &b, const Tensor &c,
                                 const OptTensor &skip, const OptTensor &z, const OptTensor &delta_bias, const OptTensor &initial,
                                 const OptTensor &lengths, bool softplus, bool want_state, bool grad_mode) {
        const ScanInputs in{u, delta, A, b, c, skip.value_or(Tensor()), z.value_or(Tensor()), delta_bias.value_or(Tensor()),
                            initial.value_or(Tensor()), lengths.value_or(Tensor())};
        const c10::hip::HIPGuardMasqueradingAsCUDA guard(u.device());
        tgru_scan_args a = scan_args(in, softplus);
        const std::vector<bool> need{wants(u), wants(delta), wants(A), wants(b), wants(c), wants(in.skip), wants(in.z), wants(in.delta_bias),
                                     wants(in.initial)};
        bool any = false;
        for (bool n : need) any = any || n;
        Tensor y = like(u), state, reserve;
        if (want_state) state = torch::empty({a.B, a.D, a.N}, A.options());
        if (any && grad_mode) reserve = scratch(tgru_scan_reserve_bytes(a.B, a.T, a.D, a.N, a.G), u);
        const Tensor ws = scratch(tgru_scan_workspace_bytes(a.B, a.T, a.D, a.N, a.G, 0), u);
        a.y = out(y);
        strides2(a.y_stride, y);
        a.final_state = fout(state);
        a.reserve = fout(reserve);
        a.workspace = fout(ws);
        check(tgru_scan_forward(&a, stream_of(u)), "tgru_scan_forward");
        ctx->saved_data["need"] = need;
        ctx->saved_data["softplus"] = softplus;
        ctx->set_materialize_grads(false);
        if (any && grad_mode) ctx->save_for_backward({u, delta, A, b, c, in.skip, in.z, in.delta_bias, in.lengths, reserve});
        if (want_state) return {y, state};
        return {y};
    }

    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        no_second_derivative("selective_scan");
        const auto saved = ctx->get_saved_variables();
        const ScanInputs in{saved[0], saved[1], saved[2], saved[3], saved[4], saved[5], saved[6], saved[7], Tensor(), saved[8]};
        const Tensor reserve = saved[9];
        const auto need = ctx->saved_data["need"].toBoolList();
        const c10::hip::HIPGuardMasqueradingAsCUDA guard(in.u.device());
        tgru_scan_args a = scan_args(in, ctx->saved_data["softplus"].toBool());
        const Tensor dy = grads[0].defined() ? near_rows(grads[0]) : Tensor();
        const Tensor dfinal = grads.size() > 1 ? dense(grads[1]) : Tensor();
        a.dy = ptr(dy);
        strides2(a.dy_stride, dy);
        a.dfinal = fptr(dfinal);
        a.reserve = const_cast<float *>(fptr(reserve));
        const Tensor ws = scratch(tgru_scan_workspace_bytes(a.B, a.T, a.D, a.N, a.G, 1), in.u);
        a.workspace = fout(ws);
        variable_list g(13);
        auto seq = [&](int k, const Tensor &of, void *&to, int64_t (&stride)[2]) {
            if (!need[k]) return;
            g[k] = like(of);
            to = out(g[k]);
            strides2(stride, g[k]);
        };
        seq(0, in.u, a.du, a.du_stride);
        seq(1, in.delta, a.ddelta, a.ddelta_stride);
        seq(6, in.z, a.dz, a.dz_stride);
        if (need[2]) a.da = fout(g[2] = torch::empty_like(in.A));
        if (need[3]) a.db = out(g[3] = torch::empty(in.b.sizes(), in.b.options()));
        if (need[4]) a.dc = out(g[4] = torch::empty(in.c.sizes(), in.c.options()));
        if (need[5]) a.dskip = fout(g[5] = torch::empty_like(in.skip));
        if (need[7]) a.ddelta_bias = fout(g[7] = torch::empty_like(in.delta_bias));
        if (need[8]) a.dinitial = fout(g[8] = torch::empty({a.B, a.D, a.N}, in.A.options()));
        check(tgru_scan_backward(&a, stream_of(in.u)), "tgru_scan_backward");
        return g;
    }
};

// The checks that a scan over sequences and a scan of one token share; `lead` is (B, T) or (B).
void check_scan(const Tensor &u, const Tensor &delta, const Tensor &A, const Tensor &b, const Tensor &c, const OptTensor &skip,
                const OptTensor &z, const OptTensor &delta_bias, std::vector<int64_t> lead) {
    dtype_code(u, "input");
    const int64_t D = as_int(u.size(-1), "the number of channels");
    for (int64_t n : lead) as_int(n, "the batch and the number of steps");
    TORCH_CHECK(A.dim() == 2 && A.size(0) == D, "A must be (D, N) = (", D, ", N), got ", shape_of(A));
    const int64_t N = A.size(1);
    TORCH_CHECK(N >= 1 && N <= TGRU_SCAN_MAX_STATES, "A has ", N, " states a channel, 1 to ", TGRU_SCAN_MAX_STATES, " are built");
    require_shape(delta, u.sizes(), "delta");
    require_like(delta, u, "delta");
    TORCH_CHECK(b.dim() == u.dim() + 1, "B must have a dimension of groups and one of states behind the input's leading ones, got ", shape_of(b));
    const int64_t G = b.size(-2);
    TORCH_CHECK(G >= 1 && D % G == 0, "the number of groups, ", G, ", must divide the number of channels, ", D);
    lead.push_back(G);
    lead.push_back(N);
    require_shape(b, lead, "B");
    require_shape(c, lead, "C");
    require_like(b, u, "B");
    require_like(c, u, "C");
    if (skip) require_shape(*skip, {D}, "D");
    if (delta_bias) require_shape(*delta_bias, {D}, "delta_bias");
    if (z) {
        require_shape(*z, u.sizes(), "z");
        require_like(*z, u, "z");
    }
}

OptTensor opt_param(const OptTensor &t, const Tensor &first, const char *what) {
    if (!t) return t;
    return param(*t, first, what);
}

std::vector<Tensor> selective_scan(const Tensor &u, const Tensor &delta, const Tensor &A, const Tensor &b, const Tensor &c,
                                   const OptTensor &skip, const OptTensor &z, const OptTensor &delta_bias, bool softplus,
                                   const OptTensor &initial_, const OptTensor &lengths, bool return_state) {
    TORCH_CHECK(u.dim() == 3, "input must be (B, T, D), got ", shape_of(u));
    check_scan(u, delta, A, b, c, skip, z, delta_bias, {u.size(0), u.size(1)});
    OptTensor initial, zz;
    if (initial_) {
        require_shape(*initial_, {u.size(0), u.size(2), A.size(1)}, "initial_state");
        initial = param(*initial_, u, "initial_state");
    }
    if (z) zz = near_rows(*z);
    require_index(lengths, u.size(0), u, "lengths");
    const Tensor A32 = param(A, u, "A");
    const OptTensor skip32 = opt_param(skip, u, "D"), bias32 = opt_param(delta_bias, u, "delta_bias");
    require_gpu(u);
    return ScanFunction::apply(near_rows(u), near_rows(delta), A32, near_rows(b), near_rows(c), skip32, zz, bias32, initial, lengths, softplus, return_state,
                               torch::GradMode::is_enabled());
}

// ---- one token -------------------------------------------------------------------------------------------------------

// Neither direction of automatic differentiation passes through a one-token call.  (Tangents of forward mode are there under
// torch.no_grad() too.)
void no_gradient(std::initializer_list<const Tensor *> ts, const char *what) {
    for (const Tensor *t : ts) {
        if (!t || !t->defined()) continue;
        TORCH_CHECK(!t->_fw_grad(/*level=*/0).defined(), what, " has no forward-mode derivative: its inputs must not be dual tensors");
        TORCH_CHECK(!(torch::GradMode::is_enabled() && t->requires_grad()), what, " has no backward pass: call it under torch.no_grad()");
    }
}

const Tensor *at(const OptTensor &t) { return t ? &*t : nullptr; }

// The pools of a one-token call: `state` is read, `state_out` (or `state` itself) is written.
Tensor check_pools(const Tensor &state, const OptTensor &state_out, bool slots, int64_t B, at::IntArrayRef shape) {
    require_shape(state, shape, "state");
    TORCH_CHECK(state.is_contiguous(), "state must be dense (it is updated where it lies)");
    TORCH_CHECK(slots || shape[0] >= B, "state holds ", shape[0], " sequences, the batch has ", B);
    if (!state_out) return state;
    require_shape(*state_out, shape, "state_out");
    TORCH_CHECK(state_out->scalar_type() == state.scalar_type() && state_out->device() == state.device() && state_out->is_contiguous(),
                "state_out must be a dense tensor of the element type of state, on its device");
    const char *p = (const char *)state.data_ptr(), *q = (const char *)state_out->data_ptr();
    const int64_t bytes = state.numel() * state.element_size();
    TORCH_CHECK(p == q || p + bytes <= q || q + bytes <= p, "state and state_out overlap in part");
    return *state_out;
}

// An input of a one-token call lies outside the pool that the call writes.
void apart(const Tensor &t, const Tensor &pool, const char *what) {
    int64_t span = 1;
    for (int64_t i = 0; i < t.dim(); ++i) span += (t.size(i) - 1) * t.stride(i);
    const char *p = (const char *)t.data_ptr(), *q = (const char *)pool.data_ptr();
    TORCH_CHECK(p + span * t.element_size() <= q || q + pool.numel() * pool.element_size() <= p || !pool.numel(), what,
                " overlaps the state that the call writes");
}

void written(const Tensor &t) {
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

Tensor short_conv_step(const Tensor &x_, const Tensor &state, const Tensor &weight_, const OptTensor &bias_, bool silu, const OptTensor &slots,
                       const OptTensor &state_out) {
    const int dtype = dtype_code(x_, "input");
    TORCH_CHECK(x_.dim() == 2, "input must be (B, D), got ", shape_of(x_));
    const int64_t B = as_int(x_.size(0), "the batch"), D = as_int(x_.size(1), "the number of channels");
    TORCH_CHECK(weight_.dim() == 2 && weight_.size(0) == D, "weight must be (D, K) = (", D, ", K), got ", shape_of(weight_));
    const int64_t K = weight_.size(1);
    TORCH_CHECK(K >= 1 && K <= TGRU_CONV_MAX_TAPS, "weight has ", K, " taps, 1 to ", TGRU_CONV_MAX_TAPS, " are built");
    if (bias_) require_shape(*bias_, {D}, "bias");
    TORCH_CHECK(state.dim() == 3, "state must be (P, K - 1, D), got ", shape_of(state));
    require_like(state, x_, "state");
    const Tensor to = check_pools(state, state_out, slots.has_value(), B, {as_int(state.size(0), "the pool"), K - 1, D});
    require_index(slots, B, x_, "slots");
    no_gradient({&x_, &state, &weight_, at(bias_), &to}, "short_conv_step");
    const Tensor x = rows(x_), weight = param(weight_, x_, "weight"), bias = bias_ ? param(*bias_, x_, "bias") : Tensor();
    apart(x, to, "input");
    require_gpu(x_);
    const c10::hip::HIPGuardMasqueradingAsCUDA guard(x.device());
    Tensor y = torch::empty({B, D}, x.options());
    tgru_conv_step_args a{};
    a.x = ptr(x);
    a.state = ptr(state);
    a.state_out = out(to);
    a.weight = fptr(weight);
    a.bias = fptr(bias);
    a.slots = slots ? iptr(*slots) : nullptr;
    a.y = out(y);
    a.x_stride = x.stride(0);
    a.y_stride = D;
    a.B = (int)B;
    a.P = (int)state.size(0);
    a.D = (int)D;
    a.K = (int)K;
    a.dtype = dtype;
    a.silu = silu;
    check(tgru_conv_step(&a, stream_of(x)), "tgru_conv_step");
    written(to);
    return y;
}

Tensor selective_scan_step(const Tensor &u_, const Tensor &delta_, const Tensor &state, const Tensor &A, const Tensor &b_, const Tensor &c_,
                           const OptTensor &skip, const OptTensor &z_, const OptTensor &delta_bias, bool softplus, const OptTensor &slots,
                           const OptTensor &state_out) {
    TORCH_CHECK(u_.dim() == 2, "input must be (B, D), got ", shape_of(u_));
    check_scan(u_, delta_, A, b_, c_, skip, z_, delta_bias, {u_.size(0)});
    const int64_t B = u_.size(0), D = u_.size(1), N = A.size(1);
    TORCH_CHECK(state.dim() == 3, "state must be (P, D, N), got ", shape_of(state));
    TORCH_CHECK(state.scalar_type() == torch::kFloat32 && state.device() == u_.device(), "state must be a float32 tensor on the input's device");
    const Tensor to = check_pools(state, state_out, slots.has_value(), B, {as_int(state.size(0), "the pool"), D, N});
    require_index(slots, B, u_, "slots");
    no_gradient({&u_, &delta_, &state, &A, &b_, &c_, at(skip), at(z_), at(delta_bias), &to}, "selective_scan_step");
    const Tensor u = rows(u_), delta = rows(delta_), b = rows(b_), c = rows(c_), z = z_ ? rows(*z_) : Tensor();
    const Tensor A32 = param(A, u, "A"), skip32 = skip ? param(*skip, u, "D") : Tensor();
    const Tensor bias32 = delta_bias ? param(*delta_bias, u, "delta_bias") : Tensor();
    apart(u, to, "input");
    apart(delta, to, "delta");
    apart(b, to, "B");
    apart(c, to, "C");
    if (z.defined()) apart(z, to, "z");
    require_gpu(u_);
    const c10::hip::HIPGuardMasqueradingAsCUDA guard(u.device());
    Tensor y = torch::empty({B, D}, u.options());
    tgru_scan_step_args a{};
    a.u = ptr(u);
    a.delta = ptr(delta);
    a.z = ptr(z);
    a.b = ptr(b);
    a.c = ptr(c);
    a.a = fptr(A32);
    a.skip = fptr(skip32);
    a.delta_bias = fptr(bias32);
    a.state = fptr(state);
    a.state_out = fout(to);
    a.slots = slots ? iptr(*slots) : nullptr;
    a.y = out(y);
    a.u_stride = u.stride(0);
    a.delta_stride = delta.stride(0);
    a.z_stride = z.defined() ? z.stride(0) : 0;
    a.y_stride = D;
    a.b_stride[0] = b.stride(0);
    a.b_stride[1] = b.stride(1);
    a.c_stride[0] = c.stride(0);
    a.c_stride[1] = c.stride(1);
    a.B = (int)B;
    a.P = (int)state.size(0);
    a.D = (int)D;
    a.N = (int)N;
    a.G = (int)b.size(1);
    a.dtype = dtype_code(u, "input");
    a.softplus = softplus;
    check(tgru_scan_step(&a, stream_of(u)), "tgru_scan_step");
    written(to);
    return y;
}

}  // namespace

void bind_ssm(py::module_ &m) {
    py::register_exception_translator([](std::exception_ptr p) {
        try {
            if (p) std::rethrow_exception(p);
        } catch (const NoGpu &e) {
            PyErr_SetString(py::module_::import("timegan_amd._lib").attr("TgruError").ptr(), e.what());
        }
    });
    m.def("short_conv", &short_conv, "differentiable short causal convolution");
    m.def("short_conv_step", &short_conv_step, "one more step of it on a pool of states");
    m.def("selective_scan", &selective_scan, "differentiable selective scan");
    m.def("selective_scan_step", &selective_scan_step, "one more step of it on a pool of states");
}
