// sequence_torch.cpp -- torch binding of the sequence operators (layer norm, rotary positions, windowed attention and its step): argument checks, allocation, autograd
// nodes.  Host code only; the kernels are reached through the C ABI of libgfpp_radnerf.so (include/gfpp_radnerf.h), whose entry points Python hands over by address.
//
// Why compiled: these operators are small and called many times per step.  From Python, the checks, the ctypes conversion and an autograd node whose backward waits
// for the interpreter in the engine's thread cost 150 us per forward + backward pass on the host, three times what the kernels of a clip's layer norm take on the GPU;
// from here they are 66 us, two thirds of which is the engine's own.
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/utils/pybind.h>
#include <ATen/ATen.h>
#include <ATen/TracerMode.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>

#include <algorithm>
#include <array>
#include <cmath>
#include <limits>
#include <optional>
#include <sstream>

#include "../../include/gfpp_radnerf.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
namespace py = pybind11;

constexpr int64_t kFar = 1 << 29;      // most tokens, and a window side without an end

// ---- errors: GfppError of the package's _lib.py --------------------------------------------------------------------------------------------------------------------
struct Error : std::runtime_error {
    using std::runtime_error::runtime_error;
};
template <typename... A>
[[noreturn]] void fail(const A &...parts) {
    std::ostringstream s;
    (s << ... << parts);
    throw Error(s.str());
}
template <typename... A>
inline void require(bool ok, const A &...parts) {
    if (__builtin_expect(!ok, 0)) fail(parts...);
}

// ---- the C ABI, by address -----------------------------------------------------------------------------------------------------------------------------------------
struct Api {
    decltype(&::gfpp_last_error) last_error = nullptr;
    decltype(&::gfpp_layer_norm_forward) layer_norm_forward = nullptr;
    decltype(&::gfpp_layer_norm_backward) layer_norm_backward = nullptr;
    decltype(&::gfpp_layer_norm_backward_scratch_floats) layer_norm_scratch = nullptr;
    decltype(&::gfpp_rotary) rotary = nullptr;
    decltype(&::gfpp_window_attn_two_part) two_part = nullptr;
    decltype(&::gfpp_window_attn_forward) window_forward = nullptr;
    decltype(&::gfpp_window_attn_backward) window_backward = nullptr;
    decltype(&::gfpp_window_attn_backward_scratch_floats) window_scratch = nullptr;
    decltype(&::gfpp_window_attn_step) step = nullptr;
    decltype(&::gfpp_window_attn_step_scratch_floats) step_scratch = nullptr;
} api;

template <typename F>
void bind_one(const py::dict &d, const char *name, F &slot) {
    slot = reinterpret_cast<F>(d[name].cast<uintptr_t>());
}
void bind(const py::dict &d) {
    bind_one(d, "gfpp_last_error", api.last_error);
    bind_one(d, "gfpp_layer_norm_forward", api.layer_norm_forward);
    bind_one(d, "gfpp_layer_norm_backward", api.layer_norm_backward);
    bind_one(d, "gfpp_layer_norm_backward_scratch_floats", api.layer_norm_scratch);
    bind_one(d, "gfpp_rotary", api.rotary);
    bind_one(d, "gfpp_window_attn_two_part", api.two_part);
    bind_one(d, "gfpp_window_attn_forward", api.window_forward);
    bind_one(d, "gfpp_window_attn_backward", api.window_backward);
    bind_one(d, "gfpp_window_attn_backward_scratch_floats", api.window_scratch);
    bind_one(d, "gfpp_window_attn_step", api.step);
    bind_one(d, "gfpp_window_attn_step_scratch_floats", api.step_scratch);
}
void check(int rc, const char *name) {
    if (rc != 0) {
        const char *m = api.last_error();
        fail(name, " failed (code ", rc, "): ", m ? m : "");
    }
}
gfpp_stream_t stream_of(const Tensor &t) { return c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.device().index()).stream(); }

int type_code(const char *what, const Tensor &t) {
    switch (t.scalar_type()) {
        case at::kFloat: return GFPP_F32;
        case at::kHalf: return GFPP_F16;
        case at::kBFloat16: return GFPP_BF16;
        default: fail(what, ": float32, float16 or bfloat16 expected, got ", t.scalar_type());
    }
}
void same_device(const char *what, const char *name, const Tensor &t, const Tensor &like) {
    require(t.device() == like.device(), what, ": ", name, " is on ", t.device(), ", expected ", like.device());
}
// (the last check of every operator: what else is wrong with a call is told without a GPU too)
void on_gpu(const char *what, const Tensor &t) { require(t.is_cuda(), what, ": tensors must be on the GPU (no CPU path)"); }

// Derivatives in forward mode: a tensor with a tangent need not ask for a gradient, and no operation is recorded that would carry the tangent on.
template <typename... T>
void no_tangents(const char *what, const T &...tensors) {
    require(!((tensors.defined() && tensors._fw_grad(0).defined()) || ...), what, ": no derivatives in forward mode (an input has a tangent)");
}

// Tracers (torch.jit.trace, make_fx) see the allocation of an output and not the kernel that fills it: what they recorded would return memory as it comes.
void not_traced(const char *what) {
    require(!at::tracer::impl::is_dispatch_enabled() && !c10::impl::TorchDispatchModeTLS::get_mode(c10::impl::TorchDispatchModeKey::PROXY).has_value(), what,
            ": cannot be traced (its kernels are no operations of torch)");
}

// (an absent tensor reaches an autograd node as an empty optional: it is no input of the node then)
std::optional<Tensor> given(const Tensor &t) { return t.defined() ? std::optional<Tensor>(t) : std::nullopt; }
bool wants_grad(const Tensor &t) { return t.defined() && t.requires_grad(); }
const void *ptr(const Tensor &t) { return t.defined() ? t.const_data_ptr() : nullptr; }
void *mut(const Tensor &t) { return t.defined() ? t.mutable_data_ptr() : nullptr; }

// Gradients are first derivatives: where the backward pass is itself recorded its results get a node that raises when it is asked for a gradient.
variable_list once(variable_list grads) {
    if (!at::GradMode::is_enabled()) return grads;
    variable_list in;
    for (auto &g : grads) in.push_back(g.defined() ? g.detach().set_requires_grad(true) : g);
    auto node = std::make_shared<torch::autograd::DelayedError>("the sequence operators have first derivatives only", (int64_t)in.size());
    return (*node)(std::move(in));
}

// ---- layer norm ----------------------------------------------------------------------------------------------------------------------------------------------------
// t as rows [M, N] of one pitch: a view where the layout has one, a copy otherwise
Tensor rows_of(const Tensor &t, int64_t N) {
    if (t.dim() == 2 && t.stride(1) == 1 && t.stride(0) >= 0) return t;
    return t.contiguous().view({-1, N});
}

Tensor norm_forward(const Tensor &x, const Tensor &rows, const Tensor &weight, const Tensor &bias, double eps, const Tensor &stats) {
    const Tensor &param = weight.defined() ? weight : bias;
    Tensor y = at::empty(x.sizes(), x.options());
    const int64_t M = rows.size(0);
    float *st = stats.defined() ? stats.mutable_data_ptr<float>() : nullptr;
    check(api.layer_norm_forward(rows.const_data_ptr(), rows.stride(0), ptr(weight), ptr(bias), param.defined() ? type_code("layer_norm", param) : GFPP_F32, (uint64_t)M,
                                 (uint32_t)rows.size(1), (float)eps, type_code("layer_norm", x), y.mutable_data_ptr(), st, st ? st + M : nullptr, stream_of(x)),
          "gfpp_layer_norm_forward");
    return y;
}

struct LayerNormFn : torch::autograd::Function<LayerNormFn> {
    static Tensor forward(AutogradContext *ctx, const Tensor &x, const std::optional<Tensor> &w, const std::optional<Tensor> &b, double eps) {
        const Tensor weight = w.value_or(Tensor()), bias = b.value_or(Tensor());
        const Tensor rows = rows_of(x, x.size(-1));
        const Tensor stats = at::empty({2, rows.size(0)}, x.options().dtype(at::kFloat));
        Tensor y = norm_forward(x, rows, weight, bias, eps, stats);
        ctx->save_for_backward({rows, weight, bias, stats});
        return y;
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        not_traced("layer_norm");
        const auto saved = ctx->get_saved_variables();
        const Tensor &rows = saved[0], &weight = saved[1], &bias = saved[2], &stats = saved[3];
        const Tensor &dy = grads[0];
        const int64_t M = rows.size(0), N = rows.size(1);
        const Tensor dyr = rows_of(dy, N);
        const bool want_x = ctx->needs_input_grad(0), want_w = weight.defined() && ctx->needs_input_grad(1), want_b = bias.defined() && ctx->needs_input_grad(weight.defined() ? 2 : 1);
        Tensor dx, dw, db, scratch;
        if (want_x) dx = at::empty(dy.sizes(), rows.options());
        if (want_w) dw = at::empty_like(weight);
        if (want_b) db = at::empty_like(bias);
        if (want_w || want_b) scratch = at::empty({(int64_t)api.layer_norm_scratch((uint64_t)M, (uint32_t)N)}, stats.options());
        const Tensor &param = weight.defined() ? weight : bias;
        const float *st = stats.const_data_ptr<float>();
        check(api.layer_norm_backward(dyr.const_data_ptr(), dyr.stride(0), rows.const_data_ptr(), rows.stride(0), ptr(weight),
                                      param.defined() ? type_code("layer_norm", param) : GFPP_F32, st, st + M, (uint64_t)M, (uint32_t)N, type_code("layer_norm", rows), mut(dx), mut(dw),
                                      mut(db), static_cast<float *>(mut(scratch)), stream_of(rows)),
              "gfpp_layer_norm_backward");
        return once({dx, dw, db, Tensor()});
    }
};

Tensor layer_norm(const Tensor &x, const std::optional<Tensor> &w, const std::optional<Tensor> &b, double eps) {
    const char *what = "layer_norm";
    type_code(what, x);
    require(x.dim() >= 1 && x.size(-1) >= 1, what, ": the last axis must not be empty, got ", x.sizes());
    const Tensor weight = w.value_or(Tensor()), bias = b.value_or(Tensor());
    for (int k = 0; k < 2; ++k) {
        const Tensor &p = k ? bias : weight;
        if (!p.defined()) continue;
        const char *name = k ? "bias" : "weight";
        same_device(what, name, p, x);
        require(p.dim() == 1 && p.size(0) == x.size(-1) && p.is_contiguous(), what, ": ", name, " must be a contiguous [", x.size(-1), "], got ", p.sizes());
        require(p.scalar_type() == at::kFloat || p.scalar_type() == x.scalar_type(), what, ": ", name, " must be float32 or ", x.scalar_type(), ", got ", p.scalar_type());
    }
    require(!weight.defined() || !bias.defined() || weight.scalar_type() == bias.scalar_type(), what, ": weight is ", weight.defined() ? weight.scalar_type() : at::kFloat, ", bias ",
            bias.defined() ? bias.scalar_type() : at::kFloat);
    require(eps >= 0.0, what, ": eps must not be negative, got ", eps);
    no_tangents(what, x, weight, bias);
    not_traced(what);
    on_gpu(what, x);
    const c10::DeviceGuard guard(x.device());
    if (at::GradMode::is_enabled() && (wants_grad(x) || wants_grad(weight) || wants_grad(bias))) return LayerNormFn::apply(x, given(weight), given(bias), eps);
    return norm_forward(x, rows_of(x, x.size(-1)), weight, bias, eps, Tensor());
}

// ---- rotary positions ----------------------------------------------------------------------------------------------------------------------------------------------
variable_list rotary_launch(const variable_list &xs, const Tensor &positions, const Tensor &frequencies, const std::vector<int64_t> &sections, bool interleaved, bool backward) {
    const Tensor &first = xs[0];
    const int64_t B = first.size(0), T = first.size(1), D = first.size(3);
    variable_list dense, out;
    int64_t strides[2][3] = {};
    for (size_t k = 0; k < xs.size(); ++k) {
        dense.push_back(xs[k].stride(3) == 1 ? xs[k] : xs[k].contiguous());
        out.push_back(at::empty(xs[k].sizes(), xs[k].options()));
        for (int i = 0; i < 3; ++i) strides[k][i] = dense[k].stride(i);
    }
    uint32_t sec[4] = {};
    for (size_t k = 0; k < sections.size(); ++k) sec[k] = (uint32_t)sections[k];
    const bool two = xs.size() == 2;
    const int type = positions.scalar_type() == at::kInt ? 0 : positions.scalar_type() == at::kLong ? 1 : 2;
    check(api.rotary(dense[0].const_data_ptr(), strides[0], (uint32_t)first.size(2), out[0].mutable_data_ptr(), two ? dense[1].const_data_ptr() : nullptr, strides[1],
                     two ? (uint32_t)xs[1].size(2) : 0, two ? out[1].mutable_data_ptr() : nullptr, positions.const_data_ptr(), type, positions.dim() == 3 ? positions.stride(0) : 0,
                     frequencies.const_data_ptr<double>(), sec, (uint32_t)sections.size(), (uint32_t)B, (uint32_t)T, (uint32_t)D, interleaved, backward, type_code("rotary_embed", first),
                     stream_of(first)),
          "gfpp_rotary");
    return out;
}

struct RotaryFn : torch::autograd::Function<RotaryFn> {
    static variable_list forward(AutogradContext *ctx, const Tensor &a, const std::optional<Tensor> &b, const Tensor &positions, const Tensor &frequencies, const std::vector<int64_t> &sections,
                                 bool interleaved) {
        ctx->save_for_backward({positions, frequencies});
        ctx->saved_data["sections"] = sections;
        ctx->saved_data["interleaved"] = interleaved;
        return rotary_launch(b ? variable_list{a, *b} : variable_list{a}, positions, frequencies, sections, interleaved, false);
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        not_traced("rotary_embed");
        const auto saved = ctx->get_saved_variables();
        // the transpose of a turn is the turn by the opposite angle (a tensor that needs no gradient still takes its place in the launch: they come in pairs)
        variable_list out = once(rotary_launch(grads, saved[0], saved[1], ctx->saved_data["sections"].toIntVector(), ctx->saved_data["interleaved"].toBool(), true));
        out.resize(6);
        return out;
    }
};

variable_list rotary_embed(const variable_list &xs, Tensor positions, Tensor frequencies, const std::vector<int64_t> &sections, bool interleaved) {
    const char *what = "rotary_embed";
    require(xs.size() == 1 || xs.size() == 2, what, ": one tensor or two, got ", xs.size());
    const Tensor &first = xs[0];
    type_code(what, first);
    for (const Tensor &t : xs) {
        require(t.dim() == 4 && t.scalar_type() == first.scalar_type() && t.size(0) == first.size(0) && t.size(1) == first.size(1) && t.size(3) == first.size(3), what,
                ": [B, T, H, D] tensors of one type that differ in H alone, got ", first.sizes(), " ", first.scalar_type(), " and ", t.sizes(), " ", t.scalar_type());
        same_device(what, "a tensor", t, first);
    }
    const int64_t B = first.size(0), T = first.size(1), D = first.size(3), axes = (int64_t)sections.size();
    int64_t P = 0;
    bool ok = axes >= 1 && axes <= 4;
    for (int64_t n : sections) {
        ok = ok && n >= 0 && n <= 512;
        P += n;
    }
    require(ok && P >= 1 && P <= 512 && 2 * P <= D, what, ": sections ", c10::IntArrayRef(sections), ": 1 .. 4 axes, 1 .. 512 pairs, ", D, " features");
    const bool own = positions.dim() == 3;
    require((positions.scalar_type() == at::kInt || positions.scalar_type() == at::kLong || positions.scalar_type() == at::kFloat) && (own || positions.dim() == 2) &&
                (!own || positions.size(0) == B) && positions.size(own ? 1 : 0) == T && positions.size(-1) == axes,
            what, ": positions must be int32, int64 or float32 [", T, ", ", axes, "] or [", B, ", ", T, ", ", axes, "], got ", positions.scalar_type(), " ", positions.sizes());
    require(frequencies.scalar_type() == at::kDouble && frequencies.dim() == 1 && frequencies.size(0) == P, what, ": frequencies must be float64 [", P, "], got ",
            frequencies.scalar_type(), " ", frequencies.sizes());
    same_device(what, "positions", positions, first);
    same_device(what, "frequencies", frequencies, first);
    require(!at::GradMode::is_enabled() || !(wants_grad(positions) || wants_grad(frequencies)), what, ": positions and frequencies get no gradient");
    for (const Tensor &t : xs) no_tangents(what, t);
    no_tangents(what, positions, frequencies);
    not_traced(what);
    on_gpu(what, first);
    const c10::DeviceGuard guard(first.device());
    positions = positions.contiguous();
    frequencies = frequencies.contiguous();
    if (at::GradMode::is_enabled() && (wants_grad(xs[0]) || (xs.size() == 2 && wants_grad(xs[1]))))
        return RotaryFn::apply(xs[0], xs.size() == 2 ? given(xs[1]) : std::nullopt, positions, frequencies, sections, interleaved);
    return rotary_launch(xs, positions, frequencies, sections, interleaved, false);
}

// ---- attention with a sliding window and sinks ---------------------------------------------------------------------------------------------------------------------
struct Window {
    int32_t left, right, sinks, start;
    double scale;
};

Tensor dense_heads(const Tensor &t) { return t.stride(-1) == 1 || t.size(-1) == 1 ? t : t.contiguous(); }
void put_strides(int64_t *&to, const Tensor &t) {
    for (int i = 0; i < 3; ++i) *to++ = t.stride(i);
}

Tensor window_forward(const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &lengths, const Window &w, const Tensor &lse, Tensor *low) {
    const int code = type_code("window_attention", q);
    Tensor out = at::empty(q.sizes(), q.options());
    if (low && api.two_part((uint32_t)k.size(1), w.left, w.right, w.sinks, code)) *low = at::empty(q.sizes(), q.options());
    int64_t strides[12], *s = strides;
    for (const Tensor *t : {&q, &k, &v, static_cast<const Tensor *>(&out)}) put_strides(s, *t);
    check(api.window_forward(q.const_data_ptr(), k.const_data_ptr(), v.const_data_ptr(), out.mutable_data_ptr(), low ? mut(*low) : nullptr, static_cast<float *>(mut(lse)), strides,
                             (uint32_t)q.size(0), (uint32_t)q.size(1), (uint32_t)k.size(1), (uint32_t)q.size(2), (uint32_t)k.size(2), (uint32_t)q.size(3), w.left, w.right, w.sinks,
                             w.start, static_cast<const int32_t *>(ptr(lengths)), (float)w.scale, code, stream_of(q)),
          "gfpp_window_attn_forward");
    return out;
}

struct WindowAttentionFn : torch::autograd::Function<WindowAttentionFn> {
    static Tensor forward(AutogradContext *ctx, const Tensor &q, const Tensor &k, const Tensor &v, const std::optional<Tensor> &lens, const Window &w) {
        const Tensor lengths = lens.value_or(Tensor());
        const Tensor lse = at::empty({q.size(0), q.size(2), q.size(1)}, q.options().dtype(at::kFloat));
        Tensor low;
        Tensor out = window_forward(q, k, v, lengths, w, lse, &low);
        ctx->save_for_backward({q, k, v, out, lse, lengths, low});
        ctx->saved_data["window"] = std::vector<int64_t>{w.left, w.right, w.sinks, w.start};
        ctx->saved_data["scale"] = w.scale;
        return out;
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        not_traced("window_attention");
        const auto saved = ctx->get_saved_variables();
        const Tensor &q = saved[0], &k = saved[1], &v = saved[2], &out = saved[3], &lse = saved[4], &lengths = saved[5], &low = saved[6];
        const Tensor dout = dense_heads(grads[0]);
        const Tensor dq = at::empty(q.sizes(), q.options()), dk = at::empty(k.sizes(), k.options()), dv = at::empty(v.sizes(), v.options());
        const auto w = ctx->saved_data["window"].toIntVector();
        const uint32_t B = (uint32_t)q.size(0), Tq = (uint32_t)q.size(1), Tk = (uint32_t)k.size(1), Hq = (uint32_t)q.size(2), Hk = (uint32_t)k.size(2), D = (uint32_t)q.size(3);
        const Tensor scratch = at::empty({(int64_t)api.window_scratch(B, Tq, Tk, Hq, Hk, D, (int32_t)w[0], (int32_t)w[1], (int32_t)w[2], (int32_t)w[3], type_code("window_attention", q))}, lse.options());
        int64_t strides[24], *s = strides;
        for (const Tensor *t : {&q, &k, &v, &out, &dout, &dq, &dk, &dv}) put_strides(s, *t);
        check(api.window_backward(q.const_data_ptr(), k.const_data_ptr(), v.const_data_ptr(), out.const_data_ptr(), ptr(low), dout.const_data_ptr(), lse.const_data_ptr<float>(),
                                  dq.mutable_data_ptr(), dk.mutable_data_ptr(), dv.mutable_data_ptr(), scratch.mutable_data_ptr<float>(), strides, B, Tq, Tk, Hq, Hk, D, (int32_t)w[0],
                                  (int32_t)w[1], (int32_t)w[2], (int32_t)w[3], static_cast<const int32_t *>(ptr(lengths)), (float)ctx->saved_data["scale"].toDouble(),
                                  type_code("window_attention", q), stream_of(q)),
              "gfpp_window_attn_backward");
        return once({dq, dk, dv, Tensor(), Tensor()});
    }
};

void check_heads(const char *what, const Tensor &q, const Tensor &k, const Tensor &v, int64_t axes) {
    type_code(what, q);
    require(q.dim() == axes && k.dim() == axes && k.sizes() == v.sizes(), what, ": q, k, v must have ", axes, " axes and k the shape of v, got ", q.sizes(), ", ", k.sizes(), ", ",
            v.sizes());
    require(k.scalar_type() == q.scalar_type() && v.scalar_type() == q.scalar_type(), what, ": q, k, v must have one type, got ", q.scalar_type(), ", ", k.scalar_type(), ", ",
            v.scalar_type());
    require(q.size(0) == k.size(0) && q.size(-1) == k.size(-1), what, ": q and k differ in batch or head width: ", q.sizes(), ", ", k.sizes());
    const int64_t Hq = q.size(-2), Hk = k.size(-2), D = q.size(-1);
    require(Hk >= 1 && Hq >= 1 && Hq % Hk == 0, what, ": ", Hq, " query heads are no multiple of ", Hk, " key heads");
    require(D >= 1 && D <= 128, what, ": head width ", D, " (1 .. 128 are supported)");
    require(q.size(0) <= kFar && Hq <= kFar, what, ": more than 2^29 sequences or heads");
    same_device(what, "k", k, q);
    same_device(what, "v", v, q);
}
double checked_scale(const char *what, const std::optional<double> &scale, int64_t D) {
    const double s = scale.value_or(1.0 / std::sqrt((double)D));
    require((float)s > 0.0f && (float)s < std::numeric_limits<float>::infinity(), what, ": scale must be positive, got ", s);
    return s;
}
int32_t whole(const char *what, const char *name, const std::optional<int64_t> &n) {
    if (!n) return (int32_t)kFar;
    require(*n >= 0, what, ": ", name, " must be a whole number from 0, got ", *n);
    return (int32_t)std::min(*n, kFar);
}

Tensor window_attention(const Tensor &q0, const Tensor &k0, const Tensor &v0, std::optional<int64_t> left, std::optional<int64_t> right, int64_t sinks, std::optional<Tensor> lens,
                        std::optional<double> scale, std::optional<int64_t> q_start) {
    const char *what = "window_attention";
    check_heads(what, q0, k0, v0, 4);
    const int64_t B = q0.size(0), Tq = q0.size(1), Tk = k0.size(1);
    require(Tq <= kFar && Tk <= kFar, what, ": more than 2^29 tokens");
    Window w{whole(what, "left", left), whole(what, "right", right), whole(what, "sinks", sinks), 0, checked_scale(what, scale, q0.size(3))};
    const int64_t start = q_start.value_or(Tk - Tq);
    require(start >= 0 && start <= kFar, what, ": q_start ", start, " must be 0 .. 2^29 (more queries than keys need it given)");
    w.start = (int32_t)start;
    Tensor lengths;
    if (lens) {
        lengths = *lens;
        require(lengths.dim() == 1 && lengths.size(0) == B && (lengths.scalar_type() == at::kInt || lengths.scalar_type() == at::kLong), what,
                ": lengths must be an int32 or int64 tensor [", B, "]");
        same_device(what, "lengths", lengths, q0);
    }
    no_tangents(what, q0, k0, v0);
    not_traced(what);
    on_gpu(what, q0);
    const c10::DeviceGuard guard(q0.device());
    if (lengths.defined()) lengths = lengths.scalar_type() == at::kLong ? lengths.clamp(0, Tk).to(at::kInt) : lengths.contiguous();
    const Tensor q = dense_heads(q0), k = dense_heads(k0), v = dense_heads(v0);
    if (at::GradMode::is_enabled() && (wants_grad(q) || wants_grad(k) || wants_grad(v))) return WindowAttentionFn::apply(q, k, v, given(lengths), w);
    return window_forward(q, k, v, lengths, w, Tensor(), nullptr);
}

// ---- the step over a rolling cache ---------------------------------------------------------------------------------------------------------------------------------
// Whether all elements of some axes (size, stride) lie apart: sorted by stride, every axis steps over what the ones before it span.
using Axes = std::array<std::pair<int64_t, int64_t>, 5>;
bool axes_apart(Axes axes) {
    std::sort(axes.begin(), axes.end(), [](const auto &a, const auto &b) { return a.second < b.second; });
    int64_t span = 1;
    for (const auto &[size, stride] : axes) {
        if (size <= 1) continue;
        if (stride < span) return false;
        span += (size - 1) * stride;
    }
    return true;
}
Axes axes_of(const Tensor &t) {
    Axes axes{};
    for (int64_t i = 0; i < 4; ++i) axes[i] = {t.size(i), t.stride(i)};
    axes[4] = {1, 0};
    return axes;
}
// Caches are written in place, each slot by whoever has it: two slots in one memory, within a cache or between the two, would be a race.
bool caches_apart(const Tensor &a, const Tensor &b) {
    if (a.numel() == 0) return true;
    Axes axes = axes_of(a);
    const Axes other = axes_of(b);
    if (!axes_apart(axes) || !axes_apart(other)) return false;
    const auto bytes = [](const Tensor &t) {
        int64_t span = 1;
        for (int64_t i = 0; i < t.dim(); ++i) span += (t.size(i) - 1) * t.stride(i);
        return span * (int64_t)t.element_size();
    };
    const int64_t apart = (int64_t)((intptr_t)b.const_data_ptr() - (intptr_t)a.const_data_ptr()), size = (int64_t)a.element_size();
    if (apart >= bytes(a) || -apart >= bytes(b)) return true;
    // One inside the other's reach.  Blocks of keys and of values in turn along an axis, each block as it likes:
    for (int64_t i = 0; i < 4; ++i) {
        if (axes[i].first <= 1 || axes[i].second != other[i].second) continue;
        const int64_t period = axes[i].second * size, rest = (axes[i].first - 1) * period, from = (apart % period + period) % period;
        if (from >= bytes(a) - rest && period - from >= bytes(b) - rest) return true;
    }
    // ... or side by side at any axis with the same strides, which is one more axis of two
    for (int64_t i = 0; i < 4; ++i)
        if (axes[i].first > 1 && axes[i].second != other[i].second) return false;
    axes[4] = {2, std::abs(apart) / size};
    return apart % size == 0 && axes_apart(axes);
}

Tensor window_attention_step(const Tensor &q0, const Tensor &k0, const Tensor &v0, const Tensor &cache_k, const Tensor &cache_v, const Tensor &positions, int64_t sinks,
                             std::optional<double> scale) {
    const char *what = "window_attention_step";
    check_heads(what, q0, k0, v0, 3);
    const int64_t B = q0.size(0), Hq = q0.size(1), D = q0.size(2), Hk = k0.size(1);
    for (int c = 0; c < 2; ++c) {
        const Tensor &t = c ? cache_v : cache_k;
        const char *name = c ? "cache_v" : "cache_k";
        require(t.dim() == 4 && t.size(0) == B && t.size(2) == Hk && t.size(3) == D && t.sizes() == cache_k.sizes(), what, ": ", name, " must be [", B, ", slots, ", Hk, ", ", D,
                "] like the other, got ", t.sizes());
        require(t.scalar_type() == q0.scalar_type(), what, ": ", name, " must be ", q0.scalar_type(), ", got ", t.scalar_type());
        bool apart = D == 1 || t.stride(3) == 1;
        for (int64_t i = 0; i < 3; ++i) apart = apart && (t.size(i) <= 1 || t.stride(i) > 0);
        require(apart, what, ": ", name, " needs a dense last axis and rows of its own (strides ", t.strides(), "): it is written in place");
        same_device(what, name, t, q0);
    }
    const int64_t slots = cache_k.size(1);
    require(sinks >= 0 && sinks < slots, what, ": sinks ", sinks, " must be 0 .. slots - 1 (", slots, " slots)");
    require(slots <= kFar, what, ": more than 2^29 slots");
    require(positions.dim() == 1 && positions.size(0) == B && (positions.scalar_type() == at::kInt || positions.scalar_type() == at::kLong) && positions.is_contiguous(), what,
            ": positions must be a contiguous int32 or int64 tensor [", B, "]");
    same_device(what, "positions", positions, q0);
    require(!at::GradMode::is_enabled() || !(wants_grad(q0) || wants_grad(k0) || wants_grad(v0) || wants_grad(cache_k) || wants_grad(cache_v)), what,
            ": no gradients (call it under torch.no_grad(); window_attention is the differentiable form)");
    const double sc = checked_scale(what, scale, D);
    no_tangents(what, q0, k0, v0, cache_k, cache_v);
    not_traced(what);
    on_gpu(what, q0);
    require(caches_apart(cache_k, cache_v), what, ": slots of cache_k and cache_v lie in one memory (strides ", cache_k.strides(), ", ", cache_v.strides(), "): they are written in place");
    const c10::DeviceGuard guard(q0.device());
    const Tensor q = dense_heads(q0), k = dense_heads(k0), v = dense_heads(v0);
    const Tensor out = at::empty(q.sizes(), q.options());
    Tensor scratch;
    if (const auto n = api.step_scratch((uint32_t)B, (uint32_t)Hq, (uint32_t)Hk, (uint32_t)D, (uint32_t)slots)) scratch = at::empty({(int64_t)n}, q.options().dtype(at::kFloat));
    const int64_t strides[14] = {q.stride(0),       q.stride(1),       k.stride(0),       k.stride(1),       v.stride(0),       v.stride(1),   cache_k.stride(0),
                                 cache_k.stride(1), cache_k.stride(2), cache_v.stride(0), cache_v.stride(1), cache_v.stride(2), out.stride(0), out.stride(1)};
    check(api.step(q.const_data_ptr(), k.const_data_ptr(), v.const_data_ptr(), cache_k.mutable_data_ptr(), cache_v.mutable_data_ptr(), positions.const_data_ptr(),
                   positions.scalar_type() == at::kLong, out.mutable_data_ptr(), strides, (uint32_t)B, (uint32_t)Hq, (uint32_t)Hk, (uint32_t)D, (uint32_t)slots, (uint32_t)sinks, (float)sc,
                   type_code(what, q), static_cast<float *>(mut(scratch)), stream_of(q)),
          "gfpp_window_attn_step");
    // written in place: whoever has kept them for a backward pass is told (torch raises there)
    for (const Tensor *t : {&cache_k, &cache_v})
        if (!t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
    return out;
}

}  // namespace

PYBIND11_MODULE(_sequence, m) {
    // the package's error class, held for the process' life
    static PyObject *error = py::object(py::module_::import("genefaceplusplus_amd._lib").attr("GfppError")).release().ptr();
    py::register_exception_translator([](std::exception_ptr p) {
        try {
            if (p) std::rethrow_exception(p);
        } catch (const Error &e) {
            PyErr_SetString(error, e.what());
        }
    });
    m.def("bind", &bind);
    m.def("layer_norm", &layer_norm);
    m.def("rotary_embed", &rotary_embed);
    m.def("window_attention", &window_attention);
    m.def("window_attention_step", &window_attention_step);
}
