// torch_layers.cpp -- the `attention` ops of the layer around attention over the C ABI: normed
// rotation, the gated feed-forward block, dropout.  Argument checks, layout, workspace, autograd.
#include "torch_support.h"

namespace {

using namespace tmsupport;

// ---- norm_rotate ------------------------------------------------------------------

// Features contiguous, and rows and heads at multiples of 16 bytes where a head's features fill
// such: the order of a head's sum, and so its bits, goes by its size alone.
Tensor lined_up(const Tensor &t) {
    const int64_t unit = 16 / t.element_size(), d = t.size(3);
    const bool ok = (d == 1 || t.stride(3) == 1) &&
                    (d % unit != 0 ||
                     (step_of(t, 0) % unit == 0 && step_of(t, 1) % unit == 0 &&
                      step_of(t, 2) % unit == 0 &&
                      reinterpret_cast<uintptr_t>(t.const_data_ptr()) % 16 == 0));
    return ok ? t : t.clone(at::MemoryFormat::Contiguous);
}

// The arguments, checked, as the library takes them.
struct Normed {
    tm_norm_rotation n = {};
    Rotation t;
    Tensor in, weight; // as read; weight undefined where there is none
    Normed(const Tensor &x, const OptTensor &w, const Tensor &positions, const Tensor &freqs,
           at::IntArrayRef sections, at::IntArrayRef heads, double eps, bool interleaved)
        : t("norm_rotate", x, positions, freqs, sections, interleaved, false) {
        const int64_t H = x.size(2), D = x.size(3);
        TORCH_CHECK_VALUE(H >= 1 && H <= TM_NORM_MAX_HEADS, "norm_rotate: x must have 1 to ",
                          (int)TM_NORM_MAX_HEADS, " heads, got ", x.sizes());
        TORCH_CHECK_VALUE(D <= TM_NORM_MAX_HEAD_DIM, "norm_rotate: heads hold 1 to ",
                          (int)TM_NORM_MAX_HEAD_DIM, " features, got ", D);
        TORCH_CHECK_VALUE(eps >= 0. && (float)eps <= 3e38f,
                          "norm_rotate: eps must be finite and not negative, got ", eps);
        const int64_t groups = (int64_t)heads.size();
        TORCH_CHECK_VALUE(groups >= 1 && groups <= TM_NORM_MAX_GROUPS,
                          "norm_rotate: heads must be 1 to ", (int)TM_NORM_MAX_GROUPS,
                          " counts, got ", groups);
        int64_t sum = 0;
        for (int64_t g = 0; g < groups; ++g) {
            TORCH_CHECK_VALUE(heads[g] >= 1 && heads[g] <= H,
                              "norm_rotate: heads must be positive and sum to ", H, ", got ",
                              heads);
            n.heads[g] = (int32_t)heads[g];
            sum += heads[g];
        }
        TORCH_CHECK_VALUE(sum == H, "norm_rotate: heads must be positive and sum to ", H,
                          ", got ", heads);
        n.groups = (int32_t)groups;
        n.eps = (float)eps;
        n.weight_type = t.r.dtype;
        if (w.has_value()) {
            TORCH_CHECK_VALUE(w->device() == x.device(),
                              "norm_rotate: weight must be on x's device");
            TORCH_CHECK_TYPE(w->scalar_type() == x.scalar_type() ||
                                 w->scalar_type() == at::kFloat,
                             "norm_rotate: weight must be float32 or ", x.scalar_type(),
                             " as x is, got ", w->scalar_type());
            TORCH_CHECK_VALUE(w->dim() == 2 && w->size(0) == groups && w->size(1) == D,
                              "norm_rotate: weight must be (", groups, ", ", D, "), got ",
                              w->sizes());
            weight = w->contiguous();
            n.weight = weight.const_data_ptr();
            n.weight_type = dtype_code(weight, "norm_rotate", "weight");
        }
        in = lined_up(t.in);
        t.r.x = in.const_data_ptr();
        t.r.x_b = step_of(in, 0), t.r.x_l = step_of(in, 1), t.r.x_h = step_of(in, 2);
        n.rotation = t.r;
    }
};

Tensor norm_rotate_hip(const Tensor &x, const OptTensor &weight, const Tensor &positions,
                       const Tensor &freqs, at::IntArrayRef sections, at::IntArrayRef heads,
                       double eps, bool interleaved) {
    const c10::DeviceGuard guard(x.device());
    const Normed p(x, weight, positions, freqs, sections, heads, eps, interleaved);
    Tensor out = at::empty(x.sizes(), x.options());
    if (out.numel())
        check_rc(tm_norm_rotate(&p.n, out.data_ptr(), current_stream(x)), "norm_rotate");
    return out;
}

// what is not asked for is empty
std::tuple<Tensor, Tensor>
norm_rotate_backward_hip(const Tensor &dout, const Tensor &x, const OptTensor &weight,
                         const Tensor &positions, const Tensor &freqs, at::IntArrayRef sections,
                         at::IntArrayRef heads, double eps, bool interleaved, bool need_x,
                         bool need_weight) {
    const c10::DeviceGuard guard(x.device());
    const Normed p(x, weight, positions, freqs, sections, heads, eps, interleaved);
    TORCH_CHECK_VALUE(dout.sizes() == x.sizes() && dout.device() == x.device(),
                      "norm_rotate_backward: dout must be as x");
    TORCH_CHECK_TYPE(dout.scalar_type() == x.scalar_type(),
                     "norm_rotate_backward: dout must have x's dtype");
    need_weight = need_weight && weight.has_value();
    Tensor dx = at::empty(need_x ? x.sizes() : at::IntArrayRef{0}, x.options());
    Tensor dw = need_weight ? at::empty(p.weight.sizes(), p.weight.options())
                            : at::empty({0}, x.options());
    const Tensor g = lined_up(dout);
    Tensor ws;
    const size_t bytes = need_weight ? tm_norm_rotate_backward_workspace_bytes(&p.n) : 0;
    if (bytes)
        ws = at::empty({(int64_t)bytes}, x.options().dtype(at::kByte));
    check_rc(tm_norm_rotate_backward(&p.n, g.const_data_ptr(), step_of(g, 0), step_of(g, 1),
                                     step_of(g, 2), need_x && x.numel() ? dx.data_ptr() : nullptr,
                                     need_weight ? dw.data_ptr() : nullptr,
                                     bytes ? ws.data_ptr() : nullptr, bytes, current_stream(x)),
             "norm_rotate_backward");
    return {dx, dw};
}

struct NormRotateFunction : torch::autograd::Function<NormRotateFunction> {
    static Tensor forward(AutogradContext *ctx, const Tensor &x, const OptTensor &weight,
                          const Tensor &positions, const Tensor &freqs, at::IntArrayRef sections,
                          at::IntArrayRef heads, double eps, bool interleaved) {
        at::AutoDispatchBelowADInplaceOrView below;
        ctx->save_for_backward({x, weight.value_or(Tensor()), positions, freqs});
        ctx->saved_data["sections"] = sections.vec();
        ctx->saved_data["heads"] = heads.vec();
        ctx->saved_data["eps"] = eps;
        ctx->saved_data["interleaved"] = interleaved;
        static auto op =
            c10::Dispatcher::singleton()
                .findSchemaOrThrow("attention::norm_rotate", "")
                .typed<Tensor(const Tensor &, const OptTensor &, const Tensor &, const Tensor &,
                              at::IntArrayRef, at::IntArrayRef, double, bool)>();
        return op.call(x, weight, positions, freqs, sections, heads, eps, interleaved);
    }
    static variable_list backward(AutogradContext *ctx, const variable_list &grads) {
        variable_list result(8);
        if (!grads[0].defined())
            return result;
        const auto s = ctx->get_saved_variables();
        const bool need_x = ctx->needs_input_grad(0);
        const bool need_weight = s[1].defined() && ctx->needs_input_grad(1);
        static auto op = c10::Dispatcher::singleton()
                             .findSchemaOrThrow("attention::norm_rotate_backward", "")
                             .typed<std::tuple<Tensor, Tensor>(
                                 const Tensor &, const Tensor &, const OptTensor &,
                                 const Tensor &, const Tensor &, at::IntArrayRef,
                                 at::IntArrayRef, double, bool, bool, bool)>();
        auto [dx, dw] = op.call(
            grads[0], s[0], s[1].defined() ? OptTensor(s[1]) : OptTensor(), s[2], s[3],
            ctx->saved_data["sections"].toIntVector(), ctx->saved_data["heads"].toIntVector(),
            ctx->saved_data["eps"].toDouble(), ctx->saved_data["interleaved"].toBool(), need_x,
            need_weight);
        if (need_x)
            result[0] = dx;
        if (need_weight)
            result[1] = dw;
        return result;
    }
};

Tensor norm_rotate_autograd(const Tensor &x, const OptTensor &weight, const Tensor &positions,
                            const Tensor &freqs, at::IntArrayRef sections, at::IntArrayRef heads,
                            double eps, bool interleaved) {
    constant(positions, "norm_rotate", "positions");
    constant(freqs, "norm_rotate", "freqs");
    TORCH_CHECK_NOT_IMPLEMENTED(!has_tangent(x) && !(weight.has_value() && has_tangent(*weight)),
                                "norm_rotate: no forward-mode derivative");
    if (wants_grad(x) || (weight.has_value() && wants_grad(*weight)))
        return NormRotateFunction::apply(x, weight, positions, freqs, sections, heads, eps,
                                         interleaved);
    at::AutoDispatchBelowADInplaceOrView below;
    static auto op =
        c10::Dispatcher::singleton()
            .findSchemaOrThrow("attention::norm_rotate", "")
            .typed<Tensor(const Tensor &, const OptTensor &, const Tensor &, const Tensor &,
                          at::IntArrayRef, at::IntArrayRef, double, bool)>();
    return op.call(x, weight, positions, freqs, sections, heads, eps, interleaved);
}

// ---- feed_forward -----------------------------------------------------------------

int activation_code(c10::string_view name) {
    static const char *const names[] = {"silu", "gelu", "gelu_tanh", "relu"}; // TM_SILU ..
    for (int i = 0; i < 4; ++i)
        if (name == names[i])
            return i;
    TORCH_CHECK_VALUE(false, "feed_forward: activation must be silu, gelu, gelu_tanh or relu, got ",
                      name);
}

// (rows, n) as the kernels read it: features contiguous and padded with zeros to 16 bytes, rows at
// multiples of 16 bytes.  Views that are, are read in place; others are copied.
Tensor rows_of(const Tensor &t) {
    const int64_t n = t.size(-1), unit = 16 / t.element_size();
    const Tensor r = t.dim() == 2 ? t : t.reshape({t.numel() / n, n});
    const int64_t l = step_of(r, 0);
    if (n % unit) {
        const Tensor t1 = n == 1 || r.stride(1) == 1 ? r : r.contiguous();
        Tensor padded = at::empty({r.size(0), (n + unit - 1) / unit * unit}, r.options());
        check_rc(tm_pad_rows(t1.const_data_ptr(), step_of(t1, 0), r.size(0), (int32_t)n,
                             dtype_code(r, "feed_forward", "x"), padded.data_ptr(),
                             current_stream(r)),
                 "feed_forward");
        return padded;
    }
    const bool ok = (n == 1 || r.stride(1) == 1) && l % unit == 0 && (l == 0 || l >= n) &&
                    l * r.element_size() < TM_FF_MAX_ROW_BYTES &&
                    reinterpret_cast<uintptr_t>(r.const_data_ptr()) % 16 == 0;
    return ok ? r : r.clone(at::MemoryFormat::Contiguous);
}

// The arguments, checked, as the library takes them.
struct Block {
    tm_feed_forward f = {};
    Tensor x, gate, up, down; // as read
    std::vector<int64_t> out; // the output's shape
    Block(const Tensor &x_, const Tensor &gate_, const Tensor &up_, const Tensor &down_,
          c10::string_view activation) {
        TORCH_CHECK_VALUE(x_.dim() >= 1 && gate_.dim() == 2 && up_.dim() == 2 && down_.dim() == 2,
                          "feed_forward: x must be (..., C), gate and up (F, C) and down (O, F), got ",
                          x_.sizes(), ", ", gate_.sizes(), ", ", up_.sizes(), " and ",
                          down_.sizes());
        f.dtype = dtype_code(x_, "feed_forward", "x");
        for (const Tensor *w : {&gate_, &up_, &down_}) {
            TORCH_CHECK_VALUE(w->device() == x_.device(),
                              "feed_forward: x and the weights must be on one device");
            TORCH_CHECK_TYPE(w->scalar_type() == x_.scalar_type(),
                             "feed_forward: x and the weights must have one dtype, got ",
                             x_.scalar_type(), " and ", w->scalar_type());
        }
        f.activation = activation_code(activation);
        const int64_t C = x_.size(-1), F = gate_.size(0), O = down_.size(0);
        TORCH_CHECK_VALUE(C >= 1 && F >= 1 && O >= 1, "feed_forward: sizes must be positive, got x ",
                          x_.sizes(), ", gate ", gate_.sizes(), ", down ", down_.sizes());
        TORCH_CHECK_VALUE(gate_.size(1) == C && up_.sizes() == gate_.sizes(),
                          "feed_forward: gate and up must be (F, ", C, ") as x is, got ",
                          gate_.sizes(), " and ", up_.sizes());
        TORCH_CHECK_VALUE(down_.size(1) == F, "feed_forward: down must be (O, ", F,
                          ") as gate is, got ", down_.sizes());
        const int64_t T = x_.numel() / C;
        const int64_t most = TM_FF_MAX_ROW_BYTES / x_.element_size() - 16;
        const auto blocks = [](int64_t m, int64_t n) {
            return ((double)m + 127.) / 128. * (((double)n + 63.) / 64.);
        };
        TORCH_CHECK_VALUE(T <= INT32_MAX - 256 && C < most && F < most && O < most &&
                              std::max({blocks(T, F), blocks(T, O), blocks(T, C),
                                        2. * blocks(F, C), blocks(O, F)}) <=
                                  TM_FF_MAX_BLOCKS,
                          "feed_forward: too many rows for one call: x ", x_.sizes(), ", gate ",
                          gate_.sizes(), ", down ", down_.sizes());
        out = x_.sizes().vec();
        out.back() = O;
        f.T = (int32_t)T, f.C = (int32_t)C, f.F = (int32_t)F, f.O = (int32_t)O;
        x = rows_of(x_), gate = rows_of(gate_), up = rows_of(up_), down = rows_of(down_);
        if (step_of(gate, 0) != step_of(up, 0)) // the kernels take one stride for both
            gate = gate.contiguous(), up = up.contiguous();
        f.x = x.const_data_ptr(), f.gate = gate.const_data_ptr();
        f.up = up.const_data_ptr(), f.down = down.const_data_ptr();
        f.x_l = step_of(x, 0), f.w_l = step_of(gate, 0), f.down_l = step_of(down, 0);
    }
};

std::tuple<Tensor, Tensor> feed(const Tensor &x, const Tensor &gate, const Tensor &up,
                                const Tensor &down, c10::string_view activation, bool save) {
    const c10::DeviceGuard guard(x.device());
    const Block p(x, gate, up, down, activation);
    const auto bytes = x.options().dtype(at::kByte);
    Tensor out = at::empty(p.out, x.options());
    Tensor saved = at::empty({save ? (int64_t)tm_feed_forward_saved_bytes(&p.f) : 0}, bytes);
    if (p.f.T) {
        const Tensor ws = at::empty({(int64_t)tm_feed_forward_workspace_bytes(&p.f)}, bytes);
        check_rc(tm_feed_forward_forward(&p.f, out.data_ptr(), save ? saved.data_ptr() : nullptr,
                                         ws.data_ptr(), (size_t)ws.numel(), current_stream(x)),
                 "feed_forward");
    }
    return {out, saved};
}

Tensor feed_forward_hip(const Tensor &x, const Tensor &gate, const Tensor &up, const Tensor &down,
                        c10::string_view activation) {
    return std::get<0>(feed(x, gate, up, down, activation, false));
}

std::tuple<Tensor, Tensor> feed_forward_save_hip(const Tensor &x, const Tensor &gate,
                                                 const Tensor &up, const Tensor &down,
                                                 c10::string_view activation) {
    return feed(x, gate, up, down, activation, true);
}

// what is not asked for is empty
std::tuple<Tensor, Tensor, Tensor, Tensor>
feed_forward_backward_hip(const Tensor &dout, const Tensor &x, const Tensor &gate,
                          const Tensor &up, const Tensor &down, const Tensor &saved,
                          c10::string_view activation, bool need_x, bool need_gate, bool need_up,
                          bool need_down) {
    const c10::DeviceGuard guard(x.device());
    const Block p(x, gate, up, down, activation);
    TORCH_CHECK_VALUE(dout.sizes() == at::IntArrayRef(p.out) && dout.device() == x.device(),
                      "feed_forward_backward: dout must be as the output ",
                      at::IntArrayRef(p.out), ", got ", dout.sizes());
    TORCH_CHECK_TYPE(dout.scalar_type() == x.scalar_type(),
                     "feed_forward_backward: dout must have x's dtype");
    TORCH_CHECK_VALUE(saved.device() == x.device() && saved.scalar_type() == at::kByte &&
                          saved.is_contiguous() &&
                          saved.numel() == (int64_t)tm_feed_forward_saved_bytes(&p.f),
                      "feed_forward_backward: saved must be what the forward pass saved");
    const bool pair = need_gate || need_up;
    const auto made = [&](bool need, const Tensor &t) {
        return at::empty(need ? t.sizes() : at::IntArrayRef{0}, x.options());
    };
    Tensor dx = made(need_x, x), dgate = made(pair, gate), dup = made(pair, up),
           ddown = made(need_down, down);
    const auto place = [](bool need, Tensor &t) { return need ? t.data_ptr() : nullptr; };
    const Tensor g = rows_of(dout);
    const Tensor ws = at::empty({(int64_t)tm_feed_forward_backward_workspace_bytes(&p.f)},
                                x.options().dtype(at::kByte));
    check_rc(tm_feed_forward_backward(&p.f, saved.const_data_ptr(), g.const_data_ptr(),
                                      step_of(g, 0), place(need_x && p.f.T, dx),
                                      place(pair, dgate), place(pair, dup),
                                      place(need_down, ddown), ws.data_ptr(), (size_t)ws.numel(),
                                      current_stream(x)),
             "feed_forward_backward");
    return {dx, need_gate ? dgate : made(false, gate), need_up ? dup : made(false, up), ddown};
}

struct FeedForwardFunction : torch::autograd::Function<FeedForwardFunction> {
    static Tensor forward(AutogradContext *ctx, const Tensor &x, const Tensor &gate,
                          const Tensor &up, const Tensor &down, std::string activation) {
        at::AutoDispatchBelowADInplaceOrView below;
        static auto op = c10::Dispatcher::singleton()
                             .findSchemaOrThrow("attention::feed_forward_save", "")
                             .typed<std::tuple<Tensor, Tensor>(
                                 const Tensor &, const Tensor &, const Tensor &, const Tensor &,
                                 c10::string_view)>();
        auto [out, saved] = op.call(x, gate, up, down, activation);
        ctx->save_for_backward({x, gate, up, down, saved});
        ctx->saved_data["activation"] = activation;
        return out;
    }
    static variable_list backward(AutogradContext *ctx, const variable_list &grads) {
        variable_list result(5);
        if (!grads[0].defined())
            return result;
        const auto s = ctx->get_saved_variables();
        bool need[4];
        for (int i = 0; i < 4; ++i)
            need[i] = ctx->needs_input_grad(i);
        static auto op =
            c10::Dispatcher::singleton()
                .findSchemaOrThrow("attention::feed_forward_backward", "")
                .typed<std::tuple<Tensor, Tensor, Tensor, Tensor>(
                    const Tensor &, const Tensor &, const Tensor &, const Tensor &,
                    const Tensor &, const Tensor &, c10::string_view, bool, bool, bool, bool)>();
        auto [dx, dgate, dup, ddown] =
            op.call(grads[0], s[0], s[1], s[2], s[3], s[4],
                    ctx->saved_data["activation"].toStringRef(), need[0], need[1], need[2],
                    need[3]);
        const Tensor all[] = {dx, dgate, dup, ddown};
        for (int i = 0; i < 4; ++i)
            if (need[i])
                result[i] = all[i];
        return result;
    }
};

Tensor feed_forward_autograd(const Tensor &x, const Tensor &gate, const Tensor &up,
                             const Tensor &down, c10::string_view activation) {
    TORCH_CHECK_NOT_IMPLEMENTED(!has_tangent(x) && !has_tangent(gate) && !has_tangent(up) &&
                                    !has_tangent(down),
                                "feed_forward: no forward-mode derivative");
    if (wants_grad(x) || wants_grad(gate) || wants_grad(up) || wants_grad(down))
        return FeedForwardFunction::apply(x, gate, up, down, std::string(activation));
    at::AutoDispatchBelowADInplaceOrView below;
    static auto op = c10::Dispatcher::singleton()
                         .findSchemaOrThrow("attention::feed_forward", "")
                         .typed<Tensor(const Tensor &, const Tensor &, const Tensor &,
                                       const Tensor &, c10::string_view)>();
    return op.call(x, gate, up, down, activation);
}

// ---- dropout ----------------------------------------------------------------------

Tensor dropout_hip(const Tensor &x, double p, int64_t seed, int64_t offset,
                   const OptTensor &seed_at, const OptTensor &residual) {
    const c10::DeviceGuard guard(x.device());
    const int dtype = dtype_code(x, "dropout", "x");
    TORCH_CHECK_VALUE(p >= 0. && p <= 1., "dropout: p must be from 0 to 1, got ", p);
    if (seed_at.has_value()) {
        TORCH_CHECK_TYPE(seed_at->scalar_type() == at::kLong,
                         "dropout: a seed on the device must be int64, got ",
                         seed_at->scalar_type());
        TORCH_CHECK_VALUE(seed_at->numel() == 1 && seed_at->device() == x.device(),
                          "dropout: seed must be one number on x's device, got ",
                          seed_at->sizes(), " on ", seed_at->device());
    }
    if (residual.has_value()) {
        TORCH_CHECK_TYPE(residual->scalar_type() == x.scalar_type(),
                         "dropout: residual must have x's dtype, got ", residual->scalar_type());
        TORCH_CHECK_VALUE(residual->sizes() == x.sizes() && residual->device() == x.device(),
                          "dropout: residual must have x's shape ", x.sizes(), ", got ",
                          residual->sizes());
    }
    const Tensor in = x.contiguous();
    Tensor add, out = at::empty(x.sizes(), x.options());
    if (residual.has_value())
        add = residual->contiguous();
    check_rc(tm_dropout(in.const_data_ptr(), add.defined() ? add.const_data_ptr() : nullptr,
                        out.data_ptr(), x.numel(), dtype, p, (uint64_t)seed,
                        seed_at.has_value() ? seed_at->const_data_ptr<int64_t>() : nullptr,
                        (uint64_t)offset, current_stream(x)),
             "dropout");
    return out;
}

Tensor call_dropout(const Tensor &x, double p, int64_t seed, int64_t offset,
                    const OptTensor &seed_at, const OptTensor &residual) {
    static auto op = c10::Dispatcher::singleton()
                         .findSchemaOrThrow("attention::dropout", "")
                         .typed<Tensor(const Tensor &, double, int64_t, int64_t,
                                       const OptTensor &, const OptTensor &)>();
    return op.call(x, p, seed, offset, seed_at, residual);
}

struct DropoutFunction : torch::autograd::Function<DropoutFunction> {
    static Tensor forward(AutogradContext *ctx, const Tensor &x, double p, int64_t seed,
                          int64_t offset, const OptTensor &seed_at, const OptTensor &residual) {
        at::AutoDispatchBelowADInplaceOrView below;
        ctx->save_for_backward({seed_at.value_or(Tensor())});
        ctx->saved_data["p"] = p;
        ctx->saved_data["seed"] = seed;
        ctx->saved_data["offset"] = offset;
        ctx->saved_data["added"] = residual.has_value();
        return call_dropout(x, p, seed, offset, seed_at, residual);
    }
    static variable_list backward(AutogradContext *ctx, const variable_list &grads) {
        variable_list result(6);
        if (!grads[0].defined())
            return result;
        const auto s = ctx->get_saved_variables();
        // the same mask again, differentiable again
        if (ctx->needs_input_grad(0))
            result[0] = call_dropout(grads[0], ctx->saved_data["p"].toDouble(),
                                     ctx->saved_data["seed"].toInt(),
                                     ctx->saved_data["offset"].toInt(),
                                     s[0].defined() ? OptTensor(s[0]) : OptTensor(), OptTensor());
        if (ctx->saved_data["added"].toBool())
            result[5] = grads[0];
        return result;
    }
};

Tensor dropout_autograd(const Tensor &x, double p, int64_t seed, int64_t offset,
                        const OptTensor &seed_at, const OptTensor &residual) {
    const bool turned = has_tangent(x), added = residual.has_value() && has_tangent(*residual);
    if (turned || added) { // linear in both
        const auto [x0, x1] = at::_unpack_dual(x, /*level=*/0);
        OptTensor r0, r1;
        if (residual.has_value()) {
            const auto [primal, tangent] = at::_unpack_dual(*residual, /*level=*/0);
            r0 = primal;
            if (added)
                r1 = tangent;
        }
        const Tensor tangent = turned ? dropout_autograd(x1, p, seed, offset, seed_at, r1)
                                      : r1->clone(at::MemoryFormat::Contiguous);
        return at::_make_dual(dropout_autograd(x0, p, seed, offset, seed_at, r0), tangent,
                              /*level=*/0);
    }
    if (wants_grad(x) || (residual.has_value() && wants_grad(*residual)))
        return DropoutFunction::apply(x, p, seed, offset, seed_at, residual);
    at::AutoDispatchBelowADInplaceOrView below;
    return call_dropout(x, p, seed, offset, seed_at, residual);
}

} // namespace

TORCH_LIBRARY_FRAGMENT(attention, m) {
    m.def("norm_rotate(Tensor x, Tensor? weight, Tensor positions, Tensor freqs, int[] sections, "
          "int[] heads, float eps, bool interleaved=False) -> Tensor");
    m.def("norm_rotate_backward(Tensor dout, Tensor x, Tensor? weight, Tensor positions, "
          "Tensor freqs, int[] sections, int[] heads, float eps, bool interleaved=False, "
          "bool need_x=True, bool need_weight=True) -> (Tensor, Tensor)");
    m.def("feed_forward(Tensor x, Tensor gate, Tensor up, Tensor down, str activation) -> Tensor");
    // the same with what feed_forward_backward needs of the hidden features
    m.def("feed_forward_save(Tensor x, Tensor gate, Tensor up, Tensor down, str activation) -> "
          "(Tensor, Tensor)");
    m.def("feed_forward_backward(Tensor dout, Tensor x, Tensor gate, Tensor up, Tensor down, "
          "Tensor saved, str activation, bool need_x=True, bool need_gate=True, "
          "bool need_up=True, bool need_down=True) -> (Tensor, Tensor, Tensor, Tensor)");
    // the seed lies in seed_at where it is given
    m.def("dropout(Tensor x, float p, int seed=0, int offset=0, Tensor? seed_at=None, "
          "Tensor? residual=None) -> Tensor");
}

TORCH_LIBRARY_IMPL(attention, CUDA, m) {
    m.impl("norm_rotate", &norm_rotate_hip);
    m.impl("norm_rotate_backward", &norm_rotate_backward_hip);
    m.impl("feed_forward", &feed_forward_hip);
    m.impl("feed_forward_save", &feed_forward_save_hip);
    m.impl("feed_forward_backward", &feed_forward_backward_hip);
    m.impl("dropout", &dropout_hip);
}

TORCH_LIBRARY_IMPL(attention, Autograd, m) {
    m.impl("norm_rotate", &norm_rotate_autograd);
    m.impl("norm_rotate_backward", torch::autograd::autogradNotImplementedFallback());
    m.impl("feed_forward", &feed_forward_autograd);
    m.impl("feed_forward_save", torch::autograd::autogradNotImplementedFallback());
    m.impl("feed_forward_backward", torch::autograd::autogradNotImplementedFallback());
    m.impl("dropout", &dropout_autograd);
}
