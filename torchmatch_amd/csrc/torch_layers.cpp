// torch_layers.cpp -- the `attention` ops of the layer around attention over the C ABI: normed
// rotation, dropout.  Argument checks, layout, workspace, autograd.
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
        TORCH_CHECK_VALUE(H >= 1, "norm_rotate: x must have a head, got ", x.sizes());
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
    // the seed lies in seed_at where it is given
    m.def("dropout(Tensor x, float p, int seed=0, int offset=0, Tensor? seed_at=None, "
          "Tensor? residual=None) -> Tensor");
}

TORCH_LIBRARY_IMPL(attention, CUDA, m) {
    m.impl("norm_rotate", &norm_rotate_hip);
    m.impl("norm_rotate_backward", &norm_rotate_backward_hip);
    m.impl("dropout", &dropout_hip);
}

TORCH_LIBRARY_IMPL(attention, Autograd, m) {
    m.impl("norm_rotate", &norm_rotate_autograd);
    m.impl("norm_rotate_backward", torch::autograd::autogradNotImplementedFallback());
    m.impl("dropout", &dropout_autograd);
}
