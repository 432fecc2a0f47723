// torch_attention.cpp -- the `attention` ops over the C ABI: argument checks, layout,
// workspace, autograd.
//
// Shapes and values that cannot be are ValueError (TORCH_CHECK_VALUE), wrong dtypes
// TypeError, as the package's Python layer raises them.
#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/autograd_not_implemented_fallback.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/library.h>

#include <algorithm>
#include <cmath>
#include <tuple>
#include <vector>

#include "../../include/torchmatch_amd.h"

namespace {

using at::Tensor;
using OptTensor = c10::optional<Tensor>;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

hipStream_t current_stream(const Tensor &t) {
    return c10::hip::getCurrentHIPStream(t.get_device()).stream();
}

void check_rc(int rc, const char *op) {
    TORCH_CHECK(rc != TM_ERR_LAUNCH, op, ": kernel launch failed"); // the entry took the error
    TORCH_CHECK(rc == TM_OK, op, ": the library refused the call (code ", rc, ")");
}

int dtype_code(const Tensor &t, const char *op, const char *name) {
    switch (t.scalar_type()) {
    case at::kBFloat16: return TM_BF16;
    case at::kHalf: return TM_F16;
    case at::kFloat: return TM_F32;
    default:
        TORCH_CHECK_TYPE(false, op, ": ", name, " must be bfloat16, float16 or float32, got ",
                         t.scalar_type());
    }
}

// strides of dimensions of one element are never used
int64_t step_of(const Tensor &t, int64_t dim) { return t.size(dim) > 1 ? t.stride(dim) : 0; }

// A (B, L, heads, D) tensor as the kernels read it: features contiguous and padded to 16
// bytes, rows and heads 16-byte aligned.  Projections' views are; others are copied.
Tensor readable(const Tensor &t) {
    const int64_t unit = 16 / t.element_size(), d = t.size(3);
    if (d % unit)
        return at::constant_pad_nd(t, {0, unit - d % unit}).contiguous();
    const bool ok = (d == 1 || t.stride(3) == 1) && step_of(t, 0) % unit == 0 &&
                    step_of(t, 1) % unit == 0 &&
                    step_of(t, 1) * t.element_size() < TM_ATTENTION_MAX_ROW_BYTES &&
                    step_of(t, 2) % unit == 0 &&
                    reinterpret_cast<uintptr_t>(t.const_data_ptr()) % 16 == 0;
    return ok ? t : t.clone(at::MemoryFormat::Contiguous);
}

struct Problem {
    tm_attention a = {};
    Tensor q, k, v; // as read; the rest is held by the caller
    int64_t d = 0;  // before padding
};

const float *floats(const OptTensor &t, const Tensor &q, const char *name, at::IntArrayRef sizes) {
    if (!t.has_value())
        return nullptr;
    TORCH_CHECK_TYPE(t->scalar_type() == at::kFloat, "attend: ", name, " must be float32, got ",
                     t->scalar_type());
    TORCH_CHECK_VALUE(t->device() == q.device(), "attend: ", name, " must be on q's device");
    TORCH_CHECK_VALUE(t->sizes() == sizes && t->is_contiguous(), "attend: ", name,
                      " must be contiguous of shape ", sizes, ", got ", t->sizes());
    // never null where given: an empty one stands for rows that are not there
    static const float none = 0.f;
    return t->numel() ? t->const_data_ptr<float>() : &none;
}

const int32_t *ints(const OptTensor &t, const Tensor &q, const char *name, at::IntArrayRef sizes) {
    if (!t.has_value())
        return nullptr;
    TORCH_CHECK_TYPE(t->scalar_type() == at::kInt, "attend: ", name, " must be int32, got ",
                     t->scalar_type());
    TORCH_CHECK_VALUE(t->device() == q.device(), "attend: ", name, " must be on q's device");
    TORCH_CHECK_VALUE(t->sizes() == sizes && t->is_contiguous(), "attend: ", name,
                      " must be contiguous of shape ", sizes, ", got ", t->sizes());
    static const int32_t none = 0;
    return t->numel() ? t->const_data_ptr<int32_t>() : &none;
}

Problem problem(const Tensor &q, const Tensor &k, const Tensor &v, const OptTensor &slopes,
                const OptTensor &q_pos, const OptTensor &k_pos, const OptTensor &q_docs,
                const OptTensor &k_docs, const OptTensor &prefix, const OptTensor &lengths,
                double scale, double cap, bool causal) {
    TORCH_CHECK_VALUE(q.dim() == 4 && k.dim() == 4 && v.dim() == 4,
                      "attend: q, k and v must be 4D (B, L, heads, D), got ", q.dim(), "D, ",
                      k.dim(), "D and ", v.dim(), "D");
    TORCH_CHECK_VALUE(k.device() == q.device() && v.device() == q.device(),
                      "attend: q, k and v must be on one device");
    TORCH_CHECK_TYPE(k.scalar_type() == q.scalar_type() && v.scalar_type() == q.scalar_type(),
                     "attend: q, k and v must have one dtype, got ", q.scalar_type(), ", ",
                     k.scalar_type(), " and ", v.scalar_type());
    Problem p;
    p.a.dtype = dtype_code(q, "attend", "q");
    const int64_t B = q.size(0), Lq = q.size(1), H = q.size(2), D = q.size(3);
    const int64_t Lk = k.size(1), Hkv = k.size(2);
    TORCH_CHECK_VALUE(k.sizes() == v.sizes(), "attend: k and v must have one shape, got ",
                      k.sizes(), " and ", v.sizes());
    TORCH_CHECK_VALUE(k.size(0) == B && k.size(3) == D, "attend: k must be (", B,
                      ", Lk, heads, ", D, ") as q is, got ", k.sizes());
    TORCH_CHECK_VALUE(H > 0 && Hkv > 0 && H % Hkv == 0,
                      "attend: the heads of q must be a multiple of those of k, got ", H, " and ",
                      Hkv);
    TORCH_CHECK_VALUE(D >= 1 && D <= tm_attention_max_head_dim(), "attend: heads hold 1 to ",
                      tm_attention_max_head_dim(), " features, got ", D);
    TORCH_CHECK_VALUE(B <= INT32_MAX && Lq <= INT32_MAX - 256 && Lk <= INT32_MAX - 256 &&
                          H <= INT32_MAX &&
                          (double)B * std::max((double)H * (double)((Lq + 31) / 32),
                                               (double)Hkv * (double)((Lk + 127) / 128)) <
                              TM_ATTENTION_MAX_BLOCKS,
                      "attend: too many rows for one call: q ", q.sizes(), ", k ", k.sizes());
    // as float32 numbers, with room for the factors that the kernels put to them
    const double most = 0x1p126;
    TORCH_CHECK_VALUE(std::abs(scale) <= most, "attend: scale must be finite in float32, got ",
                      scale);
    TORCH_CHECK_VALUE(cap >= 0. && cap <= most && (cap == 0.) == ((float)cap == 0.f),
                      "attend: cap must be positive in float32, or 0 for none, got ", cap);
    TORCH_CHECK_VALUE(cap == 0. || std::abs((float)scale / (float)cap) <= (float)most,
                      "attend: cap is too small for a scale of ", scale, ", got ", cap);
    TORCH_CHECK_VALUE(p.a.dtype == TM_F32 || cap <= TM_ATTENTION_MAX_CAP_16,
                      "attend: cap must be at most ", (int)TM_ATTENTION_MAX_CAP_16,
                      " for 16-bit types, got ", cap);
    TORCH_CHECK_VALUE(q_pos.has_value() == k_pos.has_value(),
                      "attend: give both q_positions and k_positions, or neither");
    TORCH_CHECK_VALUE(!q_pos.has_value() || slopes.has_value(),
                      "attend: positions have no effect without slopes");
    TORCH_CHECK_VALUE(q_docs.has_value() == k_docs.has_value(),
                      "attend: give both q_docs and k_docs, or neither");
    TORCH_CHECK_VALUE(!prefix.has_value() || causal, "attend: prefix needs causal=True");
    p.a.slopes = floats(slopes, q, "slopes", {H});
    if (q_pos.has_value()) {
        const int64_t axes = q_pos->dim() == 3 ? q_pos->size(2) : 0;
        TORCH_CHECK_VALUE(axes >= 1 && axes <= 3,
                          "attend: q_positions must be (B, Lq, 1 to 3 axes), got ",
                          q_pos->sizes());
        p.a.axes = (int32_t)axes;
        p.a.q_positions = floats(q_pos, q, "q_positions", {B, Lq, axes});
        p.a.k_positions = floats(k_pos, q, "k_positions", {B, Lk, axes});
    }
    p.a.q_docs = ints(q_docs, q, "q_docs", {B, Lq});
    p.a.k_docs = ints(k_docs, q, "k_docs", {B, Lk});
    p.a.prefix = ints(prefix, q, "prefix", {B});
    p.a.lengths = ints(lengths, q, "lengths", {B});
    p.q = readable(q);
    p.k = readable(k);
    p.v = readable(v);
    p.d = D;
    p.a.q = p.q.const_data_ptr();
    p.a.k = p.k.const_data_ptr();
    p.a.v = p.v.const_data_ptr();
    p.a.q_b = step_of(p.q, 0), p.a.q_l = step_of(p.q, 1), p.a.q_h = step_of(p.q, 2);
    p.a.k_b = step_of(p.k, 0), p.a.k_l = step_of(p.k, 1), p.a.k_h = step_of(p.k, 2);
    p.a.v_b = step_of(p.v, 0), p.a.v_l = step_of(p.v, 1), p.a.v_h = step_of(p.v, 2);
    p.a.B = (int32_t)B, p.a.Lq = (int32_t)Lq, p.a.Lk = (int32_t)Lk;
    p.a.H = (int32_t)H, p.a.Hkv = (int32_t)Hkv, p.a.D = (int32_t)p.q.size(3);
    p.a.causal = causal;
    p.a.scale = (float)scale, p.a.cap = (float)cap;
    return p;
}

Tensor narrowed(const Tensor &t, int64_t d) {
    return t.size(3) == d ? t : t.narrow(3, 0, d).contiguous();
}

// `with_low`: also what rounding took off the output (empty for float32)
std::tuple<Tensor, Tensor, Tensor>
forward(const Tensor &q, const Tensor &k, const Tensor &v, const OptTensor &slopes,
        const OptTensor &q_pos, const OptTensor &k_pos, const OptTensor &q_docs,
        const OptTensor &k_docs, const OptTensor &prefix, const OptTensor &lengths, double scale,
        double cap, bool causal, bool with_low) {
    const c10::DeviceGuard guard(q.device());
    const Problem p = problem(q, k, v, slopes, q_pos, k_pos, q_docs, k_docs, prefix, lengths,
                              scale, cap, causal);
    Tensor out = at::empty({p.a.B, p.a.Lq, p.a.H, p.a.D}, q.options());
    Tensor lse = at::empty({p.a.B, p.a.H, p.a.Lq}, q.options().dtype(at::kFloat)), low;
    with_low = with_low && p.a.dtype != TM_F32;
    if (with_low)
        low = at::empty_like(out);
    if (out.numel()) {
        const size_t bytes = tm_attention_workspace_bytes(&p.a);
        Tensor ws;
        if (bytes)
            ws = at::empty({(int64_t)bytes}, q.options().dtype(at::kByte));
        check_rc(tm_attention_forward(&p.a, out.data_ptr(), with_low ? low.data_ptr() : nullptr,
                                      lse.data_ptr<float>(), bytes ? ws.data_ptr() : nullptr,
                                      bytes, current_stream(q)),
                 "attend");
    }
    return {narrowed(out, p.d), with_low ? narrowed(low, p.d) : low, lse};
}

std::tuple<Tensor, Tensor> attend_hip(const Tensor &q, const Tensor &k, const Tensor &v,
                                      const OptTensor &slopes, const OptTensor &q_pos,
                                      const OptTensor &k_pos, const OptTensor &q_docs,
                                      const OptTensor &k_docs, const OptTensor &prefix,
                                      const OptTensor &lengths, double scale, double cap,
                                      bool causal) {
    auto [out, low, lse] = forward(q, k, v, slopes, q_pos, k_pos, q_docs, k_docs, prefix,
                                   lengths, scale, cap, causal, false);
    return {out, lse};
}

std::tuple<Tensor, Tensor, Tensor>
attend_forward_hip(const Tensor &q, const Tensor &k, const Tensor &v, const OptTensor &slopes,
                   const OptTensor &q_pos, const OptTensor &k_pos, const OptTensor &q_docs,
                   const OptTensor &k_docs, const OptTensor &prefix, const OptTensor &lengths,
                   double scale, double cap, bool causal) {
    auto [out, low, lse] = forward(q, k, v, slopes, q_pos, k_pos, q_docs, k_docs, prefix,
                                   lengths, scale, cap, causal, true);
    return {out, low.defined() ? low : at::empty({0}, q.options()), lse};
}

std::tuple<Tensor, Tensor, Tensor>
attend_backward_hip(const Tensor &dout, const Tensor &q, const Tensor &k, const Tensor &v,
                    const Tensor &out, const Tensor &out_low, const Tensor &lse,
                    const OptTensor &slopes, const OptTensor &q_pos, const OptTensor &k_pos,
                    const OptTensor &q_docs, const OptTensor &k_docs, const OptTensor &prefix,
                    const OptTensor &lengths, const OptTensor &dlse, double scale, double cap,
                    bool causal) {
    const c10::DeviceGuard guard(q.device());
    const Problem p = problem(q, k, v, slopes, q_pos, k_pos, q_docs, k_docs, prefix, lengths,
                              scale, cap, causal);
    TORCH_CHECK_VALUE(dout.sizes() == q.sizes() && out.sizes() == q.sizes(),
                      "attend_backward: dout and out must have q's shape");
    TORCH_CHECK_TYPE(dout.scalar_type() == q.scalar_type() &&
                         out.scalar_type() == q.scalar_type() && lse.scalar_type() == at::kFloat,
                     "attend_backward: dout and out must have q's dtype and lse float32");
    TORCH_CHECK_VALUE(dout.device() == q.device() && out.device() == q.device() &&
                          lse.device() == q.device(),
                      "attend_backward: tensors must be on one device");
    TORCH_CHECK_VALUE(lse.dim() == 3 && lse.size(0) == q.size(0) && lse.size(1) == q.size(2) &&
                          lse.size(2) == q.size(1) && lse.is_contiguous(),
                      "attend_backward: lse must be a contiguous (B, H, Lq)");
    Tensor dl;
    if (dlse.has_value()) {
        TORCH_CHECK_TYPE(dlse->scalar_type() == at::kFloat,
                         "attend_backward: dlse must be float32, got ", dlse->scalar_type());
        TORCH_CHECK_VALUE(dlse->sizes() == lse.sizes() && dlse->device() == q.device(),
                          "attend_backward: dlse must be as lse, got ", dlse->sizes());
        dl = dlse->contiguous();
    }
    const bool has_low = out_low.numel() && p.a.dtype != TM_F32;
    TORCH_CHECK_VALUE(!has_low || (out_low.sizes() == q.sizes() &&
                                   out_low.device() == q.device() &&
                                   out_low.scalar_type() == q.scalar_type()),
                      "attend_backward: out_low must be as out, or empty");
    const Tensor o = readable(out).contiguous(), g = readable(dout);
    const Tensor low = has_low ? readable(out_low).contiguous() : out_low;
    Tensor dq = at::empty(p.q.sizes(), q.options()), dk = at::empty(p.k.sizes(), q.options()),
           dv = at::empty(p.k.sizes(), q.options());
    if (dq.numel() || dk.numel()) {
        const size_t bytes = tm_attention_backward_workspace_bytes(&p.a);
        Tensor ws = at::empty({(int64_t)bytes}, q.options().dtype(at::kByte));
        check_rc(tm_attention_backward_lse(
                     &p.a, o.const_data_ptr(), has_low ? low.const_data_ptr() : nullptr,
                     lse.const_data_ptr<float>(),
                     dl.defined() ? dl.const_data_ptr<float>() : nullptr, g.const_data_ptr(),
                     step_of(g, 0), step_of(g, 1), step_of(g, 2), dq.data_ptr(), dk.data_ptr(),
                     dv.data_ptr(), ws.data_ptr(), bytes, current_stream(q)),
                 "attend_backward");
    }
    return {narrowed(dq, p.d), narrowed(dk, p.d), narrowed(dv, p.d)};
}

Tensor rotate_hip(const Tensor &x, const Tensor &positions, const Tensor &freqs,
                  at::IntArrayRef sections, bool interleaved, bool inverse) {
    const c10::DeviceGuard guard(x.device());
    TORCH_CHECK_VALUE(x.dim() == 4, "rotate: x must be 4D (B, L, heads, D), got ", x.dim(), "D");
    tm_rotation r = {};
    r.dtype = dtype_code(x, "rotate", "x");
    const int64_t B = x.size(0), L = x.size(1), H = x.size(2), D = x.size(3);
    TORCH_CHECK_VALUE(B <= INT32_MAX && L <= INT32_MAX && D >= 1 && H * D <= (1 << 24) &&
                          D <= 8192,
                      "rotate: shape not supported: ", x.sizes());
    const int64_t axes = (int64_t)sections.size();
    TORCH_CHECK_VALUE(axes >= 1 && axes <= TM_ROTATE_MAX_AXES, "rotate: 1 to ",
                      (int)TM_ROTATE_MAX_AXES, " sections, one an axis, got ", axes);
    int64_t pairs = 0;
    for (int64_t a = 0; a < axes; ++a) {
        TORCH_CHECK_VALUE(sections[a] >= 0 && sections[a] <= D,
                          "rotate: sections must be pair counts, got ", sections);
        r.sections[a] = (int32_t)sections[a];
        pairs += sections[a];
    }
    TORCH_CHECK_VALUE(2 * pairs <= D, "rotate: sections hold ", pairs,
                      " pairs, more than half of the ", D, " features");
    TORCH_CHECK_VALUE(positions.device() == x.device() && freqs.device() == x.device(),
                      "rotate: x, positions and freqs must be on one device");
    TORCH_CHECK_VALUE(positions.dim() == 3 && positions.size(0) == B && positions.size(1) == L &&
                          positions.size(2) == axes,
                      "rotate: positions must be (", B, ", ", L, ", ", axes, "), got ",
                      positions.sizes());
    TORCH_CHECK_TYPE(freqs.scalar_type() == at::kFloat, "rotate: freqs must be float32, got ",
                     freqs.scalar_type());
    TORCH_CHECK_VALUE(freqs.dim() == 1 && freqs.size(0) == pairs && freqs.is_contiguous(),
                      "rotate: freqs must be a contiguous (", pairs, "), got ", freqs.sizes());
    switch (positions.scalar_type()) {
    case at::kFloat: r.pos_type = TM_POS_F32; break;
    case at::kInt: r.pos_type = TM_POS_I32; break;
    case at::kLong: r.pos_type = TM_POS_I64; break;
    default:
        TORCH_CHECK_TYPE(false, "rotate: positions must be float32, int32 or int64, got ",
                         positions.scalar_type());
    }
    // rows of positions shared by the batch (an expanded tensor) are read in place
    const bool rows = step_of(positions, 2) == (axes > 1 ? 1 : 0) &&
                      step_of(positions, 1) == (L > 1 ? axes : 0);
    const Tensor pos = rows ? positions : positions.contiguous();
    const Tensor in = D == 1 || x.stride(3) == 1 ? x : x.contiguous();
    Tensor out = at::empty(x.sizes(), x.options());
    if (!out.numel())
        return out;
    r.x = in.const_data_ptr();
    r.positions = pos.const_data_ptr();
    r.freqs = freqs.const_data_ptr<float>();
    r.x_b = step_of(in, 0), r.x_l = step_of(in, 1), r.x_h = step_of(in, 2);
    r.pos_b = step_of(pos, 0);
    r.B = (int32_t)B, r.L = (int32_t)L, r.H = (int32_t)H, r.D = (int32_t)D;
    r.axes = (int32_t)axes, r.interleaved = interleaved, r.inverse = inverse;
    check_rc(tm_rotate(&r, out.data_ptr(), current_stream(x)), "rotate");
    return out;
}

// ---- autograd ---------------------------------------------------------------------

bool wants_grad(const Tensor &t) { return at::GradMode::is_enabled() && t.requires_grad(); }

// Whether forward-mode differentiation is under way (it goes by no grad mode): below autograd
// the tangent would be lost without a word.
bool has_tangent(const Tensor &t) { return t.defined() && t._fw_grad(/*level=*/0).defined(); }

void constant(const OptTensor &t, const char *op, const char *name) {
    TORCH_CHECK_NOT_IMPLEMENTED(!t.has_value() || !(wants_grad(*t) || has_tangent(*t)), op,
                                ": no gradient for ", name);
}

template <typename... R>
using AttendOp = std::tuple<R...>(const Tensor &, const Tensor &, const Tensor &,
                                  const OptTensor &, const OptTensor &, const OptTensor &,
                                  const OptTensor &, const OptTensor &, const OptTensor &,
                                  const OptTensor &, double, double, bool);

struct AttendFunction : torch::autograd::Function<AttendFunction> {
    static variable_list forward(AutogradContext *ctx, const Tensor &q, const Tensor &k,
                                 const Tensor &v, const std::vector<OptTensor> &masks,
                                 double scale, double cap, bool causal) {
        at::AutoDispatchBelowADInplaceOrView below;
        static auto op = c10::Dispatcher::singleton()
                             .findSchemaOrThrow("attention::attend_forward", "")
                             .typed<AttendOp<Tensor, Tensor, Tensor>>();
        auto [out, low, lse] = op.call(q, k, v, masks[0], masks[1], masks[2], masks[3], masks[4],
                                       masks[5], masks[6], scale, cap, causal);
        variable_list saved = {q, k, v, out, low, lse};
        for (const auto &m : masks)
            saved.push_back(m.has_value() ? *m : Tensor());
        ctx->save_for_backward(saved);
        ctx->saved_data["scale"] = scale;
        ctx->saved_data["cap"] = cap;
        ctx->saved_data["causal"] = causal;
        // either output may go unused: no zeros are made up for its gradient
        ctx->set_materialize_grads(false);
        return {out, lse};
    }
    static variable_list backward(AutogradContext *ctx, const variable_list &grads) {
        const auto s = ctx->get_saved_variables();
        variable_list result(7);
        if (!grads[0].defined() && !grads[1].defined())
            return result;
        const Tensor dout = grads[0].defined() ? grads[0] : at::zeros_like(s[3]);
        const auto opt = [&](int i) { return s[i].defined() ? OptTensor(s[i]) : OptTensor(); };
        static auto op =
            c10::Dispatcher::singleton()
                .findSchemaOrThrow("attention::attend_backward", "")
                .typed<std::tuple<Tensor, Tensor, Tensor>(
                    const Tensor &, const Tensor &, const Tensor &, const Tensor &,
                    const Tensor &, const Tensor &, const Tensor &, const OptTensor &,
                    const OptTensor &, const OptTensor &, const OptTensor &, const OptTensor &,
                    const OptTensor &, const OptTensor &, const OptTensor &, double, double,
                    bool)>();
        auto [dq, dk, dv] =
            op.call(dout, s[0], s[1], s[2], s[3], s[4], s[5], opt(6), opt(7), opt(8), opt(9),
                    opt(10), opt(11), opt(12),
                    grads[1].defined() ? OptTensor(grads[1]) : OptTensor(),
                    ctx->saved_data["scale"].toDouble(), ctx->saved_data["cap"].toDouble(),
                    ctx->saved_data["causal"].toBool());
        result[0] = dq;
        result[1] = dk;
        result[2] = dv;
        return result;
    }
};

std::tuple<Tensor, Tensor> attend_autograd(const Tensor &q, const Tensor &k, const Tensor &v,
                                           const OptTensor &slopes, const OptTensor &q_pos,
                                           const OptTensor &k_pos, const OptTensor &q_docs,
                                           const OptTensor &k_docs, const OptTensor &prefix,
                                           const OptTensor &lengths, double scale, double cap,
                                           bool causal) {
    const std::vector<OptTensor> masks = {slopes, q_pos, k_pos, q_docs, k_docs, prefix, lengths};
    constant(slopes, "attend", "slopes");
    constant(q_pos, "attend", "q_positions");
    constant(k_pos, "attend", "k_positions");
    TORCH_CHECK_NOT_IMPLEMENTED(!has_tangent(q) && !has_tangent(k) && !has_tangent(v),
                                "attend: no forward-mode derivative");
    if (wants_grad(q) || wants_grad(k) || wants_grad(v)) {
        auto r = AttendFunction::apply(q, k, v, masks, scale, cap, causal);
        return {r[0], r[1]};
    }
    at::AutoDispatchBelowADInplaceOrView below;
    static auto op = c10::Dispatcher::singleton()
                         .findSchemaOrThrow("attention::attend", "")
                         .typed<AttendOp<Tensor, Tensor>>();
    return op.call(q, k, v, slopes, q_pos, k_pos, q_docs, k_docs, prefix, lengths, scale, cap,
                   causal);
}

Tensor call_rotate(const Tensor &x, const Tensor &positions, const Tensor &freqs,
                   at::IntArrayRef sections, bool interleaved, bool inverse) {
    static auto op = c10::Dispatcher::singleton()
                         .findSchemaOrThrow("attention::rotate", "")
                         .typed<Tensor(const Tensor &, const Tensor &, const Tensor &,
                                       at::IntArrayRef, bool, bool)>();
    return op.call(x, positions, freqs, sections, interleaved, inverse);
}

struct RotateFunction : torch::autograd::Function<RotateFunction> {
    static Tensor forward(AutogradContext *ctx, const Tensor &x, const Tensor &positions,
                          const Tensor &freqs, at::IntArrayRef sections, bool interleaved,
                          bool inverse) {
        at::AutoDispatchBelowADInplaceOrView below;
        ctx->save_for_backward({positions, freqs});
        ctx->saved_data["sections"] = sections.vec();
        ctx->saved_data["interleaved"] = interleaved;
        ctx->saved_data["inverse"] = inverse;
        return call_rotate(x, positions, freqs, sections, interleaved, inverse);
    }
    static variable_list backward(AutogradContext *ctx, const variable_list &grads) {
        variable_list result(6);
        if (!grads[0].defined())
            return result;
        const auto s = ctx->get_saved_variables();
        // a rotation of the other sense, differentiable again
        result[0] = call_rotate(grads[0], s[0], s[1], ctx->saved_data["sections"].toIntVector(),
                                ctx->saved_data["interleaved"].toBool(),
                                !ctx->saved_data["inverse"].toBool());
        return result;
    }
};

Tensor rotate_autograd(const Tensor &x, const Tensor &positions, const Tensor &freqs,
                       at::IntArrayRef sections, bool interleaved, bool inverse) {
    constant(positions, "rotate", "positions");
    constant(freqs, "rotate", "freqs");
    if (has_tangent(x)) { // linear in x: the tangent turns as x does
        const auto [primal, tangent] = at::_unpack_dual(x, /*level=*/0);
        return at::_make_dual(
            rotate_autograd(primal, positions, freqs, sections, interleaved, inverse),
            rotate_autograd(tangent, positions, freqs, sections, interleaved, inverse),
            /*level=*/0);
    }
    if (wants_grad(x))
        return RotateFunction::apply(x, positions, freqs, sections, interleaved, inverse);
    at::AutoDispatchBelowADInplaceOrView below;
    return call_rotate(x, positions, freqs, sections, interleaved, inverse);
}

} // namespace

TORCH_LIBRARY(attention, m) {
    m.def("attend(Tensor q, Tensor k, Tensor v, Tensor? slopes=None, Tensor? q_positions=None, "
          "Tensor? k_positions=None, Tensor? q_docs=None, Tensor? k_docs=None, "
          "Tensor? prefix=None, Tensor? lengths=None, *, float scale, float cap=0., "
          "bool causal=False) -> (Tensor, Tensor)");
    // the same with what rounding took off the output, for attend_backward
    m.def("attend_forward(Tensor q, Tensor k, Tensor v, Tensor? slopes=None, "
          "Tensor? q_positions=None, Tensor? k_positions=None, Tensor? q_docs=None, "
          "Tensor? k_docs=None, Tensor? prefix=None, Tensor? lengths=None, *, float scale, "
          "float cap=0., bool causal=False) -> (Tensor, Tensor, Tensor)");
    m.def("attend_backward(Tensor dout, Tensor q, Tensor k, Tensor v, Tensor out, "
          "Tensor out_low, Tensor lse, "
          "Tensor? slopes=None, Tensor? q_positions=None, Tensor? k_positions=None, "
          "Tensor? q_docs=None, Tensor? k_docs=None, Tensor? prefix=None, "
          "Tensor? lengths=None, Tensor? dlse=None, *, float scale, float cap=0., "
          "bool causal=False) -> (Tensor, Tensor, Tensor)");
    m.def("rotate(Tensor x, Tensor positions, Tensor freqs, int[] sections, "
          "bool interleaved=False, bool inverse=False) -> Tensor");
}

TORCH_LIBRARY_IMPL(attention, CUDA, m) {
    m.impl("attend", &attend_hip);
    m.impl("attend_forward", &attend_forward_hip);
    m.impl("attend_backward", &attend_backward_hip);
    m.impl("rotate", &rotate_hip);
}

TORCH_LIBRARY_IMPL(attention, Autograd, m) {
    m.impl("attend", &attend_autograd);
    m.impl("attend_forward", torch::autograd::autogradNotImplementedFallback());
    m.impl("attend_backward", torch::autograd::autogradNotImplementedFallback());
    m.impl("rotate", &rotate_autograd);
}
