// torch_support.h -- what the `attention` ops' files share: argument checks, layout, streams,
// gradients' conditions.
//
// Shapes and values that cannot be are ValueError (TORCH_CHECK_VALUE), wrong dtypes
// TypeError, as the package's Python layer raises them.
#ifndef TORCHMATCH_AMD_TORCH_SUPPORT_H
#define TORCHMATCH_AMD_TORCH_SUPPORT_H

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

namespace tmsupport {

using at::Tensor;
using OptTensor = c10::optional<Tensor>;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

inline hipStream_t current_stream(const Tensor &t) {
    return c10::hip::getCurrentHIPStream(t.get_device()).stream();
}

inline void check_rc(int rc, const char *op) {
    TORCH_CHECK(rc != TM_ERR_LAUNCH, op, ": kernel launch failed"); // the entry took the error
    TORCH_CHECK(rc == TM_OK, op, ": the library refused the call (code ", rc, ")");
}

inline int dtype_code(const Tensor &t, const char *op, const char *name) {
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
inline int64_t step_of(const Tensor &t, int64_t dim) { return t.size(dim) > 1 ? t.stride(dim) : 0; }

// A (B, L, heads, D) tensor as the kernels read it: features contiguous and padded to 16
// bytes, rows and heads 16-byte aligned.  Projections' views are; others are copied.
inline Tensor readable(const Tensor &t) {
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

// A rotation's arguments, checked, as the library takes them.
struct Rotation {
    tm_rotation r = {};
    Tensor in, pos; // as read; the rest is held by the caller
    Rotation(const char *op, const Tensor &x, const Tensor &positions, const Tensor &freqs,
             at::IntArrayRef sections, bool interleaved, bool inverse) {
        TORCH_CHECK_VALUE(x.dim() == 4, op, ": x must be 4D (B, L, heads, D), got ", x.dim(), "D");
        r.dtype = dtype_code(x, op, "x");
        const int64_t B = x.size(0), L = x.size(1), H = x.size(2), D = x.size(3);
        TORCH_CHECK_VALUE(B <= INT32_MAX && L <= INT32_MAX && D >= 1 && H * D <= (1 << 24) &&
                              D <= 8192,
                          op, ": shape not supported: ", x.sizes());
        const int64_t axes = (int64_t)sections.size();
        TORCH_CHECK_VALUE(axes >= 1 && axes <= TM_ROTATE_MAX_AXES, op, ": 1 to ",
                          (int)TM_ROTATE_MAX_AXES, " sections, one an axis, got ", axes);
        int64_t pairs = 0;
        for (int64_t a = 0; a < axes; ++a) {
            TORCH_CHECK_VALUE(sections[a] >= 0 && sections[a] <= D,
                              op, ": sections must be pair counts, got ", sections);
            r.sections[a] = (int32_t)sections[a];
            pairs += sections[a];
        }
        TORCH_CHECK_VALUE(2 * pairs <= D, op, ": sections hold ", pairs,
                          " pairs, more than half of the ", D, " features");
        TORCH_CHECK_VALUE(positions.device() == x.device() && freqs.device() == x.device(),
                          op, ": x, positions and freqs must be on one device");
        TORCH_CHECK_VALUE(positions.dim() == 3 && positions.size(0) == B && positions.size(1) == L &&
                              positions.size(2) == axes,
                          op, ": positions must be (", B, ", ", L, ", ", axes, "), got ",
                          positions.sizes());
        TORCH_CHECK_TYPE(freqs.scalar_type() == at::kFloat, op, ": freqs must be float32, got ",
                         freqs.scalar_type());
        TORCH_CHECK_VALUE(freqs.dim() == 1 && freqs.size(0) == pairs && freqs.is_contiguous(),
                          op, ": freqs must be a contiguous (", pairs, "), got ", freqs.sizes());
        switch (positions.scalar_type()) {
        case at::kFloat: r.pos_type = TM_POS_F32; break;
        case at::kInt: r.pos_type = TM_POS_I32; break;
        case at::kLong: r.pos_type = TM_POS_I64; break;
        default:
            TORCH_CHECK_TYPE(false, op, ": positions must be float32, int32 or int64, got ",
                             positions.scalar_type());
        }
        // rows of positions shared by the batch (an expanded tensor) are read in place
        const bool rows = step_of(positions, 2) == (axes > 1 ? 1 : 0) &&
                          step_of(positions, 1) == (L > 1 ? axes : 0);
        pos = rows ? positions : positions.contiguous();
        in = D == 1 || x.stride(3) == 1 ? x : x.contiguous();
        r.x = in.const_data_ptr();
        r.positions = pos.const_data_ptr();
        r.freqs = freqs.const_data_ptr<float>();
        r.x_b = step_of(in, 0), r.x_l = step_of(in, 1), r.x_h = step_of(in, 2);
        r.pos_b = step_of(pos, 0);
        r.B = (int32_t)B, r.L = (int32_t)L, r.H = (int32_t)H, r.D = (int32_t)D;
        r.axes = (int32_t)axes, r.interleaved = interleaved, r.inverse = inverse;
    }
};

inline bool wants_grad(const Tensor &t) { return at::GradMode::is_enabled() && t.requires_grad(); }

// Whether forward-mode differentiation is under way (it goes by no grad mode): below autograd
// the tangent would be lost without a word.
inline bool has_tangent(const Tensor &t) { return t.defined() && t._fw_grad(/*level=*/0).defined(); }

inline void constant(const OptTensor &t, const char *op, const char *name) {
    TORCH_CHECK_NOT_IMPLEMENTED(!t.has_value() || !(wants_grad(*t) || has_tangent(*t)), op,
                                ": no gradient for ", name);
}

} // namespace tmsupport

#endif
