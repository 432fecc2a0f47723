// attn_backward_f16.hip -- attention backward, _Float16 inputs (a file per type, so that they compile side by side).
#include "attn_backward.h"

namespace attn {

int backward_kv_f16(const Args &a, int dp, hipStream_t s) {
    switch (dp) {
    case 32: return run_backward_kv<_Float16, 32>(a, s);
    case 64: return run_backward_kv<_Float16, 64>(a, s);
    case 96: return run_backward_kv<_Float16, 96>(a, s);
    case 128: return run_backward_kv<_Float16, 128>(a, s);
    case 256: return run_backward_kv<_Float16, 256>(a, s);
    default: return 1;
    }
}

int backward_q_f16(const Args &a, int dp, hipStream_t s) {
    switch (dp) {
    case 32: return run_backward_q<_Float16, 32>(a, s);
    case 64: return run_backward_q<_Float16, 64>(a, s);
    case 96: return run_backward_q<_Float16, 96>(a, s);
    case 128: return run_backward_q<_Float16, 128>(a, s);
    case 256: return run_backward_q<_Float16, 256>(a, s);
    default: return 1;
    }
}

int backward_join_f16(const Args &a, hipStream_t s) { return run_backward_join<_Float16>(a, s); }

int delta_f16(const Args &a, const float *lse, float *base2, float *delta, hipStream_t s) {
    return run_delta<_Float16>(a, lse, base2, delta, s);
}

} // namespace attn
