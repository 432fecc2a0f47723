// attn_backward_f32.hip -- attention backward, float inputs (a file per type, so that they compile side by side).
#include "attn_backward.h"

namespace attn {

int backward_kv_f32(const Args &a, int dp, hipStream_t s) {
    switch (dp) {
    case 32: return run_backward_kv<float, 32>(a, s);
    case 64: return run_backward_kv<float, 64>(a, s);
    case 96: return run_backward_kv<float, 96>(a, s);
    case 128: return run_backward_kv<float, 128>(a, s);
    case 256: return run_backward_kv<float, 256>(a, s);
    default: return 1;
    }
}

int backward_q_f32(const Args &a, int dp, hipStream_t s) {
    switch (dp) {
    case 32: return run_backward_q<float, 32>(a, s);
    case 64: return run_backward_q<float, 64>(a, s);
    case 96: return run_backward_q<float, 96>(a, s);
    case 128: return run_backward_q<float, 128>(a, s);
    case 256: return run_backward_q<float, 256>(a, s);
    default: return 1;
    }
}

int backward_join_f32(const Args &a, hipStream_t s) { return run_backward_join<float>(a, s); }

int delta_f32(const Args &a, const float *lse, float *base2, float *delta, hipStream_t s) {
    return run_delta<float>(a, lse, base2, delta, s);
}

} // namespace attn
