// attn_backward_bf16.hip -- attention backward, __bf16 inputs (a file per type, so that they compile side by side).
#include "attn_backward.h"

namespace attn {

int backward_kv_bf16(const Args &a, int dp, hipStream_t s) {
    switch (dp) {
    case 32: return run_backward_kv<__bf16, 32>(a, s);
    case 64: return run_backward_kv<__bf16, 64>(a, s);
    case 96: return run_backward_kv<__bf16, 96>(a, s);
    case 128: return run_backward_kv<__bf16, 128>(a, s);
    case 256: return run_backward_kv<__bf16, 256>(a, s);
    default: return 1;
    }
}

int backward_q_bf16(const Args &a, int dp, hipStream_t s) {
    switch (dp) {
    case 32: return run_backward_q<__bf16, 32>(a, s);
    case 64: return run_backward_q<__bf16, 64>(a, s);
    case 96: return run_backward_q<__bf16, 96>(a, s);
    case 128: return run_backward_q<__bf16, 128>(a, s);
    case 256: return run_backward_q<__bf16, 256>(a, s);
    default: return 1;
    }
}

int backward_join_bf16(const Args &a, hipStream_t s) { return run_backward_join<__bf16>(a, s); }

int delta_bf16(const Args &a, const float *lse, float *base2, float *delta, hipStream_t s) {
    return run_delta<__bf16>(a, lse, base2, delta, s);
}

} // namespace attn
