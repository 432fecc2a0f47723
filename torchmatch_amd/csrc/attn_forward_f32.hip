// attn_forward_f32.hip -- attention forward, float inputs (a file per type, so that they compile side by side).
#include "attn_forward.h"
#include "attn_tokens.h"

namespace attn {

int forward_f32(const Args &a, int dp, hipStream_t s) {
    switch (dp) {
    case 32: return run_forward<float, 32>(a, s);
    case 64: return run_forward<float, 64>(a, s);
    case 96: return run_forward<float, 96>(a, s);
    case 128: return run_forward<float, 128>(a, s);
    case 256: return run_forward<float, 256>(a, s);
    default: return 1;
    }
}

int tokens_f32(const Args &a, int dp, hipStream_t s) {
    switch (dp) {
    case 32: return run_tokens<float, 32>(a, s);
    case 64: return run_tokens<float, 64>(a, s);
    case 96: return run_tokens<float, 96>(a, s);
    case 128: return run_tokens<float, 128>(a, s);
    case 256: return run_tokens<float, 256>(a, s);
    default: return 1;
    }
}

int join_f32(const Args &a, int dp, hipStream_t s) {
    switch (dp) {
    case 32: return run_join<float, 32>(a, s);
    case 64: return run_join<float, 64>(a, s);
    case 96: return run_join<float, 96>(a, s);
    case 128: return run_join<float, 128>(a, s);
    case 256: return run_join<float, 256>(a, s);
    default: return 1;
    }
}

} // namespace attn
