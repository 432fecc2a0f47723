// attn_forward_bf16.hip -- attention forward, __bf16 inputs (a file per type, so that they compile side by side).
#include "attn_forward.h"
#include "attn_tokens.h"

namespace attn {

int forward_bf16(const Args &a, int dp, hipStream_t s) {
    switch (dp) {
    case 32: return run_forward<__bf16, 32>(a, s);
    case 64: return run_forward<__bf16, 64>(a, s);
    case 96: return run_forward<__bf16, 96>(a, s);
    case 128: return run_forward<__bf16, 128>(a, s);
    case 256: return run_forward<__bf16, 256>(a, s);
    default: return 1;
    }
}

int tokens_bf16(const Args &a, int dp, hipStream_t s) {
    switch (dp) {
    case 32: return run_tokens<__bf16, 32>(a, s);
    case 64: return run_tokens<__bf16, 64>(a, s);
    case 96: return run_tokens<__bf16, 96>(a, s);
    case 128: return run_tokens<__bf16, 128>(a, s);
    case 256: return run_tokens<__bf16, 256>(a, s);
    default: return 1;
    }
}

int join_bf16(const Args &a, int dp, hipStream_t s) {
    switch (dp) {
    case 32: return run_join<__bf16, 32>(a, s);
    case 64: return run_join<__bf16, 64>(a, s);
    case 96: return run_join<__bf16, 96>(a, s);
    case 128: return run_join<__bf16, 128>(a, s);
    case 256: return run_join<__bf16, 256>(a, s);
    default: return 1;
    }
}

} // namespace attn
