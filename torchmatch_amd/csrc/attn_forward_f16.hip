// attn_forward_f16.hip -- attention forward, _Float16 inputs (a file per type, so that they compile side by side).
#include "attn_forward.h"
#include "attn_tokens.h"

namespace attn {

int forward_f16(const Args &a, int dp, hipStream_t s) {
    switch (dp) {
    case 32: return run_forward<_Float16, 32>(a, s);
    case 64: return run_forward<_Float16, 64>(a, s);
    case 96: return run_forward<_Float16, 96>(a, s);
    case 128: return run_forward<_Float16, 128>(a, s);
    case 256: return run_forward<_Float16, 256>(a, s);
    default: return 1;
    }
}

int tokens_f16(const Args &a, int dp, hipStream_t s) {
    switch (dp) {
    case 32: return run_tokens<_Float16, 32>(a, s);
    case 64: return run_tokens<_Float16, 64>(a, s);
    case 96: return run_tokens<_Float16, 96>(a, s);
    case 128: return run_tokens<_Float16, 128>(a, s);
    case 256: return run_tokens<_Float16, 256>(a, s);
    default: return 1;
    }
}

int join_f16(const Args &a, int dp, hipStream_t s) {
    switch (dp) {
    case 32: return run_join<_Float16, 32>(a, s);
    case 64: return run_join<_Float16, 64>(a, s);
    case 96: return run_join<_Float16, 96>(a, s);
    case 128: return run_join<_Float16, 128>(a, s);
    case 256: return run_join<_Float16, 256>(a, s);
    default: return 1;
    }
}

} // namespace attn
