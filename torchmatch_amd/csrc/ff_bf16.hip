// ff_bf16.hip -- the feed-forward products of one type.
#include "ff_tokens.h"

namespace ff {

int product_bf16(const Args &p, Kind kind, int size, hipStream_t stream) {
    return run<__bf16>(p, kind, size, stream);
}
int tokens_bf16(const Args &p, Kind kind, hipStream_t stream) {
    return run_tokens<__bf16>(p, kind, stream);
}

} // namespace ff
