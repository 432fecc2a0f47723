// ff_f16.hip -- the feed-forward products of one type.
#include "ff_tokens.h"

namespace ff {

int product_f16(const Args &p, Kind kind, int size, hipStream_t stream) {
    return run<_Float16>(p, kind, size, stream);
}
int tokens_f16(const Args &p, Kind kind, hipStream_t stream) {
    return run_tokens<_Float16>(p, kind, stream);
}

} // namespace ff
