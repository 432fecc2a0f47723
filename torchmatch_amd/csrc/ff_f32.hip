// ff_f32.hip -- the feed-forward products of one type.
#include "ff_tokens.h"

namespace ff {

int product_f32(const Args &p, Kind kind, int size, hipStream_t stream) {
    return run<float>(p, kind, size, stream);
}
int tokens_f32(const Args &p, Kind kind, hipStream_t stream) {
    return run_tokens<float>(p, kind, stream);
}

} // namespace ff
