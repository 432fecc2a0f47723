// ff_bf16.hip -- the feed-forward products of one type.
#include "ff_tile.h"

namespace ff {

int product_bf16(const Args &p, Kind kind, bool big, hipStream_t stream) {
    return run<__bf16>(p, kind, big, stream);
}
int join_bf16(const Args &p, hipStream_t stream) { return run_join<__bf16>(p, stream); }

} // namespace ff
