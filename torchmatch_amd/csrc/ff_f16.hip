// ff_f16.hip -- the feed-forward products of one type.
#include "ff_tile.h"

namespace ff {

int product_f16(const Args &p, Kind kind, bool big, hipStream_t stream) {
    return run<_Float16>(p, kind, big, stream);
}
int join_f16(const Args &p, hipStream_t stream) { return run_join<_Float16>(p, stream); }

} // namespace ff
