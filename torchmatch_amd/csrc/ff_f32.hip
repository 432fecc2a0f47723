// ff_f32.hip -- the feed-forward products of one type.
#include "ff_tile.h"

namespace ff {

int product_f32(const Args &p, Kind kind, bool big, hipStream_t stream) {
    return run<float>(p, kind, big, stream);
}
int join_f32(const Args &p, hipStream_t stream) { return run_join<float>(p, stream); }

} // namespace ff
