// ff.h -- the arguments of the feed-forward kernels and what their files call of each other.
#ifndef TORCHMATCH_AMD_FF_H
#define TORCHMATCH_AMD_FF_H

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace ff {

// One product, or two of one shape:  out[m][n] = sum over k of a[m][k] b[n][k].
// An operand's rows hold consecutive k, or (strided) consecutive m or n, a row for each k.
struct Args {
    const void *a[2], *b[2]; // a second one: of the next `k`s (segments), of the next product
                             // (batches), or b of the up projection (gated)
    void *out[2];            // rows of out_l, T; gated: h; hidden: not used
    int64_t a_l, b_l, out_l; // elements from row to row
    // what the gated product saves and the hidden one reads, each (m, hidden) with rows of
    // out_l: a and b, or the upper halves of their float32 bits and a third of the next
    // eight bits of each
    void *saved[3];
    void *da, *db;      // hidden: gradients of a and b, rows of out_l
    // half precision (null: no scale): kMostParts maxima of |dy|; the bits of the largest finite |da|
    // or |db| that the scale they give brings past half precision's range, or zero: written
    // (hidden, the first time) or read
    const float *most;
    uint32_t *past_out;
    const uint32_t *past;
    float *part;        // sums of the tiles that are split
    int32_t M, N, K;    // K: of one segment
    int32_t segments, batches;
    int32_t whole, splits, split_steps; // tiles that are not split; the other ones' blocks
    int32_t activation, wide; // wide: out rows are at multiples of 16 bytes
};

constexpr int kMostParts = 256;
enum Kind { kUp, kDown, kHidden, kInput, kWeights };
// Tiles: 128 x 128, with four in LDS in place of two, 64 x 64 with four, 256 x 256
enum { kSmall, kDeep, kTiny, kLarge };

// Products of more rows than this do not take product_tokens.
constexpr int kTokens = 2048;
// Its rows a block: 16 while 32 would give no more than two blocks a compute unit (64 float32 rows of
// 1024 through 2816: 22 us with 16, 28 with 32; 512 rows 116 and 106).
inline int tokens_rows(int64_t M, int64_t N) {
    return M <= 16 || (M + 31) / 32 * ((N + 15) / 16) <= 512 ? 16 : 32;
}

// Non-zero: a launch failed.
#define FF_DECLARE(type)                                                                         \
    int product_##type(const Args &, Kind, int size, hipStream_t);                               \
    int tokens_##type(const Args &, Kind, hipStream_t);
FF_DECLARE(bf16)
FF_DECLARE(f16)
FF_DECLARE(f32)
#undef FF_DECLARE

} // namespace ff

#endif
