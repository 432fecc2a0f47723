// attn.h -- the arguments of the attention kernels and what their files call
// of each other.
#ifndef TORCHMATCH_AMD_ATTN_H
#define TORCHMATCH_AMD_ATTN_H

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace attn {

struct Args {
    const void *q, *k, *v, *dout;
    void *out, *out_low, *dq, *dk, *dv; // contiguous (B, L, heads, D); out_low may be null
    float *lse; // (B, H, Lq), natural logarithm, -inf for empty rows; backward: see attend_delta
    const float *delta;       // (B, H, Lq): sum over d of out * dout, less dlse
    const float *dlse;        // (B, H, Lq): the gradient of lse, or null
    const float *slopes;      // (H) or null
    const float *q_pos, *k_pos; // (B, L, axes), or null: distance of indices
    const int32_t *q_docs, *k_docs; // (B, L) or null
    const int4 *q_tiles, *k_tiles;  // (B, L / 64) summaries of the documents, or null
    const int32_t *q_order, *k_order; // (B, blocks of 128), which to start with first, or null
    const int32_t *prefix, *lengths;  // (B) or null
    // partial results of a split over keys
    float *part_o;  // (splits, B, H, Lq, DP)
    float2 *part_ml; // (splits, B, H, Lq): what weights are relative to (base 2), their sum
    // gradients of k and v split over the heads of a group (kv_heads each) and the queries
    // (kv_tiles tiles of 64 each): their partial sums (kv_splits, B, Lk, Hkv, D), or null
    float *part_dk, *part_dv;
    int32_t kv_splits, kv_heads, kv_tiles;
    // strides in elements
    int64_t q_b, q_l, q_h, k_b, k_l, k_h, v_b, v_l, v_h, do_b, do_l, do_h;
    int32_t B, Lq, Lk, H, Hkv, D;
    int32_t axes, causal, splits, tiles_per_split;
    float scale, cap; // cap 0: none
};

// One file per type; dp is D padded to 32, 64, 96, 128 or 256.  Non-zero: a launch failed.
#define ATTN_DECLARE(type)                                                                        \
    int forward_##type(const Args &, int dp, hipStream_t);                                        \
    int tokens_##type(const Args &, int dp, hipStream_t);                                         \
    int join_##type(const Args &, int dp, hipStream_t);                                           \
    int backward_kv_##type(const Args &, int dp, hipStream_t);                                    \
    int backward_join_##type(const Args &, hipStream_t);                                          \
    int backward_q_##type(const Args &, int dp, hipStream_t);                                     \
    int delta_##type(const Args &, const float *lse, float *base2, float *delta, hipStream_t);
ATTN_DECLARE(bf16)
ATTN_DECLARE(f16)
ATTN_DECLARE(f32)
#undef ATTN_DECLARE

} // namespace attn

#endif
