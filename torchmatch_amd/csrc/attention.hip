// attention.hip -- the C entries of the attention operators: checks, workspace, launches.
#include <algorithm>
#include <cmath>

#include "../../include/torchmatch_amd.h"
#include "attn_tile.h"

namespace {

using attn::Args;

// Summaries of the documents of 64 rows each: the smallest and the largest id that is not
// negative (INT_MAX, -1 without one), and whether one is negative.  A wave for each.
__global__ __launch_bounds__(256) void attend_docs(const int32_t *q_docs, const int32_t *k_docs,
                                                   int B, int Lq, int Lk, int4 *q_tiles,
                                                   int4 *k_tiles) {
    const int64_t nq = (Lq + 63) / 64, nk = (Lk + 63) / 64;
    int64_t t = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int lane = threadIdx.x & 63;
    if (t >= B * (nq + nk))
        return;
    const bool keys = t >= B * nq;
    if (keys)
        t -= B * nq;
    const int64_t n = keys ? nk : nq, len = keys ? Lk : Lq;
    const int64_t b = t / n, i = t % n * 64 + lane;
    const int id = i < len ? (keys ? k_docs : q_docs)[b * len + i] : -1;
    int lo = id < 0 ? 0x7fffffff : id, hi = id < 0 ? -1 : id;
    const bool hidden = __any(i < len && id < 0);
#pragma unroll
    for (int x = 32; x; x >>= 1) {
        lo = min(lo, __shfl_xor(lo, x));
        hi = max(hi, __shfl_xor(hi, x));
    }
    if (!lane)
        (keys ? k_tiles : q_tiles)[t] = make_int4(lo, hi, hidden, 0);
}

// With documents, how long a block of 128 queries or keys takes has nothing to do with where it
// stands.  Puts those that visit most tiles first, for each batch row: a workgroup brings the
// summaries of both sides into LDS, counts for each of its row's blocks the tiles that meet it
// and ranks the blocks, a wave a block (blockIdx.y + first_side 0: queries, 1: keys).
constexpr int kMaxOrdered = 2048;
__global__ __launch_bounds__(1024) void attend_order(const Args p, int first_side,
                                                     int32_t *q_order, int32_t *k_order) {
    __shared__ int2 own[2 * kMaxOrdered], others[2 * kMaxOrdered];
    __shared__ int cost[kMaxOrdered];
    const int b = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const bool keys = blockIdx.y + first_side;
    const int nq = (p.Lq + 63) / 64, nk = (p.Lk + 63) / 64;
    const int n_own = keys ? nk : nq, n_others = keys ? nq : nk, blocks = (n_own + 1) / 2;
    const int4 *from_own = (keys ? p.k_tiles : p.q_tiles) + (int64_t)b * n_own;
    const int4 *from_others = (keys ? p.q_tiles : p.k_tiles) + (int64_t)b * n_others;
    const attn::Limits lim(p, b);
    for (int t = threadIdx.x; t < n_own; t += 1024)
        own[t] = make_int2(from_own[t].x, from_own[t].y);
    for (int t = threadIdx.x; t < n_others; t += 1024)
        others[t] = make_int2(from_others[t].x, from_others[t].y);
    __syncthreads();
    for (int i = wave; i < blocks; i += 16) {
        const int2 m = own[2 * i], o = own[min(2 * i + 1, n_own - 1)];
        const int lo = min(m.x, o.x), hi = max(m.y, o.y);
        int first = 0, end;
        if (keys) {
            end = 128 * i < lim.length ? nq : 0;
            if (lim.causal && 128 * i >= lim.prefix)
                first = min(nq, max(0, 128 * i - lim.offset) / 64);
        } else {
            end = (lim.of(min(128 * i + 128, p.Lq) - 1) + 63) / 64;
        }
        int n = 0;
        for (int t = first; t < end; t += 64) {
            const int2 x = others[min(t + lane, end - 1)];
            n += __popcll(__ballot(t + lane < end && x.x <= hi && lo <= x.y));
        }
        if (!lane)
            cost[i] = n;
    }
    __syncthreads();
    int32_t *order = (keys ? k_order : q_order) + (int64_t)b * blocks;
    for (int i = wave; i < blocks; i += 16) {
        const int c = cost[i];
        int rank = 0;
        for (int t = 0; t < blocks; t += 64) {
            const int j = t + lane, x = cost[min(j, blocks - 1)];
            const bool before = x > c || (x == c && (keys ? j < i : j > i));
            rank += __popcll(__ballot(j < blocks && before));
        }
        if (!lane)
            order[rank] = i;
    }
}

int padded(int d) { return d <= 32 ? 32 : d <= 64 ? 64 : d <= 96 ? 96 : d <= 128 ? 128 : 256; }

size_t align256(size_t n) { return (n + 255) & ~(size_t)255; }

size_t docs_bytes(const tm_attention *a) {
    if (!a->q_docs)
        return 0;
    const size_t tiles = (size_t)a->B * ((a->Lq + 63) / 64 + (a->Lk + 63) / 64);
    const size_t blocks = (size_t)a->B * ((a->Lq + 127) / 128 + (a->Lk + 127) / 128);
    return align256(tiles * sizeof(int4)) + align256(blocks * sizeof(int32_t));
}

// Worth a launch where the blocks of `rows` rows and `heads` heads are more than run at once.
bool ordered(const tm_attention *a, int64_t rows, int64_t heads, int at_once) {
    return std::max(a->Lq, a->Lk) <= 128 * kMaxOrdered &&
           (rows + 127) / 128 * heads * a->B > at_once;
}

// One block has no order.  Two or more in a batch row also keep the launch, B workgroups of
// 1024 threads, below 2^32 of them: B is then below TM_ATTENTION_MAX_BLOCKS / 2.
bool several(int64_t rows) { return rows > 128; }

// Few queries: the kernel that packs the queries of a key head's group into 32 rows.
// Above 32 queries the other kernel's 128 rows a block are no longer mostly empty.
bool few(const tm_attention *a) { return a->Lq <= 32; }

// Keys are split over blocks when there are too few rows to fill the chip.  Few queries are
// bound by reading the keys, by one block of 8 waves a compute unit: two such blocks for each
// of the 256 in turn where rows are equally long, four where their lengths differ, so that
// the short ones leave no unit idle, and at least 32 keys a wave.  Else a block needs at least
// four tiles, so that its start and the join are worth it.
struct Splits {
    int n, tiles;
};
Splits splits_of(const tm_attention *a) {
    const int tiles = std::max((a->Lk + 63) / 64, 1);
    int64_t blocks, want, most;
    if (a->B == 0 || a->Lq == 0)
        return {1, tiles};
    if (few(a)) {
        blocks = (int64_t)((a->H / a->Hkv * a->Lq + 31) / 32) * a->Hkv * a->B;
        want = std::max<int64_t>(1, (a->lengths ? 1024 : 512) / blocks);
        most = tiles / 4;
    } else {
        blocks = (int64_t)((a->Lq + 127) / 128) * a->H * a->B;
        want = blocks >= 256 ? 1 : (512 + blocks - 1) / blocks;
        most = tiles / 4;
    }
    const int n = (int)std::max<int64_t>(1, std::min(want, most));
    const int per = (tiles + n - 1) / n;
    return {(tiles + per - 1) / per, per};
}

// The kernel over keys has a block for 128 keys of a key head that takes the group's query heads
// in turn: few blocks, and long ones, where one key head serves many.  Up to a block a compute
// unit, the group's heads and then the queries are split over up to 512 blocks of at least two
// tiles of 64 queries each, whose float32 sums a second kernel adds in their order.  The whole
// backward pass, whole against split, us: 16384 causal, H 8, Hkv 1, D 128, bf16 (128 blocks)
// 5562, 2272; 4096 causal, H 4, Hkv 1, D 64 (32) 590, 169; 3 x 515 causal, H 32, Hkv 8, D 128,
// f32 (120) 836, 479; 333, H 4, D 64, f32 (12) 109, 80; 4 x 2048 causal, H 16, Hkv 4, D 128, bf16
// (256) 453, 358; 4096, H 6, D 128, bf16 (192) 329, 351.  256 blocks and 1024 were as fast or
// slower.
struct KvSplits {
    int n, heads, tiles;
};
KvSplits kv_splits_of(const tm_attention *a) {
    const int group = a->H / a->Hkv, tiles = (a->Lq + 63) / 64;
    const int64_t blocks = (int64_t)((a->Lk + 127) / 128) * a->Hkv * a->B;
    const int64_t want =
        blocks > 256 || !blocks ? 1
                                : std::min<int64_t>(512 / blocks, (int64_t)group * tiles / 2);
    if (want <= 1)
        return {1, group, tiles};
    const int heads = (int)((group + std::min<int64_t>(group, want) - 1) /
                            std::min<int64_t>(group, want));
    const int over_heads = (group + heads - 1) / heads;
    const int over_tiles = (int)std::max<int64_t>(
        1, std::min<int64_t>(want / over_heads, tiles / 2));
    const int per = (tiles + over_tiles - 1) / over_tiles;
    return {over_heads * ((tiles + per - 1) / per), heads, per};
}
size_t kv_part_bytes(const tm_attention *a) { // of dk, or dv
    const KvSplits s = kv_splits_of(a);
    return s.n > 1 ? align256((size_t)s.n * a->B * a->Lk * a->Hkv * a->D * sizeof(float)) : 0;
}

// What every call must hold; sizes of zero are the callers' to answer.
int check(const tm_attention *a) {
    if (!a || a->B < 0 || a->Lq < 0 || a->Lk < 0 || a->H < 1 || a->Hkv < 1 || a->H % a->Hkv ||
        a->D < 1)
        return TM_ERR_INVALID_ARGUMENT;
    if (a->dtype < TM_BF16 || a->dtype > TM_F32)
        return TM_ERR_INVALID_ARGUMENT;
    const int unit = a->dtype == TM_F32 ? 4 : 8;
    if (a->D > tm_attention_max_head_dim() || a->D % unit)
        return TM_ERR_UNSUPPORTED_SHAPE;
    // blocks of up to 512 threads, of which a launch takes less than 2^32 (attend_order, of 1024,
    // is launched where this admits half as many batch rows: see several())
    if (a->Lq > INT32_MAX - 256 || a->Lk > INT32_MAX - 256 ||
        a->B * std::max((int64_t)a->H * ((a->Lq + 31) / 32),
                        (int64_t)a->Hkv * ((a->Lk + 127) / 128)) >= TM_ATTENTION_MAX_BLOCKS)
        return TM_ERR_UNSUPPORTED_SHAPE;
    if (a->dtype != TM_F32 && a->cap > TM_ATTENTION_MAX_CAP_16)
        return TM_ERR_UNSUPPORTED_SHAPE;
    // what the kernels make of these, up to 4 times as much, stays finite
    const float most = 0x1p126f;
    if (!(std::fabs(a->scale) <= most) || !(a->cap >= 0.f) || !(a->cap <= most) ||
        (a->cap > 0.f && !(std::fabs(a->scale / a->cap) <= most)))
        return TM_ERR_INVALID_ARGUMENT;
    if ((!a->q_docs != !a->k_docs) ||
        (!a->q_positions != !a->k_positions) || (a->q_positions && !a->slopes))
        return TM_ERR_INVALID_ARGUMENT;
    if (a->q_positions && (a->axes < 1 || a->axes > 3))
        return TM_ERR_UNSUPPORTED_SHAPE;
    const int64_t strides[] = {a->q_b, a->q_l, a->q_h, a->k_b, a->k_l, a->k_h,
                               a->v_b, a->v_l, a->v_h};
    for (int64_t s : strides)
        if (s % unit)
            return TM_ERR_INVALID_ARGUMENT;
    // a tile's rows are reached by 32 bits from its first
    const int64_t size = a->dtype == TM_F32 ? 4 : 2;
    if (a->q_l < 0 || a->k_l < 0 || a->v_l < 0 ||
        std::max({a->q_l, a->k_l, a->v_l}) * size >= TM_ATTENTION_MAX_ROW_BYTES)
        return TM_ERR_UNSUPPORTED_SHAPE;
    if (((uintptr_t)a->q | (uintptr_t)a->k | (uintptr_t)a->v) % 16)
        return TM_ERR_INVALID_ARGUMENT;
    return TM_OK;
}

Args args_of(const tm_attention *a) {
    Args p = {};
    p.q = a->q;
    p.k = a->k;
    p.v = a->v;
    p.slopes = a->slopes;
    p.q_pos = a->q_positions;
    p.k_pos = a->k_positions;
    p.q_docs = a->q_docs;
    p.k_docs = a->k_docs;
    p.prefix = a->causal ? a->prefix : nullptr;
    p.lengths = a->lengths;
    p.q_b = a->q_b, p.q_l = a->q_l, p.q_h = a->q_h;
    p.k_b = a->k_b, p.k_l = a->k_l, p.k_h = a->k_h;
    p.v_b = a->v_b, p.v_l = a->v_l, p.v_h = a->v_h;
    p.B = a->B, p.Lq = a->Lq, p.Lk = a->Lk, p.H = a->H, p.Hkv = a->Hkv, p.D = a->D;
    p.axes = a->axes, p.causal = a->causal ? 1 : 0;
    p.scale = a->scale, p.cap = a->cap;
    p.splits = 1;
    return p;
}

#define ATTN_BY_TYPE(call, ...)                                                                   \
    (a->dtype == TM_BF16  ? attn::call##_bf16(__VA_ARGS__)                                        \
     : a->dtype == TM_F16 ? attn::call##_f16(__VA_ARGS__)                                         \
                          : attn::call##_f32(__VA_ARGS__))

int summarise_docs(const tm_attention *a, Args &p, char *ws, bool q_order, bool k_order,
                   hipStream_t stream) {
    if (!a->q_docs)
        return 0;
    const int64_t nq = (a->Lq + 63) / 64, nk = (a->Lk + 63) / 64;
    int4 *q_tiles = (int4 *)ws, *k_tiles = q_tiles + a->B * nq;
    p.q_tiles = q_tiles;
    p.k_tiles = k_tiles;
    attend_docs<<<dim3((unsigned)((a->B * (nq + nk) + 3) / 4)), 256, 0, stream>>>(
        a->q_docs, a->k_docs, a->B, a->Lq, a->Lk, q_tiles, k_tiles);
    if (q_order || k_order) {
        int32_t *order = (int32_t *)(ws + align256(a->B * (nq + nk) * sizeof(int4)));
        int32_t *of_keys = order + (int64_t)a->B * ((a->Lq + 127) / 128);
        attend_order<<<dim3(a->B, q_order + k_order), 1024, 0, stream>>>(p, !q_order, order,
                                                                         of_keys);
        if (q_order)
            p.q_order = order;
        if (k_order)
            p.k_order = of_keys;
    }
    return hipGetLastError() == hipSuccess ? 0 : 1;
}

} // namespace

extern "C" int32_t tm_attention_max_head_dim(void) { return 256; }

extern "C" size_t tm_attention_workspace_bytes(const tm_attention *a) {
    if (check(a) != TM_OK)
        return 0;
    size_t n = docs_bytes(a);
    const Splits s = splits_of(a);
    if (s.n > 1) {
        const size_t rows = (size_t)s.n * a->B * a->H * a->Lq;
        n += align256(rows * padded(a->D) * sizeof(float)) + align256(rows * sizeof(float2));
    }
    return n;
}

extern "C" int tm_attention_forward(const tm_attention *a, void *out, void *out_low,
                                    float *lse, void *workspace, size_t workspace_bytes,
                                    hipStream_t stream) {
    const int rc = check(a);
    if (rc != TM_OK)
        return rc;
    if (a->B == 0 || a->Lq == 0)
        return TM_OK;
    if (!a->q || !out || (a->Lk && (!a->k || !a->v)))
        return TM_ERR_INVALID_ARGUMENT;
    const size_t need = tm_attention_workspace_bytes(a);
    if (workspace_bytes < need || (need && !workspace))
        return TM_ERR_WORKSPACE;
    Args p = args_of(a);
    p.out = out;
    p.out_low = a->dtype == TM_F32 ? nullptr : out_low;
    p.lse = lse;
    char *ws = (char *)workspace;
    if (summarise_docs(a, p, ws, several(a->Lq) && ordered(a, a->Lq, a->H, 512), false, stream))
        return TM_ERR_LAUNCH;
    ws += docs_bytes(a);
    const Splits s = splits_of(a);
    const int dp = padded(a->D);
    p.splits = s.n;
    p.tiles_per_split = s.tiles;
    if (s.n > 1) {
        const size_t rows = (size_t)s.n * a->B * a->H * a->Lq;
        p.part_o = (float *)ws;
        p.part_ml = (float2 *)(ws + align256(rows * dp * sizeof(float)));
    }
    if (few(a) ? ATTN_BY_TYPE(tokens, p, dp, stream) : ATTN_BY_TYPE(forward, p, dp, stream))
        return TM_ERR_LAUNCH;
    if (s.n > 1 && ATTN_BY_TYPE(join, p, dp, stream))
        return TM_ERR_LAUNCH;
    return TM_OK;
}

extern "C" size_t tm_attention_backward_workspace_bytes(const tm_attention *a) {
    if (check(a) != TM_OK)
        return 0;
    return docs_bytes(a) + 2 * align256((size_t)a->B * a->H * a->Lq * sizeof(float)) +
           2 * kv_part_bytes(a);
}

extern "C" int tm_attention_backward(const tm_attention *a, const void *out,
                                     const void *out_low, const float *lse, const void *dout,
                                     int64_t do_b, int64_t do_l, int64_t do_h, void *dq,
                                     void *dk, void *dv, void *workspace,
                                     size_t workspace_bytes, hipStream_t stream) {
    return tm_attention_backward_lse(a, out, out_low, lse, nullptr, dout, do_b, do_l, do_h, dq,
                                     dk, dv, workspace, workspace_bytes, stream);
}

extern "C" int tm_attention_backward_lse(const tm_attention *a, const void *out,
                                         const void *out_low, const float *lse,
                                         const float *dlse, const void *dout, int64_t do_b,
                                         int64_t do_l, int64_t do_h, void *dq, void *dk,
                                         void *dv, void *workspace, size_t workspace_bytes,
                                         hipStream_t stream) {
    const int rc = check(a);
    if (rc != TM_OK)
        return rc;
    if (a->B == 0 || (a->Lq == 0 && a->Lk == 0))
        return TM_OK;
    const int unit = a->dtype == TM_F32 ? 4 : 8;
    if ((a->Lq && (!a->q || !out || !lse || !dout || !dq)) ||
        (a->Lk && (!a->k || !a->v || !dk || !dv)) || (uintptr_t)dout % 16 || do_b % unit ||
        do_l % unit || do_h % unit)
        return TM_ERR_INVALID_ARGUMENT;
    if (do_l < 0 || do_l * (a->dtype == TM_F32 ? 4 : 2) >= TM_ATTENTION_MAX_ROW_BYTES)
        return TM_ERR_UNSUPPORTED_SHAPE;
    const size_t need = tm_attention_backward_workspace_bytes(a);
    if (workspace_bytes < need || (need && !workspace))
        return TM_ERR_WORKSPACE;
    Args p = args_of(a);
    p.out = const_cast<void *>(out);
    p.out_low = a->dtype == TM_F32 ? nullptr : const_cast<void *>(out_low);
    p.dout = dout;
    p.dlse = dlse;
    p.do_b = do_b, p.do_l = do_l, p.do_h = do_h;
    p.dq = dq, p.dk = dk, p.dv = dv;
    char *ws = (char *)workspace;
    const bool many = a->Lq && ordered(a, a->Lq, a->H, 512), q_order = many && several(a->Lq);
    const bool k_order = many && several(a->Lk) && ordered(a, a->Lk, a->Hkv, 256);
    if (summarise_docs(a, p, ws, q_order, k_order, stream))
        return TM_ERR_LAUNCH;
    float *delta = (float *)(ws + docs_bytes(a));
    float *base2 = (float *)((char *)delta +
                             align256((size_t)a->B * a->H * a->Lq * sizeof(float)));
    p.delta = delta;
    p.lse = base2;
    const KvSplits kv = kv_splits_of(a);
    p.kv_splits = kv.n, p.kv_heads = kv.heads, p.kv_tiles = kv.tiles;
    p.part_dk = (float *)((char *)base2 +
                          align256((size_t)a->B * a->H * a->Lq * sizeof(float)));
    p.part_dv = (float *)((char *)p.part_dk + kv_part_bytes(a));
    const int dp = padded(a->D);
    if (a->Lq && ATTN_BY_TYPE(delta, p, lse, base2, delta, stream))
        return TM_ERR_LAUNCH;
    if (a->Lk && ATTN_BY_TYPE(backward_kv, p, dp, stream))
        return TM_ERR_LAUNCH;
    if (a->Lk && kv.n > 1 && ATTN_BY_TYPE(backward_join, p, stream))
        return TM_ERR_LAUNCH;
    if (a->Lq && ATTN_BY_TYPE(backward_q, p, dp, stream))
        return TM_ERR_LAUNCH;
    return TM_OK;
}
