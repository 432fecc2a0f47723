// attn_tokens.h -- attention forward for a few queries over many keys (new tokens over a
// cache): bound by reading k and v once.
//
// The queries of all heads that share a key head are packed into rows of 32, so that one
// pass over the keys serves them all.  A block's waves take tiles of 64 keys in turn, each
// for itself: a wave brings 32 keys at a time into its own part of LDS, with the next 32 on
// their way into registers meanwhile (16 KB a wave in flight at 128 features), and no
// barrier holds it up.  At the end the waves' results are joined through LDS, and those of
// a split over blocks by attend_join.  The matrix cores are idle most of the time: 32 rows
// cost them a tenth of what reading the keys takes, so rows left empty do not matter.
#ifndef TORCHMATCH_AMD_ATTN_TOKENS_H
#define TORCHMATCH_AMD_ATTN_TOKENS_H

#include "attn_tile.h"

namespace attn {

template <typename T, int DP> struct TokensShape {
    static constexpr int kTile = 32 * Tile<T, DP>::U; // units of 32 keys in LDS
    // as many waves as LDS holds tiles for, up to 8
    static constexpr int kWaves =
        kTile * 2 * 16 * 8 <= 131072 ? 8 : kTile * 2 * 16 * 4 <= 131072 ? 4 : 2;
    // float32 rows of 256 leave no registers for the next tile
    static constexpr bool kAhead = sizeof(T) * DP <= 512;
};

template <typename T, int DP>
__global__ __launch_bounds__((64 * TokensShape<T, DP>::kWaves), 1) void
attend_tokens(const Args p) {
    using L = Tile<T, DP>;
    using S = TokensShape<T, DP>;
    constexpr int NW = S::kWaves, C = DP / 16, DB = DP / 32;
    __shared__ u32x4 tiles[NW][2][S::kTile];
    __shared__ __attribute__((aligned(16))) int s_docs[NW][32];
    __shared__ __attribute__((aligned(16))) float s_pos[NW][3][32];
    __shared__ float s_top[NW][32], s_sum[NW][32];

    const int lane = threadIdx.x & 63, half = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int group = p.H / p.Hkv, packed = group * p.Lq;
    const int row_blocks = (packed + 31) / 32;
    // the row blocks of the same keys together
    int id = xcd_order(blockIdx.x, gridDim.x);
    const int rb = id % row_blocks;
    id /= row_blocks;
    const int split = id % p.splits;
    id /= p.splits;
    const int kvh = id % p.Hkv, b = id / p.Hkv;

    const int r = 32 * rb + (lane & 31);
    const bool q_real = r < packed;
    const int qi = q_real ? r % p.Lq : p.Lq;
    const int head = kvh * group + (q_real ? r / p.Lq : 0);
    const Limits lim(p, b);
    const uint32_t row_at = L::row_lane(lane), col_at = L::col_lane(lane);
    const int all_limit = lim.of(p.Lq - 1), full_limit = lim.of(0);
    const QueryLane<T, true> rows(p, lim, b, head, qi);

    const T *q = (const T *)p.q + b * p.q_b + head * p.q_h;
    const T *k = (const T *)p.k + b * p.k_b + kvh * p.k_h;
    const T *v = (const T *)p.v + b * p.v_b + kvh * p.v_h;
    const int32_t *k_docs = p.k_docs ? p.k_docs + (int64_t)b * p.Lk : nullptr;
    const float *k_pos = p.k_pos ? p.k_pos + (int64_t)b * p.Lk * p.axes : nullptr;
    x8<T> qf[C];
#pragma unroll
    for (int c = 0; c < C; ++c)
        qf[c] = global8<T>(q + (int64_t)(q_real ? qi : 0) * p.q_l, 16 * c + 8 * half, p.D, q_real);

    const int t_end = min((all_limit + 63) / 64, (split + 1) * p.tiles_per_split);
    const int4 *k_tiles = p.k_tiles ? p.k_tiles + (int64_t)b * ((p.Lk + 63) / 64) : nullptr;
    const int4 mine = p.q_tiles ? p.q_tiles[(int64_t)b] : (int4){0, 0, 0, 0}; // Lq <= 64
    TileWalk walk;
    // with documents the waves deal out the tiles that meet them, else all of them
    walk.start(k_tiles, mine, split * p.tiles_per_split + (k_tiles ? 0 : wave), t_end, lane);
    auto advance = [&](bool first) {
        if (!k_tiles) {
            const int t = min(walk.base, t_end);
            walk.base += NW;
            return t;
        }
        int t = t_end;
        for (int n = first ? wave + 1 : NW; n; --n)
            t = walk.next(lane);
        return t;
    };

    f32x16 o[DB];
#pragma unroll
    for (int i = 0; i < DB; ++i)
        o[i] = f32x16{};
    float top = -kInf, sum = 0.f;
    const float factor = rows.factor(p);

    u32x4 *sk = tiles[wave][0], *sv = tiles[wave][1];
    Stage<T, DP, 32, 64> gk, gv;
    int g_doc = -1;
    float g_pos[3];
    const int seen = min(all_limit, p.Lk); // keys past it may hold anything
    auto fetch = [&](int k0) {
        if constexpr (S::kAhead) {
            gk.load(k, p.k_l, k0, seen, p.D, k_docs, lane);
            gv.load(v, p.v_l, k0, seen, p.D, k_docs, lane);
        }
        const bool real = lane < 32 && k0 + lane < seen;
        if (k_docs)
            g_doc = real ? k_docs[k0 + lane] : -1;
        if (k_pos) {
#pragma unroll
            for (int a = 0; a < 3; ++a)
                if (a < p.axes)
                    g_pos[a] = real ? k_pos[(int64_t)(k0 + lane) * p.axes + a] : 0.f;
        }
    };

    int t64 = advance(true), sub = 0;
    if (t64 < t_end)
        fetch(t64 * 64);
    while (t64 < t_end) {
        const int k0 = t64 * 64 + 32 * sub;
        wave_fence();
        if constexpr (!S::kAhead)
            gk.load(k, p.k_l, k0, seen, p.D, k_docs, lane);
        gk.store(sk, lane);
        if constexpr (!S::kAhead)
            gv.load(v, p.v_l, k0, seen, p.D, k_docs, lane);
        gv.store(sv, lane);
        if (lane < 32) {
            if (k_docs)
                s_docs[wave][lane] = g_doc;
            if (k_pos) {
#pragma unroll
                for (int a = 0; a < 3; ++a)
                    if (a < p.axes)
                        s_pos[wave][a][lane] = g_pos[a];
            }
        }
        wave_fence();
        bool masked = k0 + 32 > full_limit;
        if (k_tiles)
            masked = masked || !docs_same(walk.docs, mine);
        sub ^= 1;
        if (!sub || k0 + 32 >= seen) {
            sub = 0;
            t64 = advance(false);
        }
        if (t64 < t_end)
            fetch(t64 * 64 + 32 * sub);

        f32x16 s[1] = {f32x16{}};
#pragma unroll
        for (int c = 0; c < C; ++c)
            s[0] = mma32(L::row8(sk, row_at, 0, c), qf[c], s[0]);
        rows.score(p, s[0], k0, half, &s_pos[wave][0][0], 32);
        if (masked)
            rows.hide(p, s[0], -kInf, k0, half, s_docs[wave]);
        soften<T>(s, o, factor, top, sum);
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const x8<T> w = pack8<T>(s[0], t);
#pragma unroll
            for (int i = 0; i < DB; ++i)
                o[i] = mma32(L::col8(sv, col_at, 16 * t, i), w, o[i]);
        }
    }

    // join the waves: each leaves its output in its own part of LDS (a row's units of 4
    // floats permuted, so that the lanes' rows do not meet in one bank)
    sum += __shfl_xor(sum, 32);
    wave_fence();
    f32x4 *mine_o = (f32x4 *)tiles[wave];
    constexpr int U = DP / 4;
    static_assert(32 * U <= 2 * S::kTile, "a wave's output fits in its tiles");
#pragma unroll
    for (int i = 0; i < DB; ++i)
#pragma unroll
        for (int e = 0; e < 16; e += 4)
            mine_o[(lane & 31) * U + ((8 * i + e / 2 + half) ^ (lane & 7))] =
                (f32x4){o[i][e], o[i][e + 1], o[i][e + 2], o[i][e + 3]};
    if (!half) {
        s_top[wave][lane] = top;
        s_sum[wave][lane] = sum;
    }
    __syncthreads();
    for (int n = threadIdx.x; n < 32 * U; n += 64 * NW) {
        const int row = n / U, u = n % U;
        const int rr = 32 * rb + row;
        if (rr >= packed)
            break;
        float all = -kInf, total = 0.f;
#pragma unroll
        for (int w = 0; w < NW; ++w)
            all = fmaxf(all, s_top[w][row]);
        const float from = all == -kInf ? 0.f : all;
        f32x4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            const float f = __builtin_amdgcn_exp2f(s_top[w][row] - from);
            total = fmaf(s_sum[w][row], f, total);
            const f32x4 y = ((const f32x4 *)tiles[w])[row * U + (u ^ (row & 7))];
#pragma unroll
            for (int j = 0; j < 4; ++j)
                x[j] = fmaf(y[j], f, x[j]);
        }
        const int i = rr % p.Lq, h = kvh * group + rr / p.Lq;
        const int64_t at_row = ((int64_t)b * p.H + h) * p.Lq + i;
        if (p.splits > 1) {
            const int64_t at = (int64_t)split * p.B * p.H * p.Lq + at_row;
            *(f32x4 *)(p.part_o + at * DP + 4 * u) = x;
            if (u == 0)
                p.part_ml[at] = make_float2(all, total);
        } else {
            x *= total == 0.f ? 0.f : 1.f / total;
            if (4 * u < p.D)
                put<T>(p, (((int64_t)b * p.Lq + i) * p.H + h) * p.D + 4 * u,
                       __builtin_convertvector(x, x4<T>), x);
            if (u == 0 && p.lse)
                p.lse[at_row] =
                    total == 0.f ? -kInf : kLn2 * (all + __builtin_amdgcn_logf(total));
        }
    }
}

template <typename T, int DP> int run_tokens(const Args &a, hipStream_t s) {
    const int64_t blocks =
        (int64_t)((a.H / a.Hkv * a.Lq + 31) / 32) * a.splits * a.Hkv * a.B;
    attend_tokens<T, DP><<<dim3((unsigned)blocks), 64 * TokensShape<T, DP>::kWaves, 0, s>>>(a);
    return hipGetLastError() == hipSuccess ? 0 : 1;
}

} // namespace attn

#endif
