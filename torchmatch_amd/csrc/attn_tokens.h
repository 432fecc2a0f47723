// attn_tokens.h -- attention forward for a few queries over many keys (new tokens over a
// cache): bound by reading k and v once.
//
// The queries of all heads that share a key head are packed into rows of 32, so that one
// pass over the keys serves them all.  A block's waves take 32 keys at a time in turn, each for
// itself: a wave brings them straight into its own part of LDS, the next keys as soon as
// the scores are formed and the next values as soon as these are added, waits for no other
// wave, and with eight of them a compute unit has 128 KB on their way (128 features of 16
// bits).  At the end the waves' results are joined through LDS, and those of a split over
// blocks by attend_join.  The matrix cores are idle most of the time with 16-bit types: 32 rows
// cost them a tenth of what reading the keys takes, so rows left empty do not matter.  float32
// products take 16 times the cycles for twice the bytes, over half of the time of reading, and
// still go on beside it (16 tokens, 16384 keys, 128 features: 455 us, 4.7 TB/s).
#ifndef TORCHMATCH_AMD_ATTN_TOKENS_H
#define TORCHMATCH_AMD_ATTN_TOKENS_H

#include "attn_tile.h"

namespace attn {

template <typename T, int DP> struct TokensShape {
    static constexpr int kTile = 32 * Tile<T, DP>::U; // units of 32 keys in LDS
    // as many waves as LDS holds tiles for, up to 8
    static constexpr int kWaves =
        kTile * 2 * 16 * 8 <= 131072 ? 8 : kTile * 2 * 16 * 4 <= 131072 ? 4 : 2;
};

template <typename T, int DP, bool SIDE>
__global__ __launch_bounds__((64 * TokensShape<T, DP>::kWaves), 1) void
attend_tokens(const Args p) {
    using L = Tile<T, DP>;
    using S = TokensShape<T, DP>;
    constexpr int NW = S::kWaves, C = DP / 16, DB = DP / 32;
    using B = Bring<T, DP, 32, 64>;
    __shared__ u32x4 all_k[NW * S::kTile], all_v[NW * S::kTile];
    // by parity of the wave's tiles
    __shared__ __attribute__((aligned(16))) int all_docs[SIDE ? 2 * NW : 1][64];
    __shared__ __attribute__((aligned(16))) float all_pos[SIDE ? 2 * NW : 1][3][64];
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
    const QueryLane<T, SIDE> rows(p, lim, b, head, qi);

    const T *q = (const T *)p.q + b * p.q_b + head * p.q_h;
    const T *k = (const T *)p.k + b * p.k_b + kvh * p.k_h;
    const T *v = (const T *)p.v + b * p.v_b + kvh * p.v_h;
    const int32_t *k_docs = SIDE && p.k_docs ? p.k_docs + (int64_t)b * p.Lk : nullptr;
    const float *k_pos = SIDE && p.k_pos ? p.k_pos + (int64_t)b * p.Lk * p.axes : nullptr;
    x8<T> qf[C];
#pragma unroll
    for (int c = 0; c < C; ++c)
        qf[c] = global8<T>(q + (int64_t)(q_real ? qi : 0) * p.q_l, 16 * c + 8 * half, p.D, q_real);

    // the waves' turns: tiles of 32 keys, with documents those of 64 that meet them
    const int seen = min(all_limit, p.Lk); // keys past it may hold anything
    const int t_end = min((all_limit + 63) / 64, (split + 1) * p.tiles_per_split);
    const int end = min(64 * t_end, seen);
    const int4 *k_tiles =
        SIDE && p.k_tiles ? p.k_tiles + (int64_t)b * ((p.Lk + 63) / 64) : nullptr;
    const int4 mine = k_tiles ? p.q_tiles[b] : (int4){0, 0, 0, 0}; // Lq <= 64: one each row
    TileWalk walk;
    if (k_tiles)
        walk.start(k_tiles, mine, split * p.tiles_per_split, t_end, lane);
    int k0 = 64 * split * p.tiles_per_split + 32 * wave; // this wave's tile, `end` or more: none
    int4 kd = {0, 0, 0, 0};
    auto turn = [&](int turns) {
        int t = t_end;
        for (int n = 0; n < turns; ++n)
            t = walk.next(lane);
        kd = walk.docs;
        k0 = t < t_end ? 64 * t : 0x7fffffff;
    };
    if (k_tiles)
        turn(wave + 1);
    auto advance = [&]() {
        if (!k_tiles)
            k0 = min(k0, end) + 32 * NW;
        else if (!(k0 & 32) && k0 + 32 < end)
            k0 += 32;
        else
            turn(NW);
    };

    f32x16 o[DB];
#pragma unroll
    for (int i = 0; i < DB; ++i)
        o[i] = f32x16{};
    float top = -kInf, sum = 0.f;
    const float factor = rows.factor(p);

    u32x4 *sk = all_k + wave * S::kTile, *sv = all_v + wave * S::kTile;
    if (p.D < DP) {
        B::pad(sk, p.D, lane);
        B::pad(sv, p.D, lane);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }
    int parity = 0;
    auto fetch_k = [&](int at) {
        if (SIDE) {
            const int64_t j = min(at + lane, seen - 1);
            if (k_docs)
                bring_word(all_docs[parity * NW + wave], k_docs + j);
            if (k_pos) {
#pragma unroll
                for (int a = 0; a < 3; ++a)
                    if (a < p.axes)
                        bring_word(all_pos[parity * NW + wave][a], k_pos + j * p.axes + a);
            }
        }
        B::load(sk, k, p.k_l, at, seen, p.D, lane);
    };
    auto fetch_v = [&](int at) { B::load(sv, v, p.v_l, at, seen, p.D, lane); };
    if (k0 < end) {
        fetch_k(k0);
        fetch_v(k0);
    }
    while (k0 < end) {
        const int now = k0;
        bool masked = now + 32 > full_limit, dirty = now + 32 > seen;
        if (k_tiles) {
            masked = masked || !docs_same(kd, mine);
            dirty = dirty || kd.z;
        }
        const int *s_docs = all_docs[SIDE ? parity * NW + wave : 0];
        const float(*s_pos)[64] = all_pos[SIDE ? parity * NW + wave : 0];
        advance();
        parity ^= 1;

        arrived<B::N>(); // the keys; the values were sent for after them
        f32x16 s[1] = {f32x16{}};
#pragma unroll
        for (int c = 0; c < C; ++c)
            s[0] = mma32(L::row8(sk, row_at, 0, c), qf[c], s[0]);
        made_here(s[0]); // the keys have been read
        if (k0 < end)
            fetch_k(k0);
        rows.score(p, s[0], now, half, &s_pos[0][0], 64);
        if (masked)
            rows.hide(p, s[0], -kInf, now, half, s_docs);
        soften<T>(s, o, factor, top, sum);
        if (k0 < end)
            arrived<B::N>(); // the values; the next keys were sent for after them
        else
            arrived<0>();
        if (dirty) {
            B::clear(sv, now, seen, k_docs, s_docs, lane);
            wave_fence();
        }
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const x8<T> w = pack8<T>(s[0], t);
#pragma unroll
            for (int i = 0; i < DB; ++i)
                o[i] = mma32(L::col8(sv, col_at, 16 * t, i), w, o[i]);
        }
#pragma unroll
        for (int i = 0; i < DB; ++i)
            made_here(o[i]); // the values have been read
        if (k0 < end)
            fetch_v(k0);
    }

    // join the waves: each leaves its output in its own part of LDS (a row's units of 4
    // floats permuted, so that the lanes' rows do not meet in one bank)
    sum += __shfl_xor(sum, 32);
    wave_fence();
    constexpr int U = DP / 4, H = 32 * U / 2; // half of the rows in the place of the keys
    static_assert(H <= S::kTile, "a wave's output fits in its tiles");
    f32x4 *mine_o = (f32x4 *)((lane & 16 ? all_v : all_k) + wave * S::kTile);
#pragma unroll
    for (int i = 0; i < DB; ++i)
#pragma unroll
        for (int e = 0; e < 16; e += 4)
            mine_o[(lane & 15) * U + ((8 * i + e / 2 + half) ^ (lane & 7))] =
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
            const f32x4 y = ((const f32x4 *)((row & 16 ? all_v : all_k) +
                                             w * S::kTile))[(row & 15) * U + (u ^ (row & 7))];
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
    constexpr int N = 64 * TokensShape<T, DP>::kWaves;
    if (a.q_docs || a.q_pos)
        attend_tokens<T, DP, true><<<dim3((unsigned)blocks), N, 0, s>>>(a);
    else
        attend_tokens<T, DP, false><<<dim3((unsigned)blocks), N, 0, s>>>(a);
    return hipGetLastError() == hipSuccess ? 0 : 1;
}

} // namespace attn

#endif
