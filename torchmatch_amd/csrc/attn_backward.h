// attn_backward.h -- attention's gradients, in two kernels that each write every output
// once, in a fixed order (no atomics, so the same call gives the same bits).
//
// Both form the weights again from the forward pass's log of the sum:
//     p = exp(s - lse),  dp = do v^T,  ds = p (dp - delta) (1 - tanh^2)
// with delta = sum over d of out do, less the gradient of lse (whose own is p).
// attend_backward_kv owns keys (32 a wave) and runs over the queries, of every head that shares
// them, or of a part of these where blocks are few (attend_join_kv adds the parts):
//     dv^T += do^T p,  dk^T += q^T ds      (weights as queries by keys)
// attend_backward_q owns queries and runs over the keys:
//     dq^T += k^T ds^T                      (weights as keys by queries)
// Eight products (dq takes two; seven for float32, whose ds is not rounded) in place of the five
// of one kernel that would have to add dq from many blocks.  p and ds are rounded to the inputs'
// type for the second products, as the forward pass rounds its weights, and held in half
// precision's range (grad_shift, Column); sums stay in float32.
#ifndef TORCHMATCH_AMD_ATTN_BACKWARD_H
#define TORCHMATCH_AMD_ATTN_BACKWARD_H

#include <algorithm>

#include "attn_tile.h"

namespace attn {

template <typename T, int DP> struct BackwardShape {
    static constexpr int kRows = sizeof(T) == 4 && DP == 256 ? 32 : 64; // rows of a tile in LDS
    static constexpr int kOccupancy = sizeof(T) * DP <= 128 ? 3 : sizeof(T) * DP <= 256 ? 2 : 1;
    // The kernel over keys takes 32 keys a wave and needs two waves a SIMD that hide each
    // other's waits.  Rows of 128 bytes and less leave the registers for that.  With rows of 256
    // bytes k and v move to LDS, and two teams of four waves share the same 128 keys, each with
    // every other tile of queries (2 x 8192 packed in documents, 128 features, with blocks as
    // they stand: 440 us; 595 with one team and k and v in registers, 700 with a pass for dk and
    // one for dv; but 125 in place of 104 for pairs of sets of 64 features).  With the longest
    // blocks first these two take 336 and 87 us: waits (for tiles, barriers and, at 128 features,
    // nine registers in scratch) bound them, with matrix products under way in a fifth and a
    // sixth of the cycles.  Larger rows leave room for one team.
    static constexpr int kTeams = Tile<T, DP>::U == 16 ? 2 : 1;
    static constexpr int kKvRows = kTeams == 2 ? 32 : kRows;
    static constexpr bool kKeysInLds = kTeams == 2;
    static constexpr int kKvOccupancy = Tile<T, DP>::U <= 8 ? 2 : 1; // blocks a compute unit
    // rows of 256: dk and dv by a pass each, the registers hold one of them
    static constexpr bool kTwoPasses = DP == 256;
};

// WHICH: 1 dv, 2 dk, 3 both
template <typename T, int DP, bool SIDE, int WHICH>
__global__ __launch_bounds__((256 * BackwardShape<T, DP>::kTeams),
                             (BackwardShape<T, DP>::kKvOccupancy)) void
attend_backward_kv(const Args p) {
    using S = BackwardShape<T, DP>;
    using L = Tile<T, DP>;
    constexpr int QT = S::kKvRows, QB = QT / 32, C = DP / 16, DB = DP / 32, TEAMS = S::kTeams;
    constexpr bool DV = WHICH & 1, DK = WHICH & 2;
    using B = Bring<T, DP, QT, 256>;
    __shared__ u32x4 sq0[TEAMS][QT * L::U], sq1[TEAMS][QT * L::U];
    __shared__ u32x4 so0[TEAMS][QT * L::U], so1[TEAMS][QT * L::U];
    // of the tile's queries: where exponents start, delta, positions; documents
    __shared__ __attribute__((aligned(16))) float s_row0[TEAMS][5][64], s_row1[TEAMS][5][64];
    __shared__ __attribute__((aligned(16))) int s_docs0[TEAMS][64], s_docs1[TEAMS][64];
    // k and v, and at the end the second team's results, 32 x DP floats a wave
    constexpr int SUM = TEAMS == 2 ? 32 * DP : 1, KEEP = S::kKeysInLds ? 128 * L::U : 0;
    __shared__ u32x4 keep[2 * KEEP > SUM ? 2 * KEEP : SUM];

    const int all_waves = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int team = all_waves >> 2, wave = all_waves & 3;
    const int tid = threadIdx.x & 255, lane = tid & 63, half = lane >> 5;
    const int k_blocks = (p.Lk + 127) / 128;
    const int group = p.H / p.Hkv;
    const Share share(blockIdx.x, k_blocks, p.B * p.Hkv * p.kv_splits);
    const int split = share.head % p.kv_splits;
    const int kvh = share.head / p.kv_splits % p.Hkv, b = share.head / p.kv_splits / p.Hkv;
    const int kb = SIDE && p.k_order ? scalar(p.k_order[(int64_t)b * k_blocks + share.block])
                                     : share.block; // the first are seen by most
    const int k0 = 128 * kb, kw = k0 + 32 * wave, kj = kw + (lane & 31);
    const Limits lim(p, b);
    const uint32_t row_at = L::row_lane(lane), col_at = L::col_lane(lane);
    const int my_doc = SIDE && p.k_docs && kj < p.Lk ? p.k_docs[(int64_t)b * p.Lk + kj] : -1;
    const bool k_real = kj < lim.length && !(SIDE && p.k_docs && my_doc < 0);
    // the first query that sees this lane's key; the last that must be asked for
    const int my_first = !k_real ? 0x7fffffff
                         : lim.causal && kj >= lim.prefix ? max(0, kj - lim.offset)
                                                          : 0;

    const T *k = (const T *)p.k + b * p.k_b + kvh * p.k_h + (k_real ? kj : 0) * p.k_l;
    const T *v = (const T *)p.v + b * p.v_b + kvh * p.v_h + (k_real ? kj : 0) * p.v_l;
    x8<T> kf[S::kKeysInLds ? 1 : C], vf[S::kKeysInLds ? 1 : C];
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const x8<T> x = global8<T>(k, 16 * c + 8 * half, p.D, k_real);
        const x8<T> y = global8<T>(v, 16 * c + 8 * half, p.D, k_real);
        if constexpr (S::kKeysInLds) { // the same by either team
            L::put8(keep, row_at, 32 * wave, c, x);
            L::put8(keep + KEEP, row_at, 32 * wave, c, y);
        } else {
            kf[c] = x;
            vf[c] = y;
        }
    }
    float my_pos[3] = {0.f, 0.f, 0.f};
    if (SIDE && p.k_pos && kj < p.Lk)
#pragma unroll
        for (int a = 0; a < 3; ++a)
            if (a < p.axes)
                my_pos[a] = p.k_pos[((int64_t)b * p.Lk + kj) * p.axes + a];

    // the first query that sees the block's first key
    int first = 0;
    if (k0 >= lim.length)
        first = p.Lq;
    else if (lim.causal && k0 >= lim.prefix)
        first = min(p.Lq, max(0, k0 - lim.offset));
    const int nq = (p.Lq + 63) / 64, nk = (p.Lk + 63) / 64;
    // this split's heads of the group, and tiles of queries
    const int head_splits = (group + p.kv_heads - 1) / p.kv_heads;
    const int g_begin = split % head_splits * p.kv_heads;
    const int g_end = min(group, g_begin + p.kv_heads);
    const int t_begin = max(first / 64, split / head_splits * p.kv_tiles);
    const int t_end = first < p.Lq ? min(nq, (split / head_splits + 1) * p.kv_tiles) : 0;
    const int4 *q_tiles = SIDE && p.q_tiles ? p.q_tiles + (int64_t)b * nq : nullptr;
    const int32_t *q_docs = SIDE && p.q_docs ? p.q_docs + (int64_t)b * p.Lq : nullptr;
    const float *q_pos = SIDE && p.q_pos ? p.q_pos + (int64_t)b * p.Lq * p.axes : nullptr;
    int4 mine = {0, 0, 0, 0}, wave_docs = {0, 0, 0, 0};
    if (SIDE && p.k_tiles) {
        const int4 *t = p.k_tiles + (int64_t)b * nk;
        mine = t[k0 / 64];
        for (int n = k0 / 64 + 1; n < min(nk, (k0 + 128) / 64); ++n) {
            mine.x = min(mine.x, t[n].x);
            mine.y = max(mine.y, t[n].y);
        }
        wave_docs = kw < p.Lk ? t[kw / 64] : (int4){0x7fffffff, -1, 0, 0};
    }

    f32x16 dk[DB], dv[DB];
#pragma unroll
    for (int i = 0; i < DB; ++i) {
        dk[i] = f32x16{};
        dv[i] = f32x16{};
    }
    Column<T> column;

    // the tiles of one query head after the other's, dealt to the teams in turn: this team's is
    // at (g, t64, sub), the last given out at (all_g, all_t, all_sub)
    int all_g = g_begin, all_t, all_sub = 0, g, t64, sub;
    int4 qd_next = {0, 0, 0, 0}; // documents of this team's tile
    bool first_team_more = false;
    TileWalk walk;
    auto advance = [&]() {
        all_t = walk.next(lane);
        while (all_t >= t_end && all_g + 1 < g_end) {
            ++all_g;
            walk.start(q_tiles, mine, t_begin, t_end, lane);
            all_t = walk.next(lane);
        }
    };
    auto deal = [&]() {
#pragma unroll
        for (int n = 0; n < TEAMS; ++n) {
            if (n == 0)
                first_team_more = all_t < t_end;
            if (n == team) {
                g = all_g;
                t64 = all_t;
                sub = all_sub;
                qd_next = walk.docs;
            }
            if (all_t < t_end && (++all_sub == 64 / QT || all_t * 64 + all_sub * QT >= p.Lq)) {
                all_sub = 0;
                advance();
            }
        }
    };
    auto fetch = [&](u32x4 *sq, u32x4 *so, float (*s_row)[64], int *s_docs) {
        const int q0 = t64 * 64 + sub * QT, head = kvh * group + g;
        B::load(sq, (const T *)p.q + b * p.q_b + head * p.q_h, p.q_l, q0, p.Lq, p.D, tid);
        B::load(so, (const T *)p.dout + b * p.do_b + head * p.do_h, p.do_l, q0, p.Lq, p.D, tid);
        const int i = min(q0 + lane, p.Lq - 1);
        const int64_t row = ((int64_t)b * p.H + head) * p.Lq + i;
        if (wave == 0) {
            bring_word(s_row[0], p.lse + row);
            if (DK)
                bring_word(s_row[1], p.delta + row);
        } else if (SIDE && wave == 1) {
            if (q_docs)
                bring_word(s_docs, q_docs + i);
            if (q_pos) {
#pragma unroll
                for (int a = 0; a < 3; ++a)
                    if (a < p.axes)
                        bring_word(s_row[2 + a], q_pos + (int64_t)i * p.axes + a);
            }
        }
    };
    auto step = [&](u32x4 *sq, u32x4 *so, float (*s_row)[64], int *s_docs, u32x4 *next_q,
                    u32x4 *next_o, float (*next_row)[64], int *next_docs) {
        const int q0 = t64 * 64 + sub * QT, head = kvh * group + g;
        const int4 qd = qd_next;
        const bool here = t64 < t_end; // the last tile may be the other team's
        arrived();
        __syncthreads(); // this tile is here, and the other buffer is done with
        deal();
        if (t64 < t_end)
            fetch(next_q, next_o, next_row, next_docs);
        if (!here)
            return;

        const int last = min(q0 + QT, p.Lq) - 1;
        bool use = kw < lim.of(last), dirty = q0 + QT > p.Lq;
        bool masked = kw + 32 > lim.of(q0) || q0 + QT > p.Lq;
        if (q_docs) {
            use = use && docs_meet(qd, wave_docs);
            masked = masked || !docs_same(qd, wave_docs);
            dirty = dirty || qd.z;
        }
        if (dirty && use) {
            // Each wave clears all of the rows itself (with the others, the same zeros), so that
            // none has to wait: the teams are not at the same tile.
            for (int n = lane; n < QT * L::U; n += 64) {
                const int r = n / L::U;
                if (q0 + r >= p.Lq || (q_docs && s_docs[r] < 0))
                    sq[n] = so[n] = u32x4{0u, 0u, 0u, 0u};
            }
            wave_fence();
        }
        if (!use)
            return;
        const float slope = p.slopes ? p.slopes[head] * kLog2e : 0.f;

#pragma unroll 1
        for (int qb = 0; qb < QB; ++qb) {
            f32x16 s = {}, ds = {};
#pragma unroll
            for (int c = 0; c < C; ++c) {
                x8<T> kc, vc;
                if constexpr (S::kKeysInLds) {
                    kc = L::row8(keep, row_at, 32 * wave, c);
                    vc = L::row8(keep + KEEP, row_at, 32 * wave, c);
                } else {
                    kc = kf[c];
                    vc = vf[c];
                }
                s = mma32(L::row8(sq, row_at, 32 * qb, c), kc, s);
                if constexpr (DK)
                    ds = mma32(L::row8(so, row_at, 32 * qb, c), vc, ds);
            }
            const float from = (float)(kj - q0 - 32 * qb - 4 * half - lim.offset);
            weigh<T, DK>(
                p, s, ds, slope,
                [&](int n) -> f32x4 {
                    const int j = 32 * qb + 8 * n + 4 * half;
                    f32x4 d;
                    if (SIDE && q_pos) {
                        d = away(*(const f32x4 *)(s_row[2] + j), my_pos[0]);
                        if (p.axes > 1)
                            d += away(*(const f32x4 *)(s_row[3] + j), my_pos[1]);
                        if (p.axes > 2)
                            d += away(*(const f32x4 *)(s_row[4] + j), my_pos[2]);
                    } else {
                        d = away(f32x4{8.f * n, 8.f * n + 1.f, 8.f * n + 2.f, 8.f * n + 3.f},
                                 from);
                    }
                    return d;
                },
                [&](int n) { return *(const f32x4 *)(s_row[0] + 32 * qb + 8 * n + 4 * half); },
                [&](int n) { return *(const f32x4 *)(s_row[1] + 32 * qb + 8 * n + 4 * half); });
            if (masked) {
                const int row0 = q0 + 32 * qb + 4 * half;
                const int from = my_first - row0, to = p.Lq - row0;
#pragma unroll
                for (int n = 0; n < 4; ++n) {
                    i32x4 doc = {my_doc, my_doc, my_doc, my_doc};
                    if (SIDE && q_docs)
                        doc = *(const i32x4 *)(s_docs + 32 * qb + 8 * n + 4 * half);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const bool see =
                            (8 * n + e >= from) & (8 * n + e < to) & (doc[e] == my_doc);
                        s[4 * n + e] = see ? s[4 * n + e] : 0.f;
                        ds[4 * n + e] = see ? ds[4 * n + e] : 0.f;
                    }
                }
            }
            if constexpr (DK)
                column.fit(ds, dk);
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                if constexpr (DV) {
                    const x8<T> w = pack8<T>(s, t);
#pragma unroll
                    for (int i = 0; i < DB; ++i)
                        dv[i] = mma32(L::col8(so, col_at, 32 * qb + 16 * t, i), w, dv[i]);
                }
                if constexpr (DK) {
                    const x8<T> w = column.pack(ds, t);
#pragma unroll
                    for (int i = 0; i < DB; ++i)
                        dk[i] = mma32(L::col8(sq, col_at, 32 * qb + 16 * t, i), w, dk[i]);
                }
            }
        }
    };

    B::pad(sq0[team], p.D, tid);
    B::pad(sq1[team], p.D, tid);
    B::pad(so0[team], p.D, tid);
    B::pad(so1[team], p.D, tid);
    if (p.D < DP)
        __syncthreads();
    walk.start(q_tiles, mine, t_begin, t_end, lane);
    advance();
    deal();
    if (t64 < t_end)
        fetch(sq0[team], so0[team], s_row0[team], s_docs0[team]);
    // the first team has a tile wherever the second one has
    while (first_team_more) {
        step(sq0[team], so0[team], s_row0[team], s_docs0[team], sq1[team], so1[team],
             s_row1[team], s_docs1[team]);
        if (!first_team_more)
            break;
        step(sq1[team], so1[team], s_row1[team], s_docs1[team], sq0[team], so0[team],
             s_row0[team], s_docs0[team]);
    }

    if constexpr (DK)
        column.undo(dk);
    if constexpr (DV && grad_shift<T>() != 0) {
#pragma unroll
        for (int i = 0; i < DB; ++i)
            dv[i] *= 1.f / (1 << grad_shift<T>());
    }
    if constexpr (TEAMS == 2) { // the second team's results to the first, dk and then dv
        const auto join = [&](f32x16 (&x)[DB]) {
            f32x4 *at = (f32x4 *)keep + wave * (8 * DP) + lane;
            __syncthreads();
            if (team == 1) {
#pragma unroll
                for (int i = 0; i < DB; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        at[64 * (4 * i + e)] = (f32x4){x[i][4 * e], x[i][4 * e + 1],
                                                       x[i][4 * e + 2], x[i][4 * e + 3]};
            }
            __syncthreads();
            if (team == 0) {
#pragma unroll
                for (int i = 0; i < DB; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const f32x4 y = at[64 * (4 * i + e)];
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            x[i][4 * e + j] += y[j];
                    }
            }
        };
        if constexpr (DK)
            join(dk);
        if constexpr (DV)
            join(dv);
        if (team == 1)
            return;
    }
    if (kj >= p.Lk)
        return;
    const float out_scale = grad_scale(p);
    const int64_t at = (((int64_t)b * p.Lk + kj) * p.Hkv + kvh) * p.D;
    if (p.kv_splits > 1) {
        const int64_t part = (int64_t)split * p.B * p.Lk * p.Hkv * p.D + at;
#pragma unroll
        for (int i = 0; i < DB; ++i)
#pragma unroll
            for (int e = 0; e < 16; e += 4) {
                const int d = 32 * i + 2 * e + 4 * half;
                if (d < p.D) {
                    if constexpr (DK)
                        *(f32x4 *)(p.part_dk + part + d) =
                            f32x4{dk[i][e], dk[i][e + 1], dk[i][e + 2], dk[i][e + 3]} * out_scale;
                    if constexpr (DV)
                        *(f32x4 *)(p.part_dv + part + d) =
                            f32x4{dv[i][e], dv[i][e + 1], dv[i][e + 2], dv[i][e + 3]};
                }
            }
        return;
    }
#pragma unroll
    for (int i = 0; i < DB; ++i)
#pragma unroll
        for (int e = 0; e < 16; e += 4) {
            const int d = 32 * i + 2 * e + 4 * half;
            if (d < p.D) {
                x4<T> y, z;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    y[j] = (T)(dk[i][e + j] * out_scale);
                    z[j] = (T)dv[i][e + j];
                }
                if constexpr (DK)
                    *(x4<T> *)((T *)p.dk + at + d) = y;
                if constexpr (DV)
                    *(x4<T> *)((T *)p.dv + at + d) = z;
            }
        }
}

template <typename T, int DP, bool SIDE>
__global__ __launch_bounds__(256, (BackwardShape<T, DP>::kOccupancy)) void
attend_backward_q(const Args p) {
    using L = Tile<T, DP>;
    constexpr int KT = BackwardShape<T, DP>::kRows, KB = KT / 32, C = DP / 16, DB = DP / 32;
    using B = Bring<T, DP, KT, 256>;
    __shared__ u32x4 sk0[KT * L::U], sk1[KT * L::U];
    __shared__ u32x4 sv0[KT * L::U], sv1[KT * L::U];
    __shared__ __attribute__((aligned(16))) int s_docs0[64], s_docs1[64];
    __shared__ __attribute__((aligned(16))) float s_pos0[3][64], s_pos1[3][64];

    const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int q_blocks = (p.Lq + 127) / 128;
    const Share share(blockIdx.x, q_blocks, p.B * p.H);
    const int head = share.head % p.H, b = share.head / p.H;
    const int qb = SIDE && p.q_order ? scalar(p.q_order[(int64_t)b * q_blocks + share.block])
                                     : q_blocks - 1 - share.block; // the last see most
    const int kvh = head / (p.H / p.Hkv);

    const int q0 = qb * 128, qw = q0 + 32 * wave, qi = qw + (lane & 31);
    const Limits lim(p, b);
    const uint32_t row_at = L::row_lane(lane), col_at = L::col_lane(lane);
    const int block_limit = lim.of(min(q0 + 128, p.Lq) - 1);
    const int wave_limit = qw < p.Lq ? lim.of(min(qw + 32, p.Lq) - 1) : 0;
    const int full_limit = qw < p.Lq ? lim.of(qw) : 0;
    const QueryLane<T, SIDE> rows(p, lim, b, head, qi);
    const bool q_real = qi < p.Lq && !(SIDE && p.q_docs && rows.doc < 0);

    const T *q = (const T *)p.q + b * p.q_b + head * p.q_h + (q_real ? qi : 0) * p.q_l;
    const T *dout = (const T *)p.dout + b * p.do_b + head * p.do_h + (q_real ? qi : 0) * p.do_l;
    const T *k = (const T *)p.k + b * p.k_b + kvh * p.k_h;
    const T *v = (const T *)p.v + b * p.v_b + kvh * p.v_h;
    const int32_t *k_docs = SIDE && p.k_docs ? p.k_docs + (int64_t)b * p.Lk : nullptr;
    const float *k_pos = SIDE && p.k_pos ? p.k_pos + (int64_t)b * p.Lk * p.axes : nullptr;

    x8<T> qf[C], of[C];
#pragma unroll
    for (int c = 0; c < C; ++c) {
        qf[c] = global8<T>(q, 16 * c + 8 * half, p.D, q_real);
        of[c] = global8<T>(dout, 16 * c + 8 * half, p.D, q_real);
    }
    const int64_t row = ((int64_t)b * p.H + head) * p.Lq + qi;
    const float base = qi < p.Lq ? p.lse[row] : -kInf;
    const float delta = qi < p.Lq ? p.delta[row] : 0.f;

    constexpr int per64 = 64 / KT;
    int4 wave_docs = {0, 0, 0, 0};
    const int64_t nk = (p.Lk + 63) / 64, nq = (p.Lq + 63) / 64;
    const int t_end = (block_limit + 63) / 64;
    TileWalk walk;
    {
        int4 mine = {0, 0, 0, 0};
        if (SIDE && p.q_tiles) {
            const int4 *t = p.q_tiles + b * nq;
            mine = t[q0 / 64];
            if (q0 / 64 + 1 < nq) {
                const int4 o = t[q0 / 64 + 1];
                mine.x = min(mine.x, o.x);
                mine.y = max(mine.y, o.y);
            }
            wave_docs = qw < p.Lq ? t[qw / 64] : (int4){0x7fffffff, -1, 0, 0};
        }
        walk.start(SIDE && p.k_tiles ? p.k_tiles + b * nk : nullptr, mine, 0, t_end, lane);
    }

    f32x16 dq[DB];
#pragma unroll
    for (int i = 0; i < DB; ++i)
        dq[i] = f32x16{};
    Column<T> column;

    const int seen = min(block_limit, p.Lk); // keys past it may hold anything
    int t64 = walk.next(lane), sub = 0;
    auto fetch = [&](int k0, u32x4 *sk, u32x4 *sv, int *s_docs, float (*s_pos)[64]) {
        B::load(sk, k, p.k_l, k0, seen, p.D, tid);
        B::load(sv, v, p.v_l, k0, seen, p.D, tid);
        if (SIDE && wave == 0) {
            const int64_t j = min(k0 + lane, seen - 1);
            if (k_docs)
                bring_word(s_docs, k_docs + j);
            if (k_pos) {
#pragma unroll
                for (int a = 0; a < 3; ++a)
                    if (a < p.axes)
                        bring_word(s_pos[a], k_pos + j * p.axes + a);
            }
        }
    };
    auto step = [&](u32x4 *sk, u32x4 *sv, int *s_docs, float (*s_pos)[64], u32x4 *next_k,
                    u32x4 *next_v, int *next_docs, float (*next_pos)[64]) {
        const int k0 = t64 * 64 + sub * KT;
        const int4 kd = walk.docs;
        arrived();
        __syncthreads(); // this tile is here, and the other buffer is done with
        if (++sub == per64 || k0 + KT >= seen) { // no row of the second half may be there
            sub = 0;
            t64 = walk.next(lane);
        }
        if (t64 < t_end)
            fetch(t64 * 64 + sub * KT, next_k, next_v, next_docs, next_pos);

        bool use = k0 < wave_limit, masked = k0 + KT > full_limit, dirty = k0 + KT > seen;
        if (k_docs) {
            use = use && docs_meet(kd, wave_docs);
            masked = masked || !docs_same(kd, wave_docs);
            dirty = dirty || kd.z;
        }
        if (dirty) { // the same for all waves
            B::clear(sk, k0, seen, k_docs, s_docs, tid);
            __syncthreads();
        }
        if (!use)
            return;

#pragma unroll 1
        for (int kb = 0; kb < KB; ++kb) {
            f32x16 s = {}, ds = {};
#pragma unroll
            for (int c = 0; c < C; ++c) {
                s = mma32(L::row8(sk, row_at, 32 * kb, c), qf[c], s);
                ds = mma32(L::row8(sv, row_at, 32 * kb, c), of[c], ds);
            }
            weigh<T, true>(
                p, s, ds, rows.slope,
                [&](int n) {
                    return rows.distance(p, n, k0 + 32 * kb, half, &s_pos[0][32 * kb], 64);
                },
                [&](int) { return f32x4{base, base, base, base}; },
                [&](int) { return f32x4{delta, delta, delta, delta}; });
            if (masked)
                rows.hide(p, ds, 0.f, k0 + 32 * kb, half, s_docs + 32 * kb);
            column.fit(ds, dq);
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const x8<T> w = column.pack(ds, t);
                x8<T> rest = w;
                if constexpr (sizeof(T) == 2)
                    rest = column.rest(ds, t, w);
#pragma unroll
                for (int i = 0; i < DB; ++i) {
                    const x8<T> kt = L::col8(sk, col_at, 32 * kb + 16 * t, i);
                    dq[i] = mma32(kt, w, dq[i]);
                    if constexpr (sizeof(T) == 2)
                        dq[i] = mma32(kt, rest, dq[i]);
                }
            }
        }
    };

    B::pad(sk0, p.D, tid);
    B::pad(sk1, p.D, tid);
    B::pad(sv0, p.D, tid);
    B::pad(sv1, p.D, tid);
    if (p.D < DP)
        __syncthreads();
    if (t64 < t_end)
        fetch(t64 * 64, sk0, sv0, s_docs0, s_pos0);
    while (t64 < t_end) {
        step(sk0, sv0, s_docs0, s_pos0, sk1, sv1, s_docs1, s_pos1);
        if (t64 >= t_end)
            break;
        step(sk1, sv1, s_docs1, s_pos1, sk0, sv0, s_docs0, s_pos0);
    }

    column.undo(dq);
    if (qi >= p.Lq)
        return;
    const float out_scale = grad_scale(p);
    T *dst = (T *)p.dq + (((int64_t)b * p.Lq + qi) * p.H + head) * p.D;
#pragma unroll
    for (int i = 0; i < DB; ++i)
#pragma unroll
        for (int e = 0; e < 16; e += 4) {
            const int d = 32 * i + 2 * e + 4 * half;
            if (d < p.D) {
                x4<T> y;
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    y[j] = (T)(dq[i][e + j] * out_scale);
                *(x4<T> *)(dst + d) = y;
            }
        }
}

// delta of each query and head, and what the exponents of its weights start from: minus the log
// of its sum in base 2, plus the cap's share (Cap) and grad_shift(); -inf for an empty row,
// which makes all its weights zero.  16 bytes a thread, DP / E threads a row.  From the output as
// it was before it was rounded, in two parts: the rounding alone would add as much error to dq
// and dk as that of ds does.
template <typename T, int N> // N threads a row: a power of two, N * E >= D
__global__ __launch_bounds__(256) void attend_delta(const Args p, const float *lse,
                                                    float *base2, float *delta) {
    constexpr int E = 16 / (int)sizeof(T);
    typedef T unit __attribute__((ext_vector_type(E)));
    const int d = (int)threadIdx.x % N * E;
    const int64_t rows = (int64_t)p.B * p.Lq * p.H;
    for (int64_t first = (int64_t)blockIdx.x * (256 / N); first < rows;
         first += (int64_t)gridDim.x * (256 / N)) {
        const int64_t row = first + threadIdx.x / N;
        const int head = (int)(row % p.H), i = (int)(row / p.H % p.Lq);
        const int64_t b = row / p.H / p.Lq;
        float x = 0.f;
        if (row < rows && d < p.D) {
            const unit u = *(const unit *)((const T *)p.out + row * p.D + d);
            const unit w = *(const unit *)((const T *)p.dout + b * p.do_b + i * p.do_l +
                                           head * p.do_h + d);
            unit r = u;
            if (p.out_low)
                r = *(const unit *)((const T *)p.out_low + row * p.D + d);
#pragma unroll
            for (int j = 0; j < E; ++j)
                x = fmaf((float)u[j] + (p.out_low ? (float)r[j] : 0.f), (float)w[j], x);
        }
#pragma unroll
        for (int n = N / 2; n; n >>= 1)
            x += __shfl_xor(x, n);
        if (row < rows && d == 0) {
            const int64_t at = (b * p.H + head) * p.Lq + i;
            const float l = lse[at];
            // an empty row has no gradient, whatever a loss makes of its -inf
            delta[at] = l == -kInf ? 0.f : p.dlse ? x - p.dlse[at] : x;
            base2[at] = l == -kInf ? -kInf : Cap<T>::share(p) - l * kLog2e + grad_shift<T>();
        }
    }
}

template <typename T>
int run_delta(const Args &a, const float *lse, float *base2, float *delta, hipStream_t s) {
    const int64_t rows = (int64_t)a.B * a.Lq * a.H;
    const int units = a.D * (int)sizeof(T) / 16;
    const auto grid = [&](int n) {
        return dim3((unsigned)std::min<int64_t>((rows * n + 255) / 256, 1 << 20));
    };
    if (units <= 8)
        attend_delta<T, 8><<<grid(8), 256, 0, s>>>(a, lse, base2, delta);
    else if (units <= 16)
        attend_delta<T, 16><<<grid(16), 256, 0, s>>>(a, lse, base2, delta);
    else
        attend_delta<T, 64><<<grid(64), 256, 0, s>>>(a, lse, base2, delta);
    return hipGetLastError() == hipSuccess ? 0 : 1;
}

// Sums the splits' partial gradients, in their order: 4 elements of dk and dv a thread.
// Bound by memory: 11 us for 4 parts of 3 x 515 keys of 8 heads of 128 float32 features.
template <typename T> __global__ __launch_bounds__(256) void attend_join_kv(const Args p) {
    const int64_t n = (int64_t)p.B * p.Lk * p.Hkv * p.D;
    for (int64_t i = 4 * ((int64_t)blockIdx.x * 256 + threadIdx.x); i < n;
         i += (int64_t)gridDim.x * 1024) {
        f32x4 dk = *(const f32x4 *)(p.part_dk + i), dv = *(const f32x4 *)(p.part_dv + i);
        for (int s = 1; s < p.kv_splits; ++s) {
            dk += *(const f32x4 *)(p.part_dk + s * n + i);
            dv += *(const f32x4 *)(p.part_dv + s * n + i);
        }
        *(x4<T> *)((T *)p.dk + i) = __builtin_convertvector(dk, x4<T>);
        *(x4<T> *)((T *)p.dv + i) = __builtin_convertvector(dv, x4<T>);
    }
}

template <typename T> int run_backward_join(const Args &a, hipStream_t s) {
    const int64_t blocks = ((int64_t)a.B * a.Lk * a.Hkv * a.D + 1023) / 1024;
    attend_join_kv<T><<<dim3((unsigned)std::min<int64_t>(blocks, 4096)), 256, 0, s>>>(a);
    return hipGetLastError() == hipSuccess ? 0 : 1;
}

template <typename T, int DP, bool SIDE> void start_backward_kv(const Args &a, hipStream_t s) {
    constexpr int N = 256 * BackwardShape<T, DP>::kTeams;
    const dim3 grid((unsigned)((int64_t)((a.Lk + 127) / 128) * a.Hkv * a.B *
                               a.kv_splits));
    if constexpr (BackwardShape<T, DP>::kTwoPasses) {
        attend_backward_kv<T, DP, SIDE, 1><<<grid, N, 0, s>>>(a);
        attend_backward_kv<T, DP, SIDE, 2><<<grid, N, 0, s>>>(a);
    } else {
        attend_backward_kv<T, DP, SIDE, 3><<<grid, N, 0, s>>>(a);
    }
}

template <typename T, int DP> int run_backward_kv(const Args &a, hipStream_t s) {
    if (a.q_docs || a.q_pos)
        start_backward_kv<T, DP, true>(a, s);
    else
        start_backward_kv<T, DP, false>(a, s);
    return hipGetLastError() == hipSuccess ? 0 : 1;
}

template <typename T, int DP> int run_backward_q(const Args &a, hipStream_t s) {
    const dim3 grid((unsigned)((int64_t)((a.Lq + 127) / 128) * a.H * a.B));
    if (a.q_docs || a.q_pos)
        attend_backward_q<T, DP, true><<<grid, 256, 0, s>>>(a);
    else
        attend_backward_q<T, DP, false><<<grid, 256, 0, s>>>(a);
    return hipGetLastError() == hipSuccess ? 0 : 1;
}

} // namespace attn

#endif
