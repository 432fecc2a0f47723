// attn_backward.h -- attention's gradients, in two kernels that each write every output
// once, in a fixed order (no atomics, so the same call gives the same bits).
//
// Both form the weights again from the forward pass's log of the sum:
//     p = exp(s - lse),  dp = do v^T,  ds = p (dp - delta) (1 - tanh^2)
// with delta = sum over d of out do.  attend_backward_kv owns keys (32 a wave) and runs over the
// queries, of every head that shares them:
//     dv^T += do^T p,  dk^T += q^T ds      (weights as queries by keys)
// attend_backward_q owns queries and runs over the keys:
//     dq^T += k^T ds^T                      (weights as keys by queries)
// Seven products in place of the five of one kernel that would have to add dq from many
// blocks.  p and ds are rounded to the inputs' type for the second products, as the forward
// pass rounds its weights; sums stay in float32.
#ifndef TORCHMATCH_AMD_ATTN_BACKWARD_H
#define TORCHMATCH_AMD_ATTN_BACKWARD_H

#include "attn_tile.h"

namespace attn {

template <typename T, int DP> struct BackwardShape {
    static constexpr int kRows = sizeof(T) == 4 && DP == 256 ? 32 : 64; // rows of a tile in LDS
    // float32 rows of 256: dk and dv by a pass each, the registers hold one of them
    static constexpr bool kTwoPasses = sizeof(T) == 4 && DP == 256;
};

// WHICH: 1 dv, 2 dk, 3 both
template <typename T, int DP, int WHICH>
__global__ __launch_bounds__(256, 1) void attend_backward_kv(const Args p) {
    using L = Tile<T, DP>;
    constexpr int QT = BackwardShape<T, DP>::kRows, QB = QT / 32, C = DP / 16, DB = DP / 32;
    constexpr bool DV = WHICH & 1, DK = WHICH & 2;
    __shared__ u32x4 sq[QT * L::U];
    __shared__ u32x4 sdo[QT * L::U];
    __shared__ __attribute__((aligned(16))) float s_lse[QT], s_delta[QT], s_pos[3][QT];
    __shared__ __attribute__((aligned(16))) int s_limit[QT], s_doc[QT];

    const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int k_blocks = (p.Lk + 127) / 128;
    const int group = p.H / p.Hkv;
    int id = xcd_order(blockIdx.x, gridDim.x);
    const int kb = id % k_blocks; // early keys, which most causal rows see, first
    id /= k_blocks;
    const int kvh = id % p.Hkv, b = id / p.Hkv;
    const int k0 = 128 * kb, kw = k0 + 32 * wave, kj = kw + (lane & 31);
    const Limits lim(p, b);
    const int my_doc = p.k_docs && kj < p.Lk ? p.k_docs[(int64_t)b * p.Lk + kj] : -1;
    const bool k_real = kj < lim.length && !(p.k_docs && my_doc < 0);

    const T *k = (const T *)p.k + b * p.k_b + kvh * p.k_h + (k_real ? kj : 0) * p.k_l;
    const T *v = (const T *)p.v + b * p.v_b + kvh * p.v_h + (k_real ? kj : 0) * p.v_l;
    x8<T> kf[C], vf[C];
#pragma unroll
    for (int c = 0; c < C; ++c) {
        kf[c] = global8<T>(k, 16 * c + 8 * half, p.D, k_real);
        if constexpr (DK)
            vf[c] = global8<T>(v, 16 * c + 8 * half, p.D, k_real);
    }
    float my_pos[3] = {0.f, 0.f, 0.f};
    if (p.k_pos && kj < p.Lk)
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
    const int t_end = first < p.Lq ? nq : 0;
    const int4 *q_tiles = p.q_tiles ? p.q_tiles + (int64_t)b * nq : nullptr;
    int4 mine = {0, 0, 0, 0}, wave_docs = {0, 0, 0, 0};
    if (p.k_tiles) {
        const int4 *t = p.k_tiles + (int64_t)b * nk;
        mine = t[k0 / 64];
        if (k0 / 64 + 1 < nk) {
            const int4 o = t[k0 / 64 + 1];
            mine.x = min(mine.x, o.x);
            mine.y = max(mine.y, o.y);
        }
        wave_docs = kw < p.Lk ? t[kw / 64] : (int4){0x7fffffff, -1, 0, 0};
    }

    f32x16 dk[DB], dv[DB];
#pragma unroll
    for (int i = 0; i < DB; ++i) {
        dk[i] = f32x16{};
        dv[i] = f32x16{};
    }

    for (int g = 0; g < group; ++g) {
        const int head = kvh * group + g;
        const T *q = (const T *)p.q + b * p.q_b + head * p.q_h;
        const T *dout = (const T *)p.dout + b * p.do_b + head * p.do_h;
        const int64_t row = ((int64_t)b * p.H + head) * p.Lq;
        const int32_t *q_docs = p.q_docs ? p.q_docs + (int64_t)b * p.Lq : nullptr;
        const float slope = p.slopes ? p.slopes[head] * kLog2e : 0.f;

        Stage<T, DP, QT, 256> gq, gdo;
        float g_lse = 0.f, g_delta = 0.f, g_pos[3];
        int g_doc = -1;
        auto fetch = [&](int q0) {
            gq.load(q, p.q_l, q0, p.Lq, p.D, q_docs, tid);
            gdo.load(dout, p.do_l, q0, p.Lq, p.D, q_docs, tid);
            if (tid < QT) {
                const int i = q0 + tid;
                const bool real = i < p.Lq;
                g_lse = real ? p.lse[row + i] * kLog2e : -kInf;
                g_delta = real ? p.delta[row + i] : 0.f;
                g_doc = q_docs && real ? q_docs[i] : -1;
                if (p.q_pos)
#pragma unroll
                    for (int a = 0; a < 3; ++a)
                        if (a < p.axes)
                            g_pos[a] = real ? p.q_pos[((int64_t)b * p.Lq + i) * p.axes + a] : 0.f;
            }
        };

        TileWalk walk;
        walk.start(q_tiles, mine, first / 64, t_end, lane);
        constexpr int per64 = 64 / QT;
        int t64 = walk.next(lane), sub = 0;
        if (t64 < t_end)
            fetch(t64 * 64);
        while (t64 < t_end) {
            const int q0 = t64 * 64 + sub * QT;
            __syncthreads();
            gq.store(sq, tid);
            gdo.store(sdo, tid);
            if (tid < QT) {
                // an empty row: every weight 2^-inf
                s_lse[tid] = g_lse == -kInf ? kInf : g_lse;
                s_delta[tid] = g_delta;
                s_limit[tid] = q0 + tid < p.Lq ? lim.of(q0 + tid) : 0;
                s_doc[tid] = g_doc;
                if (p.q_pos)
#pragma unroll
                    for (int a = 0; a < 3; ++a)
                        if (a < p.axes)
                            s_pos[a][tid] = g_pos[a];
            }
            __syncthreads();
            const int this64 = t64;
            if (++sub == per64) {
                sub = 0;
                t64 = walk.next(lane);
            }
            if (t64 < t_end)
                fetch(t64 * 64 + sub * QT);

            const int last = min(q0 + QT, p.Lq) - 1;
            if (last < q0)
                continue;
            bool use = kw < lim.of(last);
            bool masked = kw + 32 > lim.of(q0) || q0 + QT > p.Lq;
            if (q_tiles) {
                use = use && docs_meet(q_tiles[this64], wave_docs);
                masked = masked || !docs_same(q_tiles[this64], wave_docs);
            }
            if (!use)
                continue;

#pragma unroll 1
            for (int qb = 0; qb < QB; ++qb) {
                f32x16 s = {}, ds = {};
#pragma unroll
                for (int c = 0; c < C; ++c) {
                    s = mma32(L::row8(sq, 32 * qb + (lane & 31), 2 * c + half), kf[c], s);
                    if constexpr (DK)
                        ds = mma32(L::row8(sdo, 32 * qb + (lane & 31), 2 * c + half), vf[c], ds);
                }
                f32x16 slant;
                if (p.cap > 0.f) {
                    const float in = p.scale / p.cap, out = p.cap * kLog2e;
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const float t = cap_tanh<T>(s[i] * in);
                        slant[i] = fmaf(-t, t, 1.f);
                        s[i] = out * t;
                    }
                } else {
                    const float m = p.scale * kLog2e;
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        s[i] *= m;
                }
                if (p.q_pos) {
#pragma unroll
                    for (int n = 0; n < 4; ++n) {
                        const int j = 32 * qb + 8 * n + 4 * half;
                        f32x4 dist = away(*(const f32x4 *)(s_pos[0] + j), my_pos[0]);
                        if (p.axes > 1)
                            dist += away(*(const f32x4 *)(s_pos[1] + j), my_pos[1]);
                        if (p.axes > 2)
                            dist += away(*(const f32x4 *)(s_pos[2] + j), my_pos[2]);
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            s[4 * n + e] = fmaf(-slope, dist[e], s[4 * n + e]);
                    }
                } else if (p.slopes) {
                    const float from = (float)(q0 + 32 * qb + 4 * half + lim.offset - kj);
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        s[i] = fmaf(-slope, fabsf(from + (float)(8 * (i / 4) + i % 4)), s[i]);
                }
#pragma unroll
                for (int n = 0; n < 4; ++n) {
                    const int j = 32 * qb + 8 * n + 4 * half;
                    const f32x4 lse = *(const f32x4 *)(s_lse + j);
                    const f32x4 delta = *(const f32x4 *)(s_delta + j);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int i = 4 * n + e;
                        s[i] = __builtin_amdgcn_exp2f(s[i] - lse[e]);
                        if constexpr (DK)
                            ds[i] = s[i] * (ds[i] - delta[e]);
                    }
                }
                if (DK && p.cap > 0.f) {
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        ds[i] *= slant[i];
                }
                if (masked) {
#pragma unroll
                    for (int n = 0; n < 4; ++n) {
                        const int j = 32 * qb + 8 * n + 4 * half;
                        const i32x4 limit = *(const i32x4 *)(s_limit + j);
                        i32x4 doc = {my_doc, my_doc, my_doc, my_doc};
                        if (q_docs)
                            doc = *(const i32x4 *)(s_doc + j);
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const bool see = (kj < limit[e]) & (doc[e] == my_doc) &
                                             (my_doc >= 0 || !q_docs);
                            s[4 * n + e] = see ? s[4 * n + e] : 0.f;
                            ds[4 * n + e] = see ? ds[4 * n + e] : 0.f;
                        }
                    }
                }
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    if constexpr (DV) {
                        const x8<T> w = pack8<T>(s, t);
#pragma unroll
                        for (int i = 0; i < DB; ++i)
                            dv[i] = mma32(L::col8(sdo, 32 * qb + 16 * t, i, lane), w, dv[i]);
                    }
                    if constexpr (DK) {
                        const x8<T> w = pack8<T>(ds, t);
#pragma unroll
                        for (int i = 0; i < DB; ++i)
                            dk[i] = mma32(L::col8(sq, 32 * qb + 16 * t, i, lane), w, dk[i]);
                    }
                }
            }
        }
    }

    if (kj >= p.Lk)
        return;
    const int64_t at = (((int64_t)b * p.Lk + kj) * p.Hkv + kvh) * p.D;
#pragma unroll
    for (int i = 0; i < DB; ++i)
#pragma unroll
        for (int e = 0; e < 16; e += 4) {
            const int d = 32 * i + 2 * e + 4 * half;
            if (d < p.D) {
                x4<T> y, z;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    y[j] = (T)(dk[i][e + j] * p.scale);
                    z[j] = (T)dv[i][e + j];
                }
                if constexpr (DK)
                    *(x4<T> *)((T *)p.dk + at + d) = y;
                if constexpr (DV)
                    *(x4<T> *)((T *)p.dv + at + d) = z;
            }
        }
}

template <typename T, int DP>
__global__ __launch_bounds__(256, 1) void attend_backward_q(const Args p) {
    using L = Tile<T, DP>;
    constexpr int KT = BackwardShape<T, DP>::kRows, KB = KT / 32, C = DP / 16, DB = DP / 32;
    __shared__ u32x4 sk[KT * L::U];
    __shared__ u32x4 sv[KT * L::U];
    __shared__ __attribute__((aligned(16))) int s_docs[KT];
    __shared__ __attribute__((aligned(16))) float s_pos[3][KT];

    const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int q_blocks = (p.Lq + 127) / 128;
    int id = xcd_order(blockIdx.x, gridDim.x);
    const int qb = q_blocks - 1 - id % q_blocks;
    id /= q_blocks;
    const int head = id % p.H, b = id / p.H;
    const int kvh = head / (p.H / p.Hkv);

    const int q0 = qb * 128, qw = q0 + 32 * wave, qi = qw + (lane & 31);
    const Limits lim(p, b);
    const int block_limit = lim.of(min(q0 + 128, p.Lq) - 1);
    const int wave_limit = qw < p.Lq ? lim.of(min(qw + 32, p.Lq) - 1) : 0;
    const int full_limit = qw < p.Lq ? lim.of(qw) : 0;
    const QueryLane<T, true> rows(p, lim, b, head, qi);
    const bool q_real = qi < p.Lq && !(p.q_docs && rows.doc < 0);

    const T *q = (const T *)p.q + b * p.q_b + head * p.q_h + (q_real ? qi : 0) * p.q_l;
    const T *dout = (const T *)p.dout + b * p.do_b + head * p.do_h + (q_real ? qi : 0) * p.do_l;
    const T *k = (const T *)p.k + b * p.k_b + kvh * p.k_h;
    const T *v = (const T *)p.v + b * p.v_b + kvh * p.v_h;
    const int32_t *k_docs = p.k_docs ? p.k_docs + (int64_t)b * p.Lk : nullptr;
    const float *k_pos = p.k_pos ? p.k_pos + (int64_t)b * p.Lk * p.axes : nullptr;

    x8<T> qf[C], of[C];
#pragma unroll
    for (int c = 0; c < C; ++c) {
        qf[c] = global8<T>(q, 16 * c + 8 * half, p.D, q_real);
        of[c] = global8<T>(dout, 16 * c + 8 * half, p.D, q_real);
    }
    const int64_t row = ((int64_t)b * p.H + head) * p.Lq + qi;
    float lse = qi < p.Lq ? p.lse[row] * kLog2e : kInf;
    lse = lse == -kInf ? kInf : lse; // an empty row: every weight 2^-inf
    const float delta = qi < p.Lq ? p.delta[row] : 0.f;
    const float mul = rows.factor(p);

    constexpr int per64 = 64 / KT;
    int4 wave_docs = {0, 0, 0, 0};
    const int64_t nk = (p.Lk + 63) / 64, nq = (p.Lq + 63) / 64;
    const int4 *k_tiles = p.k_tiles ? p.k_tiles + b * nk : nullptr;
    const int t_end = (block_limit + 63) / 64;
    TileWalk walk;
    {
        int4 mine = {0, 0, 0, 0};
        if (p.q_tiles) {
            const int4 *t = p.q_tiles + b * nq;
            mine = t[q0 / 64];
            if (q0 / 64 + 1 < nq) {
                const int4 o = t[q0 / 64 + 1];
                mine.x = min(mine.x, o.x);
                mine.y = max(mine.y, o.y);
            }
            wave_docs = qw < p.Lq ? t[qw / 64] : (int4){0x7fffffff, -1, 0, 0};
        }
        walk.start(k_tiles, mine, 0, t_end, lane);
    }

    f32x16 dq[DB];
#pragma unroll
    for (int i = 0; i < DB; ++i)
        dq[i] = f32x16{};

    Stage<T, DP, KT, 256> gk, gv;
    int g_doc = -1;
    float g_pos[3];
    const int seen = min(block_limit, p.Lk);
    auto fetch = [&](int k0) {
        gk.load(k, p.k_l, k0, seen, p.D, k_docs, tid);
        gv.load(v, p.v_l, k0, seen, p.D, k_docs, tid);
        if (k_docs && tid < KT)
            g_doc = k0 + tid < seen ? k_docs[k0 + tid] : -1;
        if (k_pos && tid < KT)
#pragma unroll
            for (int a = 0; a < 3; ++a)
                if (a < p.axes)
                    g_pos[a] = k0 + tid < seen ? k_pos[(int64_t)(k0 + tid) * p.axes + a] : 0.f;
    };
    int t64 = walk.next(lane), sub = 0;
    if (t64 < t_end)
        fetch(t64 * 64);
    while (t64 < t_end) {
        const int k0 = t64 * 64 + sub * KT;
        __syncthreads();
        gk.store(sk, tid);
        gv.store(sv, tid);
        if (k_docs && tid < KT)
            s_docs[tid] = g_doc;
        if (k_pos && tid < KT)
#pragma unroll
            for (int a = 0; a < 3; ++a)
                if (a < p.axes)
                    s_pos[a][tid] = g_pos[a];
        __syncthreads();
        const int this64 = t64;
        if (++sub == per64) {
            sub = 0;
            t64 = walk.next(lane);
        }
        if (t64 < t_end)
            fetch(t64 * 64 + sub * KT);

        bool use = k0 < wave_limit, masked = k0 + KT > full_limit;
        if (k_docs) {
            use = use && docs_meet(k_tiles[this64], wave_docs);
            masked = masked || !docs_same(k_tiles[this64], wave_docs);
        }
        if (!use)
            continue;

#pragma unroll 1
        for (int kb = 0; kb < KB; ++kb) {
            f32x16 s = {}, ds = {}, slant;
#pragma unroll
            for (int c = 0; c < C; ++c) {
                s = mma32(L::row8(sk, 32 * kb + (lane & 31), 2 * c + half), qf[c], s);
                ds = mma32(L::row8(sv, 32 * kb + (lane & 31), 2 * c + half), of[c], ds);
            }
            rows.score(p, s, &slant, k0 + 32 * kb, half, &s_pos[0][32 * kb], KT);
#pragma unroll
            for (int i = 0; i < 16; ++i)
                ds[i] = __builtin_amdgcn_exp2f(fmaf(s[i], mul, -lse)) * (ds[i] - delta);
            if (p.cap > 0.f) {
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    ds[i] *= slant[i];
            }
            if (masked)
                rows.hide(p, ds, 0.f, k0 + 32 * kb, half, s_docs + 32 * kb);
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const x8<T> w = pack8<T>(ds, t);
#pragma unroll
                for (int i = 0; i < DB; ++i)
                    dq[i] = mma32(L::col8(sk, 32 * kb + 16 * t, i, lane), w, dq[i]);
            }
        }
    }

    if (qi >= p.Lq)
        return;
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
                    y[j] = (T)(dq[i][e + j] * p.scale);
                *(x4<T> *)(dst + d) = y;
            }
        }
}

// delta: a wave for each query and head.  From the output as it was before it was rounded,
// in two parts: the rounding alone would add as much error to dq and dk as that of ds does.
template <typename T>
__global__ __launch_bounds__(256) void attend_delta(const Args p, float *delta) {
    const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int lane = threadIdx.x & 63;
    if (row >= (int64_t)p.B * p.Lq * p.H)
        return;
    const int head = (int)(row % p.H), i = (int)(row / p.H % p.Lq);
    const int64_t b = row / p.H / p.Lq;
    const T *o = (const T *)p.out + row * p.D, *low = (const T *)p.out_low + row * p.D;
    const T *dout = (const T *)p.dout + b * p.do_b + i * p.do_l + head * p.do_h;
    float x = 0.f;
    for (int d = 4 * lane; d < p.D; d += 256) {
        const x4<T> u = *(const x4<T> *)(o + d), w = *(const x4<T> *)(dout + d);
#pragma unroll
        for (int j = 0; j < 4; ++j)
            x = fmaf((float)u[j], (float)w[j], x);
        if (p.out_low) {
            const x4<T> r = *(const x4<T> *)(low + d);
#pragma unroll
            for (int j = 0; j < 4; ++j)
                x = fmaf((float)r[j], (float)w[j], x);
        }
    }
#pragma unroll
    for (int n = 32; n; n >>= 1)
        x += __shfl_xor(x, n);
    if (!lane)
        delta[(b * p.H + head) * p.Lq + i] = x;
}

template <typename T> int run_delta(const Args &a, float *delta, hipStream_t s) {
    const int64_t rows = (int64_t)a.B * a.Lq * a.H;
    attend_delta<T><<<dim3((unsigned)((rows + 3) / 4)), 256, 0, s>>>(a, delta);
    return hipGetLastError() == hipSuccess ? 0 : 1;
}

template <typename T, int DP> int run_backward_kv(const Args &a, hipStream_t s) {
    const dim3 grid((unsigned)((int64_t)((a.Lk + 127) / 128) * a.Hkv * a.B));
    if constexpr (BackwardShape<T, DP>::kTwoPasses) {
        attend_backward_kv<T, DP, 1><<<grid, 256, 0, s>>>(a);
        attend_backward_kv<T, DP, 2><<<grid, 256, 0, s>>>(a);
    } else {
        attend_backward_kv<T, DP, 3><<<grid, 256, 0, s>>>(a);
    }
    return hipGetLastError() == hipSuccess ? 0 : 1;
}

template <typename T, int DP> int run_backward_q(const Args &a, hipStream_t s) {
    const dim3 grid((unsigned)((int64_t)((a.Lq + 127) / 128) * a.H * a.B));
    attend_backward_q<T, DP><<<grid, 256, 0, s>>>(a);
    return hipGetLastError() == hipSuccess ? 0 : 1;
}

} // namespace attn

#endif
