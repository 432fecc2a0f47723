// attn_forward.h -- attention forward: out = softmax(scores) v in one pass over
// the keys.
//
// A wave owns 32 queries.  It forms the transposed scores, keys by queries
// (k q^T), so that a lane holds scores of one query only: the running maximum
// and sum need one exchange between the two halves of the wave, the rescaling
// of the output is by a scalar per lane, and the weights lie as the next product
// (v^T p^T) wants them.  q stays in registers; tiles of 64 keys pass through LDS in two
// buffers, brought by all four waves, one on its way while the other is used.
//
// Weights are rounded to the inputs' type for the second product, as they lie
// between 0 and 2^8 and every weight of a row errs by as much, relatively, as an
// input does; scores, maxima, sums and the output accumulate in float32.
#ifndef TORCHMATCH_AMD_ATTN_FORWARD_H
#define TORCHMATCH_AMD_ATTN_FORWARD_H

#include "attn_tile.h"

namespace attn {

template <typename T, int DP, bool SIDE> struct ForwardShape {
    static constexpr int kWaves = 4;
    static constexpr int kQueries = 32 * kWaves;
    // One wave issues a vector instruction every 8 cycles at most, two or three together one
    // every 4, and the weights take as long as the products: what counts is waves a SIMD, and
    // with it registers.  Three up to 128 bytes a row; with 256 bytes only where there are no
    // documents and positions, and 32 keys at a time (causal, 32768 rows of 128 features, 16
    // heads: 4.5 to 4.6 ms in place of 4.8, 0.96 PFLOP/s, though five registers are in scratch;
    // 2 x 8192 packed in documents, with blocks as they stand, 192 us, 267 with three, and 160
    // with the longest blocks first).
    static constexpr int kBytes = sizeof(T) * DP;
    static constexpr int kOccupancy = kBytes <= 128 || (kBytes <= 256 && !SIDE) ? 3
                                      : kBytes <= 256                          ? 2
                                                                               : 1;
    // float32 rows of 256: 32 keys at a time, so that two tiles of k and v fit in LDS
    static constexpr int kKeys = kBytes == 1024 || (kBytes > 128 && kBytes <= 256 && !SIDE)
                                     ? 32
                                     : 64;
};

template <typename T, int DP, bool SIDE>
__global__ __launch_bounds__(256, (ForwardShape<T, DP, SIDE>::kOccupancy)) void
attend_forward(const Args p) {
    using S = ForwardShape<T, DP, SIDE>;
    using L = Tile<T, DP>;
    constexpr int KT = S::kKeys, KB = KT / 32, QT = S::kQueries, C = DP / 16, DB = DP / 32;
    __shared__ u32x4 sk0[KT * L::U], sk1[KT * L::U];
    __shared__ u32x4 sv0[KT * L::U], sv1[KT * L::U];
    __shared__ __attribute__((aligned(16))) int s_docs0[64], s_docs1[64];
    __shared__ __attribute__((aligned(16))) float s_pos0[3][64], s_pos1[3][64];

    const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int q_blocks = (p.Lq + QT - 1) / QT;
    const int group = p.H / p.Hkv;
    const Share share(blockIdx.x, q_blocks, p.B * p.H * p.splits);
    const int split = share.head % p.splits, head = share.head / p.splits % p.H;
    const int b = share.head / p.splits / p.H;
    const int qb = SIDE && p.q_order ? scalar(p.q_order[(int64_t)b * q_blocks + share.block])
                                     : q_blocks - 1 - share.block; // the last see most
    const int kvh = head / group;

    const int q0 = qb * QT, qw = q0 + 32 * wave, qi = qw + (lane & 31);
    const bool q_real = qi < p.Lq;
    const Limits lim(p, b);
    const uint32_t row_at = L::row_lane(lane), col_at = L::col_lane(lane);
    const int block_limit = lim.of(min(q0 + QT, p.Lq) - 1);
    const int wave_limit = qw < p.Lq ? lim.of(min(qw + 32, p.Lq) - 1) : 0;
    const int full_limit = qw < p.Lq ? lim.of(qw) : 0; // keys that all of the wave see

    const T *q = (const T *)p.q + b * p.q_b + head * p.q_h;
    const T *k = (const T *)p.k + b * p.k_b + kvh * p.k_h;
    const T *v = (const T *)p.v + b * p.v_b + kvh * p.v_h;
    const int32_t *k_docs = SIDE && p.k_docs ? p.k_docs + (int64_t)b * p.Lk : nullptr;
    const float *k_pos = SIDE && p.k_pos ? p.k_pos + (int64_t)b * p.Lk * p.axes : nullptr;
    const QueryLane<T, SIDE> rows(p, lim, b, head, qi);

    x8<T> qf[C];
#pragma unroll
    for (int c = 0; c < C; ++c)
        qf[c] = global8<T>(q + (int64_t)(q_real ? qi : 0) * p.q_l, 16 * c + 8 * half, p.D, q_real);
    // documents: of the block (which tiles to visit) and of the wave (which to use)
    constexpr int per64 = 64 / KT; // key tiles to a summary
    int4 wave_docs = {0, 0, 0, 0};
    TileWalk walk;
    const int t_end = min((block_limit + 63) / 64, (split + 1) * p.tiles_per_split);
    {
        const int64_t nk = (p.Lk + 63) / 64, nq = (p.Lq + 63) / 64;
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
        walk.start(SIDE && p.k_tiles ? p.k_tiles + b * nk : nullptr, mine, split * p.tiles_per_split,
                   t_end, lane);
    }

    f32x16 o[DB];
#pragma unroll
    for (int i = 0; i < DB; ++i)
        o[i] = f32x16{};
    float top = -kInf, sum = 0.f; // of this lane's query; the sum of this half's keys

    using B = Bring<T, DP, KT, 256>;
    const int seen = min(block_limit, p.Lk); // keys past it may hold anything
    const float mul = rows.factor(p);
    int t64 = walk.next(lane), sub = 0;

    // The tile from key k0 on into a buffer.
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
    // One tile from its buffer while the next one is on its way into the other.
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
            B::clear(sv, k0, seen, k_docs, s_docs, tid);
            __syncthreads();
        }
        if (!use)
            return;

        // scores: keys by queries
        f32x16 s[KB];
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
            s[kb] = f32x16{};
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int kb = 0; kb < KB; ++kb)
                s[kb] = mma32(L::row8(sk, row_at, 32 * kb, c), qf[c], s[kb]);
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
            rows.score(p, s[kb], k0 + 32 * kb, half, &s_pos[0][32 * kb], 64);
        if (masked) {
#pragma unroll
            for (int kb = 0; kb < KB; ++kb)
                rows.hide(p, s[kb], -kInf, k0 + 32 * kb, half, s_docs + 32 * kb);
        }
        soften<T>(s, o, mul, top, sum);

        // output, transposed: v^T p^T
#pragma unroll
        for (int t = 0; t < KT / 16; ++t) {
            const x8<T> w = pack8<T>(s[t / 2], t % 2);
#pragma unroll
            for (int i = 0; i < DB; ++i)
                o[i] = mma32(L::col8(sv, col_at, 16 * t, i), w, o[i]);
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

    sum += __shfl_xor(sum, 32);
    if (!q_real)
        return;
    const int64_t row = ((int64_t)b * p.H + head) * p.Lq + qi;
    if (p.splits > 1) {
        const int64_t at = (int64_t)split * p.B * p.H * p.Lq + row;
        float *dst = p.part_o + at * DP;
#pragma unroll
        for (int i = 0; i < DB; ++i)
#pragma unroll
            for (int e = 0; e < 16; e += 4)
                *(f32x4 *)(dst + 32 * i + 2 * e + 4 * half) =
                    (f32x4){o[i][e], o[i][e + 1], o[i][e + 2], o[i][e + 3]};
        if (!half)
            p.part_ml[at] = make_float2(top, sum);
        return;
    }
    const float r = sum == 0.f ? 0.f : 1.f / sum;
    const int64_t at = (((int64_t)b * p.Lq + qi) * p.H + head) * p.D;
#pragma unroll
    for (int i = 0; i < DB; ++i)
#pragma unroll
        for (int e = 0; e < 16; e += 4) {
            const int d = 32 * i + 2 * e + 4 * half;
            if (d < p.D) {
                const f32x4 x = {o[i][e] * r, o[i][e + 1] * r, o[i][e + 2] * r, o[i][e + 3] * r};
                put<T>(p, at + d, __builtin_convertvector(x, x4<T>), x);
            }
        }
    if (!half && p.lse)
        p.lse[row] = sum == 0.f ? -kInf : kLn2 * (top + __builtin_amdgcn_logf(sum));
}

// Joins the partial results of a split over keys: 64 threads for each query, 4 features each
// thread; where a row has fewer than 256, the rest of them take other splits.
template <typename T, int DP>
__global__ __launch_bounds__(256) void attend_join(const Args p) {
    constexpr int N = DP / 4, P = 64 / N; // threads of a part's row, parts at a time
    const int64_t rows = (int64_t)p.B * p.H * p.Lq;
    const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int lane = threadIdx.x & 63;
    if (row >= rows)
        return;
    float top = -kInf;
    for (int s = lane; s < p.splits; s += 64)
        top = fmaxf(top, p.part_ml[s * rows + row].x);
#pragma unroll
    for (int x = 32; x; x >>= 1)
        top = fmaxf(top, __shfl_xor(top, x));
    const float from = top == -kInf ? 0.f : top;
    const int part = lane / N, d = 4 * (lane % N);
    float sum = 0.f;
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
    if (part < P) {
#pragma unroll 4
        for (int s = part; s < p.splits; s += P) {
            const int64_t at = s * rows + row;
            const float2 ml = p.part_ml[at];
            const float w = __builtin_amdgcn_exp2f(ml.x - from);
            const f32x4 x = *(const f32x4 *)(p.part_o + at * DP + d);
            sum = fmaf(ml.y, w, sum);
#pragma unroll
            for (int j = 0; j < 4; ++j)
                o[j] = fmaf(w, x[j], o[j]);
        }
    }
#pragma unroll
    for (int x = 1; x < P; ++x) {
        const float more = __shfl(sum, lane % N + x * N);
        sum = part == 0 ? sum + more : sum;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float y = __shfl(o[j], lane % N + x * N);
            o[j] = part == 0 ? o[j] + y : o[j];
        }
    }
    if (part == 0 && d < p.D) {
        const int i = (int)(row % p.Lq), head = (int)(row / p.Lq % p.H);
        const int64_t b = row / p.Lq / p.H;
        o *= sum == 0.f ? 0.f : 1.f / sum;
        put<T>(p, ((b * p.Lq + i) * p.H + head) * p.D + d, __builtin_convertvector(o, x4<T>), o);
    }
    if (!lane && p.lse)
        p.lse[row] = sum == 0.f ? -kInf : kLn2 * (top + __builtin_amdgcn_logf(sum));
}

template <typename T, int DP> int run_forward(const Args &a, hipStream_t s) {
    constexpr int Q = ForwardShape<T, DP, true>::kQueries;
    const int64_t blocks = (int64_t)((a.Lq + Q - 1) / Q) * a.splits * a.H * a.B;
    if (a.q_docs || a.q_pos)
        attend_forward<T, DP, true><<<dim3((unsigned)blocks), 256, 0, s>>>(a);
    else
        attend_forward<T, DP, false><<<dim3((unsigned)blocks), 256, 0, s>>>(a);
    return hipGetLastError() == hipSuccess ? 0 : 1;
}

template <typename T, int DP> int run_join(const Args &a, hipStream_t s) {
    const int64_t rows = (int64_t)a.B * a.H * a.Lq;
    attend_join<T, DP><<<dim3((unsigned)((rows + 3) / 4)), 256, 0, s>>>(a);
    return hipGetLastError() == hipSuccess ? 0 : 1;
}

} // namespace attn

#endif
