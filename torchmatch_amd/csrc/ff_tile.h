// ff_tile.h -- matrix products of the feed-forward block on tiles in LDS, and what is done with
// their results before they are written.
//
//     h = act(x G^T) * (x U^T),  y = h D^T                               (rows by rows)
//     dh = dy D -> da, db, h;  dx = da G + db U                            (rows by columns)
//     dG = da^T x, dU = db^T x, dD = dy^T h                                (columns by columns)
//
// A block has BM x BN of the result, a wave 64 columns of it.  Tiles of 128 bytes of k go from memory
// straight into LDS, two buffers, one barrier a tile.  Operands whose rows hold k are read by rows, others
// by transposed reads (attn_tile.h has the tiles' layout), so nothing is transposed in memory.  The
// result's columns lie along a lane's registers; a wave turns them through LDS, 32 rows at a
// time, and writes whole rows of its tile.
#ifndef TORCHMATCH_AMD_FF_TILE_H
#define TORCHMATCH_AMD_FF_TILE_H

#include "attn_tile.h"
#include "ff.h"

#include "../../include/torchmatch_amd.h"

namespace ff {

using attn::f32x16;
using attn::f32x4;
using attn::f32x8;
using attn::mma32;
using attn::u32x4;
using attn::x8;

typedef uint16_t u16x8 __attribute__((ext_vector_type(8)));

// ---- activations ------------------------------------------------------------------

// The activation's value and slope.  16-bit types take the hardware's exponential and reciprocal
// (2^-22), float32 the library's.
template <typename T> __device__ inline float exp_of(float x) {
    return sizeof(T) == 2 ? __builtin_amdgcn_exp2f(x * attn::kLog2e) : expf(x);
}
template <typename T> __device__ inline float over(float x) { // 1 / x
    return sizeof(T) == 2 ? __builtin_amdgcn_rcpf(x) : 1.f / x;
}
template <typename T> __device__ inline float2 activate(float a, int kind) {
    switch (kind) {
    case TM_SILU: {
        const float s = over<T>(1.f + exp_of<T>(-a));
        return make_float2(a * s, s * (1.f + a * (1.f - s)));
    }
    case TM_RELU: return make_float2(fmaxf(a, 0.f), a > 0.f ? 1.f : 0.f);
    case TM_GELU: {
        const float cdf = 0.5f * erfcf(-0.70710678118654752440f * a);
        return make_float2(a * cdf, cdf + a * 0.39894228040143267794f * exp_of<T>(-0.5f * a * a));
    }
    default: { // the approximation by tanh
        const float k = 0.79788456080286535588f;
        const float t = tanhf(k * (a + 0.044715f * a * a * a));
        const float half = 0.5f * (1.f + t);
        return make_float2(a * half, half + 0.5f * a * (1.f - t * t) * k *
                                                (1.f + 3.f * 0.044715f * a * a));
    }
    }
}

// ---- tiles ------------------------------------------------------------------------

template <typename T> constexpr int kStep = 128 / (int)sizeof(T); // k a tile

// One operand's tile, ROWS x kStep, brought by NT threads.  STRIDED: a row for each k.
template <typename T, int ROWS, bool STRIDED, int NT> struct Feed {
    static constexpr int BK = kStep<T>, E = 16 / (int)sizeof(T);
    using L = attn::Tile<T, STRIDED ? ROWS : BK>;
    static constexpr int SIZE = (STRIDED ? BK : ROWS) * L::U; // units
    static constexpr int N = SIZE / NT, STEP = NT / L::U;
    static_assert(SIZE % NT == 0 && NT % L::U == 0 && L::U == L::U0);

    uint32_t off[N]; // bytes from the tile's first element, its k aside
    int unit[N];     // not strided: the unit of k

    // left: rows (columns) from the tile's first on; GATED: 32 rows of the one matrix, 32 of the
    // other, in turn
    template <bool GATED>
    __device__ inline void start(int tid, int64_t stride, int left) {
        const int row = tid / L::U, pos = tid % L::U;
        const uint32_t bytes = (uint32_t)stride * (uint32_t)sizeof(T);
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const int r = row + n * STEP, u = pos ^ L::swz(r);
            unit[n] = u;
            if constexpr (STRIDED) {
                off[n] = (uint32_t)r * bytes + 16u * min(u, (left - 1) / E);
            } else {
                const int real = GATED ? (r >> 6) * 32 + (r & 31) : r;
                off[n] = (uint32_t)min(real, left - 1) * bytes + 16u * u;
            }
        }
    }
    // which matrix of a gated pair load n is of: the same for a whole wave
    __device__ static inline int of_pair(int tid, int n) {
        return attn::scalar((tid / L::U + n * STEP) >> 5) & 1;
    }
    // from: the tile's first element; second: of the other matrix (gated)
    template <bool GATED>
    __device__ inline void load(u32x4 *t, const char *from, const char *second, int tid) const {
        u32x4 *to = t + attn::scalar(tid & ~63);
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const char *s = GATED && of_pair(tid, n) ? second : from;
            __builtin_amdgcn_global_load_lds(
                (const __attribute__((address_space(1))) void *)(s + off[n]),
                (__attribute__((address_space(3))) void *)(to + n * NT), 16, 0, 0);
        }
    }
    // the last tile, of which `left` k are there: zeros past them
    template <bool GATED>
    __device__ inline void load_last(u32x4 *t, const char *from, const char *second, int tid,
                                     int left) const {
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const char *s = GATED && of_pair(tid, n) ? second : from;
            const bool real = STRIDED ? tid / L::U + n * STEP < left : unit[n] * E < left;
            u32x4 x = {0u, 0u, 0u, 0u};
            if (real)
                x = *(const u32x4 *)(s + off[n]);
            t[tid + n * NT] = x;
        }
    }

    // Where a lane reads.
    __device__ static inline uint32_t lane_at(int lane) {
        if constexpr (!STRIDED) {
            return L::row_lane(lane);
        } else if constexpr (sizeof(T) == 2) {
            const int d = (lane & 16) + 4 * (lane & 3);
            return 16u * L::at(8 * (lane >> 5) + ((lane & 15) >> 2), d >> 3) + 2u * (d & 7);
        } else {
            return 16u * L::at(8 * (lane >> 5), (lane & 31) / E) + 4u * (lane & 3);
        }
    }
    // An operand: row (column) 32 rb + lane % 32, k 16 c + 8 (lane / 32) + 0 .. 7
    __device__ static inline x8<T> operand(const u32x4 *t, uint32_t at, int rb, int c) {
        if constexpr (!STRIDED) {
            return L::row8(t, at, 32 * rb, c);
        } else {
            const char *from = (const char *)t + 16 * c * L::U * 16;
            x8<T> r;
            if constexpr (sizeof(T) == 2) {
                // the transposed read: each 16 lanes load 4 rows of 16 elements (4 a lane) and
                // each lane gets one column of them
#pragma unroll
                for (int jj = 0; jj < 2; ++jj) {
                    const char *p = from + 4 * jj * L::U * 16 + (at ^ (64u * rb + 16u * jj));
                    const attn::s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                        (__attribute__((address_space(3))) attn::s16x4 *)p);
                    const attn::x4<T> y = __builtin_bit_cast(attn::x4<T>, x);
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        r[4 * jj + j] = y[j];
                }
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    r[j] = *(const float *)(from + j * L::U * 16 +
                                            (at ^ (16u * (8 * rb ^ L::swz(j)))));
            }
            return r;
        }
    }
};

// ---- results ----------------------------------------------------------------------

template <typename T> __device__ inline void put8(T *to, f32x8 x) {
    typedef T U __attribute__((ext_vector_type(8)));
    if constexpr (sizeof(T) == 2) {
        U y;
#pragma unroll
        for (int j = 0; j < 8; ++j)
            y[j] = (T)x[j];
        *(U *)to = y;
    } else {
        *(f32x4 *)to = (f32x4){x[0], x[1], x[2], x[3]};
        *(f32x4 *)(to + 4) = (f32x4){x[4], x[5], x[6], x[7]};
    }
}

// a and b as they are saved: float32, or its first 24 bits (truncated: what a gradient then is off
// by, 2^-15, is far below the rounding of the gradients to 16 bits)
template <typename T> __device__ inline void save(const Args &p, int64_t at, f32x8 a, f32x8 b) {
    if constexpr (sizeof(T) == 4) {
        put8((float *)p.saved[0] + at, a);
        put8((float *)p.saved[1] + at, b);
    } else {
        u16x8 x, y, z;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const uint32_t u = __float_as_uint(a[j]), v = __float_as_uint(b[j]);
            x[j] = (uint16_t)(u >> 16);
            y[j] = (uint16_t)(v >> 16);
            z[j] = (uint16_t)((u & 0xff00u) | (v >> 8 & 0xffu));
        }
        *(u16x8 *)((uint16_t *)p.saved[0] + at) = x;
        *(u16x8 *)((uint16_t *)p.saved[1] + at) = y;
        *(u16x8 *)((uint16_t *)p.saved[2] + at) = z;
    }
}
template <typename T> __device__ inline void saved(const Args &p, int64_t at, f32x8 &a, f32x8 &b) {
    if constexpr (sizeof(T) == 4) {
        const f32x4 *u = (const f32x4 *)((const float *)p.saved[0] + at);
        const f32x4 *v = (const f32x4 *)((const float *)p.saved[1] + at);
        const f32x4 u0 = u[0], u1 = u[1], v0 = v[0], v1 = v[1];
        a = (f32x8){u0[0], u0[1], u0[2], u0[3], u1[0], u1[1], u1[2], u1[3]};
        b = (f32x8){v0[0], v0[1], v0[2], v0[3], v1[0], v1[1], v1[2], v1[3]};
    } else {
        const u16x8 x = *(const u16x8 *)((const uint16_t *)p.saved[0] + at);
        const u16x8 y = *(const u16x8 *)((const uint16_t *)p.saved[1] + at);
        const u16x8 z = *(const u16x8 *)((const uint16_t *)p.saved[2] + at);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            a[j] = __uint_as_float((uint32_t)x[j] << 16 | (z[j] & 0xff00u));
            b[j] = __uint_as_float((uint32_t)y[j] << 16 | (uint32_t)(z[j] & 0xffu) << 8);
        }
    }
}

// The power of two that brings the largest |dy| to 1 .. 2: half precision holds gradients of the
// hidden features times this (they are as small as the loss makes them, and lose bits below 2^-14).
template <typename T> __device__ inline int grad_up(const Args &p, int lane) {
    if constexpr (__is_same(T, _Float16)) {
        if (!p.most)
            return 0;
        float m = 0.f;
        for (int i = lane; i < kMostParts; i += 64)
            m = fmaxf(m, p.most[i]);
#pragma unroll
        for (int n = 1; n < 64; n *= 2)
            m = fmaxf(m, __shfl_xor(m, n));
        return m > 0.f && m < attn::kInf ? 1 - __builtin_amdgcn_frexp_expf(m) : 0;
    }
    return 0;
}

// One row's 8 results from column n on.
template <typename T>
__device__ inline void put_row(const Args &p, int batch, int split, int64_t m, int n, f32x8 x) {
    if (p.part) {
        float *to = p.part + (((int64_t)split * p.batches + batch) * p.M + m) * p.N + n;
        if (p.N % 4 == 0 && n + 8 <= p.N) {
            put8(to, x);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (n + j < p.N)
                    to[j] = x[j];
        }
        return;
    }
    T *to = (T *)p.out[batch] + m * p.out_l + n;
    if (p.wide && n + 8 <= p.N) {
        put8(to, x);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (n + j < p.N)
                to[j] = (T)x[j];
    }
}

// h, and a and b where they are saved; zeros past the hidden features
template <typename T>
__device__ inline void put_hidden(const Args &p, int64_t m, int n, f32x8 a, f32x8 b) {
    f32x8 h;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        h[j] = activate<T>(a[j], p.activation).x * b[j];
        if (n + j >= p.N)
            h[j] = a[j] = b[j] = 0.f;
    }
    const int64_t at = m * p.out_l + n;
    if (p.saved[0])
        save<T>(p, at, a, b);
    put8((T *)p.out[0] + at, h);
}

template <typename T>
__device__ inline void put_grads(const Args &p, int64_t m, int n, f32x8 dh, int up) {
    const int64_t at = m * p.out_l + n;
    const float by = __builtin_ldexpf(1.f, up);
    f32x8 a, b, h, da, db;
    saved<T>(p, at, a, b);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const float2 act = activate<T>(a[j], p.activation);
        const bool real = n + j < p.N;
        h[j] = real ? act.x * b[j] : 0.f;
        da[j] = real ? dh[j] * by * b[j] * act.y : 0.f;
        db[j] = real ? dh[j] * by * act.x : 0.f;
    }
    put8((T *)p.out[0] + at, h);
    put8((T *)p.da + at, da);
    put8((T *)p.db + at, db);
}

// ---- the product ------------------------------------------------------------------

template <Kind K> struct Shape { // which operands are strided
    static constexpr bool kA = K == kWeights, kB = K != kUp && K != kDown;
};

template <bool BIG> struct Size {
    static constexpr int BM = BIG ? 256 : 128, BN = BM, MB = BIG ? 4 : 2; // MB: 32 rows each
    static constexpr int NT = BIG ? 512 : 256;
};

template <typename T, Kind KIND, bool BIG>
__global__ __launch_bounds__((Size<BIG>::NT), 2) void product(const Args p) {
    using Z = Size<BIG>;
    constexpr int BM = Z::BM, BN = Z::BN, NT = Z::NT, MB = Z::MB, NB = 2, BK = kStep<T>;
    constexpr bool GATED = KIND == kUp;
    constexpr int TN = GATED ? BN / 2 : BN; // columns of the result a block
    using FA = Feed<T, BM, Shape<KIND>::kA, NT>;
    using FB = Feed<T, BN, Shape<KIND>::kB, NT>;
    __shared__ u32x4 a0[FA::SIZE], a1[FA::SIZE], b0[FB::SIZE], b1[FB::SIZE];

    const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5;
    const int wave = attn::scalar(tid >> 6), wm = wave / (BN / 64), wn = wave % (BN / 64);
    const int mt = (p.M + BM - 1) / BM, nt = (p.N + TN - 1) / TN;
    // tiles in bands of 8 rows of tiles, a run of them an XCD: those which share operands meet
    // in its L2
    int id = attn::xcd_order(blockIdx.x, gridDim.x);
    const int split = id % p.splits;
    id /= p.splits;
    const int batch = id / (mt * nt);
    id -= batch * mt * nt;
    const int band = id / (8 * nt), in_band = id - band * 8 * nt;
    const int rows = min(8, mt - 8 * band);
    const int m0 = (8 * band + in_band % rows) * BM, n0 = in_band / rows * TN;

    FA fa;
    FB fb;
    fa.template start<false>(tid, p.a_l, p.M - m0);
    fb.template start<GATED>(tid, p.b_l, p.N - n0);
    const int spk = (p.K + BK - 1) / BK; // steps a segment
    const int s0 = split * p.split_steps, s1 = min(s0 + p.split_steps, spk * p.segments);
    const uint32_t at_a = FA::lane_at(lane), at_b = FB::lane_at(lane);

    const auto fetch = [&](int s, u32x4 *ta, u32x4 *tb) {
        const int seg = s >= spk ? 1 : 0, k = (s - seg * spk) * BK;
        const int which = KIND == kInput ? seg : batch;
        const T *pa = (const T *)p.a[which], *pb = (const T *)p.b[which];
        pa += Shape<KIND>::kA ? k * p.a_l + m0 : m0 * p.a_l + k;
        pb += Shape<KIND>::kB ? k * p.b_l + n0 : n0 * p.b_l + k;
        const T *pu = GATED ? (const T *)p.b[1] + n0 * p.b_l + k : nullptr;
        if (k + BK <= p.K) {
            fa.template load<false>(ta, (const char *)pa, nullptr, tid);
            fb.template load<GATED>(tb, (const char *)pb, (const char *)pu, tid);
        } else {
            fa.template load_last<false>(ta, (const char *)pa, nullptr, tid, p.K - k);
            fb.template load_last<GATED>(tb, (const char *)pb, (const char *)pu, tid, p.K - k);
        }
    };

    f32x16 acc[NB][MB];
#pragma unroll
    for (int i = 0; i < NB; ++i)
#pragma unroll
        for (int j = 0; j < MB; ++j)
            acc[i][j] = f32x16{};
    const auto step = [&](int s, const u32x4 *ta, const u32x4 *tb, u32x4 *next_a, u32x4 *next_b) {
        attn::arrived();
        __syncthreads(); // this tile is here, and the other buffer is done with
        if (s + 1 < s1)
            fetch(s + 1, next_a, next_b);
#pragma unroll
        for (int c = 0; c < BK / 16; ++c) {
            x8<T> x[MB], y[NB];
#pragma unroll
            for (int i = 0; i < NB; ++i)
                y[i] = FB::operand(tb, at_b, NB * wn + i, c);
#pragma unroll
            for (int j = 0; j < MB; ++j)
                x[j] = FA::operand(ta, at_a, MB * wm + j, c);
#pragma unroll
            for (int i = 0; i < NB; ++i)
#pragma unroll
                for (int j = 0; j < MB; ++j)
                    acc[i][j] = mma32(y[i], x[j], acc[i][j]);
        }
    };
    if (s0 < s1)
        fetch(s0, a0, b0);
    for (int s = s0; s < s1; s += 2) {
        step(s, a0, b0, a1, b1);
        if (s + 1 < s1)
            step(s + 1, a1, b1, a0, b0);
    }

    const int up = KIND == kHidden || KIND == kInput || KIND == kWeights ? grad_up<T>(p, lane) : 0;
    const float down = __builtin_ldexpf(1.f, -up);
    // 32 rows at a time through LDS: what was a lane's column becomes rows
    __syncthreads();
    constexpr int ROW = 68; // floats: 16 bytes more than 64, so that rows meet other banks
    constexpr int PER = NT / 64 / 4; // waves that share a buffer
    static_assert(PER * 32 * ROW * 4 <= FA::SIZE * 16 && PER * 32 * ROW * 4 <= FB::SIZE * 16);
    u32x4 *buffer = wave / PER == 0 ? a0 : wave / PER == 1 ? a1 : wave / PER == 2 ? b0 : b1;
    float *turn = (float *)buffer + wave % PER * 32 * ROW;
#pragma unroll
    for (int j = 0; j < MB; ++j) {
        attn::wave_fence();
#pragma unroll
        for (int i = 0; i < NB; ++i)
#pragma unroll
            for (int q = 0; q < 4; ++q)
                *(f32x4 *)(turn + (lane & 31) * ROW + 32 * i + 8 * q + 4 * half) =
                    (f32x4){acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2],
                            acc[i][j][4 * q + 3]};
        attn::wave_fence();
        const int mw = m0 + 32 * (MB * wm + j);
        const auto read8 = [&](int r, int col) {
            const f32x4 *from = (const f32x4 *)(turn + r * ROW + col);
            const f32x4 lo = from[0], hi = from[1];
            return (f32x8){lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
        };
        if constexpr (GATED) {
#pragma unroll
            for (int n16 = 0; n16 < 2; ++n16) {
                const int r = (lane >> 2) + 16 * n16;
                const int col = 8 * (lane & 3), n = n0 + 32 * wn + col;
                if (mw + r < p.M && n < p.out_l)
                    put_hidden<T>(p, mw + r, n, read8(r, col), read8(r, col + 32));
            }
        } else {
#pragma unroll KIND == kHidden ? 1 : 4
            for (int n8 = 0; n8 < 4; ++n8) {
                const int r = (lane >> 3) + 8 * n8;
                const int col = 8 * (lane & 7), n = n0 + 64 * wn + col;
                if constexpr (KIND == kHidden) {
                    if (mw + r < p.M && n < p.out_l)
                        put_grads<T>(p, mw + r, n, read8(r, col), up);
                } else {
                    if (mw + r < p.M && n < p.N)
                        put_row<T>(p, batch, split, mw + r, n, read8(r, col) * down);
                }
            }
        }
    }
}

// The sums of a split product, in order, 4 columns a thread where rows allow it.
template <typename T> __global__ __launch_bounds__(256) void join(const Args p) {
    const int64_t count = (int64_t)p.batches * p.M * p.N;
    const int v = p.N % 4 ? 1 : 4;
    const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * v;
    if (i >= count)
        return;
    f32x4 sum = {0.f, 0.f, 0.f, 0.f};
    for (int s = 0; s < p.splits; ++s) {
        if (v == 4)
            sum += *(const f32x4 *)(p.part + s * count + i);
        else
            sum[0] += p.part[s * count + i];
    }
    const int64_t row = i / p.N, batch = row / p.M;
    T *to = (T *)p.out[batch] + (row - batch * p.M) * p.out_l + (i - row * p.N);
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (j < v)
            to[j] = (T)sum[j];
}

template <typename T, Kind KIND, bool BIG> int launch(const Args &p, hipStream_t stream) {
    using Z = Size<BIG>;
    const int tn = KIND == kUp ? Z::BN / 2 : Z::BN;
    const int64_t blocks = (int64_t)((p.M + Z::BM - 1) / Z::BM) * ((p.N + tn - 1) / tn) *
                           p.batches * p.splits;
    if (!blocks)
        return 0;
    product<T, KIND, BIG><<<dim3((unsigned)blocks), Z::NT, 0, stream>>>(p);
    return hipGetLastError() != hipSuccess;
}

template <typename T> int run(const Args &p, Kind kind, bool big, hipStream_t stream) {
    switch (kind) {
    case kUp: return big ? launch<T, kUp, true>(p, stream) : launch<T, kUp, false>(p, stream);
    case kDown: return big ? launch<T, kDown, true>(p, stream) : launch<T, kDown, false>(p, stream);
    case kHidden:
        return big ? launch<T, kHidden, true>(p, stream) : launch<T, kHidden, false>(p, stream);
    case kInput:
        return big ? launch<T, kInput, true>(p, stream) : launch<T, kInput, false>(p, stream);
    default:
        return big ? launch<T, kWeights, true>(p, stream) : launch<T, kWeights, false>(p, stream);
    }
}

template <typename T> int run_join(const Args &p, hipStream_t stream) {
    const int64_t count = (int64_t)p.batches * p.M * p.N / (p.N % 4 ? 1 : 4);
    if (!count)
        return 0;
    join<T><<<dim3((unsigned)((count + 255) / 256)), 256, 0, stream>>>(p);
    return hipGetLastError() != hipSuccess;
}

} // namespace ff

#endif
