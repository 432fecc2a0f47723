// ff_tokens.h -- the feed-forward block's forward products of few rows, where reading the weights
// once bounds them.
//
// A block has 16 rows of the weights (of gate and of up), its waves a part of k each, so that a product
// of few rows of weights still fills the card; their sums meet in LDS, in order.  A wave loads 64
// bytes of 16 rows at once, straight into the operands of 16 x 16 products with up to 16 GROUPS
// rows of x, which all blocks share in L2.  The contraction takes its indices in the order in
// which lanes hold them, for both operands alike.
#ifndef TORCHMATCH_AMD_FF_TOKENS_H
#define TORCHMATCH_AMD_FF_TOKENS_H

#include "ff_tile.h"

namespace ff {

// 16 bytes of a row: an operand of as many indices for each quarter of the wave
template <typename T> struct Unit16;
template <> struct Unit16<__bf16> {
    __device__ static inline f32x4 mma(u32x4 a, u32x4 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(attn::b16x8, a),
                                                       __builtin_bit_cast(attn::b16x8, b), c, 0,
                                                       0, 0);
    }
};
template <> struct Unit16<_Float16> {
    __device__ static inline f32x4 mma(u32x4 a, u32x4 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(attn::h16x8, a),
                                                      __builtin_bit_cast(attn::h16x8, b), c, 0, 0,
                                                      0);
    }
};
template <> struct Unit16<float> {
    __device__ static inline f32x4 mma(u32x4 a, u32x4 b, f32x4 c) {
        const f32x4 x = __builtin_bit_cast(f32x4, a), y = __builtin_bit_cast(f32x4, b);
#pragma unroll
        for (int i = 0; i < 4; ++i)
            c = __builtin_amdgcn_mfma_f32_16x16x4f32(x[i], y[i], c, 0, 0, 0);
        return c;
    }
};

constexpr int kTokenWaves = 16;

// split_steps: pieces of 64 bytes of k a wave
template <typename T, bool GATED, int GROUPS>
__global__ __launch_bounds__(64 * kTokenWaves) void product_tokens(const Args p) {
    constexpr int E = 16 / (int)sizeof(T), MATRICES = GATED ? 2 : 1;
    constexpr int AT_ONCE = GROUPS == 1 ? 8 : 4; // pieces under way
    __shared__ f32x4 sums[kTokenWaves][MATRICES * GROUPS][64];
    const int lane = threadIdx.x & 63, quarter = lane >> 4, col = lane & 15;
    const int wave = attn::scalar(threadIdx.x >> 6), waves = blockDim.x >> 6;
    const int n0 = blockIdx.x * 16;
    const char *w[MATRICES], *x[GROUPS];
    bool real[GROUPS];
#pragma unroll
    for (int i = 0; i < MATRICES; ++i)
        w[i] = (const char *)((const T *)p.b[i] + (int64_t)min(n0 + col, p.N - 1) * p.b_l) +
               16 * quarter;
#pragma unroll
    for (int g = 0; g < GROUPS; ++g) {
        real[g] = 16 * g + col < p.M;
        x[g] = (const char *)((const T *)p.a[0] +
                              (int64_t)min(16 * g + col, p.M - 1) * p.a_l) + 16 * quarter;
    }
    f32x4 acc[MATRICES][GROUPS];
#pragma unroll
    for (int i = 0; i < MATRICES; ++i)
#pragma unroll
        for (int g = 0; g < GROUPS; ++g)
            acc[i][g] = f32x4{0.f, 0.f, 0.f, 0.f};
    const int pieces = (p.K + 4 * E - 1) / (4 * E);
    const int end = min(pieces, (wave + 1) * p.split_steps);
    const int units = (p.K + E - 1) / E; // of a row; the last one ends in zeros
    for (int c0 = wave * p.split_steps; c0 < end; c0 += AT_ONCE) {
        u32x4 a[AT_ONCE][MATRICES], b[AT_ONCE][GROUPS];
#pragma unroll
        for (int c = 0; c < AT_ONCE; ++c) {
            const bool here = c0 + c < end && 4 * (c0 + c) + quarter < units;
#pragma unroll
            for (int i = 0; i < MATRICES; ++i) {
                a[c][i] = u32x4{0u, 0u, 0u, 0u};
                if (here) // read once: not kept in the caches
                    a[c][i] = __builtin_nontemporal_load((const u32x4 *)(w[i] + 64 * (c0 + c)));
            }
#pragma unroll
            for (int g = 0; g < GROUPS; ++g) {
                b[c][g] = u32x4{0u, 0u, 0u, 0u};
                if (here && real[g])
                    b[c][g] = *(const u32x4 *)(x[g] + 64 * (c0 + c));
            }
        }
#pragma unroll
        for (int c = 0; c < AT_ONCE; ++c)
#pragma unroll
            for (int g = 0; g < GROUPS; ++g)
#pragma unroll
                for (int i = 0; i < MATRICES; ++i)
                    acc[i][g] = Unit16<T>::mma(a[c][i], b[c][g], acc[i][g]);
    }
#pragma unroll
    for (int i = 0; i < MATRICES; ++i)
#pragma unroll
        for (int g = 0; g < GROUPS; ++g)
            sums[wave][i * GROUPS + g][lane] = acc[i][g];
    __syncthreads();
    // a wave each group: token 16 g + col, weights' rows n .. n + 3
    for (int g = wave; g < GROUPS; g += waves) {
        const int m = 16 * g + col, n = n0 + 4 * quarter;
        f32x4 s[MATRICES];
#pragma unroll
        for (int i = 0; i < MATRICES; ++i) {
            s[i] = sums[0][i * GROUPS + g][lane];
            for (int v = 1; v < waves; ++v)
                s[i] += sums[v][i * GROUPS + g][lane];
        }
        if (m >= p.M)
            continue;
        if constexpr (GATED) {
            if (n < p.out_l)
                put_hidden<T, 4>(p, m, n, s[0], s[1]);
        } else {
            T *to = (T *)p.out[0] + m * p.out_l + n;
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (n + j < p.N)
                    to[j] = (T)s[0][j];
        }
    }
}

template <typename T, bool GATED> int launch_tokens(Args p, hipStream_t stream) {
    const int64_t blocks = (p.out_l > p.N && GATED ? p.out_l + 15 : (int64_t)p.N + 15) / 16;
    const int pieces = (p.K + 64 / (int)sizeof(T) - 1) / (64 / (int)sizeof(T));
    // eight waves or more for each compute unit, of two pieces or more each
    int waves = 1;
    while (waves < kTokenWaves && blocks * waves < 2048 && pieces >= 4 * waves)
        waves *= 2;
    p.split_steps = (pieces + waves - 1) / waves;
    if (p.M <= 16)
        product_tokens<T, GATED, 1><<<dim3((unsigned)blocks), 64 * waves, 0, stream>>>(p);
    else
        product_tokens<T, GATED, 2><<<dim3((unsigned)blocks), 64 * waves, 0, stream>>>(p);
    return hipGetLastError() != hipSuccess;
}

template <typename T> int run_tokens(const Args &p, Kind kind, hipStream_t stream) {
    return kind == kUp ? launch_tokens<T, true>(p, stream) : launch_tokens<T, false>(p, stream);
}

} // namespace ff

#endif
