// ff_tokens.h -- the feed-forward block's forward products where there are few rows, or so little all
// told that tiles would leave the card idle: reading the weights bounds them, or a few steps' latency.
//
// A block has 16 rows of the weights (of gate and of up) and 16 or 32 of x, its waves a part of k each, so
// that a small product still fills the card; their sums meet in LDS, in order.  A wave brings whole
// lines of 16 rows and of x into its own part of LDS, two or three pieces ahead of its 16 x 16
// products, and meets the others at the end only.  (Operands straight from memory, 64 bytes of
// each row a load: 26 us for a token of 2048 through 5632 in bfloat16, 77 for 15 of 4096 through 11264,
// in place of 15.6, 4.4 TB/s, and 56, 4.9.)  The contraction
// takes its indices in the order in which lanes hold them, for both operands alike.
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

// 16 rows of 128 bytes, brought straight into LDS by one wave, whole lines of memory; units of 16
// bytes are permuted by the row, so that a unit of each row is read without bank conflicts.
struct Rows16 {
    uint32_t off[2]; // bytes from the first row
    int unit[2];
    __device__ inline void start(int lane, int64_t row_bytes, int rows) {
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            const int row = (lane >> 3) + 8 * n;
            unit[n] = (lane & 7) ^ swz16(row);
            off[n] = (uint32_t)min(row, rows - 1) * (uint32_t)row_bytes;
        }
    }
    // piece: which 8 units of the rows; past the last of `units` that one again
    __device__ inline void load(u32x4 *t, const char *from, int piece, int units) const {
#pragma unroll
        for (int n = 0; n < 2; ++n)
            __builtin_amdgcn_global_load_lds(
                (const __attribute__((address_space(1))) void *)(
                    from + off[n] + 16u * (uint32_t)min(8 * piece + unit[n], units - 1)),
                (__attribute__((address_space(3))) void *)(t + 64 * n), 16, 0, 0);
    }
    // row lane % 16, unit 4 half + lane / 16
    __device__ static inline u32x4 operand(const u32x4 *t, int lane, int half) {
        const int row = lane & 15;
        return t[8 * row + ((4 * half + (lane >> 4)) ^ swz16(row))];
    }
};

// WAVES share k; split_steps: pieces of 128 bytes of k a wave
template <typename T, bool GATED, int GROUPS, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void product_tokens(const Args p) {
    constexpr int E = 16 / (int)sizeof(T), MATRICES = GATED ? 2 : 1, PER = MATRICES + GROUPS;
    constexpr int SLOTS = GATED ? 2 : 3, LOADS = 2 * PER; // pieces on their way, their loads
    // Apart, so that the compiler sees that what is on its way is not what is read.
    __shared__ u32x4 s0[WAVES][PER * 128], s1[WAVES][PER * 128],
        s2[SLOTS > 2 ? WAVES : 1][SLOTS > 2 ? PER * 128 : 1];
    const int lane = threadIdx.x & 63, quarter = lane >> 4, col = lane & 15;
    const int wave = attn::scalar(threadIdx.x >> 6);
    const int n0 = blockIdx.x * 16, m0 = blockIdx.y * 16 * GROUPS, rows = p.M - m0;
    Rows16 w, x[GROUPS];
    w.start(lane, p.b_l * (int)sizeof(T), p.N - n0);
#pragma unroll
    for (int g = 0; g < GROUPS; ++g)
        x[g].start(lane, p.a_l * (int)sizeof(T), max(rows - 16 * g, 1));
    const int units = (p.K + E - 1) / E, pieces = (units + 7) / 8;
    const int c0 = wave * p.split_steps, c1 = min(pieces, c0 + p.split_steps);

    const auto fetch = [&](int c, u32x4 *t) {
        // past the end: the last piece again, which nobody reads
        c = min(c, pieces - 1);
#pragma unroll
        for (int i = 0; i < MATRICES; ++i)
            w.load(t + 128 * i, (const char *)((const T *)p.b[i] + n0 * p.b_l), c, units);
#pragma unroll
        for (int g = 0; g < GROUPS; ++g)
            x[g].load(t + 128 * (MATRICES + g), (const char *)((const T *)p.a[0] +
                      (int64_t)(m0 + min(16 * g, rows - 1)) * p.a_l), c, units);
    };
    f32x4 acc[MATRICES][GROUPS];
#pragma unroll
    for (int i = 0; i < MATRICES; ++i)
#pragma unroll
        for (int g = 0; g < GROUPS; ++g)
            acc[i][g] = f32x4{0.f, 0.f, 0.f, 0.f};
    const auto step = [&](int c, u32x4 *t) {
        attn::arrived<(SLOTS - 1) * LOADS>();
        u32x4 v[2][PER];
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < PER; ++i)
                v[h][i] = Rows16::operand(t + 128 * i, lane, h);
        if (8 * c + 8 > units) { // zeros past the end
#pragma unroll
            for (int h = 0; h < 2; ++h)
                if (8 * c + 4 * h + quarter >= units)
#pragma unroll
                    for (int i = 0; i < PER; ++i)
                        v[h][i] = u32x4{0u, 0u, 0u, 0u};
        }
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int g = 0; g < GROUPS; ++g)
#pragma unroll
                for (int i = 0; i < MATRICES; ++i)
                    acc[i][g] = Unit16<T>::mma(v[h][i], v[h][MATRICES + g], acc[i][g]);
        // what was read has arrived in registers: its place is free
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        fetch(c + SLOTS, t);
    };
    if (c0 < c1) {
        fetch(c0, s0[wave]);
        fetch(c0 + 1, s1[wave]);
        if constexpr (SLOTS > 2)
            fetch(c0 + 2, s2[wave]);
        for (int c = c0; c < c1; c += SLOTS) {
            step(c, s0[wave]);
            if (c + 1 < c1)
                step(c + 1, s1[wave]);
            if constexpr (SLOTS > 2)
                if (c + 2 < c1)
                    step(c + 2, s2[wave]);
        }
        attn::arrived();
    }
    __syncthreads();
    f32x4(*sums)[64] = (f32x4(*)[64])s0; // [wave][MATRICES * GROUPS][64]
    static_assert(MATRICES * GROUPS * 64 <= PER * 128);
#pragma unroll
    for (int i = 0; i < MATRICES; ++i)
#pragma unroll
        for (int g = 0; g < GROUPS; ++g)
            sums[(wave * MATRICES + i) * GROUPS + g][lane] = acc[i][g];
    __syncthreads();
    // a wave each group: token 16 g + col, weights' rows n .. n + 3
    for (int g = wave; g < GROUPS; g += WAVES) {
        const int m = m0 + 16 * g + col, n = n0 + 4 * quarter;
        f32x4 s[MATRICES];
#pragma unroll
        for (int i = 0; i < MATRICES; ++i) {
            s[i] = sums[i * GROUPS + g][lane];
#pragma unroll
            for (int v = 1; v < WAVES; ++v)
                s[i] += sums[(v * MATRICES + i) * GROUPS + g][lane];
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

template <typename T, bool GATED, int GROUPS> void launch_waves(Args p, hipStream_t stream) {
    const unsigned blocks = (unsigned)(((GATED ? p.out_l : (int64_t)p.N) + 15) / 16);
    const unsigned groups = (unsigned)((p.M + 16 * GROUPS - 1) / (16 * GROUPS));
    const int pieces = (int)(((int64_t)p.K * (int)sizeof(T) + 127) / 128);
    // few blocks: more waves each, so that enough is on its way (LDS has room for that once)
    if (blocks * groups <= 256 && pieces > 4) {
        p.split_steps = (pieces + 7) / 8;
        product_tokens<T, GATED, GROUPS, 8><<<dim3(blocks, groups), 512, 0, stream>>>(p);
        return;
    }
    p.split_steps = (pieces + 3) / 4;
    product_tokens<T, GATED, GROUPS, 4><<<dim3(blocks, groups), 256, 0, stream>>>(p);
}

template <typename T, bool GATED> int launch_tokens(const Args &p, hipStream_t stream) {
    if (tokens_rows(p.M, p.N) == 16)
        launch_waves<T, GATED, 1>(p, stream);
    else
        launch_waves<T, GATED, 2>(p, stream);
    return hipGetLastError() != hipSuccess;
}

template <typename T> int run_tokens(const Args &p, Kind kind, hipStream_t stream) {
    return kind == kUp ? launch_tokens<T, true>(p, stream) : launch_tokens<T, false>(p, stream);
}

} // namespace ff

#endif
