// dropout.hip -- dropout whose mask is never stored.
//
// Element i (in row-major order) stays where word i % 4 of the ten-round Philox generator (Salmon,
// Moraes, Dror, Shaw: "Parallel random numbers: as easy as 1, 2, 3", 2011) of the counter
// (i / 4, offset) under the key `seed` is at least round(p 2^32):
//     y = residual + x / (1 - p) where it stays, residual elsewhere
// The mask is the same whatever the type, so the gradient is the same call on dy without a residual.
//
// Bound by memory: x and the residual are read once, y is written once.  A thread takes 16 bytes at
// a time; a round of the generator is two 32 x 32 -> 64 bit products and two exclusive ors of three for
// four elements, which hide behind the memory: 16 x 2047 x 4099 half-precision elements 93 us, 5.8
// TB/s; 8192 x 2048 bfloat16 with a residual 17.5 us (5.8), without 14.9 (4.5, short).
#include "../../include/torchmatch_amd.h"

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <cmath>

namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

struct DropArgs {
    const void *x, *residual;
    void *out;
    const int64_t *seed_at; // or null: `seed`
    uint64_t seed, offset;
    int64_t count;
    uint32_t threshold;
    int32_t none; // nothing stays
    float scale;
};

__device__ inline u32x4 philox(uint64_t at, uint64_t offset, uint64_t seed) {
    uint32_t c0 = (uint32_t)at, c1 = (uint32_t)(at >> 32);
    uint32_t c2 = (uint32_t)offset, c3 = (uint32_t)(offset >> 32);
    uint32_t k0 = (uint32_t)seed, k1 = (uint32_t)(seed >> 32);
#pragma unroll
    for (int n = 0; n < 10; ++n) {
        const uint64_t m0 = (uint64_t)c0 * 0xD2511F53u, m1 = (uint64_t)c2 * 0xCD9E8D57u;
        c0 = (uint32_t)(m1 >> 32) ^ c1 ^ k0;
        c2 = (uint32_t)(m0 >> 32) ^ c3 ^ k1;
        c1 = (uint32_t)m1;
        c3 = (uint32_t)m0;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    return u32x4{c0, c1, c2, c3};
}

// V elements a thread, a multiple of 4; WIDE: read and written whole
template <typename T, int V, bool WIDE, bool RESIDUAL>
__global__ __launch_bounds__(256) void drop(const DropArgs p) {
    typedef T U __attribute__((ext_vector_type(V)));
    const uint64_t seed = p.seed_at ? (uint64_t)*p.seed_at : p.seed;
    const int64_t step = (int64_t)gridDim.x * 256 * V;
    for (int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * V; i < p.count; i += step) {
        const bool whole = WIDE && i + V <= p.count;
        U x, r;
        if (whole) {
            x = *(const U *)((const T *)p.x + i);
            if (RESIDUAL)
                r = *(const U *)((const T *)p.residual + i);
        } else {
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const int64_t e = min(i + j, p.count - 1);
                x[j] = ((const T *)p.x)[e];
                if (RESIDUAL)
                    r[j] = ((const T *)p.residual)[e];
            }
        }
        U y;
#pragma unroll
        for (int n = 0; n < V / 4; ++n) {
            const u32x4 word = philox((uint64_t)i / 4 + n, p.offset, seed);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int e = 4 * n + j;
                const bool stays = word[j] >= p.threshold && !p.none;
                float kept = (float)x[e] * p.scale;
                // a float32 product in every variant: else some take it and the conversion to half
                // precision as one instruction that rounds once, and bits go by the alignment
                asm("" : "+v"(kept));
                kept = stays ? kept : 0.f;
                y[e] = (T)(RESIDUAL ? (float)r[e] + kept : kept);
            }
        }
        if (whole) {
            *(U *)((T *)p.out + i) = y;
        } else {
#pragma unroll
            for (int j = 0; j < V; ++j)
                if (i + j < p.count)
                    ((T *)p.out)[i + j] = y[j];
        }
    }
}

template <typename T, bool WIDE> void launch(const DropArgs &p, unsigned blocks, hipStream_t s) {
    constexpr int V = 16 / sizeof(T);
    p.residual ? drop<T, V, WIDE, true><<<dim3(blocks), 256, 0, s>>>(p)
               : drop<T, V, WIDE, false><<<dim3(blocks), 256, 0, s>>>(p);
}

} // namespace

extern "C" int tm_dropout(const void *x, const void *residual, void *out, int64_t count,
                          int32_t dtype, double p, uint64_t seed, const int64_t *seed_at,
                          uint64_t offset, hipStream_t stream) {
    if (count < 0 || dtype < TM_BF16 || dtype > TM_F32 || !(p >= 0. && p <= 1.))
        return TM_ERR_INVALID_ARGUMENT;
    if (!count)
        return TM_OK;
    if (!x || !out)
        return TM_ERR_INVALID_ARGUMENT;
    DropArgs a = {};
    a.x = x, a.residual = residual, a.out = out, a.count = count;
    a.seed = seed, a.seed_at = seed_at, a.offset = offset;
    const double threshold = std::nearbyint(p * 0x1p32);
    a.none = threshold >= 0x1p32;
    a.threshold = a.none ? 0 : (uint32_t)threshold;
    a.scale = a.none ? 0.f : (float)(1. / (1. - p));
    const bool wide = !(((uintptr_t)x | (uintptr_t)residual | (uintptr_t)out) % 16);
    const int64_t per = 256 * (dtype == TM_F32 ? 4 : 8);
    const int64_t most = 1 << 20; // longer calls go round
    const unsigned blocks = (unsigned)std::min(most, (count + per - 1) / per);
    if (dtype == TM_BF16)
        wide ? launch<__bf16, true>(a, blocks, stream) : launch<__bf16, false>(a, blocks, stream);
    else if (dtype == TM_F16)
        wide ? launch<_Float16, true>(a, blocks, stream)
             : launch<_Float16, false>(a, blocks, stream);
    else
        wide ? launch<float, true>(a, blocks, stream) : launch<float, false>(a, blocks, stream);
    return hipGetLastError() == hipSuccess ? TM_OK : TM_ERR_LAUNCH;
}
