// rotate.h -- what the rotation kernels share: units of 16 bytes, positions, and the cosines
// and sines of a block's tokens.
#ifndef TORCHMATCH_AMD_ROTATE_H
#define TORCHMATCH_AMD_ROTATE_H

#include "../../include/torchmatch_amd.h"

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace rot {

typedef __bf16 b16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 h16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

template <typename T, int V> struct Unit {
    typedef T type __attribute__((ext_vector_type(V)));
};
template <> struct Unit<__bf16, 8> { using type = b16x8; };
template <> struct Unit<_Float16, 8> { using type = h16x8; };
template <> struct Unit<float, 4> { using type = f32x4; };

// Where tokens stand and by which axis each pair turns.
struct Places {
    const void *pos;
    const float *freqs;
    int64_t pos_b;
    int32_t L, pairs, axes, pos_type;
    int32_t ends[TM_ROTATE_MAX_AXES]; // the first pair past each axis
    float sign;
};

__device__ inline double position(const Places &p, int64_t i) {
    switch (p.pos_type) {
    case TM_POS_F32: return (double)((const float *)p.pos)[i];
    case TM_POS_I32: return (double)((const int32_t *)p.pos)[i];
    default: return (double)((const int64_t *)p.pos)[i];
    }
}

// (cos, sin) of a token's pair, sines times p.sign; row: the token's place in `positions`.  The
// angle is reduced to a fraction of a turn in double precision (positions may be in the hundred
// thousands; a float32 product would be off by 1e-2 there).
template <typename T> __device__ inline float2 turn_of(const Places &p, int64_t row, int pair) {
    int axis = 0;
#pragma unroll
    for (int a = 0; a + 1 < TM_ROTATE_MAX_AXES; ++a)
        axis += a + 1 < p.axes && pair >= p.ends[a];
    const double turns =
        position(p, row + axis) * (double)p.freqs[pair] * 0.15915494309189533577;
    const float r = (float)(turns - rint(turns));
    float c, s;
    if constexpr (sizeof(T) == 4) {
        sincospif(2.f * r, &s, &c);
    } else { // to 2^-20, which 16 bits do not show
        s = __builtin_amdgcn_sinf(r);
        c = __builtin_amdgcn_cosf(r);
    }
    return make_float2(c, p.sign * s);
}

// (cos, sin) of N consecutive pairs, N even, read 16 bytes at a time
template <int N> struct Turns {
    f32x4 w[N / 2];
    __device__ inline explicit Turns(const float2 *from) {
#pragma unroll
        for (int n = 0; n < N / 2; ++n)
            w[n] = ((const f32x4 *)from)[n];
    }
    __device__ inline float2 at(int j) const {
        return make_float2(w[j / 2][2 * (j % 2)], w[j / 2][2 * (j % 2) + 1]);
    }
};

constexpr int kTable = 4096; // (cos, sin) of a block, 32 KB

// The parts of a rotation that have to do with places; not whether x fits.
inline int places(const tm_rotation &r, Places &p) {
    if (r.axes < 1 || r.axes > TM_ROTATE_MAX_AXES || r.pos_type < TM_POS_F32 ||
        r.pos_type > TM_POS_I64)
        return TM_ERR_INVALID_ARGUMENT;
    p.pairs = 0;
    for (int a = 0; a < r.axes; ++a) {
        if (r.sections[a] < 0 || r.sections[a] > r.D)
            return TM_ERR_INVALID_ARGUMENT;
        p.pairs += r.sections[a];
        p.ends[a] = p.pairs;
    }
    if (2 * (int64_t)p.pairs > r.D)
        return TM_ERR_INVALID_ARGUMENT;
    p.pos = r.positions, p.freqs = r.freqs, p.pos_b = r.pos_b;
    p.L = r.L, p.axes = r.axes, p.pos_type = r.pos_type;
    p.sign = r.inverse ? -1.f : 1.f;
    return TM_OK;
}

} // namespace rot

#endif
