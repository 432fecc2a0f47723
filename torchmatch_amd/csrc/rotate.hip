// rotate.hip -- pairs of features turned by positions on several axes.
//
// Pair p of a token turns by the angle  pos[axis(p)] * freq[p]:
//     (x1, x2) -> (x1 cos - x2 sin, x2 cos + x1 sin)
// and back by the opposite angle, which is the gradient.  Bound by memory: x is read once
// and written once.  A block takes a few tokens; it computes their cosines and sines once
// into LDS, whatever the number of heads, and then streams the heads through.
//
// The angle is reduced to a fraction of a turn in double precision (positions may be in the
// hundred thousands; a float32 product would be off by 1e-2 there), a few operations per
// token and pair that the heads share.
#include "../../include/torchmatch_amd.h"

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>

namespace {

typedef __bf16 b16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 h16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

template <typename T, int V> struct Unit;
template <> struct Unit<__bf16, 8> { using type = b16x8; };
template <> struct Unit<_Float16, 8> { using type = h16x8; };
template <> struct Unit<float, 4> { using type = f32x4; };

struct RotateArgs {
    const void *x, *pos;
    const float *freqs;
    void *out;
    int64_t x_b, x_l, x_h, pos_b, tokens;
    int32_t L, H, D, pairs, axes, pos_type, interleaved, per_block;
    int32_t ends[TM_ROTATE_MAX_AXES]; // the first pair past each axis
    float sign;
};

__device__ inline double position(const RotateArgs &p, int64_t i) {
    switch (p.pos_type) {
    case TM_POS_F32: return (double)((const float *)p.pos)[i];
    case TM_POS_I32: return (double)((const int32_t *)p.pos)[i];
    default: return (double)((const int64_t *)p.pos)[i];
    }
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

// V: elements a load (16 bytes, or 1 where strides, sizes or addresses do not allow it)
template <typename T, int V>
__global__ __launch_bounds__(256) void rotate_pairs(const RotateArgs p) {
    __shared__ __attribute__((aligned(16))) float2 table[kTable];
    const int64_t first = (int64_t)blockIdx.x * p.per_block;
    const int tokens = (int)min((int64_t)p.per_block, p.tokens - first);
    for (int i = threadIdx.x; i < tokens * p.pairs; i += 256) {
        const int pair = i % p.pairs;
        const int64_t t = first + i / p.pairs;
        int axis = 0;
#pragma unroll
        for (int a = 0; a + 1 < TM_ROTATE_MAX_AXES; ++a)
            axis += a + 1 < p.axes && pair >= p.ends[a];
        const double turns = position(p, t / p.L * p.pos_b + t % p.L * p.axes + axis) *
                             (double)p.freqs[pair] * 0.15915494309189533577;
        const float r = (float)(turns - rint(turns));
        float c, s;
        if constexpr (sizeof(T) == 4) {
            sincospif(2.f * r, &s, &c);
        } else { // to 2^-20, which 16 bits do not show
            s = __builtin_amdgcn_sinf(r);
            c = __builtin_amdgcn_cosf(r);
        }
        table[i] = make_float2(c, p.sign * s);
    }
    __syncthreads();

    // items of a head: V pairs (in halves), V / 2 pairs (interleaved), V features passed on
    const int step = p.interleaved ? (V + 1) / 2 : V;
    const int turned = p.pairs / step, per_head = turned + (p.D - 2 * p.pairs) / V;
    const int per_token = per_head * p.H;
    const T *x = (const T *)p.x;
    T *out = (T *)p.out;
    for (int i = threadIdx.x; i < tokens * per_token; i += 256) {
        const int token = i / per_token, in_token = i % per_token;
        const int head = in_token / per_head, item = in_token % per_head;
        const int64_t t = first + token;
        const T *src = x + t / p.L * p.x_b + t % p.L * p.x_l + head * p.x_h;
        T *dst = out + (t * p.H + head) * p.D;
        const float2 *cs = table + token * p.pairs + item * step;
        if constexpr (V == 1) {
            if (item >= turned) {
                const int e = 2 * p.pairs + item - turned;
                dst[e] = src[e];
            } else {
                const int e1 = p.interleaved ? 2 * item : item;
                const int e2 = p.interleaved ? e1 + 1 : p.pairs + item;
                const float a = (float)src[e1], b = (float)src[e2];
                dst[e1] = (T)(a * cs->x - b * cs->y);
                dst[e2] = (T)(b * cs->x + a * cs->y);
            }
        } else {
            using U = typename Unit<T, V>::type;
            if (item >= turned) {
                const int e = 2 * p.pairs + (item - turned) * V;
                *(U *)(dst + e) = *(const U *)(src + e);
            } else if (p.interleaved) {
                const U a = *(const U *)(src + item * V);
                U y;
                Turns<V / 2> turns(cs);
#pragma unroll
                for (int j = 0; j < V / 2; ++j) {
                    const float2 w = turns.at(j);
                    const float u = (float)a[2 * j], v = (float)a[2 * j + 1];
                    y[2 * j] = (T)(u * w.x - v * w.y);
                    y[2 * j + 1] = (T)(v * w.x + u * w.y);
                }
                *(U *)(dst + item * V) = y;
            } else {
                const U a = *(const U *)(src + item * V);
                const U b = *(const U *)(src + p.pairs + item * V);
                U y, z;
                Turns<V> turns(cs);
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const float2 w = turns.at(j);
                    const float u = (float)a[j], v = (float)b[j];
                    y[j] = (T)(u * w.x - v * w.y);
                    z[j] = (T)(v * w.x + u * w.y);
                }
                *(U *)(dst + item * V) = y;
                *(U *)(dst + p.pairs + item * V) = z;
            }
        }
    }
}

template <typename T, int V> void launch(const RotateArgs &p, unsigned blocks, hipStream_t s) {
    rotate_pairs<T, V><<<dim3(blocks), 256, 0, s>>>(p);
}

} // namespace

extern "C" int tm_rotate(const tm_rotation *r, void *out, hipStream_t stream) {
    if (!r || r->B < 0 || r->L < 0 || r->H < 0 || r->D < 1 || r->axes < 1 ||
        r->axes > TM_ROTATE_MAX_AXES || r->dtype < TM_BF16 || r->dtype > TM_F32 ||
        r->pos_type < TM_POS_F32 || r->pos_type > TM_POS_I64)
        return TM_ERR_INVALID_ARGUMENT;
    RotateArgs p = {};
    for (int a = 0; a < r->axes; ++a) {
        if (r->sections[a] < 0 || r->sections[a] > r->D)
            return TM_ERR_INVALID_ARGUMENT;
        p.pairs += r->sections[a];
        p.ends[a] = p.pairs;
    }
    if (2 * (int64_t)p.pairs > r->D)
        return TM_ERR_INVALID_ARGUMENT;
    if (p.pairs > kTable || r->D > 2 * kTable || (int64_t)r->H * r->D > (1 << 24))
        return TM_ERR_UNSUPPORTED_SHAPE;
    p.tokens = (int64_t)r->B * r->L;
    if (!p.tokens || !r->H)
        return TM_OK;
    if (!r->x || !out || !r->positions || (p.pairs && !r->freqs))
        return TM_ERR_INVALID_ARGUMENT;
    p.x = r->x, p.pos = r->positions, p.freqs = r->freqs, p.out = out;
    p.x_b = r->x_b, p.x_l = r->x_l, p.x_h = r->x_h, p.pos_b = r->pos_b;
    p.L = r->L, p.H = r->H, p.D = r->D, p.axes = r->axes, p.pos_type = r->pos_type;
    p.interleaved = r->interleaved ? 1 : 0;
    p.sign = r->inverse ? -1.f : 1.f;

    const int size = r->dtype == TM_F32 ? 4 : 2, unit = 16 / size;
    const bool wide = !(((uintptr_t)r->x | (uintptr_t)out) % 16) && !(r->x_b % unit) &&
                      !(r->x_l % unit) && !(r->x_h % unit) && !(r->D % unit) &&
                      !(p.pairs % (p.interleaved ? unit / 2 : unit));
    const int v = wide ? unit : 1;
    const int step = p.interleaved ? (v + 1) / 2 : v;
    const int64_t per_token = (int64_t)(p.pairs / step + (p.D - 2 * p.pairs) / v) * p.H;
    // four items a thread where there are tokens enough, as long as that leaves four blocks
    // for each compute unit; the table's size bounds it too
    int64_t per = std::max<int64_t>(1, 1024 / per_token);
    per = std::min(per, std::max<int64_t>(1, p.tokens / 1024));
    // and a launch takes less than 2^32 threads, 2^24 blocks
    const int64_t most = (1 << 24) - 1;
    per = std::max(per, (p.tokens + most - 1) / most);
    if (p.pairs)
        per = std::min<int64_t>(per, kTable / p.pairs);
    p.per_block = (int32_t)per;
    const int64_t blocks = (p.tokens + per - 1) / per;
    if (blocks > most)
        return TM_ERR_UNSUPPORTED_SHAPE;
    const unsigned n = (unsigned)blocks;
    if (r->dtype == TM_BF16)
        wide ? launch<__bf16, 8>(p, n, stream) : launch<__bf16, 1>(p, n, stream);
    else if (r->dtype == TM_F16)
        wide ? launch<_Float16, 8>(p, n, stream) : launch<_Float16, 1>(p, n, stream);
    else
        wide ? launch<float, 4>(p, n, stream) : launch<float, 1>(p, n, stream);
    return hipGetLastError() == hipSuccess ? TM_OK : TM_ERR_LAUNCH;
}
