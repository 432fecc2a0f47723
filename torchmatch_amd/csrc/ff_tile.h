// ff_tile.h -- matrix products of the feed-forward block on tiles in LDS, and what is done with
// their results before they are written.
//
//     h = act(x G^T) * (x U^T),  y = h D^T                               (rows by rows)
//     dh = dy D -> da, db;  dx = da G + db U                               (rows by columns)
//     dG = da^T x, dU = db^T x, dD = dy^T h                                (columns by columns)
//
// A block has BM x BN of the result.  Tiles of 128 bytes of k go from memory
// straight into LDS, two buffers, one barrier a tile.  (Loads of whole lines run at 133 bytes/ns a compute
// unit, of half lines, tiles of 64 bytes of k, at 38.)  Operands whose rows hold k are read by rows, others
// by transposed reads (attn_tile.h has the tiles' layout), so nothing is transposed in memory.  The
// result's columns lie along a lane's registers; a wave turns them through LDS, 32 rows at a
// time, and writes whole rows of its tile.
//
// Long products, 8192 x 2048 x 5632 bfloat16: y 145 us (1.3 PFLOP/s), dG and dU 353 (1.07), where
// products without loads reach 2.0 to 2.1; waves wait for a third to a half of their time, and a
// block alone on its compute unit has nothing beside a wait.  h with what is saved 405 and dh with da and
// db 250, of which writing 369 and 461 MB is 95 and 100, not hidden either.  float32 is bound by the
// vector work of taking numbers apart: 105 to 133 TFLOP/s of 32768 rows of 256 through 683.
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

// ---- activations ------------------------------------------------------------------

// The activation's value and slope.  16-bit types take the hardware's exponential and reciprocal
// (2^-22), float32 the library's.
template <typename T> __device__ inline float exp_of(float x) {
    return sizeof(T) == 2 ? __builtin_amdgcn_exp2f(x * attn::kLog2e) : expf(x);
}
template <typename T> __device__ inline float over(float x) { // 1 / x
    return sizeof(T) == 2 ? __builtin_amdgcn_rcpf(x) : 1.f / x;
}
template <typename T, int KIND> __device__ inline float2 activate(float a) {
    if constexpr (KIND == TM_SILU) {
        const float s = over<T>(1.f + exp_of<T>(-a)), v = a * s;
        return make_float2(v, fmaf(v, 1.f - s, s));
    } else if constexpr (KIND == TM_RELU) {
        // not a maximum, which loses NaN
        return make_float2(a < 0.f ? 0.f : a, a > 0.f ? 1.f : 0.f);
    } else if constexpr (KIND == TM_GELU) {
        const float cdf = 0.5f * erfcf(-0.70710678118654752440f * a);
        return make_float2(a * cdf, cdf + a * 0.39894228040143267794f * exp_of<T>(-0.5f * a * a));
    } else { // the approximation by tanh
        const float k = 0.79788456080286535588f;
        const float t = tanhf(k * (a + 0.044715f * a * a * a));
        const float half = 0.5f * (1.f + t);
        // its square bounded: past it 1 - t^2 is zero, and infinity times that no number
        return make_float2(a * half, half + 0.5f * a * (1.f - t * t) * k *
                                                (1.f + fminf(3.f * 0.044715f * a * a, 1e30f)));
    }
}
// f(j, the activation) for j < V, the choice outside the loop
template <typename T, int V, typename F>
__device__ inline void activate_all(int kind, F f) {
    const auto all = [&](auto act) {
#pragma unroll
        for (int j = 0; j < V; ++j)
            f(j, act);
    };
    if (kind == TM_SILU)
        all([](float a) { return activate<T, TM_SILU>(a); });
    else if (kind == TM_RELU)
        all([](float a) { return activate<T, TM_RELU>(a); });
    else if (kind == TM_GELU)
        all([](float a) { return activate<T, TM_GELU>(a); });
    else
        all([](float a) { return activate<T, TM_GELU_TANH>(a); });
}

// ---- tiles ------------------------------------------------------------------------

template <typename T> constexpr int kStep = 128 / (int)sizeof(T); // k a tile: whole lines of memory

// What units of 16 rows of 128 bytes are permuted by, for reads of row lane % 16, unit lane / 16
__device__ inline int swz16(int row) {
    return (row >> 1 & 1) << 2 | ((row >> 2 ^ row >> 3) & 1) << 1 | (row >> 3 & 1);
}

// One operand's tile, ROWS x kStep, brought by NT threads.  STRIDED: a row for each k.  HALF: HALF rows of one
// matrix, HALF of another, in turn (0: one matrix).
template <typename T, int ROWS, bool STRIDED, int NT, int HALF> struct Feed {
    static constexpr int BK = kStep<T>, E = 16 / (int)sizeof(T);
    using L = attn::Tile<T, STRIDED ? ROWS : BK>;
    static constexpr int SIZE = (STRIDED ? BK : ROWS) * L::U; // units
    static constexpr int N = SIZE / NT, STEP = NT / L::U;
    static_assert(SIZE % NT == 0 && NT % L::U == 0 && L::U == L::U0);

    static constexpr int READS = STRIDED ? 2 : 1; // an operand's (16-bit types)

    uint32_t off[N]; // bytes from the tile's first element, its k aside

    // A row's units are permuted by it.  Rows of 128 bytes: lanes 0-3, 12-15, 20-23, 24-27 of a read take
    // their 256 bytes at once, so fours of rows at one unit and at its neighbour are to differ.
    __device__ static inline int swz(int row) {
        return sizeof(T) == 2 && !STRIDED ? swz16(row) : L::swz(row);
    }

    // left: rows (columns) from the tile's first on
    __device__ inline void start(int tid, int64_t stride, int left) {
        const int row = tid / L::U, pos = tid % L::U;
        const uint32_t bytes = (uint32_t)stride * (uint32_t)sizeof(T);
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const int r = row + n * STEP, u = pos ^ swz(r);
            if constexpr (STRIDED) {
                off[n] = (uint32_t)r * bytes + 16u * min(u, (left - 1) / E);
            } else {
                const int real = HALF ? r / (2 * HALF + !HALF) * HALF + r % (HALF + !HALF) : r;
                off[n] = (uint32_t)min(real, left - 1) * bytes + 16u * u;
            }
        }
    }
    // whether load n is of the second matrix: the same for a whole wave
    __device__ static inline bool of_second(int tid, int n) {
        return HALF && attn::scalar((tid / L::U + n * STEP) / (HALF + !HALF)) & 1;
    }
    // from: the tile's first element; second: of the other matrix; mask: 0 for its first 16 bytes
    // over and over
    __device__ inline void load(u32x4 *t, const char *from, const char *second, int tid,
                                uint32_t mask) const {
        u32x4 *to = t + attn::scalar(tid & ~63);
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const char *s = of_second(tid, n) ? second : from;
            uint32_t at = off[n] & mask;
            asm("" : "+v"(at)); // so that it stays 32 bits beside a scalar address
            __builtin_amdgcn_global_load_lds(
                (const __attribute__((address_space(1))) void *)(s + at),
                (__attribute__((address_space(3))) void *)(to + n * NT), 16, 0, 0);
        }
    }
    // the last tile, of which `left` k are there: zeros past them
    __device__ inline void load_last(u32x4 *t, const char *from, const char *second, int tid,
                                     int left) const {
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const char *s = of_second(tid, n) ? second : from;
            const int r = tid / L::U + n * STEP;
            const bool real = STRIDED ? r < left : (tid % L::U ^ swz(r)) * E < left;
            u32x4 x = {0u, 0u, 0u, 0u};
            if (real)
                x = *(const u32x4 *)(s + off[n]);
            t[tid + n * NT] = x;
        }
    }

    // Where a lane reads: a byte offset from which all reads differ by an exclusive or with a constant
    // and a constant number of rows.
    __device__ static inline uint32_t lane_at(int lane) {
        if constexpr (sizeof(T) == 2 && !STRIDED) {
            return 16u * ((lane & 15) * L::U + ((lane >> 4) ^ swz(lane & 15)));
        } else if constexpr (sizeof(T) == 2) {
            const int d = 4 * (lane & 3);
            return 16u * L::at(8 * (lane >> 4) + ((lane & 15) >> 2), d >> 3) + 2u * (d & 7);
        } else if constexpr (!STRIDED) {
            return L::row_lane(lane);
        } else {
            return 16u * L::at(8 * (lane >> 5), (lane & 31) / E) + 4u * (lane & 3);
        }
    }
    // An operand of run c: 16-bit types row (column) 16 rb + lane % 16, k 32 c + 8 (lane / 16) + 0 .. 7;
    // float32 row (column) 32 rb + lane % 32, k 16 c + 8 (lane / 32) + 0 .. 7
    __device__ static inline x8<T> operand(const u32x4 *t, uint32_t at, int rb, int c) {
        if constexpr (sizeof(T) == 2 && !STRIDED) {
            return *(const x8<T> *)((const char *)t + rb * 16 * L::U * 16 + (at ^ (64u * c)));
        } else if constexpr (sizeof(T) == 2) {
            // the transposed read: each 16 lanes load 4 rows of 16 elements (4 a lane) and
            // each lane gets one column of them
            const char *from = (const char *)t + 32 * c * L::U * 16;
            x8<T> r;
#pragma unroll
            for (int jj = 0; jj < 2; ++jj) {
                const char *p = from + 4 * jj * L::U * 16 + (at ^ (32u * rb + 16u * jj));
                const attn::s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                    (__attribute__((address_space(3))) attn::s16x4 *)p);
                const attn::x4<T> y = __builtin_bit_cast(attn::x4<T>, x);
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    r[4 * jj + j] = y[j];
            }
            return r;
        } else if constexpr (!STRIDED) {
            return L::row8(t, at, 32 * rb, c);
        } else {
            const char *from = (const char *)t + 16 * c * L::U * 16;
            x8<T> r;
#pragma unroll
            for (int j = 0; j < 8; ++j)
                r[j] = *(const float *)(from + j * L::U * 16 +
                                        (at ^ (16u * (8 * rb ^ L::swz(j)))));
            return r;
        }
    }
};

// ---- products ---------------------------------------------------------------------

// The matrix cores' products: SIDE x SIDE of the result over K indices.  Of products alone, sides of
// 16 run at 2000 TFLOP/s and of 32 at 1880.
template <typename T> struct Core {
    static constexpr int SIDE = sizeof(T) == 2 ? 16 : 32, K = sizeof(T) == 2 ? 32 : 16;
    using Sum = float __attribute__((ext_vector_type(SIDE * SIDE / 64)));
};
__device__ inline f32x4 mma(attn::b16x8 a, attn::b16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ inline f32x4 mma(attn::h16x8 a, attn::h16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// float32 numbers as sums of three bfloat16 ones of 8 bits each, exactly: six products of these,
// at sixteen times the rate of float32 ones, leave out 2^-24 of |y x| at most, with
// either sign.  Infinite numbers become NaN.
struct Parts {
    u32x4 hi, mid, lo; // eight bfloat16 each
    __device__ inline void set(f32x8 x) {
        typedef float f32x2 __attribute__((ext_vector_type(2)));
        typedef __bf16 b16x2 __attribute__((ext_vector_type(2)));
        const auto pair = [](f32x2 v) {
            return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, b16x2));
        };
        const auto left = [](f32x2 v, uint32_t of) {
            return f32x2{v[0] - __uint_as_float(of << 16), v[1] - __uint_as_float(of & 0xffff0000u)};
        };
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            f32x2 v = {x[2 * j], x[2 * j + 1]};
            hi[j] = pair(v);
            v = left(v, hi[j]);
            mid[j] = pair(v);
            lo[j] = pair(left(v, mid[j]));
        }
    }
};
// An operand as the products take it.
template <typename T> struct Operand {
    x8<T> x;
    __device__ inline void set(x8<T> v) { x = v; }
    __device__ inline void made_here() {}
};
template <> struct Operand<float> : Parts {
    // not after the next branch, away from the products that it is to run beside
    __device__ inline void made_here() { asm volatile("" : "+v"(hi), "+v"(mid), "+v"(lo)); }
};

// c[i][j] += y[i] x[j] over a run of k
template <typename T, int NB, int MB>
__device__ inline void multiply(const Operand<T> (&y)[NB], const Operand<T> (&x)[MB],
                                typename Core<T>::Sum (&c)[NB][MB]) {
    if constexpr (sizeof(T) == 4) {
        const auto all = [&](u32x4 Parts::*u, u32x4 Parts::*v) {
#pragma unroll
            for (int j = 0; j < MB; ++j)
#pragma unroll
                for (int i = 0; i < NB; ++i)
                    c[i][j] = mma32(__builtin_bit_cast(attn::b16x8, y[i].*u),
                                    __builtin_bit_cast(attn::b16x8, x[j].*v), c[i][j]);
        };
        all(&Parts::hi, &Parts::lo); // the smallest first
        all(&Parts::lo, &Parts::hi);
        all(&Parts::mid, &Parts::mid);
        all(&Parts::hi, &Parts::mid);
        all(&Parts::mid, &Parts::hi);
        all(&Parts::hi, &Parts::hi);
    } else {
#pragma unroll
        for (int j = 0; j < MB; ++j)
#pragma unroll
            for (int i = 0; i < NB; ++i)
                c[i][j] = mma(y[i].x, x[j].x, c[i][j]);
    }
}

// ---- results ----------------------------------------------------------------------

template <int V> using fv = float __attribute__((ext_vector_type(V)));

// V floats as T, in units of up to 16 bytes
template <typename T, int V> __device__ inline void put(T *to, fv<V> x) {
    constexpr int N = sizeof(T) == 4 ? 4 : V;
    typedef T U __attribute__((ext_vector_type(N)));
#pragma unroll
    for (int k = 0; k < V; k += N) {
        U y;
#pragma unroll
        for (int j = 0; j < N; ++j)
            y[j] = (T)x[k + j];
        *(U *)(to + k) = y;
    }
}

// a and b as they are saved: float32, or its first 24 bits (truncated: what a gradient then is off
// by, 2^-15, is far below the rounding of the gradients to 16 bits), the upper 16 in a plane
// each and the next eight of both in a third.
__device__ inline uint32_t bytes(uint32_t hi, uint32_t lo, uint32_t which) {
    return __builtin_amdgcn_perm(hi, lo, which); // bytes 0 - 3 of lo, 4 - 7 of hi, 12: zero
}
template <typename T, int V>
__device__ inline void save(const Args &p, int64_t at, fv<V> a, fv<V> b) {
    if constexpr (sizeof(T) == 4) {
        put<float, V>((float *)p.saved[0] + at, a);
        put<float, V>((float *)p.saved[1] + at, b);
    } else {
        typedef uint32_t U __attribute__((ext_vector_type(V / 2)));
        U x, y, z;
#pragma unroll
        for (int j = 0; j < V / 2; ++j) {
            const uint32_t a0 = __float_as_uint(a[2 * j]), a1 = __float_as_uint(a[2 * j + 1]);
            const uint32_t b0 = __float_as_uint(b[2 * j]), b1 = __float_as_uint(b[2 * j + 1]);
            x[j] = bytes(a1, a0, 0x07060302);
            y[j] = bytes(b1, b0, 0x07060302);
            z[j] = bytes(bytes(a1, b1, 0x0c0c0501), bytes(a0, b0, 0x0c0c0501), 0x05040100);
        }
        *(U *)((uint16_t *)p.saved[0] + at) = x;
        *(U *)((uint16_t *)p.saved[1] + at) = y;
        *(U *)((uint16_t *)p.saved[2] + at) = z;
    }
}
template <typename T> struct Saved { // 8 of them, as they lie in memory
    u32x4 u[sizeof(T) == 4 ? 4 : 3];
    __device__ inline void load(const Args &p, int64_t at) {
#pragma unroll
        for (int n = 0; n < (sizeof(T) == 4 ? 4 : 3); ++n)
            u[n] = sizeof(T) == 4 ? ((const u32x4 *)((const float *)p.saved[n / 2] + at))[n % 2]
                                  : *(const u32x4 *)((const uint16_t *)p.saved[n] + at);
    }
    __device__ inline void give(f32x8 &a, f32x8 &b) const {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            if constexpr (sizeof(T) == 4) {
                a[j] = __uint_as_float(u[j / 4][j % 4]);
                b[j] = __uint_as_float(u[2 + j / 4][j % 4]);
            } else {
                const uint32_t x = u[0][j / 2], y = u[1][j / 2], z = u[2][j / 2];
                a[j] = __uint_as_float(bytes(x, z, j % 2 ? 0x0706030c : 0x0504010c));
                b[j] = __uint_as_float(bytes(y, z, j % 2 ? 0x0706020c : 0x0504000c));
            }
        }
    }
};

// The power of two that half precision holds gradients of the hidden features times (they are as
// small as the loss makes them, and lose bits below 2^-14): what brings the largest |dy| to 1 .. 2, if
// that is up; where it brings a gradient past the range, the largest that does not.  So none is
// infinite and none loses bits that would not without it.
constexpr float kMostHalf = 65504.f;
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
        int up = m > 0.f ? max(0, 1 - __builtin_amdgcn_frexp_expf(m)) : 0;
        const uint32_t past = p.past ? *p.past : 0u;
        if (past) {
            const float most = __uint_as_float(past);
            const int by = __builtin_amdgcn_frexp_expf(most) - 16; // to 2^15 .. 2^16
            up -= __builtin_ldexpf(most, -by) > kMostHalf ? by + 1 : by;
        }
        return up;
    }
    return 0;
}

// One row's 8 results from column n on.
template <typename T>
__device__ inline void put_row(const Args &p, int batch, int64_t m, int n, f32x8 x) {
    T *to = (T *)p.out[batch] + m * p.out_l + n;
    if (p.wide && n + 8 <= p.N) {
        put<T, 8>(to, x);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (n + j < p.N)
                to[j] = (T)x[j];
    }
}

// h, and a and b where they are saved; zeros past the hidden features
template <typename T, int V>
__device__ inline void put_hidden(const Args &p, int64_t m, int n, fv<V> a, fv<V> b) {
    fv<V> h;
    activate_all<T, V>(p.activation, [&](int j, auto act) { h[j] = act(a[j]).x * b[j]; });
    if (n + V > p.N) {
#pragma unroll
        for (int j = 0; j < V; ++j)
            if (n + j >= p.N)
                h[j] = a[j] = b[j] = 0.f;
    }
    const int64_t at = m * p.out_l + n;
    if (p.saved[0])
        save<T, V>(p, at, a, b);
    put<T, V>((T *)p.out[0] + at, h);
}

// The gradients of a and b from that of h (half precision: times 2^up); what was saved past the
// hidden features is zero, dh there anything.  most: raised to the largest finite one.
template <typename T>
__device__ inline void put_grads(const Args &p, int64_t m, int n, f32x8 dh, const Saved<T> &kept,
                                 int up, float &most) {
    const int64_t at = m * p.out_l + n;
    f32x8 a, b, da, db;
    kept.give(a, b);
    if constexpr (__is_same(T, _Float16))
        dh *= __builtin_ldexpf(1.f, up);
    activate_all<T, 8>(p.activation, [&](int j, auto act) {
        const float2 v = act(a[j]);
        da[j] = dh[j] * b[j] * v.y;
        db[j] = dh[j] * v.x;
    });
    if (n + 8 > p.N) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (n + j >= p.N)
                da[j] = db[j] = 0.f;
    }
    if constexpr (__is_same(T, _Float16)) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float u = fabsf(da[j]), v = fabsf(db[j]);
            most = u < attn::kInf ? fmaxf(most, u) : most;
            most = v < attn::kInf ? fmaxf(most, v) : most;
        }
    }
    put<T, 8>((T *)p.da + at, da);
    put<T, 8>((T *)p.db + at, db);
}

// ---- the product ------------------------------------------------------------------

// The order of a tile's instructions: PRODUCTS a run of k, spread over them the READS of the
// next run (an operand takes the place of one that was multiplied) and, in the first run from its
// first quarter on, the LOADS of the next tile.  Sent for at once, the loads hold up every wave, later
// they are late; reads that end earlier need more registers than there are.
template <int RUNS, int PRODUCTS, int READS, int LOADS> struct Order {
    template <int R, int I> __device__ static inline void one() {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0); // matrix products
        constexpr int reads = READS * (I + 1) / PRODUCTS - READS * I / PRODUCTS;
        if constexpr (reads > 0)
            __builtin_amdgcn_sched_group_barrier(0x100, reads, 0); // reads of LDS
        constexpr int F = PRODUCTS / 4, P = PRODUCTS - F, J = R * PRODUCTS + I - F;
        constexpr int loads = J >= 0 && J < P ? LOADS * (J + 1) / P - LOADS * J / P : 0;
        if constexpr (loads > 0)
            __builtin_amdgcn_sched_group_barrier(0x020, loads, 0); // loads from memory
        if constexpr (I + 1 < PRODUCTS)
            one<R, I + 1>();
        else if constexpr (R + 1 < RUNS)
            one<R + 1, 0>();
    }
    __device__ static inline void runs() { one<0, 0>(); }
};

// float32: a run's numbers are read and taken apart while the run before is multiplied.
template <int RUNS, int PRODUCTS, int READS, int LOADS> struct OrderParts {
    template <int R, int I> __device__ static inline void one() {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0); // matrix products
        if constexpr (I < 4)
            __builtin_amdgcn_sched_group_barrier(0x100, READS / 4, 0); // reads of LDS
        else
            __builtin_amdgcn_sched_group_barrier(0x002, 8, 0); // taking apart
        if constexpr (R == 0 && I >= 4 && I < 4 + LOADS)
            __builtin_amdgcn_sched_group_barrier(0x020, 1, 0); // loads from memory
        if constexpr (I + 1 < PRODUCTS)
            one<R, I + 1>();
        else if constexpr (R + 1 < RUNS)
            one<R + 1, 0>();
    }
    __device__ static inline void runs() { one<0, 0>(); }
};

template <Kind K> struct Shape { // which operands are strided
    static constexpr bool kA = K == kWeights, kB = K != kUp && K != kDown;
};

// Meets the block's other waves when all but LATER of this one's loads have arrived and its reads and
// writes of LDS are done.  (__syncthreads() would wait for every load, those of later tiles too.)
template <int LATER> __device__ inline void meet() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(LATER) : "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// A block's waves by rows and columns, what each has of the result, in 32 x 32, and the tiles in LDS.
// Large tiles: one block of eight waves a compute unit, small ones: two of four.  Where there is no
// second block to hide the waits, four tiles do (128 x 2048 through 5632: 56 -> 49 us).  The
// large gated one's waves have 64 columns of either projection, so that rows of 128 bytes are written.
// 64 x 64 where a product is small: shorter steps, more of the card (512 x 256 from 1376 of k in
// float32 77 -> 36 us, in bfloat16 17 -> 11; 2048 x 688 from 256 26 -> 17 and 12 -> 8).
template <Kind K, int SIZE> struct Size {
    static constexpr int WM = 2, WN = SIZE == kLarge ? 4 : 2, MB = SIZE == kLarge ? 4 : 2, NB = 2;
    static constexpr int TILES = SIZE == kDeep ? 4 : 2;
};
template <Kind K> struct Size<K, kTiny> {
    static constexpr int WM = 2, WN = 2, MB = 1, NB = 1, TILES = 4;
};
template <> struct Size<kUp, kLarge> {
    static constexpr int WM = 4, WN = 2, MB = 2, NB = 4, TILES = 2;
};

// The first p.whole tiles are a block's each; the k of every other one is split over p.splits blocks, which
// leave their sums in p.part as they lie in their registers.  JOIN: adds these, in order, and
// does with them what is done with a whole tile's; a block of one wave for 32 rows of one
// wave's (as many splits' sums come by fast only where many ask for them).
template <typename T, Kind KIND, int SIZE, bool JOIN>
__global__ __launch_bounds__((JOIN ? 64 : 64 * Size<KIND, SIZE>::WM * Size<KIND, SIZE>::WN),
                             (SIZE == kDeep || JOIN ? 1 : 2)) void
product(const Args p) {
    constexpr bool HALF_GRADS = KIND == kHidden && __is_same(T, _Float16);
    if constexpr (HALF_GRADS)
        if (p.past && !*p.past) // a second time only where the first one's scale was too large
            return;
    using Z = Size<KIND, SIZE>;
    constexpr int MB = Z::MB, NB = Z::NB, BM = 32 * MB * Z::WM, BN = 32 * NB * Z::WN;
    constexpr int PARTS32 = 32 / Core<T>::SIDE; // of the matrix cores' products in 32 rows
    constexpr int M = PARTS32 * MB, N = PARTS32 * NB;
    using Sum = typename Core<T>::Sum;
    constexpr int NT = 64 * Z::WM * Z::WN, BK = kStep<T>;
    constexpr bool GATED = KIND == kUp;
    constexpr int TN = GATED ? BN / 2 : BN; // columns of the result a block
    constexpr int HALF = 16 * NB; // gated: columns of either projection a wave
    using FA = Feed<T, BM, Shape<KIND>::kA, NT, 0>;
    using FB = Feed<T, BN, Shape<KIND>::kB, NT, GATED ? HALF : 0>;
    // Apart, so that the compiler sees that a tile on its way is not the one that is read.
    constexpr int TILES = Z::TILES, LOADS = FA::N + FB::N; // a thread's, of a tile
    constexpr int ROW = 8 * NB, PER = FA::SIZE / (32 * ROW); // see the end
    __shared__ u32x4 a0[JOIN ? 32 * ROW : FA::SIZE], a1[JOIN ? 1 : FA::SIZE],
        b0[JOIN ? 1 : FB::SIZE], b1[JOIN ? 1 : FB::SIZE];
    constexpr bool MORE = TILES > 2 && !JOIN;
    __shared__ u32x4 a2[MORE ? FA::SIZE : 1], a3[MORE ? FA::SIZE : 1], b2[MORE ? FB::SIZE : 1],
        b3[MORE ? FB::SIZE : 1];

    constexpr int WAVES = Z::WM * Z::WN;
    const int lane = threadIdx.x & 63, half = lane >> 5;
    const int wave = JOIN ? (int)blockIdx.x / MB % WAVES : attn::scalar(threadIdx.x >> 6);
    const int tid = 64 * wave + lane, wm = wave / Z::WN, wn = wave % Z::WN;
    const int mt = (p.M + BM - 1) / BM, nt = (p.N + TN - 1) / TN;
    // tiles in bands of 8 rows of tiles, a run of them an XCD: those which share operands meet
    // in its L2
    int id, split = 0, tail = -1;
    if (JOIN) {
        tail = blockIdx.x / (MB * WAVES);
        id = p.whole + tail;
    } else if ((int)blockIdx.x < p.whole) {
        id = attn::xcd_order(blockIdx.x, p.whole);
    } else {
        id = attn::xcd_order(blockIdx.x - p.whole, gridDim.x - p.whole);
        split = id % p.splits;
        tail = id / p.splits;
        id = p.whole + tail;
    }
    const int batch = id / (mt * nt);
    id -= batch * mt * nt;
    const int band = id / (8 * nt), in_band = id - band * 8 * nt;
    const int rows = min(8, mt - 8 * band);
    const int m0 = (8 * band + in_band % rows) * BM, n0 = in_band / rows * TN;

    FA fa;
    FB fb;
    fa.start(tid, p.a_l, p.M - m0);
    fb.start(tid, p.b_l, p.N - n0);
    const int spk = (p.K + BK - 1) / BK; // steps a segment
    const int steps = spk * p.segments, s0 = split * p.split_steps;
    const int s1 = tail < 0 ? steps : min(s0 + p.split_steps, steps);
    uint32_t at_a = FA::lane_at(lane), at_b = FB::lane_at(lane);

    // the tiles' first elements at k = 0, of either segment; gated: of gate and up
    const int64_t off_a = Shape<KIND>::kA ? m0 : m0 * p.a_l, step_a = Shape<KIND>::kA ? p.a_l : 1;
    const int64_t off_b = Shape<KIND>::kB ? n0 : n0 * p.b_l, step_b = Shape<KIND>::kB ? p.b_l : 1;
    const T *from_a0 = (const T *)p.a[batch] + off_a, *from_a1 = (const T *)p.a[1] + off_a;
    const T *from_b0 = (const T *)p.b[batch] + off_b, *from_b1 = (const T *)p.b[1] + off_b;

    const auto is_whole = [&](int s) { return (s < spk ? s + 1 : s + 1 - spk) * BK <= p.K; };
    // sends for tile s where there is one and it is whole; else for what nobody reads (the first 16
    // bytes over and over), so that there is no branch among the products
    const auto fetch = [&](int s, u32x4 *ta, u32x4 *tb) {
        const bool here = s < s1 && is_whole(s);
        const int seg = here && s >= spk ? 1 : 0, k = here ? (s - seg * spk) * BK : 0;
        const T *pa = (KIND == kInput && seg ? from_a1 : from_a0) + k * step_a;
        const T *pb = (KIND == kInput && seg ? from_b1 : from_b0) + k * step_b;
        const T *pu = GATED ? from_b1 + k : nullptr;
        const uint32_t mask = here ? ~0u : 0u;
        fa.load(ta, (const char *)pa, nullptr, tid, mask);
        fb.load(tb, (const char *)pb, (const char *)pu, tid, mask);
    };
    // the last tile of a segment, if it is not whole
    const auto fetch_rest = [&](int s, u32x4 *ta, u32x4 *tb) {
        if (s >= s1 || is_whole(s))
            return;
        const int seg = s >= spk ? 1 : 0, k = (s - seg * spk) * BK;
        const T *pa = (KIND == kInput && seg ? from_a1 : from_a0) + k * step_a;
        const T *pb = (KIND == kInput && seg ? from_b1 : from_b0) + k * step_b;
        const T *pu = GATED ? from_b1 + k : nullptr;
        attn::arrived(); // what fetch() sent for is not to land on it
        fa.load_last(ta, (const char *)pa, nullptr, tid, p.K - k);
        fb.load_last(tb, (const char *)pb, (const char *)pu, tid, p.K - k);
    };

    Sum acc[N][M];
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
        for (int j = 0; j < M; ++j)
            acc[i][j] = Sum{};
    // operands of two runs of k
    Operand<T> x0[M], y0[N], x1[M], y1[N];
    const auto read = [&](const u32x4 *ta, const u32x4 *tb, int c, Operand<T>(&x)[M],
                          Operand<T>(&y)[N]) {
#pragma unroll
        for (int i = 0; i < N; ++i)
            y[i].set(FB::operand(tb, at_b, N * wn + i, c));
#pragma unroll
        for (int j = 0; j < M; ++j)
            x[j].set(FA::operand(ta, at_a, M * wm + j, c));
    };
    // One tile: while a run of k is multiplied the next one is read, in the first the last of the
    // tile before, so that the matrix cores wait neither for LDS nor for the barrier between
    // tiles.
    static_assert(BK == 2 * Core<T>::K);
    const auto tile = [&](const u32x4 *ta, const u32x4 *tb) {
        asm("" : "+v"(at_a), "+v"(at_b)); // addresses a constant apart are not all held
        read(ta, tb, 0, x0, y0);
        multiply<T>(y1, x1, acc);
        read(ta, tb, 1, x1, y1);
        multiply<T>(y0, x0, acc);
#pragma unroll
        for (int j = 0; j < M; ++j)
            x1[j].made_here();
#pragma unroll
        for (int i = 0; i < N; ++i)
            y1[i].made_here();
    };
    // tile s; its place's neighbour, which is free, takes the last one that is on its way.  Each
    // fetch() is LOADS loads, so that counts tell which have arrived.
    const auto step = [&](int s, u32x4 *ta, u32x4 *tb, u32x4 *next_a, u32x4 *next_b) {
        fetch(s + TILES - 1, next_a, next_b);
        tile(ta, tb);
        if constexpr (sizeof(T) == 2)
            Order<2, N * M, N * FB::READS + M * FA::READS, FA::N + FB::N>::runs();
        else
            OrderParts<2, N * M * 6, 2 * (N + M), FA::N + FB::N>::runs();
        fetch_rest(s + TILES - 1, next_a, next_b);
        meet<(TILES - 2) * LOADS>();
    };
#pragma unroll
    for (int j = 0; j < M; ++j)
        x1[j] = {};
#pragma unroll
    for (int i = 0; i < N; ++i)
        y1[i] = {};
    if (!JOIN && s0 < s1) {
        const auto first = [&](int s, u32x4 *ta, u32x4 *tb) {
            fetch(s, ta, tb);
            fetch_rest(s, ta, tb);
        };
        first(s0, a0, b0);
        if constexpr (TILES > 2) {
            first(s0 + 1, a1, b1);
            first(s0 + 2, a2, b2);
        }
        meet<(TILES - 2) * LOADS>();
    }
    for (int s = JOIN ? s1 : s0; s < s1; s += TILES) {
        if constexpr (TILES == 2) {
            step(s, a0, b0, a1, b1);
            if (s + 1 < s1)
                step(s + 1, a1, b1, a0, b0);
        } else {
            step(s, a0, b0, a3, b3);
            if (s + 1 < s1)
                step(s + 1, a1, b1, a0, b0);
            if (s + 2 < s1)
                step(s + 2, a2, b2, a1, b1);
            if (s + 3 < s1)
                step(s + 3, a3, b3, a2, b2);
        }
    }
    if constexpr (!JOIN)
        multiply<T>(y1, x1, acc);
    // 32 rows are PARTS32 sums of each column, fours of results all told
    constexpr int PER_SUM = Core<T>::SIDE * Core<T>::SIDE / 256, QUADS = PARTS32 * PER_SUM;
    // where a split tile's sums lie, 16 bytes of each thread in turn
    constexpr int SUMS = 16 * NB * MB * NT * 4; // bytes of a tile's
    const int tails =
        JOIN ? (int)gridDim.x / (MB * WAVES) : (int)(gridDim.x - p.whole) / p.splits;
    const uint32_t mine = 16u * tid;
    char *sums = (char *)p.part + ((int64_t)split * tails + tail) * SUMS;
    const int first = JOIN ? (int)blockIdx.x % MB : 0, last = JOIN ? first + 1 : MB;
    if constexpr (JOIN) {
        sums += first * (N * QUADS * 16 * NT);
#pragma unroll 4
        for (int n = 0; n < p.splits; ++n) {
            const char *from = sums + (int64_t)n * tails * SUMS;
#pragma unroll
            for (int i = 0; i < N; ++i)
#pragma unroll
                for (int q = 0; q < QUADS; ++q) {
                    const f32x4 x = *(const f32x4 *)(from + mine);
                    from += 16 * NT;
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        acc[i][q / PER_SUM][4 * (q % PER_SUM) + e] += x[e];
                }
        }
    }
    const bool leave = !JOIN && tail >= 0;

    const int up = KIND == kHidden || KIND == kInput || KIND == kWeights ? grad_up<T>(p, lane) : 0;
    const float down = __builtin_ldexpf(1.f, -up);
    attn::arrived(); // the last fetches, of nothing, are not to land on what follows
    // A wave's rows, 32 at a time, through LDS: what was a lane's column becomes rows.  Units of 16
    // bytes are permuted by the row, so that rows meet other banks.
    __syncthreads();
    // ROW units a row, PER waves a buffer
    constexpr int FLIP = ROW < 16 ? ROW - 1 : 15;
    static_assert(FA::SIZE == FB::SIZE && 4 * PER >= WAVES);
    const int place = JOIN ? 0 : wave / PER;
    f32x4 *turn = (f32x4 *)(place == 0 ? a0 : place == 1 ? a1 : place == 2 ? b0 : b1) +
                  (JOIN ? 0 : wave % PER * 32 * ROW);
    // a lane has 8 columns of PARTS rows of 32
    constexpr int LANES = (GATED ? HALF : 32 * NB) / 8, PARTS = LANES / 2;
    const int row = lane / LANES, col = lane % LANES * 8;
    const int n = n0 + (GATED ? HALF : 32 * NB) * wn + col;
    const bool here = n < (GATED || KIND == kHidden ? p.out_l : (int64_t)p.N);
    const int mw = m0 + 32 * (MB * wm + first) + row;
    Saved<T> kept[KIND == kHidden ? PARTS : 1]; // sent for 32 rows ahead
    if constexpr (KIND == kHidden) {
#pragma unroll
        for (int k = 0; k < PARTS; ++k) {
            const int m = mw + 64 / LANES * k;
            if (m < p.M && here && !leave)
                kept[k].load(p, m * p.out_l + n);
        }
    }
    float most = 0.f; // of a lane's da and db
    // one copy of what follows: the sums move up in the registers
#pragma unroll 1
    for (int j = first; j < last; ++j) {
        attn::wave_fence();
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
            for (int q = 0; q < QUADS; ++q) {
                const Sum &c = acc[i][q / PER_SUM];
                constexpr int S = Core<T>::SIDE;
                const int e = 4 * (q % PER_SUM);
                const f32x4 x = {c[e], c[e + 1], c[e + 2], c[e + 3]};
                if (leave) {
                    *(f32x4 *)(sums + mine) = x;
                    sums += 16 * NT;
                    continue;
                }
                // its row, and its four columns
                const int r = S * (q / PER_SUM) + lane % S;
                const int unit = S / 4 * i + (S == 16 ? lane >> 4 : 2 * q + half);
                turn[r * ROW + (unit ^ (r & FLIP))] = x;
            }
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
            for (int k = 0; k + PARTS32 < M; ++k)
                acc[i][k] = acc[i][k + PARTS32];
        if (leave)
            continue;
        attn::wave_fence();
        const auto read8 = [&](int r, int c) {
            const f32x4 lo = turn[r * ROW + ((c >> 2) ^ (r & FLIP))];
            const f32x4 hi = turn[r * ROW + (((c >> 2) + 1) ^ (r & FLIP))];
            return (f32x8){lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
        };
#pragma unroll
        for (int k = 0; k < PARTS; ++k) {
            const int r = row + 64 / LANES * k, m = mw + 32 * (j - first) + 64 / LANES * k;
            if (m < p.M && here) {
                if constexpr (GATED) {
                    put_hidden<T, 8>(p, m, n, read8(r, col), read8(r, col + HALF));
                } else if constexpr (KIND == kHidden) {
                    put_grads<T>(p, m, n, read8(r, col), kept[k], up, most);
                    if (j + 1 < last && m + 32 < p.M)
                        kept[k].load(p, (m + 32) * p.out_l + n);
                } else {
                    put_row<T>(p, batch, m, n, read8(r, col) * down);
                }
            }
        }
    }
    if constexpr (HALF_GRADS)
        if (most > kMostHalf && !p.past) // a maximum: in any order the same
            atomicMax(p.past_out, __float_as_uint(most));
}

template <typename T, Kind KIND, int SIZE> int launch(const Args &p, hipStream_t stream) {
    using Z = Size<KIND, SIZE>;
    constexpr int BM = 32 * Z::MB * Z::WM, TN = (KIND == kUp ? 16 : 32) * Z::NB * Z::WN;
    const int64_t tiles = (int64_t)((p.M + BM - 1) / BM) * ((p.N + TN - 1) / TN) * p.batches;
    const int64_t blocks = p.whole + (tiles - p.whole) * p.splits;
    if (!blocks)
        return 0;
    product<T, KIND, SIZE, false><<<dim3((unsigned)blocks), 64 * Z::WM * Z::WN, 0, stream>>>(p);
    if (tiles > p.whole)
        product<T, KIND, SIZE == kDeep ? kSmall : SIZE, true> // their sums lie alike
            <<<dim3((unsigned)(tiles - p.whole) * Z::MB * Z::WM * Z::WN), 64, 0, stream>>>(p);
    return hipGetLastError() != hipSuccess;
}

template <typename T, Kind KIND> int launch_size(const Args &p, int size, hipStream_t stream) {
    if constexpr (sizeof(T) == 2) // float32's operands do not fit in registers with large tiles
        if (size == kLarge)
            return launch<T, KIND, kLarge>(p, stream);
    return size == kTiny   ? launch<T, KIND, kTiny>(p, stream)
           : size == kDeep ? launch<T, KIND, kDeep>(p, stream)
                           : launch<T, KIND, kSmall>(p, stream);
}

template <typename T> int run(const Args &p, Kind kind, int size, hipStream_t stream) {
    switch (kind) {
    case kUp: return launch_size<T, kUp>(p, size, stream);
    case kDown: return launch_size<T, kDown>(p, size, stream);
    case kHidden: return launch_size<T, kHidden>(p, size, stream);
    case kInput: return launch_size<T, kInput>(p, size, stream);
    default: return launch_size<T, kWeights>(p, size, stream);
    }
}

} // namespace ff

#endif
