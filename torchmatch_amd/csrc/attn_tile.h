// attn_tile.h -- the pieces the attention kernels share: matrix-core steps on
// 32 x 32 tiles, tiles in LDS that are read by rows and by columns without
// bank conflicts, and the scores' cap, bias and masks.
//
// Register layouts of one wave (lane l, half h = l / 32):
//   operand   8 elements of row l % 32, contraction indices 8h .. 8h + 7
//   result    16 floats of column l % 32, element i is row 8(i/4) + 4h + i%4
// A contraction may take its indices in any order as long as both operands
// agree, so elements 8t .. 8t + 7 of a result serve, as they lie, as an operand
// of the next product over rows 16t + 8(j/4) + 4h + j%4 (j = 0..7): scores go
// from one product to the next without leaving the registers.
#ifndef TORCHMATCH_AMD_ATTN_TILE_H
#define TORCHMATCH_AMD_ATTN_TILE_H

#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "attn.h"

namespace attn {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 b16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 b16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 h16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 h16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));

constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLn2 = 0.69314718055994530942f;
constexpr float kInf = __builtin_inff();

template <typename T> struct Vec;
template <> struct Vec<__bf16> {
    using x4 = b16x4;
    using x8 = b16x8;
};
template <> struct Vec<_Float16> {
    using x4 = h16x4;
    using x8 = h16x8;
};
template <> struct Vec<float> {
    using x4 = f32x4;
    using x8 = f32x8;
};
template <typename T> using x4 = typename Vec<T>::x4;
template <typename T> using x8 = typename Vec<T>::x8;

// c += a b over 16 contraction indices
__device__ inline f32x16 mma32(b16x8 a, b16x8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ inline f32x16 mma32(h16x8 a, h16x8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
// float32: the step takes two indices, one per half; element i of both halves
__device__ inline f32x16 mma32(f32x8 a, f32x8 b, f32x16 c) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
        c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[i], b[i], c, 0, 0, 0);
    return c;
}

template <typename T> __device__ inline x8<T> pack8(const f32x16 &c, int t) {
    x8<T> r;
#pragma unroll
    for (int j = 0; j < 8; ++j)
        r[j] = (T)c[8 * t + j];
    return r;
}

// A tile of ROWS x DP elements in LDS, in units of 16 bytes.  Rows are padded
// to a power of two (U units) and a row's units are permuted by an exclusive
// or with a function of the row, so that both ways of reading spread over all
// banks: 8 consecutive rows at one unit (row operands), and 4 consecutive rows
// over 4 aligned units (column operands).
template <typename T, int DP> struct Tile {
    static constexpr int E = 16 / (int)sizeof(T); // elements a unit
    static constexpr int U0 = DP / E;
    static constexpr int U = U0 <= 4 ? 4 : U0 <= 8 ? 8 : U0 <= 16 ? 16 : U0 <= 32 ? 32 : 64;

    __device__ static inline int swz(int row) {
        if constexpr (U == 4)
            return (row >> 2) & 3;
        else if constexpr (U == 8)
            return (((row >> 1) & 1) << 2) | ((row >> 2) & 3);
        else
            return ((row & 3) << 2) | ((row >> 2) & 3);
    }
    __device__ static inline int at(int row, int unit) { return row * U + (unit ^ swz(row)); }

    // Where a lane reads: a byte offset from which every read of one kind differs by an
    // exclusive or with a constant and a constant number of rows, so that few registers
    // hold addresses.  Rows r0 are multiples of 16, over which swz() repeats.
    __device__ static inline uint32_t row_lane(int lane) {
        const int row = lane & 31, half = lane >> 5;
        return 16u * at(row, sizeof(T) == 2 ? half : 2 * half);
    }
    __device__ static inline uint32_t col_lane(int lane) {
        if constexpr (sizeof(T) == 2) {
            const int d = (lane & 16) + 4 * (lane & 3);
            return 16u * at(4 * (lane >> 5) + ((lane & 15) >> 2), d >> 3) + 2u * (d & 7);
        } else {
            return 16u * at(4 * (lane >> 5), (lane & 31) / E) + 4u * (lane & 3);
        }
    }

    // row operand: row r0 + lane % 32, elements 16 c + 8 (lane / 32) + 0 .. 7
    __device__ static inline x8<T> row8(const u32x4 *t, uint32_t row, int r0, int c) {
        const char *from = (const char *)t + r0 * U * 16;
        if constexpr (sizeof(T) == 2) {
            return *(const x8<T> *)(from + (row ^ (32u * c)));
        } else {
            const f32x4 lo = *(const f32x4 *)(from + (row ^ (64u * c)));
            const f32x4 hi = *(const f32x4 *)(from + (row ^ (64u * c + 16u)));
            return (x8<T>){lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
        }
    }

    // writes what row8() reads
    __device__ static inline void put8(u32x4 *t, uint32_t row, int r0, int c, x8<T> x) {
        char *to = (char *)t + r0 * U * 16;
        if constexpr (sizeof(T) == 2) {
            *(x8<T> *)(to + (row ^ (32u * c))) = x;
        } else {
            *(f32x4 *)(to + (row ^ (64u * c))) = (f32x4){x[0], x[1], x[2], x[3]};
            *(f32x4 *)(to + (row ^ (64u * c + 16u))) = (f32x4){x[4], x[5], x[6], x[7]};
        }
    }

    // column operand: column 32 db + lane % 32, rows r0 + 8(j/4) + 4(lane / 32) + j%4
    __device__ static inline x8<T> col8(const u32x4 *t, uint32_t col, int r0, int db) {
        const char *from = (const char *)t + r0 * U * 16;
        x8<T> r;
        if constexpr (sizeof(T) == 2) {
            // the transposed read: each 16 lanes load 4 rows of 16 elements (4 a
            // lane) and each lane gets one column of them
#pragma unroll
            for (int jj = 0; jj < 2; ++jj) {
                const char *at = from + 8 * jj * U * 16 + (col ^ (64u * db + 32u * jj));
                const s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                    (__attribute__((address_space(3))) s16x4 *)at);
                const x4<T> y = __builtin_bit_cast(x4<T>, x);
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    r[4 * jj + j] = y[j];
            }
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int row = 8 * (j >> 2) + (j & 3);
                r[j] = *(const float *)(from + row * U * 16 +
                                        (col ^ (16u * (8 * db ^ swz(row)))));
            }
        }
        return r;
    }
};

// A tile brought from memory straight into LDS by NT threads, without passing through
// registers.  A wave's 64 units land next to each other, so the permutation of a row's units
// is made on the side of the addresses: a scalar row and 32 bits a lane.  Features past the
// d real ones are not brought: pad() zeroes their place once.  arrived() before the barrier
// that lets others read.
template <typename T, int DP, int ROWS, int NT> struct Bring {
    using L = Tile<T, DP>;
    static constexpr int N = ROWS * L::U / NT, STEP = NT / L::U; // rows from load to load
    static_assert(ROWS * L::U % NT == 0 && NT % L::U == 0);

    // rows row0 + 0 .. ROWS - 1 of a matrix of `rows` > row0 rows; those past the last repeat it
    __device__ static inline void load(u32x4 *t, const T *base, int64_t stride, int row0, int rows,
                                       int d, int tid) {
        const int row = tid / L::U, pos = tid % L::U;
        const int left = rows - row0;
        u32x4 *to = t + __builtin_amdgcn_readfirstlane(tid & ~63);
        const char *from = (const char *)(base + (int64_t)row0 * stride);
        const uint32_t bytes = (uint32_t)stride * (uint32_t)sizeof(T);
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const int u = pos ^ L::swz(row + n * STEP);
            const char *s = from;
            uint32_t off;
            if (left >= ROWS) {
                s += (int64_t)n * STEP * stride * (int)sizeof(T);
                off = (uint32_t)row * bytes + 16u * u;
            } else {
                off = (uint32_t)max(min(row + n * STEP, left - 1), 0) * bytes + 16u * u;
            }
            if ((L::U == L::U0 && d == DP) || u * L::E < d)
                __builtin_amdgcn_global_load_lds(
                    (const __attribute__((address_space(1))) void *)(s + off),
                    (__attribute__((address_space(3))) void *)(to + n * NT), 16, 0, 0);
        }
    }
    __device__ static inline void pad(u32x4 *t, int d, int tid) {
        if (d < DP) {
#pragma unroll
            for (int n = 0; n < N; ++n)
                t[tid + n * NT] = u32x4{0u, 0u, 0u, 0u};
        }
    }
    // zeros in the rows that nobody may see: past `rows`, or of a negative document
    __device__ static inline void clear(u32x4 *t, int row0, int rows, bool by_doc, const int *docs,
                                        int tid) {
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const int r = tid / L::U + n * STEP;
            if (row0 + r >= rows || (by_doc && docs[r] < 0))
                t[tid + n * NT] = u32x4{0u, 0u, 0u, 0u};
        }
    }
};

// 64 words from memory into LDS by one wave, a word each lane
__device__ inline void bring_word(void *to, const void *from) {
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)from,
                                     (__attribute__((address_space(3))) void *)to, 4, 0, 0);
}

// Waits until at most LATER of this wave's loads are not there yet; they arrive in order.
template <int LATER = 0> __device__ inline void arrived() {
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(LATER) : "memory");
}

// What is read from LDS into the result x has been read past this point.
__device__ inline void made_here(f32x16 &x) { asm volatile("" : "+v"(x)::"memory"); }

// LDS writes of a wave are seen by its later reads as they are: both go through in order.
// This keeps the compiler from moving them.
__device__ inline void wave_fence() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// 8 elements of a row in memory (a row operand that stays in registers)
template <typename T>
__device__ inline x8<T> global8(const T *row, int e, int d, bool valid) {
    x8<T> r;
#pragma unroll
    for (int j = 0; j < 8; ++j)
        r[j] = (T)0.f;
    if constexpr (sizeof(T) == 2) {
        if (valid && e < d)
            r = *(const x8<T> *)(row + e);
    } else {
        if (valid && e < d) {
            const f32x4 a = *(const f32x4 *)(row + e);
#pragma unroll
            for (int j = 0; j < 4; ++j)
                r[j] = a[j];
        }
        if (valid && e + 4 < d) {
            const f32x4 a = *(const f32x4 *)(row + e + 4);
#pragma unroll
            for (int j = 0; j < 4; ++j)
                r[4 + j] = a[j];
        }
    }
    return r;
}

// How many leading keys query i of batch row b may see, masks by document aside.
struct Limits {
    int length, offset, prefix, causal;
    __device__ inline Limits(const Args &p, int b) {
        length = p.lengths ? min(max(p.lengths[b], 0), p.Lk) : p.Lk;
        offset = length - p.Lq;
        prefix = p.prefix ? min(max(p.prefix[b], 0), length) : 0;
        causal = p.causal;
    }
    __device__ inline int of(int i) const {
        return causal ? min(length, max(max(i + offset + 1, prefix), 0)) : length;
    }
};

// The cap, cap tanh(scale x / cap) in base 2.  For 16-bit inputs by exp and a reciprocal: with
// r = 1 / (e^(2 y) + 1), tanh y = 1 - 2 r and its derivative is 4 r (1 - r).  The error, 2e-7 of
// the cap, is absolute, and what it is added to is a score: caps up to 1024 stay below
// the rounding of float16 weights.  float32 products leave the time for the library's tanh.
template <typename T> struct Cap {
    static constexpr bool kByExp = sizeof(T) == 2;
    float in, out;
    __device__ inline Cap(const Args &p)
        : in(p.scale / p.cap * (kByExp ? 2.f * kLog2e : 1.f)), out(p.cap * kLog2e) {}
    // r, or tanh
    __device__ inline float part(float x) const {
        if constexpr (kByExp)
            return __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(x * in) + 1.f);
        else
            return tanhf(x * in);
    }
    // the score's distance from share()
    __device__ inline float add(float part, float to) const {
        return fmaf(kByExp ? -2.f * out : out, part, to);
    }
    __device__ static inline float share(const Args &p) { return kByExp ? p.cap * kLog2e : 0.f; }
    // a quarter of the derivative
    __device__ inline float slope(float part) const {
        return kByExp ? fmaf(-part, part, part) : fmaf(-0.25f * part, part, 0.25f);
    }
};

__device__ inline f32x4 away(f32x4 a, float b) {
    return (f32x4){fabsf(a[0] - b), fabsf(a[1] - b), fabsf(a[2] - b), fabsf(a[3] - b)};
}

// One lane's query against results of k q^T, 32 keys a block: the scores in base 2, what the
// lane may see.
// SIDE: there may be documents or positions (without them a kernel needs fewer registers).
template <typename T, bool SIDE> struct QueryLane {
    int limit, doc, at;
    float slope, pos[3];

    __device__ inline QueryLane(const Args &p, const Limits &lim, int b, int head, int i) {
        const bool real = i < p.Lq;
        limit = real ? lim.of(i) : 0;
        doc = SIDE && p.q_docs && real ? p.q_docs[(int64_t)b * p.Lq + i] : -1;
        at = i + lim.offset;
        slope = p.slopes ? p.slopes[head] * kLog2e : 0.f;
        pos[0] = pos[1] = pos[2] = 0.f;
        if (SIDE && p.q_pos && real)
#pragma unroll
            for (int a = 0; a < 3; ++a)
                if (a < p.axes)
                    pos[a] = p.q_pos[((int64_t)b * p.Lq + i) * p.axes + a];
    }

    // What scores must be multiplied with after score(): plain products wait for the
    // exponential, which takes the factor along.
    __device__ static inline float factor(const Args &p) {
        return p.cap > 0.f || p.slopes || !(p.scale > 0.f) ? 1.f : p.scale * kLog2e;
    }
    // s: products with keys k0 ..; to scores times log2 e but for factor().  k_pos: the block's
    // positions in LDS, `axis` apart.
    __device__ inline void score(const Args &p, f32x16 &s, int k0, int half, const float *k_pos,
                                 int axis) const {
        if (p.cap > 0.f) {
            const Cap<T> cap(p);
            const float from = Cap<T>::share(p);
#pragma unroll
            for (int i = 0; i < 16; ++i)
                s[i] = cap.add(cap.part(s[i]), from);
        } else if (p.slopes || !(p.scale > 0.f)) {
            const float m = p.scale * kLog2e;
#pragma unroll
            for (int i = 0; i < 16; ++i)
                s[i] *= m;
        }
        if (p.slopes) {
#pragma unroll
            for (int n = 0; n < 4; ++n) {
                const f32x4 d = distance(p, n, k0, half, k_pos, axis);
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    s[4 * n + e] = fmaf(-slope, d[e], s[4 * n + e]);
            }
        }
    }
    // to keys k0 + 8 n + 4 half + 0 .. 3
    __device__ inline f32x4 distance(const Args &p, int n, int k0, int half, const float *k_pos,
                                     int axis) const {
        if (SIDE && p.q_pos) {
            const float *at_n = k_pos + 8 * n + 4 * half;
            f32x4 d = away(*(const f32x4 *)at_n, pos[0]);
            if (p.axes > 1)
                d += away(*(const f32x4 *)(at_n + axis), pos[1]);
            if (p.axes > 2)
                d += away(*(const f32x4 *)(at_n + 2 * axis), pos[2]);
            return d;
        }
        const float from = (float)(at - k0 - 4 * half);
        return away(f32x4{8.f * n, 8.f * n + 1.f, 8.f * n + 2.f, 8.f * n + 3.f}, from);
    }
    // x where the lane does not see the key; docs: the block's documents in LDS
    __device__ inline void hide(const Args &p, f32x16 &s, float x, int k0, int half,
                                const int *docs) const {
        const int last = limit - k0 - 4 * half;
        if (SIDE && p.k_docs) {
#pragma unroll
            for (int n = 0; n < 4; ++n) {
                const i32x4 d = *(const i32x4 *)(docs + 8 * n + 4 * half);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const bool see = (8 * n + e < last) & (d[e] == doc) & (doc >= 0);
                    s[4 * n + e] = see ? s[4 * n + e] : x;
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < 16; ++i)
                s[i] = 8 * (i / 4) + i % 4 < last ? s[i] : x;
        }
    }
};

// Weights of half precision are held 2^7 up: its smallest normal number is 2^-14, and weights
// below it lose bits that count where many keys share a row.  At most 2^(8 + 7) then.
template <typename T> constexpr float weight_shift() {
    return __is_same(T, _Float16) ? 7.f : 0.f;
}

// max over the wave's halves, of each column
__device__ inline float max_halves(float x) {
    const auto y = __builtin_amdgcn_permlane32_swap(__float_as_int(x), __float_as_int(x), false,
                                                    false);
    return fmaxf(__int_as_float(y[0]), __int_as_float(y[1]));
}

// The gradients' kernels hold weights, which are 1 at most, as many powers of two up: 2^-14 may be
// shared by many keys (2^-28 keeps all of its bits this way).
template <typename T> constexpr int grad_shift() { return __is_same(T, _Float16) ? 14 : 0; }

// Gradients of scores, ds, are as large or small as the output's gradient makes them, and half
// precision holds 2^-14 to 2^15 with all bits.  A lane's results are of one column (a query or a
// key), whose sums any factor leaves as they are but for itself: its ds go by a power of two
// that brings the largest to 2^8 and follows when one passes 2^15, the sums with it (exactly).
// What then lies below the normal numbers is 2^-22 of the column's largest or less.  Other
// types have float32's range and no factor.  Without it ds of 2^-14 lost bits and ds past 65504
// made gradients NaN that are finite; it costs a gradient in half precision 4 to 6 % (2 x 2048,
// 8 heads, us: 64 features 128, 133; 128 features 215, 226), and 17 % at 256 features (521, 607),
// where the sums no longer stay in the accumulation registers.
template <typename T> struct Column {
    static constexpr bool kScaled = __is_same(T, _Float16);
    int up = 60; // 2^60 times the largest that a finite call can have is finite in float32

    // Before a block x of the column's ds is packed: `up` for it, and `sums` along.
    template <int DB> __device__ inline void fit(const f32x16 &x, f32x16 (&sums)[DB]) {
        if constexpr (kScaled) {
            float most = 0.f;
#pragma unroll
            for (int i = 0; i < 16; ++i)
                most = fmaxf(most, fabsf(x[i]));
            if (__any(__builtin_ldexpf(most, up) >= 32768.f)) {
                most = max_halves(most);
                const bool past = __builtin_ldexpf(most, up) >= 32768.f;
                const int by = past ? 9 - __builtin_amdgcn_frexp_expf(most) - up : 0;
                const float r = __builtin_ldexpf(1.f, by);
                up += by;
#pragma unroll
                for (int i = 0; i < DB; ++i)
#pragma unroll
                    for (int e = 0; e < 16; ++e)
                        sums[i][e] *= r;
            }
        }
    }
    // elements 8t .. of x by that factor, and what rounding took off them: a multiplication and
    // a conversion are one instruction
    __device__ inline x8<T> pack(const f32x16 &x, int t) const {
        if constexpr (!kScaled)
            return pack8<T>(x, t);
        const float by = __builtin_ldexpf(1.f, up);
        x8<T> r;
#pragma unroll
        for (int j = 0; j < 8; ++j)
            r[j] = (T)fmaf(x[8 * t + j], by, 0.f);
        return r;
    }
    __device__ inline x8<T> rest(const f32x16 &x, int t, x8<T> w) const {
        const float by = __builtin_ldexpf(1.f, up);
        x8<T> r;
#pragma unroll
        for (int j = 0; j < 8; ++j)
            r[j] = kScaled ? (T)fmaf(x[8 * t + j], by, -(float)w[j])
                           : (T)(x[8 * t + j] - (float)w[j]);
        return r;
    }
    // the sums as they would be without scale and grad_shift()
    template <int DB> __device__ inline void undo(f32x16 (&sums)[DB]) const {
        if constexpr (kScaled) {
            const float r = __builtin_ldexpf(1.f, -up - grad_shift<T>());
#pragma unroll
            for (int i = 0; i < DB; ++i)
#pragma unroll
                for (int e = 0; e < 16; ++e)
                    sums[i][e] *= r;
        }
    }
};

// One step of the running softmax: scores s (keys by queries), which times mul >= 0 are in
// base 2, become weights 2^(s mul - top).  `top` follows the largest score seen only when that
// grew by more than 2^8: weights up to 2^8 cost no precision in float32 sums, and the output
// is rarely rescaled.  `sum` adds this lane's half of the keys.
template <typename T, int KB, int DB>
__device__ inline void soften(f32x16 (&s)[KB], f32x16 (&o)[DB], float mul, float &top,
                              float &sum) {
    float m = s[0][0];
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int i = 0; i < 16; ++i)
            m = fmaxf(m, s[kb][i]);
    m = max_halves(m);
    // s mul - top in one rounding leaves the rounding of top in the weights, all of a row by
    // the same factor; past 2^11 that would show in 16 bits, so there products come first and
    // the largest weight stays a power of two
    if (__any(fabsf(m) * mul > 2048.f && m != -kInf)) {
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
            for (int i = 0; i < 16; ++i)
                s[kb][i] *= mul;
        m *= mul;
        mul = 1.f;
    }
    m = m == -kInf ? m : fmaf(m, mul, -weight_shift<T>());
    if (__any(m > top + 8.f)) {
        const float now = fmaxf(m, top);
        const float r = now == -kInf ? 1.f : __builtin_amdgcn_exp2f(top - now);
        top = now;
        sum *= r;
#pragma unroll
        for (int i = 0; i < DB; ++i)
#pragma unroll
            for (int e = 0; e < 16; ++e)
                o[i][e] *= r;
    }
    const float from = top == -kInf ? 0.f : top;
    float part[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            s[kb][i] = __builtin_amdgcn_exp2f(fmaf(s[kb][i], mul, -from));
            part[i % 4] += s[kb][i];
        }
    sum += (part[0] + part[1]) + (part[2] + part[3]);
}

// A result in the outputs' type, and what the rounding took off (for the gradient)
template <typename T> __device__ inline void put(const Args &p, int64_t at, x4<T> y, f32x4 x) {
    *(x4<T> *)((T *)p.out + at) = y;
    if (sizeof(T) == 2 && p.out_low) {
        x4<T> z;
#pragma unroll
        for (int j = 0; j < 4; ++j)
            z[j] = (T)(x[j] - (float)y[j]);
        *(x4<T> *)((T *)p.out_low + at) = z;
    }
}

// For the gradients: products s become weights p (times 2^grad_shift, which base() holds), products
// ds = do v become p (ds - delta), with a cap times a quarter of its slope (grad_scale() has
// the rest).  Four elements at a time, so
// that nothing but s and ds is held: dist(n), base(n) and delta(n) give what belongs to elements
// 4n .. 4n + 3: the distance, what attend_delta left of the log of the row's sum, and delta.
__device__ inline float grad_scale(const Args &p) {
    return p.cap > 0.f ? 4.f * p.scale : p.scale;
}
template <typename T, bool DS, typename Dist, typename Base, typename Delta>
__device__ inline void weigh(const Args &p, f32x16 &s, f32x16 &ds, float slope, Dist dist,
                             Base base, Delta delta) {
    const auto exponent = [&](int n) {
        f32x4 x = base(n);
        if (p.slopes) {
            const f32x4 d = dist(n);
#pragma unroll
            for (int e = 0; e < 4; ++e)
                x[e] = fmaf(-slope, d[e], x[e]);
        }
        return x;
    };
    if (p.cap > 0.f) {
        const Cap<T> cap(p);
#pragma unroll
        for (int n = 0; n < 4; ++n) {
            const f32x4 x = exponent(n);
            f32x4 d;
            if constexpr (DS)
                d = delta(n);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int i = 4 * n + e;
                const float r = cap.part(s[i]);
                s[i] = __builtin_amdgcn_exp2f(cap.add(r, x[e]));
                if constexpr (DS)
                    ds[i] = s[i] * (ds[i] - d[e]) * cap.slope(r);
            }
        }
    } else {
        const float m = p.scale * kLog2e;
#pragma unroll
        for (int n = 0; n < 4; ++n) {
            const f32x4 x = exponent(n);
            f32x4 d;
            if constexpr (DS)
                d = delta(n);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int i = 4 * n + e;
                s[i] = __builtin_amdgcn_exp2f(fmaf(s[i], m, x[e]));
                if constexpr (DS)
                    ds[i] = s[i] * (ds[i] - d[e]);
            }
        }
    }
}

// Documents of 64 consecutive keys or queries: the smallest and the largest id
// that is not negative, and whether any is negative.
__device__ inline bool docs_meet(int4 a, int4 b) { return a.x <= b.y && b.x <= a.y; }
__device__ inline bool docs_same(int4 a, int4 b) {
    return a.x == a.y && b.x == b.y && a.x == b.x && !a.z && !b.z;
}

// Walks the tiles of 64 rows in [t, end) that can hold something to see: all of them, or
// those whose documents meet `mine`.  A lane holds the summary of one tile of 64.
struct TileWalk {
    const int4 *tiles;
    int4 mine;
    int base, end;
    uint64_t left;
    int4 held, docs; // docs: of the tile that next() gave

    __device__ inline void start(const int4 *tiles_, int4 mine_, int t, int end_, int lane) {
        tiles = tiles_;
        mine = mine_;
        base = t;
        end = end_;
        left = 0;
        held = docs = int4{0, 0, 0, 0};
        if (tiles)
            fill(lane);
    }
    __device__ inline void fill(int lane) {
        for (left = 0; base < end; base += 64) {
            const int i = base + lane;
            held = tiles[min(i, end - 1)];
            left = __ballot(i < end && docs_meet(held, mine));
            if (left)
                return;
        }
    }
    // the next tile, or `end`
    __device__ inline int next(int lane) {
        if (!tiles)
            return base < end ? base++ : end;
        if (!left)
            return end;
        const int i = __builtin_ctzll(left), t = base + i;
        docs.x = __builtin_amdgcn_readlane(held.x, i);
        docs.y = __builtin_amdgcn_readlane(held.y, i);
        docs.z = __builtin_amdgcn_readlane(held.z, i);
        left &= left - 1;
        if (!left) {
            base += 64;
            fill(lane);
        }
        return t;
    }
};

// Blocks are dealt to the 8 XCDs in turn; each has its own L2.  xcd_order() gives every XCD a
// run of consecutive work items, so that those which read the same keys meet.
__device__ inline int xcd_order(int id, int n) {
    const int per = n >> 3, rest = n & 7, x = id & 7;
    return x * per + min(x, rest) + (id >> 3);
}

// a value that is the same in all lanes
__device__ inline int scalar(int x) { return __builtin_amdgcn_readfirstlane(x); }

// Blocks of rows of many heads, the first blocks of a head taking longest (causal): an XCD has
// its own heads, up to four of them at a time, and starts the long blocks of these first.
// Where heads do not divide by 8, all XCDs take the long blocks of all heads first.
struct Share {
    int block, head;
    __device__ inline Share(int id, int blocks, int heads) {
        if (heads & 7) {
            block = id / heads;
            head = id % heads;
            return;
        }
        const int own = heads >> 3, at_once = own & 1 ? 1 : own & 2 ? 2 : 4;
        const int j = id >> 3, run = at_once * blocks;
        block = j % run / at_once;
        head = (id & 7) * own + j / run * at_once + j % at_once;
    }
};

} // namespace attn

#endif
