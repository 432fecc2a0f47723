// norm_rotate.hip -- heads normed by their root mean square and turned by positions, in one pass.
//
//     r = (mean_d x_d^2 + eps)^-1/2,  y = R (r x w),  R the rotation of rotate.hip
//
// and with g = R^T dy:  dw = sum over tokens and heads of r g x,
//                       dx = r (g w - x r^2 mean_d(g w x)).
//
// Bound by memory: x is read once and y written once, x and dy read once and dx written once.  A
// head is held by as many lanes as it has items (V pairs or V features: 16 bytes or two times 16), so
// the norm's sum is a few exchanges between neighbouring lanes and nothing is read twice.  The
// cosines, sines and weights of a block's tokens lie in LDS, shared by the heads.
//
// 27306 tokens, 32 heads of 128, bfloat16: 109 us, 4.1 TB/s.  16396 tokens, 20 heads of 128: forward 33,
// backward 59 (4.3 TB/s) and 4 for the blocks' sums.
//
// dw: a block has one row of the weight, so a lane adds what belongs to its own features in
// registers over all of the block's tokens and heads; a block's lanes are joined in LDS and the
// blocks by a second kernel, each in a fixed order (no atomics: the same call, the same bits).
#include "rotate.h"

#include <algorithm>

namespace {

using rot::kTable;
using rot::Turns;
using rot::Unit;

// V floats; vectors, as arrays of eight are not kept in registers
template <int V> struct Floats {
    typedef float type __attribute__((ext_vector_type(V)));
};
template <int V> using fv = typename Floats<V>::type;

constexpr int kMaxPiece = 1 << 21; // heads of a block's tokens at a time: see quotient()
constexpr int kMaxItems = 8;  // a lane's, of one head
constexpr int kBlocks = 2048; // of a backward pass, about
constexpr int kJoinCols = 32; // columns of dw a block of norm_join

struct NormArgs {
    rot::Places at;
    const void *x, *dout, *weight; // weight: (groups, D), or null for ones
    void *out;                     // y, or dx (may be null: not asked for)
    float *part;                   // (blocks, D) sums for dw, or null
    int64_t x_b, x_l, x_h, do_b, do_l, do_h, tokens;
    int32_t L, H, D, interleaved, per_block, lane_bits, items, turned, groups, weight_f32;
    int32_t first_head[TM_NORM_MAX_GROUPS + 1];  // of each row of the weight
    int32_t first_block[TM_NORM_MAX_GROUPS + 1]; // backward: blocks of each row
    float eps;
};

// The features of one item: first .. first + V - 1, and with them second .. where there are two
// (halves).  pair: of its first turn.
enum Kind { kIdle, kPass, kSides, kHalves }; // kSides: pairs side by side in one unit
struct Item {
    Kind kind;
    int first, second, pair;
    template <int V> __device__ inline void set(const NormArgs &p, int n) {
        kind = kIdle;
        first = second = pair = 0;
        if (n >= p.items)
            return;
        if (n >= p.turned) {
            kind = kPass;
            first = 2 * p.at.pairs + (n - p.turned) * V;
        } else if (!p.interleaved) {
            kind = kHalves;
            pair = n * V;
            first = n * V;
            second = p.at.pairs + n * V;
        } else if (V == 1) {
            kind = kHalves;
            pair = n;
            first = 2 * n;
            second = first + 1;
        } else {
            kind = kSides;
            pair = n * (V / 2);
            first = n * V;
        }
    }
};

template <typename T, int V>
__device__ inline void read(fv<V> &a, fv<V> &b, const T *from, const Item &it) {
    using U = typename Unit<T, V>::type;
    if (it.kind == kIdle) {
#pragma unroll
        for (int j = 0; j < V; ++j)
            a[j] = b[j] = 0.f;
        return;
    }
    const U u = *(const U *)(from + it.first);
#pragma unroll
    for (int j = 0; j < V; ++j) {
        a[j] = (float)u[j];
        b[j] = 0.f;
    }
    if (it.kind == kHalves) {
        const U v = *(const U *)(from + it.second);
#pragma unroll
        for (int j = 0; j < V; ++j)
            b[j] = (float)v[j];
    }
}

template <typename T, int V>
__device__ inline void write(T *to, const fv<V> &a, const fv<V> &b, const Item &it) {
    using U = typename Unit<T, V>::type;
    if (it.kind == kIdle)
        return;
    U u;
#pragma unroll
    for (int j = 0; j < V; ++j)
        u[j] = (T)a[j];
    *(U *)(to + it.first) = u;
    if (it.kind == kHalves) {
        U v;
#pragma unroll
        for (int j = 0; j < V; ++j)
            v[j] = (T)b[j];
        *(U *)(to + it.second) = v;
    }
}

// sine: 1, or -1 to turn back
template <int V>
__device__ inline void turn(fv<V> &a, fv<V> &b, const float2 *table, const Item &it,
                            float sine) {
    if (it.kind == kHalves) {
        if constexpr (V == 1) {
            const float2 w = table[it.pair];
            const float u = a[0], v = b[0], s = sine * w.y;
            a[0] = u * w.x - v * s;
            b[0] = v * w.x + u * s;
        } else {
            const Turns<V> turns(table + it.pair);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float2 w = turns.at(j);
                const float u = a[j], v = b[j], s = sine * w.y;
                a[j] = u * w.x - v * s;
                b[j] = v * w.x + u * s;
            }
        }
    } else if (V > 1 && it.kind == kSides) {
        if constexpr (V > 1) {
            const Turns<V / 2> turns(table + it.pair);
#pragma unroll
            for (int j = 0; j < V / 2; ++j) {
                const float2 w = turns.at(j);
                const float u = a[2 * j], v = a[2 * j + 1], s = sine * w.y;
                a[2 * j] = u * w.x - v * s;
                a[2 * j + 1] = v * w.x + u * s;
            }
        }
    }
}

template <int V>
__device__ inline void weights_of(fv<V> &a, fv<V> &b, const float *w, const Item &it) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
        a[j] = w[it.first + j];
        b[j] = w[it.second + j]; // of an item without a second part: not used
    }
}

// The sum over the lanes of a head, 2^lane_bits neighbours.  Up to 16 lanes by moves within a row:
// once the lanes of four (eight) hold the same sum, a mirrored lane holds that of the others.
template <int CTRL> __device__ inline float moved(float x) {
    return __int_as_float(
        __builtin_amdgcn_update_dpp(0, __float_as_int(x), CTRL, 0xf, 0xf, false));
}
__device__ inline float over_head(float x, int lane_bits) {
    if (lane_bits > 0)
        x += moved<0xB1>(x); // quad_perm [1, 0, 3, 2]
    if (lane_bits > 1)
        x += moved<0x4E>(x); // quad_perm [2, 3, 0, 1]
    if (lane_bits > 2)
        x += moved<0x141>(x); // row_half_mirror
    if (lane_bits > 3)
        x += moved<0x140>(x); // row_mirror
    if (lane_bits > 4)
        x += __shfl_xor(x, 16);
    if (lane_bits > 5)
        x += __shfl_xor(x, 32);
    return x;
}

// i / n for 0 <= i < 2^21 by its reciprocal: the product is off by 2^-23 of itself at most, and (i + 1/2) / n
// is 1 / (2 n), 2^-22 of it, or more away from a whole number
__device__ inline int quotient(int i, float reciprocal) {
    return (int)(((float)i + 0.5f) * reciprocal);
}

// Where token `n` after (b0, l0) stands; a block's tokens cross few rows of the batch
struct At {
    int64_t b;
    uint32_t l;
    __device__ inline At(const NormArgs &p, int64_t b0, uint32_t l0, int n) : b(b0), l(l0 + n) {
        if (p.L >= p.per_block) {
            if (l >= (uint32_t)p.L) {
                l -= p.L;
                b += 1;
            }
        } else {
            const uint32_t rows = l / (uint32_t)p.L;
            l -= rows * p.L;
            b += rows;
        }
    }
};

__device__ inline float weight_at(const NormArgs &p, int i, bool f32, bool bf16) {
    if (!p.weight)
        return 1.f;
    return f32 ? ((const float *)p.weight)[i]
               : bf16 ? (float)((const __bf16 *)p.weight)[i]
                      : (float)((const _Float16 *)p.weight)[i];
}

// Cosines and sines of `tokens` tokens from (b0, l0) on.
template <typename T>
__device__ inline void fill_table(float2 *table, const NormArgs &p, int64_t b0, uint32_t l0,
                                  int tokens) {
    const float per_pair = 1.f / p.at.pairs;
    for (int i = threadIdx.x; i < tokens * p.at.pairs; i += 256) {
        const int token = quotient(i, per_pair);
        const At at(p, b0, l0, token);
        table[i] = rot::turn_of<T>(p.at, at.b * p.at.pos_b + (int64_t)at.l * p.at.axes,
                                   i - token * p.at.pairs);
    }
}

template <typename T, int V, int K>
__global__ __launch_bounds__(256) void norm_rotate(const NormArgs p) {
    extern __shared__ __attribute__((aligned(16))) float shared[];
    float2 *table = (float2 *)shared;
    float *weights = shared + ((2 * p.per_block * p.at.pairs + 3) & ~3);
    const int64_t first = (int64_t)blockIdx.x * p.per_block;
    const int tokens = (int)min((int64_t)p.per_block, p.tokens - first);
    const int64_t b0 = first / p.L;
    const uint32_t l0 = (uint32_t)(first - b0 * p.L);
    for (int i = threadIdx.x; i < p.groups * p.D; i += 256)
        weights[i] = weight_at(p, i, sizeof(T) == 4 || p.weight_f32, __is_same(T, __bf16));
    fill_table<T>(table, p, b0, l0, tokens);
    const int lane = threadIdx.x & ((1 << p.lane_bits) - 1), sub = threadIdx.x >> p.lane_bits;
    const int subs = 256 >> p.lane_bits;
    Item item[K];
#pragma unroll
    for (int k = 0; k < K; ++k)
        item[k].template set<V>(p, lane + (k << p.lane_bits));
    const float share = 1.f / p.D, per_head = 1.f / p.H;
    __syncthreads();

    constexpr int AT_ONCE = 2; // heads whose loads are under way together
    const int heads = tokens * p.H;
    for (int i0 = sub; i0 < heads; i0 += AT_ONCE * subs) {
        fv<V> a[AT_ONCE][K], b[AT_ONCE][K];
        int token[AT_ONCE], head[AT_ONCE];
#pragma unroll
        for (int n = 0; n < AT_ONCE; ++n) {
            const int i = min(i0 + n * subs, heads - 1);
            token[n] = quotient(i, per_head);
            head[n] = i - token[n] * p.H;
            const At at(p, b0, l0, token[n]);
            const T *src =
                (const T *)p.x + at.b * p.x_b + (int64_t)at.l * p.x_l + head[n] * p.x_h;
#pragma unroll
            for (int k = 0; k < K; ++k)
                read<T, V>(a[n][k], b[n][k], src, item[k]);
        }
#pragma unroll
        for (int n = 0; n < AT_ONCE; ++n) {
            const bool real = i0 + n * subs < heads; // or the last head again
            float sum = 0.f;
#pragma unroll
            for (int k = 0; k < K; ++k)
#pragma unroll
                for (int j = 0; j < V; ++j)
                    sum = fmaf(a[n][k][j], a[n][k][j], fmaf(b[n][k][j], b[n][k][j], sum));
            const float r = rsqrtf(fmaf(over_head(sum, p.lane_bits), share, p.eps));
            int row = 0;
#pragma unroll
            for (int g = 1; g < TM_NORM_MAX_GROUPS; ++g)
                row += g < p.groups && head[n] >= p.first_head[g];
            T *dst = (T *)p.out + ((first + token[n]) * p.H + head[n]) * p.D;
#pragma unroll
            for (int k = 0; k < K; ++k) {
                fv<V> wa, wb;
                weights_of<V>(wa, wb, weights + row * p.D, item[k]);
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    a[n][k][j] *= r * wa[j];
                    b[n][k][j] *= r * wb[j];
                }
                turn<V>(a[n][k], b[n][k], table + token[n] * p.at.pairs, item[k], 1.f);
                if (real)
                    write<T, V>(dst, a[n][k], b[n][k], item[k]);
            }
        }
    }
}

// A block has the heads of one row of the weight, of tokens block, block + blocks, .. in pieces of
// per_block.
template <typename T, int V, int K>
__global__ __launch_bounds__(256) void norm_rotate_backward(const NormArgs p) {
    extern __shared__ __attribute__((aligned(16))) float shared[];
    float2 *table = (float2 *)shared;
    int row = 0;
#pragma unroll
    for (int g = 1; g < TM_NORM_MAX_GROUPS; ++g)
        row += g < p.groups && (int)blockIdx.x >= p.first_block[g];
    const int lane = threadIdx.x & ((1 << p.lane_bits) - 1), sub = threadIdx.x >> p.lane_bits;
    const int subs = 256 >> p.lane_bits;
    Item item[K];
    fv<V> wa[K], wb[K], da[K], db[K];
#pragma unroll
    for (int k = 0; k < K; ++k) {
        item[k].template set<V>(p, lane + (k << p.lane_bits));
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const bool f32 = sizeof(T) == 4 || p.weight_f32, bf16 = __is_same(T, __bf16);
            wa[k][j] = weight_at(p, row * p.D + item[k].first + j, f32, bf16);
            wb[k][j] = weight_at(p, row * p.D + item[k].second + j, f32, bf16);
            da[k][j] = db[k][j] = 0.f;
        }
    }
    const float share = 1.f / p.D;
    const int head0 = p.first_head[row], n_heads = p.first_head[row + 1] - head0;
    const float per_head = 1.f / n_heads;
    const int blocks = p.first_block[row + 1] - p.first_block[row];
    for (int64_t first = (int64_t)(blockIdx.x - p.first_block[row]) * p.per_block;
         first < p.tokens; first += (int64_t)blocks * p.per_block) {
        const int tokens = (int)min((int64_t)p.per_block, p.tokens - first);
        const int64_t b0 = first / p.L;
        const uint32_t l0 = (uint32_t)(first - b0 * p.L);
        __syncthreads(); // the table of the piece before is done with
        fill_table<T>(table, p, b0, l0, tokens);
        __syncthreads();
        const int heads = tokens * n_heads;
        for (int i = sub; i < heads; i += subs) {
            const int token = quotient(i, per_head), head = head0 + i - token * n_heads;
            const At at(p, b0, l0, token);
            const T *src =
                (const T *)p.x + at.b * p.x_b + (int64_t)at.l * p.x_l + head * p.x_h;
            const T *grad =
                (const T *)p.dout + at.b * p.do_b + (int64_t)at.l * p.do_l + head * p.do_h;
            fv<V> xa[K], xb[K], ga[K], gb[K];
#pragma unroll
            for (int k = 0; k < K; ++k) {
                read<T, V>(xa[k], xb[k], src, item[k]);
                read<T, V>(ga[k], gb[k], grad, item[k]);
            }
            float sum = 0.f, dot = 0.f;
#pragma unroll
            for (int k = 0; k < K; ++k) {
                turn<V>(ga[k], gb[k], table + token * p.at.pairs, item[k], -1.f);
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    sum = fmaf(xa[k][j], xa[k][j], fmaf(xb[k][j], xb[k][j], sum));
                    dot = fmaf(xa[k][j] * wa[k][j], ga[k][j],
                               fmaf(xb[k][j] * wb[k][j], gb[k][j], dot));
                }
            }
            const float r = rsqrtf(fmaf(over_head(sum, p.lane_bits), share, p.eps));
            // x's part of dx: r^3 mean(g w x), in an order that stays in range as r x does
            const float f = r * (over_head(dot, p.lane_bits) * r) * share * r;
            T *dst = (T *)p.out + ((first + token) * p.H + head) * p.D;
#pragma unroll
            for (int k = 0; k < K; ++k) {
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const float ra = r * ga[k][j], rb = r * gb[k][j];
                    da[k][j] = fmaf(ra, xa[k][j], da[k][j]);
                    db[k][j] = fmaf(rb, xb[k][j], db[k][j]);
                    xa[k][j] = fmaf(-f, xa[k][j], ra * wa[k][j]);
                    xb[k][j] = fmaf(-f, xb[k][j], rb * wb[k][j]);
                }
                if (p.out)
                    write<T, V>(dst, xa[k], xb[k], item[k]);
            }
        }
    }
    if (!p.part)
        return;
    // the block's lanes of one feature, joined in order
    __syncthreads();
#pragma unroll
    for (int k = 0; k < K; ++k)
        if (item[k].kind != kIdle) {
#pragma unroll
            for (int j = 0; j < V; ++j)
                shared[sub * p.D + item[k].first + j] = da[k][j];
            if (item[k].kind == kHalves)
#pragma unroll
                for (int j = 0; j < V; ++j)
                    shared[sub * p.D + item[k].second + j] = db[k][j];
        }
    __syncthreads();
    for (int d = threadIdx.x; d < p.D; d += 256) {
        float sum = 0.f;
        for (int s = 0; s < subs; ++s)
            sum += shared[s * p.D + d];
        p.part[(int64_t)blockIdx.x * p.D + d] = sum;
    }
}

// dw of kJoinCols features of a row from the blocks' sums: 32 threads a feature take every 32nd
// block, then the 32 are added in order.
template <typename W>
__global__ __launch_bounds__(32 * kJoinCols) void norm_join(const NormArgs p, W *dw) {
    __shared__ float sums[32][kJoinCols + 1];
    const int per_row = (p.D + kJoinCols - 1) / kJoinCols;
    const int row = blockIdx.x / per_row, col = threadIdx.x % kJoinCols;
    const int d = blockIdx.x % per_row * kJoinCols + col, lane = threadIdx.x / kJoinCols;
    float sum = 0.f;
    if (d < p.D) {
        const float *from = p.part + d;
        int b = p.first_block[row] + lane;
        const int end = p.first_block[row + 1];
        for (; b + 7 * 32 < end; b += 8 * 32) { // eight on their way
            float x[8];
#pragma unroll
            for (int n = 0; n < 8; ++n)
                x[n] = from[(int64_t)(b + 32 * n) * p.D];
#pragma unroll
            for (int n = 0; n < 8; ++n)
                sum += x[n];
        }
        for (; b < end; b += 32)
            sum += from[(int64_t)b * p.D];
    }
    sums[lane][col] = sum;
    __syncthreads();
    if (lane == 0 && d < p.D) {
        for (int n = 1; n < 32; ++n)
            sum += sums[n][col];
        dw[row * p.D + d] = (W)sum;
    }
}

// Checks what both directions need and fills everything but the outputs.
int prepare(const tm_norm_rotation *n, NormArgs &p) {
    if (!n)
        return TM_ERR_INVALID_ARGUMENT;
    const tm_rotation &r = n->rotation;
    if (r.B < 0 || r.L < 0 || r.H < 1 || r.D < 1 || r.dtype < TM_BF16 || r.dtype > TM_F32 ||
        r.inverse || n->groups < 1 || n->groups > TM_NORM_MAX_GROUPS || !(n->eps >= 0.f) ||
        !(n->eps < __builtin_inff()) || (n->weight && n->weight_type != r.dtype &&
                                         n->weight_type != TM_F32))
        return TM_ERR_INVALID_ARGUMENT;
    if (const int rc = rot::places(r, p.at))
        return rc;
    int64_t heads = 0;
    for (int g = 0; g < n->groups; ++g) {
        if (n->heads[g] < 1)
            return TM_ERR_INVALID_ARGUMENT;
        p.first_head[g] = (int32_t)heads;
        heads += n->heads[g];
        if (heads > r.H)
            return TM_ERR_INVALID_ARGUMENT;
    }
    if (heads != r.H)
        return TM_ERR_INVALID_ARGUMENT;
    p.first_head[n->groups] = (int32_t)heads;
    if (r.D > TM_NORM_MAX_HEAD_DIM || r.H > TM_NORM_MAX_HEADS)
        return TM_ERR_UNSUPPORTED_SHAPE;
    p.x = r.x, p.weight = n->weight, p.weight_f32 = n->weight_type == TM_F32;
    p.x_b = r.x_b, p.x_l = r.x_l, p.x_h = r.x_h;
    p.L = r.L, p.H = r.H, p.D = r.D, p.groups = n->groups, p.eps = n->eps;
    p.interleaved = r.interleaved ? 1 : 0;
    p.tokens = (int64_t)r.B * r.L;
    return TM_OK;
}

// Whether units of 16 bytes fit, and how a head is shared out; the features of a lane.
int share_out(NormArgs &p, const tm_rotation &r, bool wide) {
    const int unit = r.dtype == TM_F32 ? 4 : 8, pairs = p.at.pairs;
    wide = wide && !((uintptr_t)r.x % 16) && !(r.x_b % unit) && !(r.x_l % unit) &&
           !(r.x_h % unit) && !(r.D % unit) && !(pairs % (p.interleaved ? unit / 2 : unit));
    const int v = wide ? unit : 1;
    p.turned = pairs / (p.interleaved ? (v + 1) / 2 : v);
    p.items = p.turned + (r.D - 2 * pairs) / v;
    for (p.lane_bits = 0; p.lane_bits < 6 && (1 << p.lane_bits) < p.items;)
        ++p.lane_bits;
    return v;
}

// f<V, K>() for v elements a load and the items a lane has
template <typename T, typename F> void with_sizes(int v, const NormArgs &p, F f) {
    constexpr int W = 16 / sizeof(T);
    const int k = (p.items + (1 << p.lane_bits) - 1) >> p.lane_bits;
    if (v == W)
        k == 1 ? f.template operator()<T, W, 1>() : f.template operator()<T, W, 2>();
    else
        k == 1 ? f.template operator()<T, 1, 1>() : f.template operator()<T, 1, kMaxItems>();
}
template <typename F> void with_type(int dtype, int v, const NormArgs &p, F f) {
    if (dtype == TM_BF16)
        with_sizes<__bf16>(v, p, f);
    else if (dtype == TM_F16)
        with_sizes<_Float16>(v, p, f);
    else
        with_sizes<float>(v, p, f);
}

struct Forward {
    const NormArgs &p;
    unsigned blocks;
    hipStream_t stream;
    template <typename T, int V, int K> void operator()() const {
        const size_t lds = 4 * (((2 * p.per_block * p.at.pairs + 3) & ~3) + p.groups * p.D);
        norm_rotate<T, V, K><<<dim3(blocks), 256, lds, stream>>>(p);
    }
};

struct Backward {
    const NormArgs &p;
    hipStream_t stream;
    template <typename T, int V, int K> void operator()() const {
        const size_t lds = std::max<size_t>(8 * (size_t)p.per_block * p.at.pairs,
                                            4 * (size_t)p.D * (256 >> p.lane_bits));
        norm_rotate_backward<T, V, K><<<dim3(p.first_block[p.groups]), 256, lds, stream>>>(p);
    }
};

// Blocks of each row of the weight: as many as fill the card for what it holds, at most one for
// each piece of tokens.
void deal_blocks(NormArgs &p) {
    const int64_t most = (p.tokens + p.per_block - 1) / p.per_block;
    int64_t at = 0;
    for (int g = 0; g < p.groups; ++g) {
        const int64_t heads = p.first_head[g + 1] - p.first_head[g];
        p.first_block[g] = (int32_t)at;
        at += std::max<int64_t>(1, std::min(most, (kBlocks * heads + p.H - 1) / p.H));
    }
    p.first_block[p.groups] = (int32_t)at;
}

int per_block(const NormArgs &p, int64_t heads, int64_t at_once) {
    // `at_once` heads a lane where there are tokens enough, as long as that leaves four blocks for
    // each compute unit; the table's size bounds it too
    const int64_t wanted = at_once * (256 >> p.lane_bits);
    int64_t per = std::max<int64_t>(1, wanted / heads);
    per = std::min(per, std::max<int64_t>(1, p.tokens / 1024));
    const int64_t most = (1 << 24) - 1;
    per = std::max(per, (p.tokens + most - 1) / most);
    if (p.at.pairs)
        per = std::min<int64_t>(per, kTable / p.at.pairs);
    return (int)std::min<int64_t>(per, kMaxPiece / p.H);
}

int backward_sizes(NormArgs &p) {
    // two heads a lane of the row with fewest: with four, pieces are left over (32768 tokens, 16 and
    // 16 half-precision heads of 64: 108 and 118 us)
    int64_t fewest = p.H;
    for (int g = 0; g < p.groups; ++g)
        fewest = std::min<int64_t>(fewest, p.first_head[g + 1] - p.first_head[g]);
    p.per_block = per_block(p, fewest, 2);
    deal_blocks(p);
    return p.first_block[p.groups];
}

} // namespace

extern "C" int tm_norm_rotate(const tm_norm_rotation *n, void *out, hipStream_t stream) {
    NormArgs p = {};
    if (const int rc = prepare(n, p))
        return rc;
    const tm_rotation &r = n->rotation;
    if (!p.tokens)
        return TM_OK;
    if (!r.x || !out || !r.positions || (p.at.pairs && !r.freqs))
        return TM_ERR_INVALID_ARGUMENT;
    p.out = out;
    const int v = share_out(p, r, !((uintptr_t)out % 16));
    p.per_block = per_block(p, p.H, 4);
    const int64_t blocks = (p.tokens + p.per_block - 1) / p.per_block;
    if (blocks >= (1 << 24))
        return TM_ERR_UNSUPPORTED_SHAPE;
    with_type(r.dtype, v, p, Forward{p, (unsigned)blocks, stream});
    return hipGetLastError() == hipSuccess ? TM_OK : TM_ERR_LAUNCH;
}

extern "C" size_t tm_norm_rotate_backward_workspace_bytes(const tm_norm_rotation *n) {
    NormArgs p = {};
    if (prepare(n, p) || !p.tokens)
        return 0;
    // an upper bound for either width of loads
    return ((size_t)kBlocks + 2 * p.groups) * p.D * sizeof(float);
}

extern "C" int tm_norm_rotate_backward(const tm_norm_rotation *n, const void *dout, int64_t do_b,
                                       int64_t do_l, int64_t do_h, void *dx, void *dweight,
                                       void *workspace, size_t workspace_bytes,
                                       hipStream_t stream) {
    NormArgs p = {};
    if (const int rc = prepare(n, p))
        return rc;
    const tm_rotation &r = n->rotation;
    if (dweight && !n->weight)
        return TM_ERR_INVALID_ARGUMENT;
    if (!dx && !dweight)
        return TM_OK;
    if (p.tokens) {
        if (!r.x || !dout || !r.positions || (p.at.pairs && !r.freqs))
            return TM_ERR_INVALID_ARGUMENT;
        if (dweight && (!workspace || (uintptr_t)workspace % 16 ||
                        workspace_bytes < tm_norm_rotate_backward_workspace_bytes(n)))
            return TM_ERR_WORKSPACE;
        const int unit = r.dtype == TM_F32 ? 4 : 8;
        const int v = share_out(p, r,
                                !(((uintptr_t)dx | (uintptr_t)dout) % 16) && !(do_b % unit) &&
                                    !(do_l % unit) && !(do_h % unit));
        p.dout = dout, p.do_b = do_b, p.do_l = do_l, p.do_h = do_h;
        p.out = dx;
        p.part = dweight ? (float *)workspace : nullptr;
        backward_sizes(p);
        with_type(r.dtype, v, p, Backward{p, stream});
        if (hipGetLastError() != hipSuccess)
            return TM_ERR_LAUNCH;
    }
    if (!dweight)
        return TM_OK;
    // without tokens: zeros
    const dim3 grid(p.groups * ((p.D + kJoinCols - 1) / kJoinCols));
    if (n->weight_type == TM_F32)
        norm_join<float><<<grid, 32 * kJoinCols, 0, stream>>>(p, (float *)dweight);
    else if (n->weight_type == TM_BF16)
        norm_join<__bf16><<<grid, 32 * kJoinCols, 0, stream>>>(p, (__bf16 *)dweight);
    else
        norm_join<_Float16><<<grid, 32 * kJoinCols, 0, stream>>>(p, (_Float16 *)dweight);
    return hipGetLastError() == hipSuccess ? TM_OK : TM_ERR_LAUNCH;
}
