// feed_forward.hip -- the gated feed-forward block: checks, sizes of tiles, launches.  The products
// are in ff_tile.h.
//
//     a = x G^T, b = x U^T, h = act(a) b, y = h D^T
//     dh = dy D; da = dh b act'(a), db = dh act(a);
//     dx = da G + db U; dG = da^T x, dU = db^T x, dD = dy^T h
//
// Forward two launches: both projections with the activation and the product in the first's
// epilogue, then D.  Backward: dh, in whose epilogue da and db; dx; dG and dU together;
// dD.  h, da and db are rounded to the inputs' type once, as operands of the next product have to be.  a and b
// are not rounded to it: they are saved with 15 bits after the leading one (truncated, off by less than
// 2^-15: ff_tile.h), since each enters two gradients that are rounded again (with a and b in
// bfloat16 those are off by 1.75 roundings, so by 1.42).
//
// Half precision's da and db carry a power of two (grad_up() in ff_tile.h): one launch for the largest |dy|,
// 8 us of 3711 x 1000, and a second one of dh, which ends at once (5 us) unless the first one's scale
// proves too large.
#include "ff.h"

#include "../../include/torchmatch_amd.h"

#include <algorithm>

namespace {

using ff::Args;
using ff::Kind;

constexpr int64_t kMaxRows = INT32_MAX - 256;
constexpr size_t kScaleBytes = ff::kMostParts * sizeof(float) + 256; // most and past, half precision

int size_of(const tm_feed_forward &f) { return f.dtype == TM_F32 ? 4 : 2; }
int64_t hidden_row(const tm_feed_forward &f) { return ((int64_t)f.F + 7) / 8 * 8; }
int64_t hidden_bytes(const tm_feed_forward &f) { // (T, hidden) of the inputs' type
    return ((int64_t)f.T * hidden_row(f) * size_of(f) + 255) / 256 * 256;
}

// Tiles of a product; the last ones, where they would leave much of the card idle, split over k.
struct Plan {
    int size;
    bool tokens;
    int whole, splits, split_steps;
    size_t part; // bytes of partial sums
};
// A step of 128 bytes of k of all the blocks that run at once, in us, as measured on 128 to 256 steps with
// part of the card's places taken: a compute unit that has its block alone is at its own pace, many share
// the card's clock and its memory.  16-bit types: 128 large tiles 1.20, 176 1.34, 224 1.50, 256
// 1.57 to 1.73; 256 small ones 0.67, 384 0.80, 512 0.88 to 0.94; 256 small ones with four tiles in
// LDS 0.52 to 0.57.  float32: 128 small ones 1.6, 256 1.77, 384 2.46, 512 2.73 to 2.96; 128 with four
// 1.6, 256 1.7.  64 x 64: up to 176 tiles 0.29 to 0.34, 352 0.46; float32 0.77 and 1.1.
double step_time(int dtype, int size, int64_t blocks) {
    const double part = (double)blocks / (size == ff::kSmall || size == ff::kTiny ? 512 : 256);
    if (size == ff::kTiny)
        return dtype == TM_F32 ? std::max(0.76, 0.3 + 1.15 * part)
                               : std::max(0.3, 0.13 + 0.45 * part);
    if (dtype == TM_F32)
        return size == ff::kDeep ? 1.58 + 0.1 * part : std::max(1.65, 0.9 + 1.9 * part);
    return size == ff::kLarge  ? std::max(1.19, 0.7 + 0.95 * part)
           : size == ff::kDeep ? 0.49 + 0.07 * part
                               : std::max(0.67, 0.45 + 0.47 * part);
}
// A round's beginning and end, us: what up and hidden read and write after their products is
// not hidden, 5 with 64 x 64, 9 and 14 with 128 x 128, 16 and 24 with 256 x 256.
double end_time(Kind kind, int size) {
    if (kind != ff::kUp && kind != ff::kHidden)
        return 3.;
    return size == ff::kTiny     ? 5.
           : size != ff::kLarge ? (kind == ff::kUp ? 9. : 14.)
                                : (kind == ff::kUp ? 16. : 24.);
}
// Chosen by these times; the split tiles' sums are written and read at 3 TB/s, by one launch more, 6.
Plan plan(const tm_feed_forward &f, Kind kind, int64_t M, int64_t N, int64_t K, int segments,
          int batches) {
    const int64_t k = 128 / size_of(f), steps = (K + k - 1) / k * segments;
    Plan best = {};
    double least = 0.;
    for (int size : {ff::kSmall, ff::kDeep, ff::kTiny, ff::kLarge}) {
        if (size == ff::kLarge && f.dtype == TM_F32)
            continue;
        const int64_t t = size == ff::kLarge ? 256 : size == ff::kTiny ? 64 : 128;
        const int64_t tn = kind == ff::kUp ? t / 2 : t;
        const int64_t tiles = (M + t - 1) / t * ((N + tn - 1) / tn) * batches;
        const int64_t at_once = size == ff::kSmall || size == ff::kTiny ? 512 : 256;
        const int64_t rounds = tiles / at_once, rest = tiles - rounds * at_once;
        if (size == ff::kDeep && tiles > at_once) // without a second block ends are not hidden either
            continue;
        for (int64_t splits = 1; splits <= 64; ++splits) {
            if (splits > 1 && (!rest || rest * splits > at_once || steps < 8 * splits))
                break;
            const int64_t split_steps = (steps + splits - 1) / splits;
            const double bytes = splits > 1 ? (double)rest * splits * t * t * 4 : 0.;
            const double time = step_time(f.dtype, size, at_once) * rounds * steps +
                                step_time(f.dtype, size, rest * splits) * split_steps * (rest > 0) +
                                end_time(kind, size) * (rounds + (rest > 0)) +
                                (splits > 1 ? 6. + 2. * bytes / 3e6 : 0.);
            if (best.splits == 0 || time < least) {
                least = time;
                best = {size, false, (int)(splits > 1 ? rounds * at_once : tiles), (int)splits,
                        (int)split_steps, (size_t)bytes};
            }
        }
    }
    // product_tokens: 4 for its beginning and end, and on each compute unit its blocks' steps of 4 x 128
    // bytes of k and one and a half each: up 0.40 with 32 rows a block (float32, at the rate of its own
    // instructions, 0.56), down 0.30 (0.40), 0.62 of that with 16
    if (M <= ff::kTokens && (kind == ff::kUp || kind == ff::kDown)) {
        const int rows = ff::tokens_rows(M, N);
        const double blocks = (double)((M + rows - 1) / rows * ((N + 15) / 16)) / 256.;
        const double step = (kind == ff::kUp ? (f.dtype == TM_F32 ? 0.56 : 0.40)
                                             : (f.dtype == TM_F32 ? 0.40 : 0.30)) *
                            (rows == 16 ? 0.62 : 1.);
        if (4. + std::max(blocks, 1.) * ((steps + 3) / 4 + 1.5) * step < least)
            return {ff::kSmall, true, 0, 1, 0, 0};
    }
    return best;
}

Plan plan_up(const tm_feed_forward &f) { return plan(f, ff::kUp, f.T, f.F, f.C, 1, 1); }
Plan plan_down(const tm_feed_forward &f) { return plan(f, ff::kDown, f.T, f.O, f.F, 1, 1); }
Plan plan_hidden(const tm_feed_forward &f) { return plan(f, ff::kHidden, f.T, f.F, f.O, 1, 1); }
Plan plan_input(const tm_feed_forward &f) { return plan(f, ff::kInput, f.T, f.C, f.F, 2, 1); }
Plan plan_weights(const tm_feed_forward &f) {
    return plan(f, ff::kWeights, f.F, f.C, f.T, 1, 2);
}
Plan plan_output(const tm_feed_forward &f) { return plan(f, ff::kWeights, f.O, f.F, f.T, 1, 1); }

int check(const tm_feed_forward *f) {
    if (!f || f->T < 0 || f->C < 1 || f->F < 1 || f->O < 1 || f->dtype < TM_BF16 ||
        f->dtype > TM_F32 || f->activation < TM_SILU || f->activation > TM_RELU)
        return TM_ERR_INVALID_ARGUMENT;
    const int64_t unit = 16 / size_of(*f);
    const auto odd = [&](const void *p, int64_t l, int64_t n) {
        return (uintptr_t)p % 16 || l % unit || l < 0 || (l && l < n);
    };
    if (odd(f->x, f->x_l, f->C) || odd(f->gate, f->w_l, f->C) || odd(f->up, f->w_l, f->C) ||
        odd(f->down, f->down_l, f->F))
        return TM_ERR_INVALID_ARGUMENT;
    const int64_t most = TM_FF_MAX_ROW_BYTES / size_of(*f);
    if (f->x_l >= most || f->w_l >= most || f->down_l >= most ||
        f->C >= most || f->O >= most || hidden_row(*f) >= most || f->T > kMaxRows)
        return TM_ERR_UNSUPPORTED_SHAPE;
    const auto blocks = [](int64_t m, int64_t n) { return ((m + 127) / 128) * ((n + 63) / 64); };
    if (std::max({blocks(f->T, f->F), blocks(f->T, f->O), blocks(f->T, f->C),
                  2 * blocks(f->F, f->C), blocks(f->O, f->F)}) > TM_FF_MAX_BLOCKS)
        return TM_ERR_UNSUPPORTED_SHAPE;
    return TM_OK;
}

int product(const tm_feed_forward &f, Args p, Kind kind, const Plan &how, void *part,
            hipStream_t stream) {
    p.whole = how.whole, p.splits = how.splits, p.split_steps = how.split_steps;
    p.part = (float *)part;
    p.activation = f.activation;
    if (how.tokens) {
        const auto tokens = f.dtype == TM_BF16  ? ff::tokens_bf16
                            : f.dtype == TM_F16 ? ff::tokens_f16
                                                : ff::tokens_f32;
        return tokens(p, kind, stream) ? TM_ERR_LAUNCH : TM_OK;
    }
    const auto run = f.dtype == TM_BF16  ? ff::product_bf16
                     : f.dtype == TM_F16 ? ff::product_f16
                                         : ff::product_f32;
    return run(p, kind, how.size, stream) ? TM_ERR_LAUNCH : TM_OK;
}

Args args(int64_t M, int64_t N, int64_t K) {
    Args p = {};
    p.M = (int32_t)M, p.N = (int32_t)N, p.K = (int32_t)K;
    p.segments = p.batches = 1;
    return p;
}

// rows of `out` at multiples of 16 bytes
int wide(const tm_feed_forward &f, const void *out, int64_t l) {
    return !((uintptr_t)out % 16) && l % (16 / size_of(f)) == 0;
}

// What is saved: (T, hidden) planes of the type's size, for a and b and then h.
int planes(const tm_feed_forward &f) { return f.dtype == TM_F32 ? 2 : 3; }
void *plane(const tm_feed_forward &f, const void *saved, int n) {
    return (char *)const_cast<void *>(saved) + n * ((int64_t)f.T * hidden_row(f) * size_of(f));
}
void set_saved(const tm_feed_forward &f, Args &p, const void *saved) {
    for (int n = 0; n < planes(f); ++n)
        p.saved[n] = plane(f, saved, n);
}

// The largest finite |x| of what each block takes of (rows, n), half precision; *past is cleared for
// the product that follows.
__global__ __launch_bounds__(256) void ff_most(const _Float16 *x, int64_t l, int rows, int n,
                                               float *most, uint32_t *past) {
    typedef _Float16 h16x8 __attribute__((ext_vector_type(8)));
    __shared__ float waves[4];
    const int units = (n + 7) / 8; // a row's last unit ends in zeros
    if (blockIdx.x == 0 && threadIdx.x == 0)
        *past = 0;
    float m = 0.f;
    for (int row = blockIdx.x; row < rows; row += ff::kMostParts)
        for (int u = threadIdx.x; u < units; u += 256) {
            const h16x8 v = *(const h16x8 *)(x + row * l + 8 * u);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float a = fabsf((float)v[j]);
                m = a < __builtin_inff() ? fmaxf(m, a) : m;
            }
        }
#pragma unroll
    for (int k = 1; k < 64; k *= 2)
        m = fmaxf(m, __shfl_xor(m, k));
    if (threadIdx.x % 64 == 0)
        waves[threadIdx.x / 64] = m;
    __syncthreads();
    if (threadIdx.x == 0)
        most[blockIdx.x] = fmaxf(fmaxf(waves[0], waves[1]), fmaxf(waves[2], waves[3]));
}

// 16 bytes a thread of rows of n elements, zeros past them
template <typename U, int E>
__global__ __launch_bounds__(256) void ff_pad(const U *x, int64_t l, int64_t rows, int n, int units,
                                              U *out) {
    typedef U V __attribute__((ext_vector_type(E)));
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int64_t row = i / units;
    if (row >= rows)
        return;
    const int e = (int)(i - row * units) * E;
    V v;
#pragma unroll
    for (int j = 0; j < E; ++j)
        v[j] = e + j < n ? x[row * l + e + j] : (U)0;
    ((V *)out)[i] = v;
}

} // namespace

extern "C" int tm_pad_rows(const void *x, int64_t x_l, int64_t rows, int32_t n, int32_t dtype,
                           void *out, hipStream_t stream) {
    if (rows < 0 || n < 1 || dtype < TM_BF16 || dtype > TM_F32 || (uintptr_t)out % 16)
        return TM_ERR_INVALID_ARGUMENT;
    if (!rows)
        return TM_OK;
    if (!x || !out)
        return TM_ERR_INVALID_ARGUMENT;
    const int e = dtype == TM_F32 ? 4 : 8, units = (int)(((int64_t)n + e - 1) / e);
    const int64_t most = (int64_t)((1 << 24) - 1) * 256;
    if (rows > most / units)
        return TM_ERR_UNSUPPORTED_SHAPE;
    const unsigned blocks = (unsigned)((rows * units + 255) / 256);
    if (e == 8)
        ff_pad<uint16_t, 8><<<dim3(blocks), 256, 0, stream>>>((const uint16_t *)x, x_l, rows, n,
                                                             units, (uint16_t *)out);
    else
        ff_pad<uint32_t, 4><<<dim3(blocks), 256, 0, stream>>>((const uint32_t *)x, x_l, rows, n,
                                                             units, (uint32_t *)out);
    return hipGetLastError() == hipSuccess ? TM_OK : TM_ERR_LAUNCH;
}

extern "C" size_t tm_feed_forward_saved_bytes(const tm_feed_forward *f) {
    if (check(f))
        return 0;
    return (size_t)(planes(*f) + 1) * f->T * hidden_row(*f) * size_of(*f);
}

extern "C" size_t tm_feed_forward_workspace_bytes(const tm_feed_forward *f) {
    if (check(f) || !f->T)
        return 0;
    return hidden_bytes(*f) + std::max(plan_up(*f).part, plan_down(*f).part);
}

extern "C" int tm_feed_forward_forward(const tm_feed_forward *f, void *out, void *saved,
                                       void *workspace, size_t workspace_bytes,
                                       hipStream_t stream) {
    if (const int rc = check(f))
        return rc;
    if (!f->T)
        return TM_OK;
    if (!f->x || !f->gate || !f->up || !f->down || !out || (uintptr_t)saved % 16)
        return TM_ERR_INVALID_ARGUMENT;
    if (!workspace || (uintptr_t)workspace % 16 ||
        workspace_bytes < tm_feed_forward_workspace_bytes(f))
        return TM_ERR_WORKSPACE;
    Args p = args(f->T, f->F, f->C);
    p.a[0] = f->x, p.a_l = f->x_l;
    p.b[0] = f->gate, p.b[1] = f->up, p.b_l = f->w_l;
    void *h = saved ? plane(*f, saved, planes(*f)) : workspace;
    p.out[0] = h, p.out_l = hidden_row(*f);
    if (saved)
        set_saved(*f, p, saved);
    char *part = (char *)workspace + hidden_bytes(*f);
    if (const int rc = product(*f, p, ff::kUp, plan_up(*f), part, stream))
        return rc;
    p = args(f->T, f->O, f->F);
    p.a[0] = h, p.a_l = hidden_row(*f);
    p.b[0] = f->down, p.b_l = f->down_l;
    p.out[0] = out, p.out_l = f->O, p.wide = wide(*f, out, f->O);
    return product(*f, p, ff::kDown, plan_down(*f), part, stream);
}

extern "C" size_t tm_feed_forward_backward_workspace_bytes(const tm_feed_forward *f) {
    if (check(f))
        return 0;
    return kScaleBytes + 2 * hidden_bytes(*f) +
           std::max({plan_hidden(*f).part, plan_input(*f).part, plan_weights(*f).part,
                     plan_output(*f).part});
}

extern "C" int tm_feed_forward_backward(const tm_feed_forward *f, const void *saved,
                                        const void *dout, int64_t do_l, void *dx, void *dgate,
                                        void *dup, void *ddown, void *workspace,
                                        size_t workspace_bytes, hipStream_t stream) {
    if (const int rc = check(f))
        return rc;
    const int64_t unit = 16 / size_of(*f);
    if (!dgate != !dup || (uintptr_t)dout % 16 || do_l % unit || do_l < 0 ||
        (do_l && do_l < f->O))
        return TM_ERR_INVALID_ARGUMENT;
    if (do_l >= TM_FF_MAX_ROW_BYTES / size_of(*f))
        return TM_ERR_UNSUPPORTED_SHAPE;
    if (!dgate && !ddown && (!dx || !f->T))
        return TM_OK;
    if (!workspace || (uintptr_t)workspace % 16 ||
        workspace_bytes < tm_feed_forward_backward_workspace_bytes(f))
        return TM_ERR_WORKSPACE;
    float *most = (float *)workspace;
    uint32_t *past = (uint32_t *)(most + ff::kMostParts);
    char *da = (char *)workspace + kScaleBytes;
    char *db = da + hidden_bytes(*f), *part = db + hidden_bytes(*f);
    Args p;
    const bool scaled = f->dtype == TM_F16 && f->T;
    if (f->T && (!f->x || !f->gate || !f->up || !f->down || !saved || (uintptr_t)saved % 16 ||
                 !dout))
        return TM_ERR_INVALID_ARGUMENT;
    if (f->T && (dx || dgate)) { // down's gradient needs h alone, which is saved
        if (scaled) {
            ff_most<<<dim3(ff::kMostParts), 256, 0, stream>>>((const _Float16 *)dout, do_l, f->T,
                                                             f->O, most, past);
            if (hipGetLastError() != hipSuccess)
                return TM_ERR_LAUNCH;
        }
        p = args(f->T, f->F, f->O);
        p.a[0] = dout, p.a_l = do_l;
        p.b[0] = f->down, p.b_l = f->down_l;
        p.da = da, p.db = db, p.out_l = hidden_row(*f);
        set_saved(*f, p, saved);
        if (scaled)
            p.most = most, p.past_out = past;
        const Plan how = plan_hidden(*f);
        if (const int rc = product(*f, p, ff::kHidden, how, part, stream))
            return rc;
        if (scaled) { // again, if the scale turns out too large; else its blocks end at once
            p.past = past;
            if (const int rc = product(*f, p, ff::kHidden, how, part, stream))
                return rc;
        }
        if (dx) {
            p = args(f->T, f->C, f->F);
            p.segments = 2;
            p.a[0] = da, p.a[1] = db, p.a_l = hidden_row(*f);
            p.b[0] = f->gate, p.b[1] = f->up, p.b_l = f->w_l;
            p.out[0] = dx, p.out_l = f->C, p.wide = wide(*f, dx, f->C);
            if (scaled)
                p.most = most, p.past = past;
            if (const int rc = product(*f, p, ff::kInput, plan_input(*f), part, stream))
                return rc;
        }
    }
    if (dgate) { // without rows: zeros, here and below
        p = args(f->F, f->C, f->T);
        p.batches = 2;
        p.a[0] = da, p.a[1] = db, p.a_l = hidden_row(*f);
        p.b[0] = p.b[1] = f->x, p.b_l = f->x_l;
        p.out[0] = dgate, p.out[1] = dup, p.out_l = f->C;
        p.wide = wide(*f, dgate, f->C) && wide(*f, dup, f->C);
        if (scaled)
            p.most = most, p.past = past;
        if (const int rc = product(*f, p, ff::kWeights, plan_weights(*f), part, stream))
            return rc;
    }
    if (ddown) {
        p = args(f->O, f->F, f->T);
        p.a[0] = dout, p.a_l = do_l;
        p.b[0] = f->T ? plane(*f, saved, planes(*f)) : nullptr, p.b_l = hidden_row(*f);
        p.out[0] = ddown, p.out_l = f->F, p.wide = wide(*f, ddown, f->F);
        if (const int rc = product(*f, p, ff::kWeights, plan_output(*f), part, stream))
            return rc;
    }
    return TM_OK;
}
