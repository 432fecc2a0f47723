/*
 * torchmatch_amd.h -- C ABI of the MI355X (gfx950) solver library
 * libtorchmatch_amd.so.
 *
 * Plain pointers and sizes only: every tensor argument is a device pointer
 * to contiguous row-major data, every size is an element count, and every
 * call is stream-ordered on the hipStream_t it is given (0 = null stream).
 * Nothing here allocates, frees or synchronises unless its comment says so.
 * Return values are TM_* codes below; kernels never raise.
 *
 * Reference interfaces replaced (paths relative to the torchmatch
 * repository root):
 *   tm_jv_dense_batch_f32   sources/torchmatch/assignment/cuda/dispatch.cu:137-177
 *                           (jonker_dense_batch_cuda) together with
 *                           assignment/cuda/cuda_common.cuh:215-284
 *                           (compute_inf_sentinel, rewrite_inf_to_sentinel);
 *                           results follow the CPU op
 *                           assignment/cpu/ops.cpp:176-289 bit for bit.
 *   tm_jv_compact_batch_f32 the CPU op assignment::jonker_compact_batch
 *                           (assignment/cpu/ops.cpp:431-433 with
 *                           jonker_compact_core.h:20-301), which has no
 *                           device counterpart in the reference; results
 *                           follow it bit for bit.
 *   tm_jv_unpack_i64        the unpack loop of solve_batch_unpacked,
 *                           assignment/cpu/ops.cpp:291-417 (the device side of
 *                           assignment::jonker_dense_batch_unpacked), which
 *                           assignment/_solve.py:124-164 restates in torch.
 *   tm_sinkhorn_prepare_f32 transport/matrix/_validate.py:58-63,108-110,149-156
 *                           (validate_cost's NaN / -inf checks, the marginal
 *                           sign checks, fuse_mask_into_cost),
 *                           transport/matrix/_schedule.py:68-69 (largest
 *                           finite cost) and _log_sinkhorn.py:36-46
 *                           (_inf_row_col_masks), fused into one pass.
 *   tm_sinkhorn_read_stats  the host readbacks (`.any()`, `.item()`) of
 *                           those checks, one synchronisation for all.
 *   tm_sinkhorn_iterate_f32 sources/torchmatch/transport/matrix/_log_sinkhorn.py:136-221
 *   tm_sinkhorn_f32         (log_sinkhorn_plan) and
 *   tm_sinkhorn_f64         transport/matrix/_unbalanced_sinkhorn.py:30-103
 *                           (unbalanced_sinkhorn_plan); the f64 entry for
 *                           float64 costs, which the reference iterates in
 *                           float64.
 */
#ifndef TORCHMATCH_AMD_H
#define TORCHMATCH_AMD_H

#include <hip/hip_runtime_api.h>
#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Return codes. */
enum {
    TM_OK = 0,
    TM_ERR_INVALID_ARGUMENT = 1, /* negative size, null pointer, bad scalar */
    TM_ERR_UNSUPPORTED_SHAPE = 2,/* shape beyond what the kernels handle */
    TM_ERR_WORKSPACE = 3,        /* workspace missing or too small */
    TM_ERR_LAUNCH = 4,           /* a kernel launch failed (hipGetLastError) */
    TM_ERR_NAN = 5,              /* input holds NaN (reported by tm_jv_check_status) */
    TM_ERR_NEG_INF = 6,          /* input holds -inf (reported by tm_jv_check_status) */
    TM_ERR_HIP = 7,              /* a HIP runtime call failed */
    TM_ERR_INTERNAL = 8          /* a kernel's iteration guard tripped (a bug) */
};

/* Status word bits written by tm_jv_dense_batch_f32 into *d_status. */
enum {
    TM_JV_FLAG_NAN = 1u,
    TM_JV_FLAG_NEG_INF = 2u,
    TM_JV_FLAG_POS_INF = 4u,
    TM_JV_FLAG_ANY_FINITE = 8u,
    TM_JV_FLAG_NEG_ZERO = 16u,  /* input holds -0.0 (informational) */
    /* Set in word [0] by the last write of a K <= 64, B <= 2048 launch whose
     * problems are all solved before its finishing workgroup ends (none holds
     * +inf): every output and both status words are then final, so a caller
     * that cleared word [0] before the launch may poll host-mapped status
     * words for this bit instead of synchronising the stream.  Launches that
     * do not set it are waited for by synchronising the stream. */
    TM_JV_FLAG_DONE = 0x80000000u
};

/* ---- batched Jonker-Volgenant (assignment::jonker_dense_batch) -------- */

/* Largest K = max(N, M) tm_jv_dense_batch_f32 accepts. */
int32_t tm_jv_max_k(void);

/* Device workspace tm_jv_dense_batch_f32 needs for a (B, N, M) batch. */
size_t tm_jv_workspace_bytes(int64_t B, int32_t N, int32_t M);

/* Workspace with which K = max(N, M) > 64 batches also take the prefill: the
 * column reduction and every row's cache of the augmenting row reduction
 * computed by many-wave launches before the solve, which then spends its
 * sequential steps on the reference order alone (C3, 64 x 512 x 768: about
 * 2.6 MB).  Equal to tm_jv_workspace_bytes for K <= 64.  Any workspace of
 * at least tm_jv_workspace_bytes is accepted; the result is the same, bit
 * for bit, with or without the prefill.  No counterpart in the reference:
 * its CPU op keeps thread-local scratch (ops.cpp:246-251). */
size_t tm_jv_workspace_bytes_prefill(int64_t B, int32_t N, int32_t M);

/* Solve B independent (N, M) float32 assignment problems.
 *   costs      device, (B, N, M) contiguous; +inf marks a forbidden pair
 *   out        device, (B, N) int64: row -> column, -1 for rows matched into
 *              padding columns (N > M); identical to the reference CPU op
 *   workspace  device, >= tm_jv_workspace_bytes(B, N, M), any contents
 *   d_status   two uint32 the kernels write with plain stores: device
 *              memory, or the device address of host-mapped pinned memory
 *              (hipHostGetDevicePointer), which saves the copy-back; [0]
 *              receives TM_JV_FLAG_* for the whole batch, [1] is non-zero if
 *              a solve hit its iteration guard
 * The +inf sentinel (max finite + 1) * (K + 1) is computed on the device over
 * the whole batch, as the reference does; no host round trip happens inside.
 * If the batch holds NaN or -inf, `out` is filled with -1 and the flag is set:
 * call tm_jv_check_status to turn the flags into TM_ERR_NAN / TM_ERR_NEG_INF.
 * B == 0, N == 0 or M == 0 launches nothing (the caller fills -1). */
int tm_jv_dense_batch_f32(const float *costs, int64_t B, int32_t N, int32_t M, int64_t *out,
                          void *workspace, size_t workspace_bytes, uint32_t *d_status,
                          hipStream_t stream);

/* tm_jv_dense_batch_f32, then the wait for its result, in one call: returns
 * once every output is final for work that follows on `stream`, with the
 * batch's status decoded (TM_OK, TM_ERR_NAN, TM_ERR_NEG_INF, TM_ERR_INTERNAL,
 * or a launch / HIP error); the replacement for the reference's launch plus
 * its status readback (dispatch.cu:137-177, cuda_common.cuh:241-249).  For
 * K <= 64 and B <= 2048 every solve workgroup also writes its problem's
 * summary to pinned host memory the library holds per host thread and
 * device, and the host folds those as they arrive, so a batch with no +inf,
 * NaN or -inf returns without a second launch or a stream synchronisation.
 * That memory (8,200 bytes per block) is the one allocation these entry
 * points make: a block is taken from a per-device pool at a thread's first
 * call on a device (allocated only when the pool is empty) and returned to
 * the pool when the thread exits, so the process holds one block per device
 * for each host thread that has called and is alive at once, and keeps the
 * blocks until it ends.
 * `replays` (host, may be NULL) receives the number of problems that left
 * the certified path for the exact replay on that path (0 otherwise).  Calls
 * on one host thread must not overlap (each returns before the next starts).
 * Same arguments, workspace and results as tm_jv_dense_batch_f32; no status
 * words are passed. */
int tm_jv_dense_batch_f32_sync(const float *costs, int64_t B, int32_t N, int32_t M,
                               int64_t *out, void *workspace, size_t workspace_bytes,
                               uint32_t *replays, hipStream_t stream);

/* The same for tm_jv_compact_batch_f32. */
int tm_jv_compact_batch_f32_sync(const float *costs, int64_t B, int32_t N, int32_t M,
                                 int64_t *out, void *workspace, size_t workspace_bytes,
                                 uint32_t *replays, hipStream_t stream);

/* tm_jv_dense_batch_f32 without a workspace argument and without any device
 * allocation.  No counterpart in the reference: it is for callers that cannot
 * allocate (code under graph capture, tight serving loops, harnesses that
 * forbid hipMalloc).  The workspace is a fixed device array inside the
 * library, tm_jv_noalloc_scratch_bytes() bytes per GPU (35,072), held from the
 * library's load until the process ends; its address is looked up once per
 * device on the first call for that device.  Calls that overlap on one GPU
 * share the array and race: order them (one stream, or events).  Arguments,
 * status words, results and error codes as tm_jv_dense_batch_f32;
 * TM_ERR_WORKSPACE if a shape would need more than the array holds (none
 * does: tm_jv_workspace_bytes never exceeds it). */
int tm_jv_dense_batch_f32_noalloc(const float *costs, int64_t B, int32_t N, int32_t M,
                                  int64_t *out, uint32_t *d_status, hipStream_t stream);

/* Size of the fixed device workspace tm_jv_dense_batch_f32_noalloc uses. */
size_t tm_jv_noalloc_scratch_bytes(void);

/* Largest K = max(N, M) tm_jv_compact_batch_f32 accepts. */
int32_t tm_jv_compact_max_k(void);

/* Solve B problems like tm_jv_dense_batch_f32 (same arguments, workspace,
 * status words and sentinel / padding rules) with the solver of
 * assignment::jonker_compact_batch instead: out is identical to that CPU op's
 * mapping, whose tie rules differ from the dense solver's. */
int tm_jv_compact_batch_f32(const float *costs, int64_t B, int32_t N, int32_t M, int64_t *out,
                            void *workspace, size_t workspace_bytes, uint32_t *d_status,
                            hipStream_t stream);

/* Problems of the last tm_jv_dense_batch_f32 / tm_jv_compact_batch_f32 call on
 * `workspace` (K <= 64) whose certified shortest-path solve did not prove a
 * unique optimum and that were solved again by the exact replay of the
 * reference's order (ties, near-ties).  Copies one word to *count and
 * synchronises `stream`.  A diagnostic with no counterpart in the reference.
 * TORCHMATCH_AMD_JV_CERTIFY=0 in the environment switches the certified path
 * off (every problem replays). */
int tm_jv_read_replays(const void *workspace, uint32_t *count, hipStream_t stream);

/* Copy the two status words to the host and synchronise `stream` (the only
 * host sync of the JV path, mirroring the reference's validation readback,
 * cuda_common.cuh:241-249).  Returns TM_OK, TM_ERR_NAN, TM_ERR_NEG_INF,
 * TM_ERR_INTERNAL or TM_ERR_HIP. */
int tm_jv_check_status(const uint32_t *d_status, hipStream_t stream);

/* The same verdict from status words already on the host (host-mapped
 * d_status after the caller synchronised the stream).  No HIP call. */
int tm_jv_status_code(const uint32_t *h_status);

/* Unpack B packed mappings (the `out` of tm_jv_dense_batch_f32: row -> column
 * in [0, M) or -1) into the tuple of assignment::jonker_dense_batch_unpacked:
 *   matches         device, (B, N, 2) int64: (row, col) of matched rows in row
 *                   order, -1 after n_matches[b] pairs
 *   unmatched_rows  device, (B, N) int64: unmatched rows, increasing, then -1
 *   unmatched_cols  device, (B, M) int64: columns no row took, increasing,
 *                   then -1
 *   n_matches       device, (B,) int64
 * Same contents as the reference CPU op (ops.cpp:387-414, -1 padding as its
 * at::full(-1) leaves).  M <= 4096. */
int tm_jv_unpack_i64(const int64_t *packed, int64_t B, int32_t N, int32_t M, int64_t *matches,
                     int64_t *unmatched_rows, int64_t *unmatched_cols, int64_t *n_matches,
                     hipStream_t stream);

/* ---- log-domain Sinkhorn (transport::log_sinkhorn / unbalanced_sinkhorn) */

/* Flag bits tm_sinkhorn_read_stats reports. */
enum {
    TM_SK_FLAG_NAN = 1u,          /* the cost holds NaN (before the mask) */
    TM_SK_FLAG_NEG_INF = 2u,      /* the cost holds -inf (before the mask) */
    TM_SK_FLAG_A_NEG = 4u,        /* a holds a negative entry */
    TM_SK_FLAG_B_NEG = 8u,        /* b holds a negative entry */
    TM_SK_FLAG_ANY_FINITE = 16u   /* the masked cost holds a finite entry */
};

/* Device workspace the Sinkhorn calls below need.  The size depends on the
 * form chosen for the shape (TORCHMATCH_AMD_SINKHORN_FUSED names a streaming
 * step, TORCHMATCH_AMD_SINKHORN_RESIDENT=0 switches the resident solve off); keep
 * those variables unchanged between this query and the calls that use the
 * workspace (a smaller workspace is refused with TM_ERR_WORKSPACE). */
size_t tm_sinkhorn_workspace_bytes(int64_t B, int64_t N, int64_t M);

/* First half of a solve: one pass over the (B, N, M) float32 cost and the
 * marginals, all on `stream`, no host synchronisation.
 *   cost       device (B, N, M); +inf = forbidden pair
 *   keep       device (B, N, M) bytes or NULL: pairs with keep == 0 are
 *              forbidden (the cost is read as +inf there), i.e. the
 *              reference's fuse_mask_into_cost (transport/matrix/
 *              _validate.py:149-156) without materialising the fused cost
 *   a, b       device marginals (B, N) and (B, M)
 *   k_eps      > 0: also write the log kernel -C/k_eps into the workspace
 *              (pass the same value to tm_sinkhorn_iterate_f32); 0: do not
 * The pass also records what the reference's validation and schedule read
 * from the cost (transport/matrix/_validate.py:58-63, 108-110 and
 * _schedule.py:68-69): NaN / -inf in the cost, negative marginal entries and
 * the largest finite (masked) cost.  tm_sinkhorn_read_stats fetches them. */
int tm_sinkhorn_prepare_f32(const float *cost, const uint8_t *keep, const float *a,
                            const float *b, int64_t B, int64_t N, int64_t M, float k_eps,
                            void *workspace, size_t workspace_bytes, hipStream_t stream);

/* Copy the statistics of the last tm_sinkhorn_prepare_f32 on `workspace` to
 * the host and synchronise `stream` (the only host sync of a solve).
 * *flags receives TM_SK_FLAG_* bits, *max_finite the largest finite masked
 * cost (-inf when TM_SK_FLAG_ANY_FINITE is clear). */
int tm_sinkhorn_read_stats(const void *workspace, int64_t B, int64_t N, int64_t M,
                           uint32_t *flags, float *max_finite, hipStream_t stream);

/* Second half: the log-domain Sinkhorn iteration of the reference over the
 * workspace tm_sinkhorn_prepare_f32 filled (same cost, keep, B, N, M), and
 * the log transport plan.
 *   eps_sched  HOST array of n_iter float64 epsilons (the reference schedule)
 *   rho        <= 0: balanced (log_sinkhorn); > 0: unbalanced with KL
 *              penalty rho (damping 1 / (1 + eps / rho) per step)
 *   k_eps      the k_eps given to tm_sinkhorn_prepare_f32
 *   log_plan   device (B, N, M) output, may be NULL to skip the plan
 *   log_u, log_v  device (B, N), (B, M) outputs: the final scaling
 *              potentials (f = -eps * log_u, g = -eps * log_v)
 * Matrices that fit the chip's registers are solved in one launch where the form
 * (below) allows it (cooperative when several workgroups share a problem; a
 * `stream` under graph capture takes the streaming steps).  Otherwise, with B >= 2, the steps of part of the batch
 * run on a side stream of the library's own (created on the first such call per
 * device of `stream`, default priority), forked and joined with events:
 * the call stays stream-ordered on `stream`.  TORCHMATCH_AMD_SINKHORN_GROUPS=1
 * keeps every launch on `stream`, and so does a `stream` under graph capture.
 * Threading: calls from several host threads, on the same or different
 * streams, are safe; each call holds a per-device lock from its fork to its
 * join, so the side streams never serve two callers' segments interleaved.
 * Calls that share a workspace must be ordered by the caller. */
int tm_sinkhorn_iterate_f32(const float *cost, const uint8_t *keep, int64_t B, int64_t N,
                            int64_t M, const double *eps_sched, int32_t n_iter, double rho,
                            float k_eps, float *log_plan, float *log_u, float *log_v,
                            void *workspace, size_t workspace_bytes, hipStream_t stream);

/* What the caller reads of a solve.  With TM_SK_PLAN, log_u and log_v may
 * differ from the plain calls' by a constant moved from one to the other
 * (float32: up to 3e-4 of their norm, float64: 5e-14), which the plan does
 * not show; every shape that fits the chip's
 * registers is then solved in one launch.  TM_SK_POTENTIALS (the plain calls)
 * does so only for float32 shapes whose steps carry float64 potentials (rows
 * of 128 columns and more, a multiple of four), TM_SK_STEPS never. */
enum { TM_SK_POTENTIALS = 0, TM_SK_PLAN = 1, TM_SK_STEPS = 2 };

/* What one form needs (the queries without a form: the most any needs). */
size_t tm_sinkhorn_workspace_bytes_form(int64_t B, int64_t N, int64_t M, int32_t form);
size_t tm_sinkhorn_f64_workspace_bytes_form(int64_t B, int64_t N, int64_t M, int32_t form);

/* The two halves with a form; give both the same. */
int tm_sinkhorn_prepare_form_f32(const float *cost, const uint8_t *keep, const float *a,
                                 const float *b, int64_t B, int64_t N, int64_t M, float k_eps,
                                 int32_t form, void *workspace, size_t workspace_bytes,
                                 hipStream_t stream);
int tm_sinkhorn_iterate_form_f32(const float *cost, const uint8_t *keep, int64_t B, int64_t N,
                                 int64_t M, const double *eps_sched, int32_t n_iter, double rho,
                                 float k_eps, int32_t form, float *log_plan, float *log_u,
                                 float *log_v, void *workspace, size_t workspace_bytes,
                                 hipStream_t stream);

/* Both halves without a mask and without reading the statistics back: the
 * cost must hold no NaN / -inf and the marginals must be non-negative.
 *   a, b       device marginals (B, N) and (B, M)
 *   other arguments as tm_sinkhorn_iterate_f32 */
int tm_sinkhorn_f32(const float *cost, const float *a, const float *b, int64_t B, int64_t N,
                    int64_t M, const double *eps_sched, int32_t n_iter, double rho,
                    float *log_plan, float *log_u, float *log_v, void *workspace,
                    size_t workspace_bytes, hipStream_t stream);

/* ---- float64 Sinkhorn ---------------------------------------------------
 * The reference iterates in the cost's dtype (transport/matrix/
 * _log_sinkhorn.py:184,191, _unbalanced_sinkhorn.py:60,67): a float64 cost
 * is solved in float64, with the same recurrence, shift rule, keep-previous
 * rule, damping and plan expression as tm_sinkhorn_iterate_f32.  The caller
 * validates the cost (no NaN / -inf), fuses any mask into it (+inf) and
 * builds the schedule; nothing is read back.
 *   cost, a, b, log_plan, log_u, log_v  device float64 tensors of the shapes
 *   and meanings of tm_sinkhorn_f32; log_plan may be NULL
 *   workspace  device, >= tm_sinkhorn_f64_workspace_bytes(B, N, M)
 * Any B: every launch strides its grid over the batch. */
size_t tm_sinkhorn_f64_workspace_bytes(int64_t B, int64_t N, int64_t M);
int tm_sinkhorn_f64(const double *cost, const double *a, const double *b, int64_t B,
                    int64_t N, int64_t M, const double *eps_sched, int32_t n_iter, double rho,
                    double *log_plan, double *log_u, double *log_v, void *workspace,
                    size_t workspace_bytes, hipStream_t stream);
/* The same with a form (TM_SK_PLAN: one launch where the matrix fits). */
int tm_sinkhorn_form_f64(const double *cost, const double *a, const double *b, int64_t B,
                         int64_t N, int64_t M, const double *eps_sched, int32_t n_iter,
                         double rho, int32_t form, double *log_plan, double *log_u,
                         double *log_v, void *workspace, size_t workspace_bytes,
                         hipStream_t stream);

/* ---- attention and rotation ---------------------------------------------
 * What produces the scores the solvers above work on: attention within and
 * between point sets, and the rotation of feature pairs by positions.  The
 * reference has no counterpart.  Nothing here reads anything back, so every
 * call may be captured into a graph. */

/* Element types of features, and of positions. */
enum { TM_BF16 = 0, TM_F16 = 1, TM_F32 = 2 };
enum { TM_POS_F32 = 0, TM_POS_I32 = 1, TM_POS_I64 = 2 };

/* One attention problem.  q is (B, Lq, H, D), k and v are (B, Lk, Hkv, D), Hkv
 * dividing H: query head h reads key head h / (H / Hkv).  They may be strided
 * (strides in elements, D contiguous); addresses and strides must be multiples
 * of 16 bytes and so must D (TM_ERR_INVALID_ARGUMENT, TM_ERR_UNSUPPORTED_SHAPE),
 * D at most tm_attention_max_head_dim(), rows must be less than
 * TM_ATTENTION_MAX_ROW_BYTES apart, and B H (Lq / 32) and B Hkv (Lk / 128), rounded
 * up, below TM_ATTENTION_MAX_BLOCKS.
 *
 *   s_ij = scale * q_i . k_j
 *   s_ij = cap * tanh(s_ij / cap)                       where cap > 0
 *   s_ij = s_ij - slopes[h] * |q_positions_i - k_positions_j|   (sum over axes)
 *   out_i = sum_j softmax_j(s_ij) v_j  over the j that query i sees
 *
 * Without positions the distance is that of indices, query i standing at
 * i + length - Lq.  Query i of batch row b sees key j where
 *   j < lengths[b] (Lk without lengths), and
 *   if causal: j <= i + length - Lq, or j < prefix[b], and
 *   with documents: q_docs_i == k_docs_j >= 0.
 * A query that sees nothing gets zeros, lse = -inf and no gradient.  Keys past
 * every limit and rows of negative documents may hold anything, NaN included. */
enum { TM_ATTENTION_MAX_ROW_BYTES = 1 << 26, TM_ATTENTION_MAX_BLOCKS = 1 << 23 };
/* |scale|, cap and, with a cap, |scale| / cap are 2^126 at most (TM_ERR_INVALID_ARGUMENT). */
enum { TM_ATTENTION_MAX_CAP_16 = 1024 }; /* 16-bit types: tanh is good to 2e-7 of the cap */
typedef struct tm_attention {
    const void *q, *k, *v;
    int64_t q_b, q_l, q_h, k_b, k_l, k_h, v_b, v_l, v_h;
    const float *slopes;                    /* (H) or NULL: no bias */
    const float *q_positions, *k_positions; /* (B, L, axes) or NULL; need slopes */
    const int32_t *q_docs, *k_docs;         /* (B, L) or NULL */
    const int32_t *prefix, *lengths;        /* (B) or NULL */
    int32_t dtype, B, Lq, Lk, H, Hkv, D, axes, causal;
    float scale, cap;
} tm_attention;

int32_t tm_attention_max_head_dim(void);

/* out: (B, Lq, H, D) contiguous, the inputs' type; out_low: what rounding took off
 * it, of the same shape and type, or NULL (16-bit types; the gradients are the
 * better for it); lse: (B, H, Lq) float32, the
 * natural logarithm of each row's sum, or NULL.  workspace: device, at least
 * tm_attention_workspace_bytes(a), 16-byte aligned, any contents. */
size_t tm_attention_workspace_bytes(const tm_attention *a);
int tm_attention_forward(const tm_attention *a, void *out, void *out_low, float *lse,
                         void *workspace, size_t workspace_bytes, hipStream_t stream);

/* Gradients of q, k and v (contiguous, the inputs' type) from out, out_low
 * (or NULL) and lse of the forward call and the output's gradient, (B, Lq, H, D) with its own strides.
 * The same call gives the same bits: nothing is added by atomics.
 * tm_attention_backward_lse also takes the gradient of lse, dlse: (B, H, Lq) float32, contiguous,
 * or NULL for none; what it holds for a row that sees nothing is not used. */
size_t tm_attention_backward_workspace_bytes(const tm_attention *a);
int tm_attention_backward(const tm_attention *a, const void *out, const void *out_low,
                          const float *lse, const void *dout, int64_t do_b, int64_t do_l,
                          int64_t do_h, void *dq, void *dk, void *dv, void *workspace, size_t workspace_bytes,
                          hipStream_t stream);
int tm_attention_backward_lse(const tm_attention *a, const void *out, const void *out_low,
                              const float *lse, const float *dlse, const void *dout, int64_t do_b,
                              int64_t do_l, int64_t do_h, void *dq, void *dk, void *dv,
                              void *workspace, size_t workspace_bytes, hipStream_t stream);

/* Rotation of feature pairs.  x is (B, L, H, D) of `dtype` with strides in
 * elements (D contiguous); out is (B, L, H, D), contiguous.  positions are
 * (B, L, axes) of `pos_type`, batch rows pos_b elements apart (0: shared).
 * sections[a] pairs turn by axis a: pair p of a token by the angle
 * positions[axis(p)] * freqs[p] (the opposite angle with `inverse`, which is the
 * gradient).  Pair p is features p and P + p, or 2p and 2p + 1 where
 * interleaved, P the number of pairs; the features past 2 P are copied.  P is at most 4096, H D
 * at most 2^24 and B L less than 2^24 (4096 / P), rounded down (TM_ERR_UNSUPPORTED_SHAPE). */
enum { TM_ROTATE_MAX_AXES = 4 };
typedef struct tm_rotation {
    const void *x, *positions;
    const float *freqs; /* (P) */
    int64_t x_b, x_l, x_h, pos_b;
    int32_t dtype, pos_type, B, L, H, D, axes, interleaved, inverse;
    int32_t sections[4];
} tm_rotation;
int tm_rotate(const tm_rotation *r, void *out, hipStream_t stream);

/* The same with each head normed first:
 *   y = R(x (mean_d x_d^2 + eps)^-1/2 w)
 * weight: (groups, D) contiguous, of weight_type (rotation.dtype or TM_F32), or NULL for ones; row g
 * is for heads[g] heads, which follow each other and make up all H.  D is at most
 * TM_NORM_MAX_HEAD_DIM and H TM_NORM_MAX_HEADS (TM_ERR_UNSUPPORTED_SHAPE), rotation.inverse 0.  Sums are float32.
 * out: (B, L, H, D), contiguous. */
enum { TM_NORM_MAX_GROUPS = 8, TM_NORM_MAX_HEAD_DIM = 512, TM_NORM_MAX_HEADS = 1 << 16 };
typedef struct tm_norm_rotation {
    tm_rotation rotation;
    const void *weight;
    int32_t weight_type, groups;
    int32_t heads[8];
    float eps;
} tm_norm_rotation;
int tm_norm_rotate(const tm_norm_rotation *n, void *out, hipStream_t stream);

/* Gradients from that of the output, (B, L, H, D) with its own strides: dx (B, L, H, D), contiguous,
 * and dweight, as weight; either may be NULL.  workspace (needed for dweight): device, at least
 * tm_norm_rotate_backward_workspace_bytes(n), 16-byte aligned, any contents.  The same call gives the
 * same bits. */
size_t tm_norm_rotate_backward_workspace_bytes(const tm_norm_rotation *n);
int tm_norm_rotate_backward(const tm_norm_rotation *n, const void *dout, int64_t do_b, int64_t do_l,
                            int64_t do_h, void *dx, void *dweight, void *workspace,
                            size_t workspace_bytes, hipStream_t stream);

/* Dropout of `count` elements that lie one after the other.  Element i stays where word i % 4 of the
 * ten-round Philox 4x32 generator is at least round(p 2^32); the counter's words are i / 4 (low, high) and
 * offset (low, high), the key's seed (low, high).
 *   out_i = residual_i + x_i / (1 - p) where it stays, residual_i elsewhere
 * residual may be NULL; out may be x or residual.  seed_at: where the seed lies on the device when
 * the kernel runs, or NULL for `seed`.  The gradient is the same call on the output's. */
int tm_dropout(const void *x, const void *residual, void *out, int64_t count, int32_t dtype, double p,
               uint64_t seed, const int64_t *seed_at, uint64_t offset, hipStream_t stream);

/* The gated feed-forward block on T rows:
 *   y = (act(x gate^T) * (x up^T)) down^T
 * x is (T, C), gate and up are (F, C), down is (O, F), of `dtype`, rows `_l` elements apart; addresses
 * and rows at multiples of 16 bytes, fewer than TM_FF_MAX_ROW_BYTES from row to row; where C (F for
 * down) elements do not fill whole units of 16 bytes, the last unit's rest is zeros.  Sums are float32; the
 * hidden features are rounded to `dtype` once, as are their gradients.  float16 holds these times a
 * power of two: what brings the largest finite |dout| to 1 .. 2, if that is up; the largest that keeps
 * every finite one within its range, if that one does not. */
enum { TM_SILU = 0, TM_GELU = 1, TM_GELU_TANH = 2, TM_RELU = 3 };
enum { TM_FF_MAX_ROW_BYTES = 1 << 23, TM_FF_MAX_BLOCKS = 1 << 22 };
typedef struct tm_feed_forward {
    const void *x, *gate, *up, *down;
    int64_t x_l, w_l, down_l; /* w_l: of gate and of up */
    int32_t dtype, activation, T, C, F, O;
} tm_feed_forward;

/* (rows, n) as the block takes it: rows of n elements, x_l apart, each followed by zeros up to 16
 * bytes, one after the other in out (16-byte aligned). */
int tm_pad_rows(const void *x, int64_t x_l, int64_t rows, int32_t n, int32_t dtype, void *out,
                hipStream_t stream);

/* out: (T, O), contiguous.  saved: for the gradients, tm_feed_forward_saved_bytes(f) bytes, or NULL.
 * workspace, saved: device, 16-byte aligned, any contents. */
size_t tm_feed_forward_workspace_bytes(const tm_feed_forward *f);
size_t tm_feed_forward_saved_bytes(const tm_feed_forward *f);
int tm_feed_forward_forward(const tm_feed_forward *f, void *out, void *saved, void *workspace,
                            size_t workspace_bytes, hipStream_t stream);

/* Gradients from that of the output, (T, O) with rows do_l elements apart as x's are: dx (T, C), dgate
 * and dup (F, C), ddown (O, F), contiguous; those not asked for are NULL, dgate and dup go together.
 * The same call gives the same bits: nothing is added by atomics. */
size_t tm_feed_forward_backward_workspace_bytes(const tm_feed_forward *f);
int tm_feed_forward_backward(const tm_feed_forward *f, const void *saved, const void *dout,
                             int64_t do_l, void *dx, void *dgate, void *dup, void *ddown,
                             void *workspace, size_t workspace_bytes, hipStream_t stream);

#ifdef __cplusplus
}
#endif

#endif /* TORCHMATCH_AMD_H */
