/*
 * dit_train.h — C ABI of the operators that train (and serve) a layer of one's
 * own around the block on MI355X (gfx950): layer norm, attention to a text
 * encoder's states, and their gradients; the gradient of a projection's weight
 * from an input that was kept in 8 bits.  No counterpart in the reference, which
 * runs its block forward only and takes text into the block's own attention
 * (dit_vk.cpp:391-439).
 *
 *   y        = layer_norm(x)                       stats kept
 *   q, s     = quant(y)                            kept in place of y (dit_ops.h)
 *   queries  = product of q, s and a weight        (dit_ops.h, or dit_gemm_bf16)
 *   o, lse   = cross(queries, text keys, text values)
 *   ...
 *   dq, dk, dv = cross_grad(do, ...)
 *   dW       = grad_weight(dq, q, s)
 *   dx       = layer_norm_grad(dy, x, stats)       x in any of the types, 8 bits too
 *
 * Conventions as awa_capi.h: device pointers, stream-ordered and asynchronous,
 * 0 / AWA_EARG / AWA_EHIP, messages through awa_last_error of the context.
 * The calls allocate nothing and use no scratch of the context (a plan is made
 * once, ahead of them): what they need beside their outputs is d_work, memory of
 * the caller's of at least the bytes that the call's *_work function names, 256-byte
 * aligned (NULL where that is 0), not shared between calls that may overlap.  So they
 * may be captured into graphs, and calls on different streams may overlap.  Sums,
 * statistics and softmax are fp32; results are rounded once (to nearest even); the
 * same call gives the same bits.
 */
#ifndef SEEDVR2_DIT_TRAIN_H
#define SEEDVR2_DIT_TRAIN_H

#include <stdint.h>

#include "awa_capi.h"
#include "dit_ops.h"

#ifdef __cplusplus
extern "C" {
#endif

/* A third type of rows: e4m3 with a power-of-two scale per row and 128 columns, as
 * dit_quant_fp8 writes them with block_rows 1 (values, and words of scales). */
enum { DIT_FP8 = 2 };

/* ---- layer norm -------------------------------------------------------------
 *
 *   mean = sum x / K,   rstd = (sum (x - mean)^2 / K + eps)^(-1/2)
 *   y    = (x - mean) rstd w + b
 *
 * of each row x of d_x [M][K], type dtype_x (AWA_F32 or AWA_BF16), rows ldx elements
 * apart; y [M][K] of type dtype_y, rows ldy apart; d_w, d_b fp32 [K], either may be
 * NULL (1 and 0).  d_stats (may be NULL): fp32 [M][2], each row's mean and rstd, for
 * the gradient.  M may be 0, K is 1 .. DIT_NORM_COLS_MAX.  Tensors need their
 * elements' alignment only (d_stats 8 bytes); y may be x itself (same type and stride).
 * A NaN or infinity makes its row NaN; a row whose squares sum past 2^128 has rstd 0
 * (y = b).  Rejected (AWA_EARG): sizes out of range, a stride under K (for M > 1), eps
 * negative or not finite, y over an input otherwise. */
enum { DIT_NORM_COLS_MAX = 16384 };
int dit_layer_norm(awa_ctx* ctx, int dtype_x, const void* d_x, int64_t ldx, const float* d_w, const float* d_b,
                   float eps, int dtype_y, void* d_y, int64_t ldy, float* d_stats, int M, int K,
                   awa_stream_t stream);

/* The gradient: with h = (x - mean) rstd from d_stats and a = dy w,
 *   dx = rstd (a - sum a / K - h sum (a h) / K),  dw = sum over rows dy h,  db = sum over rows dy.
 * dy, x, dx are [M][K] with their own types and strides; x may be 8-bit rows (dtype_x
 * DIT_FP8: d_x [M][K padded to 128] 16-byte aligned, d_xs words as dit_ops.h, ld_xs from
 * group to group; ldx is ignored; otherwise d_xs is NULL).  d_w may be NULL (1).  d_dx may
 * be NULL, and d_dw and d_db (fp32 [K], written, not added to), but not all three.  dx may
 * be dy, or x, itself (same type and stride).  M = 0: dw and db become 0.  The sums over
 * rows do not depend on timing: equal calls give equal bits. */
int64_t dit_layer_norm_grad_work(int M, int K); /* bytes of d_work; 0 without d_dw and d_db; negative: bad sizes */
int dit_layer_norm_grad(awa_ctx* ctx, int dtype_dy, const void* d_dy, int64_t lddy, int dtype_x, const void* d_x,
                        int64_t ldx, const uint32_t* d_xs, int64_t ld_xs, const float* d_stats, const float* d_w,
                        int dtype_dx, void* d_dx, int64_t lddx, float* d_dw, float* d_db, void* d_work,
                        int64_t work_bytes, int M, int K, awa_stream_t stream);

/* ---- a weight's gradient from 8-bit rows ------------------------------------
 *
 *   dW[n][k] = sum over m of dy[m][n] x[m][k]   (+ dW[n][k] before, with add)
 *   db[n]    = sum over m of dy[m][n]           (+ db[n] before, with add)
 *
 * dy [M][N] of type dtype_dy (AWA_F32 or AWA_BF16), rows lddy (at most DIT_OPS_COLS_MAX) apart; x [M][K] in 8-bit
 * rows (d_q [M][K padded to 128], 16-byte aligned, d_s words, ld_s from group to group).
 * dW [N][K] of type dtype_w, rows ldw apart; db fp32 [N], may be NULL.  add needs fp32 dW.
 * Every product enters the sums whole, for fp32 dy too (as three bf16 parts: values of x
 * under 2^-126 count as zero, and parts of dy as well).  M = 0: dW and db become 0 (or stay,
 * with add).  Tensors need their elements' alignment only. */
int64_t dit_grad_weight_work(int dtype_dy, int dtype_w, int M, int N, int K); /* bytes of d_work; negative: bad sizes */
int dit_grad_weight_fp8(awa_ctx* ctx, int dtype_dy, const void* d_dy, int64_t lddy, const uint8_t* d_q,
                        const uint32_t* d_s, int64_t ld_s, int dtype_w, void* d_dw, int64_t ldw, float* d_db,
                        int add, void* d_work, int64_t work_bytes, int M, int N, int K, awa_stream_t stream);

/* ---- attention to states of another length ----------------------------------
 *
 * A plan holds a batch's lengths: sequence i has query rows q_at[i] .. q_at[i] +
 * q_len[i] - 1 and key rows k_at[i] .. k_at[i] + k_len[i] - 1, any of them 0 long.
 * Query rows of different sequences do not overlap; key rows are the same for two
 * sequences (text that several clips share) or do not overlap either.  heads is a
 * multiple of kv_heads: head h reads key head h / (heads / kv_heads).  head_d is a
 * multiple of 8 up to 128.  The arrays are the host's and are copied.
 *
 *   S = scale q k^T over the sequence's keys whose mask byte is not 0 (all, without a mask)
 *   P = softmax of each row,  out = P v,  lse = log sum exp S
 *
 * A row for which no key is left, or whose scores are all -infinity, gets zeros, lse
 * -infinity, and no gradient, whatever it, its dout, and the keys and values that made it so, hold
 * (so does a row whose given lse is -infinity); masked keys (whatever they hold, NaN and infinities too)
 * take no part and get gradients of zero.  A row with a NaN or +infinity among its scores, or whose largest
 * score times log2(e) is past fp32, is NaN, its lse too.  Rows of tensors that belong to no sequence are
 * neither read nor written. */
typedef struct dit_cross dit_cross;
enum { DIT_CROSS_SEQ_MAX = 65536, DIT_CROSS_HEADS_MAX = 1024, DIT_CROSS_HEAD_D_MAX = 128 };
/* Allocates on the context's device and waits for the copy of its tables: not while a
 * stream is captured.  Rows reach at most DIT_OPS_ROWS_MAX.  A batch of about 2^23 blocks
 * of 64 keys (by key heads) or 2^24 of 128 query rows (by heads; a sequence's last ones count whole), or more, is rejected. */
int dit_cross_create(awa_ctx* ctx, int n_seq, const int64_t* h_q_at, const int64_t* h_q_len, const int64_t* h_k_at,
                     const int64_t* h_k_len, int heads, int kv_heads, int head_d, dit_cross** out);
/* Frees the tables; calls that use them must have finished (graphs too), and no stream may be capturing. */
void dit_cross_destroy(dit_cross* plan);
/* For a caller that does not know whether they have (a garbage collector), at any time: the plan is not used again; its
 * tables are freed when the next plan is made on its device, or, if a call that used them was captured, not before the
 * process ends. */
void dit_cross_drop(dit_cross* plan);
enum { DIT_CROSS_WHOLE = 256 };
/* Bytes of d_work of dit_cross_forward (grad 0) or dit_cross_grad (1), the same with DIT_CROSS_WHOLE; negative: bad arguments. */
int64_t dit_cross_work(const dit_cross* plan, int dtype, int grad);

/* A tensor [rows][heads][head_d]; strides in elements, a head's channels contiguous.  The
 * address and both strides are multiples of 16 bytes, strides not negative, row strides at most
 * DIT_OPS_COLS_MAX, head strides at most 2^36. */
typedef struct {
    void* p;
    int64_t row, head;
} dit_heads;

/* d_mask: NULL, or a byte per key row; scale: 1e-30 .. 1e30; d_lse: NULL, or fp32 [heads][ld_lse],
 * ld_lse at least the plan's last query row + 1.  dtype AWA_F32 or AWA_BF16, of all tensors.
 * bf16: scores and sums are fp32, probabilities are rounded to bf16 before they meet v (2^-8 of each at most).  dtype
 * AWA_BF16 | DIT_CROSS_WHOLE: they meet it with 16 bits (2^-16 of each), so that rounding the result is what is left
 * (AWA_F32 takes the flag too, and rounds nothing without it). */
int dit_cross_forward(awa_ctx* ctx, const dit_cross* plan, int dtype, const dit_heads* q, const dit_heads* k,
                      const dit_heads* v, const uint8_t* d_mask, float scale, const dit_heads* out, float* d_lse,
                      int64_t ld_lse, void* d_work, int64_t work_bytes, awa_stream_t stream);

/* Gradients dq, dk, dv for d_out, given the forward's inputs and results (out and lse): all written, none
 * added to; keys of several heads, or sequences, get the sum over them.  With P and S as above,
 *   dv = P^T dout, dS = P (dout v^T - rowsum(dout out)), dq = scale dS k, dk = scale dS^T q
 * bf16: P and dS are rounded to bf16 before they meet the tensors, or with DIT_CROSS_WHOLE have 16 bits, as above. */
int dit_cross_grad(awa_ctx* ctx, const dit_cross* plan, int dtype, const dit_heads* dout, const dit_heads* q,
                   const dit_heads* k, const dit_heads* v, const dit_heads* out, const float* d_lse, int64_t ld_lse,
                   const uint8_t* d_mask, float scale, const dit_heads* dq, const dit_heads* dk, const dit_heads* dv,
                   void* d_work, int64_t work_bytes, awa_stream_t stream);

#ifdef __cplusplus
}
#endif
#endif
