/*
 * libpmb200 — operators of a transformer block on caller device buffers,
 * beside the complete nonlinear functions of pmb200.h: the norms around a
 * block fused with its gate and residual scale (forward and backward), the
 * product of a few tokens with a matrix of 4-bit weights, and the attention
 * of one new token per sequence over a paged key-value cache.  No counterpart
 * in the reference, whose nonlinear workloads end at FP32 RMSNorm and softmax
 * (cuda/nonlinear.cuh:59-89).
 *
 * Conventions as in pmb200.h: 0 or a negative PM_E_* code, the message in
 * pm_last_error(); pointers are device memory of the current device; `stream`
 * is a cudaStream_t on it; nothing is synchronized, allocated or kept, so
 * every call may be captured into a graph.  Scratch is the caller's, 256-byte
 * aligned, of the size the *_scratch_bytes function gives; its contents need
 * no initialisation, and two calls that may overlap need two.  Outputs do not
 * overlap inputs or scratch.  Elements are row-major with a unit inner
 * stride; the other strides are given in elements (weight rows: bytes).
 * Sums, norms, softmax statistics and weights are held in 32 bits and rounded
 * once, to the nearest even, where a 16-bit output is written.
 */
#ifndef PMB200_BLOCKS_H
#define PMB200_BLOCKS_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Element types. */
enum { PM_DT_F32 = 0, PM_DT_BF16 = 1, PM_DT_F16 = 2 };

/*
 * The boundary between two blocks, per row r of `rows` rows of `width`:
 *   p      = block * rsqrt(mean(block^2) + eps) * post_weight   (post_weight NULL: p = block)
 *   hidden = residual + scale * gate[r / (rows / gate_rows)] * p  (gate_rows 0: no gate)
 *   normed = hidden * rsqrt(mean(hidden^2) + eps) * pre_weight    (from the unrounded hidden)
 * gate_rows divides rows: 1 is one gate vector for every row, `rows` a gate
 * per element, between them one row per sequence of equally long ones.
 * stats (NULL: not wanted) receives the two reciprocal root mean squares of
 * every row, [rows, 2] in the order above (the first is 1 without a post
 * norm); the backward call reads them.  dtype is that of residual, block,
 * hidden and normed; each weight and the gate are of that type or PM_DT_F32.
 * rows 0 is allowed and does nothing.  hidden and normed are contiguous.
 * Squares are summed in 32 bits: where their sum passes 3.4e38 the row's
 * reciprocal root mean square is 0.
 */
typedef struct {
  int64_t rows, gate_rows;
  int64_t residual_stride, block_stride;   /* elements between rows, >= width */
  int32_t width;                           /* 1 .. 2^20 */
  int32_t dtype, pre_dtype, post_dtype, gate_dtype;
  float scale, eps;
  const void* residual;
  const void* block;
  const void* pre_weight;                  /* [width] */
  const void* post_weight;                 /* [width] or NULL */
  const void* gate;                        /* [gate_rows, width] contiguous, NULL exactly when gate_rows is 0 */
  void* hidden;
  void* normed;
  float* stats;
} pm_block_norm;

int pm_block_norm_device(const pm_block_norm* job, void* stream);

/*
 * The gradients of pm_block_norm_device from those of hidden and normed
 * (either may be NULL: zero).  `forward` is the forward job with its inputs
 * and stats (hidden and normed are not read and may be NULL).  grad_residual
 * and grad_block are contiguous [rows, width] of dtype; grad_pre, grad_post
 * and grad_gate have the types and shapes of what they belong to and any of
 * the three may be NULL (not wanted).  Sums over rows are in 32 bits and in
 * a fixed order: the same inputs give the same bits.
 */
typedef struct {
  int64_t grad_hidden_stride, grad_normed_stride;
  const void* grad_hidden;
  const void* grad_normed;
  void* grad_residual;
  void* grad_block;
  void* grad_pre;
  void* grad_post;
  void* grad_gate;
} pm_block_norm_grads;

size_t pm_block_norm_backward_scratch_bytes(int64_t rows, int64_t gate_rows, int32_t width);
int pm_block_norm_backward_device(const pm_block_norm* forward, const pm_block_norm_grads* grads, void* scratch,
                                  size_t scratch_bytes, void* stream);

/*
 * y[m, n] = sum_k x[m, k] * scales[n, k / group] * (q[n, k] - zero[n, k / group])
 * with q the 4-bit weights of row n, two to a byte, the even k in the low
 * half (an odd k leaves the last high half unread), and zero = zeros[n, k / group]
 * (0..15, the high half of the byte unread) or 8 where zeros is NULL.  dtype (x and y) is PM_DT_BF16 or
 * PM_DT_F16; scales are of that type or PM_DT_F32, [n, ceil(k / group)]
 * contiguous, as are zeros.  group is a multiple of 32; the last may be
 * partial.  Weights may be read in aligned pieces of 16 bytes that hold one of
 * theirs at least.  y is contiguous [tokens, n].  tokens 0 is allowed and does
 * nothing; the weights are read once for every 16 tokens.  A wait for a copy
 * that does not end within the limit (2 s) gives up, and what depends on it is
 * NaN.
 */
typedef struct {
  int32_t tokens, n, k, group;
  int32_t dtype, scales_dtype;
  int64_t x_stride;                        /* elements between tokens, >= k */
  int64_t weight_stride;                   /* bytes between weight rows, >= (k + 1) / 2, at most 2^23 */
  const void* x;
  const uint8_t* weight;
  const void* scales;
  const uint8_t* zeros;
  void* y;
} pm_matvec_w4;

/* Scratch for the current device: 0 where the product needs none (scratch may then be NULL). */
size_t pm_matvec_w4_scratch_bytes(int32_t tokens, int32_t n, int32_t k);
int pm_matvec_w4_device(const pm_matvec_w4* job, void* scratch, size_t scratch_bytes, void* stream);
/* Sets the limit of such a wait for the process's calls from now on, 0 the usual one; returns the limit before. */
uint64_t pm_matvec_w4_wait_limit(uint64_t nanoseconds);

/*
 * Attention of one query token per sequence over a paged cache:
 *   out[b, h] = sum_j softmax_j(scale * q[b, h] . K[b, j, g]) V[b, j, g],  g = h / (q_heads / kv_heads)
 * over the live positions j of sequence b: max(0, length - window) <= j <
 * length (window 0: all of them), position j being entry j % page_size of
 * page table[b, j / page_size].  A page index outside [0, n_pages), or a
 * position beyond the table, is absent: its positions are not live and
 * nothing there is read.  A sequence without a live position gives zeros and
 * a log sum of -infinity, and so does one whose scores are all -infinity.
 * Entries that are not live may hold anything; an infinite value of a live one
 * makes its element of out infinite, NaN where both signs meet.
 * lse (NULL: not wanted) receives log(sum_j exp(scale * q . K)), [batch, q_heads].
 * With new_k and new_v (both or neither, [batch, kv_heads, head_dim]) the
 * token's own key and value are written to position length - 1 of each
 * sequence (where its page is present) and attended to there; two sequences
 * must not share that entry, and no other position, of this sequence or of
 * another, may be found there.
 * A weight in PM_DT_F16 is held to 2^-39 of the sequence's largest at least.
 * dtype: PM_DT_BF16 or PM_DT_F16 for all of q, the caches, new_k, new_v and
 * out.  head_dim: a multiple of 8 up to 256; q, the caches, new_k and new_v are
 * 16-byte aligned and their strides multiples of 8 elements.  page_size: 1..65536.
 * out is contiguous [batch, q_heads, head_dim].  batch 0 does nothing.
 */
typedef struct {
  int32_t batch, q_heads, kv_heads, head_dim;
  int32_t page_size, n_pages, table_columns;
  int32_t dtype, window;
  float scale;
  int64_t q_stride, q_head_stride;
  int64_t k_page_stride, k_token_stride, k_head_stride;
  int64_t v_page_stride, v_token_stride, v_head_stride;
  int64_t new_k_stride, new_k_head_stride, new_v_stride, new_v_head_stride;
  int64_t table_stride;
  const void* q;
  void* k_cache;                           /* written only at the new token's entries */
  void* v_cache;
  const int32_t* table;                    /* [batch, table_columns] */
  const int32_t* lengths;                  /* [batch], the new token counted; <= 0: none */
  const void* new_k;
  const void* new_v;
  void* out;
  float* lse;
} pm_paged_attention;

size_t pm_paged_attention_scratch_bytes(int32_t batch, int32_t q_heads, int32_t kv_heads, int32_t head_dim);
int pm_paged_attention_device(const pm_paged_attention* job, void* scratch, size_t scratch_bytes, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* PMB200_BLOCKS_H */
