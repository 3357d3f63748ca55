/*
 * mgx_policy.h -- C ABI of libmagical_hip.so, second part: what lies between a policy's action scores and mgx_engine_step()'s
 * actions.  Log probabilities of given actions with the entropy and the best alternatives, their gradient, and actions drawn with
 * given random numbers, for a batch of rows of n scores.
 *
 * Conventions are mgx.h's: plain pointers and sizes, buffers owned by the caller and borrowed for the call, mgx_status return codes,
 * all work enqueued on `stream`, nothing synchronises the host.  No call keeps anything for the next: calls on different streams,
 * devices and threads are independent, and a captured call can be replayed.  mgx_policy_last_error() is the text of the calling
 * thread's last failure here.
 *
 * The scores: `logits` points at element (0, 0) of rows x n values of type `dtype` (mgx_real), value (r, j) at r * row_stride + j
 * (elements; any stride >= 0: rows may overlap or coincide, as an expanded tensor's do; no alignment beyond the element's).  `mask`:
 * NULL, or u8 at r * mask_row_stride + j, 0 = action j is ruled out in row r.  An action is OPEN if its mask is not 0 and its
 * score is not -inf.  With the open scores x, m = max x, T = temperature:
 *     d_j = (x_j - m) / T,  s = sum e^d_j,   log p_j = d_j - log s,   entropy H = -sum p_j log p_j = log s - (sum d_j e^d_j) / s
 *   - an action that is not open has log p = -inf, takes no part in H and gets gradient 0;
 *   - a row without open actions has log p = -inf for every action, H = 0, no alternatives (-1), gradient 0, and action -1 is drawn;
 *   - a row with a NaN or +inf among the open scores (masked places may hold anything) has NaN for log p, H and the open places'
 *     gradient (unless nothing flows back into the row), no alternatives (-1), and action -1 is drawn.
 * Sums are held in 32 bits (drawing: in 64).  Each row's result depends on the row alone, and its last bits on how many rows and alternatives are
 * asked for, which decides how a row is shared out; it repeats bit for bit.
 */
#ifndef MGX_POLICY_H
#define MGX_POLICY_H
#include "mgx.h"
#ifdef __cplusplus
extern "C" {
#endif

enum mgx_real { MGX_REAL_F32 = 0, MGX_REAL_F16 = 1, MGX_REAL_BF16 = 2 };
enum mgx_policy_op { MGX_POLICY_LOG_PROBS = 0, MGX_POLICY_SAMPLE = 1 };
enum { MGX_POLICY_MAX_TOP = 64 };

const char *mgx_policy_last_error(void);
/* bytes of DEVICE scratch memory (16-byte aligned) that a call of this size needs, 0 if none; it is free again once the call's work
 * has run.  Two calls that may run at the same time need memory of their own. */
int64_t mgx_policy_workspace_bytes(int op, int dtype, int64_t rows, int64_t n, int top);
/* bytes of `stats` that the backward call of this size needs from the forward call, 0 if none (stats may then be NULL) */
int64_t mgx_policy_stats_bytes(int64_t rows, int64_t n);
/* actions: i32 or i64 [rows] (action_bytes 4 or 8); < 0: none given in this row (log_prob 0); >= n: NaN.  log_prob, entropy: f32 [rows].
 * stats: NULL, or f32 of mgx_policy_stats_bytes() for the backward call.  top (0 ... min(n, MGX_POLICY_MAX_TOP)): the best open actions of each row, best first,
 * equal scores by the lower index: top_actions i32 [rows][top] (-1: there are no more), top_log_probs f32 [rows][top] (-inf there). */
int mgx_policy_log_probs(int device, int dtype, const void *logits, int64_t rows, int64_t n, int64_t row_stride, const uint8_t *mask,
                         int64_t mask_row_stride, double temperature, const void *actions, int action_bytes, int top, float *log_prob,
                         float *entropy, float *stats, float *top_log_probs, int32_t *top_actions, void *workspace,
                         int64_t workspace_bytes, void *stream);
/* gradient of sum_r grad_log_prob[r] * log_prob[r] + grad_entropy[r] * entropy[r] to the scores, in their type: grad [rows][n], dense.
 * grad_log_prob / grad_entropy: f32, row r at r * stride (0: one value for all), NULL = zero; the other arguments are the forward
 * call's, stats and entropy its outputs.  A row whose given action is >= n has NaN at its open places, unless its grad_log_prob is 0; a row
 * into which nothing flows back (grad_log_prob 0 or no action given, grad_entropy 0) has gradient 0 whatever its scores. */
int mgx_policy_log_probs_backward(int device, int dtype, const void *logits, int64_t rows, int64_t n, int64_t row_stride,
                                  const uint8_t *mask, int64_t mask_row_stride, double temperature, const void *actions,
                                  int action_bytes, const float *stats, const float *entropy, const float *grad_log_prob,
                                  int64_t grad_log_prob_stride, const float *grad_entropy, int64_t grad_entropy_stride, void *grad,
                                  void *stream);
/* one action per row: the first j with p_0 + ... + p_j > u (in 64 bits: only a u within some n * 2^-53 of a border between two actions may fall on
 * either side of it, by how a row is shared out), u = uniforms[r] (f32 or f64: uniform_bytes 4 or 8) in [0, 1); a u below 0
 * or NaN counts as 0, a u of 1 or more draws the last action that can be drawn.  A probability below 2^-990 is none.  action: i32 [rows]; log_prob, entropy: f32 [rows]
 * (either may be NULL). */
int mgx_policy_sample(int device, int dtype, const void *logits, int64_t rows, int64_t n, int64_t row_stride, const uint8_t *mask,
                      int64_t mask_row_stride, double temperature, const void *uniforms, int uniform_bytes, int32_t *action,
                      float *log_prob, float *entropy, void *workspace, int64_t workspace_bytes, void *stream);

#ifdef __cplusplus
}
#endif
#endif /* MGX_POLICY_H */
