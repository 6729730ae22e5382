/*
 * learner_ops.h — C-ABI of the learner's operators: what stands between a policy's logits and the levels that
 * evc_step takes, and between a trajectory's rewards and a gradient step.
 *
 * Every call is asynchronous on `hip_stream` (a stream of `device`), allocates nothing, keeps nothing between
 * calls and may be captured into a graph.  Workspaces are the caller's, at least as large as the *_workspace
 * call for the same arguments says (0 = none, the pointer may be NULL), aligned to 16 bytes; a workspace is used by one call
 * at a time.  Returns 0, or a negative code with a text in lrn_last_error() (thread-local): -1 argument,
 * -2 no device, -4 HIP error.
 *
 * ROWS.  `rows = outer * inner` rows of `levels` logits; row (o, i) starts at o * stride_outer + i * stride_inner
 * ELEMENTS (strides are not negative), its logits are adjacent.  What lies between two rows may be read, and is not
 * used.  mask (NULL = all allowed): bytes, non-zero = allowed, at o * mask_outer + i * mask_inner + j * mask_level
 * (mask_level 0 or 1; strides of 0 broadcast).  What a masked place holds (infinities, NaN) is never used.  A logit of
 * -inf is a masked one.  Per-row arrays are contiguous [rows].
 *   m = max z_j, s = sum exp(z_j - m) over the allowed j
 *   logprob(l) = z_l - m - log s;   entropy = log s - sum exp(z_j - m) (z_j - m) / s
 * A row without an allowed level has nothing to decide: logprob 0, entropy 0, gradient 0, chosen level 0.
 * A NaN or +inf among the allowed logits makes the row's results NaN (the chosen level stays inside [0, levels)).
 */
#ifndef LEARNER_OPS_H
#define LEARNER_OPS_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define LRN_F32  0
#define LRN_BF16 1
#define LRN_F16  2
#define LRN_F64  3                 /* lrn_scan only */

#define LRN_MAX_TOP 64             /* alternatives per row */
#define LRN_SHORT_ROW 1024         /* rows of up to so many levels need no workspace, and lrn_score_backward no statistics */

const char* lrn_last_error(void);

typedef struct lrn_rows {
    const void* logits;
    int64_t outer, inner, levels;
    int64_t stride_outer, stride_inner;
    const uint8_t* mask;
    int64_t mask_outer, mask_inner;
    int32_t mask_level;
    int32_t dtype;
} lrn_rows;

/* The level with the largest logit + noise among the allowed ones (the lowest of equals), its log probability under
 * the logits alone and the row's entropy.  noise (NULL = none): float32, row (o, i) at o * noise_outer +
 * i * noise_inner, adjacent.  With Gumbel noise the level is a sample of the row's distribution.  Noise of -inf or NaN
 * puts a level behind all others of its row. */
int64_t lrn_choose_workspace(const lrn_rows* rows);
int lrn_choose(int32_t device, void* hip_stream, const lrn_rows* rows, const float* noise, int64_t noise_outer,
               int64_t noise_inner, int64_t* level_out, float* logprob_out, float* entropy_out, void* workspace,
               int64_t workspace_bytes);

/* Log probabilities of given levels (int64 [rows]; negative = the row is padding: logprob 0, no gradient through it;
 * >= levels: NaN; not allowed: -inf), entropies, and the `top` most probable alternatives in falling order, the lowest
 * of equals first ([rows][top] log probabilities and levels; behind the last allowed one: -inf and -1).
 * stat_out (NULL = not wanted): float32 [rows][2] = (m, s), what lrn_score_backward takes. */
int64_t lrn_score_workspace(const lrn_rows* rows, int32_t top);
int lrn_score(int32_t device, void* hip_stream, const lrn_rows* rows, const int64_t* level, float* logprob_out,
              float* entropy_out, float* stat_out, int32_t top, float* top_logprob_out, int64_t* top_level_out,
              void* workspace, int64_t workspace_bytes);
/* stat and entropy are lrn_score's for the same rows; not read (NULL) where levels <= LRN_SHORT_ROW, whose sums are computed again.
 * grad_out (the logits' type, contiguous [rows][levels]):
 *   g_logprob (1[j = level] - p_j) - g_entropy p_j (log p_j + entropy)
 * g_logprob / g_entropy: float32 [rows] with a stride of 1 or 0 elements (NULL = zero). */
int lrn_score_backward(int32_t device, void* hip_stream, const lrn_rows* rows, const int64_t* level, const float* stat,
                       const float* entropy, const float* g_logprob, int32_t g_logprob_stride, const float* g_entropy,
                       int32_t g_entropy_stride, void* grad_out);

/*
 * RECURRENCES over `steps` steps of `batch` sequences of `channels` values each; strides in elements (time, batch,
 * channel): time's of any sign, the others not negative, 0 = broadcast (inputs).
 *
 * lrn_scan:  h_t = a_t h_{t-1} + x_t,  t = 0 .. steps-1  (reverse: from the last step to the first; "before" and "last"
 * below are meant in that order).  a_t = gate_t (the type of x, or gate_const where gate is NULL), and exactly 0 where
 * resets (bytes, (time, batch) strides, NULL = none) says that the sequence starts anew: nothing of what came before
 * enters, not even a NaN (nor does it where the gate itself is exactly 0).  A gate that is not finite, where no reset
 * stands, makes the state NaN whatever it was.  Meant for |gate| <= 1: the products of larger gates over a run of steps must
 * stay in range.  A product of gates over many steps that underflows to 0 cuts as well: a NaN or an infinity of the state may
 * stay behind it.  initial [batch][channels]
 * contiguous (NULL = 0) is the state before the first step; final (NULL = not wanted) receives the last one.
 * initial / final are float32, float64 for LRN_F64; the state is carried in those types whatever the type of x and h.
 * h may not overlap an input.
 */
typedef struct lrn_seq {
    int64_t steps, batch, channels;
    int32_t reverse, dtype;
} lrn_seq;

typedef struct lrn_view {
    const void* data;
    int64_t st, sb, sc;
} lrn_view;

int64_t lrn_scan_workspace(const lrn_seq* seq);
int lrn_scan(int32_t device, void* hip_stream, const lrn_seq* seq, const lrn_view* x, const lrn_view* gate,
             double gate_const, const lrn_view* resets, const void* initial, const lrn_view* h_out, void* final_out,
             void* workspace, int64_t workspace_bytes);
/* Gradients: G_t = g_h_t + a_{t+1} G_{t+1} with g_final behind the last step;  grad_x = G, grad_gate_t = G_t h_{t-1}
 * (0 at a reset), grad_initial = a_0 G_0.  g_final NULL = zero; grad_gate (wanted only with a gate tensor; then h is read) and
 * grad_initial may be NULL.  h and g_final are not read where they are not needed.  grad_gate of LRN_BF16 / LRN_F16 is refused:
 * their h is rounded, lrn_scan_keep_backward has it. */
int lrn_scan_backward(int32_t device, void* hip_stream, const lrn_seq* seq, const lrn_view* gate, double gate_const,
                      const lrn_view* resets, const void* initial, const lrn_view* h, const lrn_view* g_h,
                      const void* g_final, const lrn_view* grad_x_out, const lrn_view* grad_gate_out,
                      void* grad_initial_out, void* workspace, int64_t workspace_bytes);

/* The two for LRN_BF16 / LRN_F16 with a gate's gradient, whose states are not to be rounded.  lrn_scan_keep is lrn_scan that also
 * writes every LRN_KEEP-th state as it is: kept, float32 with strides (element, batch, channel) that are not negative, has
 * (steps + LRN_KEEP - 1) / LRN_KEEP elements a column, of which the j-th holds the state before the step that has
 * (j + 1) * LRN_KEEP - 1 behind it (the last element, the first step's or none's, need not be written and is not read).
 * lrn_scan_keep_backward walks the states in between again from x; grad_gate_dtype: the sequence's, or LRN_F32 for a gradient that
 * is going to be summed (of a broadcast gate). */
#define LRN_KEEP 8
int lrn_scan_keep(int32_t device, void* hip_stream, const lrn_seq* seq, const lrn_view* x, const lrn_view* gate,
                  const lrn_view* resets, const void* initial, const lrn_view* h_out, const lrn_view* kept_out, void* final_out,
                  void* workspace, int64_t workspace_bytes);
int lrn_scan_keep_backward(int32_t device, void* hip_stream, const lrn_seq* seq, const lrn_view* x, const lrn_view* gate,
                           const lrn_view* resets, const void* initial, const lrn_view* kept, const lrn_view* g_h,
                           const void* g_final, const lrn_view* grad_x_out, const lrn_view* grad_gate_out, int32_t grad_gate_dtype,
                           void* grad_initial_out, void* workspace, int64_t workspace_bytes);

/* Generalised advantages of `steps` x `batch` (channels = 1, reverse ignored):
 *   d_t = r_t + gamma (1 - end_t) V_{t+1} - V_t,  A_t = d_t + gamma lam (1 - end_t) A_{t+1},  target_t = A_t + V_t
 * rewards: float64 or float32 (seq->dtype LRN_F64 / LRN_F32), values float32, ends bytes (non-zero: the episode ended with
 * this step), last_values [batch] float32 contiguous = V behind the last step.  Outputs float32.  The arithmetic is float64
 * for float64 rewards. */
int64_t lrn_advantages_workspace(const lrn_seq* seq);
int lrn_advantages(int32_t device, void* hip_stream, const lrn_seq* seq, const lrn_view* rewards, const lrn_view* values,
                   const lrn_view* ends, const float* last_values, double gamma, double lam, const lrn_view* advantage_out,
                   const lrn_view* target_out, void* workspace, int64_t workspace_bytes);

#ifdef __cplusplus
}
#endif
#endif /* LEARNER_OPS_H */
