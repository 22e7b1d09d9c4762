/* The two ends of a speculative round for MI355X (gfx950): the LM head's logits as probabilities, and the verification
 * of drafted tokens against them, which gives the accepted counts (`keep`) that the commit entry points take
 * (glm53f_kda_replay_batch, glm53f_kda_select_batch_bf16state, glm53f_kda_conv_shift_batch of glm53f_kda.h and
 * glm53f_lin_advance_batch of glm53f_lin.h) and the next token of every request, without a copy to the host in between.
 *
 * Conventions (as glm53f_kda.h): device pointers; strides in ELEMENTS; the return value is a hipError_t as int32: 0 on
 * success, 1 (hipErrorInvalidValue) when the host rejects an argument, otherwise the launch error. Asynchronous on
 * `stream`, on the current device; nothing is allocated, freed or synchronized inside; device arrays are not read on the
 * host; may be captured into a graph. A workspace's contents do not matter before a call and mean nothing after it;
 * calls that may run at the same time need one each. A call takes at most 65,535 rows or requests and a vocabulary of at most
 * 2^30.
 */
#ifndef GLM53F_SPEC_H
#define GLM53F_SPEC_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

struct ihipStream_t;

/** Bytes of workspace of glm53f_spec_probs for these sizes, or fewer rows; -1 on arguments that it would reject. */
int64_t glm53f_spec_probs_workspace_bytes(int32_t rows, int32_t vocab);

/** probs[r][t] = softmax over t < vocab of logits[r][t] / temperature[r], for r < rows (0 succeeds without a launch).
 *  logits       bf16, or f32 when logits_f32 != 0, rows ldl >= vocab elements apart, any alignment
 *  temperature  f32 [rows], NULL: 1. A temperature that is not above 0 gives the row's greatest logit (the lowest index
 *               of equal ones; NaN is never the greatest) the probability 1 and every other 0.
 *  probs        f32, rows ldp >= vocab elements apart; may be the logits' own buffer where those are f32 and ldp == ldl,
 *               otherwise disjoint from them
 *  workspace    at least glm53f_spec_probs_workspace_bytes bytes, 16-byte aligned
 *  A logit of -inf has probability 0; a row of nothing else is all zeros. A NaN or +inf (above temperature 0) makes its
 *  row NaN. Numerics: the sums in f32, the probabilities rounded once. */
int32_t glm53f_spec_probs(int32_t rows, int32_t vocab, const void* logits, int32_t logits_f32, int64_t ldl,
                          const float* temperature, float* probs, int64_t ldp, void* workspace,
                          int64_t workspace_bytes, struct ihipStream_t* stream);

/** Bytes of workspace of glm53f_spec_accept for these sizes, or fewer requests; -1 on arguments that it would reject. */
int64_t glm53f_spec_accept_workspace_bytes(int32_t batch, int32_t vocab);

/** The verification of a round's drafted tokens (speculative sampling: what is emitted is distributed as the target).
 *  Request b owns window rows [cu_rows[b], cu_rows[b+1]), n of them: row 0 of the window is the last committed token,
 *  row i >= 1 the i-th drafted token.
 *  cu_rows  int32 [batch + 1], non-decreasing
 *  tokens   int32 [all rows]: the windows' tokens (row 0's is not read)
 *  target   f32 probabilities p, rows p_stride >= vocab apart: row r is the target's distribution behind row r
 *  draft    f32 probabilities q, rows q_stride >= vocab apart: row r (i >= 1) is the distribution that row r's token was
 *           drawn from. NULL: the drafts are certain (q is 1 at the token and 0 elsewhere).
 *  uniform  f32 [all rows] in [0, 1): row i >= 1 judges that row's token, row 0 draws the next token
 *  keep     int32 [batch]: 1 + the number of accepted tokens (the rows to commit); 0 for a request without rows
 *  next     int32 [batch]: the token that follows the kept rows; -1 for a request without rows
 *  Row i's token x is accepted iff every one before it is and uniform_i * q_i(x) < p_{i-1}(x); a token outside
 *  [0, vocab) never is. The next token is drawn from p of the last kept row, where a draft was rejected behind it from
 *  max(p - q, 0) with q of the rejected row: the lowest token whose cumulative weight exceeds uniform_0 times the whole.
 *  Weights that are not positive finite numbers count as 0. If max(p - q, 0) is 0 everywhere, p itself is taken; if
 *  that is 0 everywhere too, the next token is -1. All of it in 64 bits, in an order that depends on vocab alone.
 *  workspace  at least glm53f_spec_accept_workspace_bytes bytes, 16-byte aligned. batch == 0 succeeds without a launch. */
int32_t glm53f_spec_accept(int32_t batch, int32_t vocab, const int32_t* cu_rows, const int32_t* tokens,
                           const float* target, int64_t p_stride, const float* draft, int64_t q_stride,
                           const float* uniform, int32_t* keep, int32_t* next, void* workspace,
                           int64_t workspace_bytes, struct ihipStream_t* stream);

#ifdef __cplusplus
}
#endif

#endif
