/* Linear attention with one decay per head for MI355X (gfx950): chunked prefill, recurrent decode, and the commit of a
 * verify window's accepted rows. The reference has no such layer (its linear attention is the delta rule with a decay
 * per channel, glm53f_kda.h); these entry points stand beside it with the same conventions, the same pool of states and
 * the same device metadata, so that one engine can hold layers of both kinds.
 *
 * Per head h with g = log_decay[h], state S [value_dim][key_dim], rows t = 0, 1, ... of a request:
 *
 *     S_t = exp(g) * S_{t-1} + v_t k_t^T            o_t = scale * S_t q_t
 *
 * Conventions (as glm53f_kda.h): every pointer is a DEVICE pointer; strides and offsets count ELEMENTS; the return
 * value is a hipError_t as int: 0 on success, 1 (hipErrorInvalidValue) when the host rejects an argument, otherwise the
 * launch error. Launches are asynchronous on `stream` (NULL: the default stream) and go to the current device, which
 * has to be the pointers' and the stream's. Nothing is allocated, freed or synchronized inside; device metadata (cu_rows,
 * keep, state_off, log_decay) is not read on the host. Calls may be captured into a graph.
 *
 * Layouts (row major, elements):
 *   q, k         bf16 rows of [qk_heads][key_dim] at q + r*q_stride, k + r*k_stride
 *   v, out       bf16 rows of [heads][value_dim] at v + r*v_stride, out + r*out_stride
 *                (q, k and v may be column ranges of one projection row; out overlaps none of them)
 *   state        f32 or bf16 [heads][value_dim][key_dim] of request b at state + state_off[b]
 *   log_decay    f32 [heads], at most 0 (-inf: nothing is remembered; 0: nothing is forgotten)
 * Head h reads q and k of head h / (heads / qk_heads): groups of value heads may share them (qk_heads divides heads).
 * key_dim and value_dim are 64 or 128 each.
 * States are moved in pieces of 128 bits: their base pointers are 16-byte aligned and the offsets multiples of 8
 * elements. Row pointers and strides may be any (16-byte aligned rows are read faster).
 *
 * Numerics: the state is held in f32 through a call, whatever its stored type, and rounded to bf16 at most once, when
 * the call stores it. Products of bf16 values are exact; sums are f32. Outputs are rounded to bf16 once.
 * `glm53f_lin_chain_batch` and `glm53f_lin_advance_batch` give a state the same bits for the same rows, and with f32
 * states a window of R rows has the bits of R calls with one row. The chunked form agrees within f32 rounding of the
 * terms, not bit for bit. A value of q, k or v that is not finite does not reach earlier rows' outputs or
 * other requests; where it reaches, outputs and states are infinite or NaN, not always the one that the formula gives.
 */
#ifndef GLM53F_LIN_H
#define GLM53F_LIN_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

struct ihipStream_t;

/**
 * The recurrence row by row: decode steps (one row per request) and short windows. One layer, `batch` requests.
 *
 * cu_rows    int32 [batch + 1], non-decreasing: request b owns rows [cu_rows[b], cu_rows[b+1]) of q, k, v and out.
 *            A request without rows keeps its state (it is copied where state_out is another buffer). Rows that belong
 *            to no request are neither read nor written.
 * state_off  int64 [batch]: request b's state is state_in + state_off[b], written to state_out + state_off[b].
 *            Regions of different requests must not overlap, but may be the same where state_out is NULL (several windows
 *            behind one state).
 * state_out  the states behind the last row: equal to state_in (in place), disjoint from it, or NULL (not written: a
 *            verify window).
 */
int32_t glm53f_lin_chain_batch(int32_t heads, int32_t qk_heads, int32_t key_dim, int32_t value_dim, int32_t batch,
    const int32_t* cu_rows, const uint16_t* q, int64_t q_stride, const uint16_t* k, int64_t k_stride,
    const uint16_t* v, int64_t v_stride, const float* log_decay, float scale, const float* state_in,
    float* state_out, const int64_t* state_off, uint16_t* out, int64_t out_stride, struct ihipStream_t* stream);

/** glm53f_lin_chain_batch with bf16 states (state_in, state_out, state_off in bf16 elements). */
int32_t glm53f_lin_chain_batch_bf16state(int32_t heads, int32_t qk_heads, int32_t key_dim, int32_t value_dim,
    int32_t batch, const int32_t* cu_rows, const uint16_t* q, int64_t q_stride, const uint16_t* k, int64_t k_stride,
    const uint16_t* v, int64_t v_stride, const float* log_decay, float scale, const uint16_t* state_in,
    uint16_t* state_out, const int64_t* state_off, uint16_t* out, int64_t out_stride, struct ihipStream_t* stream);

/**
 * The commit of a verify round, every layer of every request: the first keep[b] rows of request b go into its state,
 * without outputs. Layer l (of `layers` >= 1) has its rows at k + l*k_layer_stride and v + l*v_layer_stride, its decays
 * at log_decay + l*heads, its states at state_in / state_out + l*state_layer_stride.
 * keep       int32 [batch], 0 <= keep[b] <= rows of b (values outside are taken to the nearer end): the counts that
 *            glm53f_spec_accept writes. 0 leaves the state as it is.
 * state_out  equal to state_in or disjoint from it.
 */
int32_t glm53f_lin_advance_batch(int32_t heads, int32_t qk_heads, int32_t key_dim, int32_t value_dim, int32_t layers,
    int32_t batch, const int32_t* cu_rows, const int32_t* keep, const uint16_t* k, int64_t k_stride,
    int64_t k_layer_stride, const uint16_t* v, int64_t v_stride, int64_t v_layer_stride, const float* log_decay,
    const float* state_in, float* state_out, int64_t state_layer_stride, const int64_t* state_off,
    struct ihipStream_t* stream);

/** glm53f_lin_advance_batch with bf16 states. */
int32_t glm53f_lin_advance_batch_bf16state(int32_t heads, int32_t qk_heads, int32_t key_dim, int32_t value_dim,
    int32_t layers, int32_t batch, const int32_t* cu_rows, const int32_t* keep, const uint16_t* k, int64_t k_stride,
    int64_t k_layer_stride, const uint16_t* v, int64_t v_stride, int64_t v_layer_stride, const float* log_decay,
    const uint16_t* state_in, uint16_t* state_out, int64_t state_layer_stride, const int64_t* state_off,
    struct ihipStream_t* stream);

/**
 * Bytes of workspace that glm53f_lin_prefill_batch needs for these sizes: 0 where it needs none (short prompts, or
 * enough heads and requests to fill the GPU), -1 on arguments that it would reject. For exactly these sizes: fewer
 * requests or rows may need more. Never more than 1,535 * key_dim * value_dim * 4, nor than
 * heads * batch * ceil(max_rows / 256) * key_dim * value_dim * 4: the smaller of the two serves every call up to these sizes.
 */
int64_t glm53f_lin_prefill_workspace_bytes(int32_t heads, int32_t key_dim, int32_t value_dim, int32_t batch,
    int32_t max_rows);

/**
 * The chunked form on the matrix cores: prompts, and verify windows (state_out NULL). Arguments as
 * glm53f_lin_chain_batch, and
 * max_rows   (host) at least the longest request's rows; a request with more has its further rows left out.
 * workspace  at least glm53f_lin_prefill_workspace_bytes bytes, 16-byte aligned (NULL where that is 0). Its contents do
 *            not matter before a call and mean nothing after it; calls that may run at the same time need one each.
 */
int32_t glm53f_lin_prefill_batch(int32_t heads, int32_t qk_heads, int32_t key_dim, int32_t value_dim, int32_t batch,
    const int32_t* cu_rows, int32_t max_rows, const uint16_t* q, int64_t q_stride, const uint16_t* k,
    int64_t k_stride, const uint16_t* v, int64_t v_stride, const float* log_decay, float scale,
    const float* state_in, float* state_out, const int64_t* state_off, uint16_t* out, int64_t out_stride,
    void* workspace, int64_t workspace_bytes, struct ihipStream_t* stream);

/** glm53f_lin_prefill_batch with bf16 states. */
int32_t glm53f_lin_prefill_batch_bf16state(int32_t heads, int32_t qk_heads, int32_t key_dim, int32_t value_dim,
    int32_t batch, const int32_t* cu_rows, int32_t max_rows, const uint16_t* q, int64_t q_stride, const uint16_t* k,
    int64_t k_stride, const uint16_t* v, int64_t v_stride, const float* log_decay, float scale,
    const uint16_t* state_in, uint16_t* state_out, const int64_t* state_off, uint16_t* out, int64_t out_stride,
    void* workspace, int64_t workspace_bytes, struct ihipStream_t* stream);

#ifdef __cplusplus
}
#endif

#endif
