/*
 * mamba3_delta.h -- C ABI of the gated delta rule (gfx950): a recurrent mixer
 * with the scan's state layout that overwrites what a key held instead of
 * adding to it.
 *
 * Per sequence and head, with the state S [P, N] (f32), log decay g_t <= 0 and
 * write strength beta_t:
 *
 *     S~  = exp(g_t) S_{t-1}
 *     u_t = beta_t (v_t - S~ k_t)
 *     S_t = S~ + u_t k_t^T
 *     y_t = scale S_t q_t
 *
 * k and q are shared by heads / groups consecutive heads.  With qk_norm each
 * is brought to unit length first, x rsqrt(sum x^2 + 1e-6).
 *
 * Conventions are those of mamba3_ssm.h: caller-allocated device buffers,
 * asynchronous on `stream`, status codes with m3_last_error().  No reference
 * counterpart: the reference's mixers add outer products only.
 */
#ifndef MAMBA3_DELTA_H
#define MAMBA3_DELTA_H

#include <stddef.h>
#include <stdint.h>

#include "mamba3_ssm.h"

#ifdef __cplusplus
extern "C" {
#endif

typedef struct m3_delta_inputs {
    size_t batch, seq, heads, groups, head_dim, d_state;  /* B, T, H, G, P, N */
    int32_t dtype;                /* m3_dtype of q, k, v, y and their gradients */
    const void *q, *k;            /* [B, T, G, N] */
    const void *v;                /* [B, T, H, P] */
    /* elements between consecutive tokens' rows, a sequence seq rows after the
     * one before it (q, k and v read in place from the columns of a
     * projection); 0: contiguous */
    size_t q_stride, k_stride, v_stride;
    const float *g, *beta;        /* [B, T, H] */
    /* [B], or NULL: every sequence is seq tokens.  Tokens from lengths[b] on
     * are padding: nothing of them is used, whatever they hold, their y is
     * zero and so are their gradients.  Clamped to 0 .. seq. */
    const int32_t *lengths;
    const float *state;           /* S before the window [B, H, P, N], or NULL (zeros) */
    float scale;                  /* of y, usually N^-1/2 */
    int32_t qk_norm;
    void *workspace;              /* 256-byte aligned; may be NULL where none is needed */
    size_t workspace_bytes;
} m3_delta_inputs;

/* g and beta [rows, heads] from a projection's columns a and b (rows `stride`
 * elements apart, of `dtype`): g = -exp(a_log[h]) softplus(a + dt_bias[h]), beta =
 * sigmoid(b).  dt_bias [heads] may be NULL (zeros). */
m3_status m3_delta_gates(size_t rows, size_t heads, int32_t dtype, const void *a, const void *b,
                         size_t stride, const float *a_log, const float *dt_bias, float *g,
                         float *beta, void *stream);

/* The workspace of m3_delta_rule for these shapes; 0 where it needs none or
 * they are not covered. */
size_t m3_delta_rule_workspace_bytes(const m3_delta_inputs *in);

/* y [B, T, H, P] and, unless NULL, the state after the window [B, H, P, N]
 * (which may be in->state's own buffer).  head_dim up to 1024 and d_state up to
 * 256, else M3_ERR_UNSUPPORTED. */
m3_status m3_delta_rule(const m3_delta_inputs *in, void *y, float *state_out, void *stream);

/* One token a sequence on `state` [B, H, P, N] in place (in->seq is 1, in->state
 * and the workspace are not used): the serving step, one read and one write of
 * the state.  A sequence with lengths[b] = 0 keeps its state. */
m3_status m3_delta_step(const m3_delta_inputs *in, float *state, void *y, void *stream);

/* Gradients of m3_delta_rule.  dy [B, T, H, P] and dstate (of the state after
 * the window, or NULL) are given; dq, dk [B, T, G, N], dv [B, T, H, P] in the
 * inputs' type, dg, dbeta [B, T, H] and dstate0 [B, H, P, N] (NULL without
 * in->state) are written, all contiguous.  dq and dk are summed over the heads
 * that share a group.  d_state up to 128, else M3_ERR_UNSUPPORTED. */
typedef struct m3_delta_grads {
    const void *dy;
    const float *dstate;
    void *dq, *dk, *dv;
    float *dg, *dbeta;
    float *dstate0;
} m3_delta_grads;

size_t m3_delta_rule_backward_workspace_bytes(const m3_delta_inputs *in);
m3_status m3_delta_rule_backward(const m3_delta_inputs *in, const m3_delta_grads *grads, void *stream);

#ifdef __cplusplus
}
#endif

#endif /* MAMBA3_DELTA_H */
