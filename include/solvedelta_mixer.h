/* SolveDelta mixer frontend and readout, and the operators of the model around the
 * layer, on MI355X (gfx950): C-ABI of libsolvedelta_hip.so, next to the operator
 * entry points of solvedelta.h.
 *
 * The reference runs these pieces through third-party CUDA/Triton code; each
 * entry point here replaces one call site:
 *   - sd_conv4_silu_fwd / _bwd  <- causal_conv1d_fn(x^T, conv_weight, initial_states,
 *                                  return_final_states, activation="silu") in
 *                                  causallsso/model.py:119-136 (CPU semantics :146-164);
 *   - sd_kda_gate_fwd / _bwd    <- fla.ops.kda.gate.fused_kda_gate in
 *                                  causallsso/model.py:375-383 (its CPU form :384-390);
 *   - sd_rmsnorm_gated_fwd/_bwd <- layer_norm_gated_fwd / _bwd (rms, sigmoid) in
 *                                  causallsso/ops/norm_gate.py:46-150 (definition :20-43).
 *
 * Layouts: bf16 activations, FP32 parameters and parameter gradients.  Entry
 * points enqueue on `stream`, never allocate or synchronise, and return 0 or an
 * SD_ERR_* code of solvedelta.h.  Parameter gradients are reduced in two
 * deterministic stages through the caller's workspace (*_workspace_bytes).
 */
#ifndef SOLVEDELTA_MIXER_H
#define SOLVEDELTA_MIXER_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Causal depthwise conv4 + SiLU over T tokens of D channels:
 *   y[b,t,d] = silu(sum_k w[d,k] xs[b,t-3+k,d]), xs[b,-3..-1,:] = init[b,:,0..2] (or 0).
 * x: bf16, element (b,t,d) at x[b*x_sb + t*x_st + d]; w: fp32 [D][4];
 * init, final_state: bf16 [B][D][3], nullable; y: bf16 [B][T][D] contiguous.
 * final_state[b,d,m] = xs[b,T-3+m,d]. */
int sd_conv4_silu_fwd(int B, int T, int D, const void *x, int64_t x_sb, int64_t x_st,
                      const float *w, const void *init, void *y, void *final_state,
                      void *stream);
size_t sd_conv4_workspace_bytes(int B, int T, int D);
/* dy: bf16 [B][T][D]; dfinal: bf16 [B][D][3] nullable; dx: bf16 [B][T][D];
 * dw: fp32 [D][4]; dinit: fp32 [B][D][3] nullable. */
int sd_conv4_silu_bwd(int B, int T, int D, const void *x, int64_t x_sb, int64_t x_st,
                      const float *w, const void *init, const void *dy, const void *dfinal,
                      void *dx, float *dw, float *dinit, void *workspace,
                      size_t workspace_bytes, void *stream);

/* conv4 + SiLU under valid / reset masks (uint8 [B,T], element (b,t) at
 * m[b*m_sb + t*m_st], each nullable), the reference's CPU loop
 * (causallsso/model.py:146-164) that its varlen path reproduces by repacking
 * (model.py:166-220, packing.py:130-132): a reset on a valid token zeroes the
 * state first, an invalid token emits 0 and keeps the state, a valid token
 * emits silu(w . [state, x_t]) and shifts x_t in.  No repacking, no host sync.
 * Other arguments as sd_conv4_silu_fwd / _bwd; dx of invalid tokens is 0. */
int sd_conv4_silu_masked_fwd(int B, int T, int D, const void *x, int64_t x_sb, int64_t x_st,
                             const float *w, const void *init, const uint8_t *valid,
                             const uint8_t *reset, int64_t m_sb, int64_t m_st, void *y,
                             void *final_state, void *stream);
/* The backward's workspace: sd_conv4_masked_bwd_workspace_bytes for rows of T
 * tokens; sd_conv4_masked_workspace_bytes is its bound over every T. */
size_t sd_conv4_masked_bwd_workspace_bytes(int B, int T, int D);
size_t sd_conv4_masked_workspace_bytes(int B, int D);
int sd_conv4_silu_masked_bwd(int B, int T, int D, const void *x, int64_t x_sb, int64_t x_st,
                             const float *w, const void *init, const uint8_t *valid,
                             const uint8_t *reset, int64_t m_sb, int64_t m_st, const void *dy,
                             const void *dfinal, void *dx, float *dw, float *dinit,
                             void *workspace, size_t workspace_bytes, void *stream);

/* KDA decay gate over N rows of H*r columns:
 *   out[n,h*r+c] = -exp(log_rate[h]) * softplus(raw[n*raw_row_stride + h*r+c] + bias[h*r+c])
 * (softplus(x) = x above 20).  raw: bf16; out: fp32 [N][H*r]. */
int sd_kda_gate_fwd(int N, int H, int r, const void *raw, int64_t raw_row_stride,
                    const float *log_rate, const float *bias, float *out, void *stream);
size_t sd_kda_gate_workspace_bytes(int N, int H, int r);
/* dout: fp32 [N][H*r]; draw: bf16 [N][H*r]; dlog_rate fp32 [H]; dbias fp32 [H*r]. */
int sd_kda_gate_bwd(int N, int H, int r, const void *raw, int64_t raw_row_stride,
                    const float *log_rate, const float *bias, const float *dout, void *draw,
                    float *dlog_rate, float *dbias, void *workspace, size_t workspace_bytes,
                    void *stream);

/* Sigmoid-gated RMSNorm over N rows of width D <= 256 (contiguous bf16):
 *   y = x * rsqrt(mean(x^2) + eps) * weight * sigmoid(gate);  rstd fp32 [N] nullable. */
int sd_rmsnorm_gated_fwd(int N, int D, float eps, const void *x, const void *gate,
                         const float *weight, void *y, float *rstd, void *stream);
size_t sd_rmsnorm_gated_workspace_bytes(int N, int D);
/* dy: bf16 [N][D]; dx, dgate: bf16 [N][D]; dweight fp32 [D];
 * y: bf16 [N][D] nullable, the recomputed forward output (for a following Linear). */
int sd_rmsnorm_gated_bwd(int N, int D, float eps, const void *x, const void *gate,
                         const float *weight, const void *dy, void *dx, void *dgate,
                         float *dweight, void *y, void *workspace, size_t workspace_bytes,
                         void *stream);

/* ---- operators of the model shell around the layer ---------------------- */

/* Gated feed-forward block (causallsso/modeling_solvedelta.py:31-100) over N tokens:
 *   y = (silu(x Wg^T) * (x Wu^T)) Wd^T
 * x: bf16 [N][D], row n at x + n*x_st; gate_up: bf16 [2I][D] (Wg's rows, then Wu's), row
 * stride gate_up_st; down: bf16 [O][I], row stride down_st.  Strides count elements and are
 * at least the row's width; columns are contiguous. */
typedef struct {
  int64_t N;
  int D, I, O;
  const void *x; int64_t x_st;
  const void *gate_up; int64_t gate_up_st;
  const void *down; int64_t down_st;
} sd_ffn;
/* y: bf16 [N][O] contiguous.  saved: sd_ffn_saved_bytes, what sd_ffn_bwd reads; null where no
 * backward follows.  The sizes go by the shape, the strides and the addresses' alignment. */
size_t sd_ffn_saved_bytes(const sd_ffn *f);
size_t sd_ffn_fwd_workspace_bytes(const sd_ffn *f);
int sd_ffn_fwd(const sd_ffn *f, void *y, void *saved, void *workspace, size_t workspace_bytes,
               void *stream);
/* dy: bf16 [N][O], row stride dy_st; dx: bf16 [N][D]; dgate_up: bf16 [2I][D]; ddown: bf16
 * [O][I], contiguous, each nullable. */
size_t sd_ffn_bwd_workspace_bytes(const sd_ffn *f, const void *dy, int64_t dy_st);
int sd_ffn_bwd(const sd_ffn *f, const void *saved, const void *dy, int64_t dy_st, void *dx,
               void *dgate_up, void *ddown, void *workspace, size_t workspace_bytes,
               void *stream);

/* Row-wise quantisation to 8 bits: scale[n] = max_k |x[n,k]| / 127, q = rint(x / scale) (a
 * zero row: scale 0, q 0).  x: bf16, or FP32 if is_fp32, row stride x_st; q: row stride q_st.
 * A row that holds an infinity or a NaN gets the scale NaN. */
int sd_quantize_int8(int64_t N, int K, int is_fp32, const void *x, int64_t x_st, int8_t *q,
                     int64_t q_st, float *scale, void *stream);
/* y[n,o] = s_n w_scale[o] sum_k q[n,k] w[o,k] + bias[o], (q, s) the rows of x quantised as
 * above.  x: bf16 [N][K], row stride x_st; w: int8 [O][K], row stride w_st; bias: bf16 [O],
 * nullable; y: bf16 [N][O] contiguous.  K <= 132104: sums stay within 32 bits, of weights of -128 too. */
size_t sd_linear_int8_workspace_bytes(int64_t N, int K, int O, const void *w, int64_t w_st);
int sd_linear_int8(int64_t N, int K, int O, const void *x, int64_t x_st, const int8_t *w,
                   int64_t w_st, const float *w_scale, const void *bias, void *y,
                   void *workspace, size_t workspace_bytes, void *stream);

/* How a product of M x N outputs and rows of k_bytes is cut, for tests and profiles.  plan[0]: the
 * tile, 0 is 256x256, 1 and 2 are 128x128, 3 is 64x64; plan[1]: how many tiles are done whole;
 * plan[2]: how many workgroups share the others, which a second kernel joins. */
int sd_product_plan(int64_t M, int64_t N, int64_t k_bytes, int plan[3]);

/* One token per row of logits [B][V] (bf16, or FP32 if is_fp32; row stride logits_st), from
 * uniform numbers noise [B][V] (FP32, row stride noise_st; read between 2^-25 and 1 - 2^-24).
 * settings: temperature, top_k, top_p, min_p, in this order; each is `value` for all rows, or
 * rows[b] (FP32; int64 for top_k) where rows is not null.  z = (l - max l) / temperature;
 * tokens rank by (logit descending, index ascending); kept are the first top_k (all if
 * top_k <= 0), of these those whose predecessors hold less than top_p of the top_k's mass
 * sum exp(z) (all if top_p >= 1), of these those with z >= log(min_p) (all if min_p <= 0).
 * token[b]: the kept token with the largest z - log(-log noise), the lowest index of equals;
 * at a temperature that is not positive, rank 0; -1 if every logit is -infinity or NaN.
 * Masses are FP32 exponentials, each within 2^-17 of itself down to 2^-52 of the largest, and
 * their sums are right to 2^-28 of the largest.  V <= 2^22. */
typedef struct {
  double value;
  const void *rows;
} sd_sample_setting;
int sd_sample_tokens(int B, int V, int is_fp32, const void *logits, int64_t logits_st,
                     const float *noise, int64_t noise_st, const sd_sample_setting *settings,
                     int64_t *token, void *stream);

#ifdef __cplusplus
}
#endif

#endif /* SOLVEDELTA_MIXER_H */
