/*
 * C entry points of libtops_gla.so for the gated delta rule (prompts, training, and the form for
 * the next tokens of a serving batch) and for the layer norm. Conventions as in tops_gla.h (device
 * pointers, status codes, the caller's stream; nothing is allocated, nothing synchronizes, invalid
 * arguments launch nothing).
 *
 * Arguments come in one struct of 8-byte fields. `dtype` is TOPS_GLA_F32 or TOPS_GLA_BF16 and is
 * the type of every `void*` tensor without a type of its own; `float*` tensors are float32.
 * Strides are in elements; the last dimension of every tensor is contiguous, outputs and gradients
 * are contiguous.
 */
#ifndef TOPS_GLA_DELTA_H
#define TOPS_GLA_DELTA_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/*
 * Gated delta rule. Value head j reads key head j / (HV / H); per value head, with a state
 * S [K, V] that a sequence starts from h0 (zeros without one):
 *   S' = e^{g_t} S_{t-1},  n_t = beta_t (v_t - S'^T k_t),  S_t = S' + k_t n_t^T,
 *   o_t = scale S_t^T q_t.
 * With `l2norm` q_t and k_t stand for q_t / sqrt(|q_t|^2 + 1e-6) and the same of k_t.
 * Sequences are cut into chunks of tops_gla_delta_chunk(dtype) tokens, and these into segments of
 * `seg_chunks` chunks (the last of a sequence may be shorter; a sequence without tokens has one
 * segment), which run in parallel; tops_gla_delta_segment says how many. `chunks` and `nsegs` are
 * those of all sequences. Fixed length (`seqs` NULL): batch sequences of T tokens. Packed (batch ==
 * 1): `seqs` is a device int32 table of nseq + 1 token offsets (from 0 to T, not decreasing), nseq +
 * 1 chunk offsets, nseq + 1 segment offsets, and the sequence of each segment.
 * `keep` (tops_gla_delta_bytes, 256-byte aligned) is the forward's workspace; with `train` it also
 * holds what the backward reads.
 * 8 <= K <= 256, 8 <= V <= 65536, batch * T < 2^31 - 64, tokens of q, k, v, dout and o at least 0
 * and less than 2^24 elements apart (with T <= 1 the inputs' are not looked at).
 */
typedef struct tops_gla_delta_args {
  const void *q, *k;              /* [B, T, H, K] */
  const void *v;                  /* [B, T, HV, V] */
  const void *g, *beta;           /* [B, T, HV], of types g_dtype and beta_dtype */
  const float *h0;                /* [sequences, HV, K, V] or NULL */
  void *o;                        /* [B, T, HV, V] */
  float *ht;                      /* [sequences, HV, K, V] or NULL */
  const int32_t *seqs;
  void *keep;
  int64_t keep_bytes;
  int64_t nseq, chunks, nsegs, seg_chunks, batch, T, H, HV, K, V;
  int64_t q_sb, q_st, q_sh, k_sb, k_st, k_sh, v_sb, v_st, v_sh;
  int64_t g_sb, g_st, beta_sb, beta_st;
  int64_t l2norm, train, dtype, g_dtype, beta_dtype;
  double scale;
  /* backward only */
  const void *dout;               /* [B, T, HV, V] */
  int64_t do_sb, do_st, do_sh;
  const float *dht;               /* [sequences, HV, K, V] or NULL */
  void *dq, *dk, *dv;
  void *dg, *dbeta;               /* of g's and beta's types */
  float *dh0;                     /* [sequences, HV, K, V] or NULL */
  void *ws;                       /* tops_gla_delta_bytes, 256-byte aligned */
  int64_t ws_bytes;
} tops_gla_delta_args;
int tops_gla_delta_fwd(const tops_gla_delta_args *a, void *stream);
/* The gradients; keep as a forward with `train` left it. */
int tops_gla_delta_bwd(const tops_gla_delta_args *a, void *stream);
/* Tokens of a chunk (0 for a type that is refused). */
int64_t tops_gla_delta_chunk(int64_t dtype);
/* Chunks of a segment for nseq sequences of like lengths, `chunks` chunks in all; with K > 128, whose
 * blocks have half the columns, V stands for twice the values. */
int64_t tops_gla_delta_segment(int64_t nseq, int64_t chunks, int64_t HV, int64_t V);
/* Bytes of `keep`, or with `backward` of `ws` (0 for sizes that are refused). */
typedef struct tops_gla_delta_sizes {
  int64_t nseq, chunks, nsegs, HV, K, V, dtype, train;
} tops_gla_delta_sizes;
int64_t tops_gla_delta_bytes(const tops_gla_delta_sizes *z, int64_t backward);

/*
 * The next T tokens of each row b, its state at state[slot_b] ([slots, HV, K, V], updated in
 * place): slot_b = slots_idx[b] (int32 or int64, idx64) or b. A slot outside [0, slots) leaves
 * every state as it is and gives o = 0; no slot may be given twice, and slots are at least their
 * size apart (state_ss). 1 <= K <= 256, 1 <= V <= 65536.
 */
typedef struct tops_gla_delta_step_args {
  float *state;
  const void *q, *k, *v;          /* [batch, T, H, K], [batch, T, HV, V] */
  const void *g, *beta;           /* [batch, T, HV], of types g_dtype and beta_dtype */
  void *o;                        /* [batch, T, HV, V] */
  const void *slots_idx;
  int64_t idx64, slots, batch, T, H, HV, K, V, state_ss;
  int64_t q_sb, q_st, q_sh, k_sb, k_st, k_sh, v_sb, v_st, v_sh;
  int64_t g_sb, g_st, beta_sb, beta_st;
  int64_t l2norm, dtype, g_dtype, beta_dtype;
  double scale;
} tops_gla_delta_step_args;
int tops_gla_delta_step(const tops_gla_delta_step_args *a, void *stream);

/*
 * Layer norm of rows of D <= 16384 features: y = (x - mean) rstd (* w) (+ b), rstd =
 * 1 / sqrt(mean((x - mean)^2) + eps). `stats` [rows, 2] keeps mean and rstd for the backward, which
 * writes dx and, where dw or db is given, the sums over the rows, with ws of
 * tops_gla_layer_norm_ws_bytes. x and dy have rows x_st and dy_st apart; y and dx are contiguous.
 */
typedef struct tops_gla_layer_norm_args {
  const void *x;
  const float *w, *b;             /* [D] or NULL */
  void *y;
  float *stats;                   /* NULL in the forward: not wanted */
  int64_t rows, D, x_st, dtype;
  double eps;
  /* backward only */
  const void *dy;
  int64_t dy_st;
  void *dx;
  float *dw, *db;                 /* [D] or NULL */
  void *ws;
  int64_t ws_bytes;
} tops_gla_layer_norm_args;
int tops_gla_layer_norm_fwd(const tops_gla_layer_norm_args *a, void *stream);
int tops_gla_layer_norm_bwd(const tops_gla_layer_norm_args *a, void *stream);
int64_t tops_gla_layer_norm_ws_bytes(int64_t rows, int64_t D, int64_t dtype);

#ifdef __cplusplus
}
#endif

#endif /* TOPS_GLA_DELTA_H */
