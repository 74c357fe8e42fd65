/*
 * C entry points of libtops_gla.so for the selective state space scan, its causal convolution,
 * the single-token form of both, and the per-head norm of queries and keys with the position
 * rotation. Conventions as in tops_gla.h (device pointers, status codes, the caller's stream;
 * nothing is allocated, nothing synchronizes, invalid arguments launch nothing).
 *
 * Arguments come in one struct of 8-byte fields. `dtype` is TOPS_GLA_F32 or TOPS_GLA_BF16 and is
 * the type of every `void*` tensor; `float*` tensors are float32. Strides are in elements; the
 * last dimension of every tensor is contiguous, outputs and gradients are contiguous.
 *
 * Sequences: fixed length (`segs` NULL: B sequences of T tokens) or packed into one row of T
 * tokens (B == 1). A packed call passes its pieces as a device int32 table made by the caller
 * from the sequence lengths, whose offsets the library cannot read on the host.
 */
#ifndef TOPS_GLA_SSM_H
#define TOPS_GLA_SSM_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/*
 * Selective scan. For channel d with state size N, group g(d) = d / (D / G), per sequence:
 *   delta' = delta + delta_bias (softplus of it if `softplus`)
 *   h_t[n] = exp(delta'_t A[d,n]) h_{t-1}[n] + delta'_t u_t B_t[g,n]
 *   y_t    = (sum_n C_t[g,n] h_t[n] + Dskip[d] u_t) (* z_t sigmoid(z_t) with z)
 * A sequence is cut into pieces of at most `piece` tokens (a multiple of 16) that run in
 * parallel: piece_h [pieces][NP][D] and piece_dt [pieces][D] hold their own contributions
 * (NP = N rounded up to 8, 16, 32 or 64), not needed when no sequence has two pieces. Fixed
 * length: ceil(T / piece) pieces a sequence (at least one). Packed: `segs` holds, for each of
 * `nsegs` pieces in order, {sequence, first token, end token, its index in the sequence, pieces
 * of the sequence, index of its first chunk, f, 0}; f of row s is the first piece of sequence s.
 * A sequence of no tokens has one piece.
 * `chunk_h` [chunks][NP][D]: the states entering every chunk of
 * tops_gla_selective_scan_chunk(N) tokens of a sequence, kept for the backward (NULL: not kept).
 * `bc`: B, C and A as the kernels read them, (B * T * G + 1) * 2 * NP + NP * D floats, written by
 * the forward.
 * 1 <= N <= 64, B * T <= 2^31 - 64.
 */
typedef struct tops_gla_scan_args {
  const void *u, *delta, *z;      /* [B, T, D], z NULL: no gate */
  const void *B, *C;              /* [B, T, G, N] */
  const float *A;                 /* [D, N] */
  const float *Dskip, *delta_bias; /* [D] or NULL */
  const float *h0;                /* [sequences, D, N] or NULL */
  void *y;                        /* [B, T, D] */
  float *ht;                      /* [sequences, D, N] or NULL */
  float *chunk_h;
  float *piece_h, *piece_dt;
  float *bc;
  const int32_t *segs;
  int64_t nsegs, nseq, piece;
  int64_t batch, T, D, N, G;
  int64_t u_sb, u_st, delta_sb, delta_st, z_sb, z_st;
  int64_t B_sb, B_st, B_sg, C_sb, C_st, C_sg;
  int64_t softplus, dtype;
  /* backward only */
  const void *dy;                 /* [B, T, D] */
  int64_t dy_sb, dy_st;
  const float *dht;               /* [sequences, D, N] or NULL */
  void *du, *ddelta, *dz;         /* [B, T, D], dz exactly with z */
  void *dB, *dC;                  /* [B, T, G, N] */
  float *dA;                      /* [D, N] */
  float *dD, *dbias;              /* [D] */
  float *dh0;                     /* [sequences, D, N] or NULL */
  void *ws;                       /* tops_gla_selective_scan_bwd_ws_bytes */
  int64_t ws_bytes;
} tops_gla_scan_args;

int tops_gla_selective_scan_fwd(const tops_gla_scan_args *a, void *stream);
/* The gradients; chunk_h and bc as the forward left them (B and C are not read), piece_h and
 * piece_dt as workspaces. */
int tops_gla_selective_scan_bwd(const tops_gla_scan_args *a, void *stream);
/* Bytes of `ws`, and the tokens of a piece that fill the device for such a call. */
int64_t tops_gla_selective_scan_bwd_ws_bytes(int64_t tokens, int64_t nsegs, int64_t D, int64_t N,
                                             int64_t G);
int64_t tops_gla_selective_scan_piece(int64_t tokens, int64_t nseq, int64_t D, int64_t N,
                                      int64_t G);
/* Tokens between the states that the forward keeps (0 for an N that is refused). */
int64_t tops_gla_selective_scan_chunk(int64_t N);

/*
 * One token of the scan for each row b, its state at state[slot_b] ([slots, D, N], in place):
 * slot_b = slots_idx[b] (int32 or int64, idx64) or b. A slot outside [0, slots) leaves every
 * state as it is and gives y = 0; no slot may be given twice, and slots are at least their size
 * apart (state_ss).
 */
typedef struct tops_gla_scan_step_args {
  float *state;
  const void *u, *delta, *z;      /* [batch, D] */
  const void *B, *C;              /* [batch, G, N] */
  const float *A, *Dskip, *delta_bias;
  void *y;                        /* [batch, D] */
  const void *slots_idx;
  int64_t idx64, slots, batch, D, N, G;
  int64_t state_ss, u_sb, delta_sb, z_sb, B_sb, B_sg, C_sb, C_sg;
  int64_t softplus, dtype;
} tops_gla_scan_step_args;
int tops_gla_selective_scan_step(const tops_gla_scan_step_args *a, void *stream);

/*
 * Causal depthwise convolution of width W <= 8 with the window carried in and out:
 *   z_t[d] = sum_{j < W} w[d, j] x_{t - W + 1 + j}[d] (+ bias[d]),  y = z or z sigmoid(z),
 * rows before a sequence's first token from its state [sequences, W, D] (its last W - 1 rows;
 * zero without one); final_state gets the last W inputs. cu: device int32 [nseq + 1] token
 * offsets of packed sequences (non-decreasing from 0, the last one T), or NULL.
 */
typedef struct tops_gla_conv_args {
  const void *x;                  /* [B, T, D] */
  const void *w, *bias;           /* [D, W], [D] or NULL, of type w_dtype */
  const void *init;               /* [sequences, W, D] or NULL */
  void *y, *final_state;          /* final_state NULL: not wanted */
  const int32_t *cu;
  int64_t nseq, batch, T, D, W, x_sb, x_st, silu, dtype, w_dtype;
  /* backward only */
  const void *dy, *dfinal;        /* dfinal [sequences, W, D] or NULL */
  void *dx, *dinit;               /* dinit [sequences, W, D] or NULL */
  void *dw, *dbias;               /* [D, W], [D] of type w_dtype; dbias only with dw */
  void *ws;                       /* with dw: tops_gla_causal_conv_bwd_ws_bytes */
  int64_t ws_bytes, dy_sb, dy_st;
} tops_gla_conv_args;
int tops_gla_causal_conv_fwd(const tops_gla_conv_args *a, void *stream);
int tops_gla_causal_conv_bwd(const tops_gla_conv_args *a, void *stream);
int64_t tops_gla_causal_conv_bwd_ws_bytes(int64_t tokens, int64_t D, int64_t W);

/* One token: state[slot_b] ([slots, W, D]) moves up a row and takes x; slots as above. */
typedef struct tops_gla_conv_step_args {
  const void *x;                  /* [batch, D] */
  void *state;
  const void *w, *bias;           /* [D, W], [D] or NULL, of type w_dtype */
  void *y;                        /* [batch, D] */
  const void *slots_idx;
  int64_t idx64, slots, batch, D, W, state_ss, x_sb, silu, dtype, w_dtype;
} tops_gla_conv_step_args;
int tops_gla_causal_conv_step(const tops_gla_conv_step_args *a, void *stream);

/*
 * Queries q [B, T, Hq, D] and keys k [B, T, Hk, D]: per token and head
 *   n = x rsqrt(mean(x^2) + eps) (* weight),  then the pairs (i, i + R / 2), or (2 i, 2 i + 1)
 * with `interleaved`, of n's first R columns turned by positions[b, t] inv_freq[i] radians.
 * inv_freq float64 [R / 2]; positions int32 or int64 (pos64) with strides pos_sb, 1, NULL: t.
 * The backward takes the outputs' gradients dqo / dko and writes dq, dk and, when dqw / dkw are
 * given, the weights' gradients with ws of tops_gla_qk_norm_rope_ws_bytes. D <= 512.
 */
typedef struct tops_gla_qk_args {
  const void *q, *k;
  const float *qw, *kw;           /* [D] or NULL */
  const double *inv_freq;
  const void *positions;
  void *qo, *ko;
  int64_t batch, T, Hq, Hk, D, R;
  int64_t q_sb, q_st, q_sh, k_sb, k_st, k_sh, pos_sb, pos64;
  int64_t interleaved, dtype;
  double eps;
  /* backward only */
  const void *dqo, *dko;
  int64_t dq_sb, dq_st, dq_sh, dk_sb, dk_st, dk_sh;
  void *dq, *dk;
  float *dqw, *dkw;
  void *ws;
  int64_t ws_bytes;
} tops_gla_qk_args;
int tops_gla_qk_norm_rope_fwd(const tops_gla_qk_args *a, void *stream);
int tops_gla_qk_norm_rope_bwd(const tops_gla_qk_args *a, void *stream);
int64_t tops_gla_qk_norm_rope_ws_bytes(int64_t tokens, int64_t D);

#ifdef __cplusplus
}
#endif

#endif /* TOPS_GLA_SSM_H */
