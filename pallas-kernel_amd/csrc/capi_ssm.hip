// extern "C" entry points declared in include/tops_gla_ssm.h: argument validation and dispatch.
// No entry point allocates, synchronizes, or launches anything for invalid arguments.
#include <stdarg.h>
#include <stdio.h>

#include <initializer_list>

#include "ssm.hpp"

namespace {

constexpr int64_t kMax = 2147483647;
// Tokens of a scan: its kernels form token indices of 32 bits up to a tile past a piece's end.
constexpr int64_t kMaxScanTokens = (1LL << 31) - 64;

int fail(int code, const char* fmt, ...) {
  char msg[400];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(msg, sizeof(msg), fmt, ap);
  va_end(ap);
  return tops::set_error(code, msg);
}

int done(hipError_t e, const char* what) {
  if (e == hipSuccess) return tops::set_error(TOPS_GLA_OK, "");
  return fail(TOPS_GLA_EHIP, "%s: %s", what, hipGetErrorString(e));
}

bool dtype_ok(int64_t d) { return d == TOPS_GLA_F32 || d == TOPS_GLA_BF16; }

bool any_null(std::initializer_list<const void*> ps) {
  for (const void* p : ps)
    if (p == nullptr) return true;
  return false;
}

// Whether a launch has fewer than 2^32 threads, as it must.
bool grid_fits(int64_t blocks, int64_t threads) { return blocks < (1LL << 32) / threads; }

int scan_sizes(int64_t D, int64_t N, int64_t G, int64_t dtype) {
  if (!dtype_ok(dtype)) return fail(TOPS_GLA_EINVAL, "dtype must be F32 (0) or BF16 (1)");
  if (D < 1 || D > (1 << 20)) return fail(TOPS_GLA_EINVAL, "D must be in [1, 2^20] (D=%lld)",
                                          (long long)D);
  if (N < 1 || N > 64)
    return fail(TOPS_GLA_EUNSUPPORTED, "state size N must be in [1, 64] (N=%lld)", (long long)N);
  if (G < 1 || D % G) return fail(TOPS_GLA_EINVAL, "G must divide D (D=%lld, G=%lld)",
                                  (long long)D, (long long)G);
  return TOPS_GLA_OK;
}

// Channel tiles of a group in the forward's waves and the backward's blocks.
int64_t tiles_of(int64_t D, int64_t G) { return (D / G + 63) / 64; }
int64_t bwd_tiles_of(int64_t D, int64_t N, int64_t G) {
  const int64_t ct = tops::scan_bwd_channels((int)N);
  return (D / G + ct - 1) / ct;
}

int scan_setup(const tops_gla_scan_args* a, bool backward, tops::ScanParams* p) {
  if (a == nullptr) return fail(TOPS_GLA_EINVAL, "NULL arguments");
  if (int rc = scan_sizes(a->D, a->N, a->G, a->dtype)) return rc;
  if (a->batch < 0 || a->T < 0 || a->nseq < 0)
    return fail(TOPS_GLA_EINVAL, "bad batch, T or nseq");
  if (a->T > kMax || a->batch > kMax || a->batch * a->T > kMaxScanTokens)
    return fail(TOPS_GLA_EUNSUPPORTED, "B*T exceeds 2^31 - 64 tokens");
  if (a->piece < 16 || a->piece % 16 || a->piece > kMax)
    return fail(TOPS_GLA_EINVAL, "piece must be a positive multiple of 16 (piece=%lld)",
                (long long)a->piece);
  *p = tops::ScanParams{};
  p->a = *a;
  p->tokens = a->batch * a->T;
  if (a->segs) {
    if (a->batch != 1) return fail(TOPS_GLA_EINVAL, "packed sequences require batch == 1");
    if (a->nsegs < a->nseq || a->nsegs > kMax)
      return fail(TOPS_GLA_EINVAL, "bad nsegs (%lld for %lld sequences)", (long long)a->nsegs,
                  (long long)a->nseq);
    p->npieces = a->nsegs;
    p->multi = a->piece_h != nullptr && a->nsegs > 0;
  } else {
    if (a->nseq != a->batch) return fail(TOPS_GLA_EINVAL, "nseq must be the batch");
    const int64_t n = std::max<int64_t>(1, (a->T + a->piece - 1) / a->piece);
    if (n * a->batch > kMax) return fail(TOPS_GLA_EUNSUPPORTED, "too many pieces");
    p->pieces = (int)n;
    p->npieces = n * a->batch;
    p->multi = p->npieces > a->batch;   // not without a batch: there is nothing to launch for
    if (p->multi && a->piece_h == nullptr)
      return fail(TOPS_GLA_EINVAL, "piece_h and piece_dt are required for several pieces");
  }
  if (p->multi && a->piece_dt == nullptr)
    return fail(TOPS_GLA_EINVAL, "piece_dt is required with piece_h");
  const int64_t np = tops::scan_state_pad((int)a->N);
  p->tiles_g = (int)tiles_of(a->D, a->G);
  p->btiles = (int)(bwd_tiles_of(a->D, a->N, a->G) * a->G);
  if (!grid_fits((p->tiles_g * a->G * p->npieces + 3) / 4, 256) ||
      (backward && !grid_fits(p->btiles * p->npieces, tops::scan_bwd_threads((int)a->N))))
    return fail(TOPS_GLA_EUNSUPPORTED, "grid too large");
  p->ntiles = p->tiles_g * (int)a->G;
  p->at = a->bc + (p->tokens * a->G + 1) * 2 * np;
  if (any_null({a->A})) return fail(TOPS_GLA_EINVAL, "A must not be NULL");
  if (p->tokens > 0 && (any_null({a->u, a->delta}) || (!backward && any_null({a->B, a->C}))))
    return fail(TOPS_GLA_EINVAL, "u, delta, B and C must not be NULL");
  if (!backward) {
    if (p->tokens > 0 && a->y == nullptr) return fail(TOPS_GLA_EINVAL, "y must not be NULL");
    if (a->bc == nullptr) return fail(TOPS_GLA_EINVAL, "bc must not be NULL");
    return TOPS_GLA_OK;
  }
  if (p->tokens > 0 && any_null({a->dy, a->du, a->ddelta, a->dB, a->dC, a->chunk_h}))
    return fail(TOPS_GLA_EINVAL, "dy, du, ddelta, dB, dC and chunk_h must not be NULL");
  if (p->tokens > 0 && (a->z == nullptr) != (a->dz == nullptr))
    return fail(TOPS_GLA_EINVAL, "dz must be given exactly when z is");
  if (a->dA == nullptr) return fail(TOPS_GLA_EINVAL, "dA must not be NULL");
  const int64_t need =
      tops_gla_selective_scan_bwd_ws_bytes(p->tokens, p->npieces, a->D, a->N, a->G);
  if (need > 0 && (a->ws == nullptr || a->ws_bytes < need))
    return fail(TOPS_GLA_EINVAL, "ws must hold %lld bytes", (long long)need);
  if (a->bc == nullptr) return fail(TOPS_GLA_EINVAL, "bc must not be NULL");
  p->part_bc = (float*)a->ws;
  p->part_a = p->part_bc + p->btiles * p->tokens * 2 * np;
  p->part_d = p->part_a + p->npieces * a->D * np;
  return TOPS_GLA_OK;
}

int slots_ok(int64_t batch, int64_t slots, const void* idx) {
  if (batch < 0 || slots < 0) return fail(TOPS_GLA_EINVAL, "bad batch or slots");
  if (idx == nullptr && batch > slots)
    return fail(TOPS_GLA_EINVAL, "the states hold %lld rows, the batch %lld", (long long)slots,
                (long long)batch);
  return TOPS_GLA_OK;
}

// Slots of `size` elements, `ss` apart: rows that share one would read and write it at once.
int slots_apart(int64_t slots, int64_t ss, int64_t size) {
  if (slots > 1 && ss < size)
    return fail(TOPS_GLA_EINVAL, "the slots overlap (%lld elements, a stride of %lld)",
                (long long)size, (long long)ss);
  return TOPS_GLA_OK;
}

int conv_check(const tops_gla_conv_args* a) {
  if (a == nullptr) return fail(TOPS_GLA_EINVAL, "NULL arguments");
  if (!dtype_ok(a->dtype) || !dtype_ok(a->w_dtype)) return fail(TOPS_GLA_EINVAL, "dtype must be F32 (0) or BF16 (1)");
  if (a->D < 1 || a->D > (1 << 20))
    return fail(TOPS_GLA_EINVAL, "D must be in [1, 2^20] (D=%lld)", (long long)a->D);
  if (a->W < 1 || a->W > 8)
    return fail(TOPS_GLA_EUNSUPPORTED, "kernel width W in 1..8 (W=%lld)", (long long)a->W);
  if (a->batch < 0 || a->T < 0 || a->nseq < 0)
    return fail(TOPS_GLA_EINVAL, "bad batch, T or nseq");
  if (a->T > kMax || a->batch > kMax || a->batch * a->T > kMax)
    return fail(TOPS_GLA_EUNSUPPORTED, "B*T exceeds 2^31 tokens");
  if (a->cu == nullptr ? a->nseq != a->batch : a->batch != 1)
    return fail(TOPS_GLA_EINVAL, "packed sequences require batch == 1, others nseq == batch");
  const int64_t vec = 8 / (a->dtype == TOPS_GLA_BF16 ? 2 : 4), per = 64 * (a->D < vec ? 1 : vec);
  const int64_t tiles = tops::causal_conv_part_rows(a->batch * a->T, a->D);
  if (a->nseq > kMax || !grid_fits((a->D + per - 1) / per * (tiles + (a->nseq * a->W + 3) / 4), 256) ||
      !grid_fits((a->D + 255) / 256 * a->nseq, 256))
    return fail(TOPS_GLA_EUNSUPPORTED, "grid too large");
  if (a->w == nullptr) return fail(TOPS_GLA_EINVAL, "w must not be NULL");
  if (a->batch * a->T > 0 && a->x == nullptr) return fail(TOPS_GLA_EINVAL, "x must not be NULL");
  return TOPS_GLA_OK;
}

int qk_check(const tops_gla_qk_args* a) {
  if (a == nullptr) return fail(TOPS_GLA_EINVAL, "NULL arguments");
  if (!dtype_ok(a->dtype)) return fail(TOPS_GLA_EINVAL, "dtype must be F32 (0) or BF16 (1)");
  if (a->D < 1 || a->D > 512)
    return fail(TOPS_GLA_EUNSUPPORTED, "head size D must be in [1, 512] (D=%lld)", (long long)a->D);
  if (a->R < 0 || a->R > a->D || a->R % 2)
    return fail(TOPS_GLA_EINVAL, "rotated columns R must be even and at most D (R=%lld)",
                (long long)a->R);
  if (a->R > 0 && a->inv_freq == nullptr)
    return fail(TOPS_GLA_EINVAL, "inv_freq must not be NULL");
  if (a->batch < 0 || a->T < 0 || a->Hq < 0 || a->Hk < 0 || a->Hq > 65536 || a->Hk > 65536)
    return fail(TOPS_GLA_EINVAL, "bad batch, T, Hq or Hk");
  if (a->T > kMax || a->batch > kMax || a->batch * a->T > kMax)
    return fail(TOPS_GLA_EUNSUPPORTED, "B*T exceeds 2^31 tokens");
  if (!grid_fits(tops::qk_norm_rope_blocks(a->batch * a->T, a->Hq + a->Hk), 256))
    return fail(TOPS_GLA_EUNSUPPORTED, "grid too large");
  return TOPS_GLA_OK;
}

}  // namespace

extern "C" {

int64_t tops_gla_selective_scan_piece(int64_t tokens, int64_t nseq, int64_t D, int64_t N,
                                      int64_t G) {
  if (tokens <= 0 || nseq < 1 || D < 1 || N < 1 || N > 64 || G < 1 || D % G) return 64;
  // sequences and channels that make two waves a SIMD are not cut: a first pass over the tokens
  // costs more than the third to eighth wave give (D4096 N16 bf16, forward, whole and cut: 2048
  // waves of 256 tokens 200 and 293 us, 4096 of 128 157 and 315; but 1024 of 512 321 and 273)
  if (nseq * tiles_of(D, G) * G >= 2048) return 1 << 30;
  // as many waves a SIMD as the states in registers allow in the pieces' own passes, eight with 16
  // of them (62 and 64 registers), and at most 512 pieces for the fold to walk. The outputs' pass
  // holds five (82), and its last waves leave SIMDs idle: still the best of those measured (4096,
  // 5461, 6144, 8192, 10923, 16384 waves in all, N 16: 8192 packed tokens of 2048 channels 179, 179,
  // 167, 162, 162, 171 us; training B2 T4096 D4096 912, 931, 927, 870, 899, 918)
  const int64_t np = tops::scan_state_pad((int)N), waves = np <= 16 ? 8192 : 131072 / np;
  const int64_t len =
      std::max((tokens * tiles_of(D, G) * G + waves - 1) / waves, (tokens + 511) / 512);
  return std::min<int64_t>(std::max<int64_t>(16, (len + 15) / 16 * 16), 1 << 30);
}

int64_t tops_gla_selective_scan_chunk(int64_t N) {
  return N < 1 || N > 64 ? 0 : tops::scan_chunk();
}

int64_t tops_gla_selective_scan_bwd_ws_bytes(int64_t tokens, int64_t nsegs, int64_t D, int64_t N,
                                             int64_t G) {
  if (tokens < 0 || nsegs < 0 || D < 1 || N < 1 || N > 64 || G < 1 || D % G) return 0;
  const int64_t np = tops::scan_state_pad((int)N);
  return 4 * (bwd_tiles_of(D, N, G) * tokens * G * 2 * np + nsegs * D * (np + 2));
}

int tops_gla_selective_scan_fwd(const tops_gla_scan_args* a, void* stream) {
  tops::ScanParams p;
  if (int rc = scan_setup(a, false, &p)) return rc;
  return done(tops::run_selective_scan(p, false, (hipStream_t)stream), "selective_scan_fwd");
}

int tops_gla_selective_scan_bwd(const tops_gla_scan_args* a, void* stream) {
  tops::ScanParams p;
  if (int rc = scan_setup(a, true, &p)) return rc;
  return done(tops::run_selective_scan(p, true, (hipStream_t)stream), "selective_scan_bwd");
}

int tops_gla_selective_scan_step(const tops_gla_scan_step_args* a, void* stream) {
  if (a == nullptr) return fail(TOPS_GLA_EINVAL, "NULL arguments");
  if (int rc = scan_sizes(a->D, a->N, a->G, a->dtype)) return rc;
  if (int rc = slots_ok(a->batch, a->slots, a->slots_idx)) return rc;
  // 4 of a row's states a lane; many rows go in pairs
  const int64_t cpb = 256 / (a->N <= 4 ? 1 : tops::scan_state_pad((int)a->N) / 4);
  if (a->batch > kMax || !grid_fits((a->D + cpb - 1) / cpb * ((a->batch + 1) / 2), 256)) return fail(TOPS_GLA_EUNSUPPORTED, "grid too large");
  if (a->batch > 0 && any_null({a->u, a->delta, a->B, a->C, a->A, a->y}))
    return fail(TOPS_GLA_EINVAL, "u, delta, A, B, C and y must not be NULL");
  if (a->batch > 0 && a->slots > 0 && a->state == nullptr)
    return fail(TOPS_GLA_EINVAL, "state must not be NULL");
  if (int rc = slots_apart(a->slots, a->state_ss, a->D * a->N)) return rc;
  return done(tops::run_scan_step(*a, (hipStream_t)stream), "selective_scan_step");
}

int64_t tops_gla_causal_conv_bwd_ws_bytes(int64_t tokens, int64_t D, int64_t W) {
  if (tokens <= 0 || D < 1 || W < 1 || W > 8) return 0;
  return tops::causal_conv_part_rows((long)tokens, (long)D) * (W + 1) * D * 4;
}

int tops_gla_causal_conv_fwd(const tops_gla_conv_args* a, void* stream) {
  if (int rc = conv_check(a)) return rc;
  if (a->batch * a->T > 0 && a->y == nullptr) return fail(TOPS_GLA_EINVAL, "y must not be NULL");
  return done(tops::run_causal_conv_fwd(*a, (hipStream_t)stream), "causal_conv_fwd");
}

int tops_gla_causal_conv_bwd(const tops_gla_conv_args* a, void* stream) {
  if (int rc = conv_check(a)) return rc;
  if (a->batch * a->T > 0 && any_null({a->dy, a->dx}))
    return fail(TOPS_GLA_EINVAL, "dy and dx must not be NULL");
  const int64_t need = tops_gla_causal_conv_bwd_ws_bytes(a->batch * a->T, a->D, a->W);
  if (a->dw && need > 0 && (a->ws == nullptr || a->ws_bytes < need))
    return fail(TOPS_GLA_EINVAL, "dw needs ws of %lld bytes", (long long)need);
  return done(tops::run_causal_conv_bwd(*a, (hipStream_t)stream), "causal_conv_bwd");
}

int tops_gla_causal_conv_step(const tops_gla_conv_step_args* a, void* stream) {
  if (a == nullptr) return fail(TOPS_GLA_EINVAL, "NULL arguments");
  if (!dtype_ok(a->dtype) || !dtype_ok(a->w_dtype))
    return fail(TOPS_GLA_EINVAL, "dtype must be F32 (0) or BF16 (1)");
  if (a->D < 1 || a->D > (1 << 20))
    return fail(TOPS_GLA_EINVAL, "D must be in [1, 2^20] (D=%lld)", (long long)a->D);
  if (a->W < 1 || a->W > 8)
    return fail(TOPS_GLA_EUNSUPPORTED, "kernel width W in 1..8 (W=%lld)", (long long)a->W);
  if (int rc = slots_ok(a->batch, a->slots, a->slots_idx)) return rc;
  if (a->batch > kMax || !grid_fits(a->batch * ((a->D + 255) / 256), 256)) return fail(TOPS_GLA_EUNSUPPORTED, "grid too large");
  if (a->batch > 0 && any_null({a->x, a->w, a->y}))
    return fail(TOPS_GLA_EINVAL, "x, w and y must not be NULL");
  if (a->batch > 0 && a->slots > 0 && a->state == nullptr)
    return fail(TOPS_GLA_EINVAL, "state must not be NULL");
  if (int rc = slots_apart(a->slots, a->state_ss, a->W * a->D)) return rc;
  return done(tops::run_conv_step(*a, (hipStream_t)stream), "causal_conv_step");
}

int64_t tops_gla_qk_norm_rope_ws_bytes(int64_t tokens, int64_t D) {
  if (tokens <= 0 || D < 1 || D > 512) return 0;
  return tops::qk_norm_rope_part_rows((long)tokens) * 2 * D * 4;
}

int tops_gla_qk_norm_rope_fwd(const tops_gla_qk_args* a, void* stream) {
  if (int rc = qk_check(a)) return rc;
  const int64_t tokens = a->batch * a->T;
  if (tokens > 0 && ((a->Hq > 0 && any_null({a->q, a->qo})) || (a->Hk > 0 && any_null({a->k, a->ko}))))
    return fail(TOPS_GLA_EINVAL, "q, k and their outputs must not be NULL");
  return done(tops::run_qk_norm_rope(*a, false, (hipStream_t)stream), "qk_norm_rope_fwd");
}

int tops_gla_qk_norm_rope_bwd(const tops_gla_qk_args* a, void* stream) {
  if (int rc = qk_check(a)) return rc;
  const int64_t tokens = a->batch * a->T;
  if (tokens > 0 && ((a->Hq > 0 && any_null({a->q, a->dqo, a->dq})) ||
                     (a->Hk > 0 && any_null({a->k, a->dko, a->dk}))))
    return fail(TOPS_GLA_EINVAL, "q, k and their gradients must not be NULL");
  const int64_t need = tops_gla_qk_norm_rope_ws_bytes(tokens, a->D);
  if ((a->dqw || a->dkw) && need > 0 && (a->ws == nullptr || a->ws_bytes < need))
    return fail(TOPS_GLA_EINVAL, "dqw and dkw need ws of %lld bytes", (long long)need);
  return done(tops::run_qk_norm_rope(*a, true, (hipStream_t)stream), "qk_norm_rope_bwd");
}

}  // extern "C"
