// extern "C" entry points declared in include/tops_gla_delta.h: argument validation and dispatch.
// No entry point allocates, synchronizes, or launches anything for invalid arguments.
#include <stdarg.h>
#include <stdio.h>

#include <initializer_list>

#include "delta.hpp"

namespace {

constexpr int64_t kMax = 2147483647;
// Tokens of a call: the kernels form token indices of 32 bits up to a chunk past a sequence's end.
constexpr int64_t kMaxTokens = (1LL << 31) - 64;

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

// Whether a launch has fewer than 2^32 threads and 2^31 blocks, as it must.
bool grid_fits(int64_t blocks, int64_t threads) {
  return blocks < (1LL << 32) / threads && blocks <= kMax;
}

int head_sizes(int64_t H, int64_t HV, int64_t K, int64_t V) {
  if (K < 1 || K > 256)
    return fail(TOPS_GLA_EUNSUPPORTED, "key size K must be in [1, 256] (K=%lld)", (long long)K);
  if (V < 1 || V > 65536)
    return fail(TOPS_GLA_EUNSUPPORTED, "value size V must be in [1, 65536] (V=%lld)", (long long)V);
  if (H < 1 || HV < 1 || HV > 65536 || HV % H)
    return fail(TOPS_GLA_EINVAL, "H must divide HV (H=%lld, HV=%lld)", (long long)H, (long long)HV);
  return TOPS_GLA_OK;
}

int types(int64_t dtype, int64_t g_dtype, int64_t beta_dtype) {
  if (!dtype_ok(dtype) || !dtype_ok(g_dtype) || !dtype_ok(beta_dtype))
    return fail(TOPS_GLA_EINVAL, "dtype must be F32 (0) or BF16 (1)");
  return TOPS_GLA_OK;
}

bool aligned(const void* p) { return ((uintptr_t)p & 255) == 0; }

int delta_setup(const tops_gla_delta_args* a, bool backward, tops::DeltaParams* p) {
  if (a == nullptr) return fail(TOPS_GLA_EINVAL, "NULL arguments");
  if (int rc = types(a->dtype, a->g_dtype, a->beta_dtype)) return rc;
  if (int rc = head_sizes(a->H, a->HV, a->K, a->V)) return rc;
  if (a->K < 8 || a->V < 8)   // rows are read 8 columns at a time
    return fail(TOPS_GLA_EUNSUPPORTED, "K and V must be at least 8 (K=%lld, V=%lld)",
                (long long)a->K, (long long)a->V);
  if (a->batch < 0 || a->T < 0 || a->nseq < 0 || a->chunks < 0)
    return fail(TOPS_GLA_EINVAL, "bad batch, T, nseq or chunks");
  if (a->T > kMax || a->batch > kMax || a->batch * a->T >= kMaxTokens)
    return fail(TOPS_GLA_EUNSUPPORTED, "B*T exceeds 2^31 - 64 tokens");
  if (a->seg_chunks < 1 || a->seg_chunks > kMax / 64)
    return fail(TOPS_GLA_EINVAL, "bad seg_chunks");
  const int64_t C = tops::delta_chunk_of((int)a->dtype), per = (a->T + C - 1) / C;
  if (a->seqs == nullptr) {
    const int64_t segs = std::max<int64_t>(1, (per + a->seg_chunks - 1) / a->seg_chunks);
    if (a->nseq != a->batch || a->chunks != a->batch * per || a->nsegs != a->batch * segs)
      return fail(TOPS_GLA_EINVAL, "nseq must be the batch, chunks and nsegs its own");
  } else {
    if (a->batch != 1) return fail(TOPS_GLA_EINVAL, "packed sequences require batch == 1");
    if (a->nseq > kMax / 4 || a->chunks < per || a->chunks > per + a->nseq ||
        a->nsegs < a->nseq || a->nsegs > a->chunks + a->nseq)
      return fail(TOPS_GLA_EINVAL, "bad nseq, chunks or nsegs");
  }
  // the largest launches: the inverses, the gradients (refused before the forward that leads to them),
  // the passes (in 512 threads, half as many blocks), the fold
  const bool grads = a->train || backward;
  if (!grid_fits(a->chunks, 1) ||
      !grid_fits(a->chunks * a->HV, grads ? tops::delta_grad_threads((int)a->dtype) : 256) ||
      !grid_fits((a->V / 64 + 5) * a->HV, 256) ||
      !grid_fits((a->V / 64 + 5) * a->HV * a->nsegs, 256) ||
      (a->nsegs > a->nseq && !grid_fits((a->V + 15) / 16 * a->HV * a->nseq,
                                        tops::delta_fold_threads(tops::delta_key_pad(a->K)))))
    return fail(TOPS_GLA_EUNSUPPORTED, "grid too large");
  // offsets within a chunk are 32 bits of bytes; a single token has no next one
  const bool one = a->T <= 1;
  for (int64_t st : {one ? 0 : a->q_st, one ? 0 : a->k_st, one ? 0 : a->v_st,
                     one || !backward ? 0 : a->do_st, a->HV * a->V})
    if (st < 0 || st >= (1 << 24))
      return fail(TOPS_GLA_EUNSUPPORTED, "tokens must lie less than 2^24 elements apart (%lld)",
                  (long long)st);
  if (a->chunks > 0 && any_null({a->q, a->k, a->v, a->g, a->beta}))
    return fail(TOPS_GLA_EINVAL, "q, k, v, g and beta must not be NULL");
  if (!backward && a->chunks > 0 && a->o == nullptr)
    return fail(TOPS_GLA_EINVAL, "o must not be NULL");
  *p = tops::delta_layout({a->nseq, a->chunks, a->nsegs, a->HV, a->K, a->V, a->dtype,
                           a->train || backward}, a->keep, a->ws);
  if (p->keep_bytes > 0 &&
      (a->keep == nullptr || a->keep_bytes < p->keep_bytes || !aligned(a->keep)))
    return fail(TOPS_GLA_EINVAL, "keep must hold %lld bytes, 256-byte aligned",
                (long long)p->keep_bytes);
  p->a = *a;
  p->a.train = a->train || backward;
  if (one) p->a.q_st = p->a.k_st = p->a.v_st = p->a.do_st = 0;
  if (!backward) return TOPS_GLA_OK;
  if (a->chunks > 0 && any_null({a->dout, a->dq, a->dk, a->dv, a->dg, a->dbeta}))
    return fail(TOPS_GLA_EINVAL, "dout, dq, dk, dv, dg and dbeta must not be NULL");
  if (p->ws_bytes > 0 && (a->ws == nullptr || a->ws_bytes < p->ws_bytes || !aligned(a->ws)))
    return fail(TOPS_GLA_EINVAL, "ws must hold %lld bytes, 256-byte aligned",
                (long long)p->ws_bytes);
  return TOPS_GLA_OK;
}

int norm_check(const tops_gla_layer_norm_args* a) {
  if (a == nullptr) return fail(TOPS_GLA_EINVAL, "NULL arguments");
  if (!dtype_ok(a->dtype)) return fail(TOPS_GLA_EINVAL, "dtype must be F32 (0) or BF16 (1)");
  if (a->rows < 0 || a->rows > (1LL << 40)) return fail(TOPS_GLA_EINVAL, "bad rows");
  if (a->D < 1 || a->D > 16384)
    return fail(TOPS_GLA_EUNSUPPORTED, "D must be in [1, 16384] (D=%lld)", (long long)a->D);
  if (a->rows > 0 && a->x == nullptr) return fail(TOPS_GLA_EINVAL, "x must not be NULL");
  return TOPS_GLA_OK;
}

// The launches of a call, one after another.
hipError_t run_fwd(const tops::DeltaParams& p, hipStream_t st) {
  if (p.a.chunks > 0)
    if (const hipError_t e = tops::run_delta_prep(p, st)) return e;
  return p.a.nseq > 0 ? tops::run_delta_scan(p, false, st) : hipSuccess;
}
hipError_t run_bwd(const tops::DeltaParams& p, hipStream_t st) {
  if (p.a.nseq > 0)
    if (const hipError_t e = tops::run_delta_scan(p, true, st)) return e;
  return p.a.chunks > 0 ? tops::run_delta_grad(p, st) : hipSuccess;
}

}  // namespace

extern "C" {

int64_t tops_gla_delta_chunk(int64_t dtype) {
  return dtype_ok(dtype) ? tops::delta_chunk_of((int)dtype) : 0;
}

int64_t tops_gla_delta_segment(int64_t nseq, int64_t chunks, int64_t HV, int64_t V) {
  const int64_t whole = 1 << 20;
  if (nseq < 1 || chunks < 1 || HV < 1 || V < 1) return whole;
  // a block for each CU in the second pass: 8 sequences of 16 heads and 32 chunks in two segments
  // take 258 us forward (uncut 273, three segments 334), 5 of 64 chunks in three 432 (uncut 495, two
  // 433, four 460), one of 8 chunks in four 52 (uncut 70), one of 256 in 16 358 (uncut 1801). Below 6
  // chunks the first pass costs what the second saves (4 chunks in two 46, uncut 42)
  const int64_t blocks = (V + 127) / 128 * HV * nseq, per = (chunks + nseq - 1) / nseq;
  const int64_t segs = 256 / std::max<int64_t>(1, blocks);
  if (segs < 2 || per < 6) return whole;
  int64_t L = std::max<int64_t>((per + segs - 1) / segs, 2);
  // the fold goes from segment to segment, each about a quarter of two passes' chunk: least in sum
  // at L = sqrt(per / 4) (per = 256, one head: L = 4 187 us, 8 171, 16 232; 1024, two heads: 8 400,
  // 16 334, 32 451)
  while (L * L * 4 < per && L < whole) ++L;
  return std::min(L, whole);
}

int64_t tops_gla_delta_bytes(const tops_gla_delta_sizes* z, int64_t backward) {
  if (z == nullptr) {
    fail(TOPS_GLA_EINVAL, "NULL arguments");
    return 0;
  }
  if (z->nseq < 0 || z->chunks < 0 || z->chunks > kMax || z->nsegs < z->nseq || z->nsegs > kMax ||
      z->HV < 1 || z->HV > 65536 || z->K < 1 || z->K > 256 || z->V < 1 || z->V > 65536 ||
      !dtype_ok(z->dtype) || z->chunks * z->HV > kMax || z->nsegs * z->HV > kMax)
    return 0;
  const tops::DeltaParams p = tops::delta_layout(*z, nullptr, nullptr);
  return backward ? p.ws_bytes : p.keep_bytes;
}

int tops_gla_delta_fwd(const tops_gla_delta_args* a, void* stream) {
  tops::DeltaParams p;
  if (int rc = delta_setup(a, false, &p)) return rc;
  return done(run_fwd(p, (hipStream_t)stream), "delta_fwd");
}

int tops_gla_delta_bwd(const tops_gla_delta_args* a, void* stream) {
  tops::DeltaParams p;
  if (int rc = delta_setup(a, true, &p)) return rc;
  return done(run_bwd(p, (hipStream_t)stream), "delta_bwd");
}

int tops_gla_delta_step(const tops_gla_delta_step_args* a, void* stream) {
  if (a == nullptr) return fail(TOPS_GLA_EINVAL, "NULL arguments");
  if (int rc = types(a->dtype, a->g_dtype, a->beta_dtype)) return rc;
  if (int rc = head_sizes(a->H, a->HV, a->K, a->V)) return rc;
  if (a->batch < 0 || a->T < 0 || a->slots < 0)
    return fail(TOPS_GLA_EINVAL, "bad batch, T or slots");
  if (a->slots_idx == nullptr && a->batch > a->slots)
    return fail(TOPS_GLA_EINVAL, "the states hold %lld rows, the batch %lld", (long long)a->slots,
                (long long)a->batch);
  if (a->batch > kMax || a->T > kMax || !grid_fits((a->V + 31) / 32 * a->HV, 64) ||
      !grid_fits((a->V + 31) / 32 * a->HV * a->batch, 64))
    return fail(TOPS_GLA_EUNSUPPORTED, "grid too large");
  if (a->batch > 0 && a->T > 0 && any_null({a->q, a->k, a->v, a->g, a->beta, a->o}))
    return fail(TOPS_GLA_EINVAL, "q, k, v, g, beta and o must not be NULL");
  if (a->batch > 0 && a->slots > 0 && a->state == nullptr)
    return fail(TOPS_GLA_EINVAL, "state must not be NULL");
  if (a->slots > 1 && a->state_ss < a->HV * a->K * a->V)
    return fail(TOPS_GLA_EINVAL, "the slots overlap (%lld elements, a stride of %lld)",
                (long long)(a->HV * a->K * a->V), (long long)a->state_ss);
  return done(tops::run_delta_step(*a, (hipStream_t)stream), "delta_step");
}

int64_t tops_gla_layer_norm_ws_bytes(int64_t rows, int64_t D, int64_t dtype) {
  if (rows < 0 || D < 1 || D > 16384 || !dtype_ok(dtype)) return 0;
  // one row at least: the sums of no rows are written too
  return std::max<int64_t>(1, tops::layer_norm_part_rows((long)rows, (long)D, (int)dtype)) * 8 * D;
}

int tops_gla_layer_norm_fwd(const tops_gla_layer_norm_args* a, void* stream) {
  if (int rc = norm_check(a)) return rc;
  if (a->rows > 0 && a->y == nullptr) return fail(TOPS_GLA_EINVAL, "y must not be NULL");
  return done(tops::run_layer_norm_fwd(*a, (hipStream_t)stream), "layer_norm_fwd");
}

int tops_gla_layer_norm_bwd(const tops_gla_layer_norm_args* a, void* stream) {
  if (int rc = norm_check(a)) return rc;
  if (a->rows > 0 && any_null({a->stats, a->dy, a->dx}))
    return fail(TOPS_GLA_EINVAL, "stats, dy and dx must not be NULL");
  tops_gla_layer_norm_args c = *a;
  if (a->dw || a->db) {
    const int64_t need = tops_gla_layer_norm_ws_bytes(a->rows, a->D, a->dtype);
    if (a->ws == nullptr || a->ws_bytes < need)
      return fail(TOPS_GLA_EINVAL, "dw and db need ws of %lld bytes", (long long)need);
  } else {
    c.ws = nullptr;
  }
  return done(tops::run_layer_norm_bwd(c, (hipStream_t)stream), "layer_norm_bwd");
}

}  // extern "C"
