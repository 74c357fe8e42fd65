// The gated delta rule for the next tokens of a serving batch, states updated in place
// (include/tops_gla_delta.h).
//
// Bound by memory: the state of a row and head is read and written once, however many tokens come.
// A wave holds all K rows of 32 columns of the state, whole lines of 128 bytes: a lane four columns
// of K / 8 consecutive rows, so that the sums over the keys are sums of a lane and of the 8 lanes
// with its columns (a rotation in a row of lanes, two swaps of rows), without LDS. One round serves a
// token: with S' = e^g S, o = scale S_t^T q = scale (S'^T q + (q k) n), so S'^T k, S'^T q, q k and
// the norms are summed together, before n is known.
//
// Measured: 128 rows of 16 heads of 128 x 128, 268 MB, in 54.2 us, 4.95 TB/s, as a large copy has. A
// wave is a block of its own (four a block: 58.8 us), neighbouring columns on one XCD (each on the
// next: 56.3 us, and 64 so 50 us with 100 columns, where lines are shared). A token's inputs asked for
// with the state or the token before were no faster there, with one token a row (60.5 us: 252 registers
// for 131); of several tokens of few rows, where registers are free, that has not been measured (16 rows
// of 4 tokens: 16 us, 7 of bytes). One row of 16 heads takes 8 us, the time of its few memory accesses one
// after another.
#include "delta.hpp"

namespace tops {

namespace {

__device__ __forceinline__ float key_sum(float x) {
  x += dpp<0x128>(x);
  x = swap16_add(x, x);
  return swap32_add(x, x);
}

// KR: rows of the state a lane.
template <typename T, int KR>
__global__ __launch_bounds__(64) void delta_step_kernel(tops_gla_delta_step_args a) {
  const int lane = threadIdx.x;
  const int K = (int)a.K, V = (int)a.V, T_ = (int)a.T;
  const int vt = (V + 31) / 32;
  long blk = xcd_remap((int)blockIdx.x, (int)gridDim.x);
  const int vb = (int)(blk % vt);
  blk /= vt;
  const int hv = (int)(blk % a.HV);
  const long b = blk / a.HV;
  const int h = hv / (int)(a.HV / a.H);
  const int c0 = vb * 32 + (lane & 7) * 4;
  const int r0 = (lane >> 3) * KR;
  const int nc = V - c0, nr = K - r0;
  T* o = (T*)a.o + ((b * T_) * a.HV + hv) * V + c0;
  const long o_st = a.HV * V;

  long slot = b;
  if (a.slots_idx)
    slot = a.idx64 ? ((const int64_t*)a.slots_idx)[b] : (long)((const int32_t*)a.slots_idx)[b];
  if (slot < 0 || slot >= a.slots) {
    const float zero[4] = {0.f, 0.f, 0.f, 0.f};
    if (lane < 8 && nc > 0)
      for (int t = 0; t < T_; ++t) put_run<T, 4>(o + t * o_st, zero, nc);
    return;
  }
  float* S = a.state + slot * a.state_ss + (long)hv * K * V + (long)r0 * V + c0;
  float s[KR][4];
  if (V % 4 == 0) {   // loads without conditions, all on their way at once: from inside, past the end
    const float* S0 = S - r0 * (long)V - c0 + min(c0, V - 4);
#pragma unroll
    for (int r = 0; r < KR; ++r) {
      const auto x = get_run<float, 4>(S0 + (long)min(r0 + r, K - 1) * V);
#pragma unroll
      for (int e = 0; e < 4; ++e) s[r][e] = x.v[e];
    }
#pragma unroll
    for (int r = 0; r < KR; ++r)
      if (r >= nr || nc <= 0)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[r][e] = 0.f;
  } else {
#pragma unroll
    for (int r = 0; r < KR; ++r)
#pragma unroll
      for (int e = 0; e < 4; ++e) s[r][e] = r < nr && e < nc ? S[(long)r * V + e] : 0.f;
  }
  const T* q = (const T*)a.q + b * a.q_sb + h * a.q_sh + r0;
  const T* k = (const T*)a.k + b * a.k_sb + h * a.k_sh + r0;
  const T* v = (const T*)a.v + b * a.v_sb + hv * a.v_sh + c0;
  const long g0 = b * a.g_sb + hv, b0 = b * a.beta_sb + hv;
  const bool whole = K == 8 * KR && V % 32 == 0;   // no lane of a wave is past the end
  for (int t = 0; t < T_; ++t) {
    Run<T, KR> qr, kr;
    Run<T, 4> vr;
    if (whole) {
      qr = get_run<T, KR>(q + t * a.q_st);
      kr = get_run<T, KR>(k + t * a.k_st);
      vr = get_run<T, 4>(v + t * a.v_st);
    } else {
#pragma unroll
      for (int r = 0; r < KR; ++r) {
        qr.v[r] = r < nr ? q[t * a.q_st + r] : zero_elem<T>();
        kr.v[r] = r < nr ? k[t * a.k_st + r] : zero_elem<T>();
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) vr.v[e] = e < nc ? v[t * a.v_st + e] : zero_elem<T>();
    }
    const float ge = expf(get_any(a.g, (int)a.g_dtype, g0 + t * a.g_st));
    const float beta = get_any(a.beta, (int)a.beta_dtype, b0 + t * a.beta_st);
    float sk[4] = {0.f, 0.f, 0.f, 0.f}, sq[4] = {0.f, 0.f, 0.f, 0.f}, qk = 0.f, qq = 0.f, kk = 0.f;
#pragma unroll
    for (int r = 0; r < KR; ++r) {
      const float x = to_f32(qr.v[r]), y = to_f32(kr.v[r]);
      qk = fmaf(x, y, qk);
      qq = fmaf(x, x, qq);
      kk = fmaf(y, y, kk);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        sk[e] = fmaf(s[r][e], y, sk[e]);
        sq[e] = fmaf(s[r][e], x, sq[e]);
      }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      sk[e] = key_sum(sk[e]);
      sq[e] = key_sum(sq[e]);
    }
    qk = key_sum(qk);
    float rq = 1.f, rk = 1.f;
    if (a.l2norm) {
      rq = rsqrtf(key_sum(qq) + DELTA_L2_EPS);
      rk = rsqrtf(key_sum(kk) + DELTA_L2_EPS);
    }
    float n[4], y[4];
    const float fq = (float)a.scale * rq;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      n[e] = rk * beta * (to_f32(vr.v[e]) - ge * rk * sk[e]);   // what the raw key writes
      y[e] = fq * fmaf(qk, n[e], ge * sq[e]);
    }
#pragma unroll
    for (int r = 0; r < KR; ++r) {
      const float x = to_f32(kr.v[r]);
#pragma unroll
      for (int e = 0; e < 4; ++e) s[r][e] = fmaf(x, n[e], ge * s[r][e]);
    }
    if (lane < 8 && nc > 0) put_run<T, 4>(o + t * o_st, y, nc);
  }
#pragma unroll
  for (int r = 0; r < KR; ++r)
    if (r < nr && nc > 0) put_run<float, 4>(S + (long)r * V, s[r], nc);
}

template <typename T>
void launch(const tops_gla_delta_step_args& a, unsigned grid, hipStream_t st) {
  if (a.K <= 64)
    delta_step_kernel<T, 8><<<grid, 64, 0, st>>>(a);
  else if (a.K <= 128)
    delta_step_kernel<T, 16><<<grid, 64, 0, st>>>(a);
  else
    delta_step_kernel<T, 32><<<grid, 64, 0, st>>>(a);
}

}  // namespace

hipError_t run_delta_step(const tops_gla_delta_step_args& a, hipStream_t st) {
  if (a.batch == 0 || a.T == 0) return hipSuccess;
  const unsigned grid = (unsigned)((a.V + 31) / 32 * a.HV * a.batch);
  if (a.dtype == DT_BF16)
    launch<bf16>(a, grid, st);
  else
    launch<float>(a, grid, st);
  return hipGetLastError();
}

}  // namespace tops
