// The gradients of the gated delta rule over chunks (include/tops_gla_delta.h; the forward's
// formulas and names in delta_chunk.hip).
//
// With dS the gradient of the state after a chunk, P the masked and scaled scores and q, k the
// normed ones:
//   dN = P^T dO + e^{G_C - G} (K dS),   Y = Tm^T dN,
//   dS <- e^{G_C} dS + Q^T (scale e^G dO) - K^T (beta e^G Y),
// which goes from chunk to chunk (delta_scan.hip); then, here, for every chunk at once, with dP = dO N^T for j <= i and E = Y N^T for j < i:
//   dq  = scale (e^G (dO S^T) + (dP D) K),
//   z   = -(e^G (Y S^T) + (E D) K),                    (what k reads with, over beta)
//   dkw = e^{G_C - G} (N dS^T) + scale (dP D)^T Q - (beta E D)^T K,     (what k writes with)
//   dk = beta z + dkw,  dv = beta Y,  dbeta = k . z + v . Y,
//   dG_i = q . dq + beta k . z - k . dkw,  dG_C += sum k . e^{G_C - G} (N dS^T) + e^{G_C} <S, dS>,
// and dg the sums of dG from a token to its chunk's end. The terms of pairs on one side of a token
// cancel in that sum, which is why both sides of a pair multiply the same rounded operand: one that
// has all its factors, for the raw q and k. (Rounded before the factors of one side, the operands
// of the other differ by a bfloat16 step, and dg was 9e-3 off at 40 tokens of one head.)
#include "delta.hpp"

namespace tops {

namespace {

template <typename T, int KP>
struct GradLds {
  static constexpr int C = delta_c<T>(), VS = 32;   // values of a slab
  static constexpr int PK = pitch_of<T>(KP), PC = pitch_of<T>(C), PS = pitch_of<T>(VS);
  static constexpr int K0 = 0, Q0 = C * PK, N0 = 2 * C * PK, Y0 = N0 + VS * PC, S0 = Y0 + VS * PC;
  static constexpr int D0 = S0 + VS * PK, O0 = D0 + VS * PK, END = O0 + C * PS;
  static constexpr int G0 = (END * (int)sizeof(T) + 15) / 16 * 16;   // G [C] in 64 bits
  static constexpr int F0 = G0 + 8 * C;                              // [6][C] floats
  static constexpr int BYTES = F0 + (6 * C + 8) * 4;
};

__device__ __forceinline__ float group_sum(float x) {   // over the four lanes of a column
  x = swap16_add(x, x);
  return swap32_add(x, x);
}

// Row i of a [C][KP] tile times accumulators whose columns are tokens.
template <typename T, int NS>
__device__ __forceinline__ float row_dot(const T* row, const f32x4 (&acc)[2 * NS], int g) {
  float sum = 0.f;
#pragma unroll
  for (int s = 0; s < NS; ++s) {
    float x[8], y[8];
    values_of(ld_frag(row + 32 * s + 8 * g), x);
    pair_values(acc[2 * s], acc[2 * s + 1], y);
#pragma unroll
    for (int e = 0; e < 8; ++e) sum = fmaf(x[e], y[e], sum);
  }
  return group_sum(sum);
}

// A wave has 16 tokens of a chunk as columns of all its products; a block goes through the value
// heads of its key head (GROUP: more than one), so that their sums need no second launch.
template <typename T, int KP, bool GROUP>
__global__ __launch_bounds__(4 * delta_c<T>()) void delta_grad_kernel(DeltaParams p) {
  using L = GradLds<T, KP>;
  constexpr int C = L::C, NT = 4 * C, NS = KP / 32, NU = C / 32, VS = L::VS;
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  const tops_gla_delta_args& a = p.a;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int g = lane >> 4, i = 16 * wave + (lane & 15), uw = wave / 2;
  const int K = (int)a.K, V = (int)a.V, H = (int)a.H, HV = (int)a.HV;
  const int chunk = (int)(blockIdx.x / H), h = (int)(blockIdx.x % H);
  const ChunkAt at = delta_chunk_at(a, C, chunk);
  const bool in = i < at.len;
  T* sm = (T*)smem;
  T *sK = sm + L::K0, *sQ = sm + L::Q0, *sN = sm + L::N0, *sY = sm + L::Y0, *sS = sm + L::S0;
  T *sD = sm + L::D0, *sO = sm + L::O0;
  double* sG = (double*)(smem + L::G0);
  float* sf = (float*)(smem + L::F0);   // e^G, e^{G_C - G}, beta, 1 / |k|, 1 / |q|; dG; <S, dS>
  float *sdG = sf + 5 * C, *sSum = sf + 6 * C;
  {
    TileFetch<T, C, KP, NT> f;
    f.get((const T*)a.k + at.b * a.k_sb + at.t * a.k_st + h * a.k_sh, a.k_st, at.len, K, tid);
    f.put(sK, L::PK, at.len, K, tid);
    f.get((const T*)a.q + at.b * a.q_sb + at.t * a.q_st + h * a.q_sh, a.q_st, at.len, K, tid);
    f.put(sQ, L::PK, at.len, K, tid);
  }
  const T *kr = sK + i * L::PK, *qr = sQ + i * L::PK;
  const float scale = (float)a.scale;
  constexpr int NG = GROUP ? 2 * NS : 1;
  f32x4 dqs[NG], dks[NG];
  float sqs = 0.f, sks = 0.f;
#pragma unroll
  for (int x = 0; x < NG; ++x) dqs[x] = dks[x] = zero4();

  const int group = HV / H;
  for (int gi = 0; gi < group; ++gi) {
    const int hv = h * group + gi;
    const long unit = (long)chunk * HV + hv;
    const long tok = (long)at.b * a.T + at.t + i;
    const T* vp = (const T*)a.v + at.b * a.v_sb + (at.t + (long)min(i, at.len - 1)) * a.v_st +
                  hv * a.v_sh;
    const T* dop = (const T*)a.dout + at.b * a.do_sb + at.t * a.do_st + hv * a.do_sh;
    T* dvp = (T*)a.dv + (tok * HV + hv) * V;
    TileFetch<T, VS, C, NT> fn, fy;
    TileFetch<T, VS, KP, NT> fs, fd;
    TileFetch<T, C, VS, NT> fo;
    Run<T, 8> fv;
    auto fetch = [&](int v0) {
      fn.get((const T*)p.N + (unit * V + v0) * C, C, V - v0, C, tid);
      fy.get((const T*)p.Y + (unit * V + v0) * C, C, V - v0, C, tid);
      fs.get((const T*)p.S + (unit * V + v0) * KP, KP, V - v0, KP, tid);
      fd.get((const T*)p.dS + (unit * V + v0) * KP, KP, V - v0, KP, tid);
      fo.get(dop + v0, a.do_st, at.len, V - v0, tid);
      fv = get_run<T, 8>(vp + min(v0 + 8 * g, V - 8));
    };
    fetch(0);
    if (GROUP) __syncthreads();   // the vectors of the head before have been read
    {
      const float* vec = delta_vec(p, unit);
      for (int x = tid; x < 5 * C; x += NT) sf[x] = vec[x];
      if (tid < C) sG[tid] = delta_gsum(p, unit)[tid];
    }
    f32x4 dq[2 * NS], z[2 * NS], dkw[2 * NS], PT[2 * NU], ET[2 * NU], P2[2 * NU], E2[2 * NU];
#pragma unroll
    for (int x = 0; x < 2 * NS; ++x) dq[x] = z[x] = dkw[x] = zero4();
#pragma unroll
    for (int x = 0; x < 2 * NU; ++x) PT[x] = ET[x] = P2[x] = E2[x] = zero4();
    float vy = 0.f, sd = 0.f;
    float beta = 0.f;
    for (int v0 = 0; v0 < V; v0 += VS) {
      __syncthreads();
      fn.put(sN, L::PC, V - v0, C, tid);
      fy.put(sY, L::PC, V - v0, C, tid);
      fs.put(sS, L::PK, V - v0, KP, tid);
      fd.put(sD, L::PK, V - v0, KP, tid);
      fo.put(sO, L::PS, at.len, V - v0, tid);
#pragma unroll
      for (int x = 0; x < decltype(fs)::N; ++x)
#pragma unroll
        for (int e = 0; e < 8; ++e) sd = fmaf(to_f32(fs.r[x].v[e]), to_f32(fd.r[x].v[e]), sd);
      __syncthreads();
      const Run<T, 8> vr = fv;
      if (v0 + VS < V) fetch(v0 + VS);
      if (v0 == 0) beta = sf[2 * C + i];
      const Frag<T> of = ld_frag(sO + i * L::PS + 8 * g);
      const Frag<T> yf = ld_frag_t(sY + 16 * wave, L::PC, lane);
      const Frag<T> nf = ld_frag_t(sN + 16 * wave, L::PC, lane);
      const int c = v0 + 8 * g;
      {   // dv, and v . Y (Y is 0 past the end)
        float y[8], x[8];
        values_of(yf, y);
        values_of(frag_of<T>(cut_run(vr, c, V)), x);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          vy = in ? fmaf(x[e], y[e], vy) : 0.f;
          y[e] *= beta;
        }
        if (in && c < V) put_run<T, 8>(dvp + c, y, V - c);
      }
#pragma unroll
      for (int x = 0; x < 2 * NU; ++x) {
        const int u = x >> 1;
        if (u <= uw) {   // columns: this wave's tokens i, rows: tokens j
          const Frag<T> f = ld_pair_t(sN + 32 * u, L::PC, lane, x & 1);
          mma(PT[x], f, of);
          mma(ET[x], f, yf);
        }
        if (u >= uw) {   // columns: this wave's tokens as j, rows: tokens i
          mma(P2[x], ld_frag(sO + (32 * u + pair_row(lane, x & 1)) * L::PS + 8 * g), nf);
          mma(E2[x], ld_pair_t(sY + 32 * u, L::PC, lane, x & 1), nf);
        }
      }
#pragma unroll
      for (int x = 0; x < 2 * NS; ++x) {
        const Frag<T> f = ld_pair_t(sS + 32 * (x >> 1), L::PK, lane, x & 1);
        mma(dq[x], f, of);
        mma(z[x], f, yf);
        mma(dkw[x], ld_pair_t(sD + 32 * (x >> 1), L::PK, lane, x & 1), nf);
      }
    }
    const float gam = sf[i], gbar = sf[C + i], rk = sf[3 * C + i], rq = sf[4 * C + i];
    const double Gi = sG[i];
    // gradients of the raw q and k, but for the norms' own part; z times beta (times 1 where beta
    // is nothing that can be divided by: its own gradient needs z alone)
    const float aq = scale * rq, bz = fabsf(beta) < 0x1p-64f ? 1.f : beta, ak = bz * rk;
    const float zb = bz == beta ? 1.f : beta;   // beta z over the accumulated
#pragma unroll
    for (int x = 0; x < 2 * NS; ++x) {
      dq[x] *= gam * aq;
      z[x] *= gam * ak;
      dkw[x] *= gbar * rk;
    }
    const float left = row_dot<T, NS>(kr, dkw, g);
#pragma unroll
    for (int u = 0; u < NU; ++u) {
      float x[8], y[8];
      if (u <= uw) {
        pair_values(PT[2 * u], PT[2 * u + 1], x);
        pair_values(ET[2 * u], ET[2 * u + 1], y);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int j = 32 * u + 8 * g + e;
          const float d = j <= i ? gexp<T>((float)(Gi - sG[j])) : 0.f, rj = sf[3 * C + j];
          x[e] = j <= i ? x[e] * (d * (aq * rj)) : 0.f;
          y[e] = j < i ? y[e] * (d * (ak * rj)) : 0.f;
        }
        const Frag<T> fx = frag_of<T>(x), fyy = frag_of<T>(y);
#pragma unroll
        for (int s = 0; s < 2 * NS; ++s) {
          const Frag<T> f = ld_pair_t(sK + 32 * u * L::PK + 32 * (s >> 1), L::PK, lane, s & 1);
          mma(dq[s], f, fx);
          mma(z[s], f, fyy);
        }
      }
      if (u >= uw) {
        pair_values(P2[2 * u], P2[2 * u + 1], x);
        pair_values(E2[2 * u], E2[2 * u + 1], y);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int j = 32 * u + 8 * g + e;
          const float d = j >= i ? gexp<T>((float)(sG[j] - Gi)) : 0.f;
          const float aj = scale * sf[4 * C + j], bj = sf[2 * C + j] * sf[3 * C + j];
          x[e] = j >= i ? x[e] * (d * (aj * rk)) : 0.f;
          y[e] = j > i ? -(y[e] * (d * (bj * rk))) : 0.f;
        }
        const Frag<T> fx = frag_of<T>(x), fyy = frag_of<T>(y);
#pragma unroll
        for (int s = 0; s < 2 * NS; ++s) {
          const int off = 32 * u * L::PK + 32 * (s >> 1);
          mma(dkw[s], ld_pair_t(sQ + off, L::PK, lane, s & 1), fx);
          mma(dkw[s], ld_pair_t(sK + off, L::PK, lane, s & 1), fyy);
        }
      }
    }
    const float sq = row_dot<T, NS>(qr, dq, g), sw = row_dot<T, NS>(kr, dkw, g);
    const float sz = -row_dot<T, NS>(kr, z, g);
    vy = group_sum(vy);
    if (g == 0) {
      sdG[i] = sq + zb * sz - sw;
      if (in) put_any(a.dbeta, (int)a.beta_dtype, tok * HV + hv, sz / bz + vy);
    }
    {   // e^{G_C} <S, dS>, and the part of dG_C that the tokens' decays to it have
      sd *= sf[C - 1];
      sd += g == 0 ? left : 0.f;
      sd += dpp<0x121>(sd);
      sd += dpp<0x122>(sd);
      sd += dpp<0x124>(sd);
      sd += dpp<0x128>(sd);
      sd = group_sum(sd);
      if (lane == 0) sSum[wave] = sd;
    }
    __syncthreads();
    if (wave == 0) {
      float s = lane < C ? sdG[lane] : 0.f;
#pragma unroll
      for (int w = 0; w < C / 16; ++w) s += lane == C - 1 ? sSum[w] : 0.f;
#pragma unroll
      for (int o = 1; o < C; o <<= 1) {
        const float x = __shfl_down(s, o);
        if (lane + o < C) s += x;
      }
      if (lane < at.len)
        put_any(a.dg, (int)a.g_dtype,
                ((long)at.b * a.T + at.t + lane) * HV + hv, s);
    }
    const float sk = zb * sz + sw;
    if (GROUP) {
#pragma unroll
      for (int x = 0; x < 2 * NS; ++x) {
        dqs[GROUP ? x : 0] += dq[x];
        dks[GROUP ? x : 0] += dkw[x] - zb * z[x];
      }
      sqs += sq;
      sks += sk;
      if (gi + 1 < group) continue;
    }
    const float nq = a.l2norm ? rq * rq * (GROUP ? sqs : sq) : 0.f;
    const float nk = a.l2norm ? rk * rk * (GROUP ? sks : sk) : 0.f;
    if (in) {
      T* dqo = (T*)a.dq + (tok * H + h) * K;
      T* dko = (T*)a.dk + (tok * H + h) * K;
#pragma unroll
      for (int s = 0; s < NS; ++s) {
        const int c = 32 * s + 8 * g;
        if (c >= K) continue;
        float x[8], y[8];
        values_of(ld_frag(qr + c), x);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float d = GROUP ? dqs[GROUP ? 2 * s + e / 4 : 0][e % 4] : dq[2 * s + e / 4][e % 4];
          y[e] = d - nq * x[e];
        }
        put_run<T, 8>(dqo + c, y, K - c);
        values_of(ld_frag(kr + c), x);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float d = GROUP ? dks[GROUP ? 2 * s + e / 4 : 0][e % 4]
                                : dkw[2 * s + e / 4][e % 4] - zb * z[2 * s + e / 4][e % 4];
          y[e] = d - nk * x[e];
        }
        put_run<T, 8>(dko + c, y, K - c);
      }
    }
  }
}

template <typename T, int KP, bool GROUP>
hipError_t launch_grad(const DeltaParams& p, hipStream_t st) {
  constexpr int lds = GradLds<T, KP>::BYTES;
  const hipError_t e = hipFuncSetAttribute((const void*)delta_grad_kernel<T, KP, GROUP>,
                                           hipFuncAttributeMaxDynamicSharedMemorySize, lds);
  if (e != hipSuccess) return e;
  delta_grad_kernel<T, KP, GROUP>
      <<<(unsigned)(p.a.chunks * p.a.H), 4 * delta_c<T>(), lds, st>>>(p);
  return hipGetLastError();
}

template <typename T, int KP>
hipError_t run(const DeltaParams& p, hipStream_t st) {
  return p.a.HV > p.a.H ? launch_grad<T, KP, true>(p, st) : launch_grad<T, KP, false>(p, st);
}

}  // namespace

hipError_t run_delta_grad(const DeltaParams& p, hipStream_t st) {
  if (p.a.dtype == DT_BF16)
    return p.KP == 64 ? run<bf16, 64>(p, st) : p.KP == 128 ? run<bf16, 128>(p, st)
                                                           : run<bf16, 256>(p, st);
  return p.KP == 64 ? run<float, 64>(p, st) : p.KP == 128 ? run<float, 128>(p, st)
                                                          : run<float, 256>(p, st);
}

}  // namespace tops
