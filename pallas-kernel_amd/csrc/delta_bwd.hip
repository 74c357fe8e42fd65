// The gradients of the gated delta rule over chunks (include/tops_gla_delta.h; the forward's
// formulas and names in delta_chunk.hip).
//
// With dS the gradient of the state after a chunk, P the masked and scaled scores and q, k the
// normed ones:
//   dN = P^T dO + e^{G_C - G} (K dS),   Y = Tm^T dN,
//   dS <- e^{G_C} dS + Q^T (scale e^G dO) - K^T (beta e^G Y),
// which goes from chunk to chunk (delta_scan.hip); then, here, for every chunk at once, with
// dP = dO N^T for j <= i and E = Y N^T for j < i:
//   dq  = scale (e^G (dO S^T) + (dP D) K),
//   z   = -(e^G (Y S^T) + (E D) K),                    (what k reads with, over beta)
//   dkw = e^{G_C - G} (N dS^T) + scale (dP D)^T Q - (beta E D)^T K,     (what k writes with)
//   dk = beta z + dkw,  dv = beta Y,  dbeta = k . z + v . Y,
//   dG_i = q . dq + beta k . z - k . dkw,  dG_C += sum k . e^{G_C - G} (N dS^T) + e^{G_C} <S, dS>,
// and dg the sums of dG from a token to its chunk's end. The terms of pairs on one side of a token
// cancel in that sum, which is why both sides of a pair multiply the same rounded operand: one that
// has all its factors, for the raw q and k.
//
// What the products take from the passes (N, Y, S, dS) and the scores' gradients are two bfloat16 parts
// where the operands' type is that: a gradient of bfloat16 is then rounded once, its own rounding, and
// one of float32 (dg, dbeta) about 1e-5 off. (In one part gradients were 3e-3 off, where their own
// rounding is 1.7e-3, and a training step took 513 us instead of 592.)
#include "delta.hpp"

namespace tops {

namespace {

template <typename T, int KP>
struct GradLds {
  // values of a slab: K = 64, V = 128, two value heads a key head, 5000 tokens: forward and backward in
  // 225 us, 232 with 32; K = 128 has no room in LDS for 64
  static constexpr int NT = delta_grad_threads(sizeof(T) == 2 ? DT_BF16 : DT_F32);
  static constexpr int C = delta_c<T>(), VS = sizeof(T) == 2 && KP == 64 ? 64 : 32;
  static constexpr int PK = pitch_of<T>(KP), PS = pitch_of<T>(VS);
  static constexpr int PC = pitch_of<T>(TWO<T> * C), PD = pitch_of<T>(TWO<T> * KP);   // parts in a row
  static constexpr int K0 = 0, Q0 = C * PK, N0 = 2 * C * PK, Y0 = N0 + VS * PC, S0 = Y0 + VS * PC;
  static constexpr int D0 = S0 + VS * PD, O0 = D0 + VS * PD, END = O0 + C * PS;
  // beta z on its way to the waves of the keys, where the slabs were
  static constexpr int PX = KP + 4, X0 = N0 * (int)sizeof(T);
  static constexpr int G0 = (std::max(END * (int)sizeof(T), X0 + C * PX * 4) + 15) / 16 * 16;
  static constexpr int F0 = G0 + 8 * C;                // after G [C] in 64 bits: [9][C] floats
  static constexpr int BYTES = F0 + (9 * C + 8) * 4;
  // behind them the sums over value heads of dq and dk, each lane's own, where they fit: of 128 keys
  // and two value heads a key head forward and backward take 1040 us, 1126 with the sums in registers,
  // which then spill; 64 keys 218 for 224. With 256 keys there is no room
  static constexpr int SUMS = 2 * C * PX * 4;
  static constexpr bool PARK = BYTES + SUMS <= 160 * 1024;
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

// Each wave has 16 tokens of a chunk as columns of all its products: half of a block's waves have
// them as queries (dq, z, dv and their rows of the scores' gradients), half as keys (dkw and their
// columns of these), so that no wave holds more accumulators than two waves a SIMD leave it. A block
// goes through the value heads of its key head (GROUP: more than one), so that their sums need no
// second launch.
//
// Bound by latency: one block a CU (249 registers), whose loads and products take turns: 2 x 4096
// tokens, 16 heads of 128 x 128, 637 MB in 200 us, 3.2 TB/s, where the bytes alone take 129. Two blocks a
// CU spill. 20 registers spill with 128 keys and several value heads, 65 with 256 keys, 114 with both;
// float32: 97 with both.
template <typename T, int KP, bool GROUP>
__global__ __launch_bounds__((GradLds<T, KP>::NT)) void delta_grad_kernel(DeltaParams p) {
  using L = GradLds<T, KP>;
  constexpr int C = L::C, NT = L::NT, NS = KP / 32, NU = C / 32, NW = C / 16;
  constexpr int VS = L::VS, NH = VS / 32;
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  const tops_gla_delta_args& a = p.a;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, tw = wave % NW;
  const bool key = wave >= NW;
  const int g = lane >> 4, i = 16 * tw + (lane & 15), uw = tw / 2;
  const int K = (int)a.K, V = (int)a.V, H = (int)a.H, HV = (int)a.HV;
  const int chunk = (int)(blockIdx.x / H), h = (int)(blockIdx.x % H);
  const ChunkAt at = delta_chunk_at(a, C, chunk);
  const bool in = i < at.len;
  T* sm = (T*)smem;
  T *sK = sm + L::K0, *sQ = sm + L::Q0, *sN = sm + L::N0, *sY = sm + L::Y0, *sS = sm + L::S0;
  T *sD = sm + L::D0, *sO = sm + L::O0;
  float* sX = (float*)(smem + L::X0);
  double* sG = (double*)(smem + L::G0);
  float* sf = (float*)(smem + L::F0);   // the unit's vectors; dG, k . beta z, <S, dS>
  float *sdG = sf + 7 * C, *sKz = sf + 8 * C, *sSum = sf + 9 * C;
  const int group = HV / H;
  // a slab of a value head, on its way while the one before is multiplied (AHEAD); all of a block's
  // first loads start together
  constexpr int NP = TWO<T>;
  // 256 keys leave no registers for a slab on its way: 1394 us of a training step with 291 spilled ones,
  // 1129 with 65
  constexpr bool AHEAD = KP < 256 || sizeof(T) == 4;
  TileFetch<T, VS, NP * C, NT> fn, fy;
  TileFetch<T, VS, KP, NT> fs[NP], fd[NP];   // a part each, so that a thread has all of an element
  TileFetch<T, C, VS, NT> fo;
  Run<T, 8> fv[NH];
  auto fetch = [&](int hv, int v0) {
    const long unit = (long)chunk * HV + hv;
    const long row = (unit * V + v0) * NP;
    fn.get((const T*)p.N + row * C, NP * C, V - v0, NP * C, tid);
    fy.get((const T*)p.Y + row * C, NP * C, V - v0, NP * C, tid);
#pragma unroll
    for (int x = 0; x < NP; ++x) {
      fs[x].get((const T*)p.S + row * KP + x * KP, NP * KP, V - v0, KP, tid);
      fd[x].get((const T*)p.dS + row * KP + x * KP, NP * KP, V - v0, KP, tid);
    }
    fo.get((const T*)a.dout + at.b * a.do_sb + at.t * a.do_st + hv * a.do_sh + v0, a.do_st, at.len,
           V - v0, tid);
    if (!key)
#pragma unroll
      for (int u = 0; u < NH; ++u)
        fv[u] = get_run<T, 8>((const T*)a.v + at.b * a.v_sb + hv * a.v_sh +
                              (at.t + (long)min(i, at.len - 1)) * a.v_st +
                              min(v0 + 32 * u + 8 * g, V - 8));
  };
  {
    TileFetch<T, C, KP, NT> fk, fq;
    fk.get((const T*)a.k + at.b * a.k_sb + at.t * a.k_st + h * a.k_sh, a.k_st, at.len, K, tid);
    fq.get((const T*)a.q + at.b * a.q_sb + at.t * a.q_st + h * a.q_sh, a.q_st, at.len, K, tid);
    if (AHEAD) fetch(h * group, 0);
    fk.put(sK, L::PK, at.len, K, tid);
    fq.put(sQ, L::PK, at.len, K, tid);
  }
  const T *kr = sK + i * L::PK, *qr = sQ + i * L::PK;
  const float scale = (float)a.scale;
  // over the value heads: dq, or dk, in registers where LDS has no room for them
  constexpr bool HELD = GROUP && !L::PARK;
  f32x4 sum[HELD ? 2 * NS : 1];
  float* parked = (float*)(smem + L::BYTES) + ((key ? C : 0) + i) * L::PX + 8 * g;
  float dots = 0.f;   // and its product with q, or k
#pragma unroll
  for (int x = 0; x < (HELD ? 2 * NS : 1); ++x) sum[x] = zero4();

  for (int gi = 0; gi < group; ++gi) {
    const int hv = h * group + gi;
    const long unit = (long)chunk * HV + hv;
    const long tok = (long)at.b * a.T + at.t + i;
    T* dvp = (T*)a.dv + (tok * HV + hv) * V;
    if (GROUP) __syncthreads();   // the vectors of the head before have been read
    {
      const float* vec = delta_vec(p, unit);
      for (int x = tid; x < 7 * C; x += NT) sf[x] = vec[x];
      if (tid < C) sG[tid] = delta_gsum(p, unit)[tid];
    }
    // of a query: dq, z, and its rows of dP and E, transposed; of a key: dkw (and nothing), and its
    // columns of them
    f32x4 A[2][2 * NS], B[2][2 * NU];
#pragma unroll
    for (int x = 0; x < 2 * NS; ++x) A[0][x] = A[1][x] = zero4();
#pragma unroll
    for (int x = 0; x < 2 * NU; ++x) B[0][x] = B[1][x] = zero4();
    float vy = 0.f, sd = 0.f, beta = 0.f;
    for (int v0 = 0; v0 < V; v0 += VS) {
      if (!AHEAD) fetch(hv, v0);
      __syncthreads();
      fn.put(sN, L::PC, V - v0, NP * C, tid);
      fy.put(sY, L::PC, V - v0, NP * C, tid);
#pragma unroll
      for (int x = 0; x < NP; ++x) {
        fs[x].put(sS + x * KP, L::PD, V - v0, KP, tid);
        fd[x].put(sD + x * KP, L::PD, V - v0, KP, tid);
      }
      fo.put(sO, L::PS, at.len, V - v0, tid);
#pragma unroll
      for (int x = 0; x < TileFetch<T, VS, KP, NT>::N; ++x) {
        Split<T, NP> s, d;
#pragma unroll
        for (int i = 0; i < NP; ++i) {
          s.p[i] = fs[i].piece(x, V - v0, KP, tid);
          d.p[i] = fd[i].piece(x, V - v0, KP, tid);
        }
        float ss[8], dd[8];
        sum_of(s, ss);
        sum_of(d, dd);
#pragma unroll
        for (int e = 0; e < 8; ++e) sd = fmaf(ss[e], dd[e], sd);
      }
      Run<T, 8> vr[NH];
#pragma unroll
      for (int u = 0; u < NH; ++u) vr[u] = fv[u];
      __syncthreads();
      if (AHEAD && v0 + VS < V)
        fetch(hv, v0 + VS);
      else if (AHEAD && GROUP && gi + 1 < group)
        fetch(hv + 1, 0);
      beta = sf[2 * C + i];
#pragma unroll 1
      for (int u = 0; u < NH; ++u) {   // 32 values
        const T *uN = sN + 32 * u * L::PC, *uY = sY + 32 * u * L::PC, *uO = sO + 32 * u;
        if (u > 0 && v0 + 32 * u >= V) break;
        if (!key) {
          const Frag<T> of = ld_frag(uO + i * L::PS + 8 * g);
          Two<T> yf;
#pragma unroll
          for (int x = 0; x < NP; ++x) yf.p[x] = ld_frag_t(uY + 16 * tw + x * C, L::PC, lane);
          const int c = v0 + 32 * u + 8 * g;
          float y[8], x[8];   // dv, and v . Y (Y is 0 past the end)
          sum_of(yf, y);
          values_of(frag_of<T>(cut_run(u ? vr[NH - 1] : vr[0], c, V)), x);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            vy = in ? fmaf(x[e], y[e], vy) : 0.f;
            y[e] *= beta;
          }
          if (in && c < V) put_run<T, 8>(dvp + c, y, V - c);
#pragma unroll
          for (int n = 0; n < 2 * NU; ++n)
            if ((n >> 1) <= uw) {
              const Two<T> f = ld_split_t<T, NP>(uN + 32 * (n >> 1), C, L::PC, lane, n & 1);
              mma(B[0][n], f, of);
              mma(B[1][n], f, yf);
            }
#pragma unroll
          for (int n = 0; n < 2 * NS; ++n) {
            const Two<T> f =
                ld_split_t<T, NP>(sS + 32 * u * L::PD + 32 * (n >> 1), KP, L::PD, lane, n & 1);
            mma(A[0][n], f, of);
            mma(A[1][n], f, yf);
          }
        } else {
          Two<T> nf;
#pragma unroll
          for (int x = 0; x < NP; ++x) nf.p[x] = ld_frag_t(uN + 16 * tw + x * C, L::PC, lane);
#pragma unroll
          for (int n = 0; n < 2 * NU; ++n)
            if ((n >> 1) >= uw) {
              const int r = 32 * (n >> 1) + pair_row(lane, n & 1);
              mma(B[0][n], ld_frag(uO + r * L::PS + 8 * g), nf);
              mma(B[1][n], ld_split_t<T, NP>(uY + 32 * (n >> 1), C, L::PC, lane, n & 1), nf);
            }
#pragma unroll
          for (int n = 0; n < 2 * NS; ++n)
            mma(A[0][n],
                ld_split_t<T, NP>(sD + 32 * u * L::PD + 32 * (n >> 1), KP, L::PD, lane, n & 1), nf);
        }
      }
    }
    // Gradients of the raw q and k, but for the norms' own part; z times beta (times 1 where beta is
    // nothing that can be divided by: its own gradient needs z alone).
    const float rk = sf[3 * C + i], aq = scale * sf[6 * C + i];
    const float bz = fabsf(beta) < 0x1p-64f ? 1.f : beta, ak = bz * rk;
    const float zb = bz == beta ? 1.f : beta;   // beta z over the accumulated
    const double Gi = sG[i];
    float sw = 0.f;
    if (!key) {
      const float gam = sf[4 * C + i];
#pragma unroll
      for (int n = 0; n < 2 * NS; ++n) {
        A[0][n] *= gam * aq;
        A[1][n] *= gam * ak;
      }
#pragma unroll
      for (int u = 0; u < NU; ++u)
        if (u <= uw) {
          float x[8], y[8], d[8], rj[8];
          const int j = 32 * u + 8 * g;
          decays<T>(Gi, sG + j, 1.f, d);
          ld_eight(sf + 3 * C + j, rj);
          pair_values(B[0][2 * u], B[0][2 * u + 1], x);
          pair_values(B[1][2 * u], B[1][2 * u + 1], y);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            x[e] = j + e <= i ? x[e] * (d[e] * (aq * rj[e])) : 0.f;
            y[e] = j + e < i ? y[e] * (d[e] * (ak * rj[e])) : 0.f;
          }
          const Two<T> fx = split_of<T, NP>(x), fyy = split_of<T, NP>(y);
#pragma unroll
          for (int n = 0; n < 2 * NS; ++n) {
            const Frag<T> f = ld_pair_t(sK + 32 * u * L::PK + 32 * (n >> 1), L::PK, lane, n & 1);
            mma(A[0][n], f, fx);
            mma(A[1][n], f, fyy);
          }
        }
      const float sq = row_dot<T, NS>(qr, A[0], g), sz = -row_dot<T, NS>(kr, A[1], g);
      vy = group_sum(vy);
      if (g == 0) {
        sdG[i] = sq + zb * sz;
        sKz[i] = zb * sz;
        if (in) put_any(a.dbeta, (int)a.beta_dtype, tok * HV + hv, sz / bz + vy);
      }
      dots += sq;
    } else {
      const float gbar = sf[5 * C + i];
#pragma unroll
      for (int n = 0; n < 2 * NS; ++n) A[0][n] *= gbar * rk;
      const float left = row_dot<T, NS>(kr, A[0], g);
      sd = sd * sf[5 * C - 1] + (g == 0 ? left : 0.f);
#pragma unroll
      for (int u = 0; u < NU; ++u)
        if (u >= uw) {
          float x[8], y[8], d[8], rq[8], bj[8], rj[8];
          const int j = 32 * u + 8 * g;
          decays<T>(Gi, sG + j, -1.f, d);
          ld_eight(sf + 6 * C + j, rq);
          ld_eight(sf + 2 * C + j, bj);
          ld_eight(sf + 3 * C + j, rj);
          pair_values(B[0][2 * u], B[0][2 * u + 1], x);
          pair_values(B[1][2 * u], B[1][2 * u + 1], y);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            x[e] = j + e >= i ? x[e] * (d[e] * (scale * rq[e] * rk)) : 0.f;
            y[e] = j + e > i ? -(y[e] * (d[e] * (bj[e] * rj[e] * rk))) : 0.f;
          }
          const Two<T> fx = split_of<T, NP>(x), fyy = split_of<T, NP>(y);
#pragma unroll
          for (int n = 0; n < 2 * NS; ++n) {
            const int off = 32 * u * L::PK + 32 * (n >> 1);
            mma(A[0][n], ld_pair_t(sQ + off, L::PK, lane, n & 1), fx);
            mma(A[0][n], ld_pair_t(sK + off, L::PK, lane, n & 1), fyy);
          }
        }
      sw = row_dot<T, NS>(kr, A[0], g);
    }
    {   // e^{G_C} <S, dS>, and the part of dG_C that the tokens' decays to it have
      if (!key) sd *= sf[5 * C - 1];
      sd += dpp<0x121>(sd);
      sd += dpp<0x122>(sd);
      sd += dpp<0x124>(sd);
      sd += dpp<0x128>(sd);
      sd = group_sum(sd);
      if (lane == 0) sSum[wave] = sd;
    }
    __syncthreads();   // nobody reads the slabs any more
    if (!key) {
#pragma unroll
      for (int s = 0; s < NS; ++s)
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          f32x4 w = A[1][2 * s + x] * zb;
          *reinterpret_cast<f32x4*>(sX + i * L::PX + 32 * s + 8 * g + 4 * x) = w;
        }
    }
    __syncthreads();
    if (key) {
#pragma unroll
      for (int s = 0; s < NS; ++s)
#pragma unroll
        for (int x = 0; x < 2; ++x)
          A[0][2 * s + x] -=
              *reinterpret_cast<const f32x4*>(sX + i * L::PX + 32 * s + 8 * g + 4 * x);
      dots += sKz[i] + sw;
      if (g == 0) sdG[i] -= sw;
    }
    __syncthreads();
    if (wave == 0) {
      float s = lane < C ? sdG[lane] : 0.f;
#pragma unroll
      for (int w = 0; w < 2 * NW; ++w) s += lane == C - 1 ? sSum[w] : 0.f;
#pragma unroll
      for (int o = 1; o < C; o <<= 1) {
        const float x = __shfl_down(s, o);
        if (lane + o < C) s += x;
      }
      if (lane < at.len)
        put_any(a.dg, (int)a.g_dtype,
                ((long)at.b * a.T + at.t + lane) * HV + hv, s);
    }
    if (GROUP) {
#pragma unroll
      for (int x = 0; x < 2 * NS; ++x) {
        f32x4& to = HELD ? sum[HELD ? x : 0]
                         : *reinterpret_cast<f32x4*>(parked + 32 * (x >> 1) + 4 * (x & 1));
        if (HELD || gi > 0) A[0][x] += to;
        to = A[0][x];
      }
      if (gi + 1 < group) continue;
    }
    if (in) {
      const float r = sf[(key ? 3 : 6) * C + i], norm = a.l2norm ? r * r * dots : 0.f;
      const T* row = key ? kr : qr;
      T* to = (T*)(key ? a.dk : a.dq) + (tok * H + h) * K;
#pragma unroll
      for (int s = 0; s < NS; ++s) {
        const int c = 32 * s + 8 * g;
        if (c >= K) continue;
        float x[8], y[8];
        values_of(ld_frag(row + c), x);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          y[e] = A[0][2 * s + e / 4][e % 4] - norm * x[e];
        }
        put_run<T, 8>(to + c, y, K - c);
      }
    }
  }
}

template <typename T, int KP, bool GROUP>
hipError_t launch_grad(const DeltaParams& p, hipStream_t st) {
  using L = GradLds<T, KP>;
  constexpr int lds = L::BYTES + (GROUP && L::PARK ? L::SUMS : 0);
  static_assert(lds <= 160 * 1024, "LDS");
  const hipError_t e = hipFuncSetAttribute((const void*)delta_grad_kernel<T, KP, GROUP>,
                                           hipFuncAttributeMaxDynamicSharedMemorySize, lds);
  if (e != hipSuccess) return e;
  delta_grad_kernel<T, KP, GROUP>
      <<<(unsigned)(p.a.chunks * p.a.H), L::NT, lds, st>>>(p);
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
