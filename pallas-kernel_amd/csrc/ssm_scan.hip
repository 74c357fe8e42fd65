// Selective state space scan, forward and backward (include/tops_gla_ssm.h has the formulas).
//
// A wave owns 64 / LQ channels: a lane holds four consecutive states n of one channel, the LQ
// lanes of a channel are 64 / LQ apart. A block of 8 waves walks a piece of one sequence in
// tiles of 16 tokens: its threads load the tile's rows as contiguous runs of channels, form
// delta' and delta' u once for each (token, channel), and leave them in LDS for the waves.
//
// Pieces: h_t = a_t h_{t-1} + b_t is linear, so a sequence is cut into pieces that run in
// parallel: a first launch finds each piece's state from zero (L) and its summed delta' (S), and
// a piece of the second launch folds those of the pieces before it, h <- exp(A S_j) h + L_j.
#include "common.hpp"
#include "ssm.hpp"

namespace tops {

namespace {

constexpr int SS_NT = 512;   // threads of a block
constexpr int SS_K = 16;     // tokens of a tile, and of a chunk of the backward
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

template <int LQ>
struct Lay {
  static constexpr int CPW = 64 / LQ;            // channels of a wave
  static constexpr int CT = 8 * CPW;             // channels of a block
  static constexpr int NP = 4 * LQ;              // padded state size
  static constexpr int EPT = SS_K * CT / SS_NT;  // channels of a thread in a tile's row
  static constexpr int YP = CT + 16;             // row pitch of the tiles in lane order
  static constexpr int BPT = LQ / 4;             // elements of B and C a thread stages
};

struct Piece {
  int seq, t0, t1, idx, np, c0;
  long b;
};

__device__ __forceinline__ Piece piece_of(const ScanParams& p, int i) {
  Piece r;
  if (p.a.segs) {
    const int* s = p.a.segs + 8L * i;
    r.seq = s[0], r.t0 = s[1], r.t1 = s[2], r.idx = s[3], r.np = s[4], r.c0 = s[5];
    r.b = 0;
  } else {
    const int T = (int)p.a.T, len = (int)p.a.piece;
    r.np = p.pieces;
    r.seq = i / r.np;
    r.idx = i - r.seq * r.np;
    r.t0 = r.idx * len;
    r.t1 = min(T, r.t0 + len);
    r.c0 = r.seq * ((T + SS_K - 1) / SS_K) + r.t0 / SS_K;
    r.b = r.seq;
  }
  return r;
}

// N consecutive elements from `nv` valid ones (the others read as zero); `vec`: whole, aligned.
template <typename T, int N>
__device__ __forceinline__ void load_run(const T* p, int nv, bool vec, float (&x)[N]) {
  if (vec && nv >= N) {
    if constexpr (sizeof(T) == 2 && N == 4) {
      const uint2 w = *reinterpret_cast<const uint2*>(p);
      x[0] = bf16_lo(w.x), x[1] = bf16_hi(w.x), x[2] = bf16_lo(w.y), x[3] = bf16_hi(w.y);
      return;
    } else if constexpr (sizeof(T) == 2 && N == 2) {
      const uint32_t w = *reinterpret_cast<const uint32_t*>(p);
      x[0] = bf16_lo(w), x[1] = bf16_hi(w);
      return;
    } else if constexpr (sizeof(T) == 4 && N == 4) {
      const float4 w = *reinterpret_cast<const float4*>(p);
      x[0] = w.x, x[1] = w.y, x[2] = w.z, x[3] = w.w;
      return;
    } else if constexpr (sizeof(T) == 4 && N == 2) {
      const float2 w = *reinterpret_cast<const float2*>(p);
      x[0] = w.x, x[1] = w.y;
      return;
    }
  }
#pragma unroll
  for (int e = 0; e < N; ++e) x[e] = e < nv ? to_f32(p[e]) : 0.f;
}

template <typename T, int N>
__device__ __forceinline__ void store_n(T* p, int nv, bool vec, const float (&x)[N]) {
  if constexpr (N > 1) {
    if (vec && nv >= N) {
      store_run<T, N>(p, x);
      return;
    }
  }
#pragma unroll
  for (int e = 0; e < N; ++e)
    if (e < nv) p[e] = from_f32<T>(x[e]);
}

__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }

// Sum of the LQ lanes of each channel for four tokens' values; the lanes of row r = lane / 16
// end with token {0, 2, 1, 3}[r].
template <int LQ>
__device__ __forceinline__ float sum_states(float v0, float v1, float v2, float v3) {
  float v[4] = {v0, v1, v2, v3};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (LQ >= 8) v[i] += dpp<0x128>(v[i]);    // row_ror:8
    if constexpr (LQ >= 16) v[i] += dpp<0x124>(v[i]);   // row_ror:4
  }
  const float a = swap32_add(v[0], v[1]), b = swap32_add(v[2], v[3]);
  return swap16_add(a, b);
}

// ---------------------------------------------------------------------------
// Forward: MODE 0 a piece's own state and summed delta', 1 the outputs; MODE 2 the reverse of 0
// for the backward: the carry that a piece hands to the one before it, from a zero carry.
// ---------------------------------------------------------------------------
template <typename T, int LQ, int MODE>
__global__ __launch_bounds__(SS_NT) void scan_kernel(ScanParams p) {
  using L = Lay<LQ>;
  __shared__ float2 sDD[SS_K][L::CT];
  __shared__ float sB[SS_K][L::NP];
  __shared__ float sC[MODE == 1 ? SS_K : 1][L::NP];
  __shared__ float sY[MODE == 1 ? SS_K : 1][L::YP];
  const tops_gla_scan_args& a = p.a;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int tile = blockIdx.x % p.ntiles, pi = blockIdx.x / p.ntiles;
  const Piece pc = piece_of(p, pi);
  if (MODE == 0 && pc.idx == pc.np - 1) return;   // nobody folds it
  if (MODE == 2 && pc.idx == 0) return;
  const int D = (int)a.D, N = (int)a.N;
  const int DG = D / (int)a.G, grp = tile / p.tiles_g;
  const int cb = (tile % p.tiles_g) * L::CT;      // first channel of the block in its group
  const int d0 = grp * DG + cb, nch = min(L::CT, DG - cb);

  // the lane's states
  const int ch = wave * L::CPW + (lane & (L::CPW - 1)), n0 = 4 * (lane / L::CPW);
  const bool live = ch < nch;
  const long dl = d0 + (live ? ch : 0);
  float A[4], h[4] = {};
#pragma unroll
  for (int i = 0; i < 4; ++i) A[i] = live && n0 + i < N ? a.A[dl * N + n0 + i] * kLog2e : 0.f;
  float dsum = 0.f;
  if (MODE == 1) {
    if (a.h0 && live)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (n0 + i < N) h[i] = a.h0[((long)pc.seq * D + dl) * N + n0 + i];
    for (int j = pi - pc.idx; j < pi; ++j) {
      const float4 l = *reinterpret_cast<const float4*>(a.piece_h + ((long)j * D + dl) * L::NP + n0);
      const float s = a.piece_dt[(long)j * D + dl];
      const float lv[4] = {l.x, l.y, l.z, l.w};
#pragma unroll
      for (int i = 0; i < 4; ++i)   // a zero state stays zero under a decay that overflows
        h[i] = h[i] == 0.f ? lv[i] : fmaf(exp2_hw(A[i] * s), h[i], lv[i]);
    }
  }

  // the thread's part of a tile
  const int tt = tid / (L::CT / L::EPT), tc = (tid % (L::CT / L::EPT)) * L::EPT;
  const int nv = min(L::EPT, nch - tc);
  float bias[L::EPT], dskip[L::EPT];
#pragma unroll
  for (int e = 0; e < L::EPT; ++e) {
    bias[e] = a.delta_bias && e < nv ? a.delta_bias[d0 + tc + e] : 0.f;
    dskip[e] = MODE == 1 && a.Dskip && e < nv ? a.Dskip[d0 + tc + e] : 0.f;
  }
  const T* gu = (const T*)(MODE == 2 ? a.dy : a.u) +
                pc.b * (MODE == 2 ? a.dy_sb : a.u_sb) + d0 + tc;
  const long u_st = MODE == 2 ? a.dy_st : a.u_st;
  const T* gd = (const T*)a.delta + pc.b * a.delta_sb + d0 + tc;
  const T* gz = (const T*)a.z + (a.z ? pc.b * a.z_sb + d0 + tc : 0);
  const T* gB = MODE == 2 ? (const T*)a.C + pc.b * a.C_sb + (long)grp * a.C_sg
                          : (const T*)a.B + pc.b * a.B_sb + (long)grp * a.B_sg;
  const long B_st = MODE == 2 ? a.C_st : a.B_st;
  const T* gC = (const T*)a.C + pc.b * a.C_sb + (long)grp * a.C_sg;
  const bool has_z = a.z != nullptr && MODE != 0;

  float ru[L::EPT], rd[L::EPT], rz[L::EPT], rb[L::BPT];
  constexpr int BN = SS_K * L::NP;   // elements of B of a tile
  auto load = [&](int t0) {
    const int t = t0 + tt;
    const int v = t < pc.t1 ? nv : 0;
    load_run<T, L::EPT>(gu + (v > 0 ? t * u_st : 0), v, p.vec, ru);
    load_run<T, L::EPT>(gd + (v > 0 ? t * a.delta_st : 0), v, p.vec, rd);
    if (has_z) load_run<T, L::EPT>(gz + (v > 0 ? t * a.z_st : 0), v, p.vec, rz);
#pragma unroll
    for (int j = 0; j < L::BPT; ++j) {
      const int i = tid + SS_NT * j;   // B, then C: 2 BN = BPT * SS_NT elements in all
      const int r = i % BN, bt = t0 + r / L::NP, n = r % L::NP;
      const bool ok = bt < pc.t1 && n < N && (i < BN || MODE == 1);
      const T* g = i < BN ? gB + (ok ? bt * B_st : 0) : gC + (ok ? bt * a.C_st : 0);
      rb[j] = ok ? to_f32(g[n]) : 0.f;
    }
  };
  const int nt = (pc.t1 - pc.t0 + SS_K - 1) / SS_K;
  const int first = MODE == 2 ? nt - 1 : 0, step = MODE == 2 ? -1 : 1;
  if (nt > 0) load(pc.t0 + first * SS_K);
  for (int it = 0; it < nt; ++it) {
    const int k = first + it * step, t0 = pc.t0 + k * SS_K;
    const bool valid = t0 + tt < pc.t1;
    float ku[L::EPT], kz[L::EPT];
    float2 dd[L::EPT];
#pragma unroll
    for (int e = 0; e < L::EPT; ++e) {
      float d = rd[e] + bias[e], sg;
      if (a.softplus) softplus_sigmoid(d, d, sg);
      if (!valid || e >= nv) d = 0.f;   // a token past the end leaves the state as it is
      float x = d * ru[e];
      if (MODE == 2) x = has_z ? ru[e] * rz[e] * sigmoid(rz[e]) : ru[e];
      dd[e] = make_float2(d, x);
      ku[e] = ru[e];
      kz[e] = rz[e];
    }
#pragma unroll
    for (int e = 0; e < L::EPT; ++e) sDD[tt][tc + e] = dd[e];
#pragma unroll
    for (int j = 0; j < L::BPT; ++j) {
      const int i = tid + SS_NT * j, r = i % BN;
      if (i < BN)
        sB[r / L::NP][r % L::NP] = rb[j];
      else if (MODE == 1)
        sC[r / L::NP][r % L::NP] = rb[j];
    }
    __syncthreads();
    if (it + 1 < nt) load(pc.t0 + (k + step) * SS_K);
    if (MODE == 1 && a.chunk_h && live)
      *reinterpret_cast<float4*>(a.chunk_h + ((long)(pc.c0 + k) * D + dl) * L::NP + n0) =
          make_float4(h[0], h[1], h[2], h[3]);
#pragma unroll
    for (int q = 0; q < SS_K; q += 4) {
      float yv[4];
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        const int t = MODE == 2 ? SS_K - 1 - (q + s) : q + s;
        const float2 d = sDD[t][ch];
        const float4 b4 = *reinterpret_cast<const float4*>(&sB[t][n0]);
        const float bv[4] = {b4.x, b4.y, b4.z, b4.w};
        float cv[4] = {};
        if (MODE == 1) {
          const float4 c4 = *reinterpret_cast<const float4*>(&sC[t][n0]);
          cv[0] = c4.x, cv[1] = c4.y, cv[2] = c4.z, cv[3] = c4.w;
        }
        float y = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float ex = exp2_hw(A[i] * d.x);
          if (MODE == 2) {
            h[i] = ex * fmaf(bv[i], d.y, h[i]);
          } else {
            h[i] = fmaf(ex, h[i], d.y * bv[i]);
            if (MODE == 1) y = i == 0 ? cv[0] * h[0] : fmaf(cv[i], h[i], y);
          }
        }
        yv[s] = y;
        if (MODE != 1) dsum += d.x;
      }
      if (MODE == 1) {
        const float y = sum_states<LQ>(yv[0], yv[1], yv[2], yv[3]);
        const int row = lane >> 4, tm = ((row & 1) << 1) | (row >> 1);
        if ((lane & 15) < L::CPW) sY[q + tm][wave * L::CPW + (lane & (L::CPW - 1))] = y;
      }
    }
    __syncthreads();
    if (MODE == 1 && valid && nv > 0) {
      float o[L::EPT];
#pragma unroll
      for (int e = 0; e < L::EPT; ++e) {
        o[e] = fmaf(dskip[e], ku[e], sY[tt][tc + e]);
        if (has_z) o[e] *= kz[e] * sigmoid(kz[e]);
      }
      T* gy = (T*)a.y + (pc.b * a.T + t0 + tt) * D + d0 + tc;
      store_n<T, L::EPT>(gy, nv, p.vec, o);
    }
  }
  if (!live) return;
  if (MODE == 1) {
    if (a.ht && pc.idx == pc.np - 1)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (n0 + i < N) a.ht[((long)pc.seq * D + dl) * N + n0 + i] = h[i];
  } else {
    *reinterpret_cast<float4*>(a.piece_h + ((long)pi * D + dl) * L::NP + n0) =
        make_float4(h[0], h[1], h[2], h[3]);
    if (n0 == 0) a.piece_dt[(long)pi * D + dl] = dsum;
  }
}

// ---------------------------------------------------------------------------
// Backward, over a piece's chunks of 16 tokens from the last one on. With g_t the gradient of
// h_t, g_t = C_t dy_t + a_{t+1} g_{t+1}:
//   dC_t = sum_d dy_t h_t          dB_t = sum_d g_t delta' u        du = delta' sum_n g B + D dy
//   ddelta' = u sum_n g B + sum_n g a h_{t-1} A                     dA = sum_t g a h_{t-1} delta'
// A chunk's states run forward again from the one that the forward kept, with a_t and h_t of its
// 16 tokens in registers (recovering h_{t-1} from h_t would divide by a_t).
// ---------------------------------------------------------------------------
template <typename T, int LQ>
__global__ __launch_bounds__(SS_NT, 2) void scan_bwd_kernel(ScanParams p) {
  using L = Lay<LQ>;
  __shared__ float2 sDD[SS_K][L::CT];
  __shared__ float sDy[SS_K][L::CT];
  __shared__ float sB[SS_K][L::NP], sC[SS_K][L::NP];
  __shared__ float sS[3][SS_K][L::YP];            // sum_n g B, sum_n g a h A log2(e), sum_n C h
  __shared__ float sBC[8][SS_K][2 * L::NP];       // a wave's dB and dC
  const tops_gla_scan_args& a = p.a;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int tile = blockIdx.x % p.ntiles, pi = blockIdx.x / p.ntiles;
  const Piece pc = piece_of(p, pi);
  const int D = (int)a.D, N = (int)a.N;
  const int DG = D / (int)a.G, grp = tile / p.tiles_g;
  const int cb = (tile % p.tiles_g) * L::CT;
  const int d0 = grp * DG + cb, nch = min(L::CT, DG - cb);
  const int ch = wave * L::CPW + (lane & (L::CPW - 1)), n0 = 4 * (lane / L::CPW);
  const bool live = ch < nch;
  const long dl = d0 + (live ? ch : 0);
  float A[4], carry[4] = {}, dA[4] = {};
#pragma unroll
  for (int i = 0; i < 4; ++i) A[i] = live && n0 + i < N ? a.A[dl * N + n0 + i] * kLog2e : 0.f;
  if (a.dht && live)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (n0 + i < N) carry[i] = a.dht[((long)pc.seq * D + dl) * N + n0 + i];
  for (int j = pi - pc.idx + pc.np - 1; j > pi; --j) {
    const float4 l = *reinterpret_cast<const float4*>(a.piece_h + ((long)j * D + dl) * L::NP + n0);
    const float s = a.piece_dt[(long)j * D + dl];
    const float lv[4] = {l.x, l.y, l.z, l.w};
#pragma unroll
    for (int i = 0; i < 4; ++i)
      carry[i] = carry[i] == 0.f ? lv[i] : fmaf(exp2_hw(A[i] * s), carry[i], lv[i]);
  }

  const int tt = tid / (L::CT / L::EPT), tc = (tid % (L::CT / L::EPT)) * L::EPT;
  const int nv = min(L::EPT, nch - tc);
  float bias[L::EPT], dskip[L::EPT], accD[L::EPT] = {}, accB[L::EPT] = {};
#pragma unroll
  for (int e = 0; e < L::EPT; ++e) {
    bias[e] = a.delta_bias && e < nv ? a.delta_bias[d0 + tc + e] : 0.f;
    dskip[e] = a.Dskip && e < nv ? a.Dskip[d0 + tc + e] : 0.f;
  }
  const T* gu = (const T*)a.u + pc.b * a.u_sb + d0 + tc;
  const T* gd = (const T*)a.delta + pc.b * a.delta_sb + d0 + tc;
  const T* gz = (const T*)a.z + (a.z ? pc.b * a.z_sb + d0 + tc : 0);
  const T* gy = (const T*)a.dy + pc.b * a.dy_sb + d0 + tc;
  const T* gB = (const T*)a.B + pc.b * a.B_sb + (long)grp * a.B_sg;
  const T* gC = (const T*)a.C + pc.b * a.C_sb + (long)grp * a.C_sg;
  const bool has_z = a.z != nullptr;
  float ru[L::EPT], rd[L::EPT], rz[L::EPT], ry[L::EPT], rb[L::BPT];
  float4 rh;
  constexpr int BN = SS_K * L::NP;
  auto load = [&](int k) {
    const int t0 = pc.t0 + k * SS_K, t = t0 + tt;
    const int v = t < pc.t1 ? nv : 0;
    load_run<T, L::EPT>(gu + (v > 0 ? t * a.u_st : 0), v, p.vec, ru);
    load_run<T, L::EPT>(gd + (v > 0 ? t * a.delta_st : 0), v, p.vec, rd);
    if (has_z) load_run<T, L::EPT>(gz + (v > 0 ? t * a.z_st : 0), v, p.vec, rz);
    load_run<T, L::EPT>(gy + (v > 0 ? t * a.dy_st : 0), v, p.vec, ry);
#pragma unroll
    for (int j = 0; j < L::BPT; ++j) {
      const int i = tid + SS_NT * j;
      const int r = i % BN, bt = t0 + r / L::NP, n = r % L::NP;
      const bool ok = bt < pc.t1 && n < N;
      const T* g = i < BN ? gB + (ok ? bt * a.B_st : 0) : gC + (ok ? bt * a.C_st : 0);
      rb[j] = ok ? to_f32(g[n]) : 0.f;
    }
    rh = *reinterpret_cast<const float4*>(a.chunk_h + ((long)(pc.c0 + k) * D + dl) * L::NP + n0);
  };
  const int nt = (pc.t1 - pc.t0 + SS_K - 1) / SS_K;
  if (nt > 0) load(nt - 1);
  for (int k = nt - 1; k >= 0; --k) {
    const int t0 = pc.t0 + k * SS_K;
    const bool valid = t0 + tt < pc.t1;
    float kd[L::EPT], ks[L::EPT], ku[L::EPT], kz[L::EPT], ky[L::EPT];
#pragma unroll
    for (int e = 0; e < L::EPT; ++e) {
      float d = rd[e] + bias[e], sg = 1.f;
      if (a.softplus) softplus_sigmoid(d, d, sg);
      if (!valid || e >= nv) d = 0.f;
      kd[e] = d;
      ks[e] = sg;
      ku[e] = ru[e];
      kz[e] = has_z ? rz[e] : 0.f;
      ky[e] = ry[e];
      sDD[tt][tc + e] = make_float2(d, d * ru[e]);
      sDy[tt][tc + e] = has_z ? ry[e] * rz[e] * sigmoid(rz[e]) : ry[e];
    }
#pragma unroll
    for (int j = 0; j < L::BPT; ++j) {
      const int i = tid + SS_NT * j, r = i % BN;
      (i < BN ? sB : sC)[r / L::NP][r % L::NP] = rb[j];
    }
    const float hin[4] = {live ? rh.x : 0.f, live ? rh.y : 0.f, live ? rh.z : 0.f,
                          live ? rh.w : 0.f};
    __syncthreads();
    if (k > 0) load(k - 1);

    float av[SS_K][4], hv[SS_K][4];
#pragma unroll
    for (int t = 0; t < SS_K; ++t) {
      const float2 d = sDD[t][ch];
      const float4 b4 = *reinterpret_cast<const float4*>(&sB[t][n0]);
      const float bv[4] = {b4.x, b4.y, b4.z, b4.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        av[t][i] = exp2_hw(A[i] * d.x);
        hv[t][i] = fmaf(av[t][i], t ? hv[t - 1][i] : hin[i], d.y * bv[i]);
      }
    }
#pragma unroll
    for (int q = SS_K - 4; q >= 0; q -= 4) {
      float s1[4], s2[4], s3[4];
#pragma unroll
      for (int s = 3; s >= 0; --s) {
        const int t = q + s;
        const float2 d = sDD[t][ch];
        const float dy = sDy[t][ch];
        const float4 b4 = *reinterpret_cast<const float4*>(&sB[t][n0]);
        const float4 c4 = *reinterpret_cast<const float4*>(&sC[t][n0]);
        const float bv[4] = {b4.x, b4.y, b4.z, b4.w}, cv[4] = {c4.x, c4.y, c4.z, c4.w};
        float v[8];
        s1[s] = s2[s] = s3[s] = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float g = fmaf(cv[i], dy, carry[i]);
          const float hp = t ? hv[t - 1][i] : hin[i];
          v[i] = g * d.y;
          v[4 + i] = dy * hv[t][i];
          s1[s] = fmaf(g, bv[i], s1[s]);
          carry[i] = av[t][i] * g;
          const float gp = carry[i] * hp;
          s2[s] = fmaf(gp, A[i], s2[s]);
          s3[s] = fmaf(cv[i], hv[t][i], s3[s]);
          dA[i] = fmaf(gp, d.x, dA[i]);
        }
        sum_channels<L::CPW>(v, lane, &sBC[wave][t][0], n0, L::NP);
      }
      const int row = lane >> 4, tm = ((row & 1) << 1) | (row >> 1);
      const float r1 = sum_states<LQ>(s1[0], s1[1], s1[2], s1[3]);
      const float r2 = sum_states<LQ>(s2[0], s2[1], s2[2], s2[3]);
      const float r3 = has_z ? sum_states<LQ>(s3[0], s3[1], s3[2], s3[3]) : 0.f;
      if ((lane & 15) < L::CPW) {
        const int c = wave * L::CPW + (lane & (L::CPW - 1));
        sS[0][q + tm][c] = r1;
        sS[1][q + tm][c] = r2;
        sS[2][q + tm][c] = r3;
      }
    }
    __syncthreads();
    if (valid && nv > 0) {
      float odu[L::EPT], odd[L::EPT], odz[L::EPT];
#pragma unroll
      for (int e = 0; e < L::EPT; ++e) {
        const float s1 = sS[0][tt][tc + e], s2 = sS[1][tt][tc + e];
        float dy = ky[e];
        if (has_z) {
          const float sz = sigmoid(kz[e]);
          dy = ky[e] * kz[e] * sz;
          odz[e] = ky[e] * fmaf(dskip[e], ku[e], sS[2][tt][tc + e]) *
                   (sz * fmaf(kz[e], 1.f - sz, 1.f));
        }
        odu[e] = fmaf(s1, kd[e], dskip[e] * dy);
        odd[e] = fmaf(s1, ku[e], s2 * kLn2) * ks[e];
        accD[e] = fmaf(dy, ku[e], accD[e]);
        accB[e] += odd[e];
      }
      const long o = (pc.b * a.T + t0 + tt) * D + d0 + tc;
      store_n<T, L::EPT>((T*)a.du + o, nv, p.vec, odu);
      store_n<T, L::EPT>((T*)a.ddelta + o, nv, p.vec, odd);
      if (has_z) store_n<T, L::EPT>((T*)a.dz + o, nv, p.vec, odz);
    }
    // the block's share of dB and dC: [tile of the group][token][group][2][NP]
    for (int i = tid; i < SS_K * 2 * L::NP; i += SS_NT) {
      const int t = i / (2 * L::NP), c = i % (2 * L::NP);
      float s = 0.f;
#pragma unroll
      for (int w = 0; w < 8; ++w) s += sBC[w][t][c];
      if (t0 + t < pc.t1)
        p.part_bc[(((long)(tile % p.tiles_g) * p.tokens + pc.b * a.T + t0 + t) * a.G + grp) *
                      (2 * L::NP) + c] = s;
    }
    // no wave writes sS or sBC again before the next barrier
  }
  if (live) {
    if (pc.idx == 0 && a.dh0)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (n0 + i < N) a.dh0[((long)pc.seq * D + dl) * N + n0 + i] = carry[i];
    *reinterpret_cast<float4*>(p.part_a + ((long)pi * D + dl) * L::NP + n0) =
        make_float4(dA[0], dA[1], dA[2], dA[3]);
  }
  // dD and the bias: sum over the block's 16 token rows
  __syncthreads();
  float* s0 = &sS[0][0][0];
#pragma unroll
  for (int e = 0; e < L::EPT; ++e) {
    s0[tt * L::CT + tc + e] = accD[e];
    s0[(SS_K + tt) * L::CT + tc + e] = accB[e];
  }
  __syncthreads();
  for (int i = tid; i < 2 * L::CT; i += SS_NT) {
    const int w = i / L::CT, c = i % L::CT;
    float s = 0.f;
    for (int t = 0; t < SS_K; ++t) s += s0[(w * SS_K + t) * L::CT + c];
    if (c < nch) p.part_d[((long)pi * 2 + w) * D + d0 + c] = s;
  }
}

// dB, dC from the blocks' shares: one thread per (token, group, array, n).
template <typename T>
__global__ __launch_bounds__(256) void scan_bwd_bc_kernel(ScanParams p, int NP) {
  const long total = p.tokens * p.a.G * 2 * NP;
  const int N = (int)p.a.N;
  for (long i = blockIdx.x * 256L + threadIdx.x; i < total; i += gridDim.x * 256L) {
    float s = 0.f;
    for (int t = 0; t < p.tiles_g; ++t) s += p.part_bc[t * total + i];
    const int c = (int)(i % (2 * NP)), n = c % NP;
    if (n < N) ((T*)(c < NP ? p.a.dB : p.a.dC))[(i / (2 * NP)) * N + n] = from_f32<T>(s);
  }
}

// dA, dD, dbias from the pieces' shares.
__global__ __launch_bounds__(256) void scan_bwd_a_kernel(ScanParams p, int NP) {
  const long D = p.a.D, na = D * NP, total = na + 2 * D;
  const int N = (int)p.a.N;
  for (long i = blockIdx.x * 256L + threadIdx.x; i < total; i += gridDim.x * 256L) {
    float s = 0.f;
    if (i < na) {
      for (long j = 0; j < p.npieces; ++j) s += p.part_a[j * na + i];
      const long d = i / NP, n = i % NP;
      if (n < N) p.a.dA[d * N + n] = s;
    } else {
      const long r = i - na;
      for (long j = 0; j < p.npieces; ++j) s += p.part_d[j * 2 * D + r];
      float* out = r < D ? p.a.dD : p.a.dbias;
      if (out) out[r % D] = s;
    }
  }
}

template <typename T, int LQ>
hipError_t scan_fwd(const ScanParams& p, hipStream_t st) {
  const dim3 grid((unsigned)(p.npieces * p.ntiles));
  if (p.multi) {
    hipLaunchKernelGGL((scan_kernel<T, LQ, 0>), grid, dim3(SS_NT), 0, st, p);
    if (hipError_t e = hipGetLastError()) return e;
  }
  hipLaunchKernelGGL((scan_kernel<T, LQ, 1>), grid, dim3(SS_NT), 0, st, p);
  return hipGetLastError();
}

template <typename T, int LQ>
hipError_t scan_bwd(const ScanParams& p, hipStream_t st) {
  const dim3 grid((unsigned)(p.npieces * p.ntiles));
  if (p.multi) {
    hipLaunchKernelGGL((scan_kernel<T, LQ, 2>), grid, dim3(SS_NT), 0, st, p);
    if (hipError_t e = hipGetLastError()) return e;
  }
  if (p.npieces > 0) {
    hipLaunchKernelGGL((scan_bwd_kernel<T, LQ>), grid, dim3(SS_NT), 0, st, p);
    if (hipError_t e = hipGetLastError()) return e;
  }
  constexpr int NP = Lay<LQ>::NP;
  const long nbc = p.tokens * p.a.G * 2 * NP, na = p.a.D * (NP + 2);
  if (nbc > 0) {
    hipLaunchKernelGGL((scan_bwd_bc_kernel<T>), dim3((unsigned)std::min<long>((nbc + 255) / 256, 1L << 20)),
                       dim3(256), 0, st, p, NP);
    if (hipError_t e = hipGetLastError()) return e;
  }
  hipLaunchKernelGGL(scan_bwd_a_kernel, dim3((unsigned)std::min<long>((na + 255) / 256, 1L << 20)),
                     dim3(256), 0, st, p, NP);
  return hipGetLastError();
}

template <typename T>
hipError_t scan_any(const ScanParams& p, bool backward, hipStream_t st) {
  switch (scan_state_pad((int)p.a.N)) {
    case 16: return backward ? scan_bwd<T, 4>(p, st) : scan_fwd<T, 4>(p, st);
    case 32: return backward ? scan_bwd<T, 8>(p, st) : scan_fwd<T, 8>(p, st);
    default: return backward ? scan_bwd<T, 16>(p, st) : scan_fwd<T, 16>(p, st);
  }
}

}  // namespace

int scan_state_pad(int N) { return N <= 16 ? 16 : N <= 32 ? 32 : 64; }
int scan_tile_channels(int N) { return 2048 / scan_state_pad(N); }

hipError_t run_selective_scan(const ScanParams& p, bool backward, hipStream_t st) {
  if (p.a.D == 0 || (p.npieces == 0 && !backward)) return hipSuccess;
  return p.a.dtype == DT_BF16 ? scan_any<bf16>(p, backward, st) : scan_any<float>(p, backward, st);
}

}  // namespace tops
