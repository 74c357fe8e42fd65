// The states of the gated delta rule, from chunk to chunk, and their gradients the other way
// (include/tops_gla_delta.h; formulas and names in delta_chunk.hip and delta_bwd.hip).
//
// The columns of S and N are independent of one another: a wave owns 16 or 32 of them over all
// chunks of a sequence and head, with the state in its accumulators; K S, Tm R and K^T N hand their
// results on as operands without leaving a lane. A block's waves share the chunk's tiles in LDS,
// with the next chunk's on their way.
//
// What bounds it is the chain of products of a chunk, one chunk after another. Where sequences,
// heads and columns do not fill the device, sequences are cut into segments: over a segment the
// state is a linear map of the state before it, S_end = M S + E, and M's columns run like others,
// from the identity and without values. A first pass has E and M of all segments at once, the fold
// E_j <- M_j E_{j-1} + E_j the state after each, and a second pass runs all segments from there.
// The gradients run with the same maps transposed.
#include "delta.hpp"

namespace tops {

namespace {

// Where a block works: columns of a segment of a sequence and head.
struct SegAt {
  int seq, j, count;   // segment j of `count` of the sequence
  int b, t, T;         // batch row, first token in it, tokens of the segment
  int chunk, n;        // first chunk of all, chunks of the segment
  int seg;             // of all segments
};
__device__ __forceinline__ SegAt seg_at(const tops_gla_delta_args& a, int C, int seg) {
  SegAt x;
  const int L = (int)a.seg_chunks;
  int t0, c0, T_;
  if (a.seqs) {
    const int n1 = (int)a.nseq + 1;
    x.seq = a.seqs[3 * n1 + seg];
    x.j = seg - a.seqs[2 * n1 + x.seq];
    x.count = a.seqs[2 * n1 + x.seq + 1] - a.seqs[2 * n1 + x.seq];
    t0 = a.seqs[x.seq];
    T_ = a.seqs[x.seq + 1] - t0;
    c0 = a.seqs[n1 + x.seq];
    x.b = 0;
  } else {
    x.count = (int)(a.nsegs / a.nseq);
    x.seq = seg / x.count;
    x.j = seg - x.seq * x.count;
    t0 = 0;
    T_ = (int)a.T;
    c0 = x.seq * ((T_ + C - 1) / C);
    x.b = x.seq;
  }
  const int nc = (T_ + C - 1) / C, first = x.j * L;
  x.n = min(L, nc - first);
  x.t = t0 + first * C;
  x.T = min(T_ - first * C, L * C);
  x.chunk = c0 + first;
  x.seg = seg;
  return x;
}

// Blocks of a head: NW waves of 16 CW columns each, of V or, in a first pass, then of KP for M.
template <typename T, int KP, int CW, int NW>
struct ScanShape {
  static constexpr int C = delta_c<T>(), PARTS = sizeof(T) == 2 ? 2 : 1, COLS = 16 * CW * NW;
  static constexpr int PK = pitch_of<T>(KP), PT = pitch_of<T>(C), PV = pitch_of<T>(COLS);
  static constexpr int NT = 64 * NW;
};

template <typename T, int KP, int CW, int NW>
struct ScanLds : ScanShape<T, KP, CW, NW> {
  using B = ScanShape<T, KP, CW, NW>;
  static constexpr int C = B::C;
  static constexpr int K0 = 0, T0 = C * B::PK, V0 = T0 + B::PARTS * C * B::PT,
                       END = V0 + C * B::PV;
  static constexpr int F0 = END * (int)sizeof(T);   // three vectors of floats, e^{G_C}
  static constexpr int ONE = (F0 + (3 * C + 1) * 4 + 15) / 16 * 16;   // one of two buffers
  static constexpr int BYTES = 2 * ONE;
};

// FIRST: the first pass, which has E (and M) and leaves no states of chunks.
template <typename T, int KP, int CW, int NW, bool FIRST>
__global__ __launch_bounds__(64 * NW) void delta_scan_kernel(DeltaParams p) {
  using L = ScanLds<T, KP, CW, NW>;
  constexpr int C = L::C, NT = L::NT, NS = KP / 32, NU = C / 32, COLS = L::COLS;
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  const tops_gla_delta_args& a = p.a;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int g = lane >> 4, ci = lane & 15;
  const int K = (int)a.K, V = (int)a.V, HV = (int)a.HV;
  const int vt = (V + COLS - 1) / COLS, mt = FIRST ? (KP + COLS - 1) / COLS : 0;
  int blk = xcd_remap((int)blockIdx.x, (int)gridDim.x);   // a head's columns on one XCD
  const int vb = blk % (vt + mt);
  blk /= vt + mt;
  const int hv = blk % HV, h = hv / (HV / (int)a.H);
  const SegAt at = seg_at(a, C, blk / HV);
  const bool map = FIRST && vb >= vt;   // columns of M
  if (FIRST && (at.j + 1 >= at.count || (map && at.j == 0))) return;   // nobody asks for these
  const int nc = at.n;
  const T* kp = (const T*)a.k + at.b * a.k_sb + at.t * a.k_st + h * a.k_sh;
  // the block's columns; the last block's few may begin before them, where there are fewer than 8
  const int vc = map ? COLS : V - vb * COLS;
  const T* vp = (const T*)a.v + at.b * a.v_sb + at.t * a.v_st + hv * a.v_sh + (map ? 0 : vb * COLS);
  const int w0 = 16 * CW * wave, v0 = (map ? vb - vt : vb) * COLS + w0 + ci;
  const int width = map ? KP : V;
  const bool idle = v0 - ci >= width;   // a wave past the columns only helps with the tiles

  f32x4 S[CW][2 * NS];
  const float* from = nullptr;
  if (at.j > 0) {
    if (!FIRST) from = p.E + ((long)(at.seg - 1) * HV + hv) * K * V;
  } else if (a.h0) {
    from = a.h0 + ((long)at.seq * HV + hv) * K * V;
  }
#pragma unroll
  for (int c = 0; c < CW; ++c) {
    const int v = v0 + 16 * c;
#pragma unroll
    for (int i = 0; i < 2 * NS; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        S[c][i][r] = map && v == 32 * (i >> 1) + 8 * g + 4 * (i & 1) + r ? 1.f : 0.f;
    if (from && !map) load_state(S[c], from + min(v, V - 1), v < V, g, K, V);
  }

  TileStream<T, C, KP, NT> fk(a.k_st, K, tid);
  TileStream<T, L::PARTS * C, C, NT> ft(C, C, tid);
  TileStream<T, C, COLS, NT> fv(a.v_st, min(vc, V), tid);
  constexpr int NF = (3 * C + NT) / NT;
  float ff[NF], fr[NF];
  auto fetch = [&](int n) {
    const int len = min(C, at.T - n * C);
    const long unit = (long)(at.chunk + n) * HV + hv;
    fk.next(kp + (long)n * C * a.k_st, a.k_st, len, K, tid);
    ft.next((const T*)(p.Tm + unit * (C * C * 4)), C, L::PARTS * C, C, tid);
    if (!map) fv.next(vp + (long)n * C * a.v_st, a.v_st, len, vc, tid);
    const float* vec = delta_vec(p, unit);
#pragma unroll
    for (int i = 0; i < NF; ++i) {   // e^G / |k|, e^{G_C - G} / |k|, beta, e^{G_C}
      const int x = i * NT + tid;
      ff[i] = vec[x < 3 * C ? x : C - 1];
      fr[i] = vec[3 * C + x % C];
    }
  };
  auto put = [&](int n) {
    T* sm = (T*)(smem + (n & 1) * L::ONE);
    const int len = min(C, at.T - n * C);
    fk.put(sm + L::K0, L::PK, len, K, tid);
    ft.put(sm + L::T0, L::PT, L::PARTS * C, C, tid);
    fv.put(sm + L::V0, L::PV, map ? 0 : len, vc, tid);
    float* sf = (float*)(smem + (n & 1) * L::ONE + L::F0);
#pragma unroll
    for (int i = 0; i < NF; ++i)
      if (i * NT + tid <= 3 * C) sf[i * NT + tid] = i * NT + tid < 2 * C ? ff[i] * fr[i] : ff[i];
  };
  if (nc > 0) {
    fetch(0);
    put(0);
  }
  for (int n = 0; n < nc; ++n) {
    __syncthreads();
    if (n + 1 < nc) fetch(n + 1);
    const T* sm = (const T*)(smem + (n & 1) * L::ONE);
    const T *sK = sm + L::K0, *sT = sm + L::T0, *sV = sm + L::V0 + w0;
    const float* sf = (const float*)(smem + (n & 1) * L::ONE + L::F0);
    const long unit = (long)(at.chunk + n) * HV + hv;
    const float last = sf[3 * C];
    if (!idle) {
      f32x4 acc[CW][2 * NU];
#pragma unroll
      for (int c = 0; c < CW; ++c)
#pragma unroll
        for (int i = 0; i < 2 * NU; ++i) acc[c][i] = zero4();
#pragma unroll
      for (int s = 0; s < NS; ++s) {
        Split<T> f[CW];
#pragma unroll
        for (int c = 0; c < CW; ++c) {
          float x[8];
          pair_values(S[c][2 * s], S[c][2 * s + 1], x);
          f[c] = split_of<T>(x);
          if (!FIRST && v0 + 16 * c < V)
            st_frag((T*)p.S + (unit * V + v0 + 16 * c) * KP + 32 * s + 8 * g, high_of(f[c]));
        }
        mma_rows(acc, [&](int i) {
          return ld_frag(sK + (32 * (i >> 1) + pair_row(lane, i & 1)) * L::PK + 32 * s + 8 * g);
        }, f);
      }
      Split<T> R[NU][CW];
#pragma unroll
      for (int u = 0; u < NU; ++u)
#pragma unroll
        for (int c = 0; c < CW; ++c) {
          float x[8], y[8];
          values_of(ld_frag_t(sV + 16 * c + 32 * u * L::PV, L::PV, lane), y);
          pair_values(acc[c][2 * u], acc[c][2 * u + 1], x);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const int t = 32 * u + 8 * g + e;
            x[e] = sf[2 * C + t] * (y[e] - sf[t] * x[e]);
          }
          R[u][c] = split_of<T>(x);
        }
#pragma unroll
      for (int c = 0; c < CW; ++c)
#pragma unroll
        for (int i = 0; i < 2 * NU; ++i) acc[c][i] = zero4();
#pragma unroll
      for (int w = 0; w < NU; ++w)
        mma_split_rows(acc, [&](int i) {
          return ld_split<T>(sT, C * L::PT, (32 * (i >> 1) + pair_row(lane, i & 1)) * L::PT +
                                                32 * w + 8 * g);
        }, [&](int i) { return w <= (i >> 1); }, R[w]);
#pragma unroll
      for (int c = 0; c < CW; ++c)
#pragma unroll
        for (int i = 0; i < 2 * NS; ++i) S[c][i] *= last;
#pragma unroll
      for (int u = 0; u < NU; ++u) {
        Split<T> f[CW];
#pragma unroll
        for (int c = 0; c < CW; ++c) {
          float x[8];
          pair_values(acc[c][2 * u], acc[c][2 * u + 1], x);
          if (!FIRST && v0 + 16 * c < V)
            st_frag((T*)p.N + (unit * V + v0 + 16 * c) * C + 32 * u + 8 * g, frag_of<T>(x));
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] *= sf[C + 32 * u + 8 * g + e];
          f[c] = split_of<T>(x);
        }
        mma_rows(S, [&](int i) {
          return ld_pair_t(sK + 32 * u * L::PK + 32 * (i >> 1), L::PK, lane, i & 1);
        }, f);
      }
    }
    if (n + 1 < nc) put(n + 1);
  }
  if (idle) return;
#pragma unroll
  for (int c = 0; c < CW; ++c) {
    const int v = v0 + 16 * c;
    if (map) {   // [KP][KP]: column v, rows in the lane's order
      const long tile = (long)KP * KP;
      T* M = (T*)(p.M + ((long)at.seg * HV + hv) * tile * 4);
      T* Mt = (T*)(p.Mt + ((long)at.seg * HV + hv) * tile * 4);
#pragma unroll
      for (int s = 0; s < NS; ++s) {
        float x[8], y[8];
        pair_values(S[c][2 * s], S[c][2 * s + 1], x);
        const Split<T> f = split_of<T>(x);
        if (a.train) st_frag(Mt + v * KP + 32 * s + 8 * g, high_of(f));
        values_of(high_of(f), y);
#pragma unroll
        for (int e = 0; e < 8; ++e) M[(32 * s + 8 * g + e) * KP + v] = from_f32<T>(y[e]);
        if constexpr (sizeof(T) == 2) {
          if (a.train) st_frag(Mt + tile + v * KP + 32 * s + 8 * g, f.lo);
          values_of(f.lo, y);
#pragma unroll
          for (int e = 0; e < 8; ++e) M[tile + (32 * s + 8 * g + e) * KP + v] = from_f32<T>(y[e]);
        }
      }
    } else if (FIRST) {
      store_state(S[c], p.E + ((long)at.seg * HV + hv) * K * V + v, v < V, g, K, V);
    } else if (a.ht && at.j + 1 == at.count) {
      store_state(S[c], a.ht + ((long)at.seq * HV + hv) * K * V + v, v < V, g, K, V);
    }
  }
}

template <typename T, int KP, int CW, int NW>
struct DscanLds : ScanShape<T, KP, CW, NW> {
  using B = ScanShape<T, KP, CW, NW>;
  static constexpr int C = B::C;
  static constexpr int K0 = 0, Q0 = C * B::PK, T0 = 2 * C * B::PK, P0 = T0 + B::PARTS * C * B::PT;
  static constexpr int V0 = P0 + B::PARTS * C * B::PT, END = V0 + C * B::PV;
  static constexpr int F0 = END * (int)sizeof(T);   // three vectors of floats, e^{G_C}
  static constexpr int BYTES = F0 + (3 * C + 1) * 4;
};

template <typename T, int KP, int CW, int NW, bool FIRST>
__global__ __launch_bounds__(64 * NW) void delta_dscan_kernel(DeltaParams p) {
  using L = DscanLds<T, KP, CW, NW>;
  constexpr int C = L::C, NT = L::NT, NS = KP / 32, NU = C / 32, COLS = L::COLS, LO = C * L::PT;
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  const tops_gla_delta_args& a = p.a;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int g = lane >> 4, ci = lane & 15;
  const int K = (int)a.K, V = (int)a.V, HV = (int)a.HV;
  const int vt = (V + COLS - 1) / COLS;
  int blk = xcd_remap((int)blockIdx.x, (int)gridDim.x);
  const int vb = blk % vt;
  blk /= vt;
  const int hv = blk % HV, h = hv / (HV / (int)a.H);
  const SegAt at = seg_at(a, C, blk / HV);
  if (FIRST && at.j == 0) return;
  const int nc = at.n;
  const T* kp = (const T*)a.k + at.b * a.k_sb + at.t * a.k_st + h * a.k_sh;
  const T* qp = (const T*)a.q + at.b * a.q_sb + at.t * a.q_st + h * a.q_sh;
  const int vc = V - vb * COLS;
  const T* dp = (const T*)a.dout + at.b * a.do_sb + at.t * a.do_st + hv * a.do_sh + vb * COLS;
  const int w0 = 16 * CW * wave, v0 = vb * COLS + w0 + ci;
  const bool idle = v0 - ci >= V;

  f32x4 S[CW][2 * NS];   // dS, as the forward's states
  const float* from = nullptr;
  if (at.j + 1 < at.count) {
    if (!FIRST) from = p.dE + ((long)(at.seg + 1) * HV + hv) * K * V;
  } else if (a.dht) {
    from = a.dht + ((long)at.seq * HV + hv) * K * V;
  }
#pragma unroll
  for (int c = 0; c < CW; ++c) {
#pragma unroll
    for (int i = 0; i < 2 * NS; ++i) S[c][i] = zero4();
    if (from) load_state(S[c], from + min(v0 + 16 * c, V - 1), v0 + 16 * c < V, g, K, V);
  }

  TileStream<T, C, KP, NT> fk(a.k_st, K, tid), fq(a.q_st, K, tid);
  TileStream<T, L::PARTS * C, C, NT> ft(C, C, tid);
  TileStream<T, C, C, NT> fp[2] = {{C, C, tid}, {C, C, tid}};
  TileStream<T, C, COLS, NT> fd(a.do_st, vc, tid);
  constexpr int NF = (3 * C + NT) / NT;
  float ff[NF], fr[NF];
  auto fetch = [&](int n) {
    const int len = min(C, at.T - n * C);
    const long unit = (long)(at.chunk + n) * HV + hv;
    fk.next(kp + (long)n * C * a.k_st, a.k_st, len, K, tid);
    fq.next(qp + (long)n * C * a.q_st, a.q_st, len, K, tid);
    ft.next((const T*)(p.Tm + unit * (C * C * 4)), C, L::PARTS * C, C, tid);
#pragma unroll
    for (int i = 0; i < L::PARTS; ++i)   // rows past the end have not been written
      fp[i].next((const T*)(p.P + unit * (C * C * 4)) + i * C * C, C, len, C, tid);
    fd.next(dp + (long)n * C * a.do_st, a.do_st, len, vc, tid);
    const float* vec = delta_vec(p, unit);
#pragma unroll
    for (int i = 0; i < NF; ++i) {   // e^{G_C - G} / |k|, beta e^G / |k|, scale e^G / |q|
      const int x = i * NT + tid, t = x % C;
      const float e = vec[t + (x < C ? C : 0)], r = vec[t + (x < 2 * C ? 3 * C : 4 * C)];
      ff[i] = x < 3 * C ? e * r : vec[C - 1];
      fr[i] = x < C ? 1.f : x < 2 * C ? vec[2 * C + t] : x < 3 * C ? (float)a.scale : 1.f;
    }
  };
  T* sm = (T*)smem;
  T *sK = sm + L::K0, *sQ = sm + L::Q0, *sT = sm + L::T0, *sP = sm + L::P0, *sV = sm + L::V0;
  float* sf = (float*)(smem + L::F0);
  if (nc > 0) fetch(nc - 1);
  for (int n = nc - 1; n >= 0; --n) {
    __syncthreads();
    const int len = min(C, at.T - n * C);
    fk.put(sK, L::PK, len, K, tid);
    fq.put(sQ, L::PK, len, K, tid);
    ft.put(sT, L::PT, L::PARTS * C, C, tid);
#pragma unroll
    for (int i = 0; i < L::PARTS; ++i) fp[i].put(sP + i * LO, L::PT, len, C, tid);
    fd.put(sV, L::PV, len, vc, tid);
#pragma unroll
    for (int i = 0; i < NF; ++i)
      if (i * NT + tid <= 3 * C) sf[i * NT + tid] = ff[i] * fr[i];
    __syncthreads();
    if (n > 0) fetch(n - 1);
    if (idle) continue;
    const long unit = (long)(at.chunk + n) * HV + hv;
    const float last = sf[3 * C];

    f32x4 acc[CW][2 * NU];
#pragma unroll
    for (int c = 0; c < CW; ++c)
#pragma unroll
      for (int i = 0; i < 2 * NU; ++i) acc[c][i] = zero4();
#pragma unroll
    for (int s = 0; s < NS; ++s) {
      Split<T> f[CW];
#pragma unroll
      for (int c = 0; c < CW; ++c) {
        float x[8];
        pair_values(S[c][2 * s], S[c][2 * s + 1], x);
        f[c] = split_of<T>(x);
        if (!FIRST && v0 + 16 * c < V)
          st_frag((T*)p.dS + (unit * V + v0 + 16 * c) * KP + 32 * s + 8 * g, high_of(f[c]));
      }
      mma_rows(acc, [&](int i) {
        return ld_frag(sK + (32 * (i >> 1) + pair_row(lane, i & 1)) * L::PK + 32 * s + 8 * g);
      }, f);
    }
    Frag<T> df[NU][CW];
#pragma unroll
    for (int u = 0; u < NU; ++u)
#pragma unroll
      for (int c = 0; c < CW; ++c)
        df[u][c] = ld_frag_t(sV + w0 + 16 * c + 32 * u * L::PV, L::PV, lane);
#pragma unroll
    for (int i = 0; i < 2 * NU; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float d = sf[32 * (i >> 1) + 8 * g + 4 * (i & 1) + r];
#pragma unroll
        for (int c = 0; c < CW; ++c) acc[c][i][r] *= d;
      }
#pragma unroll
    for (int w = 0; w < NU; ++w)
#pragma unroll
      for (int i = 0; i < 2 * NU; ++i)
        if (w >= (i >> 1)) {
          const Split<T> f =
              ld_split_t<T>(sP + 32 * w * L::PT + 32 * (i >> 1), LO, L::PT, lane, i & 1);
#pragma unroll
          for (int c = 0; c < CW; ++c) mma(acc[c][i], f, df[w][c]);
        }
    Split<T> R[NU][CW];
#pragma unroll
    for (int u = 0; u < NU; ++u)
#pragma unroll
      for (int c = 0; c < CW; ++c) {
        float x[8];
        pair_values(acc[c][2 * u], acc[c][2 * u + 1], x);
        R[u][c] = split_of<T>(x);
      }
#pragma unroll
    for (int c = 0; c < CW; ++c)
#pragma unroll
      for (int i = 0; i < 2 * NU; ++i) acc[c][i] = zero4();
#pragma unroll
    for (int w = 0; w < NU; ++w)
      mma_split_rows(acc, [&](int i) {
        return ld_split_t<T>(sT + 32 * w * L::PT + 32 * (i >> 1), LO, L::PT, lane, i & 1);
      }, [&](int i) { return w >= (i >> 1); }, R[w]);
#pragma unroll
    for (int c = 0; c < CW; ++c)
#pragma unroll
      for (int i = 0; i < 2 * NS; ++i) S[c][i] *= last;
#pragma unroll
    for (int u = 0; u < NU; ++u) {
      Split<T> fo[CW], fy[CW];
#pragma unroll
      for (int c = 0; c < CW; ++c) {
        float x[8];
        values_of(df[u][c], x);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] *= sf[2 * C + 32 * u + 8 * g + e];
        fo[c] = split_of<T>(x);
        pair_values(acc[c][2 * u], acc[c][2 * u + 1], x);
        if (!FIRST && v0 + 16 * c < V)
          st_frag((T*)p.Y + (unit * V + v0 + 16 * c) * C + 32 * u + 8 * g, frag_of<T>(x));
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] *= -sf[C + 32 * u + 8 * g + e];
        fy[c] = split_of<T>(x);
      }
      mma_rows(S, [&](int i) {
        return ld_pair_t(sQ + 32 * u * L::PK + 32 * (i >> 1), L::PK, lane, i & 1);
      }, fo);
      mma_rows(S, [&](int i) {
        return ld_pair_t(sK + 32 * u * L::PK + 32 * (i >> 1), L::PK, lane, i & 1);
      }, fy);
    }
  }
  if (idle) return;
  float* to = FIRST ? p.dE + ((long)at.seg * HV + hv) * K * V
              : a.dh0 && at.j == 0 ? a.dh0 + ((long)at.seq * HV + hv) * K * V : nullptr;
#pragma unroll
  for (int c = 0; c < CW; ++c)
    if (to) store_state(S[c], to + v0 + 16 * c, v0 + 16 * c < V, g, K, V);
}

// E_j <- M_j E_{j-1} + E_j along the segments of a sequence and head, or dE_j <- M_j^T dE_{j+1} +
// dE_j the other way. A block has 16 columns, each of its waves KP / 4 or KP / 2 of the rows; the
// states go from wave to wave through LDS as operands, the maps and parts of the next segment are
// on their way meanwhile.
template <typename T, int KP, bool BACK>
__global__ __launch_bounds__(KP == 64 ? 128 : 256) void delta_fold_kernel(DeltaParams p) {
  constexpr int NS = KP / 32, NW = KP == 64 ? 2 : 4, NR = NS / NW, PARTS = sizeof(T) == 2 ? 2 : 1;
  __shared__ __attribute__((aligned(16))) Frag<T> sh[2][PARTS][NS][64];
  const tops_gla_delta_args& a = p.a;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4;
  const int K = (int)a.K, V = (int)a.V, HV = (int)a.HV;
  const int vt = (V + 15) / 16;
  int blk = xcd_remap((int)blockIdx.x, (int)gridDim.x);
  const int v = blk % vt * 16 + (lane & 15);
  blk /= vt;
  const int hv = blk % HV, seq = blk / HV;
  int first, count;
  if (a.seqs) {
    const int* f = a.seqs + 2 * (a.nseq + 1) + seq;
    first = f[0];
    count = f[1] - f[0];
  } else {
    count = (int)(a.nsegs / a.nseq);
    first = seq * count;
  }
  if (count < 3) return;   // the first segment to run is where it should be
  const long tile = (long)KP * KP;
  const int k0 = wave * NR * 32;   // the wave's rows: k0 + 32 s + 8 g + 4 h + r as ever
  auto state = [&](int n) {
    const int j = BACK ? count - 1 - n : n;
    return (BACK ? p.dE : p.E) + ((long)(first + j) * HV + hv) * K * V;
  };
  Split<T> M[2 * NR][NS];
  f32x4 E[2 * NR];
  auto fetch = [&](int n) {
    const int j = BACK ? count - 1 - n : n;
    const T* m = (const T*)((BACK ? p.Mt : p.M) + ((long)(first + j) * HV + hv) * tile * 4);
#pragma unroll
    for (int i = 0; i < 2 * NR; ++i)
#pragma unroll
      for (int s = 0; s < NS; ++s)
        M[i][s] = ld_split<T>(m, (int)tile, (k0 + 32 * (i >> 1) + pair_row(lane, i & 1)) * KP +
                                                32 * s + 8 * g);
    load_rows(E, state(n) + min(v, V - 1), k0 + 8 * g, K, V);
  };
  auto share = [&](int n) {   // the wave's rows of the state after step n, and to memory
#pragma unroll
    for (int s = 0; s < NR; ++s) {
      float x[8];
#pragma unroll
      for (int e = 0; e < 8; ++e)
        x[e] = v < V && k0 + 32 * s + 8 * g + e < K ? E[2 * s + e / 4][e % 4] : 0.f;
      const Split<T> f = split_of<T>(x);
      sh[n & 1][0][wave * NR + s][lane] = high_of(f);
      if constexpr (PARTS == 2) sh[n & 1][1][wave * NR + s][lane] = f.lo;
    }
    if (n > 0 && v < V) store_rows(E, state(n) + v, k0 + 8 * g, K, V);
  };
  load_rows(E, state(0) + min(v, V - 1), k0 + 8 * g, K, V);
  share(0);
  fetch(1);
  for (int n = 1; n + 1 < count; ++n) {
    __syncthreads();
    f32x4 acc[2 * NR];
#pragma unroll
    for (int i = 0; i < 2 * NR; ++i) acc[i] = E[i];
#pragma unroll
    for (int s = 0; s < NS; ++s) {
      Split<T> f;
      if constexpr (PARTS == 2)
        f = {sh[(n - 1) & 1][0][s][lane], sh[(n - 1) & 1][1][s][lane]};
      else
        f = {sh[(n - 1) & 1][0][s][lane]};
#pragma unroll
      for (int i = 0; i < 2 * NR; ++i) mma(acc[i], M[i][s], f);
    }
#pragma unroll
    for (int i = 0; i < 2 * NR; ++i) E[i] = acc[i];
    share(n);
    if (n + 2 < count) fetch(n + 1);
  }
}

template <typename T, int KP, int CW, int NW, bool BACK, bool FIRST>
hipError_t launch(const DeltaParams& p, hipStream_t st) {
  using S = ScanShape<T, KP, CW, NW>;
  constexpr int lds = BACK ? (int)DscanLds<T, KP, CW, NW>::BYTES : (int)ScanLds<T, KP, CW, NW>::BYTES;
  const void* f;
  if constexpr (BACK)
    f = (const void*)delta_dscan_kernel<T, KP, CW, NW, FIRST>;
  else
    f = (const void*)delta_scan_kernel<T, KP, CW, NW, FIRST>;
  const hipError_t e = hipFuncSetAttribute(f, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
  if (e != hipSuccess) return e;
  const long cols = (p.a.V + S::COLS - 1) / S::COLS +
                    (FIRST && !BACK ? (KP + S::COLS - 1) / S::COLS : 0);
  const unsigned grid = (unsigned)(cols * p.a.HV * p.a.nsegs);
  if constexpr (BACK)
    delta_dscan_kernel<T, KP, CW, NW, FIRST><<<grid, S::NT, lds, st>>>(p);
  else
    delta_scan_kernel<T, KP, CW, NW, FIRST><<<grid, S::NT, lds, st>>>(p);
  return hipGetLastError();
}

template <typename T, int KP, int CW, int NW, bool BACK>
hipError_t passes(const DeltaParams& p, hipStream_t st) {
  if (p.multi) {
    if (const hipError_t e = launch<T, KP, CW, NW, BACK, true>(p, st)) return e;
    const unsigned grid = (unsigned)((p.a.V + 15) / 16 * p.a.HV * p.a.nseq);
    delta_fold_kernel<T, KP, BACK><<<grid, KP == 64 ? 128 : 256, 0, st>>>(p);
    if (const hipError_t e = hipGetLastError()) return e;
  }
  return launch<T, KP, CW, NW, BACK, false>(p, st);
}

template <typename T, int KP, bool BACK>
hipError_t run(const DeltaParams& p, hipStream_t st) {
  // two lots of 16 columns a wave read each of the chunk's tiles once for both; with 256 keys their
  // states do not fit the registers
  if constexpr (KP < 256)
    if (p.a.V > 64) return passes<T, KP, 1, 8, BACK>(p, st);
  return passes<T, KP, 1, 4, BACK>(p, st);
}
template <typename T, int KP>
hipError_t run(const DeltaParams& p, bool back, hipStream_t st) {
  return back ? run<T, KP, true>(p, st) : run<T, KP, false>(p, st);
}

}  // namespace

hipError_t run_delta_scan(const DeltaParams& p, bool back, hipStream_t st) {
  if (p.a.dtype == DT_BF16)
    return p.KP == 64 ? run<bf16, 64>(p, back, st) : p.KP == 128 ? run<bf16, 128>(p, back, st)
                                                                 : run<bf16, 256>(p, back, st);
  return p.KP == 64 ? run<float, 64>(p, back, st) : p.KP == 128 ? run<float, 128>(p, back, st)
                                                                : run<float, 256>(p, back, st);
}

}  // namespace tops
